// Short causal convolution of each channel over packed or rectangular batches of sequences, with the K - 1 inputs before the first
// step as its state:  pre_t = bias + sum_k w_k x_{t-K+1+k},  y = pre or pre sigmoid(pre).
//   backward: dpre = dy act'(pre);  dx_t = sum_k w_k dpre_{t+K-1-k};  dw_k = sum_t dpre_t x_{t-K+1+k};  db = sum_t dpre_t
// HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx.  A wave takes a run of steps of a sequence with the
// window in registers, VEC channels a lane; its neighbours' K - 1 rows come from the L2.
#include "ppk_seq_rows.h"

namespace ppk {

namespace {
// a block: 256 columns of a chunk of PS_ROWS rows
__global__ __launch_bounds__(256) void k_ps_part(const float* __restrict__ part, long long P, long long C, unsigned column_blocks, double* __restrict__ out)
{
    const unsigned chunk = blockIdx.x / column_blocks;
    const long long c = (long long)(blockIdx.x - chunk * column_blocks) * 256 + threadIdx.x;
    if (c >= C) return;
    const long long p0 = (long long)chunk * PS_ROWS, p1 = p0 + PS_ROWS < P ? p0 + PS_ROWS : P;
    double s = 0;
    long long p = p0;
    for (; p + 8 <= p1; p += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = part[(p + k) * C + c];
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)v[k];
    }
    for (; p < p1; ++p) s += (double)part[p * C + c];
    out[(long long)chunk * C + c] = s;
}
__global__ __launch_bounds__(256) void k_ps_final(const double* __restrict__ part, int n, long long C, float* __restrict__ out)
{
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    double s = 0;
    for (int p = 0; p < n; ++p) s += part[p * C + c];
    out[c] = (float)s;
}
struct SumJobs { SumJob job[3]; int n; };
// up to ONE_PASS_ROWS rows: 64 columns a block, 16 interleaved slices of the rows, joined in order.  One launch for all of a call's sums.
__global__ __launch_bounds__(1024) void k_ps_one(SumJobs jobs)
{
    __shared__ double red[16][64];
    const SumJob j = jobs.job[blockIdx.y];
    const long long c0 = (long long)blockIdx.x * 64;
    if (c0 >= j.C) return;
    const int col = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const long long c = c0 + col;
    double s = 0;
    if (c < j.C) {
        long long p = slice;
        for (; p + 7 * 16 < j.P; p += 8 * 16) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = j.part[(p + k * 16) * j.C + c];
#pragma unroll
            for (int k = 0; k < 8; ++k) s += (double)v[k];
        }
        for (; p < j.P; p += 16) s += (double)j.part[p * j.C + c];
    }
    red[slice][col] = s;
    __syncthreads();
    if (slice || c >= j.C) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][col];
    if (!j.taps) { j.out[c] = (float)s; return; }
    const long long d = j.C / (j.taps + 1), k = c / d;        // rows of [taps + 1, D]: a weight's gradient [D, taps], then the bias'
    if (k < j.taps) j.out[(c - k * d) * j.taps + k] = (float)s;
    else if (j.out2) j.out2[c - k * d] = (float)s;
}
}  // namespace

size_t partial_sum_ws_bytes(long long P, long long C) { return P > ONE_PASS_ROWS ? ppk_align_up((size_t)((P + PS_ROWS - 1) / PS_ROWS) * (size_t)C * 8, 256) : 0; }
int partial_sums(const SumJob* jobs, int count, void* ws, hipStream_t stream)
{
    SumJobs small = {};
    long long widest = 0;
    for (int k = 0; k < count; ++k) {
        const SumJob& j = jobs[k];
        if (j.C <= 0 || !j.out) continue;
        if (j.P <= ONE_PASS_ROWS) { small.job[small.n++] = j; widest = j.C > widest ? j.C : widest; continue; }
        const unsigned cb = (unsigned)((j.C + 255) / 256), chunks = (unsigned)((j.P + PS_ROWS - 1) / PS_ROWS);
        k_ps_part<<<cb * chunks, 256, 0, stream>>>(j.part, j.P, j.C, cb, (double*)ws);
        k_ps_final<<<cb, 256, 0, stream>>>((const double*)ws, (int)chunks, j.C, j.out);
    }
    if (small.n) k_ps_one<<<dim3((unsigned)((widest + 63) / 64), (unsigned)small.n), 1024, 0, stream>>>(small);
    PPK_CHECK_LAUNCH("partial_sums");
    return PPK_OK;
}

}  // namespace ppk

namespace {

using ppk::SeqBatch;
using ppk::Stride;
using ppk::at;
using ppk::Rows;
using ppk::uni_len;
using ppk::uniform;

constexpr int AHEAD = 4;                      // steps whose elements are loaded before those of the steps before them are used
// Blocks of a backward launch in all, three a CU, what is resident together: each leaves a row of partial sums for its channels.  2048 x 20-100 x 512
// fp32: 195 us, 199 with 1024, 258 with 2048 and shorter runs.  Whole training passes with 384, 768 and 1536: the same batch fp32 337, 315, 315 us,
// bf16 231, 180, 178; 1 x 16384 x 4096 bf16 202, 203, 187; 64 x 256 x 1001 fp32, 3 taps, 165, 163, 162.
constexpr int SUM_BLOCKS = 768;
static_assert(SUM_BLOCKS <= ppk::ONE_PASS_ROWS, "one launch adds them");
constexpr long long WANTED_WAVES = 8192;       // 16384 and half the run: the same, 32768: 5 % (fp32 batch) to 45 % (bf16 prompt) slower

struct ConvArgs {
    SeqBatch q;
    int D, K, run, runs;                      // steps of a run, and runs of the longest sequence
    const void *x, *state, *dy, *dlast;
    const float *weight, *bias;
    void *y, *last, *dx, *dstate;
    float* part;                              // [blocks, K + 1, D]
    Stride xs, ys, dys;                       // ys: of y or dx
    int silu;
};

// VEC elements as one access of VEC * sizeof(T) bytes
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Vec { T v[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ void widen(const Vec<T, VEC>& p, float (&v)[VEC])
{
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = to_f32(p.v[e]);
}
template <typename T, int VEC> __device__ __forceinline__ Vec<T, VEC> narrow(const float (&v)[VEC])
{
    Vec<T, VEC> p;
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.v[e] = from_f32<T>(v[e]);
    return p;
}
template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) { widen<T, VEC>(*reinterpret_cast<const Vec<T, VEC>*>(p), v); }
template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) { *reinterpret_cast<Vec<T, VEC>*>(p) = narrow<T, VEC>(v); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// A wave's (CL == 64) or a row of 16 lanes' run of a sequence.  Runs at the same steps of sequences next to each other are worked on
// together: their rows are next to each other in a packed batch.
template <int CL> struct Run {
    long long b, t0, t1, len;
    bool any;
    __device__ __forceinline__ Run(const ConvArgs& a, long long item)
    {
        if (CL == 64) item = ((long long)__builtin_amdgcn_readfirstlane((int)(item >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)item);
        const long long k = item / a.q.B;
        b = item - k * a.q.B;
        any = k < a.runs;
        t0 = k * a.run;
        len = !any ? 0 : CL == 64 ? uni_len(a.q, b) : a.q.length(b);
        if (t0 >= len && t0 > 0) any = false;
        t1 = t0 + a.run < len ? t0 + a.run : len;
    }
};
template <int CL> __device__ __forceinline__ unsigned row_of(const SeqBatch& q, long long t) { return CL == 64 ? ppk::uni_row(q, t) : (unsigned)q.row(t); }

// the input of step t >= -(K - 1), which is of the state before the first step
template <typename T, int VEC, int K, int CL>
__device__ __forceinline__ void input_at(const ConvArgs& a, const Rows<T>& xs, long long t, long long b, int c, float (&v)[VEC])
{
    if (t >= 0) { widen<T, VEC>(xs.template get_as<Vec<T, VEC>>(row_of<CL>(a.q, t), c * (unsigned)sizeof(T)), v); return; }
    if (a.state) { load_vec<T, VEC>((const T*)a.state + (b * (K - 1) + t + K - 1) * a.D + c, v); return; }
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.f;
}
template <int VEC, int K> __device__ __forceinline__ void load_taps(const ConvArgs& a, int c, float (&w)[K][VEC], float (&bias)[VEC])
{
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        bias[e] = a.bias ? a.bias[c + e] : 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) w[j][e] = a.weight[(long long)(c + e) * K + j];
    }
}

// block 256 = 256 / CL runs x CL lanes of VEC channels.  Compiled for each K: more taps with weights of zero would multiply inputs that the
// operator does not reach, and 0 times an infinity is NaN.
template <typename T, int VEC, int K, int CL>
__global__ __launch_bounds__(256) void k_conv_fwd(ConvArgs a, int channel_blocks)
{
    const int c = ((int)(blockIdx.x % channel_blocks) * CL + threadIdx.x % CL) * VEC;
    const Run<CL> run(a, (long long)(blockIdx.x / channel_blocks) * (256 / CL) + threadIdx.x / CL);
    if (c >= a.D || !run.any) return;
    const long long b = run.b, t0 = run.t0, t1 = run.t1;
    const Rows<T> xs(a.x, b * a.xs.b, a.xs.t), ys(a.y, b * a.ys.b, a.ys.t);
    const unsigned cb = c * (unsigned)sizeof(T);
    Vec<T, VEC> next[AHEAD];
    unsigned rows[AHEAD], r[AHEAD];
    const auto fetch = [&](long long t) {                    // behind the last step, that one again
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) rows[i] = row_of<CL>(a.q, t + i < t1 ? t + i : t1 - 1);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) next[i] = xs.template get_as<Vec<T, VEC>>(rows[i], cb);
    };
    if (t0 < t1) fetch(t0);
    float w[K][VEC], bias[VEC], win[K][VEC];
    load_taps<VEC, K>(a, c, w, bias);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) input_at<T, VEC, K, CL>(a, xs, t0 - (K - 1) + j, b, c, win[j]);
    for (long long t = t0; t < t1; t += AHEAD) {
        float x[AHEAD][VEC];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) { widen<T, VEC>(next[i], x[i]); r[i] = rows[i]; }
        if (t + AHEAD < t1) fetch(t + AHEAD);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (t + i >= t1) break;
            float out[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                win[K - 1][e] = x[i][e];
                float s = bias[e];
#pragma unroll
                for (int j = 0; j < K; ++j) s = fmaf(w[j][e], win[j][e], s);
                out[e] = a.silu ? s * sigmoid(s) : s;
#pragma unroll
                for (int j = 0; j < K - 1; ++j) win[j][e] = win[j + 1][e];
            }
            ys.template put_as<Vec<T, VEC>>(r[i], cb, narrow<T, VEC>(out));
        }
    }
    if (t1 == run.len && a.last)
#pragma unroll
        for (int j = 0; j < K - 1; ++j) store_vec<T, VEC>((T*)a.last + (b * (K - 1) + j) * a.D + c, win[j]);
}

template <typename T, int VEC, int K, int CL>
__global__ __launch_bounds__(256) void k_conv_bwd(ConvArgs a, int channel_blocks)
{
    constexpr int IL = 256 / CL;
    __shared__ float red[IL][CL][VEC];
    const int cl = threadIdx.x % CL, il = threadIdx.x / CL, c = ((int)(blockIdx.x % channel_blocks) * CL + cl) * VEC;
    const long long first_block = blockIdx.x / channel_blocks, blocks = gridDim.x / channel_blocks;
    const unsigned cb = c * (unsigned)sizeof(T);
    float dw[K][VEC] = {}, db[VEC] = {};
    if (c < a.D) {
        float w[K][VEC], bias[VEC];
        load_taps<VEC, K>(a, c, w, bias);
        const long long items = a.q.B * a.runs;
        for (long long item = first_block * IL + il; item < items; item += blocks * IL) {
            const Run<CL> run(a, item);
            if (!run.any) continue;
            const long long b = run.b, t0 = run.t0, t1 = run.t1, len = run.len, first = t0 == 0 ? -(long long)(K - 1) : t0;
            const Rows<T> xs(a.x, b * a.xs.b, a.xs.t), dys(a.dy, b * a.dys.b, a.dys.t), dxs(a.dx, b * a.ys.b, a.ys.t);
            Vec<T, VEC> nx[AHEAD], nd[AHEAD];
            const auto fetch = [&](long long t) {            // behind the sequence's last step, that one again
                unsigned rows[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) rows[i] = row_of<CL>(a.q, t + i < len ? t + i : len - 1);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) { nx[i] = xs.template get_as<Vec<T, VEC>>(rows[i], cb); nd[i] = dys.template get_as<Vec<T, VEC>>(rows[i], cb); }
            };
            if (len > 0) fetch(t0);
            float win[K][VEC], dp[K][VEC];                   // inputs t - K + 1 .. t; dp[j] = dpre of step t - j
#pragma unroll
            for (int j = 0; j < K - 1; ++j) input_at<T, VEC, K, CL>(a, xs, t0 - (K - 1) + j, b, c, win[j]);
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) dp[j][e] = 0.f;
            const long long te = t1 + K - 1;
            for (long long tg = t0; tg < te; tg += AHEAD) {
                float x[AHEAD][VEC], dy[AHEAD][VEC];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) { widen<T, VEC>(nx[i], x[i]); widen<T, VEC>(nd[i], dy[i]); }
                if (tg + AHEAD < te && len > 0) fetch(tg + AHEAD);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const long long t = tg + i;
                    if (t >= te) break;
#pragma unroll
                    for (int j = K - 1; j > 0; --j)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) dp[j][e] = dp[j - 1][e];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) dp[0][e] = 0.f;
                    if (t < len) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            win[K - 1][e] = x[i][e];
                            float s = bias[e], d = dy[i][e];
#pragma unroll
                            for (int j = 0; j < K; ++j) s = fmaf(w[j][e], win[j][e], s);
                            if (a.silu) { const float g = sigmoid(s); d *= g * fmaf(s, 1.0f - g, 1.0f); }
                            dp[0][e] = d;
                            if (t < t1) {
                                db[e] += d;
#pragma unroll
                                for (int j = 0; j < K; ++j) dw[j][e] = fmaf(d, win[j][e], dw[j][e]);
                            }
#pragma unroll
                            for (int j = 0; j < K - 1; ++j) win[j][e] = win[j + 1][e];
                        }
                    }
                    const long long tt = t - (K - 1);        // the step whose input's gradient is complete
                    if (tt < first || tt >= t1) continue;
                    float dx[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        dx[e] = 0.f;
#pragma unroll
                        for (int j = 0; j < K; ++j) dx[e] = fmaf(w[j][e], dp[j][e], dx[e]);
                    }
                    const long long k = tt - (len - (K - 1));
                    if (k >= 0 && a.dlast) {                 // the last K - 1 inputs are the new state too
                        float g[VEC];
                        load_vec<T, VEC>((const T*)a.dlast + (b * (K - 1) + k) * a.D + c, g);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) dx[e] += g[e];
                    }
                    if (tt >= 0) dxs.template put_as<Vec<T, VEC>>(row_of<CL>(a.q, tt), cb, narrow<T, VEC>(dx));
                    else if (a.dstate) store_vec<T, VEC>((T*)a.dstate + (b * (K - 1) + tt + K - 1) * a.D + c, dx);
                }
            }
        }
    }
    // the items of a block, in order, one column of the partial sums at a time
#pragma unroll
    for (int j = 0; j <= K; ++j) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) red[il][cl][e] = j < K ? dw[j < K ? j : 0][e] : db[e];
        __syncthreads();
        if (il == 0 && c < a.D) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float s = red[0][cl][e];
                for (int i = 1; i < IL; ++i) s += red[i][cl][e];
                a.part[(first_block * (K + 1) + j) * a.D + c + e] = s;
            }
        }
    }
}

template <typename T, int KP>
__global__ __launch_bounds__(256) void k_conv_step(long long B, int D, int K, const T* __restrict__ x, long long ldx, const T* state,
                                                   const float* __restrict__ weight, const float* __restrict__ bias, int silu, T* __restrict__ y, T* next)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= B * D) return;
    const long long b = e / D;
    const int d = (int)(e % D);
    T in[KP];                                  // all of a channel's state is read before any of it is written: next may be the state itself
#pragma unroll
    for (int j = 0; j < KP - 1; ++j)
        if (j >= KP - K) in[j] = state[(b * (K - 1) + j - (KP - K)) * D + d];
    in[KP - 1] = x[b * ldx + d];
    float s = bias ? bias[d] : 0.f;
#pragma unroll
    for (int j = 0; j < KP; ++j)
        if (j >= KP - K) s = fmaf(weight[(long long)d * K + j - (KP - K)], to_f32(in[j]), s);
    y[e] = from_f32<T>(silu ? s * sigmoid(s) : s);
#pragma unroll
    for (int j = 0; j < KP - 1; ++j)
        if (j >= KP - K) next[(b * (K - 1) + j - (KP - K)) * D + d] = in[j + 1];
}

int taps(long long K) { return K <= 2 ? 2 : K <= 4 ? 4 : 8; }

template <typename T, int VEC, int K, int CL> void launch_conv(const ConvArgs& a, bool bwd, unsigned blocks, hipStream_t st)
{
    const int cb = (a.D + CL * VEC - 1) / (CL * VEC);
    if (bwd) k_conv_bwd<T, VEC, K, CL><<<blocks * (unsigned)cb, 256, 0, st>>>(a, cb);
    else k_conv_fwd<T, VEC, K, CL><<<blocks * (unsigned)cb, 256, 0, st>>>(a, cb);
}
template <typename T, int VEC, int K> void launch_conv(const ConvArgs& a, bool bwd, int cl, unsigned blocks, hipStream_t st)
{
    if (cl == 16) launch_conv<T, VEC, K, 16>(a, bwd, blocks, st);
    else launch_conv<T, VEC, K, 64>(a, bwd, blocks, st);
}
template <typename T, int VEC> void launch_conv(const ConvArgs& a, bool bwd, int cl, unsigned blocks, hipStream_t st)
{
    switch (a.K) {
        case 1: launch_conv<T, VEC, 1>(a, bwd, cl, blocks, st); break;
        case 2: launch_conv<T, VEC, 2>(a, bwd, cl, blocks, st); break;
        case 3: launch_conv<T, VEC, 3>(a, bwd, cl, blocks, st); break;
        case 4: launch_conv<T, VEC, 4>(a, bwd, cl, blocks, st); break;
        case 5: launch_conv<T, VEC, 5>(a, bwd, cl, blocks, st); break;
        case 6: launch_conv<T, VEC, 6>(a, bwd, cl, blocks, st); break;
        case 7: launch_conv<T, VEC, 7>(a, bwd, cl, blocks, st); break;
        default: launch_conv<T, VEC, 8>(a, bwd, cl, blocks, st);
    }
}
constexpr int WIDE = 4;                       // channels of a lane where they can be loaded together: 16 bytes in fp32, 8 in bf16

// accesses of WIDE elements where every row that a lane touches begins on one; single elements otherwise
bool conv_vec(const ConvArgs& a, int elem)
{
    const long long s = a.xs.t | a.xs.b | a.ys.t | a.ys.b | a.dys.t | a.dys.b | a.D;
    uintptr_t p = 0;
    for (const void* q : {a.x, a.state, a.dy, a.dlast, (const void*)a.y, (const void*)a.last, (const void*)a.dx, (const void*)a.dstate}) p |= (uintptr_t)q;
    return s % WIDE == 0 && p % (uintptr_t)(WIDE * elem) == 0;
}
// How a launch is cut.  A run's K - 1 rows on either side are read again, so runs are as long as leaves enough waves to fill the card.
struct ConvCut { int lanes, run, channel_blocks; long long runs, blocks; };
ConvCut conv_cut(long long T, long long B, long long D, bool vec, bool bwd)
{
    ConvCut k;
    const int w = vec ? WIDE : 1;
    k.lanes = D <= 16 * w ? 16 : 64;
    k.channel_blocks = (int)((D + k.lanes * w - 1) / (k.lanes * w));
    for (k.run = 64; k.run > 8; k.run /= 2)
        if (B * ((T + k.run - 1) / k.run) * k.channel_blocks * k.lanes / 64 >= WANTED_WAVES) break;
    k.runs = T > 0 ? (T + k.run - 1) / k.run : 1;
    k.blocks = (B * k.runs + 256 / k.lanes - 1) / (256 / k.lanes);
    if (bwd) {
        const long long most = k.channel_blocks >= SUM_BLOCKS / 64 ? 64 : SUM_BLOCKS / k.channel_blocks;
        if (k.blocks > most) k.blocks = most;
    }
    return k;
}

int conv_check(const char* what, int dtype, long long T, long long B, long long D, long long K, const void* x, const float* w, const int64_t* strides, int nstrides)
{
    if (dtype != PPK_F32 && dtype != PPK_BF16) PPK_FAIL(PPK_ERR_UNSUP, "%s: type %d (fp32 and bf16 are supported)", what, dtype);
    if (T < 0 || B < 0 || D < 1 || D > (1 << 20) || K < 1) PPK_FAIL(PPK_ERR_SHAPE, "%s: T=%lld B=%lld D=%lld K=%lld", what, T, B, D, K);
    if (K > 8) PPK_FAIL(PPK_ERR_UNSUP, "%s: %lld taps (at most 8)", what, K);
    if (!strides || !w || (B > 0 && T > 0 && !x)) PPK_FAIL(PPK_ERR_NULL, "%s: null pointer", what);
    if (T >= 1LL << 31 || B >= 1LL << 31) PPK_FAIL(PPK_ERR_UNSUP, "%s: T=%lld B=%lld D=%lld", what, T, B, D);
    for (int i = 0; i < nstrides; i += 2)
        if (strides[i] < 0 || strides[i] >= 1LL << 30) PPK_FAIL(PPK_ERR_UNSUP, "%s: rows 2^30 elements or more apart", what);
    return PPK_OK;
}

// row blocks of the launch, or an error
template <typename T> int conv_run(ConvArgs a, bool bwd, hipStream_t st)
{
    const bool vec = conv_vec(a, (int)sizeof(T));
    const ConvCut k = conv_cut(a.q.T, a.q.B, a.D, vec, bwd);
    if (!ppk_grid_fits(k.blocks * k.channel_blocks, 256))
        PPK_FAIL(PPK_ERR_UNSUP, "causal_conv: T=%lld B=%lld D=%d takes %lld blocks, more than a launch has", a.q.T, a.q.B, a.D, k.blocks * k.channel_blocks);
    a.run = k.run;
    a.runs = (int)k.runs;
    if (vec) launch_conv<T, WIDE>(a, bwd, k.lanes, (unsigned)k.blocks, st);
    else launch_conv<T, 1>(a, bwd, k.lanes, (unsigned)k.blocks, st);
    return (int)k.blocks;
}

}  // namespace

extern "C" {

int ppk_causal_conv_fwd(int dtype, int64_t T, int64_t B, int64_t D, int64_t K, const int64_t* step_off, const int64_t* lengths,
                        const void* x, const float* weight, const float* bias, const void* state, int silu, void* y, void* new_state,
                        const int64_t* strides_host, ppk_stream_t stream)
{
    int rc = conv_check("causal_conv_fwd", dtype, T, B, D, K, x, weight, strides_host, 4);
    if (rc) return rc;
    if (B == 0) return PPK_OK;
    if (T > 0 && !y) PPK_FAIL(PPK_ERR_NULL, "causal_conv_fwd: null pointer");
    ConvArgs a = {};
    a.q = {step_off, lengths, T, B};
    a.D = (int)D; a.K = (int)K;
    a.x = x; a.state = state; a.weight = weight; a.bias = bias; a.y = y; a.last = K > 1 ? new_state : nullptr; a.silu = silu;
    a.xs = {strides_host[0], strides_host[1]}; a.ys = {strides_host[2], strides_host[3]};
    rc = dtype == PPK_F32 ? conv_run<float>(a, false, (hipStream_t)stream) : conv_run<bf16_t>(a, false, (hipStream_t)stream);
    if (rc < 0) return rc;
    PPK_CHECK_LAUNCH("causal_conv_fwd");
    return PPK_OK;
}

size_t ppk_causal_conv_bwd_workspace_bytes(int64_t T, int64_t B, int64_t D, int64_t K)
{
    if (T < 0 || B < 0 || D < 1 || K < 1) return 0;
    const size_t cols = (size_t)(K + 1) * (size_t)D;
    return ppk_align_up((size_t)SUM_BLOCKS * cols * 4, 256);
}

int ppk_causal_conv_bwd(int dtype, int64_t T, int64_t B, int64_t D, int64_t K, const int64_t* step_off, const int64_t* lengths,
                        const void* x, const float* weight, const float* bias, const void* state, int silu, const void* dy, const void* dnew_state,
                        void* dx, float* dweight, float* dbias, void* dstate, const int64_t* strides_host,
                        void* workspace, size_t ws_bytes, ppk_stream_t stream)
{
    int rc = conv_check("causal_conv_bwd", dtype, T, B, D, K, x, weight, strides_host, 6);
    if (rc) return rc;
    if (!dweight || !workspace || (B > 0 && T > 0 && (!dy || !dx))) PPK_FAIL(PPK_ERR_NULL, "causal_conv_bwd: null pointer");
    if (ws_bytes < ppk_causal_conv_bwd_workspace_bytes(T, B, D, K)) PPK_FAIL(PPK_ERR_WS, "causal_conv_bwd: workspace of %zu bytes", ws_bytes);
    hipStream_t st = (hipStream_t)stream;
    const long long cols = (K + 1) * D;
    ConvArgs a = {};
    a.part = (float*)workspace;
    a.q = {step_off, lengths, T, B};
    a.D = (int)D; a.K = (int)K;
    a.x = x; a.state = state; a.weight = weight; a.bias = bias; a.dy = dy; a.silu = silu; a.dx = dx;
    a.dlast = K > 1 ? dnew_state : nullptr; a.dstate = K > 1 ? dstate : nullptr;
    a.xs = {strides_host[0], strides_host[1]}; a.dys = {strides_host[2], strides_host[3]}; a.ys = {strides_host[4], strides_host[5]};
    int blocks = 0;
    if (B > 0) blocks = dtype == PPK_F32 ? conv_run<float>(a, true, st) : conv_run<bf16_t>(a, true, st);
    if (blocks < 0) return blocks;
    const ppk::SumJob job = {a.part, blocks, cols, dweight, (int)K, dbias};
    rc = ppk::partial_sums(&job, 1, nullptr, st);
    if (rc) return rc;
    PPK_CHECK_LAUNCH("causal_conv_bwd");
    return PPK_OK;
}

int ppk_causal_conv_step(int dtype, int64_t B, int64_t D, int64_t K, const void* x, int64_t ldx, const void* state, const float* weight,
                         const float* bias, int silu, void* y, void* new_state, ppk_stream_t stream)
{
    if (dtype != PPK_F32 && dtype != PPK_BF16) PPK_FAIL(PPK_ERR_UNSUP, "causal_conv_step: type %d (fp32 and bf16 are supported)", dtype);
    if (B < 0 || D < 1 || K < 1 || ldx < 0) PPK_FAIL(PPK_ERR_SHAPE, "causal_conv_step: B=%lld D=%lld K=%lld", (long long)B, (long long)D, (long long)K);
    if (K > 8) PPK_FAIL(PPK_ERR_UNSUP, "causal_conv_step: %lld taps (at most 8)", (long long)K);
    if (B >= 1LL << 32 || D >= 1LL << 31 || !ppk_grid_fits((B * D + 255) / 256, 256))
        PPK_FAIL(PPK_ERR_UNSUP, "causal_conv_step: B=%lld D=%lld, more channels than a launch has threads", (long long)B, (long long)D);
    if (B == 0) return PPK_OK;
    if (!x || !weight || !y || (K > 1 && (!state || !new_state))) PPK_FAIL(PPK_ERR_NULL, "causal_conv_step: null pointer");
    const unsigned blocks = (unsigned)((B * D + 255) / 256);
    hipStream_t st = (hipStream_t)stream;
#define STEP(T, KP) k_conv_step<T, KP><<<blocks, 256, 0, st>>>(B, (int)D, (int)K, (const T*)x, ldx, (const T*)state, weight, bias, silu, (T*)y, (T*)new_state)
    const int kp = taps(K);
    if (dtype == PPK_F32) { if (kp == 2) STEP(float, 2); else if (kp == 4) STEP(float, 4); else STEP(float, 8); }
    else { if (kp == 2) STEP(bf16_t, 2); else if (kp == 4) STEP(bf16_t, 4); else STEP(bf16_t, 8); }
#undef STEP
    PPK_CHECK_LAUNCH("causal_conv_step");
    return PPK_OK;
}

}  // extern "C"
