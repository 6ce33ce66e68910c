// Log-probabilities of the tokens a generator took, and the clipped policy loss on them with a KL term towards a reference,
// from logits [rows, V] in fp32 or bf16.  With v = logits / temperature, m = max v, s = sum exp(v - m):
//   lp    = v[token] - m - log s
//   ratio = exp(lp - old);  pg = -min(ratio A, clip(ratio, 1 - lo, 1 + hi) A);  d = ref - lp;  kl = e^d - d - 1
//   loss  = sum over rows that count of (pg + beta kl) / n
//   dloss / dlp = (-ratio A where ratio A is the smaller side, else 0) + beta (1 - e^d);  dlp / dlogits = (onehot - softmax) / temperature
// All of it is bound by HBM: the logits are read once and held in registers, and a training call writes their gradient in the
// same pass.  A row belongs to a group of TG threads that hold it as NV 16-byte chunks each.
#include "ppk_common.h"
#include "ppk_vec.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int COUNT_BLOCK = 1024;                // targets per partial count
constexpr long long COUNT_INLINE = 2048;         // up to so many rows, every block counts them itself: cheaper than a launch of their own
// Blocks of the policy modes that hold several rows at once, each loading its next rows while it works on the ones before: what is resident
// together of 122880 x 575 fp32 rows (five waves a SIMD), where the kernel takes 129 us, 142 with 2048 blocks, 137 with 4096, 140 with 4096 and
// nothing loaded ahead.  Other rows would take more: whole passes with 1280, 2560 and 4096 blocks, 1000000 x 64 fp32 203, 202, 211 us, bf16 229, 212,
// 206; 122880 x 575 bf16 229, 214, 208; 70000 x 1000 fp32 153, 132-153, 131-136; 3000000 x 9 fp32 436, 404, 383.  Scores alone have eight waves a
// SIMD and need neither: 59 us with 4096 blocks, 71 with 1280.
constexpr int RESIDENT_BLOCKS = 1280;
constexpr int MAX_BLOCKS = 4096;                 // row blocks of a launch, and rows of its partial sums

// What a row of logits meets.  `old` etc. are read only in the policy modes.
struct RowArgs {
    const void* logits; long long ld;            // row stride in elements
    const int64_t* targets;
    long long rows;
    int V;
    long long ignore;
    float inv_t;                                 // 1 / temperature
    const float* old; const float* adv; const float* ref;
    float low, high, beta;                       // 1 - clip_low, 1 + clip_high
    const int* counts; int ncounts;              // partial counts of the rows that count
    void* grad; long long ldg;
    float* logp; float* saved;                   // [rows]; [rows, 2]: max logit and 1 / s
    double* part;                                // [blocks, 3]
};

enum { MODE_LOGP = 0, MODE_POLICY = 1, MODE_POLICY_GRAD = 2 };

__global__ __launch_bounds__(256) void k_count_rows(const int64_t* __restrict__ tgt, long long rows, long long ignore, int* __restrict__ counts)
{
    __shared__ int sc[4];
    const long long r0 = (long long)blockIdx.x * COUNT_BLOCK;
    int c = 0;
    for (int i = threadIdx.x; i < COUNT_BLOCK && r0 + i < rows; i += 256) c += tgt[r0 + i] != ignore;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    if ((threadIdx.x & 63) == 0) sc[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = sc[0] + sc[1] + sc[2] + sc[3];
}

// the number of rows that count, the same in every thread of a block; `red` is LDS of one int per wave
__device__ __forceinline__ int total_count(const RowArgs& a, int* red)
{
    int c = 0;
    if (a.counts)
        for (int i = threadIdx.x; i < a.ncounts; i += blockDim.x) c += a.counts[i];
    else
        for (int i = threadIdx.x; i < (int)a.rows; i += blockDim.x) c += a.targets[i] != a.ignore;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    int t = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) t += red[w];
    return t;
}

template <int TG> __device__ __forceinline__ float group_max(float v, float* red)
{
    v = lanes_max<(TG < 64 ? TG : 64)>(v);
    if (TG > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < TG / 64; ++w) v = fmaxf(v, red[w]);
    }
    return v;
}
template <int TG> __device__ __forceinline__ float group_sum(float v, float* red)
{
    v = lanes_sum<(TG < 64 ? TG : 64)>(v);
    if (TG > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < TG / 64; ++w) v += red[w];
    }
    return v;
}

// log s of a sum s >= 1 in fp64: s = 2^k f with f in [1/sqrt 2, sqrt 2), log f = 2 atanh r = 2 (r + r^3/3 + ...), r = (f - 1) / (f + 1), where
// |r| < 0.172 and seven terms leave 2e-12.  An fp32 logarithm would round at the size of log s, and d = ref - lp has to be exact
// at its own: the KL term of a row is about d^2 / 2.
__device__ __forceinline__ double log_sum(float s)
{
    int k = __builtin_amdgcn_frexp_expf(s);
    float f = __builtin_amdgcn_frexp_mantf(s);                    // [0.5, 1)
    if (f < 0.70710678f) { f += f; --k; }
    const double n = (double)f - 1.0, q = (double)f + 1.0;
    double r = (double)__builtin_amdgcn_rcpf((float)q);
    r = fma(r, fma(-q, r, 1.0), r);                               // Newton: 2^-46 from the reciprocal's 2^-23
    r *= n;
    const double r2 = r * r;
    double p = fma(r2, 1.0 / 13, 1.0 / 11);
    p = fma(r2, p, 1.0 / 9);
    p = fma(r2, p, 1.0 / 7);
    p = fma(r2, p, 1.0 / 5);
    p = fma(r2, p, 1.0 / 3);
    p = fma(r2, p, 1.0);
    return s != s || s == INFINITY ? (double)s : fma((double)k, 0.69314718055994530942, 2.0 * r * p);
}

// e^d - d - 1 and, in `em1`, e^d - 1: the first by its series where the sum would cancel (|d| < 1/4: eight terms, the first left out 8e-12 of
// the whole), the second as its sum with d there.  Each by itself elsewhere: -(e^d - d - 1) - d rounds at the size of d, where e^d - 1 is at most 1.
__device__ __forceinline__ float kl_of(float d, float& em1)
{
    if (!(fabsf(d) < 0.25f)) {
        em1 = expf(d) - 1.0f;
        return em1 - d;
    }
    float p = fmaf(d, 1.0f / 362880, 1.0f / 40320);
    p = fmaf(d, p, 1.0f / 5040);
    p = fmaf(d, p, 1.0f / 720);
    p = fmaf(d, p, 1.0f / 120);
    p = fmaf(d, p, 1.0f / 24);
    p = fmaf(d, p, 1.0f / 6);
    p = fmaf(d, p, 0.5f);
    p *= d * d;
    em1 = p + d;
    return p;
}

// The terms of one row.  lp is fp64 (above); the differences that it enters are rounded once.  Returns dloss / dlp (before the division by n).
__device__ __forceinline__ float policy_terms(const RowArgs& a, float old, float adv, float ref, double lp, float& pg, float& kl, float& clipped)
{
    const float lr = (float)(lp - (double)old), ratio = expf(lr);
    const float held_r = ratio < a.low ? a.low : (ratio > a.high ? a.high : ratio);
    // a ratio that is finite but beyond fp32, times no advantage: nothing
    const float free_ = adv == 0.0f && lr < INFINITY ? adv : ratio * adv, held = held_r * adv;
    pg = -(free_ <= held ? free_ : (free_ != free_ ? free_ : held));
    clipped = held < free_ ? 1.0f : 0.0f;
    float g = free_ <= held ? -free_ : 0.0f;
    kl = 0.0f;
    if (a.ref) {
        const float d = (float)((double)ref - lp);
        float em1;
        kl = kl_of(d, em1);
        if (a.beta != 0.0f) g = fmaf(-a.beta, em1, g);            // no KL term: nor what it could overflow to
    }
    return g;
}

// Keeps what a chunk holds as it is: without it the compiler keeps the bf16 elements that one pass unpacked for the next, twice the registers
__device__ __forceinline__ void hold(uint4& c) { asm volatile("" : "+v"(c.x), "+v"(c.y), "+v"(c.z), "+v"(c.w)); }

// One group of TG threads a row (TG <= 64: 256 / TG rows a workgroup at once; above, one), NV chunks of 16 bytes a thread.
// NV = 0: the row does not fit in registers and is read again for its gradient.
template <typename T, int TG, int NV, int MODE>
__global__ __launch_bounds__(TG > 256 ? TG : 256) void k_rows_lp(RowArgs a)
{
    constexpr int E = 16 / (int)sizeof(T), THREADS = TG > 256 ? TG : 256, GROUPS = THREADS / TG;
    constexpr bool PREFETCH = MODE != MODE_LOGP && TG <= 64 && NV > 0 && NV <= 4;      // the next row's loads fly while this one is worked on
    __shared__ float red[THREADS / 64];
    __shared__ int redc[THREADS / 64];
    __shared__ double acc_s[GROUPS][3];
    const int g = threadIdx.x / TG, l = threadIdx.x % TG;
    float scale = 1.0f;                                                   // 1 / (n temperature)
    if (MODE == MODE_POLICY_GRAD) {
        const int n = total_count(a, redc);
        scale = (float)((double)a.inv_t / (double)(n > 0 ? n : 1));
    }
    const float k2 = a.inv_t * LOG2E;
    double s_pg = 0, s_kl = 0, s_cl = 0;
    uint4 raw[NV > 0 ? NV : 1], next[NV > 0 ? NV : 1];
    long long t_next = a.ignore;
    float old_next = 0.f, adv_next = 0.f, ref_next = 0.f;
    const auto fetch = [&](long long row) {                               // a row behind the last: nothing
        const bool in = row < a.rows;
        const long long r = in ? row : 0;
        const RowChunks<T> rc((const T*)a.logits + r * a.ld, in ? a.V : 0);
        if (NV > 0)
#pragma unroll
            for (int i = 0; i < NV; ++i) next[i] = rc.load(l + i * TG, -INFINITY);
        t_next = in ? a.targets[r] : a.ignore;
        if (MODE != MODE_LOGP) { old_next = a.old[r]; adv_next = a.adv[r]; ref_next = a.ref ? a.ref[r] : 0.f; }
    };
    const long long step = (long long)gridDim.x * GROUPS;
    if (PREFETCH) fetch((long long)blockIdx.x * GROUPS + g);
    for (long long row0 = (long long)blockIdx.x * GROUPS; row0 < a.rows; row0 += step) {
        const long long row = row0 + g;
        const bool live = row < a.rows;                                   // TG <= 64: whole groups idle, no barrier inside
        const T* x = (const T*)a.logits + (live ? row : 0) * a.ld;
        const RowChunks<T> rc(x, live ? a.V : 0);
        if (!PREFETCH) fetch(row);
        const long long t = t_next;
        const bool counts = t != a.ignore, good = t >= 0 && t < a.V;
        const float taken = counts && good ? to_f32(x[t]) : 0.f;
        const float old = old_next, adv = adv_next, ref = ref_next;
#pragma unroll
        for (int i = 0; i < (NV > 0 ? NV : 1); ++i) raw[i] = next[i];
        if (PREFETCH) fetch(row + step);
        float m = -INFINITY;
        if (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[E];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
            }
        } else {
            for (int c = l; c < rc.chunks; c += TG) {
                float v[E];
                unpack<T>(rc.load(c, -INFINITY), v);
#pragma unroll
                for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
            }
        }
        m = group_max<TG>(m, red);
        if (NV > 0 && sizeof(T) == 2)
#pragma unroll
            for (int i = 0; i < NV; ++i) hold(raw[i]);
        float s = 0.f;
        if (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[E];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((v[e] - m) * k2);
            }
        } else {
            for (int c = l; c < rc.chunks; c += TG) {
                float v[E];
                unpack<T>(rc.load(c, -INFINITY), v);
#pragma unroll
                for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((v[e] - m) * k2);
            }
        }
        s = group_sum<TG>(s, red);
        if (NV > 0 && sizeof(T) == 2)
#pragma unroll
            for (int i = 0; i < NV; ++i) hold(raw[i]);
        if (!live) continue;                                              // no barrier below; the whole group leaves together
        double lp = 0.0;
        if (counts) lp = good ? ((double)taken - (double)m) * (double)a.inv_t - log_sum(s) : (double)NAN;   // an id outside the vocabulary: NaN, never a guess
        if (MODE == MODE_LOGP) {
            if (l == 0) {
                a.logp[row] = (float)lp;
                if (a.saved) { a.saved[2 * row] = m; a.saved[2 * row + 1] = 1.0f / s; }
            }
            continue;
        }
        float gr = 0.f;
        if (counts) {
            float pg, kl, cl;
            gr = policy_terms(a, old, adv, ref, lp, pg, kl, cl);
            s_pg += pg; s_kl += kl; s_cl += cl;
        }
        if (MODE == MODE_POLICY_GRAD) {
            const float gt = gr * scale;
            const float gp = -gt / s;
            T* out = (T*)a.grad + row * a.ldg;
            const RowChunks<T> oc(out, a.V);
            const bool same = oc.shift == rc.shift;
            const auto emit = [&](int c, uint4 r) {
                float v[E];
                unpack<T>(r, v);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float p = counts ? gp * __builtin_amdgcn_exp2f((v[e] - m) * k2) : 0.f;
                    if (counts && rc.at(c, e) == t) p += gt;
                    v[e] = p;
                }
                if (same) oc.store(out, c, v);
                else if (c < rc.chunks)
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (rc.has(c, e)) out[rc.at(c, e)] = from_f32<T>(v[e]);
            };
            if (NV > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i) emit(l + i * TG, raw[i]);
            } else {
                for (int c = l; c < rc.chunks; c += TG) emit(c, rc.load(c, -INFINITY));
            }
        }
    }
    if (MODE != MODE_LOGP) {
        if (l == 0) { acc_s[g][0] = s_pg; acc_s[g][1] = s_kl; acc_s[g][2] = s_cl; }
        __syncthreads();
        if (threadIdx.x < 3) {
            double t = 0;
            for (int q = 0; q < GROUPS; ++q) t += acc_s[q][threadIdx.x];
            a.part[(long long)blockIdx.x * 3 + threadIdx.x] = t;
        }
    }
}

__global__ __launch_bounds__(1024) void k_policy_final(RowArgs a, int nparts, float* __restrict__ loss, float* __restrict__ stats)
{
    __shared__ int redc[16];
    __shared__ double red[16][3];
    const int n = total_count(a, redc);
    double s[3] = {0, 0, 0};
    for (int p = threadIdx.x; p < nparts; p += 1024)
#pragma unroll
        for (int k = 0; k < 3; ++k) s[k] += a.part[(long long)p * 3 + k];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        s[k] = ppk_wave_sum_d(s[k]);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][k] = s[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const double inv = 1.0 / (double)(n > 0 ? n : 1);
        double t[3] = {0, 0, 0};
        for (int w = 0; w < 16; ++w)
            for (int k = 0; k < 3; ++k) t[k] += red[w][k];
        for (int k = 0; k < 3; ++k) t[k] *= inv;
        loss[0] = (float)(a.beta != 0.0f ? t[0] + (double)a.beta * t[1] : t[0]);
        for (int k = 0; k < 3; ++k) stats[k] = (float)t[k];
    }
}

// d logits = g / temperature (onehot - softmax) from what the forward kept of each row: its max and 1 / s
template <typename T>
__global__ __launch_bounds__(256) void k_logp_bwd(RowArgs a, const float* __restrict__ saved, const float* __restrict__ dlogp, int per_row)
{
    constexpr int E = 16 / (int)sizeof(T);
    const float k2 = a.inv_t * LOG2E;
    const long long tasks = a.rows * per_row;
    for (long long task = blockIdx.x; task < tasks; task += gridDim.x) {
        const long long row = task / per_row;
        const int c = (int)(task - row * per_row) * 256 + threadIdx.x;
        const T* x = (const T*)a.logits + row * a.ld;
        const RowChunks<T> rc(x, a.V);
        if (c >= rc.chunks) continue;
        T* out = (T*)a.grad + row * a.ldg;
        const RowChunks<T> oc(out, a.V);
        const long long t = a.targets[row];
        const bool counts = t != a.ignore;
        const float g = t >= 0 && t < a.V ? dlogp[row] * a.inv_t : NAN, m = saved[2 * row], gp = -g * saved[2 * row + 1];
        float v[E];
        unpack<T>(rc.load(c, -INFINITY), v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float p = counts ? gp * __builtin_amdgcn_exp2f((v[e] - m) * k2) : 0.f;
            if (counts && rc.at(c, e) == t) p += g;
            v[e] = p;
        }
        if (oc.shift == rc.shift) oc.store(out, c, v);
        else
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (rc.has(c, e)) out[rc.at(c, e)] = from_f32<T>(v[e]);
    }
}

// grad *= scale[0], and nothing at all where that is 1 (the upstream gradient of a loss that is the root of the backward pass).  A bf16 gradient
// is rounded a second time here: two half-steps in all, where a factor is not a power of two.
template <typename T>
__global__ __launch_bounds__(256) void k_scale_unless_one(T* __restrict__ g, long long n, const float* __restrict__ scale)
{
    const float s = scale[0];
    if (s == 1.0f) return;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) g[e] = from_f32<T>(to_f32(g[e]) * s);
}

template <typename T, int TG, int NV>
void launch_rows(const RowArgs& a, int mode, int blocks, hipStream_t st)
{
    const dim3 block(TG > 256 ? TG : 256);
    if (mode == MODE_LOGP) k_rows_lp<T, TG, NV, MODE_LOGP><<<blocks, block, 0, st>>>(a);
    else if (mode == MODE_POLICY) k_rows_lp<T, TG, NV, MODE_POLICY><<<blocks, block, 0, st>>>(a);
    else k_rows_lp<T, TG, NV, MODE_POLICY_GRAD><<<blocks, block, 0, st>>>(a);
}

// The threads of a row of `chunks` 16-byte chunks: as few as hold it in 64 registers each (more rows at once hide each other's waits)
int group_width(long long chunks) { return chunks <= 64 ? 16 : chunks <= 512 ? 64 : chunks <= 4096 ? 256 : chunks <= 8192 ? 512 : 1024; }      // 1024: read again instead
int row_blocks(long long rows, int tg, int mode)
{
    const int groups = tg >= 256 ? 1 : 256 / tg;
    const long long b = (rows + groups - 1) / groups, most = tg <= 64 && mode != MODE_LOGP ? RESIDENT_BLOCKS : MAX_BLOCKS;
    return (int)(b < most ? b : most);
}

template <typename T>
void dispatch_rows(const RowArgs& a, int mode, int blocks, long long chunks, hipStream_t st)
{
    const int tg = group_width(chunks);
    const long long nv = (chunks + tg - 1) / tg;
#define ROWS(TG, NV) if (tg == TG && nv <= NV) return launch_rows<T, TG, NV>(a, mode, blocks, st)
    ROWS(16, 1); ROWS(16, 2); ROWS(16, 4);
    ROWS(64, 2); ROWS(64, 3); ROWS(64, 4); ROWS(64, 6); ROWS(64, 8);
    ROWS(256, 3); ROWS(256, 4); ROWS(256, 6); ROWS(256, 8); ROWS(256, 12); ROWS(256, 16);
    ROWS(512, 12); ROWS(512, 16);
#undef ROWS
    launch_rows<T, 1024, 0>(a, mode, blocks, st);
}

int elem_bytes(int dtype) { return dtype == PPK_F32 ? 4 : 2; }
// chunks of a row at worst: one more than its bytes need where it begins inside a chunk
long long row_chunks(long long V, int dtype) { return (V * elem_bytes(dtype) + 15) / 16 + 1; }

int check_rows(const char* what, int dtype, long long rows, long long V, const void* logits, long long ld, const void* targets, float temperature)
{
    if (dtype != PPK_F32 && dtype != PPK_BF16) PPK_FAIL(PPK_ERR_UNSUP, "%s: logits of type %d (fp32 and bf16 are supported)", what, dtype);
    if (rows < 0 || V < 1 || ld < V || V > (1LL << 30)) PPK_FAIL(PPK_ERR_SHAPE, "%s: rows=%lld V=%lld row stride=%lld", what, rows, V, ld);
    if (!(temperature >= 1.0e-30f) || temperature > 1.0e30f) PPK_FAIL(PPK_ERR_SHAPE, "%s: temperature %g", what, (double)temperature);
    if (rows > 0 && (!logits || !targets)) PPK_FAIL(PPK_ERR_NULL, "%s: null pointer", what);
    if ((uintptr_t)logits % (unsigned)elem_bytes(dtype)) PPK_FAIL(PPK_ERR_ALIGN, "%s: logits not aligned to their elements", what);
    return PPK_OK;
}

struct PolicyWs { int* counts; double* part; };
int count_blocks(long long rows) { return rows <= COUNT_INLINE ? 0 : (int)((rows + COUNT_BLOCK - 1) / COUNT_BLOCK); }
size_t policy_ws_bytes(long long rows) { return ppk_align_up((size_t)count_blocks(rows) * 4, 256) + ppk_align_up((size_t)MAX_BLOCKS * 24, 256); }

}  // namespace

extern "C" {

int ppk_token_logp_fwd(int dtype, const void* logits, int64_t ldl, const int64_t* targets, int64_t rows, int64_t V, int64_t ignore_index,
                       float temperature, float* logp, float* saved, ppk_stream_t stream)
{
    int rc = check_rows("token_logp_fwd", dtype, rows, V, logits, ldl, targets, temperature);
    if (rc) return rc;
    if (rows == 0) return PPK_OK;
    if (!logp) PPK_FAIL(PPK_ERR_NULL, "token_logp_fwd: null pointer");
    RowArgs a = {};
    a.logits = logits; a.ld = ldl; a.targets = targets; a.rows = rows; a.V = (int)V; a.ignore = ignore_index; a.inv_t = 1.0f / temperature;
    a.logp = logp; a.saved = saved;
    const long long ch = row_chunks(V, dtype);
    const int blocks = row_blocks(rows, group_width(ch), MODE_LOGP);
    if (dtype == PPK_F32) dispatch_rows<float>(a, MODE_LOGP, blocks, ch, (hipStream_t)stream);
    else dispatch_rows<bf16_t>(a, MODE_LOGP, blocks, ch, (hipStream_t)stream);
    PPK_CHECK_LAUNCH("token_logp_fwd");
    return PPK_OK;
}

int ppk_token_logp_bwd(int dtype, const void* logits, int64_t ldl, const int64_t* targets, int64_t rows, int64_t V, int64_t ignore_index,
                       float temperature, const float* saved, const float* dlogp, void* dlogits, int64_t ldd, ppk_stream_t stream)
{
    int rc = check_rows("token_logp_bwd", dtype, rows, V, logits, ldl, targets, temperature);
    if (rc) return rc;
    if (ldd < V) PPK_FAIL(PPK_ERR_SHAPE, "token_logp_bwd: row stride %lld < V", (long long)ldd);
    if (rows == 0) return PPK_OK;
    if (!saved || !dlogp || !dlogits) PPK_FAIL(PPK_ERR_NULL, "token_logp_bwd: null pointer");
    RowArgs a = {};
    a.logits = logits; a.ld = ldl; a.targets = targets; a.rows = rows; a.V = (int)V; a.ignore = ignore_index; a.inv_t = 1.0f / temperature;
    a.grad = dlogits; a.ldg = ldd;
    const int per_row = (int)((row_chunks(V, dtype) + 255) / 256);
    const long long tasks = rows * per_row;
    const unsigned blocks = (unsigned)(tasks < 16384 ? tasks : 16384);
    if (dtype == PPK_F32) k_logp_bwd<float><<<blocks, 256, 0, (hipStream_t)stream>>>(a, saved, dlogp, per_row);
    else k_logp_bwd<bf16_t><<<blocks, 256, 0, (hipStream_t)stream>>>(a, saved, dlogp, per_row);
    PPK_CHECK_LAUNCH("token_logp_bwd");
    return PPK_OK;
}

size_t ppk_policy_loss_workspace_bytes(int64_t rows) { return rows < 0 ? 0 : policy_ws_bytes(rows); }

int ppk_policy_loss(int dtype, const void* logits, int64_t ldl, const int64_t* targets, int64_t rows, int64_t V, int64_t ignore_index,
                    float temperature, const float* old_logp, const float* advantages, const float* ref_logp,
                    float clip_low, float clip_high, float kl_coef, float* loss, float* stats, void* dlogits, int64_t ldd,
                    void* workspace, size_t ws_bytes, ppk_stream_t stream)
{
    int rc = check_rows("policy_loss", dtype, rows, V, logits, ldl, targets, temperature);
    if (rc) return rc;
    if (!(clip_low >= 0.f && clip_low <= 1.f) || !(clip_high >= 0.f)) PPK_FAIL(PPK_ERR_SHAPE, "policy_loss: clip range [%g, %g]", (double)clip_low, (double)clip_high);
    if (!loss || !stats || !workspace || (rows > 0 && (!old_logp || !advantages))) PPK_FAIL(PPK_ERR_NULL, "policy_loss: null pointer");
    if (rows > 0 && kl_coef != 0.f && !ref_logp) PPK_FAIL(PPK_ERR_NULL, "policy_loss: a KL term needs the reference's log-probabilities");
    if (dlogits && ldd < V) PPK_FAIL(PPK_ERR_SHAPE, "policy_loss: row stride %lld < V", (long long)ldd);
    if (rows > (1LL << 31) - 1) PPK_FAIL(PPK_ERR_UNSUP, "policy_loss: %lld rows", (long long)rows);
    if (ws_bytes < policy_ws_bytes(rows)) PPK_FAIL(PPK_ERR_WS, "policy_loss: workspace of %zu bytes, %zu needed", ws_bytes, policy_ws_bytes(rows));
    hipStream_t st = (hipStream_t)stream;
    char* cur = (char*)workspace;
    const int nc = count_blocks(rows);
    int* counts = (int*)ppk_carve(cur, (size_t)nc * 4);
    RowArgs a = {};
    a.logits = logits; a.ld = ldl; a.targets = targets; a.rows = rows; a.V = (int)V; a.ignore = ignore_index; a.inv_t = 1.0f / temperature;
    a.old = old_logp; a.adv = advantages; a.ref = ref_logp;
    a.low = 1.0f - clip_low; a.high = 1.0f + clip_high; a.beta = kl_coef;
    a.counts = nc ? counts : nullptr; a.ncounts = nc; a.grad = dlogits; a.ldg = ldd;
    a.part = (double*)cur;
    const long long ch = row_chunks(V, dtype);
    const int blocks = row_blocks(rows, group_width(ch), MODE_POLICY);
    if (nc) k_count_rows<<<nc, 256, 0, st>>>(targets, rows, ignore_index, counts);
    const int mode = dlogits ? MODE_POLICY_GRAD : MODE_POLICY;
    if (rows > 0) {
        if (dtype == PPK_F32) dispatch_rows<float>(a, mode, blocks, ch, st);
        else dispatch_rows<bf16_t>(a, mode, blocks, ch, st);
    }
    k_policy_final<<<1, 1024, 0, st>>>(a, rows > 0 ? blocks : 0, loss, stats);
    PPK_CHECK_LAUNCH("policy_loss");
    return PPK_OK;
}

int ppk_scale_unless_one(int dtype, void* g, int64_t n, const float* scale, ppk_stream_t stream)
{
    if (dtype != PPK_F32 && dtype != PPK_BF16) PPK_FAIL(PPK_ERR_UNSUP, "scale_unless_one: type %d", dtype);
    if (n < 0) PPK_FAIL(PPK_ERR_SHAPE, "scale_unless_one: n=%lld", (long long)n);
    if (n == 0) return PPK_OK;
    if (!g || !scale) PPK_FAIL(PPK_ERR_NULL, "scale_unless_one: null pointer");
    const long long b = (n + 2047) / 2048;
    const unsigned blocks = (unsigned)(b < 2048 ? b : 2048);
    if (dtype == PPK_F32) k_scale_unless_one<float><<<blocks, 256, 0, (hipStream_t)stream>>>((float*)g, n, scale);
    else k_scale_unless_one<bf16_t><<<blocks, 256, 0, (hipStream_t)stream>>>((bf16_t*)g, n, scale);
    PPK_CHECK_LAUNCH("scale_unless_one");
    return PPK_OK;
}

}  // extern "C"
