// Selective state space scan over packed or rectangular batches of sequences.  A channel d of a sequence holds N states:
//   dt = softplus(raw + bias);  a_n = exp(dt A_n);  h_n = a_n h_n' + dt x B_n;  y = (sum_n C_n h_n + D x) z sigmoid(z)
// B and C are shared by the channels of a group.  Backward, with dy' = dout silu(z) and dh running from the last step to the first:
//   dh_n = dy' C_n + (a_n dh_n of the next step);  da_n = dh_n h_n' a_n;  ddt = sum da_n A_n + x sum dh_n B_n;  dA_n = sum da_n dt
//   dx = dt sum dh_n B_n + D dy';  dB_n = sum_d dh_n dt x;  dC_n = sum_d dy' h_n;  draw = ddt sigmoid(raw + bias)
// States, sums and gradients of states are fp32.  The forward pass keeps the state before every TILE steps; the backward pass
// walks the tiles backwards and makes the states inside one again, in registers.
#include "ppk_seq_rows.h"

namespace {

using ppk::SeqBatch;
using ppk::Stride;
using ppk::at;

constexpr int TILE = 16;                     // steps between two kept states
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct ScanArgs {
    SeqBatch q;
    const int64_t* tiles;                    // device [B + 1]: first tile of each sequence, or null: rectangular
    int D, N, G, per;                        // per = D / G channels of a group
    int blocks_per_group;                    // channel blocks of a launch in a group
    const void *x, *raw, *Bm, *Cm, *z, *dy;
    const float *A, *skip, *bias, *state, *dlast;
    Stride xs, raws, Bs, Cs, zs, dys, rows;  // rows: of the outputs, in rows of their width
    long long Bg, Cg;                        // group strides
    int softplus;
    void *y, *dx, *draw, *dz;
    float *last, *kept, *dstate;             // kept: [tiles, D, N]
    float *pA, *pD, *pBC;                    // partial sums: [items, D, N], [2, items, D], [blocks_per_group, rows, G, 2, N]
    long long nrows;
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2_(-LOG2E * x)); }
__device__ __forceinline__ float softplus(float x) { return x > 20.0f ? x : log1pf(__expf(x)); }
__device__ __forceinline__ float lane_value(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

// One wave: 64 channels of a group of one sequence, every lane a channel with its NP >= N states in registers.  B and C of a step are
// loaded by the lanes n < N and handed to the multiplications as scalars.
template <typename T, int NP>
__global__ __launch_bounds__(64) void k_scan_fwd(ScanArgs a)
{
    const int lane = threadIdx.x;
    const int nb = a.G * a.blocks_per_group;
    const long long b = blockIdx.x / nb;
    const int cb = (int)(blockIdx.x % nb), g = cb / a.blocks_per_group;
    const int dl = (cb % a.blocks_per_group) * 64 + lane;
    const bool live = dl < a.per;
    const int d = g * a.per + (live ? dl : 0), N = a.N;
    const long long len = a.q.length(b);
    float A2[NP], h[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        A2[n] = n < N ? a.A[(long long)d * N + n] * LOG2E : 0.f;
        h[n] = n < N && a.state ? a.state[(b * a.D + d) * N + n] : 0.f;
    }
    const float skip = a.skip ? a.skip[d] : 0.f, bias = a.bias ? a.bias[d] : 0.f;
    const long long tile0 = a.tiles ? a.tiles[b] : b * ((a.q.T + TILE - 1) / TILE);
    const T* Bp = (const T*)a.Bm + g * a.Bg + (lane < N ? lane : 0);
    const T* Cp = (const T*)a.Cm + g * a.Cg + (lane < N ? lane : 0);
    for (long long t = 0; t < len; ++t) {
        if (a.kept && t % TILE == 0 && live)
#pragma unroll
            for (int n = 0; n < NP; ++n)
                if (n < N) a.kept[((tile0 + t / TILE) * a.D + d) * N + n] = h[n];
        const long long r = a.q.row(t);
        const float x = to_f32(((const T*)a.x)[at(a.xs, r, b) + d]);
        const float raw = to_f32(((const T*)a.raw)[at(a.raws, r, b) + d]) + bias;
        const float Bv = to_f32(Bp[at(a.Bs, r, b)]), Cv = to_f32(Cp[at(a.Cs, r, b)]);
        const float dt = a.softplus ? softplus(raw) : raw, dx = dt * x;
        float y[4] = {skip * x, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (n < N) {
                h[n] = fmaf(exp2_(dt * A2[n]), h[n], dx * lane_value(Bv, n));
                y[n & 3] = fmaf(h[n], lane_value(Cv, n), y[n & 3]);
            }
        float out = (y[0] + y[1]) + (y[2] + y[3]);
        if (a.z) { const float z = to_f32(((const T*)a.z)[at(a.zs, r, b) + d]); out *= z * sigmoid(z); }
        if (live) ((T*)a.y)[at(a.rows, r, b) * a.D + d] = from_f32<T>(out);
    }
    if (live)
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (n < N) a.last[(b * a.D + d) * N + n] = h[n];
}

// v + v of the lane that `ctrl` names, in one instruction
template <int CTRL> __device__ __forceinline__ float dpp_add(float v)
{
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, HALF_MIRROR = 0x141, MIRROR = 0x140, ROR4 = 0x124, ROR8 = 0x128;
// sum over the low bits of the lane number, LPC lanes; every one of them holds it.  A mirror reverses lanes that hold the same
// sum already within each half, which is what an xor of that half's width would reach.
template <int LPC> __device__ __forceinline__ float sum_low(float v)
{
    if (LPC > 1) v = dpp_add<XOR1>(v);
    if (LPC > 2) v = dpp_add<XOR2>(v);
    if (LPC > 4) v = dpp_add<HALF_MIRROR>(v);
    if (LPC > 8) v = dpp_add<MIRROR>(v);
    return v;
}
// sum over the lanes of a row of 16 that share their low bits (LPC of them)
template <int LPC> __device__ __forceinline__ float sum_high16(float v)
{
    if (LPC <= 1) v = dpp_add<XOR1>(v);
    if (LPC <= 2) v = dpp_add<XOR2>(v);
    if (LPC <= 4) v = dpp_add<ROR4>(v);
    if (LPC <= 8) v = dpp_add<ROR8>(v);
    return v;
}

// Block: 256 / LPC channels of a group of one sequence; lane = channel * LPC + slice, a thread holds the 4 states 4 slice .. of its channel.
template <typename T, int LPC>
__global__ __launch_bounds__(256) void k_scan_bwd(ScanArgs a)
{
    constexpr int NP = 4 * LPC, BC = 256 / LPC, PE = TILE * BC / 256;
    __shared__ float s_dt[TILE][BC], s_dx[TILE][BC], s_dy[TILE][BC];           // dt, dt x, dy'; then the sums over n of dh B, da A, C h
    __shared__ __align__(16) float s_B[TILE][NP], s_C[TILE][NP];
    __shared__ float s_red[TILE][4][2 * NP];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int ch = tid / LPC, ns = tid % LPC;                                  // the scan's channel and slice
    const int pc = tid % BC, pt = tid / BC;                                    // the channel and first step of the per-element work
    const int nb = a.G * a.blocks_per_group, N = a.N;
    const long long b = blockIdx.x / nb;
    const int cb = (int)(blockIdx.x % nb), g = cb / a.blocks_per_group, cg = cb % a.blocks_per_group;
    const int base = cg * BC;                                                  // of the block's channels in the group
    const bool live = base + ch < a.per, plive = base + pc < a.per;
    const int d = g * a.per + (live ? base + ch : 0), pd = g * a.per + (plive ? base + pc : 0);
    const long long len = a.q.length(b);
    const long long tile0 = a.tiles ? a.tiles[b] : b * ((a.q.T + TILE - 1) / TILE);
    float A2[4], dA[4] = {0.f, 0.f, 0.f, 0.f}, dh[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = ns * 4 + j;
        A2[j] = live && n < N ? a.A[(long long)d * N + n] * LOG2E : 0.f;
        dh[j] = live && n < N && a.dlast ? a.dlast[(b * a.D + d) * N + n] : 0.f;
    }
    const float skip = a.skip && plive ? a.skip[pd] : 0.f, bias = a.bias && plive ? a.bias[pd] : 0.f;
    float dskip = 0.f, dbias = 0.f;
    for (long long tile = (len + TILE - 1) / TILE - 1; tile >= 0; --tile) {
        const long long t0 = tile * TILE;
        const int steps = (int)(len - t0 < TILE ? len - t0 : TILE);
        float x[PE], dt[PE], slope[PE], dy[PE], dout[PE], z[PE], sig[PE];
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            const int t = pt + i * (256 / BC);
            const bool in = plive && t < steps;
            const long long r = a.q.row(t0 + (t < steps ? t : 0));
            x[i] = in ? to_f32(((const T*)a.x)[at(a.xs, r, b) + pd]) : 0.f;
            const float raw = in ? to_f32(((const T*)a.raw)[at(a.raws, r, b) + pd]) + bias : 0.f;
            dout[i] = in ? to_f32(((const T*)a.dy)[at(a.dys, r, b) + pd]) : 0.f;
            z[i] = in && a.z ? to_f32(((const T*)a.z)[at(a.zs, r, b) + pd]) : 0.f;
            sig[i] = sigmoid(z[i]);
            dt[i] = in ? (a.softplus ? softplus(raw) : raw) : 0.f;
            slope[i] = a.softplus ? sigmoid(raw) : 1.0f;
            dy[i] = a.z ? dout[i] * z[i] * sig[i] : dout[i];
            s_dt[t][pc] = dt[i];
            s_dx[t][pc] = dt[i] * x[i];
            s_dy[t][pc] = dy[i];
        }
        for (int e = tid; e < TILE * NP; e += 256) {
            const int t = e / NP, n = e % NP;
            const bool in = t < steps && n < N;
            const long long r = a.q.row(t0 + (t < steps ? t : 0));
            s_B[t][n] = in ? to_f32(((const T*)a.Bm)[at(a.Bs, r, b) + g * a.Bg + n]) : 0.f;
            s_C[t][n] = in ? to_f32(((const T*)a.Cm)[at(a.Cs, r, b) + g * a.Cg + n]) : 0.f;
        }
        float h[TILE + 1][4], av[TILE][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = ns * 4 + j;
            h[0][j] = live && n < N ? a.kept[((tile0 + tile) * a.D + d) * N + n] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TILE; ++t) {
            const float dtv = s_dt[t][ch], dxv = s_dx[t][ch];
            const float4 Bv = *reinterpret_cast<const float4*>(&s_B[t][ns * 4]);
            const float Bj[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                av[t][j] = exp2_(dtv * A2[j]);
                h[t + 1][j] = fmaf(av[t][j], h[t][j], dxv * Bj[j]);
            }
        }
#pragma unroll
        for (int t = TILE - 1; t >= 0; --t) {
            const float dtv = s_dt[t][ch], dxv = s_dx[t][ch], dyv = s_dy[t][ch];
            const float4 Bv = *reinterpret_cast<const float4*>(&s_B[t][ns * 4]), Cv = *reinterpret_cast<const float4*>(&s_C[t][ns * 4]);
            const float Bj[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, Cj[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
            float q1 = 0.f, q2 = 0.f, q3 = 0.f, v[8];                           // v: dB of the four states, then dC
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                dh[j] = fmaf(dyv, Cj[j], dh[j]);
                q1 = fmaf(dh[j], Bj[j], q1);
                v[j] = dh[j] * dxv;
                v[4 + j] = dyv * h[t + 1][j];
                q3 = fmaf(Cj[j], h[t + 1][j], q3);
                dh[j] *= av[t][j];
                const float da = dh[j] * h[t][j];
                q2 = fmaf(da, A2[j], q2);
                dA[j] = fmaf(da, dtv, dA[j]);
            }
            q1 = sum_low<LPC>(q1);
            q2 = sum_low<LPC>(q2);
            q3 = sum_low<LPC>(q3);
            if (ns == 0) { s_dt[t][ch] = q1; s_dx[t][ch] = q2; s_dy[t][ch] = q3; }       // this wave's channels: read above by the same wave
            // over the wave's channels: two exchanges leave a lane the sums of two of the eight, bits 5 and 4 of the lane say which
            float u[4], w[2];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[k]), __float_as_uint(v[k + 4]), false, false);
                u[k] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(u[k]), __float_as_uint(u[k + 2]), false, false);
                w[k] = sum_high16<LPC>(__uint_as_float(p[0]) + __uint_as_float(p[1]));
            }
            if ((lane & 15) < LPC) {
                const int n = (lane & (LPC - 1)) * 4 + ((lane >> 4) & 1) * 2, side = (lane >> 5) * NP;
                s_red[t][wave][side + n] = w[0];
                s_red[t][wave][side + n + 1] = w[1];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            const int t = pt + i * (256 / BC);
            if (!(plive && t < steps)) continue;
            const long long o = at(a.rows, a.q.row(t0 + t), b) * a.D + pd;
            const float q1 = s_dt[t][pc], q2 = s_dx[t][pc] * LN2, q3 = s_dy[t][pc];
            const float dr = fmaf(x[i], q1, q2) * slope[i];
            ((T*)a.dx)[o] = from_f32<T>(fmaf(dt[i], q1, skip * dy[i]));
            ((T*)a.draw)[o] = from_f32<T>(dr);
            if (a.z) ((T*)a.dz)[o] = from_f32<T>(dout[i] * fmaf(skip, x[i], q3) * sig[i] * fmaf(z[i], 1.0f - sig[i], 1.0f));
            dskip = fmaf(dy[i], x[i], dskip);
            dbias += dr;
        }
        for (int e = tid; e < TILE * 2 * NP; e += 256) {
            const int t = e / (2 * NP), k = e % (2 * NP), n = k % NP;
            if (t >= steps || n >= N) continue;
            const long long row = at(a.rows, a.q.row(t0 + t), b);
            a.pBC[(((long long)cg * a.nrows + row) * a.G + g) * 2 * N + (k / NP) * N + n] = (s_red[t][0][k] + s_red[t][1][k]) + (s_red[t][2][k] + s_red[t][3][k]);
        }
        __syncthreads();
    }
    if (live)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = ns * 4 + j;
            if (n >= N) continue;
            a.pA[(b * a.D + d) * N + n] = dA[j];
            if (a.dstate) a.dstate[(b * a.D + d) * N + n] = dh[j];
        }
    __syncthreads();
    s_dt[pt][pc] = dskip;
    s_dx[pt][pc] = dbias;
    __syncthreads();
    if (pt == 0 && plive) {
        float u = s_dt[0][pc], v = s_dx[0][pc];
        for (int i = 1; i < 256 / BC; ++i) { u += s_dt[i][pc]; v += s_dx[i][pc]; }
        a.pD[b * a.D + pd] = u;
        a.pD[(a.q.B + b) * a.D + pd] = v;
    }
}

// dB, dC [rows, G, N]: the channel blocks of a group, in order
template <typename T>
__global__ __launch_bounds__(256) void k_scan_bc(const float* __restrict__ p, int blocks, long long nrows, int G, int N, T* __restrict__ dB, T* __restrict__ dC)
{
    const long long n = nrows * G * 2 * N, e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= n) return;
    float s = p[e];
    for (int k = 1; k < blocks; ++k) s += p[k * n + e];
    const long long rg = e / (2 * N);
    const int k = (int)(e % (2 * N));
    (k < N ? dB : dC)[rg * N + (k < N ? k : k - N)] = from_f32<T>(s);
}

// One token of each sequence: lane = channel * LPC + slice as in the backward pass, four states a thread
template <typename T, int LPC>
__global__ __launch_bounds__(256) void k_scan_step(ScanArgs a, const float* state, float* next)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const int ns = (int)(e % LPC), N = a.N;
    const long long bd = e / LPC;
    if (bd >= a.q.B * a.D) return;                                             // whole groups of LPC lanes
    const long long b = bd / a.D;
    const int d = (int)(bd % a.D), g = d / a.per;
    const float x = to_f32(((const T*)a.x)[b * a.xs.b + d]);
    const float raw = to_f32(((const T*)a.raw)[b * a.raws.b + d]) + (a.bias ? a.bias[d] : 0.f);
    const float dt = a.softplus ? softplus(raw) : raw, dx = dt * x;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = ns * 4 + j;
        if (n >= N) continue;
        const float Bv = to_f32(((const T*)a.Bm)[b * a.Bs.b + g * a.Bg + n]), Cv = to_f32(((const T*)a.Cm)[b * a.Cs.b + g * a.Cg + n]);
        const float h = fmaf(exp2_(dt * (a.A[(long long)d * N + n] * LOG2E)), state[bd * N + n], dx * Bv);
        next[bd * N + n] = h;
        y = fmaf(h, Cv, y);
    }
    y = sum_low<LPC>(y) + (a.skip ? a.skip[d] * x : 0.f);
    if (a.z) { const float z = to_f32(((const T*)a.z)[b * a.zs.b + d]); y *= z * sigmoid(z); }
    if (ns == 0) ((T*)a.y)[bd] = from_f32<T>(y);
}

int slices(long long N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

template <typename T> void run_fwd(const ScanArgs& a, unsigned blocks, hipStream_t st)
{
    if (a.N <= 8) k_scan_fwd<T, 8><<<blocks, 64, 0, st>>>(a);
    else if (a.N <= 16) k_scan_fwd<T, 16><<<blocks, 64, 0, st>>>(a);
    else if (a.N <= 32) k_scan_fwd<T, 32><<<blocks, 64, 0, st>>>(a);
    else k_scan_fwd<T, 64><<<blocks, 64, 0, st>>>(a);
}
template <typename T> void run_bwd(const ScanArgs& a, unsigned blocks, hipStream_t st)
{
    switch (slices(a.N)) {
        case 1: k_scan_bwd<T, 1><<<blocks, 256, 0, st>>>(a); break;
        case 2: k_scan_bwd<T, 2><<<blocks, 256, 0, st>>>(a); break;
        case 4: k_scan_bwd<T, 4><<<blocks, 256, 0, st>>>(a); break;
        case 8: k_scan_bwd<T, 8><<<blocks, 256, 0, st>>>(a); break;
        default: k_scan_bwd<T, 16><<<blocks, 256, 0, st>>>(a);
    }
}
template <typename T> void run_step(const ScanArgs& a, unsigned blocks, const float* state, float* next, hipStream_t st)
{
    switch (slices(a.N)) {
        case 1: k_scan_step<T, 1><<<blocks, 256, 0, st>>>(a, state, next); break;
        case 2: k_scan_step<T, 2><<<blocks, 256, 0, st>>>(a, state, next); break;
        case 4: k_scan_step<T, 4><<<blocks, 256, 0, st>>>(a, state, next); break;
        case 8: k_scan_step<T, 8><<<blocks, 256, 0, st>>>(a, state, next); break;
        default: k_scan_step<T, 16><<<blocks, 256, 0, st>>>(a, state, next);
    }
}

int scan_check(const char* what, int dtype, long long T, long long B, long long D, long long N, long long G)
{
    if (dtype != PPK_F32 && dtype != PPK_BF16) PPK_FAIL(PPK_ERR_UNSUP, "%s: type %d (fp32 and bf16 are supported)", what, dtype);
    if (T < 0 || B < 0 || D < 1 || N < 1 || G < 1 || D % G) PPK_FAIL(PPK_ERR_SHAPE, "%s: T=%lld B=%lld D=%lld N=%lld G=%lld", what, T, B, D, N, G);
    if (N > 64) PPK_FAIL(PPK_ERR_UNSUP, "%s: %lld states a channel (at most 64)", what, N);
    if (D > (1 << 20)) PPK_FAIL(PPK_ERR_UNSUP, "%s: %lld channels", what, D);
    return PPK_OK;
}

struct BwdWs { size_t a, d, bc, sum, total; long long blocks_per_group; };
BwdWs bwd_ws(long long B, long long D, long long N, long long G, long long rows)
{
    BwdWs w;
    w.blocks_per_group = ceil_div(D / G, 256 / slices(N));
    w.a = ppk_align_up((size_t)B * D * N * 4, 256);
    w.d = ppk_align_up((size_t)B * 2 * D * 4, 256);
    w.bc = ppk_align_up((size_t)w.blocks_per_group * rows * G * 2 * N * 4, 256);
    w.sum = ppk::partial_sum_ws_bytes(B, D * N);
    w.total = w.a + w.d + w.bc + w.sum;
    return w;
}

// host array of strides, in elements, of (step, sequence[, group]): x, raw, B, C, z, out rows, dy
void set_strides(ScanArgs& a, const int64_t* s)
{
    a.xs = {s[0], s[1]}; a.raws = {s[2], s[3]};
    a.Bs = {s[4], s[5]}; a.Bg = s[6];
    a.Cs = {s[7], s[8]}; a.Cg = s[9];
    a.zs = {s[10], s[11]}; a.rows = {s[12], s[13]};
    a.dys = {s[14], s[15]};
}

}  // namespace

extern "C" {

int64_t ppk_selective_scan_tile(void) { return TILE; }

int ppk_selective_scan_fwd(int dtype, int64_t T, int64_t B, int64_t D, int64_t N, int64_t G, const int64_t* step_off, const int64_t* lengths,
                           const int64_t* tiles, const void* x, const void* raw, const float* A, const void* Bm, const void* Cm, const float* skip,
                           const void* z, const float* bias, const float* state, int softplus, void* y, float* last_state, float* kept,
                           const int64_t* strides_host, ppk_stream_t stream)
{
    int rc = scan_check("selective_scan_fwd", dtype, T, B, D, N, G);
    if (rc) return rc;
    if (B == 0) return PPK_OK;
    if (!A || !last_state || !strides_host || (T > 0 && (!x || !raw || !Bm || !Cm || !y))) PPK_FAIL(PPK_ERR_NULL, "selective_scan_fwd: null pointer");
    if (step_off && (!lengths || !tiles)) PPK_FAIL(PPK_ERR_NULL, "selective_scan_fwd: a packed batch needs its lengths and tiles");
    ScanArgs a = {};
    a.q = {step_off, lengths, T, B};
    a.tiles = tiles;
    a.D = (int)D; a.N = (int)N; a.G = (int)G; a.per = (int)(D / G); a.blocks_per_group = (int)ceil_div(a.per, 64);
    a.x = x; a.raw = raw; a.Bm = Bm; a.Cm = Cm; a.z = z; a.A = A; a.skip = skip; a.bias = bias; a.state = state; a.softplus = softplus;
    a.y = y; a.last = last_state; a.kept = kept;
    set_strides(a, strides_host);
    const long long blocks = B * G * a.blocks_per_group;
    if (blocks > 0x7fffffffLL) PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_fwd: B=%lld D=%lld", (long long)B, (long long)D);
    if (dtype == PPK_F32) run_fwd<float>(a, (unsigned)blocks, (hipStream_t)stream);
    else run_fwd<bf16_t>(a, (unsigned)blocks, (hipStream_t)stream);
    PPK_CHECK_LAUNCH("selective_scan_fwd");
    return PPK_OK;
}

size_t ppk_selective_scan_bwd_workspace_bytes(int64_t T, int64_t B, int64_t D, int64_t N, int64_t G, int64_t rows)
{
    if (T < 0 || B < 0 || D < 1 || N < 1 || N > 64 || G < 1 || rows < 0) return 0;
    return bwd_ws(B, D, N, G, rows).total;
}

int ppk_selective_scan_bwd(int dtype, int64_t T, int64_t B, int64_t D, int64_t N, int64_t G, int64_t rows, const int64_t* step_off,
                           const int64_t* lengths, const int64_t* tiles, const void* x, const void* raw, const float* A, const void* Bm, const void* Cm,
                           const float* skip, const void* z, const float* bias, int softplus, const float* kept, const void* dy, const float* dlast_state,
                           void* dx, void* draw, float* dA, void* dB, void* dC, float* dskip, void* dz, float* dbias, float* dstate,
                           const int64_t* strides_host, void* workspace, size_t ws_bytes, ppk_stream_t stream)
{
    int rc = scan_check("selective_scan_bwd", dtype, T, B, D, N, G);
    if (rc) return rc;
    if (rows < 0 || (!step_off && rows != T * B)) PPK_FAIL(PPK_ERR_SHAPE, "selective_scan_bwd: %lld rows", (long long)rows);
    if (!A || !dA || !workspace || !strides_host || (rows > 0 && (!x || !raw || !Bm || !Cm || !dy || !kept || !dx || !draw || !dB || !dC || (z && !dz))))
        PPK_FAIL(PPK_ERR_NULL, "selective_scan_bwd: null pointer");
    if (step_off && (!lengths || !tiles)) PPK_FAIL(PPK_ERR_NULL, "selective_scan_bwd: a packed batch needs its lengths and tiles");
    const BwdWs w = bwd_ws(B, D, N, G, rows);
    if (ws_bytes < w.total) PPK_FAIL(PPK_ERR_WS, "selective_scan_bwd: workspace of %zu bytes, %zu needed", ws_bytes, w.total);
    hipStream_t st = (hipStream_t)stream;
    char* cur = (char*)workspace;
    ScanArgs a = {};
    a.pA = (float*)ppk_carve(cur, (size_t)B * D * N * 4);
    a.pD = (float*)ppk_carve(cur, (size_t)B * 2 * D * 4);
    a.pBC = (float*)ppk_carve(cur, w.bc);
    void* sum_ws = cur;
    a.q = {step_off, lengths, T, B};
    a.tiles = tiles;
    a.D = (int)D; a.N = (int)N; a.G = (int)G; a.per = (int)(D / G); a.blocks_per_group = (int)w.blocks_per_group;
    a.x = x; a.raw = raw; a.Bm = Bm; a.Cm = Cm; a.z = z; a.dy = dy; a.A = A; a.skip = skip; a.bias = bias; a.dlast = dlast_state; a.softplus = softplus;
    a.dx = dx; a.draw = draw; a.dz = dz; a.kept = const_cast<float*>(kept); a.dstate = dstate; a.nrows = rows;
    set_strides(a, strides_host);
    const long long blocks = B * G * a.blocks_per_group, bc = rows * G * 2 * N;
    if (blocks > 0x7fffffffLL || ceil_div(bc, 256) > 0x7fffffffLL) PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_bwd: B=%lld D=%lld rows=%lld", (long long)B, (long long)D, (long long)rows);
    if (blocks > 0) {
        if (dtype == PPK_F32) run_bwd<float>(a, (unsigned)blocks, st);
        else run_bwd<bf16_t>(a, (unsigned)blocks, st);
    }
    if (bc > 0) {
        const unsigned nb = (unsigned)ceil_div(bc, 256);
        if (dtype == PPK_F32) k_scan_bc<float><<<nb, 256, 0, st>>>(a.pBC, a.blocks_per_group, rows, (int)G, (int)N, (float*)dB, (float*)dC);
        else k_scan_bc<bf16_t><<<nb, 256, 0, st>>>(a.pBC, a.blocks_per_group, rows, (int)G, (int)N, (bf16_t*)dB, (bf16_t*)dC);
    }
    rc = ppk::partial_sum(a.pA, B, D * N, dA, sum_ws, st);
    if (!rc && dskip) rc = ppk::partial_sum(a.pD, B, D, dskip, sum_ws, st);
    if (!rc && dbias) rc = ppk::partial_sum(a.pD + B * D, B, D, dbias, sum_ws, st);
    if (rc) return rc;
    PPK_CHECK_LAUNCH("selective_scan_bwd");
    return PPK_OK;
}

int ppk_selective_scan_step(int dtype, int64_t B, int64_t D, int64_t N, int64_t G, const void* x, const void* raw, const float* A, const void* Bm,
                            const void* Cm, const float* skip, const void* z, const float* bias, const float* state, int softplus, void* y,
                            float* new_state, const int64_t* strides_host, ppk_stream_t stream)
{
    int rc = scan_check("selective_scan_step", dtype, 1, B, D, N, G);
    if (rc) return rc;
    if (B == 0) return PPK_OK;
    if (!x || !raw || !A || !Bm || !Cm || !state || !y || !new_state || !strides_host) PPK_FAIL(PPK_ERR_NULL, "selective_scan_step: null pointer");
    ScanArgs a = {};
    a.q = {nullptr, nullptr, 1, B};
    a.D = (int)D; a.N = (int)N; a.G = (int)G; a.per = (int)(D / G);
    a.x = x; a.raw = raw; a.Bm = Bm; a.Cm = Cm; a.z = z; a.A = A; a.skip = skip; a.bias = bias; a.softplus = softplus; a.y = y;
    set_strides(a, strides_host);
    const long long blocks = ceil_div(B * D * slices(N), 256);
    if (blocks > 0x7fffffffLL) PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_step: B=%lld D=%lld", (long long)B, (long long)D);
    if (dtype == PPK_F32) run_step<float>(a, (unsigned)blocks, state, new_state, (hipStream_t)stream);
    else run_step<bf16_t>(a, (unsigned)blocks, state, new_state, (hipStream_t)stream);
    PPK_CHECK_LAUNCH("selective_scan_step");
    return PPK_OK;
}

}  // extern "C"
