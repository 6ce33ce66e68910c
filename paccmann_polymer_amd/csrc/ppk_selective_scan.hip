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
using ppk::Rows;
using ppk::uni_len;
using ppk::uniform;

constexpr int TILE = 16;                     // steps between two kept states
// Splits of the time axis: where the sequences and channels alone make less than a quarter of FWD_WAVES waves, one a SIMD (of BWD_BLOCKS blocks,
// two a CU), a split takes as many steps as make that many, and MIN_SPAN (BWD_MIN_SPAN) at least.  Measured, 16 states:
//   1 x 2048 x 1024 bf16 forward 65 us with 64 steps at least, 48 with 32, 41 with 16;
//   21 x 100 x 333 fp32 forward 41 us with 32 steps at least, 28 with 16;
//   64 x 256 x 1024 (1024 waves) fp32 forward 154 us in one piece, 170 in four splits; half the sequences 118 in one, 101 in eight;
//   32 x 256 x 1024 (512 blocks) fp32 training 266 us with the backward pass in one piece, 321 in splits;
//   1 x 16384 x 2048 bf16 training 1070 us with 1024 blocks, 1030 with 2048, 1050 with 4096;
//   21 x 100 x 333 fp32 backward 45 us in one launch, 42 in the three of a split.
constexpr long long MIN_SPAN = 16, BWD_MIN_SPAN = 64, FWD_WAVES = 4096, BWD_BLOCKS = 2048;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct ScanArgs {
    SeqBatch q;
    const int64_t* tiles;                    // device [B + 1]: first tile of each sequence, or null: rectangular
    int D, N, G, per;                        // per = D / G channels of a group
    int blocks_per_group;                    // channel blocks of a launch in a group
    int splits;                              // of the time axis, each of span steps (a multiple of TILE)
    long long span;
    const void *x, *raw, *Bm, *Cm, *z, *dy;
    const float *A, *skip, *bias, *state, *dlast;
    Stride xs, raws, Bs, Cs, zs, dys, rows;  // rows: of the outputs, in rows of their width
    long long Bg, Cg;                        // group strides
    int softplus;
    void *y, *dx, *draw, *dz;
    float *last, *kept, *dstate;             // kept: [tiles, D, N]
    float *carry, *sdt;                      // [B, splits, D, N], [B, splits, D]: what enters a split, and the sum of its dt
    float *pA, *pD, *pBC;                    // partial sums: [B splits, D, N], [2, B splits, D], [blocks_per_group, rows, G, 2, N]
    long long nrows;
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// A in the exponent of 2.  A state that forgets at once (A = -inf) keeps a finite exponent, which forgets all the same and leaves a dt of 0 one
__device__ __forceinline__ float base2(float A) { return A == -INFINITY ? -3.4e38f : A * LOG2E; }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2_(-LOG2E * x)); }
// log(1 + e^x) = max(x, 0) + log1p(u), u = e^-|x|.  w = 1 + u is rounded; log1p(u) = log(w) + (u - (w - 1)) / w to first order in what
// the rounding lost, which keeps a small dt (softplus of -7 is 1e-3) as exact as a large one.
__device__ __forceinline__ float softplus(float x)
{
    const float u = exp2_(-LOG2E * fabsf(x)), w = 1.0f + u;
    const float l = fmaf(u - (w - 1.0f), __builtin_amdgcn_rcpf(w), LN2 * __builtin_amdgcn_logf(w));
    return fmaxf(x, 0.0f) + l;                                 // a NaN comes through l
}
__device__ __forceinline__ float lane_value(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

__device__ __forceinline__ long long first_tile(const ScanArgs& a, long long b) { return a.tiles ? uniform<long long>(a.tiles)[b] : b * ((a.q.T + TILE - 1) / TILE); }

// N consecutive elements at a uniform address, 4-byte aligned, as scalars
template <typename T, int N> struct Scalars;
template <int N> struct Scalars<float, N> {
    float v[N];
    __device__ __forceinline__ void load(const float* p) { const UNIFORM float* u = uniform<float>(p);
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = u[n]; }
    __device__ __forceinline__ float at(int n) const { return v[n]; }
};
template <int N> struct Scalars<bf16_t, N> {
    unsigned v[N / 2];
    __device__ __forceinline__ void load(const bf16_t* p) { const UNIFORM unsigned* u = uniform<unsigned>(p);
#pragma unroll
        for (int n = 0; n < N / 2; ++n) v[n] = u[n]; }
    __device__ __forceinline__ float at(int n) const { return __uint_as_float(n & 1 ? v[n / 2] & 0xffff0000u : v[n / 2] << 16); }
};
// A step's B or C as the multiplications take it.  SCALAR: a row's N == NP elements begin on 4 bytes everywhere and are loaded as scalars, when
// the step begins.  Otherwise any N at any alignment: lane n has loaded element n some steps ahead (the lanes from N on: zero) and hands it over.
template <typename T, int NP, bool SCALAR> struct RowVec {
    Scalars<T, NP> s;
    float v;
    __device__ __forceinline__ void begin(const T* p, float ahead) { if constexpr (SCALAR) s.load(p); else v = ahead; }
    __device__ __forceinline__ float at(int n) const { if constexpr (SCALAR) return s.at(n); else return lane_value(v, n); }
};

// a lane's N states; `wide`: N == NP and they begin on 16 bytes in every lane
template <int NP> __device__ __forceinline__ void load_states(const float* p, int N, bool wide, float (&h)[NP])
{
    if (wide) {
#pragma unroll
        for (int n = 0; n < NP; n += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + n);
            h[n] = v.x; h[n + 1] = v.y; h[n + 2] = v.z; h[n + 3] = v.w;
        }
        return;
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) h[n] = p[n < N ? n : 0];
#pragma unroll
    for (int n = 0; n < NP; ++n) h[n] = n < N ? h[n] : 0.f;
}
template <int NP> __device__ __forceinline__ void store_states(float* p, int N, bool wide, const float (&h)[NP])
{
    if (wide) {
#pragma unroll
        for (int n = 0; n < NP; n += 4) *reinterpret_cast<float4*>(p + n) = make_float4(h[n], h[n + 1], h[n + 2], h[n + 3]);
        return;
    }
#pragma unroll
    for (int n = 0; n < NP; ++n)
        if (n < N) p[n] = h[n];
}
template <int NP> __device__ __forceinline__ bool wide_states(const void* p, int N) { return N == NP && ((uintptr_t)p & 15) == 0; }      // of an array's base

// What a wave of the kernels with a lane a channel works on: 64 channels of a group of one sequence, one split of its steps
struct Item {
    long long b;
    int t0, t1, len;                           // steps
    int s, g, d;                               // split, group, this lane's channel (a lane behind a group's last channel does that one again,
                                               // and stores the same values to the same places: no lane is masked)
    __device__ __forceinline__ Item(const ScanArgs& a)
    {
        const int nb = a.G * a.blocks_per_group, cb = (int)(blockIdx.x % nb);
        const long long rest = blockIdx.x / nb;
        s = (int)(rest % a.splits);
        b = rest / a.splits;
        g = cb / a.blocks_per_group;
        const int dl = (cb % a.blocks_per_group) * 64 + (int)threadIdx.x;
        d = g * a.per + (dl < a.per ? dl : a.per - 1);
        len = (int)uni_len(a.q, b);
        const long long first = s * a.span, last = first + a.span;
        t0 = first < len ? (int)first : len;
        t1 = last < len ? (int)last : len;
    }
};
__device__ __forceinline__ long long carry_at(const ScanArgs& a, long long b, int s, int d) { return (b * a.splits + s) * a.D + d; }

constexpr int AHEAD = 4;                       // steps whose elements are loaded before those of the steps before them are used (2: 5 % slower, 8: the same)

// rows of AHEAD steps from t on, in direction dir, none behind `last`
__device__ __forceinline__ void rows_of(const SeqBatch& q, int t, int last, int dir, unsigned (&rows)[AHEAD])
{
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) { const int u = t + dir * i; rows[i] = (unsigned)(dir > 0 ? (u < last ? u : last) : (u > last ? u : last)); }
    if (q.off)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) rows[i] = (unsigned)uniform<long long>(q.off)[rows[i]];
}

// The forward pass: a lane a channel with its NP >= N states in registers, B and C of a step in scalar registers (SCALAR) or handed over
// from lanes (at 32 states three waves a SIMD and 30 to 44 scalar registers spilled, at 64 one wave and 204 to 208: 64 x 256 x 1024 fp32 151 us at 16
// states, 252 at 32, 452 at 64; 17 and 33 do the work of 32 and 64).  PART: only the state at the end of a split that begins with none, and the sum of its dt.
template <typename T, int NP, bool SCALAR, bool PART>
__global__ __launch_bounds__(64) void k_scan_fwd(ScanArgs a)
{
    const Item it(a);
    const int lane = threadIdx.x, N = a.N;
    const int len = it.len, t0 = it.t0, t1 = it.t1;
    if (t0 >= len && it.s > 0) return;
    if (PART && t1 >= len) return;             // nothing enters a split behind the last
    float A2[NP], h[NP];
    load_states<NP>(a.A + (long long)it.d * N, N, wide_states<NP>(a.A, N), A2);
    if (PART || (a.splits == 1 && !a.state)) {
#pragma unroll
        for (int n = 0; n < NP; ++n) h[n] = 0.f;
    } else {
        const float* from = a.splits > 1 ? a.carry : a.state;
        load_states<NP>(from + (a.splits > 1 ? carry_at(a, it.b, it.s, it.d) : it.b * a.D + it.d) * N, N, wide_states<NP>(from, N), h);
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) A2[n] = base2(A2[n]);
    const float skip = !PART && a.skip ? a.skip[it.d] : 0.f, bias = a.bias ? a.bias[it.d] : 0.f;
    const long long tile_size = (long long)a.D * N;
    const bool kept_wide = wide_states<NP>(a.kept, N);
    float* kept = a.kept ? a.kept + ((first_tile(a, it.b) + t0 / TILE) * a.D + it.d) * N : nullptr;
    const Rows<T> xs(a.x, it.b * a.xs.b, a.xs.t), rs(a.raw, it.b * a.raws.b, a.raws.t), zs(a.z, it.b * a.zs.b, a.zs.t);
    const Rows<T> Bs(a.Bm, it.b * a.Bs.b + it.g * a.Bg, a.Bs.t), Cs(a.Cm, it.b * a.Cs.b + it.g * a.Cg, a.Cs.t), ys(a.y, it.b * a.rows.b * a.D, a.rows.t * a.D);
    const unsigned d = (unsigned)it.d * (unsigned)sizeof(T);
    const bool gate = !PART && a.z;
    T xv[AHEAD], rv[AHEAD], zv[AHEAD], bv[AHEAD], cv[AHEAD];
    unsigned rows[AHEAD];
    const unsigned own = (lane < N ? lane : 0) * (unsigned)sizeof(T);
    const auto fetch = [&](int t) {            // steps t, t + 1, ...; behind the last one, the last one
        rows_of(a.q, t, t1 - 1, 1, rows);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) { xv[i] = xs.get(rows[i], d); rv[i] = rs.get(rows[i], d); }
        if (!SCALAR)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) { bv[i] = Bs.get(rows[i], own); if (!PART) cv[i] = Cs.get(rows[i], own); }
        if (gate)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) zv[i] = zs.get(rows[i], d);
    };
    float sum = 0.f;
    if (t0 < t1) fetch(t0);
    for (int t = t0; t < t1; t += AHEAD) {
        if (!PART && kept && t % TILE == 0) { store_states<NP>(kept, N, kept_wide, h); kept += tile_size; }
        float x[AHEAD], raw[AHEAD], z[AHEAD], bl[AHEAD], cl[AHEAD];
        unsigned r[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            bl[i] = !SCALAR && lane < N ? to_f32(bv[i]) : 0.f;
            cl[i] = !SCALAR && !PART && lane < N ? to_f32(cv[i]) : 0.f;
            x[i] = to_f32(xv[i]); raw[i] = to_f32(rv[i]) + bias; z[i] = gate ? to_f32(zv[i]) : 0.f; r[i] = rows[i]; }
        if (t + AHEAD < t1) fetch(t + AHEAD);
        const auto step = [&](int i) {
            __builtin_amdgcn_sched_barrier(0);     // one step's scalars at a time: those of all do not fit
            RowVec<T, NP, SCALAR> Bv, Cv;
            Bv.begin((const T*)Bs.row(r[i]), bl[i]);
            if (!PART) Cv.begin((const T*)Cs.row(r[i]), cl[i]);
            const float dt = a.softplus ? softplus(raw[i]) : raw[i], dx = dt * x[i];
            float y[4] = {!PART && a.skip ? skip * x[i] : 0.f, 0.f, 0.f, 0.f};     // no D: no term, which an infinite x would make NaN of
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                h[n] = fmaf(exp2_(dt * A2[n]), h[n], dx * Bv.at(n));
                if (!SCALAR && !PART) h[n] = n < N ? h[n] : 0.f;               // an infinite dx makes NaN of a state that does not exist
                if (!PART) y[n & 3] = fmaf(h[n], Cv.at(n), y[n & 3]);
            }
            if (PART) { sum += dt; return; }
            float out = (y[0] + y[1]) + (y[2] + y[3]);
            if (gate) out *= z[i] * sigmoid(z[i]);
            ys.put(r[i], d, from_f32<T>(out));
        };
        if (PART || t + AHEAD <= t1) {             // a split that is not a sequence's last has whole groups only
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) step(i);
        } else {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (t + i < t1) step(i);
        }
    }
    if (PART) {
        store_states<NP>(a.carry + carry_at(a, it.b, it.s, it.d) * N, N, wide_states<NP>(a.carry, N), h);
        a.sdt[carry_at(a, it.b, it.s, it.d)] = sum;
    } else if (t1 == len) store_states<NP>(a.last + (it.b * a.D + it.d) * N, N, wide_states<NP>(a.last, N), h);
}

// What the gradient of the state at the end of a split becomes at its beginning, without what enters at the end: g = a (g + dy' C),
// from the last step to the first, and the sum of its dt.  Laid out as the forward pass.
template <typename T, int NP, bool SCALAR>
__global__ __launch_bounds__(64) void k_scan_bwd_part(ScanArgs a)
{
    const Item it(a);
    const int lane = threadIdx.x, N = a.N;
    const int t0 = it.t0, t1 = it.t1;
    if (t0 >= it.len || it.s == 0) return;     // nothing leaves the first
    float A2[NP], g[NP];
    load_states<NP>(a.A + (long long)it.d * N, N, wide_states<NP>(a.A, N), A2);
#pragma unroll
    for (int n = 0; n < NP; ++n) { A2[n] = base2(A2[n]); g[n] = 0.f; }
    const float bias = a.bias ? a.bias[it.d] : 0.f;
    const Rows<T> ds(a.dy, it.b * a.dys.b, a.dys.t), rs(a.raw, it.b * a.raws.b, a.raws.t), zs(a.z, it.b * a.zs.b, a.zs.t);
    const Rows<T> Cs(a.Cm, it.b * a.Cs.b + it.g * a.Cg, a.Cs.t);
    const unsigned d = (unsigned)it.d * (unsigned)sizeof(T);
    T dv[AHEAD], rv[AHEAD], zv[AHEAD], cv[AHEAD];
    unsigned rows[AHEAD];
    const unsigned own = (lane < N ? lane : 0) * (unsigned)sizeof(T);
    const auto fetch = [&](int t) {            // steps t - 1, t - 2, ...; before the first one, the first one
        rows_of(a.q, t - 1, t0, -1, rows);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) { dv[i] = ds.get(rows[i], d); rv[i] = rs.get(rows[i], d); if (!SCALAR) cv[i] = Cs.get(rows[i], own); }
        if (a.z)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) zv[i] = zs.get(rows[i], d);
    };
    float sum = 0.f;
    fetch(t1);
    for (int t = t1; t > t0; t -= AHEAD) {
        float dy[AHEAD], raw[AHEAD], cl[AHEAD];
        unsigned r[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            cl[i] = !SCALAR && lane < N ? to_f32(cv[i]) : 0.f;
            const float z = a.z ? to_f32(zv[i]) : 0.f;
            dy[i] = to_f32(dv[i]) * (a.z ? z * sigmoid(z) : 1.0f);
            raw[i] = to_f32(rv[i]) + bias;
            r[i] = rows[i];
        }
        if (t - AHEAD > t0) fetch(t - AHEAD);
        const auto step = [&](int i) {
            __builtin_amdgcn_sched_barrier(0);
            RowVec<T, NP, SCALAR> Cv;
            Cv.begin((const T*)Cs.row(r[i]), cl[i]);
            const float dt = a.softplus ? softplus(raw[i]) : raw[i];
            sum += dt;
#pragma unroll
            for (int n = 0; n < NP; ++n) g[n] = exp2_(dt * A2[n]) * fmaf(dy[i], Cv.at(n), g[n]);
        };
        if (t - AHEAD >= t0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) step(i);
        } else {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (t - 1 - i >= t0) step(i);
        }
    }
    store_states<NP>(a.carry + carry_at(a, it.b, it.s, it.d) * N, N, wide_states<NP>(a.carry, N), g);
    a.sdt[carry_at(a, it.b, it.s, it.d)] = sum;
}

// Joins the splits of a sequence: carry[s] holds what split s gives alone and receives what enters it.  Forward from the state before
// the first step, backward (REV) from the gradient of the state behind the last.  h' = decay h + own is associative: a block takes
// JOIN_STATES states and as many slices of the splits as make 256 threads, each slice joins its own, then the slices.  Bound by the latency of its
// loads: 128 splits of 1024 channels x 16 states 8.2 us (a thread a state, one split after the other: 12; 16 states a block: 12, 64: 9.0).
constexpr int JOIN_STATES = 32;
// decay x + own.  No step's decay is 0 or infinite, but that of many steps may be beyond fp32: a state of 0 stays 0 and an infinite one infinite all the same.
__device__ __forceinline__ float carried(float decay, float x, float own)
{
    constexpr int ZERO_OR_INF = 0x264;
    return __builtin_amdgcn_classf(x, ZERO_OR_INF) ? x + own : fmaf(decay, x, own);
}
template <bool REV, int U>
__global__ __launch_bounds__(256) void k_scan_join(ScanArgs a)
{
    constexpr int S = 256 / JOIN_STATES;                             // slices of the splits; U of a slice's are held at once
    __shared__ float s_end[S][JOIN_STATES], s_decay[S][JOIN_STATES];
    const int slice = threadIdx.x / JOIN_STATES, el = threadIdx.x % JOIN_STATES;
    const long long dn = (long long)a.D * a.N, e0 = (long long)blockIdx.x * JOIN_STATES + el, b = blockIdx.y;
    const bool live = e0 < dn;
    const long long e = live ? e0 : 0;
    const int d = (int)(e / a.N);
    const float A2 = base2(a.A[e]);
    const float* from = REV ? a.dlast : a.state;
    const long long len = uni_len(a.q, b);
    const int used = len > 0 ? (int)((len + a.span - 1) / a.span) : 1;          // no steps: the first split still hands on what enters it
    float in = from ? from[b * dn + e] : 0.f;
    const long long dir = REV ? -1 : 1, first = b * a.splits + (REV ? used - 1 : 0);
    float* c = a.carry + first * dn + e;
    const float* sd = a.sdt + first * a.D + d;
    for (int k0 = 0; k0 < used; k0 += S * U) {
        const int many = used - k0 < S * U ? used - k0 : S * U, per = (many + S - 1) / S, k1 = k0 + slice * per;
        const int n = many - slice * per < per ? many - slice * per : per;      // 0 or less: nothing left for this slice
        float own[U], by[U], end = 0.f, decay = 0.f;                             // decay: its exponent
        // The part of the last split on the way (forward the sequence's last, backward its first) is not made: nobody asks for it.  Loads are
        // not masked, so that all of them fly together: one behind the last made is that one again.
        const int last = used > 1 ? used - 2 : 0;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int k = k1 + i < last ? k1 + i : last;
            own[i] = c[dir * k * dn];
            by[i] = sd[dir * k * a.D];
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const bool made = i < n && k1 + i + 1 < used;
            own[i] = made ? own[i] : 0.f;
            by[i] = made ? by[i] * A2 : 0.f;
            decay += by[i];
            by[i] = exp2_(by[i]);
            end = carried(by[i], end, own[i]);
        }
        s_end[slice][el] = end;
        s_decay[slice][el] = exp2_(decay);
        __syncthreads();
        float mine = in;
#pragma unroll
        for (int k = 0; k < S; ++k) {
            if (k == slice) mine = in;
            in = carried(s_decay[k][el], in, s_end[k][el]);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (live && i < n) c[dir * (k1 + i) * dn] = mine;
            mine = carried(by[i], mine, own[i]);
        }
        __syncthreads();
    }
}

// sum over the LPC lanes of a row of 16 that share their low bits (of which there are 16 / LPC values)
template <int LPC> __device__ __forceinline__ float sum_slices(float v)
{
    if (LPC > 8) v += dpp_of<DPP_XOR1>(v);
    if (LPC > 4) v += dpp_of<DPP_XOR2>(v);
    v += dpp_of<DPP_ROR4>(v);
    v += dpp_of<DPP_ROR8>(v);
    return v;
}
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// Parts of a tile: a sequence's last tile is worked on as far as the part that its last step is in.  Least times of 2048 sequences of 20 to 100
// steps, 512 channels, 16 states, fp32: 1130-1170 us with parts of two steps, 1177 with three parts, 1223 with whole tiles; 1 x 16384 x 2048 bf16
// (whole tiles only): 535-550, 530 with three.  Parts of two steps: only their second can be one that does not exist.
constexpr int NPARTS = 8, PART = TILE / NPARTS, FETCH_PART = 4;

// The backward pass.  A block takes 256 / LPC channels of a group of one sequence and walks a split's tiles backwards; a thread holds the
// four states 4 slice .. of a channel.  In a wave, lane % 16 = slice * (16 / LPC) + low bits of the channel, lane / 16 = its high bits:
//   sums over states go over the slices, within a row of 16 lanes (two to four DPP additions);
//   sums over channels (dB, dC of a step: eight values a thread) halve what a lane holds at each exchange of half waves.
//   The matrix unit can make them too, with the value as one operand and a unit column as the other: 128 products a tile instead of
//   256 vector instructions, and slower: 1574 against 1222 us on 2048 sequences of 20 to 100 steps, 512 channels, 16 states, fp32, where the
//   matrix unit and the vector unit were busy for 80 % of the time together, one after the other.
// Elements of a tile are loaded while the tile behind it is worked on, and what the tile's end needs of them waits in LDS.
// FULL: N is 4 LPC and the channels of a group are whole blocks.  Otherwise states and channels that do not exist are kept at zero: their products
// with an infinite input, B, C or gradient would be NaN, and sums over states and channels take them in (21 sequences, 333 channels of three
// groups, 11 states: 47 us, 44 without).
// Bound by the vector unit at two waves a SIMD: 16 steps of states and decays are 132 of 256 registers, and at 16 states 4 more and 70 to 76 scalar
// ones are spilled (up to 84 bytes of scratch a lane).
template <typename T, int LPC, bool FULL>
__global__ __launch_bounds__(256, 2) void k_scan_bwd(ScanArgs a)
{
    constexpr int NP = 4 * LPC, BC = 256 / LPC, PE = TILE * BC / 256, CL = 16 / LPC, BCE = TILE * 2 * NP / 256;
    __shared__ float s_dt[TILE][BC], s_dx[TILE][BC], s_dy[TILE][BC];           // dt, dt x, dy'
    __shared__ float s_x[TILE][BC], s_slope[TILE][BC], s_gz[TILE][BC];         // x, d dt / d raw, dout silu'(z)
    __shared__ float s_q[4][TILE][BC];                                         // sums over n of dh B, da A, C h
    __shared__ __align__(16) float s_BC[TILE][2 * NP];
    __shared__ __align__(16) float s_red[TILE][4][2 * NP];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int ns = (lane & 15) / CL, ch = wave * (64 / LPC) + (lane >> 4) * CL + (lane & (CL - 1));    // the scan's slice and channel
    const int pc = tid % BC, pt = BC >= 64 ? __builtin_amdgcn_readfirstlane(tid / BC) : tid / BC;      // channel and first step of the per-element work
    const int nb = a.G * a.blocks_per_group, N = a.N;
    const long long item = blockIdx.x / nb, b = item / a.splits;               // item: sequence and split
    const int s = (int)(item % a.splits);
    const int cb = (int)(blockIdx.x % nb), g = cb / a.blocks_per_group, cg = cb % a.blocks_per_group;
    const int base = cg * BC;                                                  // of the block's channels in the group
    const bool live = base + ch < a.per, plive = base + pc < a.per;
    const int d = g * a.per + (live ? base + ch : 0), pd = g * a.per + (plive ? base + pc : 0);
    const long long len = uni_len(a.q, b), end = (s + 1) * a.span < len ? (s + 1) * a.span : len;
    const long long tile0 = first_tile(a, b);
    float A2[4], dA[4] = {0.f, 0.f, 0.f, 0.f}, dh[4];
    bool exists[4];
    const float* into = a.splits > 1 && s * a.span < len ? a.carry + carry_at(a, b, s, d) * N : (a.dlast ? a.dlast + (b * a.D + d) * N : nullptr);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = ns * 4 + j;
        exists[j] = live && n < N;
        A2[j] = live ? base2(a.A[(long long)d * N + (n < N ? n : 0)]) : 0.f;          // a state that does not exist decays as one that does
        dh[j] = exists[j] && into ? into[n] : 0.f;
    }
    const float skip = a.skip && plive ? a.skip[pd] : 0.f, bias = a.bias && plive ? a.bias[pd] : 0.f;
    const bool has_skip = a.skip != nullptr;
    float dskip = 0.f, dbias = 0.f;

    const Rows<T> xs(a.x, b * a.xs.b, a.xs.t), rs(a.raw, b * a.raws.b, a.raws.t), ds(a.dy, b * a.dys.b, a.dys.t);
    const Rows<T> zs(a.z ? a.z : a.x, b * (a.z ? a.zs.b : a.xs.b), a.z ? a.zs.t : a.xs.t);      // no gate: x again, unused
    const unsigned pb = (unsigned)pd * (unsigned)sizeof(T);
    // this thread's element of a row's B and C: column (tid % (2 NP)) of every 256 / (2 NP)-th row
    const int bk = tid % (2 * NP), bn = bk % NP, bt = tid / (2 * NP);
    const Rows<T> bcs(bk < NP ? a.Bm : a.Cm, (bk < NP ? b * a.Bs.b + g * a.Bg : b * a.Cs.b + g * a.Cg) + (bn < N ? bn : 0), bk < NP ? a.Bs.t : a.Cs.t);
    const Rows<T> dxs(a.dx, b * a.rows.b * a.D, a.rows.t * a.D), drs(a.draw, b * a.rows.b * a.D, a.rows.t * a.D), dzs(a.dz, b * a.rows.b * a.D, a.rows.t * a.D);
    const float* h0 = a.kept + (tile0 * a.D + d) * N + (ns * 4 < N ? ns * 4 : 0);
    T xv[PE], rv[PE], dv[PE], zv[PE], bv[BCE];
    unsigned row[PE], brow[BCE];
    f32x4 hv;
    const auto locate = [&](long long tile) {                                  // the rows of a tile; a step behind the last is the first one again
        const unsigned t0 = (unsigned)(tile * TILE);
        const int steps = (int)(end - tile * TILE < TILE ? end - tile * TILE : TILE);
#pragma unroll
        for (int i = 0; i < PE; ++i) { const int t = pt + i * (256 / BC); row[i] = t0 + (t < steps ? t : 0); }
#pragma unroll
        for (int i = 0; i < BCE; ++i) { const int t = bt + i * (256 / (2 * NP)); brow[i] = t0 + (t < steps ? t : 0); }
        if (!a.q.off) return;
#pragma unroll
        for (int i = 0; i < PE; ++i) row[i] = BC >= 64 ? (unsigned)uniform<long long>(a.q.off)[row[i]] : (unsigned)a.q.off[row[i]];
#pragma unroll
        for (int i = 0; i < BCE; ++i) brow[i] = (unsigned)a.q.off[brow[i]];
    };
    const auto fetch = [&](long long tile) {
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            xv[i] = xs.get(row[i], pb);
            rv[i] = rs.get(row[i], pb);
            dv[i] = ds.get(row[i], pb);
            zv[i] = zs.get(row[i], pb);
        }
#pragma unroll
        for (int i = 0; i < BCE; ++i) bv[i] = bcs.get(brow[i], 0);
        const float* p = h0 + tile * (long long)a.D * N;
#pragma unroll
        for (int j = 0; j < 4; ++j) hv[j] = p[ns * 4 + j < N ? j : 0];
    };
    const long long tile_end = (end + TILE - 1) / TILE, tile_begin = s * (a.span / TILE);
    if (tile_end > tile_begin) { locate(tile_end - 1); fetch(tile_end - 1); }
    for (long long tile = tile_end - 1; tile >= tile_begin; --tile) {
        const long long t0 = tile * TILE;
        const int steps = (int)(end - t0 < TILE ? end - t0 : TILE);
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            const int t = pt + i * (256 / BC);
            const bool in = plive && t < steps;
            const float x = in ? to_f32(xv[i]) : 0.f, raw = in ? to_f32(rv[i]) + bias : 0.f, dout = in ? to_f32(dv[i]) : 0.f;
            const float dt = in ? (a.softplus ? softplus(raw) : raw) : 0.f;
            float dy = dout, gz = 0.f;
            if (a.z) {
                const float z = in ? to_f32(zv[i]) : 0.f, sg = sigmoid(z), zs = z * sg;
                dy = dout * zs;
                gz = dout * fmaf(zs, 1.0f - sg, sg);
            }
            s_dt[t][pc] = dt;
            s_dx[t][pc] = dt * x;
            s_dy[t][pc] = dy;
            s_x[t][pc] = x;
            s_slope[t][pc] = a.softplus ? sigmoid(raw) : 1.0f;
            s_gz[t][pc] = gz;
        }
#pragma unroll
        for (int i = 0; i < BCE; ++i) {
            const int t = bt + i * (256 / (2 * NP));
            s_BC[t][bk] = t < steps && bn < N ? to_f32(bv[i]) : 0.f;
        }
        float h[TILE + 1][4], av[TILE][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[0][j] = live && ns * 4 + j < N ? hv[j] : 0.f;
        const long long next = tile > tile_begin ? tile - 1 : tile;
        locate(next);
        __syncthreads();
#pragma unroll
        for (int part = 0; part < NPARTS; ++part) {
            if (part * PART >= steps) break;
#pragma unroll
            for (int t = part * PART; t < (part + 1) * PART; ++t) {
                const float dtv = s_dt[t][ch], dxv = s_dx[t][ch];
                const f32x4 Bv = *reinterpret_cast<const f32x4*>(&s_BC[t][ns * 4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    av[t][j] = exp2_(dtv * A2[j]);
                    h[t + 1][j] = fmaf(av[t][j], h[t][j], FULL || exists[j] ? dxv * Bv[j] : 0.f);
                }
            }
        }
        asm volatile("" ::: "memory");           // the steps' values are read from LDS again: kept, they would be 96 registers
#pragma unroll
        for (int part = NPARTS - 1; part >= 0; --part) {
            if (part == FETCH_PART) fetch(next);                                // where the registers of the parts behind it are free again
            if (part * PART >= steps) continue;
#pragma unroll
            for (int t = (part + 1) * PART - 1; t >= part * PART; --t) {
                const float dtv = s_dt[t][ch], dxv = s_dx[t][ch], dyv = s_dy[t][ch];
                const f32x4 Bv = *reinterpret_cast<const f32x4*>(&s_BC[t][ns * 4]), Cv = *reinterpret_cast<const f32x4*>(&s_BC[t][NP + ns * 4]);
                float q1 = 0.f, q2 = 0.f, q3 = 0.f, v[8];                           // v: dB of the four states, then dC
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    dh[j] = FULL || exists[j] ? fmaf(dyv, Cv[j], dh[j]) : 0.f;
                    q1 = fmaf(dh[j], Bv[j], q1);
                    v[j] = dh[j] * dxv;
                    v[4 + j] = dyv * h[t + 1][j];
                    q3 = fmaf(Cv[j], h[t + 1][j], q3);
                    dh[j] *= av[t][j];
                    const float da = dh[j] * h[t][j];
                    q2 = fmaf(da, A2[j], q2);
                    // a step that does not exist has a dt of 0, but an infinite state may enter it; nothing has been added before the sequence's last step
                    dA[j] = t == part * PART || t < steps ? fmaf(da, dtv, dA[j]) : 0.f;
                }
                q1 = sum_slices<LPC>(q1);
                q2 = sum_slices<LPC>(q2);
                q3 = sum_slices<LPC>(q3);
                s_q[ns & 3][t][ch] = (ns & 3) == 0 ? q1 : (ns & 3) == 1 ? q2 : q3;   // every slice holds all three: the fourth writes nobody's
                // over the wave's channels: two exchanges of halves leave a lane the sums of two of the eight values (bit 5 of the lane: dC,
                // bit 4: the upper two states), the low bits of the channel follow within a row of 16
                float u[4], w[2];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[k]), __float_as_uint(v[k + 4]), false, false);
                    u[k] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(u[k]), __float_as_uint(u[k + 2]), false, false);
                    w[k] = lanes_sum<CL>(__uint_as_float(p[0]) + __uint_as_float(p[1]));
                }
                // CL lanes hold the same two sums and store them to the same place
                *reinterpret_cast<f32x2*>(&s_red[t][wave][(lane >> 5) * NP + ns * 4 + ((lane >> 4) & 1) * 2]) = f32x2{w[0], w[1]};
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PE; ++i) {
            const int t = pt + i * (256 / BC);
            if (!(plive && t < steps)) continue;
            const unsigned r = BC >= 64 ? uni_row(a.q, t0 + t) : (unsigned)a.q.row(t0 + t);
            const float q1 = s_q[0][t][pc], x = s_x[t][pc], dy = s_dy[t][pc];
            const float dr = fmaf(x, q1, s_q[1][t][pc] * LN2) * s_slope[t][pc];
            dxs.put(r, pb, from_f32<T>(fmaf(s_dt[t][pc], q1, skip * (has_skip ? dy : 0.f))));
            drs.put(r, pb, from_f32<T>(dr));
            if (a.z) dzs.put(r, pb, from_f32<T>(s_gz[t][pc] * fmaf(skip, has_skip ? x : 0.f, s_q[2][t][pc])));
            dskip = fmaf(dy, x, dskip);
            dbias += dr;
        }
#pragma unroll
        for (int i = 0; i < BCE; ++i) {
            const int t = bt + i * (256 / (2 * NP));
            if (t >= steps || bn >= N) continue;
            const long long row = at(a.rows, a.q.row(t0 + t), b);
            a.pBC[(((long long)cg * a.nrows + row) * a.G + g) * 2 * N + (bk < NP ? 0 : N) + bn] = (s_red[t][0][bk] + s_red[t][1][bk]) + (s_red[t][2][bk] + s_red[t][3][bk]);
        }
        __syncthreads();
    }
    if (live)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = ns * 4 + j;
            if (n >= N) continue;
            a.pA[(item * a.D + d) * N + n] = dA[j];
            if (a.dstate && s == 0) a.dstate[(b * a.D + d) * N + n] = dh[j];
        }
    s_dt[pt][pc] = dskip;
    s_dx[pt][pc] = dbias;
    __syncthreads();
    if (pt == 0 && plive) {
        float u = s_dt[0][pc], v = s_dx[0][pc];
        for (int i = 1; i < 256 / BC; ++i) { u += s_dt[i][pc]; v += s_dx[i][pc]; }
        a.pD[item * a.D + pd] = u;
        a.pD[(a.q.B * a.splits + item) * a.D + pd] = v;
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

// One token of each sequence: lane = channel * LPC + slice, four states a thread.  WIDE: they begin on 16 bytes, and those of B and C
// on four elements, everywhere: a wave then reads and writes a kilobyte of states at a time.
template <typename T> struct alignas(4 * sizeof(T)) Quad { T v[4]; };
template <typename T, int LPC, bool WIDE>
__global__ __launch_bounds__(256) void k_scan_step(ScanArgs a, const float* state, float* next)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const int ns = (int)(e % LPC), N = a.N;
    const long long bd = e / LPC;
    if (bd >= a.q.B * a.D) return;                                             // whole groups of LPC lanes
    const long long b = bd / a.D;
    const int d = (int)(bd - b * a.D), g = d / a.per;
    float A[4], h[4], Bv[4], Cv[4];
    const T *Bp = (const T*)a.Bm + b * a.Bs.b + g * a.Bg + ns * 4, *Cp = (const T*)a.Cm + b * a.Cs.b + g * a.Cg + ns * 4;
    const long long at_A = (long long)d * N + ns * 4, at_h = bd * N + ns * 4;
    if (WIDE) {
        const float4 u = *reinterpret_cast<const float4*>(state + at_h), v = *reinterpret_cast<const float4*>(a.A + at_A);
        const Quad<T> p = *reinterpret_cast<const Quad<T>*>(Bp), q = *reinterpret_cast<const Quad<T>*>(Cp);
        h[0] = u.x; h[1] = u.y; h[2] = u.z; h[3] = u.w;
        A[0] = v.x; A[1] = v.y; A[2] = v.z; A[3] = v.w;
#pragma unroll
        for (int j = 0; j < 4; ++j) { Bv[j] = to_f32(p.v[j]); Cv[j] = to_f32(q.v[j]); }
    } else
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = ns * 4 + j < N;
            h[j] = in ? state[at_h + j] : 0.f;
            A[j] = in ? a.A[at_A + j] : 0.f;
            Bv[j] = in ? to_f32(Bp[j]) : 0.f;
            Cv[j] = in ? to_f32(Cp[j]) : 0.f;
        }
    const float x = to_f32(((const T*)a.x)[b * a.xs.b + d]);
    const float raw = to_f32(((const T*)a.raw)[b * a.raws.b + d]) + (a.bias ? a.bias[d] : 0.f);
    const float z = a.z ? to_f32(((const T*)a.z)[b * a.zs.b + d]) : 0.f;
    const float skip = (a.skip ? a.skip : a.A)[d];                             // no D: any of A's, unused; behind a branch the load is late (15.0 -> 15.6 us)
    const float dt = a.softplus ? softplus(raw) : raw, dx = dt * x;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = fmaf(exp2_(dt * base2(A[j])), h[j], dx * Bv[j]);
        if (!WIDE) h[j] = ns * 4 + j < N ? h[j] : 0.f;                         // an infinite dx makes NaN of a state that does not exist
        y = fmaf(h[j], Cv[j], y);
    }
    if (WIDE) *reinterpret_cast<float4*>(next + at_h) = make_float4(h[0], h[1], h[2], h[3]);
    else
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (ns * 4 + j < N) next[at_h + j] = h[j];
    y = lanes_sum<LPC>(y) + (a.skip ? skip * x : 0.f);
    if (a.z) y *= z * sigmoid(z);
    if (ns == 0) ((T*)a.y)[bd] = from_f32<T>(y);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
int slices(long long N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
int bwd_slices(long long N) { return N <= 16 ? 4 : N <= 32 ? 8 : 16; }
int padded(long long N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

// How many steps a split of the time axis takes.  `units`: what runs at once without one, `want`: what fills the card.
long long span_of(long long T, long long units, long long want, long long least)
{
    const long long all = ceil_div(T > 0 ? T : 1, TILE) * TILE;
    if (units * 4 >= want || all <= 2 * least) return all;
    const long long span = ceil_div(ceil_div(all * units, want), TILE) * TILE;
    return span > least ? span : least;
}
struct Plan { long long blocks_per_group, span, splits; };
Plan plan_of(long long T, long long B, long long D, long long G, long long channels, long long want, long long least)
{
    Plan p;
    p.blocks_per_group = ceil_div(D / G, channels);
    p.span = span_of(T, B * G * p.blocks_per_group, want, least);
    p.splits = ceil_div(T > 0 ? T : 1, p.span);
    return p;
}
Plan fwd_plan(long long T, long long B, long long D, long long G) { return plan_of(T, B, D, G, 64, FWD_WAVES, MIN_SPAN); }
Plan bwd_plan(long long T, long long B, long long D, long long N, long long G) { return plan_of(T, B, D, G, 256 / bwd_slices(N), BWD_BLOCKS, BWD_MIN_SPAN); }
size_t carry_bytes(long long B, long long D, long long N, long long splits)
{
    return splits > 1 ? ppk_align_up((size_t)B * splits * D * N * 4, 256) + ppk_align_up((size_t)B * splits * D * 4, 256) : 0;
}

// SCALAR of the kernels: rows of exactly NP elements that begin on 4 bytes
template <typename T> bool scalar_rows(const void* p, const Stride& s, long long group, int N)
{
    const long long per = 4 / (long long)sizeof(T);
    return N == padded(N) && ((uintptr_t)p & 3) == 0 && s.t % per == 0 && s.b % per == 0 && group % per == 0;
}
template <typename T, int NP, bool SCALAR> void launch_fwd(const ScanArgs& a, bool part, unsigned blocks, hipStream_t st)
{
    if (part) k_scan_fwd<T, NP, SCALAR, true><<<blocks, 64, 0, st>>>(a);
    else k_scan_fwd<T, NP, SCALAR, false><<<blocks, 64, 0, st>>>(a);
}
template <typename T> void run_fwd(const ScanArgs& a, bool part, unsigned blocks, hipStream_t st)
{
    const bool sc = scalar_rows<T>(a.Bm, a.Bs, a.Bg, a.N) && scalar_rows<T>(a.Cm, a.Cs, a.Cg, a.N);
    switch (padded(a.N)) {
        case 8: if (sc) launch_fwd<T, 8, true>(a, part, blocks, st); else launch_fwd<T, 8, false>(a, part, blocks, st); break;
        case 16: if (sc) launch_fwd<T, 16, true>(a, part, blocks, st); else launch_fwd<T, 16, false>(a, part, blocks, st); break;
        case 32: launch_fwd<T, 32, false>(a, part, blocks, st); break;
        default: launch_fwd<T, 64, false>(a, part, blocks, st);
    }
}
template <typename T> void run_bwd_part(const ScanArgs& a, unsigned blocks, hipStream_t st)
{
    const bool sc = scalar_rows<T>(a.Cm, a.Cs, a.Cg, a.N);
    switch (padded(a.N)) {
        case 8: if (sc) k_scan_bwd_part<T, 8, true><<<blocks, 64, 0, st>>>(a); else k_scan_bwd_part<T, 8, false><<<blocks, 64, 0, st>>>(a); break;
        case 16: if (sc) k_scan_bwd_part<T, 16, true><<<blocks, 64, 0, st>>>(a); else k_scan_bwd_part<T, 16, false><<<blocks, 64, 0, st>>>(a); break;
        case 32: k_scan_bwd_part<T, 32, false><<<blocks, 64, 0, st>>>(a); break;
        default: k_scan_bwd_part<T, 64, false><<<blocks, 64, 0, st>>>(a);
    }
}
template <bool REV> void join(const ScanArgs& a, long long B, hipStream_t st)
{
    const dim3 grid((unsigned)ceil_div((long long)a.D * a.N, JOIN_STATES), (unsigned)B);
    if (a.splits <= 4 * 256 / JOIN_STATES) k_scan_join<REV, 4><<<grid, 256, 0, st>>>(a);
    else k_scan_join<REV, 16><<<grid, 256, 0, st>>>(a);
}
template <typename T, int LPC> void launch_bwd(const ScanArgs& a, unsigned blocks, hipStream_t st)
{
    if (a.N == 4 * LPC && a.per % (256 / LPC) == 0) k_scan_bwd<T, LPC, true><<<blocks, 256, 0, st>>>(a);
    else k_scan_bwd<T, LPC, false><<<blocks, 256, 0, st>>>(a);
}
template <typename T> void run_bwd(const ScanArgs& a, unsigned blocks, hipStream_t st)
{
    switch (bwd_slices(a.N)) {
        case 4: launch_bwd<T, 4>(a, blocks, st); break;
        case 8: launch_bwd<T, 8>(a, blocks, st); break;
        default: launch_bwd<T, 16>(a, blocks, st);
    }
}
template <typename T, int LPC> void launch_step(const ScanArgs& a, unsigned blocks, const float* state, float* next, hipStream_t st)
{
    const uintptr_t p = (uintptr_t)state | (uintptr_t)next | (uintptr_t)a.A, q = (uintptr_t)a.Bm | (uintptr_t)a.Cm;
    const long long s = a.Bs.b | a.Bg | a.Cs.b | a.Cg;
    if (a.N == 4 * LPC && p % 16 == 0 && q % (4 * sizeof(T)) == 0 && s % 4 == 0) k_scan_step<T, LPC, true><<<blocks, 256, 0, st>>>(a, state, next);
    else k_scan_step<T, LPC, false><<<blocks, 256, 0, st>>>(a, state, next);
}
template <typename T> void run_step(const ScanArgs& a, unsigned blocks, const float* state, float* next, hipStream_t st)
{
    switch (slices(a.N)) {
        case 1: launch_step<T, 1>(a, blocks, state, next, st); break;
        case 2: launch_step<T, 2>(a, blocks, state, next, st); break;
        case 4: launch_step<T, 4>(a, blocks, state, next, st); break;
        case 8: launch_step<T, 8>(a, blocks, state, next, st); break;
        default: launch_step<T, 16>(a, blocks, state, next, st);
    }
}

// rows are at most 2^32 bytes apart (a tensor of strides that reach further is copied by its caller)
bool near_rows(const int64_t* s, long long D)
{
    for (int i : {0, 2, 4, 7, 10, 14})
        if (s[i] < 0 || s[i] >= 1LL << 30) return false;
    return s[12] >= 0 && s[12] < (1LL << 30) / D;
}
int scan_check(const char* what, int dtype, long long T, long long B, long long D, long long N, long long G)
{
    if (dtype != PPK_F32 && dtype != PPK_BF16) PPK_FAIL(PPK_ERR_UNSUP, "%s: type %d (fp32 and bf16 are supported)", what, dtype);
    if (T < 0 || B < 0 || D < 1 || N < 1 || G < 1 || D % G) PPK_FAIL(PPK_ERR_SHAPE, "%s: T=%lld B=%lld D=%lld N=%lld G=%lld", what, T, B, D, N, G);
    if (N > 64) PPK_FAIL(PPK_ERR_UNSUP, "%s: %lld states a channel (at most 64)", what, N);
    if (D > (1 << 20)) PPK_FAIL(PPK_ERR_UNSUP, "%s: %lld channels", what, D);
    if (T >= 1LL << 30 || B >= 1LL << 31) PPK_FAIL(PPK_ERR_UNSUP, "%s: %lld steps of B=%lld sequences", what, T, B);
    return PPK_OK;
}

struct BwdWs { size_t a, d, bc, carry, sum, total; Plan p; };
BwdWs bwd_ws(long long T, long long B, long long D, long long N, long long G, long long rows)
{
    BwdWs w;
    w.p = bwd_plan(T, B, D, N, G);
    const long long items = B * w.p.splits;
    w.a = ppk_align_up((size_t)items * D * N * 4, 256);
    w.d = ppk_align_up((size_t)items * 2 * D * 4, 256);
    w.bc = ppk_align_up((size_t)w.p.blocks_per_group * rows * G * 2 * N * 4, 256);
    w.carry = carry_bytes(B, D, N, w.p.splits);
    w.sum = ppk::partial_sum_ws_bytes(items, D * N);
    w.total = w.a + w.d + w.bc + w.carry + w.sum;
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

size_t ppk_selective_scan_fwd_workspace_bytes(int64_t T, int64_t B, int64_t D, int64_t N, int64_t G)
{
    if (T < 0 || B < 0 || D < 1 || N < 1 || G < 1) return 0;
    return carry_bytes(B, D, N, fwd_plan(T, B, D, G).splits);
}

int ppk_selective_scan_fwd(int dtype, int64_t T, int64_t B, int64_t D, int64_t N, int64_t G, const int64_t* step_off, const int64_t* lengths,
                           const int64_t* tiles, const void* x, const void* raw, const float* A, const void* Bm, const void* Cm, const float* skip,
                           const void* z, const float* bias, const float* state, int softplus, void* y, float* last_state, float* kept,
                           const int64_t* strides_host, void* workspace, size_t ws_bytes, ppk_stream_t stream)
{
    int rc = scan_check("selective_scan_fwd", dtype, T, B, D, N, G);
    if (rc) return rc;
    if (B == 0) return PPK_OK;
    if (!A || !last_state || !strides_host || (T > 0 && (!x || !raw || !Bm || !Cm || !y))) PPK_FAIL(PPK_ERR_NULL, "selective_scan_fwd: null pointer");
    if (step_off && (!lengths || !tiles)) PPK_FAIL(PPK_ERR_NULL, "selective_scan_fwd: a packed batch needs its lengths and tiles");
    if (!near_rows(strides_host, D)) PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_fwd: rows 2^30 elements or more apart");
    ScanArgs a = {};
    a.q = {step_off, lengths, T, B};
    a.tiles = tiles;
    const Plan p = fwd_plan(T, B, D, G);
    a.D = (int)D; a.N = (int)N; a.G = (int)G; a.per = (int)(D / G); a.blocks_per_group = (int)p.blocks_per_group;
    a.span = p.span; a.splits = (int)p.splits;
    a.x = x; a.raw = raw; a.Bm = Bm; a.Cm = Cm; a.z = z; a.A = A; a.skip = skip; a.bias = bias; a.state = state; a.softplus = softplus;
    a.y = y; a.last = last_state; a.kept = kept;
    set_strides(a, strides_host);
    const long long blocks = B * p.splits * G * a.blocks_per_group;
    if (!ppk_grid_fits(blocks, 64) || (p.splits > 1 && B > 65535))
        PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_fwd: B=%lld D=%lld takes %lld blocks, more than a launch has", (long long)B, (long long)D, blocks);
    hipStream_t st = (hipStream_t)stream;
    if (p.splits > 1) {
        if (ws_bytes < carry_bytes(B, D, N, p.splits) || !workspace) PPK_FAIL(PPK_ERR_WS, "selective_scan_fwd: workspace of %zu bytes", ws_bytes);
        char* cur = (char*)workspace;
        a.carry = (float*)ppk_carve(cur, (size_t)B * p.splits * D * N * 4);
        a.sdt = (float*)cur;
        if (dtype == PPK_F32) run_fwd<float>(a, true, (unsigned)blocks, st);
        else run_fwd<bf16_t>(a, true, (unsigned)blocks, st);
        join<false>(a, B, st);
    }
    if (dtype == PPK_F32) run_fwd<float>(a, false, (unsigned)blocks, st);
    else run_fwd<bf16_t>(a, false, (unsigned)blocks, st);
    PPK_CHECK_LAUNCH("selective_scan_fwd");
    return PPK_OK;
}

size_t ppk_selective_scan_bwd_workspace_bytes(int64_t T, int64_t B, int64_t D, int64_t N, int64_t G, int64_t rows)
{
    if (T < 0 || B < 0 || D < 1 || N < 1 || N > 64 || G < 1 || rows < 0) return 0;
    return bwd_ws(T, B, D, N, G, rows).total;
}

int ppk_selective_scan_bwd(int dtype, int64_t T, int64_t B, int64_t D, int64_t N, int64_t G, int64_t rows, const int64_t* step_off,
                           const int64_t* lengths, const int64_t* tiles, const void* x, const void* raw, const float* A, const void* Bm, const void* Cm,
                           const float* skip, const void* z, const float* bias, int softplus, const float* kept, const void* dy, const float* dlast_state,
                           void* dx, void* draw, float* dA, void* dB, void* dC, float* dskip, void* dz, float* dbias, float* dstate,
                           const int64_t* strides_host, void* workspace, size_t ws_bytes, ppk_stream_t stream)
{
    int rc = scan_check("selective_scan_bwd", dtype, T, B, D, N, G);
    if (rc) return rc;
    if (rows < 0 || rows >= 1LL << 31 || (!step_off && rows != T * B)) PPK_FAIL(PPK_ERR_SHAPE, "selective_scan_bwd: %lld rows", (long long)rows);
    if (!A || !dA || !workspace || !strides_host || (rows > 0 && (!x || !raw || !Bm || !Cm || !dy || !kept || !dx || !draw || !dB || !dC || (z && !dz))))
        PPK_FAIL(PPK_ERR_NULL, "selective_scan_bwd: null pointer");
    if (step_off && (!lengths || !tiles)) PPK_FAIL(PPK_ERR_NULL, "selective_scan_bwd: a packed batch needs its lengths and tiles");
    if (!near_rows(strides_host, D)) PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_bwd: rows 2^30 elements or more apart");
    const BwdWs w = bwd_ws(T, B, D, N, G, rows);
    const long long items = B * w.p.splits;
    if (ws_bytes < w.total) PPK_FAIL(PPK_ERR_WS, "selective_scan_bwd: workspace of %zu bytes, %zu needed", ws_bytes, w.total);
    hipStream_t st = (hipStream_t)stream;
    char* cur = (char*)workspace;
    ScanArgs a = {};
    a.pA = (float*)ppk_carve(cur, w.a);
    a.pD = (float*)ppk_carve(cur, w.d);
    a.pBC = (float*)ppk_carve(cur, w.bc);
    if (w.p.splits > 1) {
        a.carry = (float*)ppk_carve(cur, (size_t)items * D * N * 4);
        a.sdt = (float*)ppk_carve(cur, (size_t)items * D * 4);
    }
    void* sum_ws = cur;
    a.q = {step_off, lengths, T, B};
    a.tiles = tiles;
    a.D = (int)D; a.N = (int)N; a.G = (int)G; a.per = (int)(D / G); a.blocks_per_group = (int)w.p.blocks_per_group;
    a.span = w.p.span; a.splits = (int)w.p.splits;
    a.x = x; a.raw = raw; a.Bm = Bm; a.Cm = Cm; a.z = z; a.dy = dy; a.A = A; a.skip = skip; a.bias = bias; a.dlast = dlast_state; a.softplus = softplus;
    a.dx = dx; a.draw = draw; a.dz = dz; a.kept = const_cast<float*>(kept); a.dstate = dstate; a.nrows = rows;
    set_strides(a, strides_host);
    const long long blocks = items * G * a.blocks_per_group, bc = rows * G * 2 * N;
    if (!ppk_grid_fits(blocks, 256) || !ppk_grid_fits(ceil_div(bc, 256), 256) || (w.p.splits > 1 && B > 65535))
        PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_bwd: B=%lld D=%lld rows=%lld takes %lld and %lld blocks, more than a launch has", (long long)B, (long long)D, (long long)rows,
                 blocks, ceil_div(bc, 256));
    if (blocks > 0) {
        if (w.p.splits > 1) {
            ScanArgs part = a;
            part.blocks_per_group = (int)ceil_div(a.per, 64);
            const unsigned pb = (unsigned)(items * G * part.blocks_per_group);
            if (dtype == PPK_F32) run_bwd_part<float>(part, pb, st);
            else run_bwd_part<bf16_t>(part, pb, st);
            join<true>(a, B, st);
        }
        if (dtype == PPK_F32) run_bwd<float>(a, (unsigned)blocks, st);
        else run_bwd<bf16_t>(a, (unsigned)blocks, st);
    }
    if (bc > 0) {
        const unsigned nb = (unsigned)ceil_div(bc, 256);
        if (dtype == PPK_F32) k_scan_bc<float><<<nb, 256, 0, st>>>(a.pBC, a.blocks_per_group, rows, (int)G, (int)N, (float*)dB, (float*)dC);
        else k_scan_bc<bf16_t><<<nb, 256, 0, st>>>(a.pBC, a.blocks_per_group, rows, (int)G, (int)N, (bf16_t*)dB, (bf16_t*)dC);
    }
    const ppk::SumJob jobs[3] = {{a.pA, items, D * N, dA, 0, nullptr}, {a.pD, items, D, dskip, 0, nullptr}, {a.pD + items * D, items, D, dbias, 0, nullptr}};
    rc = ppk::partial_sums(jobs, 3, sum_ws, st);
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
    if (!ppk_grid_fits(blocks, 256)) PPK_FAIL(PPK_ERR_UNSUP, "selective_scan_step: B=%lld D=%lld takes %lld blocks, more than a launch has", (long long)B, (long long)D, blocks);
    if (dtype == PPK_F32) run_step<float>(a, (unsigned)blocks, state, new_state, (hipStream_t)stream);
    else run_step<bf16_t>(a, (unsigned)blocks, state, new_state, (hipStream_t)stream);
    PPK_CHECK_LAUNCH("selective_scan_step");
    return PPK_OK;
}

}  // extern "C"
