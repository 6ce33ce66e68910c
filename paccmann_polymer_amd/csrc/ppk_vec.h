// fp32 / bf16 elements, and rows of them read and written in 16-byte chunks wherever they begin.  gfx950 only.
#pragma once
#include "ppk_common.h"

// v combined with v of the lane that `ctrl` names, in one instruction
template <int CTRL> __device__ __forceinline__ float dpp_of(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)); }
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140, DPP_ROR4 = 0x124, DPP_ROR8 = 0x128;
// Sum and maximum over groups of W neighbouring lanes (W a power of two up to 64), in every one of them, without LDS.  A mirror reverses
// lanes that agree already within each half, which is what an xor of that half's width would reach; between rows of 16 and between halves
// of a wave the exchange instructions hand over whole rows.
template <int W, typename F> __device__ __forceinline__ float lanes_all(float v, F f)
{
    if (W > 1) v = f(v, dpp_of<DPP_XOR1>(v));
    if (W > 2) v = f(v, dpp_of<DPP_XOR2>(v));
    if (W > 4) v = f(v, dpp_of<DPP_HALF_MIRROR>(v));
    if (W > 8) v = f(v, dpp_of<DPP_MIRROR>(v));
    if (W > 16) { const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false); v = f(__uint_as_float(p[0]), __uint_as_float(p[1])); }
    if (W > 32) { const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false); v = f(__uint_as_float(p[0]), __uint_as_float(p[1])); }
    return v;
}
template <int W> __device__ __forceinline__ float lanes_sum(float v) { return lanes_all<W>(v, [](float a, float b) { return a + b; }); }
template <int W> __device__ __forceinline__ float lanes_max(float v) { return lanes_all<W>(v, [](float a, float b) { return fmaxf(a, b); }); }

struct bf16_t { unsigned short v; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((unsigned)x.v << 16); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float x)
{
    // round to nearest even; a NaN keeps its sign and stays a NaN
    const unsigned u = __float_as_uint(x);
    const unsigned r = u + 0x7fffu + ((u >> 16) & 1u);
    bf16_t o;
    o.v = (unsigned short)((x != x) ? ((u >> 16) | 0x40u) : (r >> 16));
    return o;
}
// the elements of a 16-byte chunk
template <typename T> __device__ __forceinline__ void unpack(uint4 c, float* v);
template <> __device__ __forceinline__ void unpack<float>(uint4 c, float* v)
{
    v[0] = __uint_as_float(c.x); v[1] = __uint_as_float(c.y); v[2] = __uint_as_float(c.z); v[3] = __uint_as_float(c.w);
}
template <> __device__ __forceinline__ void unpack<bf16_t>(uint4 c, float* v)
{
    const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <typename T> __device__ __forceinline__ uint4 pack(const float* v);
template <> __device__ __forceinline__ uint4 pack<float>(const float* v)
{
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <> __device__ __forceinline__ uint4 pack<bf16_t>(const float* v)
{
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (unsigned)from_f32<bf16_t>(v[2 * i]).v | ((unsigned)from_f32<bf16_t>(v[2 * i + 1]).v << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row of n elements as the 16-byte chunks of memory that it touches: chunk c holds the elements at(c, 0) .. at(c, E - 1), those
// outside [0, n) are none of the row's and are neither read nor written.  A chunk that is the row's in whole takes one 16-byte access.
template <typename T> struct RowChunks {
    static constexpr int E = 16 / (int)sizeof(T);
    const T* x;
    int n, shift, chunks;                  // shift: elements of the first chunk before the row
    __device__ __forceinline__ RowChunks(const T* p, int n_) : x(p), n(n_)
    {
        shift = (int)(((uintptr_t)p & 15) / sizeof(T));
        chunks = (n + shift + E - 1) / E;
    }
    __device__ __forceinline__ int at(int c, int e) const { return c * E - shift + e; }
    __device__ __forceinline__ bool has(int c, int e) const { return (unsigned)at(c, e) < (unsigned)n; }
    __device__ __forceinline__ bool whole(int c) const { const int b = at(c, 0); return b >= 0 && b + E <= n; }
    // `none` stands where the chunk holds no element of the row
    __device__ __forceinline__ uint4 load(int c, float none) const
    {
        if (whole(c)) return *reinterpret_cast<const uint4*>(x + at(c, 0));
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = none;
        if (c < chunks)
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (has(c, e)) v[e] = to_f32(x[at(c, e)]);
        return pack<T>(v);
    }
    __device__ __forceinline__ void store(T* out, int c, const float* v) const
    {
        if (whole(c)) { *reinterpret_cast<uint4*>(out + at(c, 0)) = pack<T>(v); return; }
        if (c >= chunks) return;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (has(c, e)) out[at(c, e)] = from_f32<T>(v[e]);
    }
};
