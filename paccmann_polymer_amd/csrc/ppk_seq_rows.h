// How the sequence operators address a batch: a packed one (time-major, length-sorted: step t owns rows off[t] .. off[t + 1], sequence b
// its row off[t] + b) or a rectangular one of any strides.  gfx950 only.
#pragma once
#include "ppk_vec.h"

namespace ppk {

struct Stride { long long t, b; };            // of a step and of a sequence, in elements; a packed batch has t == b == its row stride

struct SeqBatch {
    const int64_t* off;                       // device [T + 1], or null: rectangular
    const int64_t* len;                       // device [B], or null: every sequence has T steps
    long long T, B;
    __device__ __forceinline__ long long row(long long t) const { return off ? off[t] : t; }
    __device__ __forceinline__ long long length(long long b) const { return len ? len[b] : T; }
};
// element offset of (step, sequence); r = SeqBatch::row(step)
__device__ __forceinline__ long long at(const Stride& s, long long r, long long b) { return r * s.t + b * s.b; }

// memory that the kernel does not write, at an address that all lanes share: loaded into scalar registers
#define UNIFORM __attribute__((address_space(4)))
template <typename T> __device__ __forceinline__ const UNIFORM T* uniform(const void* p) { return (const UNIFORM T*)(uintptr_t)p; }
__device__ __forceinline__ unsigned uni_row(const SeqBatch& q, long long t) { return q.off ? (unsigned)uniform<long long>(q.off)[t] : (unsigned)t; }
// Addresses: a base and a step's offset that all lanes share, in scalar registers, and a lane's own 32-bit offset in bytes.  A batch has
// fewer than 2^31 steps and rows, and a row's stride is below 2^32 bytes (the host sees to it): their product is two 32-bit ones.
template <typename T> struct Rows {
    const char* base;
    unsigned stride;
    __device__ __forceinline__ Rows(const void* p, long long offset, long long stride_)
        : base((const char*)p + offset * (long long)sizeof(T)), stride((unsigned)(stride_ * (long long)sizeof(T))) {}
    __device__ __forceinline__ const char* row(unsigned r) const { return base + (unsigned long long)r * stride; }
    template <typename U> __device__ __forceinline__ U get_as(unsigned r, unsigned byte) const { return *(const U*)(row(r) + byte); }
    template <typename U> __device__ __forceinline__ void put_as(unsigned r, unsigned byte, U v) const { *(U*)(const_cast<char*>(row(r)) + byte) = v; }
    __device__ __forceinline__ T get(unsigned r, unsigned byte) const { return *(const T*)(row(r) + byte); }
    __device__ __forceinline__ void put(unsigned r, unsigned byte, T v) const { *(T*)(const_cast<char*>(row(r)) + byte) = v; }
};
__device__ __forceinline__ long long uni_len(const SeqBatch& q, long long b) { return q.len ? uniform<long long>(q.len)[b] : q.T; }

// out[c] = sum over p of part[p * C + c], in an order that the sizes alone set and in fp64: the partial sums of blocks that ran in any order.
// taps != 0: the columns are [taps + 1, D], out a weight's gradient [D, taps] and out2 (or null) a bias' [D].
struct SumJob { const float* part; long long P, C; float* out; int taps; float* out2; };
constexpr int PS_ROWS = 64;                   // rows of a first-pass sum ...
constexpr long long ONE_PASS_ROWS = 4096;     // ... where there are more than this; jobs with taps have at most so many
size_t partial_sum_ws_bytes(long long P, long long C);
int partial_sums(const SumJob* jobs, int count, void* ws, hipStream_t stream);      // at most three jobs

}  // namespace ppk
