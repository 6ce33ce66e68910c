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

// out[c] = sum over p of part[p * C + c], p ascending, in fp64: the partial sums of blocks that ran in any order, added in one
constexpr int PS_ROWS = 64;                   // rows of a first-pass sum
size_t partial_sum_ws_bytes(long long P, long long C);
int partial_sum(const float* part, long long P, long long C, float* out, void* ws, hipStream_t stream);

}  // namespace ppk
