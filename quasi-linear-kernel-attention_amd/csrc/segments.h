// Sequences of different lengths laid one after the other in T rows, and the blocks of rows that workgroups own.
//
// offsets (B + 1 numbers on the device, not decreasing) are where the sequences begin, and where the last one ends. The
// host does not know them: a launch has room for every way of cutting T rows, and a workgroup finds its sequence here.
// The rows are cut into B + 2 segments: what lies before the first sequence, the sequences, what lies behind the last
// one. Segment j begins at row e(j); its blocks of `rows` rows (of `share` rows a token) have the numbers from
//   e(j) share / rows (rounded down) + j
// on. That grows by at least one with j and by enough for the segment's blocks, since rounding down loses less than
// one; so no sum over the segments before is needed, and T share / rows + B + 2 numbers are enough. Numbers between a
// segment's last block and the next one's first have nothing to do. Rows are held to [0, T] whatever the offsets are.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace qlka {

struct Segment {
    int index;             // of its sequence; -1 and B for the rows outside
    int first, rows;       // tokens: the first one, and how many
    int block;             // of the segment's rows
};

inline int64_t segment_blocks(int64_t T, int B, int share, int rows) { return T * share / rows + B + 2; }

__device__ __forceinline__ int segment_edge(const int* offsets, int B, int T, int j) {
    return j <= 0 ? 0 : j <= B + 1 ? min(max(offsets[j - 1], 0), T) : T;
}

// The number of the first block of segment j.
__device__ __forceinline__ int segment_start(int edge, int j, int share, int rows) {
    return (int)((int64_t)edge * share / rows) + j;
}

// The last j of [0, count) with at(j) <= x, which holds for j = 0 (at: not decreasing, x the same for all lanes), by a
// wave that looks at 64 places at a time.
template <class F> __device__ __forceinline__ int last_upto(int count, int x, F at) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = count;                             // the answer is in [lo - 1, lo + n)
    while (n > 64) {
        const int step = (n + 63) / 64, i = lo + (lane + 1) * step - 1;
        const int below = __popcll(__ballot(i < lo + n && at(i) <= x));
        const int from = lo + below * step;
        n = min(step - 1, lo + n - from);
        lo = from;
    }
    return lo + __popcll(__ballot(lane < n && at(lo + lane) <= x)) - 1;
}

__device__ __forceinline__ Segment segment_of(const int* offsets, int B, int T, int share, int rows, int number) {
    int j = last_upto(B + 2, number, [&](int i) {
        return segment_start(segment_edge(offsets, B, T, i), i, share, rows); });
    j = max(__builtin_amdgcn_readfirstlane(j), 0);
    Segment s;
    s.index = j - 1;
    s.first = segment_edge(offsets, B, T, j);
    s.rows = max(segment_edge(offsets, B, T, j + 1) - s.first, 0);
    s.block = number - segment_start(s.first, j, share, rows);
    return s;
}

}  // namespace qlka
