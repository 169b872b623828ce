// Sequences of different lengths laid one after the other in T rows, and the blocks of rows that workgroups own.
//
// offsets (B + 1 numbers on the device, not decreasing) are where the sequences begin, and where the last one ends. The
// host does not know them: a launch has room for every way of cutting T rows, and a workgroup finds its sequence here.
// The rows are cut into B + 2 segments: what lies before the first sequence, the sequences, what lies behind the last
// one. Segment j begins at row e(j); its blocks of `rows` rows have the numbers from
//   e(j) / rows (rounded down) + j
// on. That grows by at least one with j and by enough for the segment's blocks, since rounding down loses less than
// one; so no sum over the segments before is needed, and T / rows + B + 2 numbers are enough. Numbers between a
// segment's last block and the next one's first have nothing to do. Rows are held to [0, T] whatever the offsets are.
#pragma once

#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>

namespace qlka {

struct Segment {
    int index;             // of its sequence; -1 and B for the rows outside
    int first, rows;       // the first row, and how many
    int block;             // of the segment's rows
};

inline int64_t segment_blocks(int64_t T, int B, int rows) { return T / rows + B + 2; }

__host__ __device__ __forceinline__ int segment_edge(const int* offsets, int B, int T, int j) {
    return j <= 0 ? 0 : j <= B + 1 ? std::min(std::max(offsets[j - 1], 0), T) : T;
}

// The number of the first block of segment j.
__host__ __device__ __forceinline__ int segment_start(int edge, int j, int rows) { return edge / rows + j; }

// A wave's lanes: how many f(lane) holds for, and what is the same in all of them.
struct Lanes {
    template <class F> __device__ __forceinline__ int count(F f) const {
        return __popcll(__ballot(f((int)(threadIdx.x & 63))));
    }
    __device__ __forceinline__ int same(int x) const { return __builtin_amdgcn_readfirstlane(x); }
};

// The last j of [0, count) with at(j) <= x, which holds for j = 0 (at: not decreasing, x the same for all lanes), by a
// wave that looks at 64 places at a time. Whatever at is, the result is in [-1, count) and at is asked for [0, count).
template <class F, class L> __host__ __device__ __forceinline__ int last_upto(int count, int x, F at, L lanes) {
    int lo = 0, n = count;                             // the answer is in [lo - 1, lo + n)
    while (n > 64) {
        const int step = (n + 63) / 64;
        const int below = lanes.count([&](int lane) {
            const int i = lo + (lane + 1) * step - 1;
            return i < lo + n && at(i) <= x;
        });
        const int from = lo + below * step;
        n = std::min(step - 1, lo + n - from);
        lo = from;
    }
    return lo + lanes.count([&](int lane) { return lane < n && at(lo + lane) <= x; }) - 1;
}
template <class F> __device__ __forceinline__ int last_upto(int count, int x, F at) {
    return last_upto(count, x, at, Lanes());
}

template <class L>
__host__ __device__ __forceinline__
Segment segment_of(const int* offsets, int B, int T, int rows, int number, L lanes) {
    const auto start = [&](int i) { return segment_start(segment_edge(offsets, B, T, i), i, rows); };
    const int j = std::max(lanes.same(last_upto(B + 2, number, start, lanes)), 0);
    Segment s;
    s.index = j - 1;
    s.first = segment_edge(offsets, B, T, j);
    s.rows = std::max(segment_edge(offsets, B, T, j + 1) - s.first, 0);
    s.block = number - segment_start(s.first, j, rows);
    if (s.block < 0) s.rows = s.block = 0;             // offsets that decrease: a vote of lanes is not the last of them
    return s;
}

}  // namespace qlka
