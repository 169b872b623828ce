// How pages are found and how the work of attention over them is cut (paged_device.h): the arithmetic, on the host and
// on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>
#include <cstdint>

namespace qlka {
namespace pg {

constexpr int MOST_POSITIONS = 1 << 28;

// ---- pages

// n / page_size = high word of 2 n * magic, >> shift, for n below 2^31
struct Division { uint32_t magic, shift; };
inline Division division_by(int page_size) {
    int log = 0;
    while (1 << log < page_size) ++log;
    return {(uint32_t)(((uint64_t(1) << (31 + log)) + page_size - 1) / page_size), (uint32_t)log};
}
__host__ __device__ __forceinline__ int divided(int n, Division by) {
    return (int)((uint32_t)((uint64_t)(2u * (uint32_t)n) * by.magic >> 32) >> by.shift);
}

// ---- sequences

// The new tokens of a sequence: `rows` of them from row `first` on, the first at position `start`.
struct Tokens { int first, rows, start; };
__host__ __device__ __forceinline__ int rows_between(int first, int end) { return std::max(end - first, 0); }
__host__ __device__ __forceinline__ Tokens tokens_at(int first, int rows, int length) {
    return {first, rows, std::min(std::max(length, 0), MOST_POSITIONS) - rows};
}
// Positions up to `seat` that have a place.
__host__ __device__ __forceinline__ int seen_upto(int seat, int num_pages, int places) {
    return num_pages ? std::min(std::max(seat + 1, 0), places) : 0;
}

// ---- units

struct Extent { int blocks, seen; };           // of a sequence: blocks of rows, positions that its last row sees
struct Cut { int blocks, parts, span; };     // of a sequence: units a key head = blocks * parts; positions of a part

// The work of the sequences so far and one more. The kernel that joins parts finds the same span as the one that left
// them only if both round alike, and products of thousands of blocks and positions are rounded: one fused operation,
// which no compiler can take apart or fuse with another one.
__host__ __device__ __forceinline__ float more_work(float work, Extent h) {
    return __builtin_fmaf((float)h.blocks, (float)h.seen, work);
}
// Positions of a part: what leaves about `aim` units of `work`, `least` at the least, a multiple of `align`. More than
// work / aim, so that the units are at most as many as the blocks and aim + 1.
__host__ __device__ __forceinline__ int span_of(float work, float aim, int least, int align) {
    const int span = std::max((int)std::fmin(work / aim, (float)MOST_POSITIONS) + 1, least);
    return (span + align - 1) / align * align;
}
// A sequence's parts, all of one length: a multiple of `align`.
__host__ __device__ __forceinline__ Cut cut_of(Extent h, int span, int align) {
    const uint32_t parts = std::max(1, (h.seen + span - 1) / span), each = ((uint32_t)h.seen + parts - 1) / parts;
    return {h.blocks, (int)parts, std::max((int)(each + align - 1) / align, 1) * align};
}
// Which part, key head (of G) and block a sequence's unit number `rest` is.
struct InSequence { int part, kvh, block; };
__host__ __device__ __forceinline__ InSequence place_in(int blocks, int rest, int G) {
    const uint32_t n = std::max(blocks, 1), all = n * (uint32_t)G;
    const uint32_t i = std::max(rest, 0);    // (sums of offsets that decrease can pass 32 bits)
    return {(int)(i / all), (int)(i % all / n), (int)(i % n)};
}

}  // namespace pg
}  // namespace qlka
