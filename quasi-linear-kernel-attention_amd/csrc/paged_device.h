// Device pieces of the paged kernels: pages found by position, held rows of 8 bits taken apart.
#pragma once

#include "paged.h"
#include "segments.h"
#include "softmax_tile.h"

namespace qlka {
namespace pg {

using sm::bf16x2;
using sm::bf16x4;
using sm::bf16x8;
using sm::f32x4;
using sm::f32x8;

// Types of held elements of 8 bits.
struct Int8 {};
struct E4m3 {};

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// EL successive held elements of a row, as they lie in memory
template <class C, int EL> struct Piece;
template <> struct Piece<__bf16, 8> { typedef bf16x8 raw; static constexpr int SIZE = 2, PARTS = 1, SEGS = 1; };
template <> struct Piece<float, 8> { typedef f32x8 raw; static constexpr int SIZE = 4, PARTS = 3, SEGS = 1; };
template <class C> struct Piece<C, 8> { typedef u32x2 raw; static constexpr int SIZE = 1, PARTS = 1, SEGS = 1; };
template <class C> struct Piece<C, 16> { typedef u32x4 raw; static constexpr int SIZE = 1, PARTS = 1, SEGS = 2; };

template <class C> constexpr bool coded = std::is_same<C, Int8>::value || std::is_same<C, E4m3>::value;

// 2^(e - 127); NaN for the mark of elements that were not finite
__device__ __forceinline__ float power_of(uint32_t e) {
    return __uint_as_float(e == 255 ? 0x7fc00000u : e << 23);
}

// Four codes times a power of two: exact in float, and in bf16, whose 8 bits hold 7 and a sign, or 4 and a sign.
template <class C> __device__ __forceinline__ f32x4 four(uint32_t w, float s) {
    f32x4 x;
    if constexpr (std::is_same<C, Int8>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> 8 * i) * s;
    } else {
        typedef __attribute__((ext_vector_type(2))) float f32x2;
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        x = f32x4{lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
    }
    return x;
}
template <class C> __device__ __forceinline__ f32x8 eight(u32x2 w, float s) {
    const f32x4 lo = four<C>(w[0], s), hi = four<C>(w[1], s);
    return f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Eight elements as the parts that matrix products take (i: which eight of the piece).
__device__ __forceinline__ sm::Frag<1> parts_of(bf16x8 x, int, float, __bf16) { return sm::frag_of(x); }
__device__ __forceinline__ sm::Frag<3> parts_of(f32x8 x, int, float, float) { return sm::frag_of(x); }
template <class C> __device__ __forceinline__ sm::Frag<1> parts_of(u32x2 x, int, float s, C) {
    return sm::frag_of(__builtin_convertvector(eight<C>(x, s), bf16x8));
}
template <class C> __device__ __forceinline__ sm::Frag<1> parts_of(u32x4 x, int i, float s, C) {
    return sm::frag_of(__builtin_convertvector(eight<C>(u32x2{x[2 * i], x[2 * i + 1]}, s), bf16x8));
}

// Where a position's page is in the table, and its row in the page.
__device__ __forceinline__ int page_at(const PgParams& p, int n) {
    return (int)((uint64_t)(uint32_t)n * p.magic >> p.shift);
}

// The new tokens of a sequence: `first` of the T rows on, `rows` of them, the first at position `start`.
struct Tokens { int first, rows, start; };
__device__ __forceinline__ Tokens tokens_of(const PgParams& p, int b, int first, int rows) {
    const int length = min(max(p.lengths[b], 0), 1 << 28);
    return {first, rows, length - rows};
}

// f(padded row length)
template <class F> int by_width(int D, F f) {
    const int DP = sm_padded(D);
    return DP == 32   ? f(std::integral_constant<int, 32>())
           : DP == 64 ? f(std::integral_constant<int, 64>())
                      : f(std::integral_constant<int, 128>());
}

// element types: q's, and what is held
template <class F> int dispatch_types(int dtype, int held, F f) {
    const auto with = [&](auto t) {
        return held == QLKA_INT8 ? f(t, Int8()) : held == QLKA_E4M3 ? f(t, E4m3()) : f(t, t);
    };
    return dtype == QLKA_BF16 ? with(__bf16()) : with(float());
}

}  // namespace pg
}  // namespace qlka
