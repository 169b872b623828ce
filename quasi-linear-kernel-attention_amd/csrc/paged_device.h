// Device pieces of the paged kernels: pages found by position, held rows of 8 bits taken apart.
#pragma once

#include "paged.h"
#include "paged_cut.h"
#include "segments.h"
#include "softmax_tile.h"

#include <limits>

namespace qlka {
namespace pg {

constexpr float LOW = -std::numeric_limits<float>::infinity();
constexpr float GROW = 4.f;                  // of a row's reference: 2^8 of the exponentials

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
        asm("" : "+v"(w));                   // (else the word may be loaded as four bytes)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> 8 * i) * s;
    } else {
        typedef __attribute__((ext_vector_type(2))) float f32x2;
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
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
__device__ __forceinline__ sm::Frag<1> parts_of(u32x2 x, int, float s, Int8) {
    return sm::frag_of(__builtin_convertvector(eight<Int8>(x, s), bf16x8));
}
__device__ __forceinline__ sm::Frag<1> parts_of(u32x2 x, int, float s, E4m3) {      // an instruction for two
    bf16x8 y;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[h], s, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[h], s, true);
        y[4 * h] = lo[0]; y[4 * h + 1] = lo[1]; y[4 * h + 2] = hi[0]; y[4 * h + 3] = hi[1];
    }
    return sm::frag_of(y);
}
template <class C> __device__ __forceinline__ sm::Frag<1> parts_of(u32x4 x, int i, float s, C c) {
    return parts_of(u32x2{x[2 * i], x[2 * i + 1]}, 0, s, c);
}

// A position's place: the index of its page in the table, and its row in the page.
struct Place { int index, row; };
__device__ __forceinline__ Place place_of(const PgParams& p, int n) {
    const int index = divided(n, p.page_division);
    return {index, n - index * p.page_size};
}
// Where a row of a page is from the first one of its head on.
__device__ __forceinline__ uint64_t bytes_to(PgStrides s, uint32_t page, uint32_t row) {
    return (uint64_t)page * s.page + (uint64_t)row * s.row;
}

// Sums over the lanes up to this one, in registers; the last lane has the sum of all.
template <int CTRL, int ROWS, class X> __device__ __forceinline__ X moved(X x) {
    union { X x; int i; } a{x}, y;
    y.i = __builtin_amdgcn_update_dpp(0, a.i, CTRL, ROWS, 0xf, false);
    return y.x;
}
template <class X> __device__ __forceinline__ X sums_upto(X x) {
    x += moved<0x111, 0xf>(x);               // row_shr 1, 2, 4, 8
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);               // row_bcast 15 into rows 1 and 3
    x += moved<0x143, 0xc>(x);               // row_bcast 31 into rows 2 and 3
    return x;
}
template <class X> __device__ __forceinline__ X last_lane(X x) {
    union { X x; int i; } a{x}, y;
    y.i = __builtin_amdgcn_readlane(a.i, 63);
    return y.x;
}

__device__ __forceinline__ Tokens tokens_of(const PgParams& p, int b) {
    int first = b, rows = 1;
    if (p.offsets) {
        first = segment_edge(p.offsets, p.B, p.T, b + 1);
        rows = rows_between(first, segment_edge(p.offsets, p.B, p.T, b + 2));
    }
    return tokens_at(first, rows, p.lengths[b]);
}
__device__ __forceinline__ int seen_from(const PgParams& p, int seat) {
    return seen_upto(seat, p.num_pages, p.places);
}

// The tokens of sequence `lane`, the first 64 together.
__device__ __forceinline__ Tokens tokens_of_lane(const PgParams& p) {
    const int lane = threadIdx.x & 63;
    return lane < p.B ? tokens_of(p, lane) : Tokens{0, 0, 0};
}
// The sequence of row t (the same for all lanes) and its tokens, from those of every lane; b < 0 outside every
// sequence.
struct Found { int b; Tokens tokens; };
__device__ __forceinline__ Found find(const PgParams& p, int t, Tokens mine) {
    Found x{t, {}};
    if (p.offsets) {
        x.b = __popcll(__ballot((int)(threadIdx.x & 63) < p.B && mine.first <= t)) - 1;
        if (x.b == 63) x.b = __builtin_amdgcn_readfirstlane(last_upto(p.B + 1, t, [&](int j) { return p.offsets[j]; }));
        if (x.b >= p.B) x.b = -1;
        if (x.b < 0) return x;
    }
    if (x.b < 64)
        x.tokens = {__builtin_amdgcn_readlane(mine.first, x.b), __builtin_amdgcn_readlane(mine.rows, x.b),
                    __builtin_amdgcn_readlane(mine.start, x.b)};
    else
        x.tokens = tokens_of(p, x.b);
    if (t < x.tokens.first || t >= x.tokens.first + x.tokens.rows) x.b = -1;
    return x;
}

// How the work of a launch is cut into units of about equal time: a block of ROWS rows of one key head over `span`
// successive positions. The span goes by what the sequences of this launch (STEP: those of few rows) hold together,
// which only the device knows, so that there are about `aim` units a key head; every workgroup finds it, and its unit,
// by itself, a lane a sequence. The parts of a sequence are of one length (4 chunks of up to 8192: the longest of 19
// tiles instead of 20, 65 us instead of 68). Units of one sequence, part and key head are next to each other, and
// successive ones on one XCD, whose L2 then serves their keys. Where a sequence's positions are one part, its rows are
// written at once, else each part's sums go to the unit's place in the workspace and paged_join adds them up. Of many
// sequences a kernel of its own writes the span and the units before each one to the workspace (u.table), where the
// others look.
struct Unit { int b, part, kvh, block, parts, span, at; };

template <bool STEP, int ROWS> struct Units {
    static constexpr int ALIGN = STEP ? PG_ALIGN : PG_ALIGN / 2;       // a turn of all waves; a tile
    const PgParams& p;
    const PgUnits& u;
    int share, span, all;                    // all: units a key head
    // of the first 64 sequences this lane's: looked up once
    Tokens mine;
    Cut cut_mine;
    int first, before;                       // its units a key head, and those up to it

    __device__ __forceinline__ Extent held(int b, Tokens t) const {
        const int rows = t.rows * share;
        const bool here = b < p.B && STEP == (rows <= p.few) && rows > 0;
        return {here ? (rows + ROWS - 1) / ROWS : 0, seen_from(p, t.start + t.rows - 1)};
    }
    // f(the first of 64 sequences, what this lane's is) for those from 64 up to `end`, until it returns true; all are
    // looked up together (256 of 100 to 1000, 8 with chunks, 12 / 4 heads, bf16: 54 us, 56 one after the other); more
    // of them are in u.table
    template <class F> __device__ __forceinline__ void others(int end, F f) const {
        constexpr int EACH = (PG_LOOKED_UP - 64) / 64;
        if (end <= 64) return;
        const int lane = threadIdx.x & 63;
        Tokens t[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) t[i] = tokens_of(p, min(64 + 64 * i + lane, p.B - 1));
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int b = 64 + 64 * i;
            if (b >= end || f(b, held(b + lane, t[i]))) return;
        }
    }
    __device__ __forceinline__ Cut cut(Extent h) const { return cut_of(h, span, ALIGN); }

    __device__ __forceinline__ Units(const PgParams& p, const PgUnits& u) : Units(p, u, tokens_of_lane(p)) {}
    __device__ __forceinline__ Units(const PgParams& p, const PgUnits& u, Tokens mine)
        : p(p), u(u), share(p.H / p.G), mine(mine) {
        if (__builtin_expect(u.table != nullptr, 0)) {
            all = __builtin_amdgcn_readfirstlane(u.table[p.B]);
            span = __builtin_amdgcn_readfirstlane(u.table[p.B + 1]);
            return;
        }
        const int lane = threadIdx.x & 63;
        const Extent held_mine = held(lane, mine);
        float work = more_work(0.f, held_mine);
        others(p.B, [&](int, Extent h) {
            work = more_work(work, h);
            return false;
        });
        set_span(last_lane(sums_upto(work)));
        cut_mine = cut(held_mine);
        first = cut_mine.blocks * cut_mine.parts;
        before = sums_upto(first);
        all = upto(p.B);
    }
    // for paged_table
    __device__ __forceinline__ Units(const PgParams& p, const PgUnits& u, int) : p(p), u(u), share(p.H / p.G) {}
    __device__ __forceinline__ void set_span(float work) {
        span = __builtin_amdgcn_readfirstlane(span_of(work, u.aim, u.least, PG_ALIGN));
    }
    // of a sequence that is the same for all lanes
    __device__ __forceinline__ Tokens tokens(int b) const {
        if (b >= 64 || u.table) return tokens_of(p, b);
        return {__builtin_amdgcn_readlane(mine.first, b), __builtin_amdgcn_readlane(mine.rows, b),
                __builtin_amdgcn_readlane(mine.start, b)};
    }
    // units of the sequences before `end`
    __device__ __forceinline__ int upto(int end) const {
        if (end <= 0) return 0;
        if (__builtin_expect(u.table != nullptr, 0)) return __builtin_amdgcn_readfirstlane(u.table[end]);
        const int n = __builtin_amdgcn_readlane(before, min(end, 64) - 1);
        if (end <= 64) return n;
        const int lane = threadIdx.x & 63;
        int more = 0;
        others(end, [&](int b, Extent h) {
            const Cut c = cut(h);
            more += b + lane < end ? c.blocks * c.parts : 0;
            return false;
        });
        return n + last_lane(sums_upto(more));
    }
    // number `rest` of a sequence's units
    __device__ __forceinline__ void place(Unit& x, Cut c, int rest) const {
        const InSequence at =
            place_in(__builtin_amdgcn_readfirstlane(c.blocks), __builtin_amdgcn_readfirstlane(rest), p.G);
        x.parts = __builtin_amdgcn_readfirstlane(c.parts);
        x.span = __builtin_amdgcn_readfirstlane(c.span);
        x.part = at.part;
        x.kvh = at.kvh;
        x.block = at.block;
    }
    // The unit of a workgroup; b < 0 where it has none.
    __device__ __forceinline__ Unit of(int wg) const {
        const int units = all * p.G, each = (units + 7) / 8;
        Unit x{};
        x.b = -1;
        x.at = (wg & 7) * each + (wg >> 3);
        // (offsets that decrease can make more units than a launch and its workspace are made for)
        if ((wg >> 3) >= each || x.at >= units || x.at >= u.room) return x;
        if (__builtin_expect(u.table != nullptr, 0)) {
            x.b = last_upto(p.B + 1, x.at, [&](int j) { return u.table[j] * p.G; });
            x.b = min(max(__builtin_amdgcn_readfirstlane(x.b), 0), p.B - 1);
            place(x, cut(held(x.b, tokens_of(p, x.b))), x.at - u.table[x.b] * p.G);
            return x;
        }
        int base = 0;                        // units a key head of the sequences before those that are looked at
        // whether the unit is of one of 64 sequences: this lane's cut, its units a key head, and those up to it
        const auto among = [&](int b0, Cut c, int n, int to) {
            const uint64_t past = __ballot((base + to) * p.G > x.at);
            if (!past) {
                base += last_lane(to);
                return false;
            }
            const int l = __builtin_ctzll(past);
            x.b = b0 + l;
            const Cut its = {__builtin_amdgcn_readlane(c.blocks, l), __builtin_amdgcn_readlane(c.parts, l),
                             __builtin_amdgcn_readlane(c.span, l)};
            place(x, its, x.at - (base + __builtin_amdgcn_readlane(to - n, l)) * p.G);
            return true;
        };
        if (!among(0, cut_mine, first, before))
            others(p.B, [&](int b0, Extent h) {
                const Cut c = cut(h);
                const int n = c.blocks * c.parts;
                return among(b0, c, n, sums_upto(n));
            });
        return x;
    }
};

// Zeros for the rows outside every sequence, by `count` workgroups of which this is number wg.
template <class T> __device__ __forceinline__ void write_outside(const PgParams& p, int wg, int count) {
    const int lo = segment_edge(p.offsets, p.B, p.T, 1), hi = segment_edge(p.offsets, p.B, p.T, p.B + 1);
    const int64_t rows = (int64_t)p.H * (lo + max(p.T - hi, 0));
    const int lanes = p.D / 4;
    for (int64_t i = (int64_t)wg * blockDim.x + threadIdx.x; i < rows * lanes; i += (int64_t)count * blockDim.x) {
        const int d = (int)(i % lanes) * 4, head = (int)(i / lanes % p.H), n = (int)(i / lanes / p.H);
        const int t = n < lo ? n : n - lo + hi;
        sm::store4((T*)p.out + head * p.so.h + t * p.so.r, d, p.D, f32x4{});
    }
}
constexpr int OUTSIDE_GROUPS = 16;

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
