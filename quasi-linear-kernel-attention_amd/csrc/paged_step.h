// Softmax attention of a few new tokens over a cache in pages (a decoder's single tokens): bound by reading the held
// keys and values once.
//
// A workgroup takes 16 rows, the query heads of one key head's new tokens, and a part of the sequence's positions; its
// waves take 32 positions each in turn and go through them by themselves (no barrier): pages found, keys and values
// loaded into registers one turn ahead, S^T = k q^T by v_mfma_f32_16x16x32_bf16 with the keys as they lie in memory as
// the first operand (a lane holds 8 elements of a key; which 8 goes by the load's width, and q is held to match), O^T
// += v^T P^T with the probabilities from the registers that they are in and the values turned by a tile in LDS that
// only this wave uses. A row's reference for the exponentials is moved when some lane's score passes it by 2^8, so
// nothing crosses lanes in most turns. Waves are joined at the end, the parts of long sequences by paged_join.
//
// Measured: 16 sequences of 2000 to 8192, 12 heads of 64, bf16: 37 us under way for 211 MB, of which the card's
// last-level cache serves a part, 50 with the joining and cold pages (shuffled pages are read at 5.1 TB/s at most); 32
// of 1000 to 16384, 12 / 4 heads, e4m3: 22 us, 32 with all; 8 of 33 to 197: 6.5 us, latency of lengths, table and rows
// in turn.
//
// Elements of 8 bits become bf16 exactly (paged_cache.hip), so products are those of what is held.
#pragma once

#include "paged_device.h"

#include <limits>

namespace qlka {
namespace pg {

constexpr int STEP_WAVES = 4;

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// A sum of products of operands in NA and NB parts, the smaller parts' apart (softmax_tile.h, Acc).
template <int NA, int NB> struct Sum {
    f32x4 main = {}, rest;
    __device__ __forceinline__ void start() {
        if constexpr (NA + NB > 2) rest = f32x4{};
    }
    __device__ __forceinline__ void add(const sm::Frag<NA>& a, const sm::Frag<NB>& b) {
        if constexpr (NB == 3) rest = mfma16(a.p[0], b.p[2], rest);
        if constexpr (NA == 3) {
            rest = mfma16(a.p[2], b.p[0], rest);
            rest = mfma16(a.p[1], b.p[1], rest);
        }
        if constexpr (NB == 3) rest = mfma16(a.p[0], b.p[1], rest);
        if constexpr (NA == 3) rest = mfma16(a.p[1], b.p[0], rest);
        main = mfma16(a.p[0], b.p[0], main);
    }
    __device__ __forceinline__ void join() {
        if constexpr (NA + NB > 2) main = main + rest;
    }
};

// Column d0 + lane % 16 of a tile's 32 rows in the order that scores stand in registers: lane group g (of 16) has rows
// 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3.
template <int NP, int DP>
__device__ __forceinline__ sm::Frag<NP> column16(const sm::Tile<NP, 32, DP>& t, int d0, int lane) {
    const int row = 4 * (lane >> 4) + ((lane & 15) >> 2), piece = (d0 >> 3) + ((lane & 3) >> 1);
    const int lo = t.at(row, piece) + (lane & 1) * 4, hi = t.at(row + 16, piece) + (lane & 1) * 4;
    sm::Frag<NP> f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        union { sm::s16x4 s[2]; bf16x8 b; } u;
        typedef __attribute__((address_space(3))) sm::s16x4 lds4;
        u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)&t.x[i * t.PLANE + lo]);
        u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)&t.x[i * t.PLANE + hi]);
        f.p[i] = u.b;
    }
    return f;
}

// Waves that a SIMD has room for: what waits for memory is other waves' time. With 4 waves bf16 rows of 64 would spill
// in the loop (16 x 12 heads of up to 8192: 70 us, 52 with 3, 59 with 2); 8 bits spill 3 registers, loaded 8 at a time
// 6 to 14, and are faster so (32 x 12 / 4: 33 us, 41 with 2).
template <class T, class C, int DP> constexpr int step_room() {
    return sm::Elem<T>::PARTS == 3 || DP == 128 ? 2 : coded<C> || DP == 32 ? 4 : 3;
}

template <class T, class C, int DP, int EL> __device__ __forceinline__ void step(const PgParams& p, int wg) {
    typedef Piece<C, EL> P;
    typedef typename P::raw Raw;
    constexpr int NQ = sm::Elem<T>::PARTS, NK = P::PARTS, NW = STEP_WAVES, ROWS = PG_STEP_ROWS;
    constexpr int PIECES = DP / (4 * EL), ND = DP / 16;
    constexpr bool AHEAD = PIECES * (int)sizeof(Raw) <= 64;            // two turns' rows in registers
    typedef sm::Tile<NK, 32, DP> TileT;
    __shared__ union {
        TileT v[NW];
        float o[NW][ROWS][DP + 4];
    } lds;
    __shared__ float join_ref[NW][ROWS], join_sum[NW][ROWS];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int share = p.H / p.G;
    const Units<true, ROWS> units(p, p.step);
    const Unit unit = units.of(wg);
    if (unit.b < 0) return;
    const Tokens seq = units.tokens(unit.b);
    const int b = unit.b, kvh = unit.kvh, rows = seq.rows * share, r0 = unit.block * ROWS;

    // this lane's row, and the positions that the block's rows see
    const int r = r0 + col, head = kvh * share + r % share, t = seq.first + r / share;
    const bool real = r < rows;
    const int last = seq.start + min(r0 + ROWS - 1, rows - 1) / share, least = seq.start + r0 / share;
    const int seat = real ? seq.start + r / share : last;
    const int seen = seen_from(p, last);
    if (unit.part && (int64_t)unit.part * unit.span >= seen) return;   // (the first part leaves zeros all the same)
    const int begin = unit.part * (unit.span / 32), end = min(begin + unit.span / 32, (seen + 31) / 32);
    int turn = begin + wave;

    const int* table = p.tables + b * p.table_stride;
    // element d of piece i of this lane
    const auto at = [&](int i) { return (4 * i + g) * EL; };

    const char* k_head = p.k_pages + (uint64_t)kvh * p.sk.head;
    const char* v_head = p.v_pages + (uint64_t)kvh * p.sv.head;
    const uint8_t* ke_head = p.k_exp + (uint64_t)kvh * p.ske.head;
    const uint8_t* ve_head = p.v_exp + (uint64_t)kvh * p.sve.head;

    struct Pages { int page[2], row[2]; };
    const auto look = [&](int turn) {
        Pages x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Place at = place_of(p, min(turn * 32 + 16 * i + col, seen - 1));
            x.page[i] = turn < end ? table[at.index] : 0;
            x.row[i] = at.row;
        }
        return x;
    };
    struct Held {
        Raw k[2][PIECES], v[2][PIECES];
        uint32_t ke[2][PIECES], ve[2][PIECES];
        uint32_t there;                      // bit i, 16 + i: positions i, 16 + i of the turn have a page
    };
    const auto fetch = [&](Pages pages) {
        Held x;
        bool ok[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ok[i] = (uint32_t)pages.page[i] < (uint32_t)p.num_pages;
            const uint32_t page = ok[i] ? pages.page[i] : 0, row = pages.row[i];       // not there: some row, not used
            const char* k = k_head + bytes_to(p.sk, page, row);
            const char* v = v_head + bytes_to(p.sv, page, row);
#pragma unroll
            for (int c = 0; c < PIECES; ++c) {
                const int d = at(c) < p.D ? at(c) : 0;
                x.k[i][c] = *reinterpret_cast<const Raw*>(k + d * P::SIZE);
                x.v[i][c] = *reinterpret_cast<const Raw*>(v + d * P::SIZE);
            }
            if constexpr (coded<C>) {
                const uint8_t* ke = ke_head + bytes_to(p.ske, page, row);
                const uint8_t* ve = ve_head + bytes_to(p.sve, page, row);
#pragma unroll
                for (int c = 0; c < PIECES; ++c) {
                    const int d = at(c) < p.D ? at(c) : 0;
                    x.ke[i][c] = ke[d / BLOCK];
                    x.ve[i][c] = ve[d / BLOCK];
                }
            }
        }
        x.there = (uint32_t)(__ballot(ok[0]) & 0xffff) | (uint32_t)(__ballot(ok[1]) & 0xffff) << 16;
        return x;
    };
    Held even;
    Pages pages = look(turn);
    if (turn < end) even = fetch(pages);
    if constexpr (AHEAD) pages = look(turn + NW);

    sm::Frag<NQ> qf[PIECES][P::SEGS];
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int i = 0; i < P::SEGS; ++i) {
            typename sm::Elem<T>::seg s = {};
            if (real) s = sm::load_seg((const T*)p.q + head * p.sq.h + t * p.sq.r, at(c) + 8 * i, p.D);
            s = s * (T)p.q_sign;
            qf[c][i] = sm::frag_of(s);
        }

    const float c1 = p.scale * sm::UNIT;
    TileT& tile = lds.v[wave];
    Sum<NK, NQ> o[ND];
    float top = LOW, ref = 0.f, sum = 0.f;

    // one turn's rows
    const auto go_through = [&](int turn, Held& here) {
        const int n0 = turn * 32;
        // positions of the turn that are not to be used: past the last one that a row sees, or without a page
        const uint32_t used = here.there & (seen - n0 >= 32 ? ~0u : (1u << (seen - n0)) - 1);
        if (used != ~0u || p.D < DP) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool mine = used >> (16 * i + col) & 1;
#pragma unroll
                for (int c = 0; c < PIECES; ++c)
                    if (!mine || at(c) >= p.D) {
                        here.k[i][c] = here.v[i][c] = Raw{};
                        here.ke[i][c] = here.ve[i][c] = 127;
                    }
            }
        }

        f32x4 s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            Sum<NK, NQ> a;
            a.start();
#pragma unroll
            for (int c = 0; c < PIECES; ++c) {
                const float power = coded<C> ? power_of(here.ke[i][c]) : 1.f;
#pragma unroll
                for (int e = 0; e < P::SEGS; ++e) a.add(parts_of(here.k[i][c], e, power, C()), qf[c][e]);
            }
            a.join();
            s[i] = a.main;
        }
        sm::wave_sync();                     // the tile's last readers are done
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < PIECES; ++c) {
                const float power = coded<C> ? power_of(here.ve[i][c]) : 1.f;
#pragma unroll
                for (int e = 0; e < P::SEGS; ++e) {
                    const sm::Frag<NK> f = parts_of(here.v[i][c], e, power, C());
#pragma unroll
                    for (int n = 0; n < NK; ++n)
                        *reinterpret_cast<bf16x8*>(
                            &tile.x[n * TileT::PLANE + TileT::at(16 * i + col, at(c) / 8 + e)]) = f.p[n];
                }
            }
        sm::wave_sync();

        // scaled after the sum, as in the tiles: equal products stay equal however large the scale is
        float hi = LOW;
        const bool edge = n0 + 31 > least;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] = __builtin_fmaf(s[i][e], c1, 0.f);             // (a product would be contracted with - ref)
                if (used != ~0u || edge) {
                    const int n = 16 * i + 4 * g + e;
                    if (!(used >> n & 1) || n0 + n > seat) s[i][e] = LOW;
                }
                hi = fmaxf(hi, s[i][e]);
            }
        if (__any(hi > top + GROW)) {                                   // top -inf: any score at all
            hi = fmaxf(hi, __shfl_xor(hi, 16));
            hi = fmaxf(hi, __shfl_xor(hi, 32));
            const bool before = top == LOW;
            const float was = ref;
            top = fmaxf(top, hi);
            ref = top == LOW ? 0.f : top;
            const float f = before ? 1.f : sm::exp_of(was - ref);       // the first time there is nothing to scale
            sum *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d].main *= f;
        }
        f32x8 e;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = sm::exp_of(s[i / 4][i % 4] - ref);
        const sm::Frag<NQ> pf = sm::split<NQ>(e);
        if constexpr (NQ == 1) {
            sum = sm::add_all(pf.p[0], sum);                            // of the rounded ones: what is added up
        } else {
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) part += e[i];
            sum += part;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            o[d].start();
            o[d].add(column16<NK, DP>(tile, 16 * d, lane), pf);
            o[d].join();
        }
    };
    if constexpr (AHEAD) {
        // in two sets of registers by turns, so that one turn's rows are waited for while the next ones are on their
        // way
        while (turn < end) {
            Held odd;
            if (turn + NW < end) odd = fetch(pages);
            pages = look(turn + 2 * NW);
            go_through(turn, even);
            turn += NW;
            if (turn >= end) break;
            if (turn + NW < end) even = fetch(pages);
            pages = look(turn + 2 * NW);
            go_through(turn, odd);
            turn += NW;
        }
    } else {
        while (turn < end) {
            pages = look(turn + NW);
            go_through(turn, even);
            turn += NW;
            if (turn < end) even = fetch(pages);
        }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    __syncthreads();                         // the tiles are not read any more
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(&lds.o[wave][col][16 * d + 4 * g]) = o[d].main;
    if (g == 0) {
        join_ref[wave][col] = sum == 0.f ? LOW : ref;
        join_sum[wave][col] = sum;
    }
    __syncthreads();

    // four elements a thread
    const int mine = min(ROWS, rows - r0);
    for (int i = tid; i < mine * (DP / 4); i += 64 * NW) {
        const int row = i / (DP / 4), d = i % (DP / 4) * 4, at_r = r0 + row;
        float to = LOW;
#pragma unroll
        for (int n = 0; n < NW; ++n) to = fmaxf(to, join_ref[n][row]);
        if (to == LOW) to = 0.f;
        f32x4 x = {};
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < NW; ++n) {
            const float f = sm::exp_of(join_ref[n][row] - to);
            s += join_sum[n][row] * f;
            x = x + *reinterpret_cast<const f32x4*>(&lds.o[n][row][d]) * f;
        }
        const int to_head = kvh * share + at_r % share, to_t = seq.first + at_r / share;
        if (unit.parts > 1) {
            const int64_t to_row = (int64_t)unit.at * ROWS + row;
            *reinterpret_cast<f32x4*>(p.step.part + to_row * DP + d) = x;
            if (d == 0) {
                p.step.part2[2 * to_row] = to;
                p.step.part2[2 * to_row + 1] = s;
            }
        } else {
            x = x * (s == 0.f ? 0.f : 1.f / s);
            sm::store4((T*)p.out + to_head * p.so.h + to_t * p.so.r, d, p.D, x);
        }
    }
}

}  // namespace pg
}  // namespace qlka
