// Softmax attention of chunks of new tokens over a cache in pages: the tiles of softmax_fwd.hip over rows that are
// found through the sequence's table.
//
// A workgroup takes 128 rows of one sequence and key head, token by token and within a token the query heads that share
// the key head, so that heads with common keys read (and take apart) them once. Each thread finds the pages of the rows
// that it brings, one tile ahead of them. bf16 rows go to LDS directly, into the other of two buffers; rows of 8 bits
// stay in registers until the tile before is done with and become bf16 on their way into the other buffer (exactly, see
// paged_cache.hip); float rows are split into three parts there, with one buffer.
//
// Bound by vector instructions: 4 chunks of 512 new tokens at 1024 to 8192, 12 / 4 heads, int8: 64 us, 378 TFLOP/s (the
// scores' work; taking 8 bits apart and bringing them 20 us; with bf16 pages 56 us). Two or three waves a SIMD are as
// fast, with four registers spill (120 us).
#pragma once

#include "paged_device.h"

#include <limits>

namespace qlka {
namespace pg {

constexpr int TILE_WAVES = PG_TILE_ROWS / 32;

// A sum of products of operands in NA and NB parts, the smaller parts' apart (softmax_tile.h, Acc).
template <int NA, int NB> struct Gather {
    sm::f32x16 main = {}, rest;
    __device__ __forceinline__ void start() {
        if constexpr (NA + NB > 2) rest = sm::f32x16{};
    }
    __device__ __forceinline__ void add(const sm::Frag<NA>& a, const sm::Frag<NB>& b) {
        if constexpr (NB == 3) rest = sm::mfma(a.p[0], b.p[2], rest);
        if constexpr (NA == 3) {
            rest = sm::mfma(a.p[2], b.p[0], rest);
            rest = sm::mfma(a.p[1], b.p[1], rest);
        }
        if constexpr (NB == 3) rest = sm::mfma(a.p[0], b.p[1], rest);
        if constexpr (NA == 3) rest = sm::mfma(a.p[1], b.p[0], rest);
        main = sm::mfma(a.p[0], b.p[0], main);
    }
    __device__ __forceinline__ void join() {
        if constexpr (NA + NB > 2) main = main + rest;
    }
};

// A key head's first rows of all pages.
struct Heads { const char *k, *v; const uint8_t *ke, *ve; };

// Tiles of keys and values on their way from pages into LDS.
template <class C, int DP, int BN> struct Bring {
    typedef Piece<C, 8> P;
    typedef typename P::raw Raw;
    static constexpr int NP = P::PARTS, NT = 64 * TILE_WAVES, PIECES = DP / 8, BUFFERS = NP == 1 ? 2 : 1;
    static constexpr int APART = NT / PIECES, EACH = BN / APART;       // rows of a thread: one in APART, EACH of them
    static constexpr bool DIRECT = std::is_same<C, __bf16>::value;
    static_assert(APART * PIECES == NT && EACH * APART == BN, "every thread brings as many pieces");
    typedef sm::Tile<NP, BN, DP> TileT;
    struct Lds { TileT k[BUFFERS], v[BUFFERS]; };

    int row, slot;                           // this thread's first row, and its place among the row's pieces
    int page[EACH], at[EACH];                // of the tile that is fetched next: its rows' pages and places in them
    uint32_t ok;                             // which of the rows being brought are there
    Raw k[DIRECT ? 1 : EACH], v[DIRECT ? 1 : EACH];
    uint32_t ke[EACH], ve[EACH];

    __device__ __forceinline__ Bring(Lds& lds, const PgParams& p, int tid)
        : row(tid / PIECES), slot(tid % PIECES), ok(0) {
        if (DIRECT && p.D < DP) {            // pieces past D stay as they are
            bf16x8* x = reinterpret_cast<bf16x8*>(&lds);
            for (int i = tid; i < (int)(sizeof(Lds) / 16); i += NT) x[i] = bf16x8{};
            __syncthreads();
        }
    }
    // the pages of tile t
    __device__ __forceinline__ void look(const PgParams& p, const int* table, int t, int seen) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int n = t * BN + row + i * APART;
            const Place place = place_of(p, min(n, seen - 1));
            page[i] = n < seen ? table[place.index] : -1;
            at[i] = place.row;
        }
    }
    // the tile whose pages have been looked up
    __device__ __forceinline__ void fetch(Lds& lds, int buffer, const PgParams& p, const Heads& heads, int tid) {
        ok = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const bool there = (uint32_t)page[i] < (uint32_t)p.num_pages;
            ok |= (uint32_t)there << i;
            // a row's pieces are turned by bits of its number: where they go, or, straight to LDS, where they come from
            const int piece = DIRECT ? slot ^ TileT::turn(row + i * APART) : slot, d = piece * 8;
            if constexpr (DIRECT) {
                const int first = (tid >> 6) * (64 / PIECES) + i * APART;        // of the wave's rows
                const uint32_t to_k = sm::lds_place(&lds.k[buffer].x[first * DP]);
                const uint32_t to_v = sm::lds_place(&lds.v[buffer].x[first * DP]);
                if (d >= p.D) continue;
                if (there) {
                    sm::load_to_lds(heads.k + bytes_to(p.sk, page[i], at[i]) + d * P::SIZE, to_k);
                    sm::load_to_lds(heads.v + bytes_to(p.sv, page[i], at[i]) + d * P::SIZE, to_v);
                } else {
                    *reinterpret_cast<bf16x8*>(&lds.k[buffer].x[(row + i * APART) * DP + slot * 8]) = bf16x8{};
                    *reinterpret_cast<bf16x8*>(&lds.v[buffer].x[(row + i * APART) * DP + slot * 8]) = bf16x8{};
                }
            } else {
                // what is not there is read from a place that is, and dropped in put(): no load waits for a test
                const uint32_t from = there ? page[i] : 0, e = d < p.D ? d : 0;
                k[i] = *reinterpret_cast<const Raw*>(heads.k + bytes_to(p.sk, from, at[i]) + e * P::SIZE);
                v[i] = *reinterpret_cast<const Raw*>(heads.v + bytes_to(p.sv, from, at[i]) + e * P::SIZE);
                if constexpr (coded<C>) {
                    ke[i] = heads.ke[bytes_to(p.ske, from, at[i]) + e / BLOCK];
                    ve[i] = heads.ve[bytes_to(p.sve, from, at[i]) + e / BLOCK];
                }
            }
        }
    }
    // the rows that were fetched into registers to LDS
    __device__ __forceinline__ void put(Lds& lds, int buffer, int D) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (!(ok >> i & 1) || slot * 8 >= D) {
                k[i] = v[i] = Raw{};
                ke[i] = ve[i] = 127;
            }
            const sm::Frag<NP> x = parts_of(k[i], 0, coded<C> ? power_of(ke[i]) : 1.f, C());
            const sm::Frag<NP> y = parts_of(v[i], 0, coded<C> ? power_of(ve[i]) : 1.f, C());
            const int at = TileT::at(row + i * APART, slot);
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                *reinterpret_cast<bf16x8*>(&lds.k[buffer].x[n * TileT::PLANE + at]) = x.p[n];
                *reinterpret_cast<bf16x8*>(&lds.v[buffer].x[n * TileT::PLANE + at]) = y.p[n];
            }
        }
    }
    // 0 or -inf for each of the tile's rows
    __device__ __forceinline__ void put_mask(float* mask) {
        if (slot == 0) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) mask[row + i * APART] = ok >> i & 1 ? 0.f : LOW;
        }
    }
};

template <class T, class C, int DP> constexpr int tiles_room() { return sm::Elem<T>::PARTS == 3 && DP == 128 ? 1 : 2; }

template <class T, class C, int DP> __device__ __forceinline__ void tiles(const PgParams& p, int wg) {
    constexpr int NQ = sm::Elem<T>::PARTS, NK = Piece<C, 8>::PARTS;
    constexpr int BN = sm_tile_rows(NK, DP), NS = BN / 32, ND = DP / 32;
    constexpr int ROWS = PG_TILE_ROWS, NT = 64 * TILE_WAVES;
    typedef Bring<C, DP, BN> BringT;
    static_assert(Units<false, ROWS>::ALIGN % BN == 0);
    __shared__ __attribute__((aligned(16))) typename BringT::Lds lds;
    __shared__ __attribute__((aligned(16))) float mask_of[BringT::BUFFERS][BN];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const int share = p.H / p.G;
    const Units<false, ROWS> units(p, p.tiles);
    const Unit unit = units.of(wg);
    if (unit.b < 0) return;
    const Tokens seq = units.tokens(unit.b);
    const int kvh = unit.kvh, rows = seq.rows * share, r0 = unit.block * ROWS, rw = r0 + wave * 32, r = rw + col;

    const bool real = r < rows;
    const int head = kvh * share + r % share, t_q = seq.first + r / share;
    const int last = seq.start + min(r0 + ROWS - 1, rows - 1) / share;              // the workgroup's last position
    const int wave_first = seq.start + rw / share, wave_last = seq.start + min(rw + 31, rows - 1) / share;
    const int seat = seq.start + r / share;
    const int seen = seen_from(p, last);
    if (unit.part && (int64_t)unit.part * unit.span >= seen) return;   // (the first part leaves zeros all the same)
    int t = unit.part * (unit.span / BN);
    const int t1 = min(t + unit.span / BN, (seen + BN - 1) / BN);

    const int* table = p.tables + unit.b * p.table_stride;
    const Heads heads = {p.k_pages + (uint64_t)kvh * p.sk.head, p.v_pages + (uint64_t)kvh * p.sv.head,
                         p.k_exp + (uint64_t)kvh * p.ske.head, p.v_exp + (uint64_t)kvh * p.sve.head};
    // whether some page here does not exist
    bool lacks = false;
    if (t < t1) {
        const int end = place_of(p, min(t1 * BN, seen) - 1).index;
        for (int i = place_of(p, t * BN).index + tid; i <= end; i += NT)
            lacks |= (uint32_t)table[i] >= (uint32_t)p.num_pages;
    }
    lacks = __syncthreads_or(lacks);
    BringT tile(lds, p, tid);
    constexpr bool DIRECT = BringT::DIRECT;
    int buffer = 0, next = t;                          // next: the tile to be fetched
    const auto fetch = [&](int to) {
        tile.fetch(lds, to, p, heads, tid);
        if (DIRECT && lacks) tile.put_mask(mask_of[to]);
        ++next;
        tile.look(p, table, min(next, t1 - 1), seen);
    };
    if (t < t1) {
        tile.look(p, table, t, seen);
        fetch(0);
    }

    sm::Frag<NQ> qf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        typename sm::Elem<T>::seg s = {};
        if (real) s = sm::load_seg((const T*)p.q + head * p.sq.h + t_q * p.sq.r, 16 * c + 8 * half, p.D);
        s = s * (T)p.q_sign;
        qf[c] = sm::frag_of(s);
    }

    const float c1 = p.scale * sm::UNIT;
    Gather<NK, NQ> o[ND];
    float top = LOW, ref = 0.f, sum = 0.f;
    bool wide = false;                                 // a row here has a large ref

    for (; t < t1; ++t) {
        const int n0 = t * BN;
        if constexpr (BringT::BUFFERS == 1) __syncthreads();             // nobody reads it any more
        if constexpr (DIRECT) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else {
            tile.put(lds, buffer, p.D);
            if (lacks) tile.put_mask(mask_of[buffer]);
        }
        __syncthreads();
        const float* mask = mask_of[buffer];
        const auto& kt = lds.k[buffer];
        const auto& vt = lds.v[buffer];
        buffer ^= BringT::BUFFERS - 1;
        // (into registers the last tile is fetched once more: what is fetched behind a test is waited for where the
        // paths meet)
        if (!DIRECT || t + 1 < t1) fetch(buffer);
        if (rw >= rows || n0 > wave_last) continue;

        sm::f32x16 s[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            Gather<NK, NQ> a;
            a.start();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) a.add(kt.row(32 * i + col, 16 * c + 8 * half), qf[c]);
            __builtin_amdgcn_s_setprio(0);
            a.join();
            s[i] = a.main;
        }
        if (lacks) {
#pragma unroll
            for (int i = 0; i < NS; ++i) s[i] = sm::masked(s[i], mask, 32 * i + 4 * half);
        }
        if (n0 + BN - 1 > min(wave_first, seen - 1)) {
            const int lim = min(seat, seen - 1) - n0 - 4 * half;         // the last key seen
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * i + sm::reg_row(e) > lim) s[i][e] = LOW;
        }
        float hi = s[0][0];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) hi = fmaxf(hi, s[i][e]);
        hi = fmaxf(hi, sm::other_half(hi)) * c1;
        if (__any(hi > top + GROW)) {                                    // top -inf: any score at all
            const bool before = top == LOW;
            const float was = ref;
            top = fmaxf(top, hi);
            ref = top == LOW ? 0.f : top;
            wide = __any(fabsf(ref) > sm::WIDE);
            const float f = before ? 1.f : sm::exp_of(was - ref);        // the first time there is nothing to scale
            sum *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d].main *= f;
        }
        float mul = 2.f * c1, add = -2.f * ref;
        if (__builtin_expect(wide, 0)) {               // scores are rounded before the reference is taken off (WIDE)
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[i][e] = __builtin_fmaf(s[i][e], c1, 0.f) - ref;      // (a product would be contracted with it)
                }
            mul = 2.f;
            add = 0.f;
        }
        float tile_sum = 0.f;                          // by tiles: thousands of terms one by one lose two digits more
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d].start();
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f32x8 e = sm::eight(s[i], c);
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = sm::fexp2(__builtin_fmaf(e[j], mul, add));
                const sm::Frag<NQ> pf = sm::split<NQ>(e);
                if constexpr (NQ == 1) {
                    sum = sm::add_all(pf.p[0], sum);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) tile_sum += e[j];
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d].add(vt.column(32 * i + 16 * c, 32 * d, lane), pf);
            }
        sum += tile_sum;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d].join();
    }
    if (!real) return;
    sum += sm::other_half(sum);
    if (unit.parts > 1) {
        const int64_t at = (int64_t)unit.at * ROWS + (r - r0);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<f32x4*>(p.tiles.part + at * DP + 32 * d + 8 * e + 4 * half) = sm::quad(o[d].main, e);
        if (half == 0) {
            p.tiles.part2[2 * at] = ref;
            p.tiles.part2[2 * at + 1] = sum;
        }
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = (T*)p.out + head * p.so.h + t_q * p.so.r;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sm::store4(out, 32 * d + 8 * e + 4 * half, p.D, sm::quad(o[d].main, e) * inv);
}

}  // namespace pg
}  // namespace qlka
