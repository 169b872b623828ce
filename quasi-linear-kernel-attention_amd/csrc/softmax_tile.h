// Device pieces of the softmax attention kernels (gfx950, wave64): matrix fragments, tiles in LDS, masks, buckets.
//
// Products run on v_mfma_f32_32x32x16_bf16 (lane l: row or column l % 32, elements 8 (l / 32) + 0..7 of a 16-element
// chunk; result: column l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4 for register r). The scores are formed with the
// other side's rows in the registers, so a lane holds scores of one row (or one key), and eight successive result
// registers are, as they are, the second operand of the next product: its 16-element chunk is taken in the order
//   slot (half, j) <- element 8 (j / 4) + 4 half + j % 4,
// and the first operand is read from LDS in that order, transposed, by ds_read_b64_tr_b16 (four successive rows of one
// column a lane). No score crosses lanes or goes through LDS.
//
// float inputs are split into three bf16 parts of 8 bits each (24 in all), and a product is the six products of parts
// whose sizes add up to 2^-16 of the largest or more; what is left out is below 2^-26 of it. At the rates of large
// products (bf16 1215 TFLOP/s, fp32 152, measured) six of them are 1.33 times as fast as one in fp32. An infinity among
// the inputs gives NaN this way.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>
#include <type_traits>

#include "softmax.h"

namespace qlka {
namespace sm {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

// Scores, biases and log sums are held in units of 2 ln 2, halves of a power of two: in units of ln 2 the number of a
// score is larger than the score, and the lowest finite bias, with which a bucket is hidden, would become -inf. exp2 of
// twice the number is e to the score.
constexpr float UNIT = 0.72134752044448170f;
// Where a row's reference (its maximum, its log sum) is larger, scores are rounded before it is taken off: it is a
// rounded score itself, and the exact product in fma(score, scale, bias - reference) would be off from it by up to half
// its last place, which is 2^-15 here and grows to any factor of the exponential.
constexpr float WIDE = 512.f;

template <class T> struct Elem;
template <> struct Elem<__bf16> { static constexpr int PARTS = 1; typedef bf16x8 seg; };
template <> struct Elem<float> { static constexpr int PARTS = 3; typedef f32x8 seg; };

template <int NP> struct Frag { bf16x8 p[NP]; };

template <int NP> __device__ __forceinline__ Frag<NP> split(f32x8 x) {
    Frag<NP> f;
    f.p[0] = __builtin_convertvector(x, bf16x8);
    if constexpr (NP == 3) {
        x = x - __builtin_convertvector(f.p[0], f32x8);
        f.p[1] = __builtin_convertvector(x, bf16x8);
        x = x - __builtin_convertvector(f.p[1], f32x8);
        f.p[2] = __builtin_convertvector(x, bf16x8);
    }
    return f;
}
__device__ __forceinline__ Frag<1> frag_of(bf16x8 x) { return Frag<1>{{x}}; }
__device__ __forceinline__ Frag<3> frag_of(f32x8 x) { return split<3>(x); }

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// A sum of products. The matrix instruction drops what of a product lies a few bits below the sum's last one, always
// downwards: 0.007 of a last place an instruction, measured, which a long sum of few signs would show. So the five
// products of the smaller parts gather in a sum of their own, 2^-8 as large, until join().
template <int NP> struct Acc {
    f32x16 main = {}, rest;
    __device__ __forceinline__ Acc() {}
    __device__ __forceinline__ explicit Acc(f32x16 from) : main(from) {}
    __device__ __forceinline__ void start() {
        if constexpr (NP == 3) rest = f32x16{};
    }
    __device__ __forceinline__ void add(const Frag<NP>& a, const Frag<NP>& b) {
        if constexpr (NP == 3) {
            rest = mfma(a.p[0], b.p[2], rest);
            rest = mfma(a.p[2], b.p[0], rest);
            rest = mfma(a.p[1], b.p[1], rest);
            rest = mfma(a.p[0], b.p[1], rest);
            rest = mfma(a.p[1], b.p[0], rest);
        }
        main = mfma(a.p[0], b.p[0], main);
    }
    // the same sum, bit for bit, as add(b, a)
    __device__ __forceinline__ void add_turned(const Frag<NP>& a, const Frag<NP>& b) {
        if constexpr (NP == 3) {
            rest = mfma(a.p[2], b.p[0], rest);
            rest = mfma(a.p[0], b.p[2], rest);
            rest = mfma(a.p[1], b.p[1], rest);
            rest = mfma(a.p[1], b.p[0], rest);
            rest = mfma(a.p[0], b.p[1], rest);
        }
        main = mfma(a.p[0], b.p[0], main);
    }
    __device__ __forceinline__ void join() {
        if constexpr (NP == 3) main = main + rest;
    }
};

__device__ __forceinline__ f32x8 floats(bf16x8 x) { return __builtin_convertvector(x, f32x8); }
__device__ __forceinline__ f32x8 floats(f32x8 x) { return x; }
// registers 4 r .. 4 r + 3: four successive rows of a result
__device__ __forceinline__ f32x4 quad(f32x16 x, int r) {
    return f32x4{x[4 * r], x[4 * r + 1], x[4 * r + 2], x[4 * r + 3]};
}
// a result's 16 rows of x from x[first] on (first includes 4 (lane / 32))
__device__ __forceinline__ f32x16 rows_of(const float* x, int first) {
    f32x16 y;
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 z = *reinterpret_cast<const f32x4*>(x + first + 8 * r4);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * r4 + j] = z[j];
    }
    return y;
}
// registers 8 c .. 8 c + 7: the second operand's chunk c
__device__ __forceinline__ f32x8 eight(f32x16 x, int c) {
    f32x8 y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = x[8 * c + j];
    return y;
}
// x[0] + x[1] + ... of eight bf16
__device__ __forceinline__ float add_all(bf16x8 x, float to) {
    const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) to = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[2 * i], x[2 * i + 1]}, one, to, false);
    return to;
}
// What this wave's lanes wrote to LDS before, its other lanes read after (LDS serves a wave in order: no instruction,
// only an order for the compiler).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }
// A row's log sum, ref + log2(sum) / 2, in two floats: the second is what the first one's rounding drops. With a large
// ref that is all of log2(sum), without which each of n equal keys would have the probability 1.
__device__ __forceinline__ void store_lse(const SmParams& p, int64_t row, float ref, float sum) {
    const float l = 0.5f * __log2f(sum), hi = ref + l, back = hi - ref;
    if (p.log2_sum) p.log2_sum[row] = sum == 0.f ? __builtin_inff() : hi + hi;
    if (p.lse) p.lse[row] = sum == 0.f ? __builtin_inff() : hi;
    if (p.lse_low) p.lse_low[row] = sum == 0.f ? 0.f : (ref - (hi - back)) + (l - back);
}
// Whether a row's log sum is one to take off in two steps, after the score is rounded (WIDE).
__device__ __forceinline__ bool large_lse(float lse) { return fabsf(lse) > WIDE && lse != __builtin_inff(); }
// P of such a row from (score - lse) - lse_low: 1 at most, however the score was rounded here and in the forward
__device__ __forceinline__ float at_most_0(float x) { return x > 0.f ? 0.f : x; }
// e to a score
__device__ __forceinline__ float exp_of(float x) { return fexp2(x + x); }
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }
__device__ __forceinline__ int reg_row(int r) { return (r >> 2) * 8 + (r & 3); }   // + 4 (lane / 32)

// Eight elements d .. d + 7 of a row of D, a multiple of 8; zeros past D.
template <class T> __device__ __forceinline__ typename Elem<T>::seg load_seg(const T* row, int d, int D) {
    typename Elem<T>::seg x = {};
    if (d < D) x = *reinterpret_cast<const typename Elem<T>::seg*>(row + d);
    return x;
}

// A tile of ROWS rows of DP elements in LDS, one plane for each part, without gaps. A row's 16-byte pieces are turned
// (exclusive or) by bits of the row's number, so that the two pieces of 4 rows that a transposing read takes in a cycle
// are on different banks: at 64 elements such reads count no conflict. LDS serves 16 lanes' pieces in a cycle, of 16
// rows when a row is read, among which the turn repeats at 64 elements: each such read takes 8 cycles for 4
// (SQ_LDS_BANK_CONFLICT is 4 cycles a read in every kernel here).
template <int NP, int ROWS, int DP> struct Tile {
    static constexpr int PLANE = ROWS * DP, PIECES = DP / 8;
    alignas(16) __bf16 x[NP * PLANE];

    static __device__ __forceinline__ int turn(int row) {
        return DP == 32 ? (row & 2) | (row >> 2 & 1) : (row & 3) << 1 | (row >> 2 & 1);
    }
    static __device__ __forceinline__ int at(int row, int piece) { return row * DP + ((piece ^ turn(row)) << 3); }

    template <class Seg> __device__ __forceinline__ void put(int row, int piece, Seg s) {
        const Frag<NP> f = frag_of(s);
#pragma unroll
        for (int i = 0; i < NP; ++i) *reinterpret_cast<bf16x8*>(&x[i * PLANE + at(row, piece)]) = f.p[i];
    }
    // elements d .. d + 7 of a row
    __device__ __forceinline__ Frag<NP> row(int row, int d) const {
        Frag<NP> f;
#pragma unroll
        for (int i = 0; i < NP; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(&x[i * PLANE + at(row, d >> 3)]);
        return f;
    }
    // column d0 + lane % 32 over rows row0 .. row0 + 15, in the slots' order
    __device__ __forceinline__ Frag<NP> column(int row0, int d0, int lane) const {
        const int row = row0 + 4 * (lane >> 5) + ((lane & 15) >> 2);
        const int from = at(row, (d0 >> 3) + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) + (lane & 1) * 4;
        Frag<NP> f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            union { s16x4 s[2]; bf16x8 b; } u;
            typedef __attribute__((address_space(3))) s16x4 lds4;
            u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)&x[i * PLANE + from]);
            u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)&x[i * PLANE + from + 8 * DP]);   // turned alike
            f.p[i] = u.b;
        }
        return f;
    }
};

// Rows of the tiles that a workgroup goes through.
template <class T, int DP> struct Shape {
    static constexpr int NP = Elem<T>::PARTS;
    static constexpr int BN = sm_tile_rows(NP, DP);
    // Waves a SIMD has room for. From 2 on a wave has 256 registers at most, and the compiler keeps sums in those that
    // vector instructions can reach; with 1 it puts them in the others and copies every score.
    static constexpr int WAVES = NP == 3 && DP == 128 ? 1 : 2;
};

// 16 bytes a lane from memory to LDS, lane l's to `to` + 16 l bytes. Written out because of the waits: before every
// transposing read the compiler would wait for its own form of this, though that goes to the other buffer.
// Pair::arrive() waits. The low half of a generic pointer into LDS is the place in LDS.
__device__ __forceinline__ uint32_t lds_place(const void* to) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)to);
}
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(to), "v"(from) : "memory", "m0");
}
// from is the same for all lanes
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t bytes, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(to), "v"(bytes), "s"(from) : "memory", "m0");
}

// Two tiles (k and v, or q and dO) of ROWS rows on their way into LDS, where a workgroup of NW waves then reads them.
//
// bf16 goes there directly (global_load_lds, 16 bytes a lane, 1 KB an instruction; the pieces are turned by reading
// from turned places), into the other one of two buffers while the current one is read: no registers hold a tile, and
// one barrier a tile is enough. float goes through registers, where it is split into parts, and has one buffer and two
// barriers. Rows that are not to be read become zeros.
template <class T, int DP, int ROWS, int NW> struct Pair {
    static constexpr int NP = Elem<T>::PARTS, NT = 64 * NW, PIECES = DP / 8, BUFFERS = NP == 1 ? 2 : 1;
    static constexpr uint64_t ALL = ROWS == 64 ? ~0ull : (1ull << ROWS % 64) - 1;
    typedef Tile<NP, ROWS, DP> TileT;
    struct Lds { TileT a[BUFFERS], b[BUFFERS]; };
    static_assert(alignof(Lds) >= 16, "pieces of 16 bytes are read, written and loaded");
    static constexpr int HELD = NP == 1 ? 1 : ROWS * PIECES / NT, STEP = NT / PIECES;
    static_assert(NP == 1 || (HELD * NT == ROWS * PIECES && STEP * PIECES == NT),
                  "a thread takes one column of HELD rows");

    // Rows whose pieces a lane takes: the first one, and every APART-th after it.
    static constexpr int RPI = 64 / PIECES, EACH = ROWS / RPI / NW, APART = RPI * NW;
    static constexpr bool ALIKE = APART % 8 == 0 || EACH == 1;       // they are turned alike

    int64_t stride_a, stride_b;
    bool near, has;                        // rows within 32 bits of their tile; this lane's piece is not past D
    uint32_t at_a, at_b;                   // bytes from a tile's first row to this lane's piece
    typename Elem<T>::seg a[HELD], b[HELD];

    __device__ __forceinline__ Pair(Lds& lds, int64_t stride_a, int64_t stride_b, int D, int tid)
        : stride_a(stride_a), stride_b(stride_b) {
        near = stride_a < 1 << 22 && stride_b < 1 << 22 && (NP != 1 || ALIKE);
        int row = tid / PIECES, piece = tid % PIECES;
        if constexpr (NP == 1) piece ^= TileT::turn(row);
        has = piece * 8 < D;
        at_a = (uint32_t)(row * stride_a + piece * 8) * sizeof(T);
        at_b = (uint32_t)(row * stride_b + piece * 8) * sizeof(T);
        if (NP == 1 && D < DP) {           // pieces past D stay as they are
            bf16x8* x = reinterpret_cast<bf16x8*>(&lds);
            for (int i = tid; i < (int)(sizeof(Lds) / 16); i += NT) x[i] = bf16x8{};
            __syncthreads();
        }
    }
    // tile_a, tile_b: first rows; bits: the rows to read
    __device__ __forceinline__ void fetch(Lds& lds, int buffer, const T* tile_a, const T* tile_b, uint64_t bits, int D,
                                          int tid) {
        if (near && bits == ALL) {                         // without a test for each row
            if constexpr (NP == 1) {
                const uint32_t to_a = lds_place(&lds.a[buffer].x[(tid >> 6) * RPI * DP]);
                const uint32_t to_b = lds_place(&lds.b[buffer].x[(tid >> 6) * RPI * DP]);
                if (has) {
#pragma unroll
                    for (int j = 0; j < EACH; ++j)
                        load_to_lds(tile_a + j * APART * stride_a, at_a, to_a + j * APART * DP * 2);
#pragma unroll
                    for (int j = 0; j < EACH; ++j)
                        load_to_lds(tile_b + j * APART * stride_b, at_b, to_b + j * APART * DP * 2);
                }
            } else {
                typedef const typename Elem<T>::seg* segs;
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    a[i] = b[i] = {};
                    if (!has) continue;
                    a[i] = *(segs)((const char*)(tile_a + i * STEP * stride_a) + at_a);
                    b[i] = *(segs)((const char*)(tile_b + i * STEP * stride_b) + at_b);
                }
            }
        } else if constexpr (NP == 1) {
#pragma unroll 1
            for (int j = 0; j < EACH; ++j) {
                const int first = (tid >> 6) * RPI + j * APART, row = first + (tid & 63) / PIECES;
                const int slot = tid % PIECES, piece = slot ^ TileT::turn(row);
                const uint32_t to_a = lds_place(&lds.a[buffer].x[first * DP]);
                const uint32_t to_b = lds_place(&lds.b[buffer].x[first * DP]);
                if (piece * 8 >= D) continue;
                if (bits >> row & 1) {
                    load_to_lds(tile_a + row * stride_a + piece * 8, to_a);
                    load_to_lds(tile_b + row * stride_b + piece * 8, to_b);
                } else {
                    *reinterpret_cast<bf16x8*>(&lds.a[buffer].x[row * DP + slot * 8]) = bf16x8{};
                    *reinterpret_cast<bf16x8*>(&lds.b[buffer].x[row * DP + slot * 8]) = bf16x8{};
                }
            }
        } else {
            const int row = tid / PIECES, d = tid % PIECES * 8;
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                a[i] = b[i] = {};
                if (!has || !(bits >> (row + i * STEP) & 1)) continue;
                a[i] = load_seg(tile_a + (row + i * STEP) * stride_a, d, D);
                b[i] = load_seg(tile_b + (row + i * STEP) * stride_b, d, D);
            }
        }
    }
    // until here the fetched tile has arrived and nobody reads the buffer that the next fetch goes to; between two
    // calls of it what `more` writes is read
    template <class F> __device__ __forceinline__ void arrive(Lds& lds, int tid, F more) {
        if constexpr (NP == 1) {
            more();
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                lds.a[0].put(tid / PIECES + i * STEP, tid % PIECES, a[i]);
                lds.b[0].put(tid / PIECES + i * STEP, tid % PIECES, b[i]);
            }
            more();
            __syncthreads();
        }
    }
};

// 4 bytes' truth as 4 bits
__device__ __forceinline__ uint32_t truth4(uint32_t w) {
    const uint32_t y = ((((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) >> 7) & 0x01010101u;
    return (y * 0x10204080u) >> 28;
}

__device__ __forceinline__ uint64_t lane_u64(uint64_t x, int lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane) << 32;
}

// The keys of each tile of BN that a batch's mask keeps, one bit a key; 64 tiles are looked at together, one a lane.
template <int BN> struct KeyBits {
    const uint8_t* keep;       // the batch's row, or null
    int N, window;             // N: keys that are seen
    uint64_t bits;             // of tile 64 * window + lane

    __device__ __forceinline__ KeyBits(const SmParams& p, int b)
        : keep(p.keep ? p.keep + b * p.keep_stride : nullptr), N(p.seen), window(-1), bits(0) {}

    __device__ __forceinline__ void look(int w) {
        if (w == window) return;
        window = w;
        const int64_t n0 = ((int64_t)w * 64 + (threadIdx.x & 63)) * BN, left = N - n0;
        bits = 0;
#pragma unroll 1
        for (int j = 0; j < BN && j < left; j += 16) {
            uint64_t t = 0;
            if (left - j >= 16) {
                typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(1)));
                const u32x4 x = *reinterpret_cast<const u32x4*>(keep + n0 + j);
                t = truth4(x.x) | truth4(x.y) << 4 | truth4(x.z) << 8 | truth4(x.w) << 12;
            } else {
                for (int i = 0; i < left - j; ++i) t |= (uint64_t)(keep[n0 + j + i] != 0) << i;
            }
            bits |= t << j;
        }
    }
    // moves t to the first tile from t on, before end, that has a key, and gives its keys; 0 where there is none
    __device__ __forceinline__ uint64_t find(int& t, int end) {
        if (!keep) {
            const int left = N - t * BN;
            return t >= end ? 0 : left >= BN ? (BN == 64 ? ~0ull : (1ull << BN % 64) - 1) : (1ull << left) - 1;
        }
        while (t < end) {
            look(t >> 6);
            const uint64_t any = __ballot(bits != 0) >> (t & 63);
            if (any) {
                t += __builtin_ctzll(any);
                return t < end ? lane_u64(bits, t & 63) : 0;
            }
            t = (t | 63) + 1;
        }
        return 0;
    }
};

// The bias of one head in LDS: its column of the table, and the borders.
struct BiasLds {
    float value[QLKA_MAX_BUCKETS];
    int border[QLKA_MAX_BUCKETS];
    __device__ __forceinline__ void fill(const SmParams& p, int head, int tid, int nt) {
        const int nb = (p.bk.n + 1) * (p.bk.both ? 2 : 1);
        for (int i = tid; i < nb; i += nt) value[i] = p.table[(int64_t)i * p.H + head] * UNIT;
        for (int i = tid; i < p.bk.n; i += nt) border[i] = p.bk.border[i];
    }
};

// The masked keys of a tile: 0 or -inf for each.
template <int BN> __device__ __forceinline__ void put_mask(float* mask, uint64_t bits, int tid) {
    if (tid < BN) mask[tid] = bits >> tid & 1 ? 0.f : -__builtin_inff();
}
// Scores with -inf for masked keys (whatever stood there); first as for rows_of.
__device__ __forceinline__ f32x16 masked(f32x16 s, const float* mask, int first) {
    const f32x16 z = rows_of(mask, first);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = z[r] == 0.f ? s[r] : z[r];
    return s;
}

// number of borders <= dist
__device__ __forceinline__ int count_borders(const int* border, int n, int dist) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (border[mid] <= dist) lo = mid + 1; else hi = mid;
    }
    return lo;
}
// bucket of the distance diff = key - query
__device__ __forceinline__ int bucket_of(const int* border, int n, int both, int diff) {
    const int dist = diff <= 0 ? -diff : both ? diff : 0;
    return count_borders(border, n, dist) + (both && diff > 0 ? n + 1 : 0);
}

// Where all distances from lo to hi are in one bucket far from the diagonal: that bucket, else -1.
__device__ __forceinline__ int far_bucket(const SmBuckets& bk, int lo, int hi) {
    if (hi <= -bk.far) return bk.n;
    if (bk.both) return lo >= bk.far && lo > 0 ? 2 * bk.n + 1 : -1;
    return lo >= 0 ? 0 : -1;
}

// The work of a workgroup: `blocks` blocks of each of `pairs` (batch, head) pairs. Workgroups go round the 8 XCDs; all
// blocks of a pair go to one of them, whose L2 then serves its keys, and successive pairs to different ones, since the
// heads of a batch with more keys are next to each other. The pairs that are left over are spread over all.
struct Work { int pair, block; };
__device__ __forceinline__ Work xcd_work(int wg, int pairs, int blocks) {
    const int full = (pairs >> 3) * blocks, slot = wg >> 3;
    if (slot < full) return {slot / blocks * 8 + (wg & 7), slot % blocks};
    const int rest = wg - 8 * full;
    return {(pairs & ~7) + rest / blocks, rest % blocks};
}

// f(element, padded row length) for a call's type and row length.
template <class F> int dispatch(int dtype, int D, F f) {
    const int DP = sm_padded(D);
    const auto at = [&](auto t) {
        return DP == 32   ? f(t, std::integral_constant<int, 32>())
               : DP == 64 ? f(t, std::integral_constant<int, 64>())
                          : f(t, std::integral_constant<int, 128>());
    };
    return dtype == QLKA_BF16 ? at(__bf16()) : at(float());
}

// Stores four successive elements d .. d + 3 of a row of D.
template <class T> __device__ __forceinline__ void store4(T* row, int d, int D, f32x4 x) {
    if (d >= D) return;
    if constexpr (sizeof(T) == 2) *reinterpret_cast<bf16x4*>(row + d) = __builtin_convertvector(x, bf16x4);
    else *reinterpret_cast<f32x4*>(row + d) = x;
}

}  // namespace sm
}  // namespace qlka
