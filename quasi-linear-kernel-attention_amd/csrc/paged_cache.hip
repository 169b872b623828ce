// A cache of keys and values in pages, written as tokens come and read back (include/qlka.h).
//
// With 8 bits held, 32 elements of a row share a power of two: the least one, 2^e, whose multiple by the largest code
// reaches the largest of them. x / 2^e, the code's rounding (nearest, ties to the even one) and code * 2^e are then
// exact but for that rounding, in any type that holds x: what is written is what the definition says, to the bit, and
// products of what is read need no further rounding (int8 and e4m3 values have at most 7 and 4 bits, bf16 has 8). A
// scale of largest / 127 would use up to one bit more of int8, but every reader would round.
//
// Both kernels are bound by memory, and at few rows by the latency of offsets and lengths, table and store, one after
// the other (the rows themselves are loaded meanwhile). DP / 8 lanes take a row, 8 elements each; 4 lanes find a
// block's largest element. A wave writes one token's rows of all heads, keys and values, so that the sequence is looked
// up once for all of them. 8 prompts of 200 to 4096 (10211 tokens of 12 heads of 64, bf16 to int8): 14 us for 49 MB;
// read back padded: 17.5 us for 117 MB; 64 tokens: 3.6 us.
#include "paged_device.h"

namespace qlka {
namespace pg {

// The exponent (plus 127) of a block whose largest element is `most`: the least of [27, top] with most <= largest *
// 2^(e - 127), largest = MANT * 2^SHIFT with MANT in [1, 2); 255 if it is not finite.
template <class C> __device__ __forceinline__ uint32_t exponent_of(float most) {
    constexpr bool INT = std::is_same<C, Int8>::value;
    constexpr uint32_t MANT = INT ? 0x7e0000u : 0x600000u;            // of 127 = 1.984375 * 2^6, of 448 = 1.75 * 2^8
    constexpr int SHIFT = INT ? 6 : 8, TOP = INT ? 248 : 246;
    const uint32_t bits = __float_as_uint(most);
    if (bits >= 0x7f800000u) return 255;
    const int e = (int)(bits >> 23) - SHIFT + ((bits & 0x7fffffu) > MANT ? 1 : 0);
    return (uint32_t)min(max(e, LEAST_EXP), TOP);
}

template <class C> __device__ __forceinline__ u32x2 codes_of(f32x8 x, uint32_t e) {
    const float s = __uint_as_float((254 - min(e, 253u)) << 23);       // 2^(127 - e)
    u32x2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (std::is_same<C, Int8>::value) {
            // next to 1.5 * 2^23 a float's last place is 1: the sum is rounded as it should be, and its low byte is the
            // code
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] = __float_as_uint(__builtin_amdgcn_fmed3f(x[4 * h + i] * s, -127.f, 127.f) + 12582912.f);
            const uint32_t lo = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400);
            const uint32_t hi = __builtin_amdgcn_perm(y[3], y[2], 0x0c0c0400);
            w[h] = e == 255 ? 0u : lo | hi << 16;
        } else {
            float c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = __builtin_amdgcn_fmed3f(x[4 * h + i] * s, -448.f, 448.f);
            int y = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
            y = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], y, true);
            w[h] = e == 255 ? 0x7f7f7f7fu : (uint32_t)y;
        }
    }
    return w;
}

// One wave a token: its rows of all heads, keys then values, DP / 8 lanes a row.
template <class T, class C, int DP> __global__ __launch_bounds__(256) void paged_write(const PgParams p) {
    constexpr int LANES = DP / 8, AT_ONCE = 64 / LANES, AHEAD = 4;
    const int lane = threadIdx.x & 63;
    const int token = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), d = lane % LANES * 8;
    if (token >= p.T) return;
    typedef typename sm::Elem<T>::seg Seg;
    const int last = 2 * p.G - 1;
    // Row i: keys, then values. What all lanes share of an address is found once, for both.
    const T *k = (const T*)p.k + token * p.snk.r, *v = (const T*)p.v + token * p.snv.r;
    const auto load = [&](int i) {
        const bool key = i < p.G;
        return sm::load_seg((key ? k : v) + (key ? i : i - p.G) * (key ? p.snk.h : p.snv.h), d, p.D);
    };
    // the first rows are on their way while the place is found
    Seg ahead[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) ahead[j] = load(min(lane / LANES + j * AT_ONCE, last));
    const Found found = find(p, token, tokens_of_lane(p));
    if (found.b < 0) return;
    // offsets and lengths are the caller's: whatever they are, a position without a place is none
    const int seat = found.tokens.start + token - found.tokens.first;
    if (seat < 0 || seat >= p.places) return;
    const Place place = place_of(p, __builtin_amdgcn_readfirstlane(seat));
    const uint32_t page = __builtin_amdgcn_readfirstlane(p.tables[found.b * p.table_stride + place.index]);
    if (page >= (uint32_t)p.num_pages) return;
    char *to_k = p.k_pages + bytes_to(p.sk, page, place.row), *to_v = p.v_pages + bytes_to(p.sv, page, place.row);
    uint8_t *to_ke = p.k_exp + bytes_to(p.ske, page, place.row), *to_ve = p.v_exp + bytes_to(p.sve, page, place.row);
    const auto put = [&](int i, Seg x) {
        const bool key = i < p.G;
        const uint32_t g = key ? i : i - p.G;
        char* at = (key ? to_k : to_v) + (uint64_t)g * (key ? p.sk.head : p.sv.head) + d * Piece<C, 8>::SIZE;
        if constexpr (!coded<C>) {
            if (d < p.D) *reinterpret_cast<Seg*>(at) = x;
        } else {
            const f32x8 y = sm::floats(x);
            // the largest of the block's bits: NaN and infinities are above every finite number
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(y[j]) & 0x7fffffffu);
            most = max(most, (uint32_t)__builtin_amdgcn_mov_dpp((int)most, 0xB1, 0xf, 0xf, true));     // quad: 1 0 3 2
            most = max(most, (uint32_t)__builtin_amdgcn_mov_dpp((int)most, 0x4E, 0xf, 0xf, true));     // quad: 2 3 0 1
            const uint32_t e = exponent_of<C>(__uint_as_float(most));
            if (d < p.D) {
                *reinterpret_cast<u32x2*>(at) = codes_of<C>(y, e);
                if (d % BLOCK == 0)
                    ((key ? to_ke : to_ve) + (uint64_t)g * (key ? p.ske.head : p.sve.head))[d / BLOCK] = (uint8_t)e;
            }
        }
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        const int i = lane / LANES + j * AT_ONCE;
        if (i <= last) put(i, ahead[j]);
    }
#pragma unroll 2
    for (int i = lane / LANES + AHEAD * AT_ONCE; i <= last; i += AT_ONCE) put(i, load(i));
}

// Rows of one sequence and head, keys and values, DP / 8 lanes a row and PG_READ_ROWS rows a lane.
template <class T, class C, int DP> __global__ __launch_bounds__(256) void paged_read(const PgParams p) {
    constexpr int LANES = DP / 8, ROWS = 256 / LANES;
    const int d = threadIdx.x % LANES * 8, g = blockIdx.x / p.blocks % p.G, b = blockIdx.x / p.blocks / p.G;
    const int length = min(max(p.lengths[b], 0), p.places);
    const int first = blockIdx.x % p.blocks * ROWS * PG_READ_ROWS + threadIdx.x / LANES;
    if (d >= p.D) return;
    typedef typename Piece<C, 8>::raw Raw;
    Raw k[PG_READ_ROWS], v[PG_READ_ROWS];
    uint32_t ke[PG_READ_ROWS], ve[PG_READ_ROWS];
#pragma unroll
    for (int i = 0; i < PG_READ_ROWS; ++i) {
        const int n = first + i * ROWS;
        k[i] = v[i] = Raw{};
        ke[i] = ve[i] = 127;
        if (n >= length || n >= p.N) continue;
        const Place place = place_of(p, n);
        const uint32_t page = p.tables[b * p.table_stride + place.index];
        if (page >= (uint32_t)p.num_pages) continue;
        k[i] = *reinterpret_cast<const Raw*>(p.k_pages + (uint64_t)g * p.sk.head + bytes_to(p.sk, page, place.row) +
                                             d * Piece<C, 8>::SIZE);
        v[i] = *reinterpret_cast<const Raw*>(p.v_pages + (uint64_t)g * p.sv.head + bytes_to(p.sv, page, place.row) +
                                             d * Piece<C, 8>::SIZE);
        if constexpr (coded<C>) {
            ke[i] = p.k_exp[(uint64_t)g * p.ske.head + bytes_to(p.ske, page, place.row) + d / BLOCK];
            ve[i] = p.v_exp[(uint64_t)g * p.sve.head + bytes_to(p.sve, page, place.row) + d / BLOCK];
        }
    }
#pragma unroll
    for (int i = 0; i < PG_READ_ROWS; ++i) {
        const int n = first + i * ROWS;
        if (n >= p.N) continue;
        typedef typename sm::Elem<T>::seg Seg;
        Seg x, y;
        if constexpr (coded<C>) {
            x = __builtin_convertvector(eight<C>(k[i], power_of(ke[i])), Seg);
            y = __builtin_convertvector(eight<C>(v[i], power_of(ve[i])), Seg);
        } else {
            x = k[i];
            y = v[i];
        }
        *reinterpret_cast<Seg*>((T*)p.out_k + b * p.sok.b + g * p.sok.h + n * p.sok.r + d) = x;
        *reinterpret_cast<Seg*>((T*)p.out_v + b * p.sov.b + g * p.sov.h + n * p.sov.r + d) = y;
    }
}

}  // namespace pg

int pg_write(int dtype, int held, const PgParams& p, hipStream_t st) {
    return pg::dispatch_types(dtype, held, [&](auto t, auto c) {
        return pg::by_width(p.D, [&](auto dp) {
            pg::paged_write<decltype(t), decltype(c), dp.value><<<dim3((unsigned)((p.T + 3) / 4)), 256, 0, st>>>(p);
            return (int)hipGetLastError(); }); });
}

int pg_read(int dtype, int held, const PgParams& p, hipStream_t st) {
    return pg::dispatch_types(dtype, held, [&](auto t, auto c) {
        return pg::by_width(p.D, [&](auto dp) {
            const dim3 grid((unsigned)((int64_t)p.B * p.G * p.blocks));
            pg::paged_read<decltype(t), decltype(c), dp.value><<<grid, 256, 0, st>>>(p);
            return (int)hipGetLastError(); }); });
}

}  // namespace qlka
