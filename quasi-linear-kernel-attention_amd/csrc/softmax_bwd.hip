// Softmax attention, backward. With P the probabilities of the forward (formed again from its row statistics),
//   dV = P^T dO,  dP = dO V^T,  delta = rowsum(dO * O),  dS = P * (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q,
// and the gradient of a bias bucket is the sum of dS over its scores.
//
// Two kernels, each forming P and dP for itself: softmax_dq goes over the keys for 32 queries a wave, softmax_dkv over
// the queries (of all the heads that share a key head) for 32 keys a wave. That is 7 products instead of the 5 of one
// pass, and no sum between workgroups: no atomics, results that do not change from run to run. Scores stay in registers
// as in the forward. Rounding P and dS to bf16 for the products with bf16 operands costs what rounding the results
// does. An error of delta is in all of a row's dS alike, so it is formed from O before that is rounded to bf16. For the
// table's gradient, which is fp32, dS is taken as it is, and O is that of P in three parts (softmax_fwd.hip, FINE).
// The waves wait for 34 to 50% of their cycles, for the next tile and for each other. Measured: 12 x 8192 x 8192 of 64
// with the table's gradient, bf16: softmax_dq 491 us (630 TFLOP/s), softmax_dkv 533 us (773); fp32, 32 x 4 heads of 600
// to 65: 41 and 42 us; bf16 of 128, 2 x 8 x 2048 x 2048: 257 us with the forward. Registers are short: at fp32 of 64
// elements and more, and at bf16 of 128, some values live in scratch memory.
#include "softmax_tile.h"

#include <limits>

namespace qlka {
namespace sm {

constexpr float HIGH = std::numeric_limits<float>::infinity();

// Twice a bias that a whole tile has, finite where it is above: a row past the last one adds -inf to it
__device__ __forceinline__ float far_twice(float x) { return fminf(2.f * x, std::numeric_limits<float>::max()); }

// delta, a wave 32 rows of a head, DP / 8 lanes a row; and whether one of the 32 has a large log sum
template <class T, int DP>
__global__ __launch_bounds__(256) void softmax_delta(const SmParams p) {
    constexpr int LANES = DP / 8;
    const int groups = (p.M + 31) / 32, lane = threadIdx.x & 63, d = lane % LANES * 8;
    const int64_t group = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (group >= (int64_t)p.B * p.H * groups) return;
    const int first = (int)(group % groups) * 32, head = (int)(group / groups % p.H), b = (int)(group / groups / p.H);
    const int64_t row0 = ((int64_t)b * p.H + head) * p.M;
    bool large = false;
#pragma unroll
    for (int i = 0; i < 32; i += 64 / LANES) {
        const int m = first + i + lane / LANES;
        float x = 0.f;
        if (m < p.M) {
            const T* out = (const T*)p.out + b * p.so.b + head * p.so.h + m * p.so.r;
            const auto g = load_seg((const T*)p.g_out + b * p.sg.b + head * p.sg.h + m * p.sg.r, d, p.D);
            const f32x8 o = p.out_full ? load_seg(p.out_full + (row0 + m) * p.D, d, p.D)
                                       : floats(load_seg(out, d, p.D));
            large |= large_lse(p.lse_unit * p.lse[row0 + m]);
#pragma unroll
            for (int j = 0; j < 8; ++j) x = __builtin_fmaf((float)g[j], o[j], x);
        }
#pragma unroll
        for (int far = 1; far < LANES; far *= 2) x += __shfl_xor(x, far);
        if (m < p.M && d == 0) p.delta[row0 + m] = x;
    }
    large = __any(large);
    if (lane == 0) p.large[group] = large;
}

// y of a lane added to x where both lanes' buckets are the same: one step of a segmented scan over a wave (CTRL: a DPP
// shift within 16 lanes, or the broadcast of a row's last lane to the next)
template <int CTRL, int ROWS> __device__ __forceinline__ void scan_step(float& x, int bucket) {
    const int c = __builtin_amdgcn_update_dpp(-1, bucket, CTRL, ROWS, 0xf, false);
    const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xf, false);
    if (c == bucket) x += __int_as_float(y);
}

// Adds a wave's 32 x 32 scores' gradients to the buckets of their distances. A lane holds one query (lane % 32) and 16
// keys; for each register the values of 32 queries are turned in the wave until lane t holds the diagonal (key - query)
// = t or t - 32, so a diagonal's sum gathers in one lane; lanes of one bucket, which are neighbours, are then summed by
// a segmented scan. buckets: those of the distances from the tile's first key and first query less 32 on. acc: this
// wave's own, in LDS.
__device__ __forceinline__ void add_band(f32x16 ds, const uint8_t* buckets, float* acc, int lane) {
    const int t = lane & 31, half = lane >> 5, from = 4 * (4 * half - t);
    float pos = 0.f, neg = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int x = __builtin_amdgcn_ds_bpermute(((from + 4 * reg_row(r)) & 124) | (lane & 32) << 2,
                                                   __float_as_int(ds[r]));
        const bool after = t <= reg_row(r) + 4 * half;
        pos += after ? __int_as_float(x) : 0.f;
        neg += after ? 0.f : __int_as_float(x);
    }
    pos += other_half(pos);
    neg += other_half(neg);
    float x = half ? pos : neg;
    const int bucket = buckets[lane];
    scan_step<0x111, 0xf>(x, bucket);        // row_shr 1, 2, 4, 8
    scan_step<0x112, 0xf>(x, bucket);
    scan_step<0x114, 0xf>(x, bucket);
    scan_step<0x118, 0xf>(x, bucket);
    scan_step<0x142, 0xa>(x, bucket);        // row_bcast 15 into rows 1 and 3
    scan_step<0x143, 0xc>(x, bucket);        // row_bcast 31 into rows 2 and 3
    const int after = __shfl_down(bucket, 1);
    if (lane == 63 || after != bucket) acc[bucket] += x;
    wave_sync();
}

// f(first half, halves together): both halves of a tile together where registers reach for it, else one after the
// other, and the second only where it has something to do
template <int NP, int NS, class F> __device__ __forceinline__ void by_halves(bool one, F f) {
    if constexpr (NP == 1) {
        f(0, std::integral_constant<int, NS>());
    } else {
#pragma unroll 1
        for (int i = 0; i < (one ? 1 : NS); ++i) f(i, std::integral_constant<int, 1>());
    }
}

// Large log sums are taken off in two steps, after the score is rounded. With bf16 operands in a loop of its own,
// f(true): a test between a tile's products and its exponentials keeps those apart (8% of softmax_dkv's time at 4 x 12
// x 1024 x 4096 of 64). With fp32 the test is in the loop, by tiles, f(false): there it costs 1% at 32 x 4 heads of 600
// to 65, and what a second loop needs before it starts, and its registers, 5%.
template <int NP, class F> __device__ __forceinline__ void by_size(bool large, F f) {
    if constexpr (NP == 1) {
        if (__builtin_expect(large, 0)) return f(std::true_type());
    }
    f(std::false_type());
}

template <class T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW, (Shape<T, DP>::WAVES)) void softmax_dq(const SmParams p) {
    constexpr int NP = Elem<T>::PARTS, BN = Shape<T, DP>::BN, NT = 64 * NW, ROWS = 32 * NW, NS = BN / 32, ND = DP / 32;
    typedef Pair<T, DP, BN, NW> PairT;
    constexpr int BUFFERS = PairT::BUFFERS;
    __shared__ typename PairT::Lds lds;
    __shared__ BiasLds table;
    __shared__ __attribute__((aligned(16))) float mask_of[BUFFERS][BN];
    __shared__ float near_bias[BUFFERS][BIAS ? ROWS + BN : 1], sums[BIAS ? NW : 1][QLKA_MAX_BUCKETS];
    __shared__ uint8_t near_bucket[BUFFERS][BIAS ? ROWS + BN : 1];     // from the distance before near_bias's first on

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const Work w = xcd_work(blockIdx.x, p.B * p.H, p.blocks * p.splits);
    const int block = w.block % p.blocks, split_i = w.block / p.blocks;
    const int head = w.pair % p.H, b = w.pair / p.H, kvh = head / (p.H / p.G);
    const int m0 = block * ROWS, mw = m0 + wave * 32, m = mw + col;
    const T* k = (const T*)p.k + b * p.sk.b + kvh * p.sk.h;
    const T* v = (const T*)p.v + b * p.sv.b + kvh * p.sv.h;
    const int64_t row = ((int64_t)b * p.H + head) * p.M + m;

    const int tiles = (p.seen + BN - 1) / BN;
    int t0 = (int)((int64_t)tiles * split_i / p.splits), t1 = (int)((int64_t)tiles * (split_i + 1) / p.splits);
    if (p.causal) {
        const int last = min(m0 + ROWS, p.M) - 1 + p.start;
        t1 = min(t1, last < 0 ? 0 : last / BN + 1);
    }
    KeyBits<BN> seen(p, b);
    PairT tile(lds, p.sk.r, p.sv.r, p.D, tid);
    const auto fetch = [&](int t, uint64_t bits, int buffer) {
        tile.fetch(lds, buffer, k + (int64_t)t * BN * p.sk.r, v + (int64_t)t * BN * p.sv.r, bits, p.D, tid);
    };
    int t = t0, buffer = 0;
    uint64_t coming = seen.find(t, t1);                // the keys of tile t, which is on its way
    if (coming) fetch(t, coming, 0);

    Frag<NP> qf[DP / 16], gf[DP / 16];
    float delta = 0.f;
    // dP is formed as -((-dO) V^T) for every other query: the matrix instruction's sums are a little low
    // (softmax_tile.h), and a bucket adds up millions of dS (12 x 8192 x 8192, four inputs: error of the table's
    // gradient 2 to 12% less)
    const float turn = BIAS && (col & 1) ? -1.f : 1.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        const int d = 16 * c + 8 * half;
        typename Elem<T>::seg s = {}, g = {};
        f32x8 o = {};
        if (m < p.M) {
            s = load_seg((const T*)p.q + b * p.sq.b + head * p.sq.h + m * p.sq.r, d, p.D);
            g = load_seg((const T*)p.g_out + b * p.sg.b + head * p.sg.h + m * p.sg.r, d, p.D);
            o = p.out_full ? load_seg(p.out_full + row * p.D, d, p.D)
                           : floats(load_seg((const T*)p.out + b * p.so.b + head * p.so.h + m * p.so.r, d, p.D));
        }
        s = s * (T)p.q_sign;
        qf[c] = frag_of(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) delta = __builtin_fmaf((float)g[i], o[i], delta);
        g = g * (T)turn;
        gf[c] = frag_of(g);
    }
    delta += other_half(delta);
    const float lse = m < p.M ? p.lse_unit * p.lse[row] : HIGH;
    const bool large = __any(large_lse(lse));
    if (split_i == 0) {                                // softmax_dkv reads them
        if (m < p.M && half == 0) p.delta[row] = delta;
        if (mw < p.M && lane == 0) p.large[((int64_t)b * p.H + head) * ((p.M + 31) / 32) + mw / 32] = large;
    }
    const int buckets = (p.bk.n + 1) * (p.bk.both ? 2 : 1);
    float left = 0.f, right = 0.f;                     // this lane's sums far below and far above the diagonal
    const bool to_table = BIAS && p.part_table;
    if constexpr (BIAS) {
        table.fill(p, head, tid, NT);
        for (int i = lane; i < buckets; i += 64) sums[wave][i] = 0.f;
    }
    bool any_large = false;
    if constexpr (NP == 1) any_large = __syncthreads_or(large);
    else if constexpr (BIAS) __syncthreads();

    const float c1 = p.scale * UNIT;
    Acc<NP> dq[ND];

    const auto go = [&](auto all_wide) {
        const bool wide = NP == 3 ? large : all_wide;
        while (coming) {
            const int n0 = t * BN;
            const uint64_t bits = coming;
            float far = 0.f;
            int fb = -1;
            float *near_here = near_bias[buffer], *mask = mask_of[buffer];
            uint8_t* bucket_here = near_bucket[buffer];
            tile.arrive(lds, tid, [&] {
                if (bits != PairT::ALL) put_mask<BN>(mask, bits, tid);
                if constexpr (BIAS) {
                    const int lo = n0 - (m0 + ROWS - 1) - p.start;
                    fb = far_bucket(p.bk, lo, n0 + BN - 1 - m0 - p.start);
                    if (fb < 0) {
                        for (int i = tid; i < ROWS + BN; i += NT) {
                            const int bucket = bucket_of(table.border, p.bk.n, p.bk.both, lo + i - 1);
                            bucket_here[i] = (uint8_t)bucket;
                            if (i) near_here[i - 1] = table.value[bucket];
                        }
                    } else {
                        far = table.value[fb];
                    }
                }
            });
            const auto& kt = lds.a[buffer];
            const auto& vt = lds.b[buffer];
            buffer ^= BUFFERS - 1;
            coming = seen.find(++t, t1);
            if (coming) fetch(t, coming, buffer);
            if (mw >= p.M || (p.causal && n0 > mw + 31 + p.start)) continue;

            const bool edge = p.causal && n0 + BN - 1 > mw + p.start;
            const int lim = m + p.start - n0 - 4 * half;                     // at an edge, the last key seen
            const float* nb = &near_here[BIAS ? ROWS - 1 - wave * 32 - col + 4 * half : 0];
            const float off = wide ? 0.f : lse, add = far_twice(far - off);
            // `count` halves of the tile together: the products of one are under way while the other's scores are
            // worked on
            const auto halves = [&](auto first, auto count) {
                f32x16 s[count], dp[count];
#pragma unroll
                for (int i = 0; i < count; ++i) {
                    Acc<NP> a;
                    a.start();
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c) a.add(kt.row(32 * (first + i) + col, 16 * c + 8 * half), qf[c]);
                    a.join();
                    s[i] = a.main;
                }
#pragma unroll
                for (int i = 0; i < count; ++i) {
                    Acc<NP> a;
                    a.start();
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c) a.add(vt.row(32 * (first + i) + col, 16 * c + 8 * half), gf[c]);
                    a.join();
                    dp[i] = a.main;
                }
#pragma unroll
                for (int i = 0; i < count; ++i) {
                    // to twice the scores less the row's log sum
                    if (wide || (BIAS && fb < 0)) {
                        if (BIAS && fb < 0) {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                s[i][r] = __builtin_fmaf(s[i][r], c1, nb[32 * (first + i) + reg_row(r)] - off);
                        } else {
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[i][r] = __builtin_fmaf(s[i][r], c1, far);
                        }
                        if (wide) {
                            const float low = m < p.M && p.lse_low ? p.lse_low[row] : 0.f;
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[i][r] = at_most_0((s[i][r] - lse) - low);
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[i][r] += s[i][r];
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[i][r] = __builtin_fmaf(s[i][r], 2.f * c1, add);
                    }
                    if (bits != PairT::ALL) s[i] = masked(s[i], mask, 32 * (first + i) + 4 * half);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[i][r] = fexp2(s[i][r]) * __builtin_fmaf(dp[i][r], turn, -delta);
                    if (edge) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (32 * (first + i) + reg_row(r) > lim) s[i][r] = 0.f;
                    }
                    if (to_table) {
                        if (fb < 0) {
                            // a half's first key and the wave's first query, less 32, after lo - 1
                            const int from = 32 * (first + i) + ROWS - 32 - 32 * wave;
                            if ((uint32_t)(bits >> (32 * (first + i))))
                                add_band(s[i], bucket_here + from, sums[wave], lane);
                        } else {
                            float a = 0.f;
#pragma unroll
                            for (int r = 0; r < 16; ++r) a += s[i][r];
                            if (fb == p.bk.n) left += a; else right += a;
                        }
                    }
                    Frag<NP> df[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) df[c] = split<NP>(eight(s[i], c));
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        dq[d].start();
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            dq[d].add(kt.column(32 * (first + i) + 16 * c, 32 * d, lane), df[c]);
                        dq[d].join();
                    }
                }
            };
            by_halves<NP, NS>(NS == 1 || !(bits >> 32), halves);
        }
    };
    by_size<NP>(any_large, go);
    if (to_table) {
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
            left += __shfl_xor(left, x);
            right += __shfl_xor(right, x);
        }
        if (lane == 0) {
            sums[wave][p.bk.n] += left;
            sums[wave][p.bk.both ? 2 * p.bk.n + 1 : 0] += right;
        }
        __syncthreads();
        const int64_t count = (int64_t)p.B * p.splits * p.blocks;
        float* part = p.part_table + (head * count + ((int64_t)b * p.splits + split_i) * p.blocks + block) * buckets;
        for (int i = tid; i < buckets; i += NT) {
            float a = 0.f;
            for (int j = 0; j < NW; ++j) a += sums[j][i];
            part[i] = a;
        }
    }
    if (m >= p.M || !p.g_q) return;
    const float f = p.scale * p.q_sign;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = 32 * d + 8 * r + 4 * half;
            const f32x4 x = quad(dq[d].main, r);
            if (p.splits > 1)
                *reinterpret_cast<f32x4*>(p.part + ((int64_t)split_i * p.B * p.H * p.M + row) * DP + at) = x;
            else
                store4((T*)p.g_q + b * p.sgq.b + head * p.sgq.h + m * p.sgq.r, at, p.D, x * f);
        }
}

template <class T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW, (Shape<T, DP>::WAVES)) void softmax_dkv(const SmParams p) {
    constexpr int NP = Elem<T>::PARTS, BM = Shape<T, DP>::BN, NT = 64 * NW, KEYS = 32 * NW, NS = BM / 32, ND = DP / 32;
    typedef Pair<T, DP, BM, NW> PairT;
    constexpr int BUFFERS = PairT::BUFFERS;
    __shared__ typename PairT::Lds lds;
    __shared__ __attribute__((aligned(16))) float lse_of[BUFFERS][BM], delta_of[BUFFERS][BM], large_of[BUFFERS][2][BM];
    __shared__ int wide_of;                            // (fp32, one buffer) a row of the tile has a large log sum
    __shared__ BiasLds table;
    __shared__ float near_bias[BUFFERS][BIAS ? KEYS + BM : 1];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const Work w = xcd_work(blockIdx.x, p.B * p.G, p.blocks * p.splits);
    const int block = w.block % p.blocks, split_i = w.block / p.blocks;
    const int kvh = w.pair % p.G, b = w.pair / p.G, share = p.H / p.G;
    const int n0 = block * KEYS, nw = n0 + wave * 32, n = nw + col;
    const bool shown = n < p.seen && (!p.keep || p.keep[b * p.keep_stride + n]);
    const bool idle = !__any(shown);

    // the tiles of queries of all heads that share these keys, one after the other
    const int tiles = (p.M + BM - 1) / BM;
    const int64_t work = (int64_t)tiles * share;
    const int t1 = (int)(work * (split_i + 1) / p.splits);
    const auto next = [&](int t) {                     // the first tile from t on with a query that sees a key here
        if (p.causal)
            while (t < t1 && t % tiles * BM + BM - 1 + p.start < n0) ++t;
        return t;
    };
    PairT tile(lds, p.sq.r, p.sg.r, p.D, tid);
    float ls = HIGH, des = 0.f;
    const auto fetch = [&](int t, int buffer) {
        const int head = kvh * share + t / tiles, m0 = t % tiles * BM, left = p.M - m0;
        const uint64_t bits = left >= BM ? PairT::ALL : (1ull << left) - 1;
        tile.fetch(lds, buffer, (const T*)p.q + b * p.sq.b + head * p.sq.h + m0 * p.sq.r,
                   (const T*)p.g_out + b * p.sg.b + head * p.sg.h + m0 * p.sg.r, bits, p.D, tid);
        ls = HIGH;
        des = 0.f;
        if (tid < BM && tid < left) {
            const int64_t row = ((int64_t)b * p.H + head) * p.M + m0 + tid;
            ls = p.lse[row];
            des = p.delta[row];
        }
    };
    int t = next((int)(work * split_i / p.splits)), buffer = 0;
    if (t < t1) fetch(t, 0);
    Frag<NP> kf[DP / 16], vf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        typename Elem<T>::seg s = {}, x = {};
        if (shown) {
            s = load_seg((const T*)p.k + b * p.sk.b + kvh * p.sk.h + n * p.sk.r, 16 * c + 8 * half, p.D);
            x = load_seg((const T*)p.v + b * p.sv.b + kvh * p.sv.h + n * p.sv.r, 16 * c + 8 * half, p.D);
        }
        s = s * (T)p.q_sign;
        kf[c] = frag_of(s);
        vf[c] = frag_of(x);
    }

    const int groups = share * ((p.M + 31) / 32);      // of 32 rows of the heads that share these keys
    bool any_large = false;
    if constexpr (NP == 1) {
        for (int i = tid; i < groups; i += NT) any_large |= p.large[((int64_t)b * p.G + kvh) * groups + i] != 0;
        any_large = __syncthreads_or(any_large);
    }

    const float c1 = p.scale * UNIT;
    Acc<NP> dk[ND], dv[ND];
    const float per_c1 = 1.f / c1;
    int filled = -1;                                   // the head whose bias stands in LDS

    const auto go = [&](auto all_wide) {
        while (t < t1) {
            const int m0 = t % tiles * BM, head = kvh * share + t / tiles;
            float far = 0.f;
            bool near = false;
            float *near_here = near_bias[buffer], *lse = lse_of[buffer], *delta = delta_of[buffer];
            float (*two)[BM] = large_of[buffer];
            if (BIAS && head != filled) {
                __syncthreads();
                table.fill(p, head, tid, NT);
                filled = head;
                __syncthreads();
            }
            tile.arrive(lds, tid, [&] {
                ls *= p.lse_unit;                          // (not where it is loaded, which would wait for it)
                const bool wide = NP == 3 ? __any(large_lse(ls)) : all_wide;      // all rows are in the first wave
                if (NP == 3 && tid == 0) wide_of = wide;
                if (tid < BM) {
                    lse[tid] = wide ? 0.f : -ls * per_c1;
                    delta[tid] = -des;
                    if (wide) {
                        two[0][tid] = ls;
                        const int64_t row = ((int64_t)b * p.H + head) * p.M + m0 + tid;
                        two[1][tid] = p.lse_low && m0 + tid < p.M ? p.lse_low[row] : 0.f;
                    }
                }
                if constexpr (BIAS) {
                    const int lo = n0 - (m0 + BM - 1) - p.start;
                    const int fb = far_bucket(p.bk, lo, n0 + KEYS - 1 - m0 - p.start);
                    near = fb < 0;
                    if (near) {
                        for (int i = tid; i < KEYS + BM - 1; i += NT)
                            near_here[i] = table.value[bucket_of(table.border, p.bk.n, p.bk.both, lo + i)];
                    } else {
                        far = table.value[fb];
                    }
                }
            });
            const auto& qt = lds.a[buffer];
            const auto& gt = lds.b[buffer];
            buffer ^= BUFFERS - 1;
            t = next(t + 1);
            if (t < t1) fetch(t, buffer);
            if (idle || (p.causal && m0 + BM - 1 + p.start < nw)) continue;

            const bool edge = p.causal && m0 + p.start < nw + 31;
            const int lim = edge ? n - p.start - m0 - 4 * half : -1;         // the first query that sees the key
            const float* nb = &near_here[BIAS ? wave * 32 + col + BM - 1 - 4 * half : 0];
            const float add = far_twice(far);
            const auto halves = [&](auto first, auto count) {
                // scores less the row's log sum (in units of the scores; a large one later), and dP less delta
                f32x16 s[count], dp[count];
#pragma unroll
                for (int i = 0; i < count; ++i) {
                    Acc<NP> a(rows_of(lse, 32 * (first + i) + 4 * half));
                    a.start();
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c)
                        a.add_turned(qt.row(32 * (first + i) + col, 16 * c + 8 * half), kf[c]);
                    a.join();
                    s[i] = a.main;
                }
#pragma unroll
                for (int i = 0; i < count; ++i) {
                    Acc<NP> a(rows_of(delta, 32 * (first + i) + 4 * half));
                    a.start();
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c) a.add(gt.row(32 * (first + i) + col, 16 * c + 8 * half), vf[c]);
                    a.join();
                    dp[i] = a.main;
                }
                const bool wide = NP == 3 ? __builtin_amdgcn_readfirstlane(wide_of) : all_wide;
#pragma unroll
                for (int i = 0; i < count; ++i) {
                    // to twice the scores less the row's log sum
                    if (wide || (BIAS && near)) {
                        if (BIAS && near) {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                s[i][r] = __builtin_fmaf(s[i][r], c1, nb[-32 * (first + i) - reg_row(r)]);
                        } else {
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[i][r] = __builtin_fmaf(s[i][r], c1, far);
                        }
                        if (wide) {
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const int row = 32 * (first + i) + 4 * half + reg_row(r);
                                s[i][r] = at_most_0((s[i][r] - two[0][row]) - two[1][row]);
                            }
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[i][r] += s[i][r];
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[i][r] = __builtin_fmaf(s[i][r], 2.f * c1, add);
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        s[i][r] = fexp2(s[i][r]);
                        dp[i][r] *= s[i][r];
                    }
                    if (edge) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (32 * (first + i) + reg_row(r) < lim) s[i][r] = dp[i][r] = 0.f;
                    }
                    Frag<NP> f[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) f[c] = split<NP>(eight(s[i], c));
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        dv[d].start();
#pragma unroll
                        for (int c = 0; c < 2; ++c) dv[d].add(gt.column(32 * (first + i) + 16 * c, 32 * d, lane), f[c]);
                        dv[d].join();
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) f[c] = split<NP>(eight(dp[i], c));
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        dk[d].start();
#pragma unroll
                        for (int c = 0; c < 2; ++c) dk[d].add(qt.column(32 * (first + i) + 16 * c, 32 * d, lane), f[c]);
                        dk[d].join();
                    }
                }
            };
            by_halves<NP, NS>(m0 + 32 >= p.M, halves);
        }
    };
    by_size<NP>(any_large, go);
    if (n >= p.N) return;
    const float f = p.scale * p.q_sign;
    const int64_t row = ((int64_t)b * p.G + kvh) * p.N + n, all = (int64_t)p.B * p.G * p.N;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = 32 * d + 8 * r + 4 * half;
            f32x4 x = quad(dk[d].main, r), y = quad(dv[d].main, r);
            if (!shown) x = y = f32x4{};                    // what was computed for a key that nothing sees
            if (p.splits > 1) {
                *reinterpret_cast<f32x4*>(p.part + (split_i * all + row) * DP + at) = x;
                *reinterpret_cast<f32x4*>(p.part2 + (split_i * all + row) * DP + at) = y;
            } else {
                store4((T*)p.g_k + b * p.sgk.b + kvh * p.sgk.h + n * p.sgk.r, at, p.D, x * f);
                store4((T*)p.g_v + b * p.sgv.b + kvh * p.sgv.h + n * p.sgv.r, at, p.D, y);
            }
        }
}

// Sum of the splits' partial rows: DP / 4 lanes a row.
template <class T, int DP>
__global__ __launch_bounds__(256) void softmax_sum(const float* part, T* out, SmStrides so, float scale,
                                                   int splits, int64_t rows, int heads, int len, int D) {
    constexpr int LANES = DP / 4;
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int d = threadIdx.x % LANES * 4;
    if (row >= rows) return;
    f32x4 x = {};
    for (int s = 0; s < splits; ++s) x = x + *reinterpret_cast<const f32x4*>(part + (s * rows + row) * DP + d);
    const int i = (int)(row % len), h = (int)(row / len % heads), b = (int)(row / len / heads);
    store4(out + b * so.b + h * so.h + i * so.r, d, D, x * scale);
}

// One workgroup for each (head, bucket).
__global__ __launch_bounds__(256) void softmax_table(const float* part, float* g_table, int H, int count, int buckets) {
    __shared__ float s[4];
    const int h = blockIdx.x, k = blockIdx.y;
    float x = 0.f;
    for (int i = threadIdx.x; i < count; i += 256) x += part[((int64_t)h * count + i) * buckets + k];
#pragma unroll
    for (int far = 1; far < 64; far *= 2) x += __shfl_xor(x, far);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) g_table[(int64_t)k * H + h] = s[0] + s[1] + s[2] + s[3];
}

template <class T, int DP> int run_delta(const SmParams& p, hipStream_t st) {
    const int64_t groups = (int64_t)p.B * p.H * ((p.M + 31) / 32);
    softmax_delta<T, DP><<<dim3((unsigned)((groups + 3) / 4)), 256, 0, st>>>(p);
    return (int)hipGetLastError();
}
template <class T, int DP, int NW> int run_dq(const SmParams& p, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)p.B * p.H * p.blocks * p.splits));
    if (p.table) softmax_dq<T, DP, NW, true><<<grid, 64 * NW, 0, st>>>(p);
    else softmax_dq<T, DP, NW, false><<<grid, 64 * NW, 0, st>>>(p);
    return (int)hipGetLastError();
}
template <class T, int DP, int NW> int run_dkv(const SmParams& p, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)p.B * p.G * p.blocks * p.splits));
    if (p.table) softmax_dkv<T, DP, NW, true><<<grid, 64 * NW, 0, st>>>(p);
    else softmax_dkv<T, DP, NW, false><<<grid, 64 * NW, 0, st>>>(p);
    return (int)hipGetLastError();
}
template <class T, int DP> int run_sum(const float* part, void* out, SmStrides so, float scale, int splits, int B,
                                       int heads, int len, int D, hipStream_t st) {
    const int64_t rows = (int64_t)B * heads * len, threads = rows * (DP / 4);
    softmax_sum<T, DP><<<dim3((unsigned)((threads + 255) / 256)), 256, 0, st>>>(part, (T*)out, so, scale, splits, rows,
                                                                               heads, len, D);
    return (int)hipGetLastError();
}

}  // namespace sm

int sm_delta(int dtype, const SmParams& p, hipStream_t st) {
    return sm::dispatch(dtype, p.D, [&](auto t, auto dp) { return sm::run_delta<decltype(t), dp.value>(p, st); });
}

int sm_dq(int dtype, const SmParams& p, int waves, hipStream_t st) {
    return sm::dispatch(dtype, p.D, [&](auto t, auto dp) {
        return waves == 2 ? sm::run_dq<decltype(t), dp.value, 2>(p, st)
                          : sm::run_dq<decltype(t), dp.value, 4>(p, st); });
}

int sm_dkv(int dtype, const SmParams& p, int waves, hipStream_t st) {
    return sm::dispatch(dtype, p.D, [&](auto t, auto dp) {
        return waves == 2 ? sm::run_dkv<decltype(t), dp.value, 2>(p, st)
                          : sm::run_dkv<decltype(t), dp.value, 4>(p, st); });
}

int sm_sum_parts(int dtype, const float* part, void* out, SmStrides so, float scale, int splits, int B, int heads,
                 int len, int D, hipStream_t st) {
    return sm::dispatch(dtype, D, [&](auto t, auto dp) {
        return sm::run_sum<decltype(t), dp.value>(part, out, so, scale, splits, B, heads, len, D, st); });
}

int sm_sum_table(const float* part, float* g_table, int H, int count, int buckets, hipStream_t st) {
    sm::softmax_table<<<dim3((unsigned)H, (unsigned)buckets), 256, 0, st>>>(part, g_table, H, count, buckets);
    return (int)hipGetLastError();
}

}  // namespace qlka
