// Softmax attention, forward: O = softmax(scale q k^T + bias) v over the visible keys, one pass over the keys with the
// running maximum and sum.
//
// A wave owns 32 queries and keeps S^T = k q^T tiles in registers (a lane holds one query's scores, softmax_tile.h), so
// the row maximum and sum need one exchange between the halves of the wave, and O^T += v^T P^T takes the probabilities
// from the registers they are in. A workgroup's waves share the tiles of k and v in LDS; the next tile's loads are
// issued before the current tile's products. The running maximum is moved only when it grows by more than 2^8, so
// that the output is hardly ever scaled; probabilities are then at most 2^8. Rounding them to bf16 for the product with
// bf16 values (not for fp32) costs what rounding the result does (error against float64 0.0023, 0.0017 with P whole;
// two parts of P: 1337 us for 965 at 12 x 16384 x 16384); the sum they are divided by is then that of the rounded ones.
// Where the table's gradient will be wanted (FINE) they are taken in three parts of 8 bits: that gradient is fp32 and a
// sum over rows of dS = P (dP - delta), in which an error of delta, the row sum of dO * O, does not average out. The
// smaller parts' products then gather in a sum of their own, as in Acc (12 x 8192 x 8192: error of the table's gradient
// 1.0e-6, 1.8e-6 without; 476 us, 250 with one part).
//
// Masked keys are read as zeros (what stands there may be anything) and their tiles, where none is left, are skipped.
// Bound by the matrix cores and by the scores' work between them (an exponential, a maximum and two multiply-adds a
// score), which other waves' products hide only in part. Measured: 12 x 16384 x 16384 of 64 with the bias, bf16, 977 to
// 1003 us, 835 TFLOP/s; 4 x 12 x 2048 x 8192, padded, 200 to 220 us; fp32, 2 x 12 x 301 x 3111, padded, 54 us with the
// joining of the splits; causal order, 12 x 8192 x 8192, 197 us. When a call has too few queries to fill the GPU, the
// keys are split: each split leaves its unscaled O with its maximum and sum, and softmax_combine joins them.
#include "softmax_tile.h"

#include <limits>

namespace qlka {
namespace sm {

constexpr float GROW = 4.f;          // 2^8 of the exponentials

// Three parts of P leave room for three waves a SIMD (of 64 elements) only if the compiler is held to it: 476 us for 524 at
// 12 x 8192 x 8192.
template <class T, int DP, int NW, bool BIAS, bool FINE>
__global__ __launch_bounds__(64 * NW, (FINE && DP <= 64 ? 3 : Shape<T, DP>::WAVES))
void softmax_fwd(const SmParams p) {
    constexpr int NP = Elem<T>::PARTS, BN = Shape<T, DP>::BN, NT = 64 * NW, ROWS = 32 * NW, NS = BN / 32, ND = DP / 32;
    typedef Pair<T, DP, BN, NW> PairT;
    constexpr int BUFFERS = PairT::BUFFERS;
    __shared__ typename PairT::Lds lds;
    __shared__ BiasLds table;
    __shared__ float near_bias[BUFFERS][BIAS ? ROWS + BN : 1];
    __shared__ __attribute__((aligned(16))) float mask_of[BUFFERS][BN];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const Work w = xcd_work(blockIdx.x, p.B * p.H, p.blocks * p.splits);
    const int block = w.block % p.blocks, split_i = w.block / p.blocks;
    const int head = w.pair % p.H, b = w.pair / p.H, kvh = head / (p.H / p.G);
    const int m0 = block * ROWS, mw = m0 + wave * 32, m = mw + col;
    const T* q = (const T*)p.q + b * p.sq.b + head * p.sq.h;
    const T* k = (const T*)p.k + b * p.sk.b + kvh * p.sk.h;
    const T* v = (const T*)p.v + b * p.sv.b + kvh * p.sv.h;

    const int tiles = (p.seen + BN - 1) / BN;
    int t0 = (int)((int64_t)tiles * split_i / p.splits), t1 = (int)((int64_t)tiles * (split_i + 1) / p.splits);
    if (p.causal) {
        const int last = min(m0 + ROWS, p.M) - 1 + p.start;          // the last key that a row here sees
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

    Frag<NP> qf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        typename Elem<T>::seg s = {};
        if (m < p.M) s = load_seg(q + m * p.sq.r, 16 * c + 8 * half, p.D);
        s = s * (T)p.q_sign;
        qf[c] = frag_of(s);
    }
    if constexpr (BIAS) {
        table.fill(p, head, tid, NT);
        __syncthreads();
    }

    const float c1 = p.scale * UNIT;
    Acc<NP> o[ND];
    float top = -std::numeric_limits<float>::infinity(), ref = 0.f, sum = 0.f;
    bool wide = false;                                 // a row here has a large ref

    while (coming) {
        const int n0 = t * BN;
        const uint64_t bits = coming;
        float far = 0.f;
        bool near = false;
        float *near_here = near_bias[buffer], *mask = mask_of[buffer];
        tile.arrive(lds, tid, [&] {
            if (bits != PairT::ALL) put_mask<BN>(mask, bits, tid);
            if constexpr (BIAS) {
                const int lo = n0 - (m0 + ROWS - 1) - p.start;
                const int fb = far_bucket(p.bk, lo, n0 + BN - 1 - m0 - p.start);
                near = fb < 0;
                if (near) {
                    for (int i = tid; i < ROWS + BN - 1; i += NT)
                        near_here[i] = table.value[bucket_of(table.border, p.bk.n, p.bk.both, lo + i)];
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

        f32x16 s[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            Acc<NP> a;
            a.start();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) a.add(kt.row(32 * i + col, 16 * c + 8 * half), qf[c]);
            __builtin_amdgcn_s_setprio(0);
            a.join();
            s[i] = a.main;
        }

        // scores are fma(s, mul, add) from here on
        float mul = c1, add = far;
        const bool edge = p.causal && n0 + BN - 1 > mw + p.start, all = bits == PairT::ALL;
        if (near || edge || !all) {
            const float* nb = &near_here[BIAS ? ROWS - 1 - wave * 32 - col + 4 * half : 0];
            if (BIAS && near) {
#pragma unroll
                for (int i = 0; i < NS; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[i][r] = __builtin_fmaf(s[i][r], c1, nb[32 * i + reg_row(r)]);
            } else {
#pragma unroll
                for (int i = 0; i < NS; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[i][r] = __builtin_fmaf(s[i][r], c1, far);
            }
            if (!all) {
#pragma unroll
                for (int i = 0; i < NS; ++i) s[i] = masked(s[i], mask, 32 * i + 4 * half);
            }
            if (edge) {
                const int lim = m + p.start - n0 - 4 * half;             // the last key seen
#pragma unroll
                for (int i = 0; i < NS; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (32 * i + reg_row(r) > lim) s[i][r] = -std::numeric_limits<float>::infinity();
            }
            mul = 1.f;
            add = 0.f;
        }
        float hi = s[0][0];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) hi = fmaxf(hi, s[i][r]);
        hi = fmaxf(hi, other_half(hi));
        hi = __builtin_fmaf(hi, mul, add);
        if (__any(hi > top + GROW)) {                                     // top -inf: any score at all
            const bool first = top == -std::numeric_limits<float>::infinity();
            const float was = ref;
            top = fmaxf(top, hi);
            ref = top == -std::numeric_limits<float>::infinity() ? 0.f : top;
            wide = __any(fabsf(ref) > WIDE);
            const float f = first ? 1.f : exp_of(was - ref);              // the first time there is nothing to scale
            sum *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d].main *= f;
        }
        const auto weigh = [&](auto wide) {
            if constexpr (wide) {
#pragma unroll
                for (int i = 0; i < NS; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[i][r] = __builtin_fmaf(s[i][r], mul, add) - ref;
                mul = 2.f;
                add = 0.f;
            } else {
                mul *= 2.f;
                add = 2.f * (add - ref);
            }
            float tile_sum = 0.f;                      // by tiles: thousands of terms one by one lose two digits more
            f32x16 small[ND];                          // FINE: the smaller parts apart, as in Acc
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                o[d].start();
                if constexpr (FINE) small[d] = f32x16{};
            }
#pragma unroll
            for (int i = 0; i < NS; ++i) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    f32x8 e = eight(s[i], c);
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = fexp2(__builtin_fmaf(e[j], mul, add));
                    const Frag<NP> pf = split<NP>(e);
                    if constexpr (NP == 1 && !FINE) {
                        sum = add_all(pf.p[0], sum);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) tile_sum += e[j];
                    }
                    Frag<NP> rest[2];
                    if constexpr (FINE) {
                        e -= floats(pf.p[0]);
                        rest[0] = split<NP>(e);
                        rest[1] = split<NP>(e - floats(rest[0].p[0]));
                    }
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const Frag<NP> vf = vt.column(32 * i + 16 * c, 32 * d, lane);
                        if constexpr (FINE) {
                            small[d] = mfma(vf.p[0], rest[1].p[0], small[d]);
                            small[d] = mfma(vf.p[0], rest[0].p[0], small[d]);
                        }
                        o[d].add(vf, pf);
                    }
                }
            }
            sum += tile_sum;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                o[d].join();
                if constexpr (FINE) o[d].main += small[d];
            }
        };
        if (__builtin_expect(wide, 0)) weigh(std::true_type());
        else weigh(std::false_type());
    }
    if (m >= p.M) return;
    sum += other_half(sum);
    const int64_t row = ((int64_t)b * p.H + head) * p.M + m;
    if (p.splits > 1) {
        const int64_t at = (int64_t)split_i * p.B * p.H * p.M + row;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4*>(p.part + at * DP + 32 * d + 8 * r + 4 * half) =
                    quad(o[d].main, r);
        if (half == 0) {
            p.part2[2 * at] = ref;
            p.part2[2 * at + 1] = sum;
        }
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = (T*)p.out + b * p.so.b + head * p.so.h + m * p.so.r;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const f32x4 x = quad(o[d].main, r) * inv;
            store4(out, 32 * d + 8 * r + 4 * half, p.D, x);
            if (p.out_full) store4(p.out_full + row * p.D, 32 * d + 8 * r + 4 * half, p.D, x);
        }
    if (half == 0) store_lse(p, row, ref, sum);
}

template <class T, int DP, int NW> int launch_fwd(const SmParams& p, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)p.B * p.H * p.blocks * p.splits));
    const bool fine = sizeof(T) == 2 && p.table && p.out_full && !p.table_kept;
    if (fine) softmax_fwd<T, DP, NW, true, sizeof(T) == 2><<<grid, 64 * NW, 0, st>>>(p);
    else if (p.table) softmax_fwd<T, DP, NW, true, false><<<grid, 64 * NW, 0, st>>>(p);
    else softmax_fwd<T, DP, NW, false, false><<<grid, 64 * NW, 0, st>>>(p);
    return (int)hipGetLastError();
}
// Joins the splits of a row, a wave a row: first a lane for each split's maximum and sum, then DP / 4 lanes for each of
// several splits at a time, four elements a lane. Both steps' loads are issued together: a row costs two memory
// latencies.
constexpr int COMBINE_ROWS = 4, MOST_SPLITS = 256;

template <class T, int DP>
__global__ __launch_bounds__(64 * COMBINE_ROWS) void softmax_combine(const SmParams p) {
    constexpr int LANES = DP / 4, AT_ONCE = 64 / LANES, LOOK = MOST_SPLITS / 64;
    constexpr float LOW = -std::numeric_limits<float>::infinity();
    __shared__ float weight[COMBINE_ROWS][MOST_SPLITS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t rows = (int64_t)p.B * p.H * p.M, row = (int64_t)blockIdx.x * COMBINE_ROWS + wave;
    if (row >= rows) return;
    float2 a[LOOK];
    float ref = LOW;
#pragma unroll
    for (int i = 0; i < LOOK; ++i) {
        const int s = lane + 64 * i;
        a[i] = float2{LOW, 0.f};
        if (s < p.splits) a[i] = *reinterpret_cast<const float2*>(p.part2 + 2 * (s * rows + row));
        if (a[i].y == 0.f) a[i].x = LOW;                                  // no key there
        ref = fmaxf(ref, a[i].x);
    }
#pragma unroll
    for (int far = 1; far < 64; far *= 2) ref = fmaxf(ref, __shfl_xor(ref, far));
    if (ref == LOW) ref = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < LOOK; ++i) {
        const float f = exp_of(a[i].x - ref);
        if (lane + 64 * i < p.splits) weight[wave][lane + 64 * i] = f;
        sum += a[i].y * f;
    }
    wave_sync();
#pragma unroll
    for (int far = 1; far < 64; far *= 2) sum += __shfl_xor(sum, far);
    const int d = lane % LANES * 4, first = lane / LANES;
    f32x4 x = {};
#pragma unroll 4
    for (int s = first; s < p.splits; s += AT_ONCE)
        x = x + *reinterpret_cast<const f32x4*>(p.part + (s * rows + row) * DP + d) * weight[wave][s];
#pragma unroll
    for (int far = LANES; far < 64; far *= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], far);
    x = x * (sum == 0.f ? 0.f : 1.f / sum);
    if (first) return;
    const int m = (int)(row % p.M), head = (int)(row / p.M % p.H), b = (int)(row / p.M / p.H);
    store4((T*)p.out + b * p.so.b + head * p.so.h + m * p.so.r, d, p.D, x);
    if (p.out_full) store4(p.out_full + row * p.D, d, p.D, x);
    if (d == 0) store_lse(p, row, ref, sum);
}

// The same for up to FEW_SPLITS splits, DP / 4 lanes a row (12 x 4096 rows of 2 splits: 23 us with a wave a row, 16 us
// so).
constexpr int FEW_SPLITS = 8;

template <class T, int DP>
__global__ __launch_bounds__(256) void softmax_combine_few(const SmParams p) {
    constexpr int LANES = DP / 4;
    constexpr float LOW = -std::numeric_limits<float>::infinity();
    const int64_t rows = (int64_t)p.B * p.H * p.M, row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int d = threadIdx.x % LANES * 4;
    if (row >= rows) return;
    float2 a[FEW_SPLITS];
    f32x4 y[FEW_SPLITS];
    float ref = LOW, sum = 0.f;
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) {
        a[s] = float2{LOW, 0.f};
        y[s] = f32x4{};
        if (s >= p.splits) continue;
        a[s] = *reinterpret_cast<const float2*>(p.part2 + 2 * (s * rows + row));
        y[s] = *reinterpret_cast<const f32x4*>(p.part + (s * rows + row) * DP + d);
    }
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) {
        if (a[s].y == 0.f) a[s].x = LOW;                                  // no key there
        ref = fmaxf(ref, a[s].x);
    }
    if (ref == LOW) ref = 0.f;
    f32x4 x = {};
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) {
        const float f = exp_of(a[s].x - ref);
        sum += a[s].y * f;
        x = x + y[s] * f;
    }
    x = x * (sum == 0.f ? 0.f : 1.f / sum);
    const int m = (int)(row % p.M), head = (int)(row / p.M % p.H), b = (int)(row / p.M / p.H);
    store4((T*)p.out + b * p.so.b + head * p.so.h + m * p.so.r, d, p.D, x);
    if (p.out_full) store4(p.out_full + row * p.D, d, p.D, x);
    if (d == 0) store_lse(p, row, ref, sum);
}

template <class T, int DP> int launch_combine(const SmParams& p, hipStream_t st) {
    const int64_t rows = (int64_t)p.B * p.H * p.M;
    if (p.splits <= FEW_SPLITS) {
        softmax_combine_few<T, DP><<<dim3((unsigned)((rows * (DP / 4) + 255) / 256)), 256, 0, st>>>(p);
        return (int)hipGetLastError();
    }
    softmax_combine<T, DP><<<dim3((unsigned)((rows + COMBINE_ROWS - 1) / COMBINE_ROWS)), 64 * COMBINE_ROWS, 0, st>>>(p);
    return (int)hipGetLastError();
}

}  // namespace sm

int sm_fwd(int dtype, const SmParams& p, hipStream_t st) {
    return sm::dispatch(dtype, p.D, [&](auto t, auto dp) {
        return sm::launch_fwd<decltype(t), dp.value, FWD_WAVES>(p, st); });
}

int sm_combine(int dtype, const SmParams& p, hipStream_t st) {
    return sm::dispatch(dtype, p.D, [&](auto t, auto dp) { return sm::launch_combine<decltype(t), dp.value>(p, st); });
}

}  // namespace qlka
