// Softmax attention for a few query rows per key head (a decoder's single tokens; with shared heads all their queries):
// bound by reading k and v once.
//
// A key row is read by DP / 8 lanes of a wave, 8 elements each, so a wave reads 512 / DP keys with one 16-byte load a
// lane (two for float) and keeps four such loads of k and four of v in flight, twice. Scores are formed with fp32
// multiply-adds and summed over a row's lanes by DPP; every group of lanes runs its own softmax over the keys that pass
// it, and the groups, then the waves, are joined at the end. The keys are split over workgroups until the GPU is full
// (softmax_combine joins the splits). A matrix tile would use one of its 32 rows here; from a few rows on it is faster
// all the same (softmax_api.hip). Near the diagonal a lane finds the bias of one key of the tile for every row, which
// the keys' groups then read from LDS. Measured: 16 x 12 heads, 8192 padded keys of 64 in bf16 (303 MB read) 52 us, 5.8
// TB/s; 8 x 12 heads, 197 keys 6.2 us.
#include "softmax_tile.h"

#include <limits>

namespace qlka {
namespace sm {

constexpr int STEP_WAVES = FWD_WAVES;

template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
// sum over groups of 4, 8 or 16 successive lanes, in every lane
template <int LANES> __device__ __forceinline__ float row_sum(float x) {
    x += dpp<0xB1>(x);                       // quad: 1 0 3 2
    x += dpp<0x4E>(x);                       // quad: 2 3 0 1
    if constexpr (LANES >= 8) x += dpp<0x141>(x);    // half row mirrored: the other quad
    if constexpr (LANES >= 16) x += dpp<0x140>(x);   // row mirrored: the other half
    return x;
}

template <class T, int DP, int R, bool BIAS>
__global__ __launch_bounds__(64 * STEP_WAVES) void softmax_step(const SmParams p) {
    constexpr int LANES = DP / 8, KEYS = 64 / LANES, U = 4, NW = STEP_WAVES, NT = 64 * NW;
    constexpr float LOW = -std::numeric_limits<float>::infinity();
    __shared__ float join_o[NW][R][DP], join_m[NW][R], join_s[NW][R];
    __shared__ float table[BIAS ? R : 1][QLKA_MAX_BUCKETS];
    __shared__ int border[BIAS ? QLKA_MAX_BUCKETS : 1];
    __shared__ float near_bias[BIAS ? NW : 1][R][64];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = lane / LANES, d = lane % LANES * 8;
    int w = blockIdx.x;                      // nothing is read twice, so any order does
    const int split_i = w % p.splits; w /= p.splits;
    const int kvh = w % p.G, b = w / p.G, share = p.H / p.G, rows = share * p.M;
    const T* k = (const T*)p.k + b * p.sk.b + kvh * p.sk.h;
    const T* v = (const T*)p.v + b * p.sv.b + kvh * p.sv.h;

    const int tiles = (p.seen + 63) / 64;
    const int t0 = (int)((int64_t)tiles * split_i / p.splits);
    const int t1 = (int)((int64_t)tiles * (split_i + 1) / p.splits);
    KeyBits<64> seen(p, b);
    struct Place { int t, u0; uint64_t bits; };        // a tile, the first key of U * KEYS of it, its keys
    const auto next = [&](Place at) {                  // the next U * KEYS keys of this wave with one to see
        at.u0 += U * KEYS;
        while (true) {
            while (at.u0 < 64) {
                if (at.bits >> at.u0 & (U * KEYS == 64 ? ~0ull : (1ull << U * KEYS % 64) - 1)) return at;
                at.u0 += U * KEYS;
            }
            at.t += NW;
            at.u0 = 0;
            if (at.t >= t1) return at;
            int t = at.t;
            at.bits = seen.find(t, t + 1);
        }
    };
    // the keys of one place are on their way while those of the place before are worked on
    struct Rows { typename Elem<T>::seg k[U], v[U]; };
    const auto fetch = [&](Place at) {
        Rows x;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int n = at.u0 + u * KEYS + group;
            x.k[u] = {};
            x.v[u] = {};
            if (at.bits >> n & 1) {
                x.k[u] = load_seg(k + (at.t * 64 + n) * p.sk.r, d, p.D);
                x.v[u] = load_seg(v + (at.t * 64 + n) * p.sv.r, d, p.D);
            }
        }
        return x;
    };
    Place at = next(Place{t0 + wave - NW, 64, 0});
    Rows rows_here;
    if (at.t < t1) rows_here = fetch(at);

    f32x8 q[R], o[R];
    float top[R], sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        o[r] = f32x8{};
        q[r] = f32x8{};
        top[r] = LOW;
        sum[r] = 0.f;
        if (r < rows) {
            const int head = kvh * share + r / p.M, m = r % p.M;
            q[r] = floats(load_seg((const T*)p.q + b * p.sq.b + head * p.sq.h + m * p.sq.r, d, p.D)) * p.q_sign;
            if constexpr (BIAS)
                for (int i = tid; i < (p.bk.n + 1) * (p.bk.both ? 2 : 1); i += NT)
                    table[r][i] = p.table[(int64_t)i * p.H + head] * UNIT;
        }
    }
    if constexpr (BIAS) {
        for (int i = tid; i < p.bk.n; i += NT) border[i] = p.bk.border[i];
        __syncthreads();
    }

    const float c1 = p.scale * UNIT;
    int near_tile = -1;
    while (at.t < t1) {
        const Place after = next(at);
        Rows rows_next;
        if (after.t < t1) rows_next = fetch(after);
        const int n0 = at.t * 64;
        int fb = -1;
        if constexpr (BIAS) {
            fb = far_bucket(p.bk, n0 - (p.M - 1) - p.start, n0 + 63 - p.start);
            if (fb < 0 && near_tile != at.t) {
                near_tile = at.t;
                wave_sync();
                for (int m = 0; m < p.M; ++m) {
                    const int bucket = bucket_of(border, p.bk.n, p.bk.both, n0 + lane - m - p.start);
                    for (int r = m; r < rows; r += p.M) near_bias[wave][r][lane] = table[r][bucket];
                }
                wave_sync();
            }
        }
        float x[R][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const f32x8 kf = floats(rows_here.k[u]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float a = q[r][0] * kf[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) a = __builtin_fmaf(q[r][i], kf[i], a);
                x[r][u] = row_sum<LANES>(a);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= rows) continue;
            const int seat = r % p.M + p.start;                        // the query's position
            float hi = LOW;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int n = at.u0 + u * KEYS + group;
                // scaled after the sum, as in the tiles: equal products stay equal however large the scale is
                x[r][u] = __builtin_fmaf(x[r][u], c1, BIAS ? fb >= 0 ? table[r][fb] : near_bias[wave][r][n] : 0.f);
                if (!(at.bits >> n & 1) || (p.causal && n0 + n > seat)) x[r][u] = LOW;
                hi = fmaxf(hi, x[r][u]);
            }
            const float to = fmaxf(top[r], hi), ref = to == LOW ? 0.f : to, f = exp_of(top[r] - ref);
            top[r] = to;
            sum[r] *= f;
            o[r] *= f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float e = exp_of(x[r][u] - ref);
                sum[r] += e;
                o[r] += floats(rows_here.v[u]) * e;
            }
        }
        at = after;
        rows_here = rows_next;
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int far = LANES; far < 64; far *= 2) {
            const float top2 = __shfl_xor(top[r], far), to = fmaxf(top[r], top2), ref = to == LOW ? 0.f : to;
            const float f = exp_of(top[r] - ref), f2 = exp_of(top2 - ref);
            sum[r] = sum[r] * f + __shfl_xor(sum[r], far) * f2;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[r][i] = o[r][i] * f + __shfl_xor(o[r][i], far) * f2;
            top[r] = to;
        }
        if (group == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) join_o[wave][r][d + i] = o[r][i];
            if (d == 0) {
                join_m[wave][r] = top[r];
                join_s[wave][r] = sum[r];
            }
        }
    }
    __syncthreads();
    const int64_t all = (int64_t)p.B * p.H * p.M;
    for (int e = tid; e < rows * DP; e += NT) {
        const int r = e / DP, c = e % DP, head = kvh * share + r / p.M, m = r % p.M;
        float to = LOW;
#pragma unroll
        for (int i = 0; i < NW; ++i) to = fmaxf(to, join_m[i][r]);
        const float ref = to == LOW ? 0.f : to;
        float s = 0.f, x = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const float f = exp_of(join_m[i][r] - ref);
            s += join_s[i][r] * f;
            x += join_o[i][r][c] * f;
        }
        const int64_t row = ((int64_t)b * p.H + head) * p.M + m;
        if (p.splits > 1) {
            p.part[(split_i * all + row) * DP + c] = x;
            if (c == 0) {
                p.part2[2 * (split_i * all + row)] = ref;
                p.part2[2 * (split_i * all + row) + 1] = s;
            }
            continue;
        }
        x = s == 0.f ? 0.f : x / s;
        if (c < p.D) {
            const int64_t at = b * p.so.b + head * p.so.h + m * p.so.r + c;
            ((T*)p.out)[at] = (T)x;
            if (p.out_full) p.out_full[row * p.D + c] = x;
        }
        if (c == 0) store_lse(p, row, ref, s);
    }
}

template <class T, int DP, int R> int launch_step(const SmParams& p, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)p.B * p.G * p.splits));
    if (p.table) softmax_step<T, DP, R, true><<<grid, 64 * STEP_WAVES, 0, st>>>(p);
    else softmax_step<T, DP, R, false><<<grid, 64 * STEP_WAVES, 0, st>>>(p);
    return (int)hipGetLastError();
}
template <class T, int DP> int pick_step(const SmParams& p, hipStream_t st) {
    const int rows = p.H / p.G * p.M;
    static_assert(STEP_MOST == 4, "the largest number of rows has an instance");
    return rows == 1   ? launch_step<T, DP, 1>(p, st)
           : rows == 2 ? launch_step<T, DP, 2>(p, st)
                       : launch_step<T, DP, 4>(p, st);
}
}  // namespace sm

int sm_step(int dtype, const SmParams& p, hipStream_t st) {
    return sm::dispatch(dtype, p.D, [&](auto t, auto dp) { return sm::pick_step<decltype(t), dp.value>(p, st); });
}

}  // namespace qlka
