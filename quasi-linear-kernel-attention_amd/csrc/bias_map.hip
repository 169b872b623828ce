// The relative position bias by buckets as a map: out[h, m, n] = table[bucket(n - (m + start))][h], and its gradient,
// the sums of the map's gradient over each bucket. Both are bound by the map's bytes. The map is constant along its
// diagonals: a workgroup finds the bucket of each diagonal of its tile once, and writes rows as windows of one array in
// LDS.
#include "softmax_tile.h"

namespace qlka {
namespace sm {

constexpr int MAP_ROWS = 64, MAP_COLS = 1024, MAP_T = 256;
constexpr int SUM_ROWS = 16, SUM_COLS = 1024;         // of the gradient

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // rows start at any float

__global__ __launch_bounds__(MAP_T) void map_fwd(const float* table, const SmBuckets bk, float* out, int H, int M,
                                                 int N, int start) {
    __shared__ float along[MAP_ROWS + MAP_COLS];
    __shared__ int border[QLKA_MAX_BUCKETS];
    const int n0 = blockIdx.x * MAP_COLS, m0 = blockIdx.y * MAP_ROWS, h = blockIdx.z, tid = threadIdx.x;
    const int rows = min(MAP_ROWS, M - m0), cols = min(MAP_COLS, N - n0);
    for (int i = tid; i < bk.n; i += MAP_T) border[i] = bk.border[i];
    __syncthreads();
    const int lo = n0 - (m0 + rows - 1) - start;
    for (int i = tid; i < rows + cols - 1; i += MAP_T)
        along[i] = table[(int64_t)bucket_of(border, bk.n, bk.both, lo + i) * H + h];
    __syncthreads();
    float* to = out + ((int64_t)h * M + m0) * N + n0;
    const int c = 4 * tid;
    for (int r = 0; r < rows; ++r, to += N) {
        const float* a = &along[rows - 1 - r + c];
        if (c + 3 < cols) {
            *reinterpret_cast<f32x4u*>(to + c) = f32x4u{a[0], a[1], a[2], a[3]};
        } else {
            for (int i = 0; c + i < cols; ++i) to[c + i] = a[i];
        }
    }
}

// A workgroup sums its rows along 1024 diagonals. A thread takes 4 x 4 values at a time, four loads of four, and goes
// down and to the right by four, so that it stays on the same seven diagonals; then the diagonals of a bucket are
// summed, at once where a wave's lie in one. Measured for 12 x 1777 x 2049 (175 MB): 35 us, a plain sum's time, where
// the last-level cache holds the map, 53 us after as many bytes were written. (64 rows a workgroup 58 us, 8 rows 53;
// one diagonal a thread, with single loads, 148.)
__global__ __launch_bounds__(MAP_T) void map_bwd(const float* g, const SmBuckets bk, float* part, int M, int N,
                                                 int start) {
    constexpr int NW = MAP_T / 64;
    __shared__ int border[QLKA_MAX_BUCKETS];
    __shared__ float sums[NW][QLKA_MAX_BUCKETS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m0 = blockIdx.x * SUM_ROWS, h = blockIdx.z;
    const int rows = min(SUM_ROWS, M - m0), buckets = (bk.n + 1) * (bk.both ? 2 : 1);
    for (int i = tid; i < bk.n; i += MAP_T) border[i] = bk.border[i];
    for (int i = lane; i < buckets; i += 64) sums[wave][i] = 0.f;
    __syncthreads();
    const int first = blockIdx.y * SUM_COLS - SUM_ROWS, c0 = first + 4 * tid;      // column of row m0
    const float* from = g + ((int64_t)h * M + m0) * N;
    float x[7] = {};                                                               // diagonals c0 - 3 .. c0 + 3
    const auto add = [&](f32x4u y, int i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[3 + j - i] += y[j];
    };
    // a wave inside the map; one at an edge, or past it
    const int lo = first + 256 * wave, hi = lo + 255 + rows - 1;                   // its columns
    if (lo >= 0 && hi < N && rows % 4 == 0) {
#pragma unroll 4
        for (int r = 0; r < rows; r += 4) {
            f32x4u y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = *reinterpret_cast<const f32x4u*>(from + (int64_t)(r + i) * N + c0 + r);
#pragma unroll
            for (int i = 0; i < 4; ++i) add(y[i], i);
        }
    } else if (hi >= 0 && lo < N) {
        // every lane loads, from the nearest value where it has none, so that the loads stay under way together
#pragma unroll 2
        for (int r = 0; r < rows; r += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float* row = from + (int64_t)min(r + i, rows - 1) * N;
                f32x4u y;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = c0 + r + j;
                    const float z = row[min(max(n, 0), N - 1)];
                    y[j] = n >= 0 && n < N && r + i < rows ? z : 0.f;
                }
                add(y, i);
            }
    }
    const int fb = far_bucket(bk, first + 256 * wave - 3 - m0 - start, first + 256 * wave + 255 - m0 - start);
    if (fb >= 0) {
        float y = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + x[6]);
#pragma unroll
        for (int k = 1; k < 64; k *= 2) y += __shfl_xor(y, k);
        if (lane == 0) sums[wave][fb] = y;
    } else {
#pragma unroll
        for (int j = 0; j < 7; ++j) {
            float y = x[j];
            const int bucket = bucket_of(border, bk.n, bk.both, c0 + j - 3 - m0 - start);
#pragma unroll
            for (int k = 1; k < 64; k *= 2) {              // lanes of one bucket are neighbours
                const float z = __shfl_up(y, k);
                const int c = __shfl_up(bucket, k);
                if (lane >= k && c == bucket) y += z;
            }
            const int after = __shfl_down(bucket, 1);
            if (lane == 63 || after != bucket) sums[wave][bucket] += y;
            wave_sync();
        }
    }
    __syncthreads();
    part += (((int64_t)h * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * buckets;
    for (int i = tid; i < buckets; i += MAP_T) part[i] = sums[0][i] + sums[1][i] + sums[2][i] + sums[3][i];
}

static dim3 map_grid(int M, int N, int H) {
    return dim3((unsigned)((N + MAP_COLS - 1) / MAP_COLS), (unsigned)((M + MAP_ROWS - 1) / MAP_ROWS), (unsigned)H);
}
static dim3 sum_grid(int M, int N, int H) {
    return dim3((unsigned)((M + SUM_ROWS - 1) / SUM_ROWS), (unsigned)((N + SUM_ROWS + SUM_COLS - 1) / SUM_COLS),
                (unsigned)H);
}

}  // namespace sm

int bias_map_fwd(const float* table, const SmBuckets& bk, float* out, int H, int M, int N, int start, hipStream_t st) {
    sm::map_fwd<<<sm::map_grid(M, N, H), sm::MAP_T, 0, st>>>(table, bk, out, H, M, N, start);
    return (int)hipGetLastError();
}

int bias_map_blocks(int M, int N) {
    const dim3 g = sm::sum_grid(M, N, 1);
    return (int)(g.x * g.y);
}

int bias_map_bwd(const float* g, const SmBuckets& bk, float* part, int H, int M, int N, int start, hipStream_t st) {
    sm::map_bwd<<<sm::sum_grid(M, N, H), sm::MAP_T, 0, st>>>(g, bk, part, M, N, start);
    return (int)hipGetLastError();
}

}  // namespace qlka
