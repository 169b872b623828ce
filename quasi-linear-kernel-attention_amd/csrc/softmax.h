// Softmax attention and the bucketed relative position bias: what the host side (softmax_api.hip) and the kernel files
// share. Not part of the public interface.
#pragma once

#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

#include "qlka.h"

namespace qlka {

// One query row and one key row are rows of D elements; b, h and r are the distances in elements between batches, heads
// and rows.
struct SmStrides { int64_t b, h, r; };

// Buckets of one side (distances dist >= 0): bucket i holds the distances from border[i - 1] up to below border[i]
// (bucket 0 from 0, the last one without end). both: keys after the query take the buckets from n + 1 on, else all
// of them take bucket 0.
struct SmBuckets {
    int n;                                   // borders
    int both;
    int far;                                 // distances from here on are in a side's last bucket
    int border[QLKA_MAX_BUCKETS];
};

struct SmParams {
    const void *q, *k, *v, *g_out;
    void *out, *g_q, *g_k, *g_v;
    float* out_full;                         // [B][H][M][D], or null
    int table_kept;                          // the table will have no gradient
    SmStrides sq, sk, sv, so, sg, sgq, sgk, sgv;
    const uint8_t* keep;                     // [B] rows of N bytes, keep_stride apart, or null
    int64_t keep_stride;
    const float* table;                      // [buckets][H], or null
    float *lse, *lse_low;                    // [B][H][M], half the log2 of the row's sum, and what lies below its last
                                             // place; +inf and 0 for a row without keys
    float* log2_sum;                         // [B][H][M], the log2 of the row's sum (each of these may be null)
    float lse_unit;                          // backward: what lse is multiplied by (lse may be a log2_sum)
    float* delta;                            // [B][H][M]
    int* large;                              // [B][H][groups of 32 rows]: whether a row has a large log sum
    float* part;                             // partial rows of DP floats: [split][B * heads][rows]
    float* part2;                            // a second set (dV), or [split][B * H][M][2] (maximum, sum) of the forward
    float* part_table;                       // [H][B * row blocks * splits][buckets]
    int B, H, G, M, N, D;
    int seen;                                // keys from here on are seen by no query, and not read
    int causal, start;
    int splits, blocks;                      // splits of the long axis; blocks of rows (or keys) per head
    float scale;                             // |scale|; its sign (or 0) is in q_sign
    float q_sign;
    SmBuckets bk;
    const int* offsets;                      // packed sequences (sm_packed_*): segments.h; then B is 1, M and N are the
    int sequences, groups;                   // rows of all, and `large` has `groups` numbers a head
};

// Elements of a row in LDS and in the partial rows.
inline int sm_padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
// Rows of the tiles that a workgroup goes through, for a number of parts an element and a padded row length.
constexpr int sm_tile_rows(int parts, int DP) { return DP == 128 || (parts == 3 && DP == 64) ? 32 : 64; }
inline int sm_buckets(const SmBuckets& b) { return (b.n + 1) * (b.both ? 2 : 1); }

// Launchers; each returns a hipError_t value. The dtype is QLKA_F32 or QLKA_BF16.
constexpr int FWD_WAVES = 4;              // waves a workgroup of the forward's kernels, of tiles and of single tokens
int sm_fwd(int dtype, const SmParams& p, hipStream_t st);
// the same for packed sequences (no mask, no bias), waves (of 32 rows) a workgroup: 1 or 4
int sm_packed_fwd(int dtype, const SmParams& p, int waves, hipStream_t st);
// waves (of 32 rows) a workgroup: 2 or 4
constexpr int STEP_MOST = 4;              // query rows a key head that sm_step takes
int sm_step(int dtype, const SmParams& p, hipStream_t st);
int sm_combine(int dtype, const SmParams& p, hipStream_t st);
int sm_delta(int dtype, const SmParams& p, hipStream_t st);
int sm_dq(int dtype, const SmParams& p, int waves, hipStream_t st);
int sm_dkv(int dtype, const SmParams& p, int waves, hipStream_t st);
int sm_packed_dq(int dtype, const SmParams& p, int waves, hipStream_t st);
int sm_packed_dkv(int dtype, const SmParams& p, int waves, hipStream_t st);
// out[row] = scale * sum over the splits of part's rows; rows of heads x len per batch
int sm_sum_parts(int dtype, const float* part, void* out, SmStrides so, float scale, int splits, int B, int heads,
                 int len, int D, hipStream_t st);
// g_table[bucket][h] = sum of part_table over its count rows
int sm_sum_table(const float* part, float* g_table, int H, int count, int buckets, hipStream_t st);

int bias_map_fwd(const float* table, const SmBuckets& bk, float* out, int H, int M, int N, int start, hipStream_t st);
int bias_map_blocks(int M, int N);
int bias_map_bwd(const float* g, const SmBuckets& bk, float* part, int H, int M, int N, int start, hipStream_t st);

// capi.hip: sets qlka_last_error() to the message and returns the code
int api_error(int code, const char* message);

}  // namespace qlka
