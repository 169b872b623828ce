/*
 * libqlka: MI355X (gfx950) weighted abs / Laplace sums, the hot path of quasi-linear kernel attention.
 *
 * A plain C ABI: device pointers, sizes and a hipStream_t passed as void*. Nothing here allocates device memory:
 * the caller passes outputs and a workspace of at least the size the matching *_ws_bytes() returns. All launches are
 * asynchronous on `stream`. Every function returns 0 on success or a QLKA_E* code; qlka_last_error() then holds a
 * message for the calling thread.
 *
 * Layouts (the reference's own, Weighted_Abs_Sum/weighted_abs_sum/ops.py:107-110): q (P, D, M), k (P, D, N),
 * v (P, N, C), row outputs (P, M, C), out_u (P, M), per-feature outputs (P, D, M) / (P, D, N); fp32, contiguous.
 * Limits (Weighted_Abs_Sum/csrc/binding.cpp:69-84): P, D, N, M >= 1; 1 <= C <= 128; N, M <= 131072;
 * P*D*max(N, M) <= INT32_MAX.
 */
#ifndef QLKA_H
#define QLKA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QLKA_OK         0
#define QLKA_EINVAL     1   /* argument validation failed (message says which) */
#define QLKA_EWORKSPACE 2   /* workspace null or smaller than *_ws_bytes() */
#define QLKA_EHIP       3   /* a HIP launch failed */

/* Message of the last error on this thread ("" if none). */
const char* qlka_last_error(void);
/* ABI version of this library. */
int qlka_version(void);
/*
 * Base cutoff B of the dense evaluation (the qlka_direct_* kernels: same results to fp32 rounding, same tie
 * conventions) in qlka_laplace_fwd, qlka_abs_fwd (path -1), qlka_abs_bwd and qlka_sgn_fwd, with L = max(N, M): the
 * abs forward goes dense for L <= 2B, the Laplace forward for L <= B, the backward and the sgn sum for L <= B or for
 * L <= 5B/4 when P * ceil(L / 32) >= 512. Whatever B (0 included) and the pinned path, the abs forward also goes
 * dense for N <= 16 keys, and the backward and the sgn sum for min(N, M) <= 16 (the walk's segment totals lose
 * accuracy with a handful of keys). Default 512; 0 sorts everything else. Process-wide; returns the previous
 * value (or -QLKA_EINVAL for n < 0). The C-level counterpart of the reference's set_keops_cutoff
 * (Weighted_Abs_Sum/weighted_abs_sum/ops.py:21-25), which picks the KeOps backend in Python.
 */
int qlka_set_direct_max(int n);
/*
 * Which sorted route a call takes, for tests and measurements: segments of N + M <= 32768 elements can run column by
 * column, all others walk. AUTO (the default) takes the columns where they were measured faster, NEVER walks
 * everything, ALWAYS takes the columns wherever they apply. Results agree to fp32 rounding. What the dense evaluation
 * takes stays there (qlka_set_direct_max). Process-wide; returns the previous mode (or -QLKA_EINVAL for another one).
 */
#define QLKA_COLUMNS_AUTO   0
#define QLKA_COLUMNS_NEVER  1
#define QLKA_COLUMNS_ALWAYS 2
int qlka_set_columns(int mode);
/*
 * Workspace budget in bytes (default 5 GiB). Every operator below runs its whole pipeline on chunks of consecutive
 * p = (batch, head) indices (every stage works on each p alone), taking the largest chunk the workspace it is given
 * holds (at least one p), so the caller bounds device memory by the workspace it passes. The *_ws_bytes() queries
 * report the workspace of the largest chunk within this budget (one p when even one p exceeds it); results do not
 * depend on the chunking. They report 0 for a call that takes the dense route at the current cutoff (qlka_laplace_fwd,
 * qlka_abs_fwd, qlka_abs_bwd, qlka_abs_bwd_sorted, qlka_sgn_fwd): such a call takes no workspace, and ws may be null
 * (a dense abs forward that keeps its sorts for a walking backward needs sort scratch only for segments longer than
 * 16384). Process-wide; returns the previous value. The reference has no counterpart: its
 * workspace is O(P*D*(N+M)) (Weighted_Abs_Sum/csrc/binding.cpp:101-111), where this build's per-feature slab of
 * contribution rows is O(P*D*M*C).
 */
size_t qlka_set_workspace_budget(size_t bytes);

/*
 * weighted_laplace_sum forward.
 *   out_w[p,m,c] = sum_{d,n} exp(-|k[p,d,n] - q[p,d,m]|) v[p,n,c],  out_u[p,m] = sum_{d,n} exp(-|k[p,d,n] - q[p,d,m]|)
 * max(N, M) <= B (the dense cutoff, default 512; see qlka_set_direct_max) runs the dense evaluation of
 * qlka_direct_fwd (no workspace: qlka_laplace_fwd_ws_bytes reports 0).
 * Replaces _ext.weighted_laplace_sum_forward (Weighted_Laplace_Sum/csrc/binding.cpp:63-100).
 */
size_t qlka_laplace_fwd_ws_bytes(int P, int D, int N, int M, int C);
int qlka_laplace_fwd(const float* q, const float* k, const float* v, float* out_w, float* out_u,
                     int P, int D, int N, int M, int C, void* ws, size_t ws_bytes, void* stream);
/*
 * qlka_laplace_fwd without a workspace argument and without any device allocation. No counterpart in the reference:
 * it is for callers that cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc). Its workspace is a static 512 MiB device array of the library, held on every device the
 * library runs on until the process ends; the call runs qlka_laplace_fwd over it one chunk of p at a time and gives
 * the same results. Shapes whose single-p workspace (qlka_laplace_fwd_ws_bytes(1, D, N, M, C)) exceeds 512 MiB are
 * refused with QLKA_EINVAL (N = M = 16384, D = C = 64 needs 297 MiB). `stream` must belong to the current device.
 * All calls on one device share the array: calls that overlap in time on one device (e.g. on two streams) race and
 * must be serialised by the caller. The array takes device memory from the first call on a device on (hipMemGetInfo
 * on MI355X: free memory unchanged by loading the library, 6 MiB less after a first qlka_laplace_fwd call, whose
 * kernels' code loads on first use, and 512 MiB less after this entry's first call; unchanged by its later calls); a
 * process that never calls it does not hold it. A thread's first uncaptured call on a
 * device may create that thread's side stream and its events (hipStreamCreateWithFlags, hipEventCreateWithFlags:
 * no device memory); under stream capture, or once they exist, the call creates nothing.
 */
int qlka_laplace_fwd_noalloc(const float* q, const float* k, const float* v, float* out_w, float* out_u,
                             int P, int D, int N, int M, int C, void* stream);

/*
 * weighted_abs_sum forward; out_u == NULL gives the plain op, out_u != NULL the _full op.
 *   out_w[p,m,c] = sum_{d,n} |k[p,d,n] - q[p,d,m]| v[p,n,c],  out_u[p,m] = sum_{d,n} |k[p,d,n] - q[p,d,m]|
 * path: -1 auto, 0 global, 1 fused (the fused path exists for max(N, M) <= 4096 only, as in the reference). Under
 * auto, short segments run the dense evaluation of qlka_direct_fwd (see qlka_set_direct_max).
 * Replaces _ext.weighted_abs_sum_forward / weighted_abs_sum_full_forward (Weighted_Abs_Sum/csrc/binding.cpp:229-239).
 */
size_t qlka_abs_fwd_ws_bytes(int P, int D, int N, int M, int C);
int qlka_abs_fwd(const float* q, const float* k, const float* v, float* out_w, float* out_u,
                 int P, int D, int N, int M, int C, int path, void* ws, size_t ws_bytes, void* stream);

/*
 * weighted_abs_sum backward; g_u == NULL gives the plain backward, g_u != NULL the _full backward.
 *   grad_q[p,d,m] = sum_n s(q_m - k_n) (<v_n, g_w[m]> + g_u[m]),
 *   grad_k[p,d,n] = sum_m s(k_n - q_m) (<g_w[m], v_n> + g_u[m]),
 *   grad_v[p,n,c] = sum_{d,m} |k_n - q_m| g_w[p,m,c];  s(x) = +1 for x > 0, -1 otherwise (a tie counts -1).
 * Replaces _ext.weighted_abs_sum_backward / weighted_abs_sum_full_backward (Weighted_Abs_Sum/csrc/binding.cpp:242-380).
 */
size_t qlka_abs_bwd_ws_bytes(int P, int D, int N, int M, int C);
int qlka_abs_bwd(const float* q, const float* k, const float* v, const float* g_w, const float* g_u,
                 float* grad_q, float* grad_k, float* grad_v,
                 int P, int D, int N, int M, int C, void* ws, size_t ws_bytes, void* stream);

/*
 * Forward and backward that share their sorts. The reference's backward sorts k and q again
 * (Weighted_Abs_Sum/csrc/binding.cpp:242-380 after :229-239); here a forward can leave the sorted k and q and their
 * permutations in caller buffers (k_sorted, k_perm: P*D*N each; q_sorted, q_perm: P*D*M each) for the backward of
 * the same inputs. qlka_abs_bwd_walks tells whether qlka_abs_bwd would sort and walk at this shape (1) or run the
 * dense kernels (0), i.e. whether keeping the sorts pays; qlka_abs_fwd_keep computes what qlka_abs_fwd computes and
 * sets *kept = 1 when it filled the four buffers (0: left untouched, the backward would not use them); after
 * *kept != 0, qlka_abs_bwd_sorted with the same q, k, v computes what qlka_abs_bwd computes without sorting. Same
 * workspace sizes as qlka_abs_fwd / qlka_abs_bwd.
 * states (optional, may be NULL; qlka_abs_keep_state_bytes() bytes, 0 when the backward would read none: it takes the
 * dense kernels, or, at C <= 64 with C % 4 == 0, walks once over the merged sorted keys and queries): the forward
 * also leaves there the range states and query bounds of its walk over the sorted keys, which the backward's grad_q
 * walk would compute again (the same range sums, scan and bounds); it sets *kept = 3 when it wrote them (its own walk
 * ran; a forward on the dense kernels or by columns keeps only the sorts). Passing them to qlka_abs_bwd_sorted after
 * *kept = 3 skips one range-sum pass, one scan and one bound search per chunk of the backward, with bit-identical
 * gradients.
 */
int qlka_abs_bwd_walks(int P, int N, int M);
size_t qlka_abs_keep_state_bytes(int P, int D, int N, int M, int C);
int qlka_abs_fwd_keep(const float* q, const float* k, const float* v, float* out_w, float* out_u,
                      int P, int D, int N, int M, int C, int path, float* k_sorted, uint32_t* k_perm,
                      float* q_sorted, uint32_t* q_perm, void* states, int* kept, void* ws, size_t ws_bytes,
                      void* stream);
int qlka_abs_bwd_sorted(const float* q, const float* k, const float* v, const float* g_w, const float* g_u,
                        float* grad_q, float* grad_k, float* grad_v, int P, int D, int N, int M, int C,
                        const float* k_sorted, const uint32_t* k_perm, const float* q_sorted, const uint32_t* q_perm,
                        const void* states, void* ws, size_t ws_bytes, void* stream);

/*
 * Dense forward and backward that share the kernel matrix A[p,m,n] = sum_d |k[p,d,n] - q[p,d,m]|. No counterpart in
 * the reference, whose dense (KeOps) route forms A again in the backward (Weighted_Abs_Sum/weighted_abs_sum/
 * keops_backend.py:19-48). qlka_abs_dense_keep_bytes is the size of A (P*M rows of (N + 3) & ~3 floats) where the
 * forward and the backward both run the dense kernels and A stays within 256 MB, else 0; then qlka_abs_fwd_dense_keep
 * computes what qlka_abs_fwd computes and also writes A, and qlka_abs_bwd_dense_kept, given that A and the same q, k, v,
 * computes what qlka_abs_bwd computes, with grad_v as the contraction of A with g_w instead of forming A again
 * (bit-identical gradients). Both take no workspace; both return QLKA_EINVAL where the size is 0.
 */
size_t qlka_abs_dense_keep_bytes(int P, int D, int N, int M, int C);
int qlka_abs_fwd_dense_keep(const float* q, const float* k, const float* v, float* out_w, float* out_u, float* A,
                            int P, int D, int N, int M, int C, void* stream);
int qlka_abs_bwd_dense_kept(const float* q, const float* k, const float* v, const float* g_w, const float* g_u,
                            float* grad_q, float* grad_k, float* grad_v, const float* A, int P, int D, int N, int M,
                            int C, void* stream);

/*
 * weighted_sgn_sum: out[p,d,m] = sum_n sgn(k[p,d,n] - q[p,d,m]) <v[p,n,:], g[p,m,:]>, with a tie counted +1
 * (it is the negated grad_q walk). Replaces _ext.weighted_sgn_sum_forward (Weighted_Abs_Sum/csrc/binding.cpp:384-439).
 */
size_t qlka_sgn_fwd_ws_bytes(int P, int D, int N, int M, int C);
int qlka_sgn_fwd(const float* q, const float* k, const float* v, const float* g, float* out,
                 int P, int D, int N, int M, int C, void* ws, size_t ws_bytes, void* stream);

/*
 * Dense evaluation for short segments: A[m,n] = sum_d f(q[p,d,m] - k[p,d,n]) with f = |x| (kind 0, the weighted abs
 * sum) or exp(-|x|) (kind 1, the weighted Laplace sum), out_w[p,m,:] = sum_n A[m,n] v[p,n,:], out_u[p,m] = sum_n
 * A[m,n] (out_u may be NULL). Same values as qlka_abs_fwd / qlka_laplace_fwd; no sort and no workspace, O(N M D)
 * work, so it is the faster route only for short segments (the ops pick it by size). The role of the reference's
 * KeOps backend below KEOPS_CUTOFF (Weighted_Abs_Sum/weighted_abs_sum/keops_backend.py:19-35).
 */
#define QLKA_DIRECT_ABS     0
#define QLKA_DIRECT_LAPLACE 1
int qlka_direct_fwd(int kind, const float* q, const float* k, const float* v, float* out_w, float* out_u,
                    int P, int D, int N, int M, int C, void* stream);

/*
 * Dense evaluation of the abs backward and of weighted_sgn_sum with an explicit value `tie` of sign(0): the
 * formulas of qlka_abs_bwd / qlka_sgn_fwd with s(0) = tie (0: the KeOps convention of keops_backend.py:40-41 and of
 * autograd through the KeOps forward; -1 for the gradients / +1 for the sgn sum: the walk's convention). g_u may be
 * NULL. No workspace; O(N M (D + C)) work, for short segments.
 */
int qlka_direct_bwd(float tie, const float* q, const float* k, const float* v, const float* g_w, const float* g_u,
                    float* grad_q, float* grad_k, float* grad_v, int P, int D, int N, int M, int C, void* stream);
int qlka_direct_sgn(float tie, const float* q, const float* k, const float* v, const float* g, float* out,
                    int P, int D, int N, int M, int C, void* stream);

/*
 * Fused additive-kernel attention layer, forward: the op(s) plus the normalising epilogue in one call.
 *   kind QLKA_ADD_LAPLACE: out = w / clamp(u - n_pad sum_d e^{-|q_d|}, 1e-6), (w, u) = weighted_laplace_sum(q, k, v)
 *   kind QLKA_ADD_RIESZ:   out = ((|q|_1 + 1e-3) sum_n v_n + sum_n |k_n|_1 v_n - w)
 *                               / clamp((|q|_1 + 1e-3) M + sum_n |k_n|_1 - u - 1e-3 n_pad, 1e-6),
 *                          (w, u) = weighted_abs_sum_full(q, k, v)
 *   kind QLKA_ADD_BUMP:    out = ((w+ + w-)/2 - w0) / clamp((u+ + u-)/2 - u0 - n_pad sum_d max(0, 1 - |q_d|), 1e-6),
 *                          (w0, u0), (w+, u+), (w-, u-) = weighted_abs_sum_full at q, q + 1, q - 1; the three share one
 *                          sort of k and q and one set of key-range summaries.
 * q (P, D, M) and k (P, D, N) already divided by tau, k and v already multiplied by the key mask; n_pad (P) is the
 * number of masked keys per p (NULL: none); out (P, M, C). No gradient.
 * Replaces _add_laplace / _add_riesz / _add_bump (Experiments/kernel_attention/attention.py:67-92).
 */
#define QLKA_ADD_LAPLACE 0
#define QLKA_ADD_RIESZ   1
#define QLKA_ADD_BUMP    2
size_t qlka_layer_fwd_ws_bytes(int kind, int P, int D, int N, int M, int C);
int qlka_layer_fwd(int kind, const float* q, const float* k, const float* v, const float* n_pad, float* out,
                   int P, int D, int N, int M, int C, void* ws, size_t ws_bytes, void* stream);

/*
 * The same layers with the key mask applied inside the sums: q (P, D, M) and k (P, D, N) divided by tau, k and v NOT
 * multiplied by the mask, keep (P, N) bytes (nonzero = real key, non-null). Masked keys weigh 0 in every sum, so w and
 * u run over the real keys only and the n_pad corrections become exact (add_laplace: out = w / clamp(u, 1e-6), ...);
 * no k * keep or v * keep is materialised. Same values as qlka_layer_fwd on k * keep, v * keep and n_pad = N - #kept,
 * without the cancellation of the n_pad terms. Workspace: qlka_layer_fwd_ws_bytes.
 * Replaces the keep branch of attention() (Experiments/kernel_attention/attention.py:122-124) around _add_laplace /
 * _add_riesz / _add_bump, and the padded-key rule of Weighted_Laplace_Sum/weighted_laplace_sum/__init__.py:12.
 */
int qlka_layer_fwd_masked(int kind, const float* q, const float* k, const float* v, const uint8_t* keep, float* out,
                          int P, int D, int N, int M, int C, void* ws, size_t ws_bytes, void* stream);

/*
 * Softmax attention to a sequence of another length, and the learned relative position bias by buckets. No counterpart
 * in the reference's operators: its "softmax" baseline is torch's scaled_dot_product_attention
 * (Experiments/kernel_attention/attention.py:99-102), for which it has no position bias.
 *
 *   S[b,h,m,n] = scale <q[b,h,m], k[b,h/(H/G),n]> + table[bucket(n - (m + start))][h]      (table may be NULL: no bias)
 *   out[b,h,m] = sum_n P[m,n] v[b,h/(H/G),n],  P = softmax of S over the keys that the query sees
 * A query sees key n if keep[b][n] is nonzero (keep may be NULL) and, with causal, n <= m + start. A row that sees no
 * key (or only scores of -inf) gives zeros, here and in every gradient. Rows of keys that are masked, or that no query
 * of the call sees, are not read. scale: 0 or of a size in [2^-96, 2^96]. The table's values are finite, up to the
 * type's lowest and largest, or -inf. Scores may be as large as fp32 holds (where their roundings pass 1, equal ones
 * share a row and others may not compare as they would in exact arithmetic); past that, and where other infinities or
 * NaN are read, a row can be NaN.
 * Sums, the softmax's statistics and every sum of the gradients are fp32; with QLKA_BF16 the probabilities and dS are
 * rounded to bf16 for their matrix products, and each result once at its end.
 *
 * q (B, H, M, D), k and v (B, G, N, D) with H a multiple of G; D a multiple of 8 up to 128, its elements contiguous;
 * *_stride are the distances in elements between batches, heads and rows, 0 or more (a dimension of size 1: any value);
 * every row starts at a multiple of 16 bytes. keep is rows of N bytes, keep_stride bytes apart. M and N may be 0.
 * A launch takes less than 2^32 threads: B * heads * ceil(rows / 128) stays below 2^24.
 *
 * Buckets: a side's bucket i holds the distances from border[i - 1] up to below border[i] (bucket 0 from 0 on, the last
 * one without end); border is non-decreasing and positive, on the host. bidirectional: distance |d| for d = n - (m +
 * start), keys after the query (d > 0) in buckets num_borders + 1 on, 2 (num_borders + 1) buckets in all. Else distance
 * max(-d, 0) and num_borders + 1 buckets. table and g_table are (buckets, H) fp32, contiguous.
 *
 * Forward: writes out and, where not NULL, lse (B, H, M) (log2 of each row's sum, +inf for a row without keys),
 * log_sums (2, B, H, M) (half of that log2, in two floats: the second is what lies below the first one's last place;
 * where scores are large, it is the log of the number of keys that share a row) and out_full (with QLKA_BF16: (B, H, M,
 * D) fp32, out before it is rounded; for the gradients' row sums, in which an error of out is common to all of a row's
 * dS). With out_full and a table the probabilities are taken whole, for the table's gradient, unless table_kept is
 * nonzero: the table will have none, and out is what the same call without out_full gives. Backward: reads q, k, v,
 * out, g_out, log_sums or (for log sums of the ordinary size) lse alone and, where not NULL, out_full, writes g_q (may
 * be NULL), g_k and g_v (both or neither NULL) and g_table (may be NULL; with QLKA_BF16 it needs out_full). No atomics:
 * results do not change from run to run.
 */
#define QLKA_F32  0
#define QLKA_BF16 1
#define QLKA_MAX_BUCKETS 256
typedef struct qlka_softmax_args {
    int dtype, B, H, G, M, N, D;
    int causal, start;
    float scale;
    const void *q, *k, *v;
    int64_t q_stride[3], k_stride[3], v_stride[3];
    const uint8_t* keep;
    int64_t keep_stride;
    const float* table;
    const int* border;
    int num_borders, bidirectional;
    void* out;
    int64_t out_stride[3];
    float* out_full;
    float* lse;
    const void* g_out;
    int64_t g_out_stride[3];
    void *g_q, *g_k, *g_v;
    int64_t g_q_stride[3], g_k_stride[3], g_v_stride[3];
    float* g_table;
    float* log_sums;
    int table_kept;
} qlka_softmax_args;
size_t qlka_softmax_fwd_ws_bytes(const qlka_softmax_args* args);
int qlka_softmax_fwd(const qlka_softmax_args* args, void* ws, size_t ws_bytes, void* stream);
size_t qlka_softmax_bwd_ws_bytes(const qlka_softmax_args* args);
int qlka_softmax_bwd(const qlka_softmax_args* args, void* ws, size_t ws_bytes, void* stream);
/*
 * The bias as a map, out (H, M, N) fp32 with out[h,m,n] = table[bucket(n - (m + start))][h], and its gradient, g_table
 * (buckets, H) = the sums of g (H, M, N) over each bucket.
 */
int qlka_bias_map_fwd(const float* table, const int* border, int num_borders, int bidirectional, float* out, int H,
                      int M, int N, int start, void* stream);
size_t qlka_bias_map_bwd_ws_bytes(int num_borders, int bidirectional, int H, int M, int N);
int qlka_bias_map_bwd(const float* g, const int* border, int num_borders, int bidirectional, float* g_table, int H,
                      int M, int N, int start, void* ws, size_t ws_bytes, void* stream);

/*
 * Softmax attention within sequences of different lengths that lie one after the other in T rows (no padding). offsets
 * (B + 1 numbers on the device, not decreasing, in [0, T]) are where the sequences begin, and where the last one ends:
 * a row sees the keys of its own sequence, with causal those up to itself. Rows outside every sequence get zeros, here
 * and in every gradient. No sequence changes another one's results, whatever it holds. No counterpart in the reference.
 *
 *   out[h,m] = sum_n P[m,n] v[h/(H/G),n],  P = softmax of scale <q[h,m], k[h/(H/G),n]> over the keys n that m sees
 *
 * q (H, T, D), k and v (G, T, D); *_stride are the distances in elements between heads and rows. Types, D, alignment,
 * scale, roundings, lse, log_sums (2, H, T), out_full (H, T, D) and the gradients are as for qlka_softmax_fwd / _bwd
 * without a table, but that log_sums are those of the exponentials before their rounding to bf16: a probability of the
 * gradients has no other error than its own rounding (where keys are split, out can then differ in its last place from
 * that of a call without log_sums). Offsets that decrease give rows that are not said, but no access outside the
 * tensors. The offsets may change between the replays of a captured call. A launch takes less than 2^32 threads, so
 * heads * (T / 32 + B) stays below 2^24.
 */
typedef struct qlka_packed_args {
    int dtype, B, H, G, T, D;
    int causal;
    float scale;
    const int* offsets;
    const void *q, *k, *v;
    int64_t q_stride[2], k_stride[2], v_stride[2];
    void* out;
    int64_t out_stride[2];
    float* out_full;
    float* log_sums;
    const void* g_out;
    int64_t g_out_stride[2];
    void *g_q, *g_k, *g_v;
    int64_t g_q_stride[2], g_k_stride[2], g_v_stride[2];
} qlka_packed_args;
size_t qlka_packed_fwd_ws_bytes(const qlka_packed_args* args);
int qlka_packed_fwd(const qlka_packed_args* args, void* ws, size_t ws_bytes, void* stream);
size_t qlka_packed_bwd_ws_bytes(const qlka_packed_args* args);
int qlka_packed_bwd(const qlka_packed_args* args, void* ws, size_t ws_bytes, void* stream);

/*
 * A cache of keys and values in pages. A sequence's token at position i is row i % page_size of page
 * tables[b][i / page_size]; pages are rows of D elements for each of G key heads, at any strides (elements, between
 * pages, heads and rows, each below 2^32 bytes). What is held (held):
 *   QLKA_F32, QLKA_BF16  the rows as they are; of the type of the call (dtype) only
 *   QLKA_INT8, QLKA_E4M3 8 bits an element, and for every 32 elements of a row a byte e (k_exp, v_exp: ceil(D / 32) a
 *                        row, contiguous; strides in bytes between pages, heads and rows): an element stands for
 *                        code * 2^(e - 127). e is the least of [27, 248] (int8; 246 with e4m3) with which the largest
 *                        code (127; 448) reaches the largest element, the codes are the nearest ones, ties to the
 *                        even one. Such values are exact in bf16 and fp32, so nothing is rounded a second time when
 *                        they are read. e = 255 marks 32 elements of which one was infinite or NaN: all read as NaN.
 *
 * tables: B rows of table_len page numbers, table_stride apart; lengths: B numbers of tokens, the new ones included;
 * offsets (B + 1): the new tokens of the sequences one after the other in T rows, or NULL: one for each, T = B. All on
 * the device; their contents may change between the replays of a captured call. Row m of sequence b is at position
 * lengths[b] - (offsets[b + 1] - m). Page numbers outside [0, num_pages), and what a table's row has no place for, are
 * pages that do not exist: nothing is written there, keys there are not seen, reading gives zeros.
 *
 * qlka_paged_write: the new tokens' k and v (G, T, D) go to their positions. Rows outside every sequence, or at
 *   negative positions, are left out; nothing else in the pages changes. Two rows of one call at one place in a page
 *   leave either one's values, or parts of both.
 * qlka_paged_read: out_k and out_v (B, G, N, D) of dtype get the first N positions of each sequence, zeros from
 *   lengths[b] on.
 * qlka_paged_attention: out (H, T, D), softmax attention of the new tokens q (H, T, D) to their sequence's held keys up
 *   to their own position, which have been written before. Rows that see none, and rows outside every sequence, get
 *   zeros.
 *   longest: the most new tokens of a sequence if the caller knows it, else 0. It only decides which kernels run.
 *
 * Strides are in elements between heads and rows ((B, heads, rows) for out_k and out_v); D a multiple of 8 up to 128,
 * rows at multiples of 16 bytes (in pages of 8 bits with D no multiple of 16: of 8 bytes). The scale is as for
 * qlka_softmax_fwd, the probabilities are rounded to bf16 for their product where q is. Infinities and NaN that a
 * sequence holds at its new tokens' positions or before can make any of its new rows NaN, no other sequence's.
 */
#define QLKA_INT8 2
#define QLKA_E4M3 3
typedef struct qlka_paged_args {
    int dtype, held, B, H, G, T, D;
    int page_size, num_pages, table_len, longest, N;
    float scale;
    const int *tables, *lengths, *offsets;
    int64_t table_stride;
    void *k_pages, *v_pages;
    int64_t k_pages_stride[3], v_pages_stride[3];
    uint8_t *k_exp, *v_exp;
    int64_t k_exp_stride[3], v_exp_stride[3];
    const void *q, *k, *v;
    int64_t q_stride[2], k_stride[2], v_stride[2];
    void *out, *out_k, *out_v;
    int64_t out_stride[2], out_k_stride[3], out_v_stride[3];
} qlka_paged_args;
int qlka_paged_write(const qlka_paged_args* args, void* stream);
int qlka_paged_read(const qlka_paged_args* args, void* stream);
size_t qlka_paged_attention_ws_bytes(const qlka_paged_args* args);
int qlka_paged_attention(const qlka_paged_args* args, void* ws, size_t ws_bytes, void* stream);

/*
 * Test entry: stable ascending sort of num_segs contiguous segments of seg_len fp32 keys; perm[i] is the in-segment
 * index of the i-th smallest key (np.argsort(kind="stable"); -0.0 ties +0.0 and is written as +0.0).
 * Replaces launch_iota + launch_cub_sort (Weighted_Abs_Sum/csrc/sort_utils.cu:85-117).
 */
size_t qlka_seg_sort_ws_bytes(int num_segs, int seg_len);
int qlka_seg_sort(const float* keys, float* sorted, uint32_t* perm, int num_segs, int seg_len,
                  void* ws, size_t ws_bytes, void* stream);

/*
 * Test entry: merge rank of every query, rank[s,m] = #{n : k[s,n] < q[s,m]} (np.searchsorted(side="left")), computed
 * by the same sort + range split + merge walk the operators use. Replaces the walk start / emit rule of
 * Weighted_Abs_Sum/csrc/walk_common.cuh:10-30 and abs_kernels.cu:324.
 */
size_t qlka_merge_rank_ws_bytes(int num_segs, int N, int M);
int qlka_merge_rank(const float* q, const float* k, int32_t* rank, int num_segs, int N, int M,
                    void* ws, size_t ws_bytes, void* stream);

/*
 * Optional per-stage timing (no reference counterpart; measurement aid for bench.py). When enabled, every kernel
 * launch is bracketed by hipEvents on its own stream; qlka_timing_read() synchronises them and reports the
 * accumulated milliseconds and launch count of one stage ("lap_range_walk", "abs_range_walk", "lds_radix_sort", ...).
 * The stage "busy" is the union of all bracketed intervals since the last reset (time in which at least one library
 * kernel ran; launches on the side stream overlap those on the caller's stream).
 */
int qlka_timing_enable(int on);
int qlka_timing_reset(void);
int qlka_timing_read(const char* stage, double* total_ms, long long* count);

#ifdef __cplusplus
}
#endif

#endif /* QLKA_H */
