// The C ABI of softmax attention and of the bias map (include/qlka.h): validation, the choice of kernel and split, the
// workspace and the launches.
#include "qlka.h"
#include "qlka_internal.h"
#include "softmax.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

using namespace qlka;

namespace {

constexpr int64_t LONGEST = 1 << 28;      // rows, keys, positions: sums of a few stay in 32 bits
constexpr int64_t MOST_ROWS = INT32_MAX;

int refuse(const char* fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return api_error(QLKA_EINVAL, buf);
}

int status(int e, const char* where) {
    if (e == 0) return QLKA_OK;
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", where, hipGetErrorString((hipError_t)e));
    return api_error(QLKA_EHIP, buf);
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int check_buckets(const int* border, int n, int both, SmBuckets* bk) {
    const int most = both ? QLKA_MAX_BUCKETS / 2 : QLKA_MAX_BUCKETS;
    if (n < 0 || n >= most) return refuse("at most %d buckets", QLKA_MAX_BUCKETS);
    if (n > 0 && !border) return refuse("border must be non-null");
    bk->n = n;
    bk->both = both ? 1 : 0;
    bk->far = 0;
    for (int i = 0; i < n; ++i) {
        if (border[i] < 1 || border[i] > LONGEST || border[i] < bk->far)
            return refuse("border must be positive, non-decreasing and at most 2^28");
        bk->border[i] = bk->far = border[i];
    }
    return QLKA_OK;
}

int check_sizes(const qlka_softmax_args* a) {
    if (!a) return refuse("args must be non-null");
    if (a->dtype != QLKA_F32 && a->dtype != QLKA_BF16) return refuse("dtype must be QLKA_F32 or QLKA_BF16");
    if (a->B < 0 || a->M < 0 || a->N < 0 || a->H < 1 || a->G < 1)
        return refuse("B, M and N must be >= 0, H and G >= 1");
    if (a->H % a->G) return refuse("H must be a multiple of G");
    if (a->D < 8 || a->D > 128 || a->D % 8) return refuse("D must be a multiple of 8 in [8, 128]");
    if (a->M > LONGEST || a->N > LONGEST || a->start > LONGEST || a->start < -LONGEST)
        return refuse("M, N and |start| must be <= 2^28");
    if ((double)a->B * a->H * a->M > (double)MOST_ROWS || (double)a->B * a->G * a->N > (double)MOST_ROWS)
        return refuse("B * H * M and B * G * N must fit int32");
    // the gradients hold log sums in units of the scale
    if (a->scale != 0.f && !(std::fabs(a->scale) >= 0x1p-96f && std::fabs(a->scale) <= 0x1p96f))
        return refuse("scale must be 0 or of a size in [2^-96, 2^96]");
    return QLKA_OK;
}

// ---- how a call runs

constexpr int CUS = 256;

// Splits of an axis of `tiles` tiles for `groups` workgroups over the other axes, by an estimate of the time: rounds of
// workgroups on a CU (one alone on a CU is not twice as fast as two, waits not being filled), each its tiles and what
// it costs by itself, and the joining of `join` bytes a split. In microseconds, the constants set by hand until 12
// shapes (prompts and gradients of 65 to 8192 keys, fp32 and bf16) came near the best of 1 to 16 splits of all their
// axes: eight of them within 4% of it or faster (1 x 4 heads, 100 x 8000: 14.4 us, 17.2 the best one number, 132 unsplit),
// the others 7 to 18% slower (1 x 12, 512 x 4096: 26.8 : 23.7, unsplit 70; 4 x 12, 1024 x 4096: 91 : 77, unsplit 88).
int splits_for(int64_t groups, int64_t tiles, double tile_us, double join_bytes) {
    int best = 1;
    double least = 0;
    for (int s = 1; s <= 64 && (s == 1 || 2 * s <= tiles); ++s) {
        const double rounds = std::max<double>(1.7, (double)ceil_div(groups * s, CUS));
        double t = rounds * (2.0 + tile_us * ceil_div(tiles, s));
        if (s > 1) t += 4.0 + s * join_bytes / 2e6;
        if (s == 1 || t < 0.95 * least) {
            best = s;
            least = t;
        }
    }
    return best;
}
// The same for the kernel of few rows, which is bound by memory: enough workgroups to fill the GPU, four tiles each or
// more.
int step_splits(int64_t groups, int64_t tiles) {
    if (groups >= 1024) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div(2048, std::max<int64_t>(groups, 1)), tiles / 4, 256}));
}

// Keys that some query may see; in causal order a longer cache's are not read.
int seen_keys(const qlka_softmax_args* a) { return a->causal ? std::max(0, std::min(a->N, a->M + a->start)) : a->N; }

int tile_rows(const qlka_softmax_args* a) { return sm_tile_rows(a->dtype == QLKA_F32 ? 3 : 1, sm_padded(a->D)); }

struct RowPlan { int waves, blocks, splits; };
// kernels that own `len` rows of each of `heads` heads and go over `tiles` tiles of the other side
// (waves: 0 for two where the rows are few, measured 6% faster there for the gradients and 5% slower for the forward)
RowPlan row_plan(const qlka_softmax_args* a, int heads, int len, int64_t tiles, double products, int waves) {
    RowPlan r;
    r.waves = waves ? waves : len <= 64 ? 2 : 4;
    r.blocks = (int)ceil_div(len, 32 * r.waves);
    const int DP = sm_padded(a->D);
    const double tile_us = products * 0.3 * DP / 64 * (a->dtype == QLKA_F32 ? 2 : 1);
    r.splits = splits_for((int64_t)a->B * heads * r.blocks, tiles, tile_us, (double)a->B * heads * len * DP * 8);
    return r;
}

// Few query rows per key head: the kernel without matrix tiles (softmax_step.hip), against the tiles, which read shared
// keys once for each query head but hardly compute in bf16. Measured (us, step : tiles), B, heads / key heads, M, N of
// 64 elements:
//   bf16  8, 12 / 12, 1,  197     6.2 :  7.9       fp32  8, 12 / 12, 4,  197    11.6 :  15.4
//   bf16 16, 12 / 12, 2, 8192      87 :   74       fp32 16, 12 / 3,  1, 4096      36 :  136
//                                                  fp32  1,  8 / 1,  1, 4096    21.3 :  15.8
// and bf16 single tokens whose heads share keys, by the bytes of k and v (MB):
//    4.2   4, 12 / 4, 1024     15.1 : 11.0          50   8, 12 / 6, 4096    20.1 : 22.5
//   16.8   4, 12 / 4, 4097     18.0 : 17.2          50   8, 12 / 3, 8192    30.0 : 35.7
//   33.6  64,  8 / 4,  512     16.1 : 14.2          67  32, 12 / 4, 2048    31.1 : 35.9
//   33.6   8, 12 / 4, 4097     21.7 : 22.6          67 128,  8 / 4,  512    23.5 : 26.8
//   33.6   4, 12 / 4, 8192     20.4 : 23.1         101  16, 12 / 6, 4096    31.9 : 37.6
//   33.6   1,  8 / 2, 65536    26.4 : 28.3         102   1,  8 / 2, 200000  49.3 : 65.5
bool steps(const qlka_softmax_args* a) {
    const int64_t rows = (int64_t)a->H / a->G * a->M;
    if (a->dtype == QLKA_F32) return rows <= STEP_MOST;
    const double bytes = 4.0 * a->B * a->G * seen_keys(a) * a->D;                 // of k and v
    return rows == 1 || (a->M == 1 && rows <= STEP_MOST && bytes > 32e6);
}

struct FwdPlan { bool step; RowPlan rows; size_t part, part2; };
FwdPlan fwd_plan(const qlka_softmax_args* a) {
    FwdPlan f{};
    f.step = steps(a);
    if (f.step) f.rows = {0, 0, step_splits((int64_t)a->B * a->G, ceil_div(seen_keys(a), 64))};
    else f.rows = row_plan(a, a->H, a->M, ceil_div(seen_keys(a), tile_rows(a)), 2, FWD_WAVES);
    if (f.rows.splits > 1) {
        const size_t rows = (size_t)f.rows.splits * a->B * a->H * a->M;
        f.part = align256(rows * sm_padded(a->D) * 4);
        f.part2 = align256(rows * 8);
    }
    return f;
}

struct BwdPlan {
    RowPlan dq, dkv;
    size_t delta, large, part, part2, table;
    size_t bytes() const { return delta + large + part + part2 + table; }
};
BwdPlan bwd_plan(const qlka_softmax_args* a, bool dq, bool dkv, bool table) {
    BwdPlan w{};
    const int t = tile_rows(a), DP = sm_padded(a->D);
    w.delta = align256((size_t)a->B * a->H * a->M * 4);
    w.large = align256((size_t)a->B * a->H * ceil_div(a->M, 32) * 4);
    if (dq || table) {
        w.dq = row_plan(a, a->H, a->M, ceil_div(seen_keys(a), t), 3, 0);
        if (w.dq.splits > 1) w.part = align256((size_t)w.dq.splits * a->B * a->H * a->M * DP * 4);
    }
    if (table)
        w.table = align256((size_t)a->H * a->B * w.dq.blocks * w.dq.splits * (a->num_borders + 1) *
                           (a->bidirectional ? 2 : 1) * 4);
    if (dkv) {
        w.dkv = row_plan(a, a->G, a->N, ceil_div(a->M, t) * (a->H / a->G), 5, 0);
        if (w.dkv.splits > 1) {
            w.part2 = align256((size_t)w.dkv.splits * a->B * a->G * a->N * DP * 4);
            w.part = std::max(w.part, w.part2);
        }
    }
    return w;
}

// ---- arguments to kernel parameters

SmStrides strides(const int64_t* s) { return {s[0], s[1], s[2]}; }

// Rows are read and written in pieces of 16 bytes, those of a tile at unsigned offsets from its first one.
int check_rows(const qlka_softmax_args* a, const char* name, const void* x, const int64_t* s, int heads, int rows) {
    const int64_t piece = a->dtype == QLKA_F32 ? 4 : 8;
    if (!x) return QLKA_OK;
    const int sizes[3] = {a->B, heads, rows};
    bool aligned = (uintptr_t)x % 16 == 0;
    for (int i = 0; i < 3; ++i) {
        if (sizes[i] <= 1) continue;
        if (s[i] < 0) return refuse("the strides of %s must not be negative", name);
        aligned = aligned && s[i] % piece == 0;
    }
    return aligned ? QLKA_OK : refuse("the rows of %s must be aligned to 16 bytes", name);
}

int params(const qlka_softmax_args* a, SmParams* p) {
    *p = SmParams{};
    p->q = a->q; p->k = a->k; p->v = a->v; p->g_out = a->g_out;
    p->out = a->out; p->out_full = a->out_full; p->table_kept = a->table_kept;
    p->g_q = a->g_q; p->g_k = a->g_k; p->g_v = a->g_v;
    p->sq = strides(a->q_stride); p->sk = strides(a->k_stride); p->sv = strides(a->v_stride);
    p->so = strides(a->out_stride); p->sg = strides(a->g_out_stride);
    p->sgq = strides(a->g_q_stride); p->sgk = strides(a->g_k_stride); p->sgv = strides(a->g_v_stride);
    p->keep = a->keep; p->keep_stride = a->keep_stride;
    p->table = a->table;
    p->log2_sum = a->lse;
    p->lse = a->log_sums;
    p->lse_low = a->log_sums ? a->log_sums + (int64_t)a->B * a->H * a->M : nullptr;
    p->lse_unit = 1.f;
    p->B = a->B; p->H = a->H; p->G = a->G; p->M = a->M; p->N = a->N; p->D = a->D;
    p->seen = seen_keys(a);
    p->causal = a->causal ? 1 : 0;
    p->start = a->start;
    p->splits = p->blocks = 1;
    // scores are held in units of the scale, so a scale of 0 goes into the sign
    p->scale = a->scale == 0.f ? 1.f : std::fabs(a->scale);
    p->q_sign = a->scale == 0.f ? 0.f : a->scale < 0.f ? -1.f : 1.f;
    const struct { const char* name; const void* x; const int64_t* s; int heads, rows; } all[] = {
        {"q", a->q, a->q_stride, a->H, a->M},          {"k", a->k, a->k_stride, a->G, a->N},
        {"v", a->v, a->v_stride, a->G, a->N},          {"out", a->out, a->out_stride, a->H, a->M},
        {"g_out", a->g_out, a->g_out_stride, a->H, a->M}, {"g_q", a->g_q, a->g_q_stride, a->H, a->M},
        {"g_k", a->g_k, a->g_k_stride, a->G, a->N},    {"g_v", a->g_v, a->g_v_stride, a->G, a->N}};
    for (const auto& o : all)
        if (int e = check_rows(a, o.name, o.x, o.s, o.heads, o.rows)) return e;
    if ((uintptr_t)a->out_full % 16) return refuse("out_full must be aligned to 16 bytes");
    return a->table ? check_buckets(a->border, a->num_borders, a->bidirectional, &p->bk) : QLKA_OK;
}

int need_ws(const void* ws, size_t have, size_t need) {
    if (need == 0) return QLKA_OK;
    if (ws && have >= need && (uintptr_t)ws % 16 == 0) return QLKA_OK;
    return api_error(QLKA_EWORKSPACE, "workspace too small, null or not aligned to 16 bytes");
}

// A launch takes less than 2^32 threads.
int fits_grid(int64_t groups, int threads) {
    if (groups <= (int64_t)UINT32_MAX / threads) return QLKA_OK;
    return refuse("too many workgroups: %lld of %d threads, a launch takes less than 2^32 threads", (long long)groups,
                  threads);
}
// a kernel of workgroups of 256 that takes `lanes` lanes a row
int fits_rows(int64_t rows, int lanes) { return fits_grid(ceil_div(rows * lanes, 256), 256); }

}  // namespace

extern "C" {

size_t qlka_softmax_fwd_ws_bytes(const qlka_softmax_args* a) {
    if (check_sizes(a)) return 0;
    const FwdPlan f = fwd_plan(a);
    return f.part + f.part2;
}

int qlka_softmax_fwd(const qlka_softmax_args* a, void* ws, size_t ws_bytes, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_sizes(a)) return e;
    SmParams p;
    if (int e = params(a, &p)) return e;
    if (a->B == 0 || a->M == 0) return QLKA_OK;
    if (!a->q || !a->out || (a->N > 0 && (!a->k || !a->v))) return refuse("q, k, v and out must be non-null");
    if (a->out_full && a->dtype == QLKA_F32) return refuse("out_full goes with QLKA_BF16");
    const FwdPlan f = fwd_plan(a);
    if (int e = need_ws(ws, ws_bytes, f.part + f.part2)) return e;
    const int64_t heads = (int64_t)a->B * (f.step ? a->G : a->H);
    if (int e = fits_grid(heads * std::max(f.rows.blocks, 1) * f.rows.splits, 64 * FWD_WAVES)) return e;
    if (f.rows.splits > 1)
        if (int e = fits_rows((int64_t)a->B * a->H * a->M, 64)) return e;
    hipStream_t st = (hipStream_t)stream;
    p.splits = f.rows.splits;
    p.blocks = f.rows.blocks;
    p.part = (float*)ws;
    p.part2 = (float*)((char*)ws + f.part);
    int e;
    if (f.step) {
        StageTimer timer("softmax_step", st);
        e = sm_step(a->dtype, p, st);
    } else {
        StageTimer timer("softmax_fwd", st);
        e = sm_fwd(a->dtype, p, st);
    }
    if (e || p.splits == 1) return status(e, "softmax attention");
    StageTimer timer("softmax_combine", st);
    return status(sm_combine(a->dtype, p, st), "softmax attention, joining of splits");
}

size_t qlka_softmax_bwd_ws_bytes(const qlka_softmax_args* a) {
    if (check_sizes(a) || (a->g_table && (a->num_borders < 0 || a->num_borders >= QLKA_MAX_BUCKETS))) return 0;
    const BwdPlan w = bwd_plan(a, a->g_q, a->g_k, a->g_table);
    return w.bytes();
}

int qlka_softmax_bwd(const qlka_softmax_args* a, void* ws, size_t ws_bytes, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_sizes(a)) return e;
    SmParams p;
    if (int e = params(a, &p)) return e;
    if (!a->g_k != !a->g_v) return refuse("g_k and g_v: both or neither");
    if (a->g_table && !a->table) return refuse("g_table needs the table");
    const bool rows = (int64_t)a->B * a->M > 0, keys = (int64_t)a->B * a->N > 0;
    if (rows && (!a->q || !a->out || (!a->lse && !a->log_sums) || !a->g_out))
        return refuse("q, out, lse or log_sums, and g_out must be non-null");
    if (!a->log_sums) {                                 // lse alone
        p.lse = a->lse;
        p.lse_unit = 0.5f;
    }
    if (keys && (!a->k || !a->v)) return refuse("k and v must be non-null");
    if (a->out_full && a->dtype == QLKA_F32) return refuse("out_full goes with QLKA_BF16");
    if (rows && a->g_table && a->dtype == QLKA_BF16 && !a->out_full)
        return refuse("g_table needs out_full with QLKA_BF16");
    const BwdPlan w = bwd_plan(a, a->g_q, a->g_k, a->g_table);
    if (int e = need_ws(ws, ws_bytes, w.bytes())) return e;
    const int64_t queries = (int64_t)a->B * a->H * a->M, kept = (int64_t)a->B * a->G * a->N;
    const int DP = sm_padded(a->D);
    if (int e = fits_grid((int64_t)a->B * a->H * w.dq.blocks * w.dq.splits, 64 * std::max(w.dq.waves, 1))) return e;
    if (int e = fits_grid((int64_t)a->B * a->G * w.dkv.blocks * w.dkv.splits, 64 * std::max(w.dkv.waves, 1))) return e;
    if (!a->g_q && !a->g_table)
        if (int e = fits_rows((int64_t)a->B * a->H * ceil_div(a->M, 32), 64)) return e;
    if (w.dq.splits > 1)
        if (int e = fits_rows(queries, DP / 4)) return e;
    if (w.dkv.splits > 1)
        if (int e = fits_rows(kept, DP / 4)) return e;
    if (a->g_table)
        if (int e = fits_grid(a->H, 256)) return e;
    hipStream_t st = (hipStream_t)stream;
    char* at = (char*)ws;
    p.delta = (float*)at; at += w.delta;
    p.large = (int*)at; at += w.large;
    p.part = (float*)at; at += w.part;
    p.part2 = (float*)at; at += w.part2;
    p.part_table = (float*)at;
    if (rows && !a->g_q && !a->g_table) {               // else softmax_dq leaves them
        StageTimer timer("softmax_delta", st);
        if (int e = sm_delta(a->dtype, p, st)) return status(e, "softmax attention backward, row sums");
    }
    if (!a->g_table) p.part_table = nullptr;
    if (rows && (a->g_q || a->g_table)) {
        p.splits = w.dq.splits;
        p.blocks = w.dq.blocks;
        {
            StageTimer timer("softmax_dq", st);
            if (int e = sm_dq(a->dtype, p, w.dq.waves, st)) return status(e, "softmax attention backward, queries");
        }
        if (p.splits > 1 && a->g_q) {
            StageTimer timer("softmax_sum", st);
            if (int e = sm_sum_parts(a->dtype, p.part, a->g_q, p.sgq, a->scale, p.splits, a->B, a->H, a->M,
                                     a->D, st))
                return status(e, "softmax attention backward, joining of splits");
        }
    }
    if (a->g_table) {
        StageTimer timer("softmax_table", st);
        const int count = rows ? a->B * w.dq.blocks * w.dq.splits : 0;
        if (int e = sm_sum_table(p.part_table, a->g_table, a->H, count, sm_buckets(p.bk), st))
            return status(e, "softmax attention backward, table");
    }
    if (keys && a->g_k) {
        p.splits = w.dkv.splits;
        p.blocks = w.dkv.blocks;
        {
            StageTimer timer("softmax_dkv", st);
            if (int e = sm_dkv(a->dtype, p, w.dkv.waves, st)) return status(e, "softmax attention backward, keys");
        }
        if (p.splits > 1) {
            StageTimer timer("softmax_sum", st);
            int e = sm_sum_parts(a->dtype, p.part, a->g_k, p.sgk, a->scale, p.splits, a->B, a->G, a->N, a->D, st);
            if (!e) e = sm_sum_parts(a->dtype, p.part2, a->g_v, p.sgv, 1.f, p.splits, a->B, a->G, a->N, a->D, st);
            if (e) return status(e, "softmax attention backward, joining of splits");
        }
    }
    return QLKA_OK;
}

static int check_map(int H, int M, int N, int start) {
    if (H < 1 || H > 65535) return refuse("H must be in [1, 65535]");
    if (M < 0 || N < 0 || M > 1 << 21 || N > 1 << 21) return refuse("M and N must be in [0, 2^21]");
    if (start > LONGEST || start < -LONGEST) return refuse("|start| must be <= 2^28");
    return QLKA_OK;
}

int qlka_bias_map_fwd(const float* table, const int* border, int num_borders, int bidirectional, float* out, int H,
                      int M, int N, int start, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_map(H, M, N, start)) return e;
    SmBuckets bk;
    if (int e = check_buckets(border, num_borders, bidirectional, &bk)) return e;
    if (M == 0 || N == 0) return QLKA_OK;
    if (!table || !out) return refuse("table and out must be non-null");
    StageTimer timer("bias_map", (hipStream_t)stream);
    return status(bias_map_fwd(table, bk, out, H, M, N, start, (hipStream_t)stream), "bias map");
}

size_t qlka_bias_map_bwd_ws_bytes(int num_borders, int bidirectional, int H, int M, int N) {
    if (check_map(H, M, N, 0) || num_borders < 0 || num_borders >= QLKA_MAX_BUCKETS || M == 0 || N == 0) return 0;
    return (size_t)H * bias_map_blocks(M, N) * (num_borders + 1) * (bidirectional ? 2 : 1) * 4;
}

int qlka_bias_map_bwd(const float* g, const int* border, int num_borders, int bidirectional, float* g_table, int H,
                      int M, int N, int start, void* ws, size_t ws_bytes, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_map(H, M, N, start)) return e;
    SmBuckets bk;
    if (int e = check_buckets(border, num_borders, bidirectional, &bk)) return e;
    const bool any = M > 0 && N > 0;
    if (!g_table || (any && !g)) return refuse("g and g_table must be non-null");
    if (int e = need_ws(ws, ws_bytes, qlka_bias_map_bwd_ws_bytes(num_borders, bidirectional, H, M, N))) return e;
    hipStream_t st = (hipStream_t)stream;
    if (any) {
        StageTimer timer("bias_map_bwd", st);
        if (int e = bias_map_bwd(g, bk, (float*)ws, H, M, N, start, st)) return status(e, "bias map backward");
    }
    StageTimer timer("softmax_table", st);
    return status(sm_sum_table((const float*)ws, g_table, H, any ? bias_map_blocks(M, N) : 0, sm_buckets(bk), st),
                  "bias map backward, table");
}

}  // extern "C"
