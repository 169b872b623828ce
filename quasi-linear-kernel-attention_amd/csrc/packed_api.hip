// The C ABI of attention within packed sequences (include/qlka.h): validation, blocks and splits, the workspace and the
// launches of softmax_fwd.hip's and softmax_bwd.hip's kernels over one sequence's rows a workgroup (segments.h).
#include "api_checks.h"
#include "segments.h"

using namespace qlka;

namespace {

int check_sizes(const qlka_packed_args* a) {
    if (!a) return refuse("args must be non-null");
    if (a->dtype != QLKA_F32 && a->dtype != QLKA_BF16) return refuse("dtype must be QLKA_F32 or QLKA_BF16");
    if (a->B < 0 || a->T < 0 || a->H < 1 || a->G < 1) return refuse("B and T must be >= 0, H and G >= 1");
    if (a->H % a->G) return refuse("H must be a multiple of G");
    if (a->D < 8 || a->D > 128 || a->D % 8) return refuse("D must be a multiple of 8 in [8, 128]");
    if (a->T > LONGEST || a->B > LONGEST) return refuse("B and T must be <= 2^28");
    if ((double)a->H * a->T > (double)MOST_ROWS) return refuse("H * T must fit int32");
    return check_scale(a->scale);
}

// ---- how a call runs

int tile_rows(const qlka_packed_args* a) { return sm_tile_rows(a->dtype == QLKA_F32 ? 3 : 1, sm_padded(a->D)); }
// The host does not know the lengths: waves go by the average one, and splits by twice that, since the longest
// sequence's workgroups are what a call waits for (64 sequences of 65 to 600, fp32 training: 313 us by the average, 273
// by twice or three times that; calls of many workgroups are not split either way). Lengths far from the average are
// not served well (12 heads of 64, causal, bf16 / fp32): one of 4096 among 300 of 10 takes 136 / 519 us, 381 / 1729
// with the gradients (alone 70 / 271, 265 / 970), since its blocks are of one wave or two and not in the order of their
// work; four of 2048 with 300 empty sequences 111 / 400 and 291 / 1290 (without those 46 / 167, 181 / 849).
int64_t average(const qlka_packed_args* a) { return ceil_div(a->T, std::max(a->B, 1)); }
int64_t longest(const qlka_packed_args* a) { return std::min<int64_t>(2 * average(a), a->T); }

struct Plan { int waves, blocks, splits; };
// Workgroups of `few` waves where sequences have no rows for more, unless they are less than the GPU has room for at
// once (two a compute unit, one of fp32 rows of 128): then waves without rows help to bring the others' (fp32 training,
// 12 heads of 64 of 8 to 30 rows: 16 sequences 27 us with all waves, 30 with few; 64: 52 and 46; 1000: 641 and 475; 12
// heads of 80 of 30 to 60 rows: 16 sequences 58 and 65, 25 111 and 88).
Plan plan(const qlka_packed_args* a, int heads, int64_t tiles, double products, int few) {
    Plan r;
    const int64_t room = a->dtype == QLKA_F32 && sm_padded(a->D) == 128 ? 256 : 512;
    const bool small = average(a) <= 32 * few && (int64_t)heads * a->B > room;
    r.waves = small ? few : FWD_WAVES;
    r.blocks = (int)segment_blocks(a->T, a->B, 32 * r.waves);
    const int DP = sm_padded(a->D);
    const double tile_us = products * 0.3 * DP / 64 * (a->dtype == QLKA_F32 ? 2 : 1);
    r.splits = splits_for((int64_t)heads * r.blocks, tiles, tile_us, (double)heads * a->T * DP * 8);
    return r;
}
Plan fwd_plan(const qlka_packed_args* a) {
    return plan(a, a->H, ceil_div(longest(a), tile_rows(a)), 2, 1);
}
size_t part_bytes(const qlka_packed_args* a, const Plan& p, int heads) {
    return p.splits > 1 ? align256((size_t)p.splits * heads * a->T * sm_padded(a->D) * 4) : 0;
}
size_t part2_bytes(const qlka_packed_args* a, const Plan& p) {
    return p.splits > 1 ? align256((size_t)p.splits * a->H * a->T * 8) : 0;
}

struct BwdPlan {
    Plan dq, dkv;
    size_t delta, large, part, part2;
    size_t bytes() const { return delta + large + part + part2; }
};
int groups(const qlka_packed_args* a) { return (int)segment_blocks(a->T, a->B, 32); }
BwdPlan bwd_plan(const qlka_packed_args* a) {
    BwdPlan w{};
    const int t = tile_rows(a);
    w.delta = align256((size_t)a->H * a->T * 4);
    w.large = align256((size_t)a->H * groups(a) * 4);
    w.dq = plan(a, a->H, ceil_div(longest(a), t), 3, 2);
    w.dkv = plan(a, a->G, ceil_div(longest(a), t) * (a->H / a->G), 5, 2);
    w.part2 = part_bytes(a, w.dkv, a->G);
    w.part = std::max(part_bytes(a, w.dq, a->H), w.part2);
    return w;
}

// ---- arguments to kernel parameters

SmStrides strides(const int64_t* s) { return {0, s[0], s[1]}; }

int params(const qlka_packed_args* a, SmParams* p) {
    *p = SmParams{};
    p->q = a->q; p->k = a->k; p->v = a->v; p->g_out = a->g_out;
    p->out = a->out; p->out_full = a->out_full;
    p->g_q = a->g_q; p->g_k = a->g_k; p->g_v = a->g_v;
    p->sq = strides(a->q_stride); p->sk = strides(a->k_stride); p->sv = strides(a->v_stride);
    p->so = strides(a->out_stride); p->sg = strides(a->g_out_stride);
    p->sgq = strides(a->g_q_stride); p->sgk = strides(a->g_k_stride); p->sgv = strides(a->g_v_stride);
    p->lse = a->log_sums;
    p->lse_low = a->log_sums ? a->log_sums + (int64_t)a->H * a->T : nullptr;
    p->lse_unit = 1.f;
    p->B = 1; p->H = a->H; p->G = a->G; p->M = p->N = p->seen = a->T; p->D = a->D;
    p->causal = a->causal ? 1 : 0;
    p->splits = p->blocks = 1;
    p->scale = a->scale == 0.f ? 1.f : std::fabs(a->scale);
    p->q_sign = a->scale == 0.f ? 0.f : a->scale < 0.f ? -1.f : 1.f;
    p->offsets = a->offsets;
    p->sequences = a->B;
    p->groups = groups(a);
    const struct { const char* name; const void* x; const int64_t* s; int heads; } all[] = {
        {"q", a->q, a->q_stride, a->H},       {"k", a->k, a->k_stride, a->G},
        {"v", a->v, a->v_stride, a->G},       {"out", a->out, a->out_stride, a->H},
        {"g_out", a->g_out, a->g_out_stride, a->H}, {"g_q", a->g_q, a->g_q_stride, a->H},
        {"g_k", a->g_k, a->g_k_stride, a->G}, {"g_v", a->g_v, a->g_v_stride, a->G}};
    for (const auto& o : all) {
        const int64_t sizes[2] = {o.heads, a->T};
        if (int e = check_rows(o.name, o.x, o.s, sizes, 2, a->dtype == QLKA_F32 ? 4 : 2)) return e;
    }
    if ((uintptr_t)a->out_full % 16) return refuse("out_full must be aligned to 16 bytes");
    if (a->out_full && a->dtype == QLKA_F32) return refuse("out_full goes with QLKA_BF16");
    if (!a->offsets) return refuse("offsets must be non-null");
    return QLKA_OK;
}

}  // namespace

extern "C" {

size_t qlka_packed_fwd_ws_bytes(const qlka_packed_args* a) {
    if (check_sizes(a)) return 0;
    const Plan f = fwd_plan(a);
    return part_bytes(a, f, a->H) + part2_bytes(a, f);
}

int qlka_packed_fwd(const qlka_packed_args* a, void* ws, size_t ws_bytes, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_sizes(a)) return e;
    SmParams p;
    if (int e = params(a, &p)) return e;
    if (a->T == 0) return QLKA_OK;
    if (!a->q || !a->k || !a->v || !a->out) return refuse("q, k, v and out must be non-null");
    const Plan f = fwd_plan(a);
    const size_t part = part_bytes(a, f, a->H);
    if (int e = need_ws(ws, ws_bytes, part + part2_bytes(a, f))) return e;
    if (int e = fits_grid((int64_t)a->H * f.blocks * f.splits, 64 * f.waves)) return e;
    if (f.splits > 1)
        if (int e = fits_rows((int64_t)a->H * a->T, 64)) return e;
    hipStream_t st = (hipStream_t)stream;
    p.splits = f.splits;
    p.blocks = f.blocks;
    p.part = (float*)ws;
    p.part2 = (float*)((char*)ws + part);
    {
        StageTimer timer("packed_fwd", st);
        const int e = sm_packed_fwd(a->dtype, p, f.waves, st);
        if (e || f.splits == 1) return status(e, "packed attention");
    }
    StageTimer timer("softmax_combine", st);
    return status(sm_combine(a->dtype, p, st), "packed attention, joining of splits");
}

size_t qlka_packed_bwd_ws_bytes(const qlka_packed_args* a) { return check_sizes(a) ? 0 : bwd_plan(a).bytes(); }

int qlka_packed_bwd(const qlka_packed_args* a, void* ws, size_t ws_bytes, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_sizes(a)) return e;
    SmParams p;
    if (int e = params(a, &p)) return e;
    if (!a->g_k != !a->g_v) return refuse("g_k and g_v: both or neither");
    if (a->T == 0) return QLKA_OK;
    if (!a->q || !a->k || !a->v || !a->out || !a->log_sums || !a->g_out)
        return refuse("q, k, v, out, log_sums and g_out must be non-null");
    const BwdPlan w = bwd_plan(a);
    if (int e = need_ws(ws, ws_bytes, w.bytes())) return e;
    const int64_t queries = (int64_t)a->H * a->T, kept = (int64_t)a->G * a->T;
    const int DP = sm_padded(a->D);
    if (int e = fits_grid((int64_t)a->H * w.dq.blocks * w.dq.splits, 64 * w.dq.waves)) return e;
    if (int e = fits_grid((int64_t)a->G * w.dkv.blocks * w.dkv.splits, 64 * w.dkv.waves)) return e;
    if (w.dq.splits > 1)
        if (int e = fits_rows(queries, DP / 4)) return e;
    if (w.dkv.splits > 1)
        if (int e = fits_rows(kept, DP / 4)) return e;
    hipStream_t st = (hipStream_t)stream;
    char* at = (char*)ws;
    p.delta = (float*)at; at += w.delta;
    p.large = (int*)at; at += w.large;
    p.part = (float*)at; at += w.part;
    p.part2 = (float*)at;
    p.splits = w.dq.splits;
    p.blocks = w.dq.blocks;
    {   // also for g_q null: softmax_dkv reads the row sums that it leaves
        StageTimer timer("packed_dq", st);
        if (int e = sm_packed_dq(a->dtype, p, w.dq.waves, st)) return status(e, "packed attention backward, queries");
    }
    if (p.splits > 1 && a->g_q) {
        StageTimer timer("softmax_sum", st);
        if (int e = sm_sum_parts(a->dtype, p.part, a->g_q, p.sgq, a->scale, p.splits, 1, a->H, a->T, a->D, st))
            return status(e, "packed attention backward, joining of splits");
    }
    if (!a->g_k) return QLKA_OK;
    p.splits = w.dkv.splits;
    p.blocks = w.dkv.blocks;
    {
        StageTimer timer("packed_dkv", st);
        if (int e = sm_packed_dkv(a->dtype, p, w.dkv.waves, st)) return status(e, "packed attention backward, keys");
    }
    if (p.splits == 1) return QLKA_OK;
    StageTimer timer("softmax_sum", st);
    int e = sm_sum_parts(a->dtype, p.part, a->g_k, p.sgk, a->scale, p.splits, 1, a->G, a->T, a->D, st);
    if (!e) e = sm_sum_parts(a->dtype, p.part2, a->g_v, p.sgv, 1.f, p.splits, 1, a->G, a->T, a->D, st);
    return status(e, "packed attention backward, joining of splits");
}

}  // extern "C"
