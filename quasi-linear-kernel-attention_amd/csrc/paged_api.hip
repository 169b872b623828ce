// The C ABI of the cache in pages and of attention over it (include/qlka.h): validation, the choice of kernels and
// splits, the workspace and the launches.
#include "api_checks.h"
#include "paged.h"
#include "segments.h"

using namespace qlka;

namespace {

bool coded(const qlka_paged_args* a) { return a->held == QLKA_INT8 || a->held == QLKA_E4M3; }
int held_size(const qlka_paged_args* a) { return coded(a) ? 1 : a->held == QLKA_F32 ? 4 : 2; }

int check_sizes(const qlka_paged_args* a) {
    if (!a) return refuse("args must be non-null");
    if (a->dtype != QLKA_F32 && a->dtype != QLKA_BF16) return refuse("dtype must be QLKA_F32 or QLKA_BF16");
    if (!coded(a) && a->held != a->dtype) return refuse("held must be dtype, QLKA_INT8 or QLKA_E4M3");
    if (a->B < 0 || a->T < 0 || a->N < 0 || a->H < 1 || a->G < 1)
        return refuse("B, T and N must be >= 0, H and G >= 1");
    if (a->H % a->G) return refuse("H must be a multiple of G");
    if (a->D < 8 || a->D > 128 || a->D % 8) return refuse("D must be a multiple of 8 in [8, 128]");
    if (a->T > LONGEST || a->B > LONGEST || a->N > LONGEST) return refuse("B, T and N must be <= 2^28");
    if (a->page_size < 1 || a->page_size > 1 << 16) return refuse("page_size must be in [1, 65536]");
    if (a->num_pages < 0 || a->table_len < 0) return refuse("num_pages and table_len must be >= 0");
    if (a->longest < 0) return refuse("longest must be >= 0");
    if ((double)a->H * a->T > (double)MOST_ROWS || (double)a->B * a->G * a->N > (double)MOST_ROWS)
        return refuse("H * T and B * G * N must fit int32");
    if (!a->offsets && a->T != a->B) return refuse("without offsets every sequence has one token: T must be B");
    return QLKA_OK;
}

// ---- how a call runs

// Sequences of up to so many rows a key head go through the step kernel, 16 at a time, others through the tiles. bf16
// rows come as fast to a tile (32 sequences of up to 16384 with 4 to 8 tokens, 12 / 4 heads: 45 us with 16, 57 with 32;
// 8 to 16 tokens: 59 and 55), others have to be taken apart or turned into bf16 (fp32, 4 sequences of up to 8000, 6 to
// 12 tokens: 24 us with 32, 39 with 16; e4m3, 12 / 12 heads, 12 to 24 tokens: 120 and 128).
int few_rows(const qlka_paged_args* a) { return a->held == QLKA_BF16 ? 16 : 32; }
// Workgroups of a launch: one round of those that registers and LDS leave room for.
// One a compute unit for fp32 rows of 128 where they are held so (96 KB of LDS) or go through tiles (372 to 388
// registers; tokens of 16 sequences of 2000 to 8192, 8 / 2 heads: 45 us, 65 with two; 8 heads 145 either way; 4 chunks
// of 256, 8 / 2 heads, fp32 115 and 119, int8 79 and 85; two of 200 among 16, fp32 86 and 100, int8 58 and 70).
bool one(const qlka_paged_args* a, bool tiles) {
    return a->dtype == QLKA_F32 && sm_padded(a->D) == 128 && (tiles || !coded(a));
}
// Two of other fp32 and of rows of 128 (tokens of 16 sequences of 2000 to 8192: 8 heads of 128, int8 41 us, 50 with
// 768, 47 with 1024; bf16 54, 57 with 1536; fp32, 12 heads of 64, 97, 107 with 768 or 1536; chunks of 512, 8 / 2 heads
// of 128, int8: 83, 91 with 768); three of bf16 rows of 64 (12 / 4 heads 20.7 us, 24.5 with 1536; 12 heads, cold pages,
// 50.4 and 51.5); four of 8 bits and of rows of 32 (12 heads of 64, int8: 31.1 us, 33.2 with 768). Beside tiles more
// and smaller ones fill what those leave (64 of up to 8192, 8 with chunks of 512, 12 heads of 64: bf16 162 us, 178 with
// one round; int8 146 and 160; 24 of 500 to 5000, fp32: 57, 60 with three rounds).
bool two(const qlka_paged_args* a) { return a->dtype == QLKA_F32 || sm_padded(a->D) == 128; }
int64_t step_groups(const qlka_paged_args* a, bool tiles) {
    if (one(a, tiles)) return 256;
    if (two(a)) return tiles ? 768 : 512;
    return tiles ? 1536 : coded(a) || sm_padded(a->D) == 32 ? 1024 : 768;
}
// Tiles alone: three a compute unit (4 chunks of 512 at up to 8192, int8, 12 / 4 heads: 68 us; 71 with two, 80 with
// six), beside tokens two, so that those have a third (32 sequences, two with chunks of 700: 46 us for 50).
int64_t tile_groups(const qlka_paged_args* a, bool step) { return one(a, true) ? 256 : two(a) || step ? 512 : 768; }
// The least positions of a part: a turn of the step kernel's waves (one sequence of 2000, int8, 12 / 4 heads: 9.3 us;
// 10.6 with 256, 17.4 as one), a few tiles of the others (300 tokens of it: 20.1 us; 24.4 with 128, 23.2 with 512). A
// call whose tables have no room for more than so many positions is not cut at all, which saves joining (one sequence
// of 250: 7.0 us for 9.3; of 500: 9.2 either way).
constexpr int64_t STEP_LEAST = 128, TILE_LEAST = 256, STEP_WHOLE = 512, TILE_WHOLE = 256;

// The units of more sequences than a workgroup looks up by itself are found once, by a kernel before the others (512 of
// 100 to 1000, 12 / 4 heads, bf16: 52 us for 57; 2000 of 100 to 500, int8: 106 for 278; but 256: 36 for 34).
bool many(const qlka_paged_args* a) { return a->B > PG_LOOKED_UP; }

struct Plan {
    bool step, tiles, join;
    int few;
    PgUnits units[2];                        // step, tiles
    size_t part[2], part2[2], table[2];
    size_t bytes() const { return part[0] + part2[0] + part[1] + part2[1] + table[0] + table[1]; }
};
Plan plan(const qlka_paged_args* a) {
    Plan r{};
    const int64_t share = a->H / a->G;
    const int64_t longest = !a->offsets ? 1 : a->longest ? std::min(a->longest, a->T) : a->T;
    const int few = few_rows(a);
    r.step = r.tiles = true;
    r.few = few;
    if (!a->offsets || longest * share <= few) {
        r.tiles = false;
        r.few = INT32_MAX;
    } else if (a->T * share >= 256 * std::max<int64_t>(a->B, 1)) {
        // Chunks, on the average: tiles alone, for tokens among them too. Measured both ways, bf16, one chunk among
        // tokens at up to 8192, tiles alone and both kinds: the average is not what tells which is faster. 12 / 4
        // heads, 2800 and 31 tokens: 90 and 60 us; 700 and 7: 55 and 51; 2048 and 7: 38 and 42; 4096 and 15: 82 and
        // 102; 12 heads, 2048 and 7: 133 and 108; 4096 and 15: 130 and 106. (int8: 106 and 65, 65 and 55, 45 and 48, 98
        // and 122, 155 and 133, 165 and 131.)
        r.step = false;
        r.few = -1;
    }
    const int64_t places = std::min<int64_t>((int64_t)a->table_len * a->page_size, LONGEST);
    const int DP = sm_padded(a->D);
    const struct { bool used; int rows; int64_t groups, least, whole; } kernels[2] = {
        {r.step, PG_STEP_ROWS, step_groups(a, r.tiles), STEP_LEAST, STEP_WHOLE},
        {r.tiles, PG_TILE_ROWS, tile_groups(a, r.step), TILE_LEAST, TILE_WHOLE}};
    for (int i = 0; i < 2; ++i) {
        const auto& k = kernels[i];
        if (!k.used) continue;
        // Sequences that have rows here, at most: of the tiles' beside the step kernel's each has more than `few` rows.
        // (A chunk of 512 among 1999 tokens, 12 heads of 64: 173 MiB of workspace, 889 with a block for each of them;
        // among 999: 360 us for 371.)
        const int64_t tokens = i == 1 && r.step ? few / share + 1 : 1;
        const int64_t sequences = std::min<int64_t>(a->B, a->T / tokens);
        // blocks of rows a key head: each of them has one that is not full at most, and more in the step kernel only
        // where it is alone
        int64_t blocks = a->T * share / k.rows + sequences;
        if (i == 0 && r.tiles) blocks = std::min<int64_t>(blocks, sequences * (few / PG_STEP_ROWS));
        // a sequence's last part is shorter than the others: room for those within the round of workgroups
        const int64_t last = a->G * (i == 0 ? sequences : blocks) / 2;
        const int64_t aim = std::max<int64_t>(std::max(k.groups - last, k.groups / 2) / a->G, 1);
        const bool parts = places > k.whole;
        const int64_t units = (blocks + (parts ? aim + 1 : 0)) * a->G;          // the sum of parts rounded up
        PgUnits& u = r.units[i];
        u.aim = (float)aim;
        u.least = parts ? (int)k.least : (int)LONGEST;
        u.room = units;
        u.groups = (int)std::min<int64_t>(ceil_div(units, 8) * 8, INT32_MAX);
        if (many(a)) r.table[i] = align256(((size_t)a->B + 2) * 4);
        if (parts) {
            r.join = true;
            r.part[i] = align256((size_t)units * k.rows * DP * 4);
            r.part2[i] = align256((size_t)units * k.rows * 8);
        }
    }
    return r;
}

// ---- arguments to kernel parameters

PgStrides page_strides(const int64_t* s, int size) {
    return {(uint32_t)(s[0] * size), (uint32_t)(s[1] * size), (uint32_t)(s[2] * size)};
}
PgOut strides2(const int64_t* s) { return {0, s[0], s[1]}; }
PgOut strides3(const int64_t* s) { return {s[0], s[1], s[2]}; }

// The cache and where the sequences are in it.
int params(const qlka_paged_args* a, PgParams* p) {
    *p = PgParams{};
    p->k_pages = (char*)a->k_pages; p->v_pages = (char*)a->v_pages;
    p->sk = page_strides(a->k_pages_stride, held_size(a)); p->sv = page_strides(a->v_pages_stride, held_size(a));
    p->k_exp = a->k_exp; p->v_exp = a->v_exp;
    p->ske = page_strides(a->k_exp_stride, 1); p->sve = page_strides(a->v_exp_stride, 1);
    p->tables = a->tables; p->lengths = a->lengths; p->offsets = a->offsets;
    p->table_stride = a->table_stride;
    p->B = a->B; p->H = a->H; p->G = a->G; p->T = a->T; p->D = a->D; p->N = a->N;
    p->page_size = a->page_size; p->num_pages = a->num_pages; p->table_len = a->table_len;
    p->places = (int)std::min<int64_t>((int64_t)a->table_len * a->page_size, LONGEST);
    p->page_division = pg::division_by(a->page_size);
    p->blocks = 1;
    const int64_t sizes[3] = {a->num_pages, a->G, a->page_size};
    const struct { const char* name; const void* x; const int64_t* s; } pages[] = {
        {"k_pages", a->k_pages, a->k_pages_stride}, {"v_pages", a->v_pages, a->v_pages_stride}};
    const int64_t unit = coded(a) && a->D % 16 ? 8 : 16;
    for (const auto& o : pages) {
        if (a->num_pages && !o.x) return refuse("%s must be non-null", o.name);
        bool aligned = (uintptr_t)o.x % unit == 0;
        for (int i = 0; i < 3; ++i) {
            if (sizes[i] <= 1) continue;
            if (o.s[i] < 0 || o.s[i] > UINT32_MAX / held_size(a))
                return refuse("the strides of %s must be in [0, 2^32) bytes", o.name);
            aligned = aligned && o.s[i] * held_size(a) % unit == 0;
        }
        if (!aligned) return refuse("the rows of %s must be aligned to %d bytes", o.name, (int)unit);
    }
    if (coded(a) && a->num_pages) {
        if (!a->k_exp || !a->v_exp) return refuse("k_exp and v_exp must be non-null where 8 bits are held");
        for (int i = 0; i < 3; ++i)
            if (sizes[i] > 1 &&
                ((uint64_t)a->k_exp_stride[i] > UINT32_MAX || (uint64_t)a->v_exp_stride[i] > UINT32_MAX))
                return refuse("the strides of k_exp and v_exp must be in [0, 2^32)");
    }
    if (a->B > 0 && (!a->lengths || (a->table_len > 0 && !a->tables)))
        return refuse("tables and lengths must be non-null");
    if (a->B > 1 && a->table_stride < 0) return refuse("table_stride must not be negative");
    return QLKA_OK;
}

int rows_of(const qlka_paged_args* a, const char* name, const void* x, const int64_t* s, int heads) {
    const int64_t sizes[2] = {heads, a->T};
    return check_rows(name, x, s, sizes, 2, a->dtype == QLKA_F32 ? 4 : 2);
}

}  // namespace

extern "C" {

int qlka_paged_write(const qlka_paged_args* a, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_sizes(a)) return e;
    PgParams p;
    if (int e = params(a, &p)) return e;
    if (int e = rows_of(a, "k", a->k, a->k_stride, a->G)) return e;
    if (int e = rows_of(a, "v", a->v, a->v_stride, a->G)) return e;
    if (a->T == 0 || a->B == 0 || p.places == 0 || a->num_pages == 0) return QLKA_OK;
    if (!a->k || !a->v) return refuse("k and v must be non-null");
    if (int e = fits_grid(ceil_div(a->T, 4), 256)) return e;
    p.k = a->k; p.v = a->v;
    p.snk = strides2(a->k_stride); p.snv = strides2(a->v_stride);
    hipStream_t st = (hipStream_t)stream;
    StageTimer timer("paged_write", st);
    return status(pg_write(a->dtype, a->held, p, st), "writing to pages");
}

int qlka_paged_read(const qlka_paged_args* a, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_sizes(a)) return e;
    PgParams p;
    if (int e = params(a, &p)) return e;
    const int64_t sizes[3] = {a->B, a->G, a->N};
    if (int e = check_rows("out_k", a->out_k, a->out_k_stride, sizes, 3, a->dtype == QLKA_F32 ? 4 : 2)) return e;
    if (int e = check_rows("out_v", a->out_v, a->out_v_stride, sizes, 3, a->dtype == QLKA_F32 ? 4 : 2)) return e;
    if (a->B == 0 || a->N == 0) return QLKA_OK;
    if (!a->out_k || !a->out_v) return refuse("out_k and out_v must be non-null");
    p.out_k = a->out_k; p.out_v = a->out_v;
    p.sok = strides3(a->out_k_stride); p.sov = strides3(a->out_v_stride);
    p.blocks = (int)ceil_div(a->N, 256 / (sm_padded(a->D) / 8) * PG_READ_ROWS);
    if (int e = fits_grid((int64_t)a->B * a->G * p.blocks, 256)) return e;
    hipStream_t st = (hipStream_t)stream;
    StageTimer timer("paged_read", st);
    return status(pg_read(a->dtype, a->held, p, st), "reading pages");
}

size_t qlka_paged_attention_ws_bytes(const qlka_paged_args* a) {
    if (check_sizes(a) || check_scale(a->scale)) return 0;
    const Plan r = plan(a);
    return r.bytes();
}

int qlka_paged_attention(const qlka_paged_args* a, void* ws, size_t ws_bytes, void* stream) {
    api_error(QLKA_OK, "");
    if (int e = check_sizes(a)) return e;
    if (int e = check_scale(a->scale)) return e;
    PgParams p;
    if (int e = params(a, &p)) return e;
    if (int e = rows_of(a, "q", a->q, a->q_stride, a->H)) return e;
    if (int e = rows_of(a, "out", a->out, a->out_stride, a->H)) return e;
    if (a->T == 0) return QLKA_OK;
    if (!a->q || !a->out) return refuse("q and out must be non-null");
    const Plan r = plan(a);
    if (int e = need_ws(ws, ws_bytes, r.bytes())) return e;
    if (int e = fits_grid((int64_t)r.units[0].groups + r.units[1].groups + 16, 256)) return e;
    if (r.join)
        if (int e = fits_rows((int64_t)a->H * a->T, 64)) return e;
    p.q = a->q; p.out = a->out;
    p.sq = strides2(a->q_stride); p.so = strides2(a->out_stride);
    p.scale = a->scale == 0.f ? 1.f : std::fabs(a->scale);
    p.q_sign = a->scale == 0.f ? 0.f : a->scale < 0.f ? -1.f : 1.f;
    p.few = r.few;
    p.step = r.units[0];
    p.tiles = r.units[1];
    char* at = (char*)ws;
    p.step.part = (float*)at; at += r.part[0];
    p.step.part2 = (float*)at; at += r.part2[0];
    p.tiles.part = (float*)at; at += r.part[1];
    p.tiles.part2 = (float*)at; at += r.part2[1];
    if (r.table[0]) p.step.table = (int*)at;
    at += r.table[0];
    if (r.table[1]) p.tiles.table = (int*)at;
    hipStream_t st = (hipStream_t)stream;
    if (many(a)) {
        StageTimer timer("paged_table", st);
        if (int e = pg_table(p, st)) return status(e, "attention over pages, units");
    }
    {
        StageTimer timer("paged_attend", st);
        const int e = a->dtype == QLKA_BF16 ? pg_attend_bf16(a->held, p, st) : pg_attend_f32(a->held, p, st);
        if (e) return status(e, "attention over pages");
    }
    if (!r.join) return QLKA_OK;
    StageTimer timer("paged_join", st);
    return status(pg_join(a->dtype, p, st), "attention over pages, joining of parts");
}

}  // extern "C"
