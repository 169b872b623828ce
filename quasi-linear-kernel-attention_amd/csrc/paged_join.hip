// Attention over pages: the sums of a row's parts (paged_device.h, Units) to the row.
#include "paged_device.h"

namespace qlka {
namespace pg {

// Adds up the parts of rows whose positions are more than one. A wave takes a row (MANY: 256 / DP rows of a token,
// since finding the sequence costs as much as a row): its lanes look at the parts' references and sums, one each, then
// DP / 4 lanes take a part's sums. Bound by latency: launch, sequence, sums (192 rows: 4.5 us; 19548 rows of 2 to 7
// parts: 7.8 us, 20 with a wave a row; of 9 parts 10.2 us, 13.3 where 8 were waited for before the ninth was asked
// for).
template <class T, int DP, bool MANY> __global__ __launch_bounds__(256) void paged_join(const PgParams p) {
    constexpr int LANES = DP / 4, GROUPS = 64 / LANES;                 // lanes of a part's row
    constexpr int LOOK = MANY ? LANES : 64, AT_ONCE = MANY ? 1 : GROUPS;
    const int lane = threadIdx.x & 63, share = p.H / p.G, i = lane % LANES, group = lane / LANES;
    const uint32_t w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const uint32_t turns = MANY ? (p.H + GROUPS - 1) / GROUPS : p.H;
    const int t = (int)(w / turns), head0 = (int)(w % turns) * (MANY ? GROUPS : 1);
    if (t >= p.T) return;
    // the sequence, looked up together with what its units are found from
    const Tokens mine = tokens_of_lane(p);
    const Found found = find(p, t, mine);
    if (found.b < 0) return;
    const int b = found.b;
    const Tokens seq = found.tokens;
    int span, before, blocks, parts;         // of the sequence: units a key head before it, its blocks and parts
    const bool step = seq.rows * share <= p.few;
    const auto look_up = [&](const auto& units) {
        const Cut c = units.cut(units.held(b, seq));
        span = c.span;
        before = units.upto(b);
        blocks = c.blocks;
        parts = c.parts;
    };
    if (step) look_up(Units<true, PG_STEP_ROWS>(p, p.step, mine));
    else look_up(Units<false, PG_TILE_ROWS>(p, p.tiles, mine));
    if (parts == 1) return;
    const int size = step ? PG_STEP_ROWS : PG_TILE_ROWS;
    const PgUnits& u = step ? p.step : p.tiles;
    const int seen = seen_from(p, seq.start + t - seq.first);
    parts = max(1, (seen + span - 1) / span);                          // that this token sees
    const int64_t next = (int64_t)p.G * blocks, apart = next * size;   // units and rows from a part to the next

    const int head = MANY ? min(head0 + group, p.H - 1) : head0, kvh = head / share;
    const int r = (t - seq.first) * share + head % share;
    const int64_t unit = (int64_t)before * p.G + (int64_t)kvh * blocks + r / size;         // of part 0
    if (unit < 0 || unit + (parts - 1) * next >= u.room) return;  // offsets that decrease
    const int64_t row = unit * size + r % size;
    float ref = LOW, sum = 0.f;
    f32x4 x = {};
    // parts s0 to s0 + LOOK - 1, of which the first `early` of a group of lanes are on their way before their weights
    // are known
    const auto add = [&](int s0, auto early) {
        constexpr int EARLY = decltype(early)::value;
        const int look = s0 + (MANY ? i : lane), count = min(LOOK, parts - s0), first = MANY ? 0 : group;
        float2 a = {LOW, 0.f};
        if (look < parts) a = *reinterpret_cast<const float2*>(u.part2 + 2 * (look * apart + row));
        f32x4 y[EARLY];
        const auto from = [&](int s) {
            return *reinterpret_cast<const f32x4*>(u.part + ((s0 + min(s, count - 1)) * apart + row) * DP + 4 * i);
        };
#pragma unroll
        for (int e = 0; e < EARLY; ++e) y[e] = from(first + e * AT_ONCE);
        if (a.y == 0.f) a.x = LOW;                                      // no key there
        float top = a.x;
#pragma unroll
        for (int far = 1; far < LOOK; far *= 2) top = fmaxf(top, __shfl_xor(top, far));
        top = fmaxf(top, ref);
        const float to = top == LOW ? 0.f : top, was = sm::exp_of(ref - to), f = sm::exp_of(a.x - to);
        ref = top;
        sum = sum * was + a.y * f;
        x = x * was;
        const auto weight = [&](int s) { return __shfl(f, MANY ? group * LANES + s % LANES : s & 63); };
#pragma unroll
        for (int e = 0; e < EARLY; ++e) {
            const int s = first + e * AT_ONCE;
            const float z = weight(s);
            if (s < count) x = x + y[e] * z;
        }
        // (all lanes go on to the last part: the one that holds its weight may have none left itself)
        for (int e = EARLY; e * AT_ONCE < count; ++e) {
            const int s = first + e * AT_ONCE;
            const float z = weight(s);
            if (s < count) x = x + from(s) * z;
        }
    };
#pragma unroll 1
    for (int s0 = 0; s0 < parts; s0 += LOOK) {
        const int count = min(LOOK, parts - s0);
        if (count <= 4 * AT_ONCE) add(s0, std::integral_constant<int, 4>());
        else if (count <= 8 * AT_ONCE) add(s0, std::integral_constant<int, 8>());
        else add(s0, std::integral_constant<int, 16 * AT_ONCE <= LOOK ? 16 : LOOK / AT_ONCE>());
    }
#pragma unroll
    for (int far = 1; far < LOOK; far *= 2) sum += __shfl_xor(sum, far);
    if constexpr (!MANY) {
#pragma unroll
        for (int far = LANES; far < 64; far *= 2)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], far);
    }
    if (MANY ? head0 + group < p.H : group == 0)
        sm::store4((T*)p.out + head * p.so.h + t * p.so.r, 4 * i, p.D, x * (sum == 0.f ? 0.f : 1.f / sum));
}
constexpr int64_t JOIN_MANY = 4096;          // rows

// The units before each of the sequences, of all, and the span: B + 2 numbers for each kind of units, of which each has
// a workgroup.
constexpr int TABLE_THREADS = 1024;
template <class U> __device__ __forceinline__ void fill_table(const PgParams& p, const PgUnits& u, U units, int* sums,
                                                              float* works) {
    const int tid = threadIdx.x, wave = tid >> 6;
    double mine = 0;                         // (of a million sequences floats would lose what the span has to spare)
    for (int b = tid; b < p.B; b += TABLE_THREADS) {
        const auto h = units.held(b, tokens_of(p, b));
        mine += (double)h.blocks * h.seen;
    }
    float work = last_lane(sums_upto((float)mine));
    if ((tid & 63) == 0) works[wave] = work;
    __syncthreads();
    work = 0.f;
    for (int w = 0; w < TABLE_THREADS / 64; ++w) work += works[w];
    units.set_span(work);
    int base = 0;
    for (int b0 = 0; b0 < p.B; b0 += TABLE_THREADS) {
        const int b = b0 + tid;
        int n = 0;
        if (b < p.B) {
            const Cut c = units.cut(units.held(b, tokens_of(p, b)));
            n = c.blocks * c.parts;
        }
        int to = sums_upto(n);
        if ((tid & 63) == 63) sums[wave] = to;
        __syncthreads();
        for (int w = 0; w < wave; ++w) to += sums[w];
        if (b < p.B) u.table[b] = base + to - n;
        for (int w = 0; w < TABLE_THREADS / 64; ++w) base += sums[w];
        __syncthreads();
    }
    if (tid == 0) {
        u.table[p.B] = base;
        u.table[p.B + 1] = units.span;
    }
}
__global__ __launch_bounds__(TABLE_THREADS) void paged_table(const PgParams p) {
    __shared__ int sums[TABLE_THREADS / 64];
    __shared__ float works[TABLE_THREADS / 64];
    if (blockIdx.x == 0 && p.step.groups)
        fill_table(p, p.step, Units<true, PG_STEP_ROWS>(p, p.step, 0), sums, works);
    if (blockIdx.x == 1 && p.tiles.groups)
        fill_table(p, p.tiles, Units<false, PG_TILE_ROWS>(p, p.tiles, 0), sums, works);
}

}  // namespace pg

int pg_table(const PgParams& p, hipStream_t st) {
    pg::paged_table<<<2, pg::TABLE_THREADS, 0, st>>>(p);
    return (int)hipGetLastError();
}

int pg_join(int dtype, const PgParams& p, hipStream_t st) {
    return sm::dispatch(dtype, p.D, [&](auto t, auto dp) {
        const int64_t rows = (int64_t)p.T * p.H, at_once = 256 / dp.value;
        const int64_t waves = p.T * ((p.H + at_once - 1) / at_once);
        if (rows >= pg::JOIN_MANY)
            pg::paged_join<decltype(t), dp.value, true><<<dim3((unsigned)((waves + 3) / 4)), 256, 0, st>>>(p);
        else
            pg::paged_join<decltype(t), dp.value, false><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, st>>>(p);
        return (int)hipGetLastError(); });
}

}  // namespace qlka
