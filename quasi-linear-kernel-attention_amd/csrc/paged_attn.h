// Attention of new tokens over a cache in pages: the kernels. A launch has workgroups for sequences of few rows
// (paged_step.h), for chunks (paged_tiles.h), or for both: a batch of chunks and tokens is one launch, in which the one
// kind fills the compute units that the other leaves (32 sequences of 12 / 4 heads, two with chunks: 66 us one after
// the other, 54 in one launch). The last workgroups write the rows outside every sequence.
#pragma once

#include "paged_step.h"
#include "paged_tiles.h"

namespace qlka {
namespace pg {

template <class T, class C, int DP, int EL, bool STEP, bool TILES> constexpr int room() {
    constexpr int AS_STEP = step_room<T, C, DP>(), AS_TILES = tiles_room<T, C, DP>();
    return STEP && TILES ? (AS_STEP < AS_TILES ? AS_STEP : AS_TILES) : STEP ? AS_STEP : AS_TILES;
}

template <class T, class C, int DP, int EL, bool STEP, bool TILES>
__global__ __launch_bounds__(256, (room<T, C, DP, EL, STEP, TILES>())) void paged_attend(const PgParams p) {
    int wg = blockIdx.x;
    if constexpr (TILES) {                   // they take longer: they begin first
        if (wg < p.tiles.groups) return tiles<T, C, DP>(p, wg);
        wg -= p.tiles.groups;
    }
    if constexpr (STEP) {
        if (wg < p.step.groups) return step<T, C, DP, EL>(p, wg);
        wg -= p.step.groups;
    }
    write_outside<T>(p, wg, OUTSIDE_GROUPS);
}

template <class T, class C, int DP, int EL> int attend(const PgParams& p, hipStream_t st) {
    const int groups = p.tiles.groups + p.step.groups + (p.offsets ? OUTSIDE_GROUPS : 0);
    const dim3 grid((unsigned)groups);
    if (!p.tiles.groups) paged_attend<T, C, DP, EL, true, false><<<grid, 256, 0, st>>>(p);
    else if (p.step.groups) paged_attend<T, C, DP, EL, true, true><<<grid, 256, 0, st>>>(p);
    else paged_attend<T, C, DP, 8, false, true><<<grid, 256, 0, st>>>(p);
    return (int)hipGetLastError();
}

}  // namespace pg

template <class T> int pg_attend_type(int held, const PgParams& p, hipStream_t st) {
    const auto with = [&](auto c) {
        return pg::by_width(p.D, [&](auto dp) {
            typedef decltype(c) C;
            if constexpr (pg::coded<C> && dp.value >= 64) {
                if (p.D % 16 == 0) return pg::attend<T, C, dp.value, 16>(p, st);
            }
            return pg::attend<T, C, dp.value, 8>(p, st);
        });
    };
    return held == QLKA_INT8 ? with(pg::Int8()) : held == QLKA_E4M3 ? with(pg::E4m3()) : with(T());
}

}  // namespace qlka
