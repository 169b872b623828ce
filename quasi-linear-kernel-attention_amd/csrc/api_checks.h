// What the host sides of the softmax kernels share: refusals, workspaces, grids and splits. Not part of the public
// interface.
#pragma once

#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "qlka.h"
#include "qlka_internal.h"
#include "softmax.h"

namespace qlka {

constexpr int64_t LONGEST = 1 << 28;      // rows, keys, positions: sums of a few stay in 32 bits
constexpr int64_t MOST_ROWS = INT32_MAX;

inline int refuse(const char* fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return api_error(QLKA_EINVAL, buf);
}

inline int status(int e, const char* where) {
    if (e == 0) return QLKA_OK;
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", where, hipGetErrorString((hipError_t)e));
    return api_error(QLKA_EHIP, buf);
}

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits of an axis of `tiles` tiles for `groups` workgroups over the other axes, by an estimate of the time: rounds of
// workgroups on a CU (one alone on a CU is not twice as fast as two, waits not being filled), each its tiles and what
// it costs by itself, and the joining of `join` bytes a split. In microseconds, the constants set by hand until 12
// shapes (prompts and gradients of 65 to 8192 keys, fp32 and bf16) came near the best of 1 to 16 splits of all their
// axes: eight of them within 4% of it or faster (1 x 4 heads, 100 x 8000: 14.4 us, 17.2 the best one number, 132
// unsplit), the others 7 to 18% slower (1 x 12, 512 x 4096: 26.8 : 23.7, unsplit 70; 4 x 12, 1024 x 4096: 91 : 77,
// unsplit 88).
inline int splits_for(int64_t groups, int64_t tiles, double tile_us, double join_bytes) {
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

// scores and log sums are held in units of the scale
inline int check_scale(float scale) {
    if (scale != 0.f && !(std::fabs(scale) >= 0x1p-96f && std::fabs(scale) <= 0x1p96f))
        return refuse("scale must be 0 or of a size in [2^-96, 2^96]");
    return QLKA_OK;
}

inline int need_ws(const void* ws, size_t have, size_t need) {
    if (need == 0) return QLKA_OK;
    if (ws && have >= need && (uintptr_t)ws % 16 == 0) return QLKA_OK;
    return api_error(QLKA_EWORKSPACE, "workspace too small, null or not aligned to 16 bytes");
}

// A launch takes less than 2^32 threads.
inline int fits_grid(int64_t groups, int threads) {
    if (groups <= (int64_t)UINT32_MAX / threads) return QLKA_OK;
    return refuse("too many workgroups: %lld of %d threads, a launch takes less than 2^32 threads", (long long)groups,
                  threads);
}
// a kernel of workgroups of 256 that takes `lanes` lanes a row
inline int fits_rows(int64_t rows, int lanes) { return fits_grid(ceil_div(rows * lanes, 256), 256); }

// Rows are read and written in pieces of 16 bytes, so those of every dimension of more than one (of n) start at
// multiples of them; strides in elements of `size` bytes.
inline int check_rows(const char* name, const void* x, const int64_t* s, const int64_t* sizes, int n, int size) {
    if (!x) return QLKA_OK;
    bool aligned = (uintptr_t)x % 16 == 0;
    for (int i = 0; i < n; ++i) {
        if (sizes[i] <= 1) continue;
        if (s[i] < 0) return refuse("the strides of %s must not be negative", name);
        aligned = aligned && s[i] * size % 16 == 0;
    }
    return aligned ? QLKA_OK : refuse("the rows of %s must be aligned to 16 bytes", name);
}

}  // namespace qlka
