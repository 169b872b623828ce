"""CPU checks of how workgroups find their sequences and rows (csrc/segments.h, csrc/paged_cut.h): every row of a valid
call in one block, positions in their pages, and no row, group, page or place outside the call's, whatever offsets and
lengths are."""

from test_paged_cut import run

# 64 lanes one after the other, which is what a wave's vote comes to.
LANES = r"""
#include "segments.h"
#include "paged_cut.h"
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
using namespace qlka;
struct OnHost {
    template <class F> int count(F f) const {
        int n = 0;
        for (int lane = 0; lane < 64; ++lane) n += f(lane) ? 1 : 0;
        return n;
    }
    int same(int x) const { return x; }
};
std::mt19937 rng(1);
int below(int n) { return (int)(rng() % (unsigned)n); }
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
"""

VALID = LANES + r"""
int main() {
    for (int i = 0; i < 600; ++i) {
        const int sizes[] = {0, 1, 31, 32, 33, 200, 1000, 5000}, rows_of[] = {32, 64, 128};
        const int T = sizes[below(8)], B = i % 3 ? below(9) : below(700), rows = rows_of[below(3)];
        std::vector<int> at(B + 1);
        for (int& x : at) x = below(T + 1);
        std::sort(at.begin(), at.end());
        std::vector<int> seen(T, 0), groups(segment_blocks(T, B, 32), 0);
        for (int number = 0; number < segment_blocks(T, B, rows); ++number) {
            const Segment s = segment_of(at.data(), B, T, rows, number, OnHost());
            CHECK(s.index >= -1 && s.index <= B && s.block >= 0);
            const int group = segment_start(s.first, s.index + 1, 32);
            for (int r = s.block * rows; r < s.rows && r < (s.block + 1) * rows; ++r) {
                ++seen[s.first + r];
                if (r % 32 == 0) ++groups.at(group + r / 32);
                if (s.index >= 0 && s.index < B)
                    CHECK(s.first == at[s.index] && s.rows == at[s.index + 1] - at[s.index]);
            }
        }
        for (int n : seen) CHECK(n == 1);
        for (int n : groups) CHECK(n <= 1);                          // groups of 32 rows have places of their own
    }
    // the last place of many, at and around the squares of what is looked at together
    for (int count : {1, 2, 63, 64, 65, 127, 128, 129, 4095, 4096, 4097, 100000})
        for (int i = 0; i < 200; ++i) {
            std::vector<int> at(count, 0);
            for (int j = 1; j < count; ++j) at[j] = at[j - 1] + (below(3) ? 0 : below(4));
            const int x = below(at[count - 1] + 3);
            int want = 0;
            for (int j = 0; j < count; ++j) if (at[j] <= x) want = j;
            const auto get = [&](int j) { if (j < 0 || j >= count) std::abort(); return at[j]; };
            CHECK(last_upto(count, x, get, OnHost()) == want);
        }
    std::puts("ok");
    return 0;
}
"""

WILD = LANES + r"""
int wild() {
    const int extremes[] = {INT32_MIN, -1, 0, 1, INT32_MAX, 1 << 28, -(1 << 28)};
    return below(3) ? (below(2) ? below(2000) : extremes[below(7)]) : (int)rng();
}
int main() {
    for (int i = 0; i < 3000; ++i) {
        const int T = below(3) ? below(300) : 0, B = below(4) ? below(9) : below(400);
        std::vector<int> at(B + 1);
        for (int& x : at) x = wild();
        for (int rows : {32, 128})
            for (int number = 0; number < segment_blocks(T, B, rows); ++number) {
                const Segment s = segment_of(at.data(), B, T, rows, number, OnHost());
                CHECK(s.index >= -1 && s.index <= B);
                CHECK(s.first >= 0 && s.rows >= 0 && s.first + s.rows <= T);
                const int group = segment_start(s.first, s.index + 1, 32);
                CHECK(group >= 0 && group + (s.rows + 31) / 32 <= segment_blocks(T, B, 32));
                CHECK(s.block >= 0 && (long long)s.block * rows <= INT32_MAX);    // kernels leave those past s.rows
            }
        for (int x : {0, T - 1, T, wild()}) {
            const int j = last_upto(B + 1, x, [&](int k) { if (k < 0 || k > B) std::abort(); return at[k]; }, OnHost());
            CHECK(j >= -1 && j <= B);
        }
        // attention over pages
        for (int b = 0; b < B; ++b) {
            const int first = segment_edge(at.data(), B, T, b + 1), end = segment_edge(at.data(), B, T, b + 2);
            const pg::Tokens t = pg::tokens_at(first, pg::rows_between(first, end), wild());
            CHECK(t.first >= 0 && t.rows >= 0 && t.first + t.rows <= T);
            const int page_size = 1 + below(below(2) ? 100 : 65536), table_len = below(50);
            const int places = (int)std::min<int64_t>((int64_t)table_len * page_size, pg::MOST_POSITIONS);
            const int seen = pg::seen_upto(t.start + t.rows - 1, below(5), places);
            CHECK(seen >= 0 && seen <= places);
            const pg::Division by = pg::division_by(page_size);
            for (int n : {0, seen / 2, seen - 1}) {
                if (n < 0 || n >= seen) continue;
                const int page = pg::divided(n, by);
                CHECK(page == n / page_size && page >= 0 && page < table_len);
            }
            const int share = 1 + below(12), G = 1 + below(12);
            for (int block_rows : {16, 128}) {
                const int rows = t.rows * share, blocks = (rows + block_rows - 1) / block_rows;
                const pg::Cut c = pg::cut_of({blocks, seen}, 128 * (1 + below(100)), 128);
                CHECK(c.parts >= 1 && c.span >= 1 && (long long)c.parts * c.span >= seen);
                const pg::InSequence u = pg::place_in(blocks, wild(), G);
                CHECK(u.part >= 0 && u.kvh >= 0 && u.kvh < G && u.block >= 0 && u.block < std::max(blocks, 1));
                for (int r = u.block * block_rows; r < rows && r < (u.block + 1) * block_rows; ++r)
                    CHECK(t.first + r / share < T && u.kvh * share + r % share < G * share);
            }
        }
    }
    std::puts("ok");
    return 0;
}
"""


def test_rows_of_valid_calls(tmp_path):
    assert run(tmp_path, VALID, "segments") == ["ok"]


def test_rows_whatever_the_offsets_are(tmp_path):
    assert run(tmp_path, WILD, "segments") == ["ok"]


def test_division_by_every_page_size(tmp_path):
    assert run(tmp_path, r"""
#include "paged_cut.h"
#include <cstdio>
int main() {
    using namespace qlka::pg;
    for (int size = 1; size <= 65536; ++size) {
        const Division by = division_by(size);
        for (int k : {0, 1, 2, 1000, MOST_POSITIONS / size - 1, MOST_POSITIONS / size, 0x7fffffff / size})
            for (int d = -1; d <= 1; ++d) {
                const long long n = (long long)k * size + d;
                if (n >= 0 && n <= 0x7fffffff && divided((int)n, by) != n / size) return 1;
            }
    }
    std::puts("ok");
    return 0;
}
""", "division") == ["ok"]
