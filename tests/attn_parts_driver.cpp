// How a step's work is shared (csrc/attn_plan.h), on the CPU under sanitizers: shares cover all groups in order and find their
// owners up to the largest numbers, one sequence's units get whole workgroups, and groups of twice the tiles cover the same
// positions.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../qwenny_amd/csrc/attn_plan.h"

using namespace qh;

#define CHECK(c)                                               \
    do {                                                       \
        if (!(c)) {                                            \
            std::printf("line %d: %s\n", __LINE__, #c);        \
            std::exit(1);                                      \
        }                                                      \
    } while (0)

int main() {
    std::mt19937_64 rng(11);
    auto in = [&](int64_t lo, int64_t hi) { return (int)std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
    for (int trial = 0; trial < 20000; trial++) {
        const int all = trial % 3 ? in(1, 5000) : in(1, 2147483647 - 1);
        const int used = in(1, all < TREE_MAX_WGS ? all : TREE_MAX_WGS);
        CHECK(first_group(0, all, used) == 0 && first_group(used, all, used) == all);
        for (int k = 0; k < 20; k++) {
            const int w = in(0, used - 1), lo = first_group(w, all, used), hi = first_group(w + 1, all, used);
            CHECK(lo < hi);
            CHECK(group_owner(lo, all, used) == w && group_owner(hi - 1, all, used) == w && group_owner(in(lo, hi - 1), all, used) == w);
        }
    }
    for (int trial = 0; trial < 20000; trial++) {
        const int units = in(1, 300), groups = in(1, 400), grid = in(1, 768), all = units * groups;
        const int used = used_workgroups(grid, all, 1, units);
        CHECK(used >= 1 && used <= grid && used <= all);
        CHECK(used_workgroups(grid, all, 2, units) == (all < grid ? all : grid));
        if (units <= grid)
            for (int u = 0; u <= units; u++) {  // a unit begins where a workgroup's part begins
                const int w = u == units ? used : group_owner(u * groups, all, used);
                CHECK(first_group(w, all, used) == u * groups);
            }
    }
    for (int trial = 0; trial < 20000; trial++) {
        const int32_t start[2] = {0, in(0, 64)}, len[1] = {in(0, 1 << 20)};
        const TreeArrays a{start, len, 1 << 15, 6, start[1], 1, 64, in(1, 8)};
        const Seq s = sequence(a, 0, 16 << in(0, 1)), w = sequence(a, 0, 16, true);
        CHECK(w.groups == (s.groups + 1) / 2 && w.total == s.total);
        CHECK(!s.groups || ((s.groups - 1) * GROUP_TILES * KV_TILE < s.total && s.total <= s.groups * GROUP_TILES * KV_TILE));
    }
    std::puts("ok");
    return 0;
}
