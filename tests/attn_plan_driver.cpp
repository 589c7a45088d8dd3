// The work plan of a step's attention (csrc/attn_plan.h) walked on the CPU as the kernels walk it, for valid and for invalid
// arrays held in buffers of exactly their sizes (AddressSanitizer catches an index past one): every (unit, group) is taken
// once, every partial slot is used by one unit at most, the joining side finds the slots that the producing side wrote, and
// every table, token and row index lies in its buffer.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "../qwenny_amd/csrc/attn_plan.h"

using namespace qh;

#define CHECK(c)                                                        \
    do {                                                                \
        if (!(c)) {                                                     \
            std::printf("trial %d line %d: %s\n", trial, __LINE__, #c); \
            std::exit(1);                                               \
        }                                                               \
    } while (0)

int main() {
    std::mt19937 rng(7);
    auto in = [&](int lo, int hi) { return (int)std::uniform_int_distribution<int>(lo, hi)(rng); };
    for (int trial = 0; trial < 3000; trial++) {
        const bool valid = trial % 3 != 0;
        const int n_seq = in(1, trial % 7 == 0 ? 300 : 6), heads = in(1, 4), group = in(1, 9), rows = 16 << in(0, 2);
        const int max_new = in(1, TREE_MAX_NEW), page_shift = in(6, 10);
        const int64_t table_ld = in(1, 12);
        const int cap = (int)(table_ld << page_shift);
        std::vector<int32_t> start{0}, len;
        for (int b = 0; b < n_seq; b++) {
            int m = in(0, 3) ? in(0, max_new) : 0;
            if (m > cap) m = cap;
            start.push_back(start.back() + m);
            len.push_back(in(0, 5) ? in(0, cap - m) : 0);
        }
        int n = start.back();
        if (!valid)
            for (int k = in(1, 4); k; k--) {
                const int wild[] = {-1, -2147483647 - 1, 2147483647, n + 1, cap, cap + 1, in(0, 1000)};
                (in(0, 1) ? start : len)[in(0, n_seq - 1)] = wild[in(0, 6)];
                if (!in(0, 4)) start[n_seq] = wild[in(0, 6)];
            }
        if (n == 0) n = 1;
        std::vector<char> table((size_t)n_seq * table_ld), tokens(n);
        const TreeArrays a{start.data(), len.data(), table_ld, page_shift, n, n_seq, max_new, group};
        std::vector<int> base(n_seq + 1, 0);
        for (int b = 0; b < n_seq; b++) {
            const Seq s = sequence(a, b, rows);
            CHECK(s.first >= 0 && s.news >= 0 && s.first + s.news <= n && s.news <= max_new);
            CHECK(s.old >= 0 && s.total == s.old + s.news && s.total <= cap);
            CHECK(!valid || (!s.bad && s.news == start[b + 1] - start[b] && s.old == len[b]));
            CHECK((s.groups > 0) == (s.news > 0) && (s.chunks > 0) == (s.news > 0));
            base[b + 1] = base[b] + heads * s.chunks * s.groups;
        }
        const int all = base[n_seq];
        if (!all) continue;
        const int grid = in(1, 600), used = grid < all ? grid : all;
        std::vector<char> taken(all, 0);
        std::map<int, int> slot_unit;  // slot -> u0
        std::set<int> direct;
        for (int w = 0; w < used; w++) {
            const int lo = first_group(w, all, used), hi = first_group(w + 1, all, used);
            CHECK(lo < hi && hi <= all);
            for (int at = lo; at < hi;) {
                int b = 0;
                for (int step = 512; step; step >>= 1)
                    if (b + step < n_seq && base[b + step] <= at) b += step;
                const Seq s = sequence(a, b, rows);
                CHECK(s.groups > 0 && at >= base[b] && at < base[b + 1]);
                const int unit = (at - base[b]) / s.groups, g0 = (at - base[b]) - unit * s.groups;
                const int g1 = s.groups < g0 + hi - at ? s.groups : g0 + hi - at;
                const int head = unit / s.chunks, row0 = (unit - head * s.chunks) * rows;
                CHECK(head < heads && row0 / group < s.news);
                const int tiles = (s.total + KV_TILE - 1) / KV_TILE;
                for (int t = g0 * GROUP_TILES; t < g1 * GROUP_TILES && t < tiles; t++)
                    table.at((size_t)b * table_ld + ((t * KV_TILE) >> page_shift))++;
                for (int r = row0; r < row0 + rows; r++)
                    if (r / group < s.news) tokens.at(s.first + r / group)++;
                const int u0 = at - g0;
                for (int k = at; k < at + g1 - g0; k++) {
                    CHECK(!taken[k]);
                    taken[k] = 1;
                    CHECK(group_owner(k, all, used) == w);
                }
                if (g0 == 0 && g1 == s.groups) {
                    direct.insert(u0);
                } else {
                    const int slot = 2 * w + (at != lo);
                    CHECK(slot == partial_slot(w, u0, all, used) && slot < 2 * used);
                    CHECK(!slot_unit.count(slot));
                    slot_unit[slot] = u0;
                }
                at += g1 - g0;
            }
        }
        for (int k = 0; k < all; k++) CHECK(taken[k]);
        for (int b = 0; b < n_seq; b++) {  // the joining side
            const Seq s = sequence(a, b, rows);
            for (int u = 0; u < heads * s.chunks; u++) {
                const int u0 = base[b] + u * s.groups;
                const int w0 = group_owner(u0, all, used), w1 = group_owner(u0 + s.groups - 1, all, used);
                CHECK((w0 == w1) == (direct.count(u0) > 0));
                if (w0 != w1)
                    for (int w = w0; w <= w1; w++) {
                        auto it = slot_unit.find(partial_slot(w, u0, all, used));
                        CHECK(it != slot_unit.end() && it->second == u0);
                    }
            }
        }
    }
    std::puts("ok");
    return 0;
}
