// Who writes each token's row of a step's attention (csrc/attn_plan.h), on the CPU under sanitizers, for arrays of any numbers in
// buffers of exactly their sizes, as the kernels walk them: the list made as if the starts were in order and again where
// they are not, the workgroups that are used, groups of four and of eight tiles, the joining side by owner(). Each row is written
// by one sequence's one workgroup, by the join alone, or as a row that no sequence has work for.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
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
    std::mt19937 rng(19);
    auto in = [&](int lo, int hi) { return (int)std::uniform_int_distribution<int>(lo, hi)(rng); };
    int joined = 0, wides = 0, alone = 0, served_beside_bad = 0;
    for (int trial = 0; trial < 6000; trial++) {
        const int n_seq = trial % 4 == 0 ? 1 : in(1, trial % 7 == 0 ? 200 : 6), heads = in(1, 4), group = in(1, 9), rows = 16 << in(0, 1);
        const int max_new = in(1, TREE_MAX_NEW), page_shift = in(6, 10), grid = in(1, 600);
        const int64_t table_ld = in(1, 12);
        const int cap = (int)(table_ld << page_shift);
        std::vector<int32_t> start{in(0, 3) ? 0 : in(0, 5)}, len;
        for (int b = 0; b < n_seq; b++) {
            const int m = in(0, 3) ? in(0, in(0, 9) ? max_new : max_new + 9) : 0;  // (now and then more than fits)
            start.push_back(start.back() + m);
            len.push_back(in(0, 9) ? in(0, cap) : in(-5, cap + 5));
        }
        const int n = start.back() + (in(0, 3) ? 0 : in(0, 5)) + (start.back() == 0);
        if (trial % 3 == 0)
            for (int k = in(1, 3); k; k--) {
                const int wild[] = {-1, -2147483647 - 1, 2147483647, n + 1, in(0, n), in(0, n)};
                start[in(0, n_seq)] = wild[in(0, 5)];
            }
        const TreeArrays a{start.data(), len.data(), table_ld, page_shift, n, n_seq, max_new, group};
        bool disorder = false;
        for (int b = 0; b < n_seq; b++) disorder |= sequence(a, b, rows).disorder;
        std::vector<int> base[2] = {{0}, {0}}, owner_of(n, -1);
        std::vector<Seq> seq;
        for (int b = 0; b < n_seq; b++) {
            const Seq s = sequence(a, b, rows, false, disorder ? start_before(a, b) : 0);
            CHECK(s.first >= 0 && s.news >= 0 && s.news <= max_new && s.first + s.news <= n);
            CHECK(s.old >= 0 && s.total == s.old + s.news && s.total <= cap);
            CHECK(!b || s.first >= seq.back().first + seq.back().news);  // one token, one sequence
            for (int t = s.first; t < s.first + s.news; t++) owner_of[t] = b;
            // what fits keeps its outputs, whatever its neighbours hold
            int64_t most = 0;
            for (int i = 0; i < b; i++)
                if (start[i] <= n && start[i] > most) most = start[i];
            const int64_t m = (int64_t)start[b + 1] - start[b];
            const bool fits = start[b] >= most && start[b] <= start[b + 1] && start[b + 1] <= n && m <= max_new && len[b] >= 0 && len[b] + m <= cap;
            CHECK(s.news == (fits ? m : 0));
            CHECK(!fits || (s.first == start[b] && s.old == len[b]) || m == 0);
            seq.push_back(s);
            for (int k = 0; k < 2; k++) base[k].push_back(base[k].back() + heads * s.chunks * (k ? (s.groups + 1) >> 1 : s.groups));
        }
        const bool wide = base[0].back() > grid;
        const std::vector<int>& at0 = base[wide];
        const int all = at0.back(), used = used_workgroups(grid, all, n_seq, heads * seq[0].chunks);
        CHECK(used <= grid && used <= all);
        std::vector<int> written(n * heads * group, 0);
        std::map<int, int> slot_unit;
        auto groups_of = [&](const Seq& s) { return group_count(s.total, wide); };
        for (int w = 0; w < used; w++) {
            const int lo = first_group(w, all, used), hi = first_group(w + 1, all, used);
            for (int at = lo; at < hi;) {
                int b = -1;
                for (int i = 0; i < n_seq; i++)
                    if (at0[i] <= at) b = i;
                const Seq& s = seq.at(b);
                const int groups = groups_of(s), past = at - at0[b], unit = past / groups, g0 = past % groups;
                CHECK(s.news > 0 && unit < heads * s.chunks);
                const int g1 = groups < g0 + hi - at ? groups : g0 + hi - at, head = unit / s.chunks, row0 = unit % s.chunks * rows;
                if (g0 == 0 && g1 == groups) {
                    for (int r = row0; r < row0 + rows && r < s.news * group; r++)
                        written.at(((s.first + r / group) * heads + head) * group + r % group)++;
                } else {
                    const int slot = 2 * w + (at != lo);
                    CHECK(slot < 2 * grid && !slot_unit.count(slot));
                    slot_unit[slot] = at - g0;
                }
                at += g1 - g0;
            }
        }
        auto find = [&](int token) {  // the last that begins at or before it
            int b = -1;
            for (int i = 0; i < n_seq; i++)
                if (seq[i].first <= token) b = i;
            return b;
        };
        const double inv_all = 1.0 / all;
        for (int t = 0; t < n; t++) {
            const int b = find(t);
            const bool served = b >= 0 && t - seq[b].first < seq[b].news;
            CHECK(served == (owner_of[t] >= 0) && (!served || owner_of[t] == b));
            if (!served) {
                const bool pad = padding(a, t, disorder);
                CHECK(!pad || t < start[0] || t >= start[n_seq]);
                CHECK(pad || disorder || (t >= start[0] && t < start[n_seq]));
                for (int r = 0; r < heads * group; r++) written.at(t * heads * group + r)++;
                continue;
            }
            served_beside_bad += disorder;
            const Seq& s = seq[b];
            for (int head = 0; head < heads; head++)
                for (int g = 0; g < group; g++) {
                    const int r = (t - s.first) * group + g, groups = groups_of(s), u0 = at0[b] + (head * s.chunks + r / rows) * groups;
                    const int w0 = owner(u0, used, inv_all), parts = owner(u0 + groups - 1, used, inv_all) - w0 + 1;
                    if (parts == 1) continue;
                    for (int i = 0; i < parts; i++) {
                        const int slot = i ? 2 * (w0 + i) : 2 * w0 + (owner(u0 - 1, used, inv_all) == w0 ? 1 : 0);
                        CHECK(slot_unit.count(slot) && slot_unit[slot] == u0);
                    }
                    written.at((t * heads + head) * group + g)++;
                    joined++;
                }
        }
        for (int v : written) CHECK(v == 1);
        wides += wide, alone += n_seq == 1 && used < grid && used < all;
    }

    const int trial = -1;
    CHECK(joined > 100000 && wides > 500 && alone > 20 && served_beside_bad > 1000);
    std::puts("ok");
    return 0;
}
