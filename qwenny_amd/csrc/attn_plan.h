// How a step's attention is shared among workgroups (tree_attn.hip), in plain C++: the kernels and a host test make the same
// plan from the same arrays. Whatever the arrays hold, every index made here lies in its buffer.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace qh {

constexpr int KV_TILE = 64;          // tokens of a tile; pages are a multiple of it
constexpr int GROUP_TILES = 4;       // tiles of a group, a workgroup's smallest part: one for each of its waves
constexpr int TREE_MAX_SEQS = 1024;  // sequences of a step
constexpr int TREE_MAX_NEW = 64;     // tokens of one sequence in a step: a mask is 64 bits
constexpr int TREE_MAX_WGS = 1024;   // workgroups of a launch

struct TreeArrays {
    const int32_t* start;  // [n_seq + 1]
    const int32_t* len;    // [n_seq]
    int64_t table_ld;      // pages of a table's row
    int page_shift;
    int n, n_seq, max_new;
    int group;  // query heads of a kv head
};

// A sequence's part of the step: tokens first .. first + news, `old` positions before them, `total` in all; its rows (token,
// query head of the kv head) in `chunks` of some rows each, its positions in `groups`. A sequence has work only if its numbers
// fit; otherwise its tokens are nobody's (news = 0). `bad`: it has such tokens. `disorder`: its start lies before an
// earlier sequence's, or its tokens are not start[b] <= start[b + 1] <= n: they are not taken, whatever they were meant to be.
struct Seq {
    int first, news, old, total, chunks, groups;
    bool bad, disorder;
};

// groups of `total` positions; `wide`: groups of twice the tiles, where there are enough for every workgroup
constexpr int group_count(int total, bool wide = false) {
    const unsigned size = KV_TILE * GROUP_TILES << (wide ? 1 : 0);
    return (int)(((unsigned)total + size - 1) / size);
}

// (`rows`: a power of two; `before`: start_before(a, b), or 0 where the starts are in order. The firsts of all sequences then
// ascend, and the tokens of those that have work follow one another: each token has one sequence at most, the last whose
// first is not past it.)
constexpr Seq sequence(const TreeArrays& a, int b, int rows, bool wide = false, int before = 0) {
    const int s0 = a.start[b], s1 = a.start[b + 1], len = a.len[b];
    const int cap = (int)(a.table_ld << a.page_shift), most = a.max_new < cap ? a.max_new : cap;
    const bool disorder = s0 < before || s1 < s0 || s1 > a.n;
    const int tokens = disorder ? 0 : s1 - s0;
    const bool fits = tokens <= most && len >= 0 && len <= cap - tokens;
    const int first = !disorder || (s0 > before && s0 <= a.n) ? s0 : before;
    const int news = fits ? tokens : 0, old = fits ? len : 0, total = old + news;
    const int chunks = (news * a.group + rows - 1) >> __builtin_ctz(rows);
    return Seq{first, news, old, total, chunks, chunks ? group_count(total, wide) : 0, disorder || news != tokens, disorder};
}

// The largest of the starts before sequence b that are numbers of tokens at all (for steps whose starts are not in order).
constexpr int start_before(const TreeArrays& a, int b) {
    int most = 0;
    for (int i = 0; i < b; i++)
        if (a.start[i] > most && a.start[i] <= a.n) most = a.start[i];
    return most;
}

// A token that no sequence has work for: outside of all sequences of a step in order (padding), or not served. `disorder`: some
// sequence's.
constexpr bool padding(const TreeArrays& a, int token, bool disorder) {
    return !disorder && (token < a.start[0] || token >= a.start[a.n_seq]);
}

// `all` groups in a row (sequence by sequence, kv head by kv head, chunk by chunk) in equal parts for `used` <= all
// workgroups: the first group of workgroup w, the workgroup of group `at`.
// (w all / used and (used (at + 1) - 1) / all, without 64-bit divisions: used <= TREE_MAX_WGS)
constexpr int first_group(int w, int all, int used) {
    return used == all ? w : w * (all / used) + w * (all % used) / used;
}
constexpr int group_owner(int at, int all, int used) {
    if (used == all) return at;
    int w = (int)((float)at * ((float)used / (float)all));  // off by one at most
    w = w < 0 ? 0 : w >= used ? used - 1 : w;
    while (w > 0 && first_group(w, all, used) > at) w--;
    while (w + 1 < used && first_group(w + 1, all, used) <= at) w++;
    return w;
}

// group_owner in few steps, as join_kernel takes it, from 1 / all in 64 bits: ((at + 1) used - 1) / all, the half keeping it off
// whole numbers (-1 for group -1). group_owner and partial_slot say what it has to give; the host tests hold it to them.
constexpr int owner(int at, int used, double inv_all) {
    return at < 0 ? -1 : (int)(((double)at * used + (used - 0.5)) * inv_all);
}

// The workgroups that take part of `grid`. One sequence's units are all alike: each gets as many workgroups as any, so that no
// workgroup has parts of two.
constexpr int used_workgroups(int grid, int all, int n_seq, int units) {
    return all <= grid ? all : n_seq == 1 && units <= grid ? units * (grid / units) : grid;
}

// Where workgroup w keeps its partial result of the unit (sequence, kv head, chunk) whose groups begin at u0: it has at most
// two, the unit that its part begins in and the one that it ends in.
constexpr int partial_slot(int w, int u0, int all, int used) { return 2 * w + (first_group(w, all, used) < u0 ? 1 : 0); }

}  // namespace qh
