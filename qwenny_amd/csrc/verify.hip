// Drafted tokens held against the target's logits (qh_verify): which of them are kept, and the token after them.
//
// For a row of logits l at temperature T: w(v) = exp((l(v) - max l) / T), Z = sum_v w(v). A row's choice by a number u in
// [0, 1) is the least v with sum_{v' <= v} w(v') > u Z. Drafts without probabilities: a sequence goes from its first token to
// the child that is its row's choice, while there is one. Drafts with probabilities q (chains): token t after row i is kept
// where u0 q(t) Z < w(t); where it is not, the choice is among max(0, w - Z q) instead of w.
// Everything behind the logits is 64-bit: in a flat distribution over 248,320 tokens a token's part of the sum is 4e-6 of it,
// and an error of 1e-7 in a sum, as 32 bits leave it, would pick the neighbour once in a few dozen choices.
// One read of the logits leaves each 4,096 of them with a maximum and a sum (bound by the read, and at few rows by one workgroup's way
// from its loads to its sum); what follows knows a row from those, reads a choice's 4,096 logits again and is bound by the chain of its trips
// to memory. Kernel times over 248,320 tokens (medians of a trace): 5 rows 6.1 us for the stats, 11.2 the choices, 3.9 the path; 64 rows 23.0
// (63 MB, 2.8 TB/s), 10.0, 3.9; 12 drafted chains of 5 16.4, 14.2 for the kept ones, 5.7 and 8.4 for the token after a rejection.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

#include "gemm.h"
#include "internal.h"
#include "kv.h"

using namespace qh;

namespace {

constexpr int THREADS = 256, PER = 16, BLOCK = THREADS * PER;  // logits of a thread, of a workgroup
constexpr int MAX_BLOCKS = 1024;                               // of a row: vocabularies up to 2^22
constexpr double LOG2E = 1.4426950408889634074;

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// A part of a row: its largest logit, where that is first, and the sum of 2^((l - max) log2e / T).
struct Stat {
    double sum;
    float max;  // NaN: the part has a NaN
    int32_t at;
};

// Where a sequence with drafts' probabilities ends: its last kept row, the row's sum and largest logit, and what is left to do.
struct End {
    double z, max;
    int32_t row, next;  // next: the token, or -1 as long as it is among max(0, w - Z q)
    int32_t open, kept;
};

struct Args {
    const float* logits;
    const float* draft;  // q, or null
    const int32_t* tokens;
    const float* temp;  // null: 1
    const float* u;     // [n][2]
    int64_t ld, draft_ld;
    int32_t vocab, blocks;
    TreeArrays t;
    const int32_t* table;
    const uint64_t* mask;
    Stat* stats;    // [n][blocks]
    int32_t* pick;  // [n]: each row's choice
    End* ends;      // [n_seq]
    double* rest;   // [n_seq][blocks]: sums of max(0, w - Z q)
    int32_t *next, *count, *emit, *src, *dst, *new_len;
};

// 2^t for t <= 0 to 1e-14 of it: the polynomial is e^x's series to its 11th power, |x| <= ln 2 / 2, of which the rest is 8.7e-15 of e^x at
// most (at x = -ln 2 / 2), beside a few roundings of 2^-53.
__device__ __forceinline__ double exp2_64(double t) {
    const double n = __builtin_rint(t), x = (t - n) * 0.69314718055994530942;
    double p = 1.0 / 39916800;
    p = fma(p, x, 1.0 / 3628800);
    p = fma(p, x, 1.0 / 362880);
    p = fma(p, x, 1.0 / 40320);
    p = fma(p, x, 1.0 / 5040);
    p = fma(p, x, 1.0 / 720);
    p = fma(p, x, 1.0 / 120);
    p = fma(p, x, 1.0 / 24);
    p = fma(p, x, 1.0 / 6);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0);
    return __builtin_ldexp(p, (int)fmax(n, -2000.0));
}

// The same where there are many: 2^(n / 64) by a table of 64 in LDS, the rest |x| <= ln 2 / 128 by four terms (what is left is below 4e-14).
// 13 operations instead of 21: the stats of 64 rows take 23 us, with the other 28.
struct Table {
    double pow2[64];
};
__device__ __forceinline__ void fill(Table& table) {
    if (threadIdx.x < 64) table.pow2[threadIdx.x] = exp2_64((double)threadIdx.x / 64.0 - 1.0) * 2.0;
}
__device__ __forceinline__ double exp2_64(const Table& table, double t64) {  // of t64 / 64
    constexpr double C = 0.69314718055994530942 / 64;
    const double n = __builtin_rint(t64), f = t64 - n;
    const int i = max((int)n, -200000);
    double p = C * C * C * C / 24;
    p = fma(p, f, C * C * C / 6);
    p = fma(p, f, C * C / 2);
    p = fma(p, f, C);
    p = fma(p, f, 1.0);
    return __builtin_ldexp(p * table.pow2[i & 63], i >> 6);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
// inclusive sums over the wave's lanes
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double left = __shfl_up(v, d);
        v += lane >= d ? left : 0.0;
    }
    return v;
}

// The sequence of a token: the first within whose start and end it lies, or -1. (Where starts are not in order another may have it too, but
// none that has work: that one begins below an earlier end.)
__device__ __forceinline__ int seq_of(const Args& a, int token) {
    const int lane = threadIdx.x & 63;
    for (int c = 0; c < a.t.n_seq; c += 64) {
        const int b = min(c + lane, a.t.n_seq - 1), end = a.t.start[b + 1];
        const uint64_t in = __ballot(a.t.start[b] <= token && token < end && end <= a.t.n);
        if (in) return min(c + __ffsll((unsigned long long)in) - 1, a.t.n_seq - 1);
    }
    return -1;
}

// The row's temperature as log2e / T, 0 where the likeliest token is wanted; negative: the row's sequence has none.
__device__ __forceinline__ double sharpness(const Args& a, int b) {
    if (!a.temp) return LOG2E;
    const float t = b < 0 ? 0.0f : a.temp[b];
    return t == 0.0f ? 0.0 : t > 0.0f && t < INFINITY ? LOG2E / (double)t : -1.0;
}

// A thread's 16 logits (or probabilities) of a row from its `at`-th on: four runs of four, a run of the wave 1 KiB.
__device__ __forceinline__ int place(int k) { return (k >> 2) * (THREADS * 4) + threadIdx.x * 4 + (k & 3); }
__device__ __forceinline__ void load(const float* row, int at, int vocab, float fill, float (&x)[PER]) {
#pragma unroll
    for (int r = 0; r < PER / 4; r++) {
        const int i = at + place(4 * r);
        f4u v = {fill, fill, fill, fill};
        if (i + 4 <= vocab) {
            v = *(const f4u*)(row + i);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < vocab) v[k] = row[i + k];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) x[4 * r + k] = v[k];
    }
}

// Each part of each row: one read of the logits.
__global__ __launch_bounds__(THREADS) void verify_stats_kernel(const Args a) {
    __shared__ float tops[THREADS / 64];
    __shared__ int32_t places[THREADS / 64];
    __shared__ double sums[THREADS / 64];
    __shared__ Table table;
    const int row = blockIdx.x / a.blocks, part = blockIdx.x - row * a.blocks, at = part * BLOCK, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float x[PER];
    load(a.logits + row * a.ld, at, a.vocab, -INFINITY, x);
    fill(table);
    const double sharp = sharpness(a, seq_of(a, row));
    if (part == 0 && threadIdx.x == 0) {  // (what no sequence has work for says nothing)
        a.emit[row] = -1;
        if (a.src) a.src[row] = a.dst[row] = -1;
    }
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int k = 0; k < PER; k++) top = fmaxf(top, x[k]), nan |= x[k] != x[k];
    int where = 0x7fffffff;
#pragma unroll
    for (int k = PER - 1; k >= 0; k--) where = x[k] == top ? at + place(k) : where;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float other = __shfl_xor(top, d);
        const int its = __shfl_xor(where, d);
        where = other > top ? its : other == top ? min(where, its) : where;
        top = fmaxf(top, other);
    }
    nan = __any(nan);
    if (lane == 0) tops[wave] = nan ? NAN : top, places[wave] = where;
    __syncthreads();
    top = tops[0], where = places[0], nan = top != top;
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) {
        nan |= tops[w] != tops[w];
        where = tops[w] > top ? places[w] : tops[w] == top ? min(where, places[w]) : where;
        top = fmaxf(top, tops[w]);
    }
    double sum = 0.0;
    if (sharp > 0.0 && top > -INFINITY && top < INFINITY) {
#pragma unroll
        for (int k = 0; k < PER; k++) sum += x[k] == -INFINITY ? 0.0 : exp2_64(table, ((double)x[k] - (double)top) * (64.0 * sharp));
    }
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int w = 0; w < THREADS / 64; w++) sum += sums[w];
        a.stats[(size_t)row * a.blocks + part] = Stat{sum, nan ? NAN : top, where};
    }
}

// A row's parts, the first 64 (of a vocabulary of 262,144 all) in the lanes' registers.
struct Parts {
    const Stat* stats;
    Stat mine;
    int blocks;
    __device__ __forceinline__ Parts(const Args& a, int row) : stats(a.stats + (size_t)row * a.blocks), blocks(a.blocks) {
        mine = stats[min((int)(threadIdx.x & 63), blocks - 1)];
    }
    __device__ __forceinline__ Stat at(int k) const { return k < 64 ? mine : stats[k]; }  // (of lane k % 64)
};

// A row from its parts, by one wave: its largest logit, where, and Z. False where it has no choice (NaN, infinity, nothing).
struct Row {
    float max;
    int32_t at;
    double z;
};
__device__ __forceinline__ bool row_of(const Parts& parts, double sharp, Row* out) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY;
    int where = 0x7fffffff;
    bool nan = false;
    for (int k = lane; k < parts.blocks; k += 64) {
        const Stat s = parts.at(k);
        nan |= s.max != s.max;
        where = s.max > top ? s.at : s.max == top ? min(where, s.at) : where;
        top = fmaxf(top, s.max);
    }
    const float mine = top;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    where = mine == top ? where : 0x7fffffff;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) where = min(where, __shfl_xor(where, d));
    double z = 0.0;
    if (sharp > 0.0)
        for (int k = lane; k < parts.blocks; k += 64) {
            const Stat s = parts.at(k);
            if (s.max > -INFINITY) z += s.sum * exp2_64(((double)s.max - (double)top) * sharp);
        }
    out->max = top, out->at = where, out->z = wave_sum(z);
    return !__any(nan) && top > -INFINITY && top < INFINITY && sharp >= 0.0;
}

// The first part in which the sum passes `goal`, by the workgroup's every wave alike, and the sum before it; the last part that
// adds anything where none does (its rounding). `part(k)`: of lane k % 64.
template <class F>
__device__ __forceinline__ int find_block(const Args& a, double goal, F&& part, double* before) {
    const int lane = threadIdx.x & 63;
    double run = 0.0;
    int last = 0;
    double last_before = 0.0;
    for (int c = 0; c < a.blocks; c += 64) {
        const double v = c + lane < a.blocks ? part(c + lane) : 0.0;
        const double upto = run + wave_scan(v);
        const uint64_t past = __ballot(upto > goal && v > 0.0), some = __ballot(v > 0.0);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            *before = __shfl(upto - v, l);
            return c + l;
        }
        if (some) {
            const int l = 63 - __clzll((long long)some);
            last = c + l, last_before = __shfl(upto - v, l);
        }
        run = __shfl(upto, 63);
    }
    *before = last_before;
    return last;
}

// A thread's 16 logits (or probabilities) one after the other, as a search among them needs them.
__device__ __forceinline__ void load_run(const float* row, int at, int vocab, float fill, float (&x)[PER]) {
#pragma unroll
    for (int r = 0; r < PER; r += 4) {
        const int i = at + (int)threadIdx.x * PER + r;
        f4u v = {fill, fill, fill, fill};
        if (i + 4 <= vocab) {
            v = *(const f4u*)(row + i);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < vocab) v[k] = row[i + k];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) x[r + k] = v[k];
    }
}

// The first token of a part in which the sum passes `goal`: weights w[k] of the tokens at + 16 tid + k. One workgroup.
__device__ __forceinline__ int find_token(int at, const double (&w)[PER], double before, double goal) {
    __shared__ double sums[THREADS / 64];
    __shared__ int32_t found[2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double mine = 0.0;
#pragma unroll
    for (int k = 0; k < PER; k++) mine += w[k];
    const double upto = wave_scan(mine);
    if (threadIdx.x == 0) found[0] = 0x7fffffff, found[1] = -1;
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    double run = before;
    for (int v = 0; v < wave; v++) run += sums[v];
    run += upto - mine;
    int first = 0x7fffffff, last = -1;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        run += w[k];
        const int token = at + threadIdx.x * PER + k;
        if (w[k] > 0.0) last = token;
        if (w[k] > 0.0 && run > goal) first = min(first, token);
    }
    if (first != 0x7fffffff) atomicMin(&found[0], first);
    if (last >= 0) atomicMax(&found[1], last);
    __syncthreads();
    return found[0] != 0x7fffffff ? found[0] : found[1];
}

// A row's choice by u, of w. One workgroup; every thread gets it.
__device__ __forceinline__ int choose(const Args& a, const Table& table, const Parts& parts, int row, double sharp, const Row& r, float u) {
    if (sharp == 0.0) return r.at;
    const double goal = (double)u * r.z;
    double before;
    const int block = find_block(a, goal, [&](int k) {
        const Stat s = parts.at(k);
        return s.max > -INFINITY ? s.sum * exp2_64(((double)s.max - (double)r.max) * sharp) : 0.0;
    }, &before);
    float x[PER];
    load_run(a.logits + row * a.ld, block * BLOCK, a.vocab, -INFINITY, x);
    double w[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) w[k] = x[k] == -INFINITY ? 0.0 : exp2_64(table, ((double)x[k] - (double)r.max) * (64.0 * sharp));
    return find_token(block * BLOCK, w, before, goal);
}

// Each row's choice, a workgroup a row.
__global__ __launch_bounds__(THREADS) void verify_pick_kernel(const Args a) {
    __shared__ Table table;
    const int row = blockIdx.x;
    const float u = a.u[2 * row + 1];
    const Parts parts(a, row);
    fill(table);
    __syncthreads();
    const double sharp = sharpness(a, seq_of(a, row));
    Row r;
    const bool any = row_of(parts, sharp, &r);
    const int token = any ? choose(a, table, parts, row, sharp, r, u) : -1;
    if (threadIdx.x == 0) a.pick[row] = token;
}

// A cached position's slot.
__device__ __forceinline__ int slot_of(const Args& a, int b, int64_t at) {
    const int64_t page = a.table[(size_t)b * a.t.table_ld + (at >> a.t.page_shift)];
    return page >= 0 && page <= 0x7fffffff >> a.t.page_shift ? (int)((page << a.t.page_shift) + (at & ((1 << a.t.page_shift) - 1))) : -1;
}

// What a sequence has said, by a wave: lane l is its l-th token of the step, `path` the tokens that are kept.
__device__ __forceinline__ void put_path(const Args& a, int b, const Seq& s, uint64_t path, int token, int next) {
    const int lane = threadIdx.x & 63;
    const int count = __popcll(path);
    // the k-th kept token's place in the step
    int node = 0;
    uint64_t left = path;
    for (int k = 0; k < count; k++) {
        const int at = __ffsll((unsigned long long)left) - 1;
        node = lane == k ? at : node;
        left &= left - 1;
    }
    const int after = __shfl(node, min(lane + 1, 63));
    const int said = __shfl(token, after & 63);
    if (lane < s.news) {
        const size_t i = (size_t)s.first + lane;
        a.emit[i] = lane + 1 < count ? said : lane + 1 == count ? next : -1;
        if (a.src) {
            const bool moved = lane < count && node != lane;
            a.src[i] = moved ? slot_of(a, b, (int64_t)s.old + node) : -1;
            a.dst[i] = moved ? slot_of(a, b, (int64_t)s.old + lane) : -1;
        }
    }
    if (lane == 0) {
        a.next[b] = next;
        a.count[b] = count - 1;
        if (a.new_len) a.new_len[b] = s.old + count;
    }
}

// The sequence of a wave: its part of the step, against all starts before it.
__device__ __forceinline__ Seq sequence_of(const Args& a, int b) {
    int most = 0;
    for (int i = threadIdx.x & 63; i < b; i += 64) {
        const int start = a.t.start[i];
        if (start <= a.t.n) most = max(most, start);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = max(most, __shfl_xor(most, d));
    return sequence(a.t, b, 1, false, most);
}

// The sequence's part of the step; one whose numbers do not fit, or without tokens, keeps nothing and says nothing.
__device__ __forceinline__ Seq seq_part(const Args& a, int b) {
    const Seq s = sequence_of(a, b);
    if (s.news == 0 && (threadIdx.x & 63) == 0) {
        a.next[b] = -1;
        a.count[b] = 0;
        if (a.new_len) a.new_len[b] = a.t.len[b];
    }
    return s;
}

// Drafts without probabilities: from the rows' choices to the paths, a wave a sequence.
__global__ __launch_bounds__(64) void verify_walk_kernel(const Args a) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const Seq s = seq_part(a, b);
    if (s.news == 0) return;
    const bool there = lane < s.news;
    const size_t i = (size_t)s.first + min(lane, s.news - 1);
    const int token = a.tokens[i], pick = a.pick[i];
    // its parent: the last that it sees before itself
    const uint64_t above = (a.mask ? a.mask[i] : ~0ull) & ((1ull << lane) - 1);
    const int parent = above ? 63 - __clzll((long long)above) : -1;
    const int choice = __shfl(pick, max(parent, 0));
    const bool right = there && parent >= 0 && choice == token && token >= 0;
    // from the first token on to the child that says the choice, of equal ones the first
    uint64_t path = 1;
    int last = 0;
    while (const uint64_t children = __ballot(right && parent == last)) {
        last = __ffsll((unsigned long long)children) - 1;  // (behind its parent)
        path |= 1ull << last;
    }
    put_path(a, b, s, path, token, __shfl(pick, last));
}

// Drafts with probabilities: how far each chain is kept, a workgroup a sequence.
__global__ __launch_bounds__(THREADS) void verify_accept_kernel(const Args a) {
    __shared__ double z[64];
    __shared__ float top[64];
    __shared__ int32_t at[64], fine[64];
    __shared__ Table table;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Seq s = seq_part(a, b);
    if (s.news == 0) {
        if (threadIdx.x == 0) a.ends[b].open = 0, a.ends[b].row = -1;
        return;
    }
    const double sharp = sharpness(a, b);
    // (what says whether a draft is kept is asked for before the rows are added up)
    const size_t mine = (size_t)s.first + min(lane, s.news - 1);
    const int t = lane + 1 < s.news ? a.tokens[mine + 1] : -1;
    const bool drafted = t >= 0 && t < a.vocab;
    const float logit = drafted ? a.logits[mine * a.ld + t] : 0.0f, likely = drafted ? a.draft[mine * a.draft_ld + t] : 0.0f;
    const float u = a.u[2 * mine];
    fill(table);
    for (int k = wave; k < s.news; k += THREADS / 64) {
        Row r;
        const bool any = row_of(Parts(a, s.first + k), sharp, &r);
        if (lane == 0) z[k] = r.z, top[k] = r.max, at[k] = r.at, fine[k] = any;
    }
    __syncthreads();
    bool kept = false;
    if (drafted && fine[lane]) {
        const double w = exp2_64(table, ((double)logit - (double)top[lane]) * (64.0 * sharp));
        kept = sharp == 0.0 ? t == at[lane] : (double)u * (double)likely * z[lane] < w;
    }
    const uint64_t no = ~__ballot(kept);
    const int k = __ffsll((unsigned long long)no) - 1;  // (the last token has no successor that could be kept)
    const int row = s.first + k;
    const bool open = fine[k] && sharp > 0.0 && k + 1 < s.news;
    int next = -1;
    if (fine[k] && !open) next = choose(a, table, Parts(a, row), row, sharp, Row{top[k], at[k], z[k]}, a.u[2 * row + 1]);
    if (threadIdx.x == 0) a.ends[b] = End{z[k], top[k], row, next, open, k};
    if (wave == 0 && !open)
        put_path(a, b, s, ~0ull >> (63 - k), lane < s.news ? a.tokens[s.first + lane] : -1, next);
}

// max(0, w - Z q) of the tokens at + 16 tid + k of a sequence's last kept row
__device__ __forceinline__ double left_over(const Table& table, float l, float q, double sharp, const End& e) {
    return l == -INFINITY ? 0.0 : fmax(exp2_64(table, ((double)l - e.max) * (64.0 * sharp)) - e.z * (double)q, 0.0);
}
__global__ __launch_bounds__(THREADS) void verify_rest_kernel(const Args a) {
    __shared__ double sums[THREADS / 64];
    __shared__ Table table;
    const int b = blockIdx.y, at = blockIdx.x * BLOCK;
    const End e = a.ends[b];
    if (!e.open) return;
    const double sharp = sharpness(a, b);
    float x[PER], q[PER];
    load(a.logits + e.row * a.ld, at, a.vocab, -INFINITY, x);
    load(a.draft + e.row * a.draft_ld, at, a.vocab, 0.0f, q);
    fill(table);
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < PER; k++) sum += left_over(table, x[k], q[k], sharp, e);
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    sum = 0.0;
    for (int w = 0; w < THREADS / 64; w++) sum += sums[w];
    a.rest[(size_t)b * a.blocks + blockIdx.x] = sum;
}

// The token after a rejection, a workgroup a sequence.
__global__ __launch_bounds__(THREADS) void verify_finish_kernel(const Args a) {
    __shared__ Table table;
    const int b = blockIdx.x;
    const End e = a.ends[b];
    if (!e.open) return;
    const Seq s = sequence_of(a, b);
    const int lane = threadIdx.x & 63, said = lane < s.news ? a.tokens[s.first + lane] : -1;
    fill(table);
    __syncthreads();
    const double sharp = sharpness(a, b);
    const double* const rest = a.rest + (size_t)b * a.blocks;
    double all = 0.0;
    for (int k = threadIdx.x & 63; k < a.blocks; k += 64) all += rest[k];
    all = wave_sum(all);
    const float u = a.u[2 * e.row + 1];
    int next;
    if (all > 0.0) {
        const double goal = (double)u * all;
        double before;
        const int block = find_block(a, goal, [&](int k) { return rest[k]; }, &before);
        float x[PER], q[PER];
        load_run(a.logits + e.row * a.ld, block * BLOCK, a.vocab, -INFINITY, x);
        load_run(a.draft + e.row * a.draft_ld, block * BLOCK, a.vocab, 0.0f, q);
        double w[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) w[k] = left_over(table, x[k], q[k], sharp, e);
        next = find_token(block * BLOCK, w, before, goal);
    } else {  // the drafts' probabilities are the target's own
        next = choose(a, table, Parts(a, e.row), e.row, sharp, Row{(float)e.max, 0, e.z}, u);
    }
    if (threadIdx.x < 64) put_path(a, b, s, ~0ull >> (63 - e.kept), said, next);
}

}  // namespace

extern "C" int qh_verify(qh_ctx* ctx, void* stream, const float* logits, size_t ld, size_t vocab, const qh_tree* step, int page,
                         const int32_t* tokens, const float* draft, size_t draft_ld, const float* temp, const float* u, int32_t* next,
                         int32_t* count, int32_t* emit, int32_t* src, int32_t* dst, int32_t* new_len) {
    if (!step) return fail(QH_EINVAL, "verify: null step");
    if (step->n == 0 || step->n_seq == 0) return QH_OK;
    if (!logits || !tokens || !u || !next || !count || !emit || !step->start || !step->len) return fail(QH_EINVAL, "verify: null");
    if (!src != !dst) return fail(QH_EINVAL, "verify: moves need both src and dst");
    if (src && !step->table) return fail(QH_EINVAL, "verify: moves need the step's tables");
    if (vocab < 1 || vocab > (size_t)BLOCK * MAX_BLOCKS) return fail(QH_EINVAL, "verify: %zu logits of a row (1 to 2^22)", vocab);
    if (ld < vocab || ld > (size_t)1 << 32 || (draft && (draft_ld < vocab || draft_ld > (size_t)1 << 32)))
        return fail(QH_EINVAL, "verify: rows of %zu logits, %zu probabilities for a vocabulary of %zu", ld, draft ? draft_ld : vocab, vocab);
    if (step->n_seq < 0 || step->n_seq > TREE_MAX_SEQS)
        return fail(QH_EINVAL, "verify: %d sequences (up to %d)", step->n_seq, TREE_MAX_SEQS);
    if (step->max_new < 1 || step->max_new > TREE_MAX_NEW)
        return fail(QH_EINVAL, "verify: up to %d tokens of a sequence, asked for %d", TREE_MAX_NEW, step->max_new);
    if (step->n > (size_t)step->n_seq * step->max_new)
        return fail(QH_EINVAL, "verify: %zu tokens of %d sequences of up to %d", step->n, step->n_seq, step->max_new);
    if (page < KV_TILE || page > 1024 || (page & (page - 1)))
        return fail(QH_EINVAL, "verify: pages of %d tokens (a power of two from 64 to 1024)", page);
    if (step->table_ld < 1 || step->table_ld > ((size_t)1 << 30) / page)
        return fail(QH_EINVAL, "verify: tables of %zu pages of %d tokens (1 to 2^30 positions)", step->table_ld, page);
    if (draft && step->mask) return fail(QH_EINVAL, "verify: drafts with probabilities are chains: no mask");
    if (!ctx) return fail(QH_EINVAL, "verify: null context");
    Args a = {};
    a.logits = logits, a.draft = draft, a.tokens = tokens, a.temp = temp, a.u = u;
    a.ld = (int64_t)ld, a.draft_ld = (int64_t)draft_ld, a.vocab = (int32_t)vocab, a.blocks = (int32_t)((vocab + BLOCK - 1) / BLOCK);
    a.t = TreeArrays{step->start, step->len, (int64_t)step->table_ld, __builtin_ctz((unsigned)page), (int)step->n, step->n_seq,
                     step->max_new, 1};
    a.table = step->table, a.mask = step->mask;
    a.next = next, a.count = count, a.emit = emit, a.src = src, a.dst = dst, a.new_len = new_len;
    const size_t n = step->n, seqs = (size_t)step->n_seq;
    const size_t stats = n * a.blocks * sizeof(Stat), ends = seqs * sizeof(End), rest = seqs * a.blocks * 8, picks = n * 4;
    if (stats + ends + rest + picks > PF_SK_PART_BYTES)
        return fail(QH_EINVAL, "verify: %zu rows of %zu logits are too many for one call", n, vocab);
    uint8_t* const scratch = (uint8_t*)ctx_partials(ctx);
    a.stats = (Stat*)scratch;
    a.ends = (End*)(scratch + stats);
    a.rest = (double*)(scratch + stats + ends);
    a.pick = (int32_t*)(scratch + stats + ends + rest);
    const hipStream_t s = (hipStream_t)stream;
    launch_kernel(verify_stats_kernel, dim3((unsigned)(a.blocks * n)), dim3(THREADS), s, a);
    if (draft) {
        launch_kernel(verify_accept_kernel, dim3((unsigned)seqs), dim3(THREADS), s, a);
        launch_kernel(verify_rest_kernel, dim3((unsigned)a.blocks, (unsigned)seqs), dim3(THREADS), s, a);
        launch_kernel(verify_finish_kernel, dim3((unsigned)seqs), dim3(THREADS), s, a);
    } else {
        launch_kernel(verify_pick_kernel, dim3((unsigned)n), dim3(THREADS), s, a);
        launch_kernel(verify_walk_kernel, dim3((unsigned)seqs), dim3(64), s, a);
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "verify launch: %s", hipGetErrorString(e));
    return QH_OK;
}
