// Attention of a step's tokens (single tokens, chains and trees of drafted tokens) over the paged, quantised KV cache, and
// the joining of its partial results (qh_tree_attn).
//
// For each row (a token and one of its query heads) over the positions t that it sees:
//   s_t = c q.k_t,  o = sum_t exp(s_t) v_t / sum_t exp(s_t),  then o * sigmoid(gate) where a gate is given,
// with k_t = sk_t * (codes), v_t = sv_t * (codes). One pass over the cache: the running maximum m and sum l of the softmax
// beside the unnormalised o, rescaled when m grows. The codes go into the products as they are: sk_t multiplies the finished
// scores, sv_t the probabilities.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

#include "gemm.h"
#include "internal.h"
#include "kv.h"

using namespace qh;

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The plan in memory, for join_kernel: -, workgroups, -, -, 1 / groups in 64 bits, -, -; then PLAN_SEQ numbers of each sequence,
// one after the other for all of them: first group; first token | tokens << 20; chunks; groups.
constexpr int PLAN_HEAD = 8, PLAN_SEQ = 4;

// buffer resource word 3 (32-bit data format, no swizzle), and the cache policy of loads past the caches
constexpr int BUF_RSRC_WORD3 = 0x00020000;
constexpr int CPOL_NT = 2;

// Workgroups of a CU: what a kernel's registers leave room for.
constexpr int wgs_per_cu(int d, int r, int w) { return w == 8 ? 1 : d == 64 ? (r == 1 ? 4 : 3) : d == 128 && r == 1 ? 3 : 2; }

struct Args {
    const __bf16* q;     // [n][heads][D]
    const __bf16* gate;  // the same, or null
    __bf16* out;
    Kv kv;
    TreeArrays t;
    const int32_t* table;  // [n_seq][table_ld]
    const uint64_t* mask;  // [n], or null: a chain
    float scale;           // softmax scale * log2(e)
    uint32_t group_inv;    // 2^20 / group rounded up: (r * group_inv) >> 20 is r / group for the rows r < 64 group <= 4096
    int32_t row_tiles;     // log2 of a chunk's tiles of 16 rows
    float* part;           // [2 * workgroups][rows of a chunk][D], then at byte ml_at f2 [2 * workgroups][rows of a chunk]:
    int32_t ml_at;         // maximum (log2) and sum
    int32_t* plan;         // [PLAN_HEAD + n_seq * PLAN_SEQ]
};

// The compiler moves nothing across: left free it converts a whole tile's codes ahead of its products and spills.
#define HOLD() __builtin_amdgcn_sched_barrier(0)

// A barrier for what the workgroup's waves wrote to LDS; loads and stores to memory stay in flight over it.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Eight codes as exact f16 operands: e4m3 by its conversion; an int8 code c = q + 128 is put into f16's low bits as it is,
// the subnormal number c 2^-24, which the matrix instructions multiply exactly. The products' sums then hold 2^-24 (q + 128):
// the 128 is taken off by the scores' first value, and from the outputs at the end, beside a sum of the probabilities.
// (Against codes made whole numbers of, one instruction a pair instead of two.)
template <int FMT>
__device__ __forceinline__ h8 operands(uint32_t a, uint32_t b) {
    h2 p[4];
    if constexpr (FMT == QH_KV_I8) {
        p[0] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0, a, 0x0c010c00u));
        p[1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0, a, 0x0c030c02u));
        p[2] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0, b, 0x0c010c00u));
        p[3] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0, b, 0x0c030c02u));
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    }
    return h8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
}
constexpr int code_exp(int fmt) { return fmt == QH_KV_I8 ? 24 : 0; }  // operands are 2^-this of the codes' values

// A lane's neighbour's value in the wave (DPP): CTRL of quad_perm, row_half_mirror, row_mirror, row_shr, row_bcast.
template <int CTRL, int ROWS = 15>
__device__ __forceinline__ int dpp(int old, int v) {
    return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 15, false);
}
// f over the N = 4, 8 or 16 neighbouring lanes that share a row of queries
template <int N, class F>
__device__ __forceinline__ int over_lanes(int v, F&& f) {
    v = f(v, dpp<0xb1>(v, v));
    v = f(v, dpp<0x4e>(v, v));
    if (N > 4) v = f(v, dpp<0x141>(v, v));
    if (N > 8) v = f(v, dpp<0x140>(v, v));
    return v;
}

// the largest / sum over the four lanes that hold one row (lanes l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float row_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

__device__ __forceinline__ float wave_max(float v) {
    v = __int_as_float(over_lanes<16>(__float_as_int(v), [](int x, int y) { return __float_as_int(fmaxf(__int_as_float(x), __int_as_float(y))); }));
    return row_max(v);
}

// f over the 16 lanes of each quarter of the wave
template <class F>
__device__ __forceinline__ float lanes16(F&& f, float v) {
    return __int_as_float(over_lanes<16>(__float_as_int(v), [&](int x, int y) { return __float_as_int(f(__int_as_float(x), __int_as_float(y))); }));
}
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// What a workgroup of 16 R rows holds in LDS.
template <int D, int R, int W>
struct Shared {
    int32_t base[2][TREE_MAX_SEQS];  // of each sequence: its first group (of 4, of 8 tiles),
    int32_t who[TREE_MAX_SEQS];   // first token | tokens << 20,
    int32_t old[TREE_MAX_SEQS];   // positions before them
    int32_t wave_sum[3][W];
    float factor[16 * R], start[16 * R];  // of each row: what its scores are multiplied by, and begin with
    uint64_t sees[16 * R];                // which of its sequence's tokens of this step a row sees,
    int32_t sees_exp[16 * R];             // and their values' largest scale (scale_exp)
    f4 largest[16 * R][W / 4];            // each wave's largest score of the row,
    f4 largest_scale[W / 4];              // and largest scale of its values
    f4 sums[16 * R][W / 2];               // each wave's sum of the row's probabilities, and of their roundings
    h8 q[R][D / 64][2][64];
    float tile_scale[W][2][KV_TILE];
    h8 p[W][R][2][64];  // probabilities of each wave's tile
};

// The sequences' places in LDS, and the number of their groups: of four tiles in .narrow, of eight in .wide. Up to 64 sequences
// each wave makes the whole list for itself, more are shared by the workgroup's threads. Starts that are not in order are
// found on the way; the list is then made anew, each sequence against all starts before it.
struct Totals {
    int narrow, wide, units;  // (units: of the first sequence)
    int rest;                 // REST_ bits
};
constexpr int REST_DISORDER = 1, REST_SOME = 2;  // starts are not in order; some tokens are in no sequence that has work
template <int D, int R, int W>
__device__ __forceinline__ Totals plan(const Args& a, Shared<D, R, W>& sh) {
    constexpr int THREADS = 64 * W;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool few = a.t.n_seq <= 64;
    for (bool in_order = true;; in_order = false) {
        int before[2] = {0, 0}, units = 0, rest = 0;
        for (int c = 0; c < a.t.n_seq; c += THREADS) {
            const int b = c + (few ? lane : (int)threadIdx.x);
            int v[2] = {0, 0}, run[2], sum[2], some = 0;
            Seq s = {};
            if (b < a.t.n_seq) {
                s = sequence(a.t, b, 16 * R, false, in_order ? 0 : start_before(a.t, b));
                units = a.kv.heads * s.chunks;
                v[0] = units * s.groups;
                v[1] = units * ((s.groups + 1) >> 1);
                some = s.bad || (b == 0 && s.first > 0) || (b == a.t.n_seq - 1 && s.first + s.news < a.t.n);
            }
            some = (__any(some) ? REST_SOME : 0) | (__any(s.disorder) ? REST_DISORDER : 0);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                run[k] = v[k];  // inclusive over the wave
                run[k] += dpp<0x111>(0, run[k]);
                run[k] += dpp<0x112>(0, run[k]);
                run[k] += dpp<0x114>(0, run[k]);
                run[k] += dpp<0x118>(0, run[k]);
                run[k] += dpp<0x142, 10>(0, run[k]);
                run[k] += dpp<0x143, 12>(0, run[k]);
                sum[k] = __builtin_amdgcn_readlane(run[k], 63);
                run[k] += before[k] - v[k];
            }
            if (!few) {
                if (lane == 0) sh.wave_sum[0][wave] = sum[0], sh.wave_sum[1][wave] = sum[1], sh.wave_sum[2][wave] = some;
                lds_barrier();
                sum[0] = sum[1] = some = 0;
                for (int w = 0; w < W; w++) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        if (w < wave) run[k] += sh.wave_sum[k][w];
                        sum[k] += sh.wave_sum[k][w];
                    }
                    some |= sh.wave_sum[2][w];
                }
                lds_barrier();
            }
            if (b < a.t.n_seq) {
                sh.base[0][b] = run[0];
                sh.base[1][b] = run[1];
                sh.who[b] = s.first | s.news << 20;
                sh.old[b] = s.old;
            }
            before[0] += sum[0], before[1] += sum[1], rest |= some;
        }
        if (!few) lds_barrier();
        rest = __builtin_amdgcn_readfirstlane(rest);
        if (in_order && (rest & REST_DISORDER)) continue;
        return Totals{__builtin_amdgcn_readfirstlane(before[0]), __builtin_amdgcn_readfirstlane(before[1]),
                      __builtin_amdgcn_readfirstlane(units), rest};
    }
}

// x / y of numbers that all lanes have alike, where the quotient is below 2^20
__device__ __forceinline__ int divide(int x, int y) {
    int q = (int)((float)x * __builtin_amdgcn_rcpf((float)y));  // off by one at most
    q -= q * y > x ? 1 : 0;
    q += x - q * y >= y ? 1 : 0;
    return __builtin_amdgcn_readfirstlane(q);
}

// The sequence that a group or token `at` lies in: the last that begins at or before it, -1 for none (empty ones share their
// successor's beginning).
template <class F>
__device__ __forceinline__ int find_seq(int n_seq, int at, F&& begin) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int c = 0; c < n_seq; c += 64) {
        const int b = c + lane;
        n += __popcll(__ballot(b < n_seq && begin(min(b, n_seq - 1)) <= at));
    }
    return n - 1;
}
constexpr int first_of(int who) { return who & 0xfffff; }

__device__ __forceinline__ b4 load_gate(const Args& a, size_t at) { return a.gate ? *(const b4*)(a.gate + at) : b4{}; }

// The least e >= NO_EXP for which a scale is below 2^e (to 2^126; such powers of two have exact reciprocals).
constexpr int NO_EXP = -126;
__device__ __forceinline__ int scale_exp(float s) { return s > 0.0f ? max(min(__builtin_amdgcn_frexp_expf(s), 126), NO_EXP) : NO_EXP; }

// A row's output: four of its dimensions, divided by the sum and gated.
__device__ __forceinline__ void put_out(const Args& a, size_t at, f4 v, float total, b4 gate) {
    v *= total > 0.0f || total != total ? __builtin_amdgcn_rcpf(total) : 0.0f;
    if (a.gate) {
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] *= sigmoid((float)gate[u]);
    }
    *(b4*)(a.out + at) = __builtin_convertvector(v, b4);
}

// The outputs of tokens that no sequence has work for, the grid's workgroups in turn: zeros for padding, else NaN.
template <int D, int R, int W>
__device__ __forceinline__ void put_rest(const Args& a, const Shared<D, R, W>& sh, int rest) {
    for (int token = blockIdx.x; token < a.t.n; token += gridDim.x) {
        const int b = find_seq(a.t.n_seq, token, [&](int b) { return first_of(sh.who[b]); });
        if (b >= 0 && token - first_of(sh.who[b]) < sh.who[b] >> 20) continue;
        const uint32_t fill = padding(a.t, token, rest & REST_DISORDER) ? 0 : 0x7fc07fc0u;
        const int pieces = a.kv.heads * a.t.group * (D / 8);
        u4* const out = (u4*)a.out + (size_t)token * pieces;
        for (int i = threadIdx.x; i < pieces; i += 64 * W) out[i] = u4{fill, fill, fill, fill};
    }
}

// The work is a row of groups: for each sequence, kv head and chunk of 16 R rows, the cache in groups of 4 x 64 tokens. The
// workgroups share it in equal parts, across the borders of sequences; consecutive parts on one XCD, whose L2 then serves
// the chunks that read the same cache. A tile for each wave at a time, a wave makes the scores of its own for all rows; the
// waves agree on the rows' largest scores, put their probabilities into LDS, and each then multiplies those of all tiles by
// its own share of the values' dimensions. So a code is read and converted once for all rows, a wave's part of the outputs
// is small, and there is nothing to join over the waves but the sums. (Each wave with whole rows and tiles of its own, joined
// over LDS, took 12.0 us against 10.3 for a short sequence, 45 against 33 for 64 drafted tokens at 8,150.) Keys are read a
// group ahead, values too or while the scores are made.
// What covers a sequence's whole cache is written out, the rest as partial results for join_kernel: at most one at the start
// of a workgroup's part and one at its end. (Summed by the last workgroup of a row to arrive instead, without a second launch:
// one workgroup reads them all then, and waits for stores and counters first. One token at 4,099 positions 13.7 us against
// 12.8, at 16,000 18.7 against 15.3, at 131,000 54.5 against 51.9.)
// Bound by HBM where the cache is long (131,000 positions of 24 x 256, e4m3: 272 MB in 45 us, 6.0 TB/s), by its chain of memory
// trips where it is short (77 positions: 7.8 us), and with many rows by what goes on beside the matrix products: operands made
// of codes, exponentials (64 tokens at 8,150: 12.8 GFLOP in 32 us).
template <int D, int FMT, int R, int W>
__global__ __launch_bounds__(64 * W, W / 4 * wgs_per_cu(D, R, W)) void tree_attn_kernel(const Args args) {
    constexpr int THREADS = 64 * W;
    constexpr int C = D / 64, ROWS = 16 * R, SL = D / 16 / W;  // SL: sixteenths of the dimensions that a wave multiplies
    constexpr int CHAINS = R == 1 ? 2 : 1;  // sums of an output, so that products need not wait for one another
    constexpr bool EARLY = R == 1 || D < 256;  // registers for a group's values beside its keys
    constexpr uint32_t NONE = ~0u;
    __shared__ Shared<D, R, W> sh;
    const Args& a = args;
    // all lines of the arguments are fetched at once: each is a trip to memory when first touched
    const auto* const line = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" ::"s"(line[0]), "s"(line[16]), "s"(line[32]));
    static_assert(sizeof(Args) > 128);
    // groups of four tiles where there are few, so that they reach more CUs; of eight where a workgroup has several: the parts are
    // then whole turns of eight waves too
    const Totals totals = plan<D, R, W>(a, sh);
    const bool wide = totals.narrow > (int)gridDim.x;
    const int groups_in_all = wide ? totals.wide : totals.narrow;
    const int workgroups = __builtin_amdgcn_readfirstlane(used_workgroups(gridDim.x, groups_in_all, a.t.n_seq, totals.units));
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) {
            a.plan[1] = workgroups;
            *(double*)(a.plan + 4) = 1.0 / groups_in_all;
        }
        for (int i = threadIdx.x; i < a.t.n_seq; i += THREADS) {
            const int who = sh.who[i], news = who >> 20;
            int32_t* const seq = a.plan + PLAN_HEAD + i;
            seq[0] = sh.base[wide][i], seq[a.t.n_seq] = who;
            seq[2 * a.t.n_seq] = (news * a.t.group + ROWS - 1) / ROWS, seq[3 * a.t.n_seq] = group_count(sh.old[i] + news, wide);
        }
    }
    if (totals.rest) put_rest(a, sh, totals.rest);
    // consecutive parts on one XCD (workgroups b, b + 8, .. run on the same one)
    const int xcd = blockIdx.x & 7, at_xcd = blockIdx.x >> 3;
    if (at_xcd >= (workgroups >> 3) + (xcd < (workgroups & 7) ? 1 : 0)) return;
    const int workgroup = xcd * (workgroups >> 3) + min(xcd, workgroups & 7) + at_xcd;
    // (what all lanes have alike is said to be so where it comes through LDS or a division: addresses are then scalar)
    const int lo = __builtin_amdgcn_readfirstlane(first_group(workgroup, groups_in_all, workgroups));
    const int hi = __builtin_amdgcn_readfirstlane(first_group(workgroup + 1, groups_in_all, workgroups));
    for (int at = lo; at < hi;) {
        // (said anew in each turn, so that nothing that follows is kept in registers across them: most workgroups take one. The
        // arguments are read again where they are used.)
        int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        int all = groups_in_all, used = workgroups, w = __builtin_amdgcn_readfirstlane(workgroup), group_tiles = __builtin_amdgcn_readfirstlane(GROUP_TILES << (wide ? 1 : 0));
        const auto* again = line;
        asm volatile("" : "+v"(tid), "+s"(wave), "+s"(all), "+s"(used), "+s"(w), "+s"(group_tiles), "+s"(again));
        const Args& a = *(const Args*)again;
        const int page_shift = a.kv.page_shift;
        const int lane = tid & 63, col = lane & 15, g = lane >> 4, page_tiles = 1 << (page_shift - 6);
        const int b = find_seq(a.t.n_seq, at, [&](int b) { return sh.base[wide][b]; });
        const int who = __builtin_amdgcn_readfirstlane(sh.who[b]), old = __builtin_amdgcn_readfirstlane(sh.old[b]);
        const int past = at - __builtin_amdgcn_readfirstlane(sh.base[wide][b]);
        const int first = first_of(who), news = who >> 20, total = old + news;
        const int chunks = (news * a.t.group + ROWS - 1) / ROWS;
        const int groups = group_count(total, wide), unit = divide(past, groups), g0 = past - unit * groups;
        const int g1 = min(groups, g0 + hi - at);
        const int head = chunks == 1 ? unit : divide(unit, chunks), row0 = (unit - head * chunks) * ROWS;
        const int live = min(ROWS, news * a.t.group - row0);
        const int t_end = min((total + KV_TILE - 1) / KV_TILE, g1 * group_tiles);

        // Whether rows may see different tokens here (a token alone in its step, without a mask, is seen by all rows there are): then
        // lane l has the scale of the step's l-th token's value (0: of a page that the cache has not). Its page is asked for ahead
        // of the tiles' places, whose wait is then for both.
        const bool apart = (news > 1 || a.mask) && t_end * KV_TILE > old;
        const int fresh_at = old + min(lane, news - 1);
        int fresh_page = 0;
        if (apart) fresh_page = a.table[(size_t)b * a.t.table_ld + (fresh_at >> page_shift)];

        // where tiles lie, 64 at a time: lane l has the l-th's place in the cache (of its keys) in tiles
        uint32_t places = 0;
        auto load_places = [&](int t) {
            const int mine = min(t + lane, t_end - 1);
            const int32_t pg = a.table[(size_t)b * a.t.table_ld + (mine >> (page_shift - 6))];
            places = (((uint32_t)pg * a.kv.heads + head) * 2 << (page_shift - 6)) + (mine & (page_tiles - 1));
            if (pg < 0 || ((int64_t)pg << page_shift) >= a.kv.slots) places = NONE;
        };
        load_places(g0 * group_tiles);
        auto node_of = [&](int r) { return (int)((uint32_t)r * a.group_inv >> 20); };  // r / group
        // first element of a row's query, gate and output
        auto row_at = [&](int r) {
            const int node = node_of(row0 + r);
            return ((size_t)(first + node) * a.kv.heads * a.t.group + head * a.t.group + (row0 + r - node * a.t.group)) * D;
        };
        // the queries: a thread has 16 dimensions of a row
        constexpr int PER_ROW = D / 16, PASS = THREADS / PER_ROW;
        const int q_row = tid / PER_ROW, q_part = tid % PER_ROW;
        b8 raw[2];
        uint64_t mask;
        auto load_query = [&](int r) {
            const int row = min(r, live - 1), node = node_of(row0 + row);
            const __bf16* const qp = a.q + row_at(row) + q_part * 16;
            raw[0] = *(const b8*)qp, raw[1] = *(const b8*)(qp + 8);
            mask = a.mask ? a.mask[first + node] : ~0ull >> (63 - node);
        };
        load_query(q_row);

        u4 kc[4][C], vc[W][SL];
        float sk, sv;
        const uint32_t in_tile = col * 64 + g * 16;
        // 1 KiB pieces of a tile, as buffer loads: of a tile that is not there they read nothing
        auto tile_at = [&](uint32_t place, int from, bool there) {
            return __builtin_amdgcn_make_buffer_rsrc(a.kv.codes + (size_t)place * (KV_TILE * D) + from, 0, there ? KV_TILE * D - from : 0,
                                                     BUF_RSRC_WORD3);
        };
        // With chunks of 16 rows past the caches. One chunk reads its codes once (24 x 256, one token at 16,000 15.3 us against 16.1
        // through them, 32 x 128 13.6 against 14.8); where a head has several, it depends (24 x 256, 5 tokens at 4,000 13.9 against
        // 14.2, but at 1,000 13.4 against 12.6, 13 at 1,000 13.9 against 13.6).
        auto piece = [&](__amdgpu_buffer_rsrc_t tile, int at) {
            return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(tile, in_tile + (at & 4095), at & ~4095, R == 1 ? CPOL_NT : 0));
        };
        // the wave's tile's keys and scales (lane l: token l's); a page that the cache has not gives NaN
        auto load_keys = [&](int turn) {
            const int t = turn + wave;
            const uint32_t at = __builtin_amdgcn_readlane(places, (t - g0 * group_tiles) & 63);
            const bool none = at == NONE;
            const uint32_t place = none ? 0 : at;
            const auto tile = tile_at(place, 0, t < t_end);
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int sub = 0; sub < 4; sub++) kc[sub][c] = piece(tile, sub * 16 * D + c * 1024);
            const float* const sc = a.kv.scales + (size_t)place * KV_TILE;
            sk = none ? NAN : sc[lane];
            sv = t * KV_TILE + lane < total ? sc[page_tiles * KV_TILE + lane] : 0.0f;
        };
        const int slice = wave * SL;
        auto load_values = [&](int turn) {
#pragma unroll
            for (int v = 0; v < W; v++) {
                const int t = turn + v;
                const uint32_t at = __builtin_amdgcn_readlane(places, (t - g0 * group_tiles) & 63);
                const auto tile = tile_at((at == NONE ? 0 : at) + page_tiles, slice * 1024, t < t_end);
#pragma unroll
                for (int i = 0; i < SL; i++) vc[v][i] = piece(tile, i * 1024);
            }
        };
        float fresh = 0.0f;
        if (apart && lane < news && fresh_page >= 0 && ((int64_t)fresh_page << page_shift) < a.kv.slots)
            fresh = a.kv.scales[((((size_t)fresh_page * a.kv.heads + head) * 2 + 1) << page_shift) + (fresh_at & ((1 << page_shift) - 1))];
        load_keys(g0 * group_tiles);
        if (EARLY) load_values(g0 * group_tiles);

        // the queries, scaled by a power of two into f16's range (the factor goes to the scores)
        for (int r = q_row;;) {
            // bf16 with the sign taken off compares as a whole number; from 0x7f80 on it is not finite
            typedef uint16_t us2 __attribute__((ext_vector_type(2)));
            us2 m = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, __builtin_bit_cast(u4, raw[i >> 2])[i & 3] & 0x7fff7fffu));
            const int top = over_lanes<PER_ROW>(max(m.x, m.y), [](int x, int y) { return max(x, y); });
            const int e = top < 0x7f80 ? __builtin_amdgcn_frexp_expf(__uint_as_float((uint32_t)top << 16)) - 15 : 0;
            float sum = 0.0f;
            h8 q[2];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                q[i >> 3][i & 7] = (_Float16)__builtin_ldexpf((float)raw[i >> 3][i & 7], -e);
                if (FMT == QH_KV_I8) sum += (float)q[i >> 3][i & 7];
            }
            if (FMT == QH_KV_I8)
                sum = __int_as_float(over_lanes<PER_ROW>(__float_as_int(sum), [](int x, int y) {
                    return __float_as_int(__int_as_float(x) + __int_as_float(y));
                }));
            if (r < ROWS) {
                sh.q[r >> 4][q_part >> 2][0][(q_part & 3) * 16 + (r & 15)] = q[0];
                sh.q[r >> 4][q_part >> 2][1][(q_part & 3) * 16 + (r & 15)] = q[1];
                if (q_part == 0) {
                    const uint64_t sees = mask & ~0ull >> (64 - news);
                    // (a row that sees nothing has nothing that is not finite either)
                    sh.factor[r] = top >= 0x7f80 && (old || sees) ? NAN : fminf(fmaxf(__builtin_ldexpf(a.scale, e + code_exp(FMT)), 1e-37f), 3e38f);
                    sh.start[r] = -0x1p-17f * sum;
                    sh.sees[r] = sees, sh.sees_exp[r] = NO_EXP;
                }
            }
            r += PASS;
            if (r - q_row >= ROWS) break;
            load_query(r);
        }
        lds_barrier();
        // A row's probabilities are rounded relative to the values that it sees: to the largest scale of those that all rows see, so
        // far (`ref`), and of the step's tokens that it sees itself (sees_exp). A sibling's, however large, takes no bits from it.
        // (Where one wave finds sees_exp from the scales' exponents, 5 tokens at 77 positions take 9.0 us; with a maximum over each
        // row's tokens in the loop 9.2, over LDS 9.1; with one maximum for all rows, at the cost of those bits, 8.7.)
        if (apart && wave == 0) {
            // from the largest power of two down: which rows see a token of it
            int mine = scale_exp(fresh < INFINITY ? fresh : 0.0f), exp[R];
            uint64_t sees[R];
#pragma unroll
            for (int rt = 0; rt < R; rt++) exp[rt] = NO_EXP, sees[rt] = sh.sees[rt * 16 + col];
            for (;;) {
                int most = over_lanes<16>(mine, [](int x, int y) { return max(x, y); });
                most = max(max(__builtin_amdgcn_readlane(most, 0), __builtin_amdgcn_readlane(most, 16)),
                           max(__builtin_amdgcn_readlane(most, 32), __builtin_amdgcn_readlane(most, 48)));
                const uint64_t tokens = __ballot(mine == most);
                bool open = false;
#pragma unroll
                for (int rt = 0; rt < R; rt++) {
                    exp[rt] = exp[rt] == NO_EXP && (sees[rt] & tokens) ? most : exp[rt];
                    open |= exp[rt] == NO_EXP;
                }
                if (most == NO_EXP || !__any(open)) break;
                mine = mine == most ? NO_EXP : mine;
            }
#pragma unroll
            for (int rt = 0; rt < R; rt++) sh.sees_exp[rt * 16 + col] = exp[rt];  // (read behind the loop's first barrier)
        }
        float top[R], sum[R], rounded[R];  // rounded: the sum of the probabilities as they are multiplied
        f4 o[R][SL][CHAINS];
        int ref = NO_EXP;  // values' scales are taken relative to 2^ref, or the row's own sees_exp above it: probabilities fit f16
#pragma unroll
        for (int rt = 0; rt < R; rt++) {
            top[rt] = -INFINITY, sum[rt] = rounded[rt] = 0.0f;
#pragma unroll
            for (int i = 0; i < SL; i++)
#pragma unroll
                for (int k = 0; k < CHAINS; k++) o[rt][i][k] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        const int whole_lane = lane;
        for (int turn = g0 * group_tiles; turn < t_end; turn += W) {
            // (said anew here and behind the loop: what follows from it would be kept in registers otherwise, and they run out)
            int said = whole_lane;
            asm volatile("" : "+v"(said));
            const int lane = said, col = lane & 15, g = lane >> 4;
            const int t0 = (turn + wave) * KV_TILE;
            const bool more = turn + W < t_end, own = turn + wave < t_end;
            // A wave at its softmax goes before one at its products, which the matrix units keep busy for longer than they take to
            // issue (64 tokens at 8,150, 24 x 256: 37.5 us against 39.8; 13 at 30,000: 40.0 against 40.9).
            __builtin_amdgcn_s_setprio(0);
            // s^T = k q^T: lane (col, g) gets row `col` of tokens 16 sub + 4 g + i
            f4 x[R][4];
#pragma unroll
            for (int rt = 0; rt < R; rt++) {
                const float start = FMT == QH_KV_I8 ? sh.start[rt * 16 + col] : 0.0f;
#pragma unroll
                for (int sub = 0; sub < 4; sub++) x[rt][sub] = f4{start, start, start, start};
            }
#pragma unroll
            for (int c = 0; c < C; c++) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    h8 q[R], codes[4];
#pragma unroll
                    for (int rt = 0; rt < R; rt++) q[rt] = sh.q[rt][c][k][lane];
#pragma unroll
                    for (int sub = 0; sub < 4; sub++) codes[sub] = operands<FMT>(kc[sub][c][2 * k], kc[sub][c][2 * k + 1]);
#pragma unroll
                    for (int rt = 0; rt < R; rt++)
#pragma unroll
                        for (int sub = 0; sub < 4; sub++)
                            x[rt][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes[sub], q[rt], x[rt][sub], 0, 0, 0);
                }
                HOLD();
            }
            __builtin_amdgcn_s_setprio(1);
            if (!EARLY) load_values(turn);

            // the scores' and the values' scales, as the lanes need them
            float(&ts)[2][KV_TILE] = sh.tile_scale[wave];
            ts[0][lane] = sk, ts[1][lane] = sv;
            const float shared = (!apart || t0 + lane < old) && sv < INFINITY ? sv : 0.0f;
            float most = 0.0f;
            if (own && __any(shared > __builtin_ldexpf(1.0f, ref))) most = wave_max(shared);
            __builtin_amdgcn_wave_barrier();
            const bool whole = own && t0 + KV_TILE <= old;  // every row sees every token
#pragma unroll
            for (int rt = 0; rt < R; rt++) {
                uint64_t seen = 0;  // bit i: the row sees token t0 + i
                if (own && !whole) {
                    const int node = t0 - old;  // above -64
                    const uint64_t sees = sh.sees[rt * 16 + col];
                    seen = node >= 64 ? 0 : node >= 0 ? sees >> node : sees << -node | ((1ull << -node) - 1);
                }
                float mx = -INFINITY;
#pragma unroll
                for (int sub = 0; sub < 4; sub++) {
                    x[rt][sub] *= *(const f4*)&ts[0][sub * 16 + g * 4];
                    if (!whole) {
                        const uint32_t bits = (uint32_t)(seen >> (sub * 16 + g * 4));
#pragma unroll
                        for (int i = 0; i < 4; i++) x[rt][sub][i] = bits & (1u << i) ? x[rt][sub][i] : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) mx = fmaxf(mx, x[rt][sub][i]);
                }
                mx = row_max(mx);
                if (g == 0) ((float*)sh.largest[rt * 16 + col])[wave] = mx;
            }
            if (lane == 0) ((float*)sh.largest_scale)[wave] = most;
            HOLD();
            lds_barrier();

            const auto over = [](const f4(&v)[W / 4]) {
                float m = fmaxf(fmaxf(v[0].x, v[0].y), fmaxf(v[0].z, v[0].w));
#pragma unroll
                for (int k = 1; k < W / 4; k++) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
                return m;
            };
            const int ref_was = ref;
            ref = __builtin_amdgcn_readfirstlane(max(ref, scale_exp(over(sh.largest_scale))));
#pragma unroll
            for (int rt = 0; rt < R; rt++) {
                const float next = fmaxf(top[rt], over(sh.largest[rt * 16 + col]));
                const float factor = sh.factor[rt * 16 + col];
                const int sees_exp = sh.sees_exp[rt * 16 + col], exp = max(ref, sees_exp);
                const float inv_ref = __builtin_ldexpf(1.0f, -exp);
                float by = __builtin_ldexpf(1.0f, max(ref_was, sees_exp) - exp);
                // the maximum is followed only where it has grown by more than 2^8 (the sums and f16 hold that)
                if (__any((next - top[rt]) * factor > 8.0f)) {
                    const float al = next > top[rt] ? __builtin_amdgcn_exp2f((top[rt] - next) * factor) : 1.0f;
                    sum[rt] *= al;
                    top[rt] = next;
                    by *= al;
                }
                if (turn != g0 * group_tiles && __any(by != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < SL; i++)
#pragma unroll
                        for (int k = 0; k < CHAINS; k++) o[rt][i][k] *= by;
                    rounded[rt] *= by;
                }
                const float off = top[rt] == -INFINITY ? 0.0f : top[rt];
                h8 p[2];
#pragma unroll
                for (int sub = 0; sub < 4; sub++) {
                    const f4 vs = *(const f4*)&ts[1][sub * 16 + g * 4] * inv_ref;  // (exact)
                    float pv[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float pr = __builtin_amdgcn_exp2f((x[rt][sub][i] - off) * factor);
                        pv[i] = pr * vs[i];
                        if (!whole) pv[i] = x[rt][sub][i] == -INFINITY ? 0.0f : pv[i];
                        sum[rt] += pr;
                    }
                    const h2 a0 = __builtin_convertvector((f2{pv[0], pv[1]}), h2);
                    const h2 a1 = __builtin_convertvector((f2{pv[2], pv[3]}), h2);
                    if (FMT == QH_KV_I8) {
                        const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
                        rounded[rt] = __builtin_amdgcn_fdot2(a0, one, rounded[rt], false);
                        rounded[rt] = __builtin_amdgcn_fdot2(a1, one, rounded[rt], false);
                    }
                    h8& to = p[sub >> 1];
                    const int k = (sub & 1) * 4;
                    to[k] = a0.x, to[k + 1] = a0.y, to[k + 2] = a1.x, to[k + 3] = a1.y;
                }
                sh.p[wave][rt][0][lane] = p[0];
                sh.p[wave][rt][1][lane] = p[1];
                HOLD();
            }
            if (more) {
                if (((turn + W - g0 * group_tiles) & 63) == 0) load_places(turn + W);
                load_keys(turn + W);
            }
            lds_barrier();

            __builtin_amdgcn_s_setprio(0);
            // o^T += v^T p^T: the k index of both operands runs over tokens 16 w + 4 g + j, as the scores lie
#pragma unroll
            for (int v = 0; v < W; v++) {
                const int t = turn + v;
                if (t < t_end) {
                    if ((t + 1) * KV_TILE > total) {  // codes that no token of this sequence wrote may be anything
                        u4 keep;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int have = total - (t * KV_TILE + k * 16 + g * 4);
                            keep[k] = have >= 4 ? ~0u : have <= 0 ? 0u : (1u << (8 * have)) - 1;
                        }
#pragma unroll
                        for (int i = 0; i < SL; i++) vc[v][i] &= keep;
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        h8 codes[SL];
#pragma unroll
                        for (int i = 0; i < SL; i++) codes[i] = operands<FMT>(vc[v][i][2 * k], vc[v][i][2 * k + 1]);
#pragma unroll
                        for (int rt = 0; rt < R; rt++) {
                            const h8 p = sh.p[v][rt][k][lane];
#pragma unroll
                            for (int i = 0; i < SL; i++)
                                o[rt][i][k % CHAINS] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes[i], p, o[rt][i][k % CHAINS], 0, 0, 0);
                        }
                    }
                }
            }
            if (EARLY && more) load_values(turn + W);
        }

        // the waves' sums joined, and the outputs written, or a partial result
        const bool direct = g0 == 0 && g1 == groups;
        const int slot = 2 * w + (at != lo);
        {
            int said = whole_lane;
            asm volatile("" : "+v"(said));
            const int lane = said, col = lane & 15, g = lane >> 4;
#pragma unroll
            for (int rt = 0; rt < R; rt++) {
                const f2 s = {row_sum(sum[rt]), FMT == QH_KV_I8 ? row_sum(rounded[rt]) : 0.0f};
                if (g == 0) ((f2*)sh.sums[rt * 16 + col])[wave] = s;
            }
            constexpr bool AHEAD = R * SL <= 4;  // (registers)
            b4 gate[R][SL];
            if (AHEAD && direct)
#pragma unroll
                for (int rt = 0; rt < R; rt++)
#pragma unroll
                    for (int i = 0; i < SL; i++) gate[rt][i] = load_gate(a, row_at(min(rt * 16 + col, live - 1)) + (slice + i) * 16 + g * 4);
            lds_barrier();
#pragma unroll
            for (int rt = 0; rt < R; rt++) {
                f4 s = sh.sums[rt * 16 + col][0];
#pragma unroll
                for (int k = 1; k < W / 2; k++) s += sh.sums[rt * 16 + col][k];
                sum[rt] = s.x + s.z;
                const float back = -128.0f * (s.y + s.w);
                const int exp = max(ref, sh.sees_exp[rt * 16 + col]);
#pragma unroll
                for (int i = 0; i < SL; i++) {
                    f4 v = o[rt][i][0];
                    if (CHAINS > 1) v += o[rt][i][CHAINS - 1];
                    if (FMT == QH_KV_I8) v = v * 0x1p24f + back;
                    o[rt][i][0] = v * __builtin_ldexpf(1.0f, exp);
                }
            }
#pragma unroll
            for (int rt = 0; rt < R; rt++) {
                const int r = rt * 16 + col;
                if (r >= live) continue;
                if (direct) {
#pragma unroll
                    for (int i = 0; i < SL; i++) {
                        const size_t to = row_at(r) + (slice + i) * 16 + g * 4;
                        put_out(a, to, o[rt][i][0], sum[rt], AHEAD ? gate[rt][i] : load_gate(a, to));
                    }
                } else {
                    const uint32_t row = slot * ROWS + r;
#pragma unroll
                    for (int i = 0; i < SL; i++) *(f4*)(a.part + row * D + (slice + i) * 16 + g * 4) = o[rt][i][0];
                    if (wave == 0 && g == 0)
                        ((f2*)((uint8_t*)a.part + a.ml_at))[row] =
                            f2{top[rt] == -INFINITY ? -INFINITY : top[rt] * sh.factor[r], sum[rt]};
                }
            }
        }
        at += g1 - g0;
        if (at < hi) lds_barrier();
    }
}

// The partial results of the rows whose cache several workgroups shared: a workgroup takes W dimensions of a row, each thread
// four; the sets of W / 4 threads take partials in turn, relative to the largest maximum, and are summed in LDS. Bound by its
// trips to memory: the plan, the partials. W is 64 for few rows (24 rows of 128 partials 4.5 us against 8.5 with whole rows, 120
// of 64 4.4 against 5.5), and whole rows for many (1536 rows of 10 partials 5.6 us against 12.4, 744 of a ragged batch 3.9
// against 6.1).
template <int D, int W>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
    constexpr int V = W / 4, SETS = 256 / V, DEEP = 4;
    __shared__ f4 sums[SETS][V];
    // all lines of the arguments are fetched at once, as above
    const auto* const line = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" ::"s"(line[0]), "s"(line[16]), "s"(line[32]));
    const int rows = 16 << a.row_tiles, token = blockIdx.x, head = blockIdx.y;
    const int piece = (int)(blockIdx.z * a.group_inv >> 20), in_group = blockIdx.z - piece * a.t.group;
    const int lane = threadIdx.x & 63, set = threadIdx.x / V, d = piece * W + threadIdx.x % V * 4;
    const size_t at = (((size_t)token * a.kv.heads + head) * a.t.group + in_group) * D + d;
    const b4 gate = load_gate(a, at);
    const int used = a.plan[1];
    const double inv_all = *(const double*)(a.plan + 4);
    // the token's sequence; up to 64 sequences all their places are read at once
    const int32_t* const seqs = a.plan + PLAN_HEAD;
    int seq[PLAN_SEQ];
    if (a.t.n_seq <= 64) {
        int mine[PLAN_SEQ];
#pragma unroll
        for (int k = 0; k < PLAN_SEQ; k++) mine[k] = seqs[k * a.t.n_seq + min(lane, a.t.n_seq - 1)];
        const int b = max(0, __popcll(__ballot(lane < a.t.n_seq && first_of(mine[1]) <= token)) - 1);
#pragma unroll
        for (int k = 0; k < PLAN_SEQ; k++) seq[k] = __builtin_amdgcn_readlane(mine[k], b);
    } else {
        const int b = max(0, find_seq(a.t.n_seq, token, [&](int b) { return first_of(seqs[a.t.n_seq + b]); }));
#pragma unroll
        for (int k = 0; k < PLAN_SEQ; k++) seq[k] = seqs[k * a.t.n_seq + b];
    }
    const int base = seq[0], news = seq[1] >> 20, chunks = seq[2], groups = seq[3];
    const int node = token - first_of(seq[1]);
    if (node < 0 || node >= news) return;  // (tree_attn_kernel wrote the row)
    const int r = node * a.t.group + in_group;
    const int u0 = base + (head * chunks + (r >> (4 + a.row_tiles))) * groups, u1 = u0 + groups;
    const int w0 = owner(u0, used, inv_all), parts = owner(u1 - 1, used, inv_all) - w0 + 1;
    if (parts == 1) return;  // one workgroup wrote the row
    const int first_slot = 2 * w0 + (owner(u0 - 1, used, inv_all) == w0 ? 1 : 0), in = r & (rows - 1);  // partial_slot
    auto slot = [&](int i) { return (size_t)(i == 0 ? first_slot : 2 * (w0 + i)) * rows + in; };
    const f2* const ml = (const f2*)((const uint8_t*)a.part + a.ml_at);
    f4 y[DEEP], v = {0.0f, 0.0f, 0.0f, 0.0f};
    float m[DEEP];
    auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < DEEP; k++) {
            const int i = i0 + k * SETS;
            if (i < parts) {
                m[k] = ml[slot(i)].x;
                y[k] = *(const f4*)(a.part + slot(i) * D + d);
            }
        }
    };
    load(set);
    f2 mine = lane < parts ? ml[slot(lane)] : f2{-INFINITY, 0.0f};
    for (int i = lane + 64; i < parts; i += 64) {
        const f2 u = ml[slot(i)];
        const float best = fmaxf(mine.x, u.x);
        mine.y = (mine.x == -INFINITY ? mine.y : mine.y * __builtin_amdgcn_exp2f(mine.x - best)) +
                 (u.x == -INFINITY ? u.y : u.y * __builtin_amdgcn_exp2f(u.x - best));
        mine.x = best;
    }
    const float best = wave_max(mine.x);
    float total = mine.x == -INFINITY ? mine.y : mine.y * __builtin_amdgcn_exp2f(mine.x - best);
    total = row_sum(lanes16([](float x, float y) { return x + y; }, total));
    for (int i0 = set; i0 < parts; i0 += SETS * DEEP) {
#pragma unroll
        for (int k = 0; k < DEEP; k++)
            if (i0 + k * SETS < parts) v += (m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - best)) * y[k];
        if (i0 + SETS * DEEP < parts) load(i0 + SETS * DEEP);
    }
    sums[set][threadIdx.x % V] = v;
    __syncthreads();
    if (set) return;
    const int there = min(parts, SETS);
    f4 u[SETS];
#pragma unroll
    for (int k = 1; k < SETS; k++) u[k] = sums[k][threadIdx.x];
#pragma unroll
    for (int k = 1; k < SETS; k++)
        if (k < there) v += u[k];
    put_out(a, at, v, total, gate);
}

template <int D, int FMT>
void launch(hipStream_t stream, const Args& a, int waves, int grid, bool join) {
    auto* f = a.row_tiles == 0 ? tree_attn_kernel<D, FMT, 1, 4> : tree_attn_kernel<D, FMT, 2, 4>;
    if constexpr (D == 256)
        if (waves == 8) f = tree_attn_kernel<D, FMT, 2, 8>;
    launch_kernel(f, dim3(grid), dim3(64 * waves), stream, a);
    if (!join) return;
    const unsigned n = (unsigned)a.t.n, heads = (unsigned)a.kv.heads, group = (unsigned)a.t.group;
    if (n * heads * group <= 512) launch_kernel(join_kernel<D, 64>, dim3(n, heads, group * (D / 64)), dim3(256), stream, a);
    else launch_kernel(join_kernel<D, D>, dim3(n, heads, group), dim3(256), stream, a);
}

}  // namespace

extern "C" int qh_tree_attn(qh_ctx* ctx, void* stream, const void* q, int q_heads, const qh_kv* kv, const qh_tree* step,
                            float scale, const void* gate, void* out) {
    if (!step) return fail(QH_EINVAL, "tree_attn: null step");
    Args a = {};
    if (int e = kv_check("tree_attn", kv, &a.kv)) return e;
    if (step->n == 0 || step->n_seq == 0) return QH_OK;
    if (!q || !out || !step->start || !step->len || !step->table) return fail(QH_EINVAL, "tree_attn: null");
    if (q_heads < 1 || q_heads % kv->heads || q_heads / kv->heads > 64)
        return fail(QH_EINVAL, "tree_attn: %d query heads over %d kv heads (a multiple, up to 64 times)", q_heads, kv->heads);
    if (step->n_seq < 0 || step->n_seq > TREE_MAX_SEQS)
        return fail(QH_EINVAL, "tree_attn: %d sequences (up to %d)", step->n_seq, TREE_MAX_SEQS);
    if (step->max_new < 1 || step->max_new > TREE_MAX_NEW)
        return fail(QH_EINVAL, "tree_attn: up to %d tokens of a sequence, asked for %d", TREE_MAX_NEW, step->max_new);
    if (step->n > (size_t)step->n_seq * step->max_new)
        return fail(QH_EINVAL, "tree_attn: %zu tokens of %d sequences of up to %d", step->n, step->n_seq, step->max_new);
    if (!(scale > 0.0f) || !(scale < INFINITY)) return fail(QH_EINVAL, "tree_attn: scale %g must be positive", scale);
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)gate % 16)
        return fail(QH_EINVAL, "tree_attn: q, gate and out must be 16-byte aligned");
    if ((uint64_t)a.kv.slots / KV_TILE * 2 * kv->heads >= 0xffffffffu)  // (a tile's place is a 32-bit number)
        return fail(QH_EINVAL, "tree_attn: a cache of %zu pages of %d tokens of %d heads is too large", kv->pages, kv->page, kv->heads);
    const int64_t cap = (int64_t)step->table_ld * kv->page;  // positions that a table can name
    if (step->table_ld < 1 || step->table_ld > ((size_t)1 << 30) / kv->page)
        return fail(QH_EINVAL, "tree_attn: tables of %zu pages of %d tokens (1 to 2^30 positions)", step->table_ld, kv->page);
    const int group = q_heads / kv->heads;
    const int64_t groups = (cap + KV_TILE * GROUP_TILES - 1) / (KV_TILE * GROUP_TILES);  // of the longest sequence there can be
    const int64_t cus = ctx ? ctx_cus(ctx) : 1;
    auto units_of = [&](int rt) { return (int64_t)kv->heads * ((step->max_new * group + (16 << rt) - 1) >> (4 + rt)); };
    // Chunks of 32 rows, where there are more than 16, read the cache half as often, but leave half as many shares: from about a
    // share for each CU (24 x 256, 5 tokens at 16,000: 20.5 us against 24.4, at 4,000: 15.6 against 13.9; 32 x 128, 5 tokens at
    // 16,000: 17.4 against 18.8, at 4,000: 13.0 against 11.7). In batches of smaller heads 16 rows stay ahead longer (32 sequences of
    // 5 tokens at up to 4,000: 32 x 128 42.4 against 40.7, 16 x 64 18.7 against 16.7), which this rule does not follow.
    // Shares are counted from what the tables could hold, since the lengths are on the device: tables wider than the sequences
    // need get the forms of the longest ones (24 x 256, 5 tokens at 4,000: 14.0 us, with tables of 131,072 positions 16.8).
    const int rt = step->max_new * group > 16 && units_of(1) * step->n_seq * groups >= (kv->head_dim == 256 ? cus * 3 / 4 : cus) ? 1 : 0;
    const int rows = 16 << rt;
    // Workgroups of four waves start soon, and are out of step with one another, so that one's products run beside another's
    // softmax (24 x 256: 32 sequences of 5 tokens 33.5 us against 41.9 of eight waves, 64 tokens at 16,000 61.6 against 65.5). One
    // long chunk alone has eight waves and half as many partial results (5 tokens at 32,700: 24.3 against 25.5, at 131,000: 59.9
    // against 64.6; of 128 dimensions 70.0 against 62.0). (31 tokens at 4,000 would gain, too: 19.9 against 22.2, of 128 dimensions
    // 16.5 against 18.5; at 16,000 they lose: 42.5 against 40.2, 34.3 against 31.0.)
    const int64_t total = units_of(rt) * step->n_seq * groups;
    const int waves = rt && kv->head_dim == 256 && step->n_seq == 1 && step->max_new * group <= 32 && total >= 2 * cus ? 8 : 4;
    const int64_t units = units_of(rt);
    if (units * step->n_seq > 0x7fffffff / groups)
        return fail(QH_EINVAL, "tree_attn: %d sequences of up to %lld positions are too many for one call", step->n_seq, (long long)cap);
    if (!ctx) return fail(QH_EINVAL, "tree_attn: null context");
    a.q = (const __bf16*)q, a.gate = (const __bf16*)gate, a.out = (__bf16*)out;
    a.t = TreeArrays{step->start, step->len, (int64_t)step->table_ld, a.kv.page_shift, (int)step->n, step->n_seq, step->max_new,
                     group};
    a.table = step->table;
    a.mask = step->mask;
    a.group_inv = ((1u << 20) + group - 1) / group;
    a.scale = scale * 1.4426950408889634f;
    const int grid = (int)std::min({cus * wgs_per_cu(kv->head_dim, 1 << rt, waves), units * step->n_seq * groups, (int64_t)TREE_MAX_WGS});
    const size_t part = (size_t)2 * grid * rows * kv->head_dim * 4, ml = (size_t)2 * grid * rows * 8;
    if (part + ml + (TREE_MAX_SEQS * PLAN_SEQ + PLAN_HEAD) * 4 > PF_SK_PART_BYTES) return fail(QH_EINVAL, "tree_attn: scratch");
    a.row_tiles = rt;
    a.part = (float*)ctx_partials(ctx);
    a.ml_at = (int32_t)part;
    a.plan = (int32_t*)((uint8_t*)ctx_partials(ctx) + part + ml);
    const bool join = groups > 1 && grid > 1;
    auto go = [&](auto d) {
        if (kv->fmt == QH_KV_I8) launch<decltype(d)::value, QH_KV_I8>((hipStream_t)stream, a, waves, grid, join);
        else launch<decltype(d)::value, QH_KV_E4M3>((hipStream_t)stream, a, waves, grid, join);
    };
    if (kv->head_dim == 64) go(std::integral_constant<int, 64>{});
    else if (kv->head_dim == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "tree_attn launch: %s", hipGetErrorString(e));
    return QH_OK;
}
