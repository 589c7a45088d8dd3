// Attention of a prompt's chunk (and of batches of chunks) over the paged, quantised KV cache (qh_chunk_attn).
//
// For each row (a token and one of its query heads) over the positions t up to its token's own:
//   s_t = c q.k_t,  o = sum_t exp(s_t) v_t / sum_t exp(s_t),  then o * sigmoid(gate) where a gate is given,
// with k_t = sk_t * (codes), v_t = sv_t * (codes). One pass over the cache for each 256 rows of a kv head (128 where there are few):
// the running maximum and sum of the softmax beside the unnormalised o, rescaled when the maximum has grown by 2^15.
//
// Bound by the matrix instructions, 4 d operations for each row and position; the cache is read once for 256 rows of them (2 bytes of codes
// for 1,024 operations: far below what memory gives, and neighbours read the same tiles from L2). So everything else goes beside the
// products:
//  - A wave has 64 rows: 64 x d outputs in accumulation registers, its queries and two blocks' scores in vector registers, 512 in all for
//    d = 256, one wave for each SIMD (and 11 to 13 more, a unit's numbers, that are put by in scratch memory while its loop runs). Scores are
//    made as s^T = k q^T, so that a lane holds its row's: the softmax needs one exchange between two lanes, and its results are the next
//    product's operands as they stand.
//  - Four waves share a tile of 64 tokens in LDS, as f16 operands, two tiles in turn: codes come from memory a tile ahead, are
//    made operands beside the score products, and one barrier a tile separates the two.
//  - The rows are two sets of 32. While one's softmax runs, the other's products do: the second set's value products stand behind the next
//    block's scores. With d = 256 a block of 32 tokens is 64 products of 32 cycles; 1,274 us of 1,647 at 2,048 tokens behind
//    30,000 cached ones are the products alone (timed without the rest; the clock falls under them), 1,345 with their operands from LDS.
// Measured at 24 heads over 4 of 256, int8: those 2,048 tokens 1.65 ms, 948 TFLOP/s (a large f16 product reaches about 1,200);
// none cached 130 us (202 with a table of more than 5,120 positions, see SHORT_TILES); 131 tokens behind 120,000 607 us. The simplest form
// that was right: 4.0 ms, 266 us, 15.0 ms. 2,048 tokens behind 29,952 of 32 heads over 8, int8: of 128 dimensions 1.32 ms, 788 TFLOP/s, of 64 0.79 ms,
// 656 (a score's exponential takes as long whatever d is: at d = 64 a block's 32 take as many cycles as its 16 products).
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>
#include <utility>

#include "gemm.h"
#include "internal.h"
#include "kv.h"

using namespace qh;

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The compiler moves nothing across: left free it fetches a whole tile's operands ahead of its products and spills.
#define HOLD() __builtin_amdgcn_sched_barrier(0)
#define LIKELY(x) __builtin_expect(x, 1)  // a branch that is taken makes a wave wait for its instructions, with none beside it
#define UNLIKELY(x) __builtin_expect(x, 0)
#define INLINE __attribute__((always_inline))  // (left out of line, a lambda's captures would be in memory)

constexpr int BUF_RSRC_WORD3 = 0x00020000;  // buffer resource word 3: 32-bit data format, no swizzle

constexpr int WAVES = 4, THREADS = 64 * WAVES;
constexpr int rows_of(int sets) { return 32 * sets * WAVES; }  // of a workgroup whose waves have so many sets of 32 rows

struct Args {
    const __bf16* q;     // [n][heads][D]
    const __bf16* gate;  // the same, or null
    __bf16* out;
    Kv kv;
    TreeArrays t;
    const int32_t* table;  // [n_seq][table_ld]
    float scale;           // softmax scale * log2(e), without its power of two:
    int32_t scale_exp;
    int32_t parts;         // workgroups that the work may be shared among in equal parts; 0: each has a unit
    float* part;           // [2 parts][256 rows x D], as the lanes hold them, and of each row (maximum, sum, unit):
    f4* part_rows;         // [2 parts][256]
    struct Cut* cuts;      // [parts]
};

// Where a part begins within a unit, for join_kernel.
struct Cut {
    int32_t begin, end;  // the unit's, in the row of all (end 0: the part begins with a unit, or another before it joins this one)
    int32_t all, used;   // the row's length, and its parts
    int32_t first, head, row0, last;
};

// Four codes as exact f16 operands: an int8 code c = q + 128 becomes 1024 + c by its bits, then q; e4m3 by its conversion.
template <int FMT>
__device__ __forceinline__ h4 operands(uint32_t a) {
    h2 p[2];
    if constexpr (FMT == QH_KV_I8) {
        const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        p[0] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + off;
        p[1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + off;
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    }
    return h4{p[0].x, p[0].y, p[1].x, p[1].y};
}

// The matrix instructions are written out, so that outputs stay in accumulation registers and scores in vector registers: of a
// function's builtins the compiler puts all into one kind, and moves the other's values back and forth around every product. It
// does not know them, so what has to be waited for stands here: a register that a vector instruction wrote is read two steps later
// (OPERANDS_READY), a product is read when it is through (PRODUCTS_READY: 8 passes and 4 steps; 20 are left). A product added to the one
// before it in the same registers needs no wait.
#define OPERANDS_READY() asm volatile("s_nop 1")
#define PRODUCTS_READY() asm volatile("s_nop 15\n\ts_nop 3")
// Of products that the compiler's own instructions read, the wait has the registers as its operands: no reader is moved before it. (Outputs are
// read by assembly, `kept`, that stays behind it as it is.)
template <int SETS>
__device__ __forceinline__ void products_ready(f16 (&x)[SETS]) {
    if constexpr (SETS == 1) asm volatile("s_nop 15\n\ts_nop 3" : "+v"(x[0]));
    else asm volatile("s_nop 15\n\ts_nop 3" : "+v"(x[0]), "+v"(x[1]));
}
// (WAIT: where the compiler may fetch an operand from elsewhere right before. It does with D = 64, whose kernel has half the registers; a
// test looks at what was built.)
template <bool WAIT>
__device__ __forceinline__ void product_first(f16& x, h8 a, h8 b) {
    if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(x) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(x) : "v"(a), "v"(b));
}
template <bool WAIT>
__device__ __forceinline__ void product(f16& x, h8 a, h8 b) {
    if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(x) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(x) : "v"(a), "v"(b));
}
template <bool WAIT>
__device__ __forceinline__ void product_kept(f16& o, h8 a, h8 b) {
    if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(b));
}
__device__ __forceinline__ void nothing_kept(f16& o, h8 zero) { asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %1, 0" : "=a"(o) : "v"(zero)); }
__device__ __forceinline__ float kept(float o) {
    float v;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(o));
    return v;
}
__device__ __forceinline__ float keep(float v) {
    float o;
    asm volatile("v_accvgpr_write_b32 %0, %1" : "=a"(o) : "v"(v));
    return o;
}

// f(0), f(1), .. f(N - 1), the numbers known to the compiler
template <class F, int... I>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each(std::make_integer_sequence<int, N>{}, f);
}
template <int R>
using Set = std::integral_constant<int, R>;

// over the two lanes that hold one row (l, l ^ 32)
__device__ __forceinline__ float both_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// The least e >= NO_EXP for which a scale is below 2^e (to 2^126; such powers of two have exact reciprocals, that a probability
// may be multiplied by).
constexpr int NO_EXP = -100;
__device__ __forceinline__ int scale_exp(float s) { return s > 0.0f ? max(min(__builtin_amdgcn_frexp_expf(s), 126), NO_EXP) : NO_EXP; }

// The sequences' places: first unit (of ROWS rows of a kv head), first token and tokens.
struct Plan {
    int32_t base[TREE_MAX_SEQS], first[TREE_MAX_SEQS], news[TREE_MAX_SEQS];
    int32_t sums[2][WAVES];
};
constexpr int REST_DISORDER = 1, REST_SOME = 2;  // starts are not in order; some tokens are in no sequence that has work

constexpr int MAX_UNITS = 2048;  // units of a call that may be shared in equal parts

// A unit: up to ROWS rows of a sequence's kv head, and the tiles that they see.
struct Unit {
    int b, first, old, head, row0, last, tiles;
};

// Fills the plan and returns the units in all. Starts that are not in order are found on the way; the plan is then made anew, each
// sequence against all starts before it.
template <int ROWS>
__device__ __forceinline__ int make_plan(const Args& a, Plan& plan, int* rest_out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (bool in_order = true;; in_order = false) {
        int before = 0, rest = 0;
        for (int c = 0; c < a.t.n_seq; c += THREADS) {
            const int b = c + threadIdx.x;
            int units = 0, some = 0;
            Seq s = {};
            if (b < a.t.n_seq) {
                s = sequence(a.t, b, ROWS, false, in_order ? 0 : start_before(a.t, b));
                units = a.kv.heads * s.chunks;
                some = s.bad || (b == 0 && s.first > 0) || (b == a.t.n_seq - 1 && s.first + s.news < a.t.n);
            }
            some = (__any(some) ? REST_SOME : 0) | (__any(s.disorder) ? REST_DISORDER : 0);
            int run = units;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int left = __shfl_up(run, d);
                run += lane >= d ? left : 0;
            }
            if (lane == 63) plan.sums[0][wave] = run, plan.sums[1][wave] = some;
            __syncthreads();
            int all = 0, left = 0;
            for (int w = 0; w < WAVES; w++) {
                left += w < wave ? plan.sums[0][w] : 0;
                all += plan.sums[0][w];
                rest |= plan.sums[1][w];
            }
            if (b < a.t.n_seq) {
                plan.base[b] = before + left + run - units;
                plan.first[b] = s.first;
                plan.news[b] = s.news;
            }
            before += all;
            __syncthreads();
        }
        rest = __builtin_amdgcn_readfirstlane(rest);
        if (in_order && (rest & REST_DISORDER)) continue;
        *rest_out = rest;
        return __builtin_amdgcn_readfirstlane(before);
    }
}

// The last sequence that begins at or before `at`, -1 for none (empty ones share their successor's beginning).
__device__ __forceinline__ int find(const int32_t* begin, int n, int at) {
    int lo = -1, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (begin[mid] <= at ? lo : hi) = mid;
    }
    return lo;
}
__device__ __forceinline__ int find_seq(const int32_t* begin, int n_seq, int at) {
    return __builtin_amdgcn_readfirstlane(find(begin, n_seq, at));
}

// The u-th unit: a sequence's longest first, the heads in turn; or head by head, so that neighbours read the same cache.
template <int ROWS>
__device__ __forceinline__ Unit unit_at(const Args& a, const Plan& plan, int u, bool by_head) {
    Unit v;
    v.b = find(plan.base, a.t.n_seq, u);
    v.first = plan.first[v.b];
    v.old = a.t.len[v.b];
    const int past = u - plan.base[v.b], rows = plan.news[v.b] * a.t.group, chunks = (rows + ROWS - 1) / ROWS;
    v.head = by_head ? past / chunks : past % a.kv.heads;
    v.row0 = (chunks - 1 - (by_head ? past % chunks : past / a.kv.heads)) * ROWS;
    v.last = min(v.row0 + ROWS, rows) - 1;
    v.tiles = (v.old + v.last / a.t.group + 1 + KV_TILE - 1) / KV_TILE;
    return v;
}

// What a unit takes beside its tiles, in tiles: queries in, outputs out, the first tile's way (24 x 256 in units of 128 rows: 14 us and
// 3.1 a tile, which is 4.5 of them; shares by 4, 6 and 9: 12 mixed chunks of 32 x 128 118, 120 and 125 us, 131 tokens of 24 x 256 behind 120,000 604, 600
// and 595, 2,048 behind 30,000 1,639, 1,643 and 1,638).
constexpr int UNIT_TILES = 6;
__device__ __forceinline__ int length(const Unit& v) { return v.tiles + UNIT_TILES; }

// The lengths before each unit (in head order), and in all; the most of a unit.
template <int ROWS>
__device__ __forceinline__ int count_tiles(const Args& a, const Plan& plan, int units, int32_t* before, int32_t* sums, int* most_out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int all = 0, most = 0;
#pragma unroll 1
    for (int c = 0; c < units; c += THREADS) {
        const int u = c + threadIdx.x;
        const int tiles = u < units ? length(unit_at<ROWS>(a, plan, u, true)) : 0;
        int run = tiles, top = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int left = __shfl_up(run, d);
            run += lane >= d ? left : 0;
            top = max(top, __shfl_xor(top, d));
        }
        if (lane == 63) sums[wave] = run, sums[WAVES + wave] = top;
        __syncthreads();
        int at = all + run - tiles;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            at += w < wave ? sums[w] : 0;
            all += sums[w];
            most = max(most, sums[WAVES + w]);
        }
        if (u < units) before[u] = at;
        __syncthreads();
    }
    *most_out = __builtin_amdgcn_readfirstlane(most);
    return __builtin_amdgcn_readfirstlane(all);
}

// The outputs of tokens that no sequence has work for, the grid's workgroups in turn: zeros for padding, else NaN.
template <int D>
__device__ __forceinline__ void put_rest(const Args& a, const Plan& plan, int rest) {
    for (int token = blockIdx.x; token < a.t.n; token += gridDim.x) {
        const int b = find_seq(plan.first, a.t.n_seq, token);
        if (b >= 0 && token - plan.first[b] < plan.news[b]) continue;
        const uint32_t fill = padding(a.t, token, rest & REST_DISORDER) ? 0 : 0x7fc07fc0u;
        const int pieces = a.kv.heads * a.t.group * (D / 8);
        u4* const out = (u4*)a.out + (size_t)token * pieces;
        for (int i = threadIdx.x; i < pieces; i += THREADS) out[i] = u4{fill, fill, fill, fill};
    }
}

// What a workgroup holds of a tile of 64 tokens, as operands: keys [D / 8][64 tokens] of 8 dimensions; values [4][2][D] of the 8
// tokens 16 s + 4 h .. + 3, 16 s + 8 + 4 h .. + 3, which the product of keys and queries leaves in one lane (its half h).
template <int D>
struct Tile {
    h8 k[D / 8][KV_TILE];
    h8 v[4][2][D];
    float key_scale[KV_TILE];    // with all that a score is multiplied by
    float value_scale[KV_TILE];
    _Float16 factor[KV_TILE];    // what the values were multiplied by
};
template <int D, int ROWS>
struct Shared {
    Tile<D> tile[2];
    int32_t top_exp[WAVES];
    int32_t sees[ROWS];        // positions that a row sees
    float row_factor[ROWS];
    Plan plan;
    int32_t tiles_before[MAX_UNITS];
};

// The rounds that unshared units take against equal parts, in tiles: equal parts cost the partial results' way through memory and a
// second launch, about as much as JOIN_TILES. With equal parts always, 2,048 tokens of
// 24 x 256, none cached, take 150 us instead of 127, of 32 x 128 132 instead of 111, of 32 x 64 75 instead of 68; without them, 12 mixed chunks of 32 x 128 take
// 153 instead of 115, 300 tokens of 24 x 256 behind 2,000 143 instead of 76, of 32 x 64 74 instead of 53. Between them, where few units leave
// most of the GPU idle, a difference of 25 tiles is too much to ask: behind 1,000 positions (16 to 21 tiles) 70 tokens of 24 x 256 take 82 us, and with
// equal parts 48, 300 of 32 x 128 69 and 52, of 32 x 64 51 and 43. No part is below PART_TILES. (All warm.)
constexpr int JOIN_TILES = 25, PART_TILES = 4;
// Tables up to so many tiles have units of 128 rows where 256 would be less than two for each workgroup: half the work at the end of the
// last round, for tiles that are read for half the rows. It goes by what a table can hold, since the lengths are on the device: with a wider one short prompts
// have units of 256 rows, too. In us, 128 rows against 256: 2,048 tokens of 24 x 256, 32 tiles in all 126 and 202, 48 237 and 278, 64 299 and 266, 80
// 370 and 322, 112 508 and 433, 500 2,020 and 1,680; 512 tokens, 8 tiles 50 and 83, 48 113 and 103, 112 187 and 164. 32 x 128, 2,048 tokens, 32 tiles
// 112 and 129, 48 204 and 179, 80 341 and 260; 512 tokens, 48 tiles 90 and 93, 112 156 and 145. 32 x 64, 2,048 tokens, 32 tiles 67 and 78, 80 156 and 157, 160
// 300 and 282; 512 tokens, 80 tiles 79 and 91, 288 180 and 183. So the two cross between 32 and 64 tiles at d = 256 and 128, and between 80 and
// 300 at d = 64. (Warm.)
constexpr int SHORT_TILES = 80;
__device__ __forceinline__ bool share(int units, int all, int most, int parts) {
    const int even = (all + parts - 1) / parts;
    return (units <= parts ? most : max(most, even + most / 2)) > even + JOIN_TILES;
}

// A lane's row's softmax: the reference m that scores are taken against (in powers of two), and the sums of 2^(score - m). A score
// may come to m + 15, since f16 holds that; m is set 7 below a largest score, so that probabilities keep f16's full bits down to 2^-21
// of the largest and are dropped below 2^-32.
constexpr float ROOM = 15.0f, BELOW = 7.0f;
constexpr int VALUE_EXP = 7;  // values are taken relative to 2^-7 of the largest scale, for the same reason
// What that leaves of a value: half of f16's smallest step is 2^-25, so its scale is off by 2^-25 2^-7 of less than twice the largest scale, 2^-31
// of it, times the code; the product's own rounding adds 2^-31 once. With codes up to 127 that is 2^-24 of the largest scale, with e4m3's 448
// 449 / 2^31 < 2^-22. Where the scale goes to the probability, of which the largest is 2^7 at least, the same.

// Waves of a SIMD: what the registers (and LDS) leave room for.
constexpr int waves_of(int d) { return d == 64 ? 2 : 1; }

template <int D, int FMT, int SETS>
__global__ __launch_bounds__(THREADS, waves_of(D)) void chunk_attn_kernel(const Args a) {
    constexpr int ROWS = rows_of(SETS);
    constexpr bool WAIT = waves_of(D) > 1;
    __shared__ Shared<D, ROWS> sh;
    int rest;
    const int units = make_plan<ROWS>(a, sh.plan, &rest);
    if (rest) put_rest<D>(a, sh.plan, rest);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // (The lane is said anew in each block: what follows from it would otherwise be kept in registers over the blocks, and they run out.)
    int lane = tid & 63;
    auto col = [&]() INLINE { return lane & 31; };
    auto half = [&]() INLINE { return lane >> 5; };
    auto l16 = [&]() INLINE { return lane & 15; };
    auto c4 = [&]() INLINE { return lane >> 4; };
    auto g4 = [&]() INLINE { return (lane >> 4 & 1) * 2 + (lane >> 5); };
    auto my_row = [&]() INLINE { return wave * (32 * SETS) + (lane & 31); };
    // A unit each; or all tiles of all units in a row, in equal parts, consecutive ones on one XCD (workgroups b, b + 8, .. run on the same
    // one), whose L2 then serves those that read the same head's cache.
    int at = 0, hi = 1, all = 0, used = 0, part = 0;
    bool shared = false;
    if (a.parts) {
        int most;
        all = count_tiles<ROWS>(a, sh.plan, units, sh.tiles_before, sh.plan.sums[0], &most);
        shared = all > 0 && share(units, all, most, a.parts);
        used = shared ? min(a.parts, max(all / PART_TILES, 1)) : 0;
        part = blockIdx.x;
        if (part < used) {
            const int xcd = part & 7, at_xcd = part >> 3;
            part = xcd * (used >> 3) + min(xcd, used & 7) + at_xcd;
        }
        if (part < a.parts && part >= used && tid == 0) a.cuts[part] = Cut{};
    }
    // where a part begins: not within what a unit takes beside its tiles, but with the unit
    auto begin_of = [&](int w) INLINE {
        const int begin = first_group(w, all, used);
        if (begin >= all) return all;
        const int unit = sh.tiles_before[find_seq(sh.tiles_before, units, begin)];
        return __builtin_amdgcn_readfirstlane(begin - unit <= UNIT_TILES ? unit : begin);  // (a tile at least before it)
    };
    if (shared) {
        if (part >= used) return;
        at = begin_of(part);
        hi = begin_of(part + 1);
        if (at >= hi) {
            if (tid == 0) a.cuts[part] = Cut{};
            return;
        }
    } else if ((int)blockIdx.x >= units) {
        return;
    }
  do {
    const int u = shared ? find_seq(sh.tiles_before, units, at) : (int)blockIdx.x;
    const int unit_begin = shared ? __builtin_amdgcn_readfirstlane(sh.tiles_before[u]) : 0;
    const Unit v = unit_at<ROWS>(a, sh.plan, u, shared);
    const int b = __builtin_amdgcn_readfirstlane(v.b), first = __builtin_amdgcn_readfirstlane(v.first);
    const int news = __builtin_amdgcn_readfirstlane(sh.plan.news[v.b]), old = __builtin_amdgcn_readfirstlane(v.old), group = a.t.group;
    const int head = __builtin_amdgcn_readfirstlane(v.head), row0 = __builtin_amdgcn_readfirstlane(v.row0);
    const int last = __builtin_amdgcn_readfirstlane(v.last), tiles = __builtin_amdgcn_readfirstlane(v.tiles);  // the last row
    const int all_see = old + row0 / group + 1;  // positions that all its rows see
    const int t_begin = shared ? max(at - unit_begin - UNIT_TILES, 0) : 0;
    const int t_end = shared ? min(tiles, hi - unit_begin - UNIT_TILES) : tiles;
    if (shared && at == begin_of(part)) {  // the first part that begins within a unit has it joined
        const bool joins = t_begin && begin_of(part - 1) <= unit_begin;
        if (tid == 0) a.cuts[part] = joins ? Cut{unit_begin, unit_begin + length(v), all, used, first, head, row0, last} : Cut{};
    }
    if (shared) __syncthreads();  // (the unit before is through with LDS)

    // the lane's row of a set, and its first query and output
    auto row_of = [&](int r) INLINE { return row0 + wave * (32 * SETS) + r * 32 + col(); };
    auto row_at = [&](int r) INLINE {
        const int row = min(row_of(r), last), node = row / group;
        return ((size_t)(first + node) * a.kv.heads * group + head * group + (row - node * group)) * D;
    };
    // (what only some tiles and waves need lies in LDS: registers run out)
#pragma unroll
    for (int r = 0; r < SETS; r++) sh.sees[my_row() + r * 32] = old + min(row_of(r), last) / group + 1;

    // where tiles lie, 64 at a time: lane l has the l-th's place in the cache (of its keys) in tiles
    constexpr uint32_t NONE = ~0u;
    const int page_tiles = 1 << (a.kv.page_shift - 6);
    uint32_t places = 0;
    auto load_places = [&](int t) INLINE {
        const int mine = min(t + lane, t_end - 1);
        const int page = a.table[(size_t)b * a.t.table_ld + (mine >> (a.kv.page_shift - 6))];
        places = (((uint32_t)page * a.kv.heads + head) * 2) * page_tiles + (mine & (page_tiles - 1));
        if (page < 0 || ((int64_t)page << a.kv.page_shift) >= a.kv.slots) places = NONE;
    };
    load_places(t_begin);

    // a thread's pieces of a tile: 16 dimensions of a token's key, 16 tokens of a dimension of the values
    constexpr int PIECES = KV_TILE * D / 16 / THREADS;
    u4 raw[PIECES];
    float ks, vs;
    bool none;
    uint32_t place;
    // (buffer loads: an address is a lane's 32 bits beside what the wave has alike)
    auto rsrc = [&](const void* p, int bytes) INLINE { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, BUF_RSRC_WORD3); };
    auto piece = [&](__amdgpu_buffer_rsrc_t codes, int at, int i) INLINE {
        return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(codes, at, (wave + i * WAVES) * 1024, 0));
    };
    auto load_keys = [&](int t) INLINE {
        if (UNLIKELY(((t - t_begin) & 63) == 0 && t > t_begin)) load_places(t);
        const uint32_t p = __builtin_amdgcn_readlane(places, (t - t_begin) & 63);
        none = p == NONE;
        place = none ? 0 : p;
        const auto sc = rsrc(a.kv.scales + (size_t)place * KV_TILE, (page_tiles + 1) * KV_TILE * 4);
        ks = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sc, lane * 4, 0, 0));
        vs = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sc, lane * 4, page_tiles * KV_TILE * 4, 0));
        const auto codes = rsrc(a.kv.codes + (size_t)place * (KV_TILE * D), KV_TILE * D);
#pragma unroll
        for (int i = 0; i < PIECES; i++) raw[i] = piece(codes, l16() * 64 + c4() * 16, i);
    };
    auto load_values = [&]() INLINE {
        const auto codes = rsrc(a.kv.codes + ((size_t)place + page_tiles) * (KV_TILE * D), KV_TILE * D);
#pragma unroll
        for (int i = 0; i < PIECES; i++) raw[i] = piece(codes, l16() * 64 + g4() * 16, i);
    };
    auto put_keys = [&](Tile<D>& to, int i) INLINE {
        const int u = wave + i * WAVES, token = u / (D / 64) * 16 + l16(), chunk = u % (D / 64) * 8 + c4() * 2;
        const h4 k0 = operands<FMT>(raw[i].x), k1 = operands<FMT>(raw[i].y), k2 = operands<FMT>(raw[i].z), k3 = operands<FMT>(raw[i].w);
        to.k[chunk][token] = __builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7);
        to.k[chunk + 1][token] = __builtin_shufflevector(k2, k3, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    h4 factor[4];  // of the thread's tokens
    auto load_factors = [&](const Tile<D>& to) INLINE {
#pragma unroll
        for (int s = 0; s < 4; s++) factor[s] = *(const h4*)&to.factor[s * 16 + g4() * 4];
    };
    auto put_values = [&](Tile<D>& to, int i, int there) INLINE {
        const int dim = (wave + i * WAVES) * 16 + l16();
        if (FMT == QH_KV_E4M3 && UNLIKELY(there < KV_TILE)) {  // what was not written may be NaN codes, which no probability takes away
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int keep = max(there - (s * 16 + g4() * 4), 0);
                raw[i][s] = keep < 4 ? raw[i][s] & ((1u << 8 * keep) - 1) : raw[i][s];
            }
        }
#pragma unroll
        for (int s = 0; s < 4; s++) ((h4*)&to.v[s][g4() & 1][dim])[g4() >> 1] = operands<FMT>(raw[i][s]) * factor[s];
    };

    // the lane's queries: dimensions 16 i + 8 half .. + 7, scaled by a power of two into f16's range. One power for the workgroup, that goes
    // into the keys' scales; in a wave with rows 2^16 and more below the largest, or not finite, each row its own, with a factor for
    // what it then differs by.
    // Where queries reach 2^55, the rest of the power is left to the differences of scores (`late`): the scores themselves might be
    // infinite. All tiles are then taken apart.
    h8 q[SETS][D / 16];
    float late;
    int key_exp;
    bool wide = false;
    {
        constexpr int LOW = -1000;
        uint32_t top[SETS];  // bf16 with the sign taken off compares as a whole number; from 0x7f80 on it is not finite
        int e[SETS], most = LOW;
        u4 raw_q[SETS][D / 16];
#pragma unroll
        for (int r = 0; r < SETS; r++) {
            const __bf16* const from = a.q + row_at(r) + half() * 8;
#pragma unroll
            for (int i = 0; i < D / 16; i++) raw_q[r][i] = *(const u4*)(from + i * 16);
        }
        typedef uint16_t us2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int r = 0; r < SETS; r++) {
            us2 largest = {0, 0};
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) largest = __builtin_elementwise_max(largest, __builtin_bit_cast(us2, raw_q[r][i][k] & 0x7fff7fffu));
            top[r] = max(largest.x, largest.y);
            const auto both = __builtin_amdgcn_permlane32_swap(top[r], top[r], false, false);
            top[r] = max(both[0], both[1]);
            e[r] = top[r] && top[r] < 0x7f80 ? __builtin_amdgcn_frexp_expf(__uint_as_float(top[r] << 16)) - 15 : LOW;
            most = max(most, e[r]);
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) most = max(most, __shfl_xor(most, d));
        if (lane == 0) sh.top_exp[wave] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; w++) most = max(most, sh.top_exp[w]);
        most = __builtin_amdgcn_readfirstlane(most == LOW ? 0 : most);
#pragma unroll
        for (int r = 0; r < SETS; r++) wide |= __any(top[r] >= 0x7f80 || (top[r] && e[r] < most - 16));
        each<SETS>([&](auto set) INLINE {
            constexpr int r = decltype(set)::value;
            sh.row_factor[my_row() + r * 32] = top[r] >= 0x7f80 ? NAN : __builtin_ldexpf(1.0f, e[r] == LOW ? 0 : e[r] - most);
            const int by = wide && e[r] != LOW ? e[r] : most;
            each<D / 16>([&](auto at) INLINE {
                constexpr int i = decltype(at)::value;
                HOLD();
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t two = raw_q[r][i][k];
                    const h2 h = __builtin_convertvector((f2{__builtin_ldexpf(__uint_as_float(two << 16), -by),
                                                             __builtin_ldexpf(__uint_as_float(two & 0xffff0000u), -by)}), h2);
                    q[r][i][2 * k] = h.x, q[r][i][2 * k + 1] = h.y;
                }
            });
        });
        auto alike = [&](float v) INLINE { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); };
        key_exp = __builtin_amdgcn_readfirstlane(a.scale_exp + min(most, 40));
        late = alike(__builtin_ldexpf(1.0f, max(most - 40, 0)));
    }

    // Values are multiplied by their scales as they become operands, relative to 2^ref, the largest scale so far: for tiles that all rows
    // see whole. In other tiles (`apart`) the scales go to the probabilities, relative to the largest that the row itself sees.
    int ref = NO_EXP;
    bool apart = false, apart_next = false;
    int ref_next = NO_EXP;
    // what is said of a tile before its values become operands
    auto put_scales = [&](Tile<D>& to, int t) INLINE {
        if (none) ks = vs = NAN;
        const bool whole = (t + 1) * KV_TILE <= all_see;
        apart_next = apart_next || !whole || late > 1.0f || __any(!(fabsf(vs) < INFINITY));  // (and so for good: units then only grow)
        if (UNLIKELY(!apart_next && __any(fabsf(vs) > __builtin_ldexpf(1.0f, ref_next)))) {
            float most = fabsf(vs);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
            ref_next = __builtin_amdgcn_readfirstlane(max(ref_next, scale_exp(most)));
        }
        to.key_scale[lane] = fabsf(vs) < INFINITY ? __builtin_ldexpf(ks * a.scale, key_exp) : NAN;
        to.value_scale[lane] = fabsf(vs) < INFINITY ? fabsf(vs) : 0.0f;
        // (A tile's unwritten tokens may have any scale. Where the scales go to the probabilities, a negative one's sign stays with the value.
        // 2^VALUE_EXP bounds nothing else; by selects instead the widest heads' kernel spills.)
        const float most = apart_next ? 1.0f : 0x1p7f;
        to.factor[lane] = (_Float16)__builtin_amdgcn_fmed3f(__builtin_ldexpf(vs, apart_next ? 250 : VALUE_EXP - ref_next), -most, most);
    };
    auto written = [&](int t) INLINE { return none ? 0 : min(old + news - t * KV_TILE, KV_TILE); };  // tokens of the tile

    f16 o[SETS][D / 32];
    float m[SETS], sum[SETS];
    int unit[SETS];  // o is in units of 2^unit
    each<SETS>([&](auto set) INLINE {
        constexpr int r = decltype(set)::value;
        m[r] = -INFINITY, sum[r] = 0.0f, unit[r] = NO_EXP;
        each<D / 32>([&](auto i) INLINE { nothing_kept(o[r][i], h8{}); });
    });
    auto scale_out = [&](auto set, float by) INLINE {
        constexpr int r = decltype(set)::value;
        if (!__any(by != 1.0f)) return;
        HOLD();
        PRODUCTS_READY();
        each<D / 32>([&](auto i) INLINE {
            HOLD();
            each<16>([&](auto k) INLINE { o[r][i][k.value] = keep(kept(o[r][i][k.value]) * by); });
        });
        HOLD();
        OPERANDS_READY();
    };

    f16 x[SETS];    // scores of 32 tokens: the lane has its rows' of tokens 8 (i / 4) + 4 half + i % 4
    h8 p[2][2];     // their probabilities, as operands: of each set; or with one set, of a block and of the one before
    float mx[SETS];
    int to[SETS];  // the units that the values then have
    // A set's scores relative to m (as yet none: as they are), in 16 steps that may go on beside products.
    f4 sc[2];  // the block's keys' scales, four tokens' and the next ones'; behind the first set's last, its first again
    auto load_scale = [&](const Tile<D>& tile, int tb, int j) INLINE { sc[j & 1] = *(const f4*)&tile.key_scale[tb * 32 + j * 8 + half() * 4]; };
    auto relative = [&](const Tile<D>& tile, int tb, auto set, auto at) INLINE {
        constexpr int r = decltype(set)::value, k = decltype(at)::value;
        x[r][k] = __builtin_fmaf(x[r][k], sc[k / 4 & 1][k & 3], m[r] == -INFINITY ? -0.0f : -m[r]);
        if constexpr (k % 2 == 1) mx[r] = fmaxf(fmaxf(k == 1 ? -INFINITY : mx[r], x[r][k - 1]), x[r][k]);
        if constexpr (k % 4 == 3 && (r + 1 < SETS || k < 8)) load_scale(tile, tb, (k / 4 + 2) % 4);
    };
    // then, in tiles taken apart, what a row does not see is left out; the units that the values have
    auto mask = [&](const Tile<D>& tile, int t, int tb, auto set) INLINE {
        constexpr int r = decltype(set)::value;
        to[r] = ref - VALUE_EXP;
        if (LIKELY(!apart)) return;
        const int t0 = t * KV_TILE + tb * 32 + half() * 4, behind = (t + 1) * KV_TILE <= all_see ? 0x7fffffff : sh.sees[my_row() + r * 32];
        float largest = 0.0f;
        mx[r] = -INFINITY;
        each<4>([&](auto at) INLINE {
            constexpr int j = decltype(at)::value;
            const f4 sv = *(const f4*)&tile.value_scale[tb * 32 + j * 8 + half() * 4];
            HOLD();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool seen = t0 + 8 * j + i < behind;
                x[r][4 * j + i] = seen ? x[r][4 * j + i] : -INFINITY;
                mx[r] = fmaxf(mx[r], x[r][4 * j + i]);
                largest = fmaxf(largest, seen ? sv[i] : 0.0f);
            }
        });
        to[r] = max(max(ref, unit[r]), scale_exp(both_max(largest)));
    };
    // whether m has to follow, or the units change
    auto moved = [&](auto set) INLINE {
        constexpr int r = decltype(set)::value;
        return __any(mx[r] * late > ROOM || m[r] == -INFINITY || unit[r] != to[r]);
    };
    // m follows the scores where some are above ROOM, by whole numbers: the power of two by which the sums are multiplied
    auto follow = [&](auto set) INLINE {
        constexpr int r = decltype(set)::value;
        const float most = both_max(mx[r]);
        const bool none = m[r] == -INFINITY;
        const float up = most * late > ROOM || (none && most > -INFINITY)
                             ? (fabsf(most * late) < 0x1p30f ? floorf(most * late - BELOW) / late : most) : 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++) x[r][k] -= up;
        m[r] = none ? (most > -INFINITY ? up : m[r]) : m[r] + up;
        const float by = none ? 1.0f : __builtin_amdgcn_exp2f(-up * late);
        sum[r] *= by;
        const float units = none ? 1.0f : __builtin_ldexpf(by, unit[r] - to[r]);  // (none: there are no outputs yet)
        unit[r] = to[r];
        return units;
    };
    // In tiles taken apart the sum is of the probabilities by themselves, and their values' scales go into the exponents.
    auto settle = [&](const Tile<D>& tile, int tb, auto set) INLINE {
        constexpr int r = decltype(set)::value;
        if (LIKELY(!apart)) return;
        each<4>([&](auto at) INLINE {
            constexpr int j = decltype(at)::value;
            const f4 sv = *(const f4*)&tile.value_scale[tb * 32 + j * 8 + half() * 4];
            HOLD();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float s = x[r][4 * j + i] * late;
                sum[r] += __builtin_amdgcn_exp2f(s);
                x[r][4 * j + i] = s + (__builtin_amdgcn_logf(sv[i]) - (float)unit[r]);  // (log2; an unseen token's score is -inf)
            }
        });
    };
    // The probabilities of a set's scores, in 16 steps beside products. (Sums are of the probabilities as they are multiplied.)
    h2 ones = {(_Float16)1.0f, (_Float16)1.0f};
    float even;
    auto soft = [&](auto set, auto at, auto to) INLINE {
        constexpr int r = decltype(set)::value, k = decltype(at)::value, q = decltype(to)::value;
        const float pr = __builtin_amdgcn_exp2f(x[r][k]);
        if constexpr (k % 2 == 0) {
            even = pr;
        } else {
            const h2 pp = __builtin_convertvector((f2{even, pr}), h2);
            sum[r] = __builtin_amdgcn_fdot2(pp, ones, sum[r], false);
            p[q][k >> 3][(k & 7) - 1] = pp.x, p[q][k >> 3][k & 7] = pp.y;
        }
    };

    // Operands are asked for DEEP - 1 products ahead of theirs, over the borders of what follows one another: `ahead(k)` has the k-th of what comes
    // after.
    constexpr int DEEP = 4;
    static_assert(D / 16 % DEEP == 0);
    h8 f[DEEP];
    auto key = [&](const Tile<D>& tile, int tb, int i) INLINE { return tile.k[2 * i + half()][tb * 32 + col()]; };
    auto value = [&](const Tile<D>& tile, int tb, int n) INLINE { return tile.v[tb * 2 + n / (D / 32)][half()][n % (D / 32) * 32 + col()]; };
    // s^T = k q^T of 32 tokens, with `beside(i)` beside the products of 16 dimensions
    auto scores = [&](const Tile<D>& tile, int tb, auto&& beside, auto&& ahead) INLINE {
        each<D / 16>([&](auto at) INLINE {
            constexpr int i = decltype(at)::value, to = (i + DEEP - 1) % DEEP;
            HOLD();
            if constexpr (i + DEEP - 1 < D / 16) f[to] = key(tile, tb, i + DEEP - 1);
            else f[to] = ahead(i + DEEP - 1 - D / 16);
            if constexpr (i >= D / 16 - 2) load_scale(tile, tb, i - D / 16 + 2);
#pragma unroll
            for (int r = 0; r < SETS; r++) {
                if constexpr (i == 0) product_first<WAIT>(x[r], f[0], q[r][0]);
                else product<WAIT>(x[r], f[i % DEEP], q[r][i]);
            }
            beside(at);
        });
        HOLD();
    };
    // o^T += v^T p^T of a set: the lane has its row's dimensions 32 i + 8 (k / 4) + 4 half + k % 4
    constexpr int PRODUCTS = D / 32 * 2;  // of 32 dimensions, then of 16 tokens
    auto outputs = [&](const Tile<D>& tile, int tb, auto set, auto from, auto&& beside, auto&& ahead) INLINE {
        constexpr int r = decltype(set)::value, q = decltype(from)::value;
        HOLD();
        OPERANDS_READY();
        each<PRODUCTS>([&](auto at) INLINE {
            constexpr int n = decltype(at)::value, to = (n + DEEP - 1) % DEEP;
            HOLD();
            if constexpr (n + DEEP - 1 < PRODUCTS) f[to] = value(tile, tb, n + DEEP - 1);
            else f[to] = ahead(n + DEEP - 1 - PRODUCTS);
            product_kept<WAIT>(o[r][n % (D / 32)], f[n % DEEP], p[q][n / (D / 32)]);
            beside(at);
        });
        HOLD();
    };
    // 16 steps spread over a set's products
    auto spread = [&](auto at, auto&& step) INLINE {
        constexpr int n = decltype(at)::value, from = 16 * n / PRODUCTS, to = 16 * (n + 1) / PRODUCTS;
        each<to - from>([&](auto k) INLINE { step(std::integral_constant<int, from + decltype(k)::value>{}); });
    };
    const auto nothing = [](auto) INLINE {};

    load_keys(t_begin);
    put_scales(sh.tile[t_begin & 1], t_begin);
#pragma unroll
    for (int i = 0; i < PIECES; i++) put_keys(sh.tile[t_begin & 1], i);
    load_values();
    __syncthreads();
    load_factors(sh.tile[t_begin & 1]);
#pragma unroll
    for (int i = 0; i < PIECES; i++) put_values(sh.tile[t_begin & 1], i, written(t_begin));
    apart = apart_next, ref = ref_next;
    __syncthreads();
    // The second set's products with the values stand behind the next block's scores: the first set's softmax then has them beside it,
    // and the second set's the first set's products. One set alone stands behind as a whole, its softmax beside the block before's products.
    // To begin with, probabilities of nothing.
#pragma unroll
    for (int k = 0; k < 8; k++) p[1][0][k] = p[1][1][k] = (_Float16)0.0f;
    auto widen = [&]() INLINE {
        if (UNLIKELY(wide)) {
#pragma unroll
            for (int r = 0; r < SETS; r++)
#pragma unroll
                for (int k = 0; k < 16; k++) x[r][k] *= sh.row_factor[my_row() + r * 32];
        }
    };
    auto first_set = [&](const Tile<D>& tile, int t, int tb) INLINE {
        products_ready(x);
        widen();
        each<16>([&](auto k) INLINE { relative(tile, tb, Set<0>{}, k); });
        mask(tile, t, tb, Set<0>{});
    };
#pragma unroll
    for (int k = 0; k < DEEP - 1; k++) f[k] = key(sh.tile[t_begin & 1], 0, k);
    scores(sh.tile[t_begin & 1], 0, nothing, [&](int k) INLINE { return value(sh.tile[t_begin & 1], 1, k); });
    first_set(sh.tile[t_begin & 1], t_begin, 0);
    (void)follow(Set<0>{});
    settle(sh.tile[t_begin & 1], 0, Set<0>{});
    int t = t_begin;
    do {  // (there is a tile at least; a loop that might not run would have its outputs in registers of their own)
        const Tile<D>& tile = sh.tile[t & 1];
        Tile<D>& next = sh.tile[(t + 1) & 1];
        const bool more = t + 1 < t_end;
        each<2>([&](auto block) INLINE {
            constexpr int tb = decltype(block)::value;
            asm volatile("" : "+v"(lane));
            const Tile<D>& before = tb ? tile : sh.tile[(max(t, t_begin + 1) - 1) & 1];
            if (LIKELY(more)) {
                if constexpr (tb == 0) load_keys(t + 1);
                else load_values();
            }
            ones = apart ? h2{(_Float16)0.0f, (_Float16)0.0f} : h2{(_Float16)1.0f, (_Float16)1.0f};
            // (behind the last tile's last block there are no scores: what is asked for then is the tile's again, and not used)
            const Tile<D>& coming = tb == 0 ? tile : next;
            auto coming_key = [&](int k) INLINE { return key(coming, tb ^ 1, k); };
            if constexpr (SETS == 1) {
                outputs(before, tb ^ 1, Set<0>{}, Set<(tb ^ 1)>{},
                        [&](auto at) INLINE { spread(at, [&](auto k) INLINE { soft(Set<0>{}, k, Set<tb>{}); }); }, coming_key);
            } else {
                outputs(before, tb ^ 1, Set<1>{}, Set<1>{}, [&](auto at) INLINE {
                    spread(at, [&](auto k) INLINE {
                        soft(Set<0>{}, k, Set<0>{});
                        relative(tile, tb, Set<1>{}, k);
                    });
                }, [&](int k) INLINE { return value(tile, tb, k); });
                mask(tile, t, tb, Set<1>{});
                if (UNLIKELY(moved(Set<1>{}))) scale_out(Set<1>{}, follow(Set<1>{}));
                settle(tile, tb, Set<1>{});
                outputs(tile, tb, Set<0>{}, Set<0>{},
                        [&](auto at) INLINE { spread(at, [&](auto k) INLINE { soft(Set<1>{}, k, Set<1>{}); }); }, coming_key);
            }
            if (tb == 0 || LIKELY(more)) {
                // the next tile's operands beside the scores, late enough for its codes to be there
                scores(coming, tb ^ 1, [&](auto at) INLINE {
                    constexpr int i = decltype(at)::value - D / 32;
                    if constexpr (i == -1) {
                        if constexpr (tb == 0) {
                            if (LIKELY(more)) put_scales(next, t + 1);
                        } else {
                            load_factors(next);
                        }
                    }
                    if constexpr (i >= 0 && i % 2 == 0 && i / 2 < PIECES) {
                        if constexpr (tb == 0) {
                            if (LIKELY(more)) put_keys(next, i / 2);
                        } else {
                            put_values(next, i / 2, written(t + 1));
                        }
                    }
                }, [&](int k) INLINE { return value(tile, tb, k); });
                if constexpr (tb == 1) apart = apart_next, ref = ref_next;
                first_set(coming, t + tb, tb ^ 1);
                if (UNLIKELY(moved(Set<0>{}))) {
                    const float by = follow(Set<0>{});
                    scale_out(Set<0>{}, by);
                    if constexpr (SETS == 1) {  // what stands behind, too
#pragma unroll
                        for (int k = 0; k < 16; k++) p[tb][k >> 3][k & 7] = (_Float16)((float)p[tb][k >> 3][k & 7] * by);
                    }
                }
                settle(coming, tb ^ 1, Set<0>{});
            }
            __syncthreads();
        });
    } while (++t < t_end);
#pragma unroll
    for (int k = 0; k < DEEP - 1; k++) f[k] = value(sh.tile[(t_end - 1) & 1], 1, k);
    outputs(sh.tile[(t_end - 1) & 1], 1, Set<SETS - 1>{}, Set<1>{}, nothing, [&](int) INLINE { return f[0]; });
    PRODUCTS_READY();

    auto put = [&](auto set, auto gated) INLINE {
        constexpr int r = decltype(set)::value, N = D / 8;
        const float total = __builtin_ldexpf(__builtin_amdgcn_rcpf(both_sum(sum[r])), unit[r]);
        const size_t at = row_at(r) + half() * 4;
        b4 g[N];  // (all at once: each is a trip to memory)
        if constexpr (decltype(gated)::value)
            each<N>([&](auto k) INLINE { g[k.value] = *(const b4*)(a.gate + at + k.value * 8); });
        const bool there = row_of(r) <= last;
        each<N>([&](auto piece) INLINE {
            constexpr int k = decltype(piece)::value, i = k / 4, j = k % 4;
            HOLD();
            f4 v = f4{kept(o[r][i][4 * j]), kept(o[r][i][4 * j + 1]), kept(o[r][i][4 * j + 2]), kept(o[r][i][4 * j + 3])} * total;
            if constexpr (decltype(gated)::value) {
#pragma unroll
                for (int n = 0; n < 4; n++) v[n] *= sigmoid((float)g[k][n]);
            }
            if (there) *(b4*)(a.out + at + k * 8) = __builtin_convertvector(v, b4);
        });
    };
    if (t_begin == 0 && t_end == tiles) {
        each<SETS>([&](auto set) INLINE {
            if (a.gate) put(set, std::true_type{});
            else put(set, std::false_type{});
        });
    } else {
        const size_t slot = partial_slot(part, unit_begin, all, used);
        f4* const rows = a.part_rows + slot * ROWS + wave * (32 * SETS) + col();
        f4* const to = (f4*)a.part + slot * (ROWS * D / 4) + (size_t)wave * SETS * (D * 8) + lane;
        each<SETS>([&](auto set) INLINE {
            constexpr int r = decltype(set)::value;
            const float total = both_sum(sum[r]);
            if (half() == 0) rows[r * 32] = f4{m[r], total, (float)unit[r], 0.0f};
            each<D / 32>([&](auto dims) INLINE {
                constexpr int i = decltype(dims)::value;
                HOLD();
#pragma unroll
                for (int j = 0; j < 4; j++)
                    to[((r * (D / 32) + i) * 4 + j) * 64] = f4{kept(o[r][i][4 * j]), kept(o[r][i][4 * j + 1]), kept(o[r][i][4 * j + 2]), kept(o[r][i][4 * j + 3])};
            });
        });
    }
    at = unit_begin + UNIT_TILES + t_end;
  } while (shared && at < hi);
}

// The partial results of a unit that several parts have: a workgroup for 32 rows of it and 64 dimensions. The maxima's powers of two and
// the units of the parts are joined; four parts' results are under way at once. Bound by their bytes: 256 parts of 256 x 256 in 27 us
// (a workgroup for all dimensions, two under way: 78).
template <int D, int SETS>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
    constexpr int ROWS = rows_of(SETS), AHEAD = 4, PIECES = 2;  // pieces of 8 dimensions that a wave has
    const int part = blockIdx.x, set = blockIdx.y;
    if (part == 0) return;
    const Cut cut = a.cuts[part];
    if (cut.end == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5, piece = (blockIdx.z * 4 + wave) * PIECES;
    const int row = cut.row0 + set * 32 + col;
    const int end = group_owner(cut.end - 1, cut.all, cut.used);
    auto slot = [&](int w) { return (size_t)partial_slot(w, cut.begin, cut.all, cut.used); };
    auto row_state = [&](int w) { return a.part_rows[slot(w) * ROWS + set * 32 + col]; };
    float m = -INFINITY, units = NO_EXP, sum = 0.0f;
    for (int w0 = part - 1; w0 <= end; w0 += AHEAD) {
        f4 s[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) s[k] = row_state(min(w0 + k, end));
#pragma unroll
        for (int k = 0; k < AHEAD; k++) m = fmaxf(m, s[k].x), units = fmaxf(units, s[k].z);
    }
    f4 o[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; i++) o[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int w0 = part - 1; w0 <= end; w0 += AHEAD) {
        f4 s[AHEAD], v[AHEAD][PIECES];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int w = min(w0 + k, end);
            s[k] = row_state(w);
            const f4* const from = (const f4*)a.part + slot(w) * (ROWS * D / 4) + (size_t)set * (D * 8) + lane;
#pragma unroll
            for (int i = 0; i < PIECES; i++) v[k][i] = from[(piece + i) * 64];
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            if (w0 + k > end) break;
            const bool none = s[k].x == -INFINITY;  // (a row that sees nothing of a part adds nothing, or that it is not finite)
            const float by = none ? 0.0f : __builtin_amdgcn_exp2f(s[k].x - m);
            sum += none ? s[k].y : s[k].y * by;
            const float scale = __builtin_ldexpf(by, (int)(s[k].z - units));
#pragma unroll
            for (int i = 0; i < PIECES; i++) o[i] += none ? f4{0.0f, 0.0f, 0.0f, 0.0f} : v[k][i] * scale;
        }
    }
    if (row > cut.last) return;
    const float total = __builtin_ldexpf(__builtin_amdgcn_rcpf(sum), (int)units);
    const int group = a.t.group, node = row / group;
    const size_t at = ((size_t)(cut.first + node) * a.kv.heads * group + cut.head * group + (row - node * group)) * D + half * 4;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const size_t d = at + (piece + i) * 8;
        f4 v = o[i] * total;
        if (a.gate) {
            const b4 g = *(const b4*)(a.gate + d);
#pragma unroll
            for (int n = 0; n < 4; n++) v[n] *= sigmoid((float)g[n]);
        }
        *(b4*)(a.out + d) = __builtin_convertvector(v, b4);
    }
}

}  // namespace

extern "C" int qh_chunk_attn(qh_ctx* ctx, void* stream, const void* q, int q_heads, const qh_kv* kv, const qh_tree* step,
                             float scale, const void* gate, void* out) {
    if (!step) return fail(QH_EINVAL, "chunk_attn: null step");
    Args a = {};
    if (int e = kv_check("chunk_attn", kv, &a.kv)) return e;
    if (step->n == 0 || step->n_seq == 0) return QH_OK;
    if (!q || !out || !step->start || !step->len || !step->table) return fail(QH_EINVAL, "chunk_attn: null");
    if (step->mask) return fail(QH_EINVAL, "chunk_attn: no mask (trees: tree_attn)");
    if (q_heads < 1 || q_heads % kv->heads || q_heads / kv->heads > 64)
        return fail(QH_EINVAL, "chunk_attn: %d query heads over %d kv heads (a multiple, up to 64 times)", q_heads, kv->heads);
    if (step->n_seq < 0 || step->n_seq > TREE_MAX_SEQS)
        return fail(QH_EINVAL, "chunk_attn: %d sequences (up to %d)", step->n_seq, TREE_MAX_SEQS);
    if (step->n > (size_t)1 << 20) return fail(QH_EINVAL, "chunk_attn: %zu tokens (up to 2^20)", step->n);
    if (step->max_new < 1) return fail(QH_EINVAL, "chunk_attn: up to %d tokens of a sequence", step->max_new);
    if (step->n > (size_t)step->n_seq * step->max_new)
        return fail(QH_EINVAL, "chunk_attn: %zu tokens of %d sequences of up to %d", step->n, step->n_seq, step->max_new);
    if (!(scale > 0.0f) || !(scale < INFINITY)) return fail(QH_EINVAL, "chunk_attn: scale %g must be positive", scale);
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)gate % 16)
        return fail(QH_EINVAL, "chunk_attn: q, gate and out must be 16-byte aligned");
    if (step->table_ld < 1 || step->table_ld > ((size_t)1 << 30) / kv->page)
        return fail(QH_EINVAL, "chunk_attn: tables of %zu pages of %d tokens (1 to 2^30 positions)", step->table_ld, kv->page);
    if ((uint64_t)a.kv.slots / KV_TILE * 2 * kv->heads >= 0xffffffffu)  // (a tile's place is a 32-bit number)
        return fail(QH_EINVAL, "chunk_attn: a cache of %zu pages of %d tokens of %d heads is too large", kv->pages, kv->page, kv->heads);
    const int group = q_heads / kv->heads;
    auto units_of = [&](int sets) { return ((uint64_t)step->n * group / rows_of(sets) + step->n_seq) * kv->heads; };  // as many as there can be
    if (units_of(1) > 0x7fffffffu) return fail(QH_EINVAL, "chunk_attn: %zu tokens of %d heads are too many for one call", step->n, q_heads);
    if (!ctx) return fail(QH_EINVAL, "chunk_attn: null context");
    a.q = (const __bf16*)q, a.gate = (const __bf16*)gate, a.out = (__bf16*)out;
    a.t = TreeArrays{step->start, step->len, (int64_t)step->table_ld, a.kv.page_shift, (int)step->n, step->n_seq, step->max_new,
                     group};
    a.table = step->table;
    a.scale = std::frexp(scale, &a.scale_exp) * 1.4426950408889634f;
    const uint64_t most = (step->table_ld * kv->page + KV_TILE - 1) / KV_TILE, wgs = (uint64_t)ctx_cus(ctx) * waves_of(kv->head_dim);
    // Units of 128 rows where there are less than two of 256 for each workgroup that runs at once, and none is long
    const int sets = most <= SHORT_TILES && units_of(2) < 2 * wgs ? 1 : 2;
    const uint64_t units = units_of(sets);
    // Work is shared in equal parts where units alone might leave compute units without: not where a table names few tiles, nor with many
    // units. (Which it is to be the device decides, from the lengths. What the step's own tokens see makes equal parts so long at least; where
    // they then gain nothing for sure, a second launch and the count of the tiles are spared: 2,048 tokens of 24 x 256 with none cached take
    // 131 us, 134 with them.)
    const uint64_t longest = most + UNIT_TILES;
    const double tokens = (double)step->n, per_head = (double)q_heads / rows_of(sets);
    const double least = per_head * tokens * (tokens / step->n_seq / (2 * KV_TILE) + UNIT_TILES) / std::min<uint64_t>(wgs, TREE_MAX_WGS);
    const bool gains = longest > 2 * JOIN_TILES || (double)longest > least + JOIN_TILES;
    const size_t rows = rows_of(sets), slot = rows * kv->head_dim * 4 + rows * sizeof(f4);
    if (gains && units <= MAX_UNITS && units * longest <= 0x7fffffff) {
        // (252 parts at d = 256. With the rows' sums elsewhere 256 fit: no faster for 2,048 tokens behind 30,000, and 779 us instead of 725 for 131
        // behind 120,000, cold, whose units' parts then all begin at the same tiles.)
        a.parts = (int32_t)std::min<uint64_t>({wgs, TREE_MAX_WGS, (PF_SK_PART_BYTES - TREE_MAX_WGS * sizeof(Cut)) / (2 * slot)});
        a.part = (float*)ctx_partials(ctx);
        a.part_rows = (f4*)((uint8_t*)a.part + 2 * a.parts * rows * kv->head_dim * 4);
        a.cuts = (Cut*)(a.part_rows + 2 * a.parts * rows);
    }
    auto go = [&](auto d, auto fmt) {
        constexpr int D = decltype(d)::value, FMT = decltype(fmt)::value;
        launch_kernel(sets == 1 ? chunk_attn_kernel<D, FMT, 1> : chunk_attn_kernel<D, FMT, 2>, dim3((unsigned)std::max<uint64_t>(units, a.parts)),
                      dim3(THREADS), (hipStream_t)stream, a);
        if (a.parts) launch_kernel(sets == 1 ? join_kernel<D, 1> : join_kernel<D, 2>, dim3((unsigned)a.parts, (unsigned)rows / 32, D / 64), dim3(256), (hipStream_t)stream, a);
    };
    auto of = [&](auto d) {
        if (kv->fmt == QH_KV_I8) go(d, std::integral_constant<int, QH_KV_I8>{});
        else go(d, std::integral_constant<int, QH_KV_E4M3>{});
    };
    if (kv->head_dim == 64) of(std::integral_constant<int, 64>{});
    else if (kv->head_dim == 128) of(std::integral_constant<int, 128>{});
    else of(std::integral_constant<int, 256>{});
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "chunk_attn launch: %s", hipGetErrorString(e));
    return QH_OK;
}
