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
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 8, THREADS = 64 * WAVES;  // of a workgroup: two waves a SIMD
constexpr int FAN = MAX_CLUSTER;

// buffer resource word 3 (32-bit data format, no swizzle), and the cache policy of agent-coherent loads and stores
constexpr int BUF_RSRC_WORD3 = 0x00020000;
constexpr int CPOL_SC1 = 16;

// Workgroups of a CU: what a kernel's registers leave room for.
constexpr int wgs_per_cu(int d) { return d == 64 ? 2 : 1; }

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
    int32_t row_tiles;     // log2 of a chunk's tiles of 16 rows; the waves share them, and then the cache's tiles
    int32_t fuse;          // partial results are summed by the last workgroup to arrive, else by join_kernel
    float* part;           // [2 * workgroups][rows of a chunk][D], then at byte ml_at f2 [2 * workgroups][rows of a chunk]:
    int32_t ml_at;         // maximum (log2) and sum
    int32_t* plan;         // [n_seq + 1]: base of each sequence's groups, then their number (for join_kernel)
    uint32_t* count;       // [3 * workgroups] arrivals, zero between launches: of clusters by slot, then of units
};

// The compiler moves nothing across: left free it converts a whole tile's codes ahead of its products and spills.
#define HOLD() __builtin_amdgcn_sched_barrier(0)

// eight codes as exact f16 operands
template <int FMT>
__device__ __forceinline__ h8 operands(uint32_t a, uint32_t b) {
    h2 p[4];
    if constexpr (FMT == QH_KV_I8) {
        // 0x6400 | code = 1024 + code, then - 1152 (codes are q + 128)
        const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const uint32_t m = 0x64646464u;
        p[0] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(m, a, 0x04010400u)) + off;
        p[1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(m, a, 0x04030402u)) + off;
        p[2] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(m, b, 0x04010400u)) + off;
        p[3] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(m, b, 0x04030402u)) + off;
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
        p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
        p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    }
    return h8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
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

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }

// What a workgroup holds in LDS. The queries and the tiles' scales are done with when its waves' results are joined there.
template <int D>
struct Shared {
    static constexpr int C = D / 64, DT = D / 16, HALF = D == 256 ? 8 : DT;
    int32_t base[TREE_MAX_SEQS];  // of each sequence: its first group,
    int32_t who[TREE_MAX_SEQS];   // first token | tokens << 20,
    int32_t old[TREE_MAX_SEQS];   // positions before them | (its numbers do not fit) << 31
    int32_t wave_sum[WAVES];
    int32_t last;
    float factor[16 * WAVES];
    f2 wave_ml[WAVES][16];
    union {
        struct {
            h8 q[WAVES][C][2][64];
            float tile_scale[WAVES][2][KV_TILE];
        } in;
        f4 joined[WAVES][HALF][64];
        struct {
            f2 ml[FAN][16];
            float weight[FAN][16];
            f2 row[16];  // the joined maximum and sum
        } parts;
    };
};

// The sequences' places in LDS; returns the number of their groups. Up to 64 sequences each wave makes the whole list for
// itself, more are shared by the workgroup's threads.
template <int D>
__device__ __forceinline__ int plan(const Args& a, Shared<D>& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool few = a.t.n_seq <= 64;
    int before = 0;
    for (int c = 0; c < a.t.n_seq; c += THREADS) {
        const int b = c + (few ? lane : (int)threadIdx.x);
        int v = 0;
        Seq s = {};
        if (b < a.t.n_seq) {
            s = sequence(a.t, b, 16 << a.row_tiles);
            v = a.kv.heads * s.chunks * s.groups;
        }
        int run = v;  // inclusive over the wave
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(run, o);
            if (lane >= o) run += up;
        }
        int sum = __builtin_amdgcn_readlane(run, 63);
        run += before - v;
        if (!few) {
            if (lane == 0) sh.wave_sum[wave] = sum;
            __syncthreads();
            sum = 0;
            for (int w = 0; w < WAVES; w++) {
                if (w < wave) run += sh.wave_sum[w];
                sum += sh.wave_sum[w];
            }
            __syncthreads();
        }
        if (b < a.t.n_seq) {
            sh.base[b] = run;
            sh.who[b] = s.first | s.news << 20;
            sh.old[b] = s.old | (s.bad ? 1 << 31 : 0);
        }
        before += sum;
    }
    if (!few) __syncthreads();
    return __builtin_amdgcn_readfirstlane(before);
}

// The sequence that group `at` lies in: the last with base <= at (empty ones share their successor's base).
__device__ __forceinline__ int find_seq(const int32_t* base, int n_seq, int at) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int c = 0; c < n_seq; c += 64) {
        const int b = c + lane;
        n += __popcll(__ballot(b < n_seq && base[min(b, n_seq - 1)] <= at));
    }
    return n - 1;
}

__device__ __forceinline__ b4 load_gate(const Args& a, size_t at) { return a.gate ? *(const b4*)(a.gate + at) : b4{}; }

// A row's output: four of its dimensions, divided by the sum and gated.
__device__ __forceinline__ void put_out(const Args& a, size_t at, f4 v, float total, b4 gate) {
    v *= total > 0.0f || total != total ? 1.0f / total : 0.0f;
    if (a.gate) {
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] *= sigmoid((float)gate[u]);
    }
    *(b4*)(a.out + at) = __builtin_convertvector(v, b4);
}

// `count` partial results of one unit, those of workgroups w0, w0 + step, .., summed relative to their largest maximum in
// that order: into the outputs (`out`), or back into the first one's place. (Chunks of 16 rows.)
template <int D, class Row>
__device__ __forceinline__ void join_parts(const Args& a, Shared<D>& sh, __amdgpu_buffer_rsrc_t rsrc, int first_slot, int w0, int step,
                                           int count, int live, bool out, Row&& row_of) {
    constexpr int V = D / 4, ITEMS = (16 * V + THREADS - 1) / THREADS, DEEP = 16 / ITEMS;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // what follows from it is made here, not kept in registers over the whole kernel
    auto slot = [&](int i) { return i == 0 ? first_slot : 2 * (w0 + i * step); };
    f4 sum[ITEMS], in[DEEP][ITEMS];
    auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < DEEP; k++)
#pragma unroll
            for (int j = 0; j < ITEMS; j++) {
                const int e = j * THREADS + tid;
                if (i0 + k < count && e < live * V)
                    in[k][j] = __builtin_bit_cast(
                        f4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (uint32_t)slot(i0 + k) * (16 * D * 4) + e * 16, 0, CPOL_SC1));
            }
    };
    __syncthreads();
    for (int e = tid; e < count * 16; e += THREADS)
        sh.parts.ml[e >> 4][e & 15] = __builtin_bit_cast(
            f2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, a.ml_at + ((uint32_t)slot(e >> 4) * 16 + (e & 15)) * 8, 0, CPOL_SC1));
    load(0);
    b4 gate[ITEMS];
    size_t at[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        const int e = j * THREADS + tid, r = min(e / V, live - 1);
        at[j] = row_of(r) + e % V * 4;
        if (out) gate[j] = load_gate(a, at[j]);
        sum[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __syncthreads();
    if (tid < live) {
        float best = -INFINITY, total = 0.0f;
#pragma unroll 4
        for (int i = 0; i < count; i++) best = fmaxf(best, sh.parts.ml[i][tid].x);
#pragma unroll 4
        for (int i = 0; i < count; i++) {
            const f2 v = sh.parts.ml[i][tid];
            const float by = v.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v.x - best);
            total += v.x == -INFINITY ? v.y : v.y * by;  // (without a maximum: 0 or NaN)
            sh.parts.weight[i][tid] = by;
        }
        sh.parts.row[tid] = f2{best, total};
    }
    __syncthreads();
    for (int i0 = 0; i0 < count; i0 += DEEP) {
#pragma unroll
        for (int k = 0; k < DEEP; k++)
#pragma unroll
            for (int j = 0; j < ITEMS; j++) {
                const int e = j * THREADS + tid;
                if (i0 + k < count && e < live * V) sum[j] += sh.parts.weight[i0 + k][e / V] * in[k][j];
            }
        if (i0 + DEEP < count) load(i0 + DEEP);
    }
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        const int e = j * THREADS + tid;
        if (e >= live * V) continue;
        if (out) put_out(a, at[j], sum[j], sh.parts.row[e / V].y, gate[j]);
        else
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, sum[j]), rsrc, (uint32_t)first_slot * (16 * D * 4) + e * 16, 0,
                                                   CPOL_SC1);
    }
    if (!out && tid < live)
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, sh.parts.row[tid]), rsrc,
                                              a.ml_at + ((uint32_t)first_slot * 16 + tid) * 8, 0, CPOL_SC1);
}

// Whether this workgroup is the last of `of` to come here since the counter was zero; it sets it back to zero.
__device__ __forceinline__ bool last_of(uint32_t* counter, int of, int32_t* flag) {
    __builtin_amdgcn_s_waitcnt(0);  // this wave's partial has been performed
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool l = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(of - 1);
        if (l) (void)__hip_atomic_exchange(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = l;
    }
    __syncthreads();
    return *flag != 0;
}

// The work is a row of groups: for each sequence, kv head and chunk of rows, the cache in groups of 8 x 64 tokens. The
// workgroups share it in equal parts, across the borders of sequences; consecutive parts on one XCD, whose L2 then serves
// the chunks that read the same cache. In a workgroup a wave has 16 of the chunk's rows, and takes turns at the cache's
// tiles with the other waves of these rows; each keeps its own softmax, and they are joined in LDS. What covers a
// sequence's whole cache is written out, the rest as partial results: at most one at the start of a workgroup's part and
// one at its end. They are summed in their order by join_kernel, or (`fuse`) here: each workgroup writes its own
// (device-coherent stores) and counts itself, and the last to arrive sums them; from more than 16 on in two steps,
// clusters of neighbours and then the clusters' sums. No workgroup waits for another.
template <int D, int FMT>
__global__ __launch_bounds__(THREADS, 2 * wgs_per_cu(D)) void tree_attn_kernel(const Args a) {
    constexpr int C = D / 64, DT = D / 16, HALF = Shared<D>::HALF;
    __shared__ Shared<D> sh;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int all = plan<D>(a, sh), used = min((int)gridDim.x, all);
    if (blockIdx.x == 0 && !a.fuse)
        for (int i = threadIdx.x; i <= a.t.n_seq; i += THREADS) a.plan[i] = i < a.t.n_seq ? sh.base[i] : all;
    // consecutive parts on one XCD (workgroups b, b + 8, .. run on the same one)
    const int xcd = blockIdx.x & 7, at_xcd = blockIdx.x >> 3;
    if (at_xcd >= (used >> 3) + (xcd < (used & 7) ? 1 : 0)) return;
    const int w = xcd * (used >> 3) + min(xcd, used & 7) + at_xcd;
    // (what all lanes have alike is said to be so where it comes through LDS or a division: addresses are then scalar)
    const int lo = __builtin_amdgcn_readfirstlane(first_group(w, all, used));
    const int hi = __builtin_amdgcn_readfirstlane(first_group(w + 1, all, used));
    const int page = 1 << a.kv.page_shift, rows = 16 << a.row_tiles;
    const int turns = WAVES >> a.row_tiles, turn = wave & (turns - 1), rt = wave >> (3 - a.row_tiles);
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(a.part, 0, (int)PF_SK_PART_BYTES, BUF_RSRC_WORD3);
    for (int at = lo; at < hi;) {
        const int b = find_seq(sh.base, a.t.n_seq, at);
        const int who = __builtin_amdgcn_readfirstlane(sh.who[b]), was = __builtin_amdgcn_readfirstlane(sh.old[b]);
        const int past = at - __builtin_amdgcn_readfirstlane(sh.base[b]);
        const int first = who & 0xfffff, news = who >> 20, old = was & 0x7fffffff, total = old + news;
        const int chunks = (news * a.t.group + rows - 1) >> (4 + a.row_tiles);
        const int groups = (total + KV_TILE * GROUP_TILES - 1) / (KV_TILE * GROUP_TILES);
        const int unit = __builtin_amdgcn_readfirstlane(past / groups), g0 = past - unit * groups;
        const int g1 = min(groups, g0 + hi - at);
        const int head = __builtin_amdgcn_readfirstlane(unit / chunks), row0 = (unit - head * chunks) * rows;
        const int live = min(rows, news * a.t.group - row0);
        const int tiles = (total + KV_TILE - 1) / KV_TILE;
        const int t_first = g0 * GROUP_TILES + turn, t_end = rt * 16 < live ? min(tiles, g1 * GROUP_TILES) : 0;

        // pages of the wave's tiles, 64 at a time: lane l has its l-th tile's
        int32_t pages = 0;
        auto load_pages = [&](int t) {
            const int mine = t + lane * turns;
            if (mine < t_end) pages = a.table[(size_t)b * a.t.table_ld + ((mine * KV_TILE) >> a.kv.page_shift)];
        };
        load_pages(t_first);

        auto node_of = [&](int r) { return (int)((uint32_t)r * a.group_inv >> 20); };  // r / group
        // first element of a row's query, gate and output
        auto row_at = [&](int r) {
            const int node = node_of(row0 + r);
            return ((size_t)(first + node) * a.kv.heads * a.t.group + head * a.t.group + (row0 + r - node * a.t.group)) * D;
        };
        // the queries: a thread has 16 dimensions of a row
        constexpr int PER_ROW = D / 16, PASS = THREADS / PER_ROW;
        const int q_row = threadIdx.x / PER_ROW, q_part = threadIdx.x % PER_ROW;
        b8 raw[2];
        auto load_query = [&](int r) {
            const __bf16* const qp = a.q + row_at(min(r, live - 1)) + q_part * 16;
            raw[0] = *(const b8*)qp, raw[1] = *(const b8*)(qp + 8);
        };
        load_query(q_row);
        const int my_node = node_of(row0 + min(rt * 16 + col, live - 1));
        // of its sequence's tokens of this step
        const uint64_t sees = (a.mask ? a.mask[first + my_node] : ~0ull >> (63 - my_node)) & ~0ull >> (64 - news);

        u4 kc[4][C], vc[DT];
        float sk, sv;
        const uint8_t* block = a.kv.codes;  // a tile's keys; its values lie one block on
        const float* scales = a.kv.scales;
        bool none = false;
        // a page that the cache has not gives NaN
        auto find = [&](int t, int i) {
            int64_t pg = __builtin_amdgcn_readlane(pages, i & 63);
            none = pg < 0 || (pg << a.kv.page_shift) >= a.kv.slots;
            if (none) pg = 0;
            const int in = (t * KV_TILE) & (page - 1);
            block = a.kv.codes + kv_block<D>(a.kv, pg, head, 0) + (size_t)in * D;
            scales = a.kv.scales + kv_scale(a.kv, pg, head, 0) + in;
        };
        const uint32_t k_lane = col * 64 + g * 16;
        auto load_keys = [&](int t) {  // keys and scales (lane l: token l's)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int sub = 0; sub < 4; sub++) kc[sub][c] = *(const u4*)(block + sub * 16 * D + c * 1024 + k_lane);
            sk = none ? NAN : scales[lane];
            sv = t * KV_TILE + lane < total ? scales[page + lane] : 0.0f;
        };
        auto load_values = [&]() {
            const uint8_t* const vp = block + ((size_t)D << a.kv.page_shift);
#pragma unroll
            for (int i = 0; i < DT; i++) vc[i] = *(const u4*)(vp + i * 1024 + k_lane);
        };
        if (t_first < t_end) {
            find(t_first, 0);
            load_keys(t_first);
        }

        // the queries, scaled by a power of two into f16's range (the factor goes to the scores)
        for (int r = q_row;;) {
            float top = 0.0f, odd = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float v = (float)raw[i >> 3][i & 7];
                top = fmaxf(top, fabsf(v));
                odd += v * 0.0f;  // NaN where v is not finite
            }
#pragma unroll
            for (int o = 1; o < PER_ROW; o <<= 1) top = fmaxf(top, __shfl_xor(top, o)), odd += __shfl_xor(odd, o);
            const int e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
            if (r < rows) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    h8 q;
#pragma unroll
                    for (int i = 0; i < 8; i++) q[i] = (_Float16)__builtin_ldexpf((float)raw[k][i], -e);
                    sh.in.q[r >> 4][q_part >> 2][k][(q_part & 3) * 16 + (r & 15)] = q;
                }
                if (q_part == 0) sh.factor[r] = fmaxf(__builtin_ldexpf(a.scale, e), 1e-37f) + odd + (was < 0 ? NAN : 0.0f);
            }
            r += PASS;
            if (r - q_row >= rows) break;
            load_query(r);
        }
        if (t_first < t_end) load_values();
        __syncthreads();
        const float factor = sh.factor[rt * 16 + col];
        float top = -INFINITY, sum = 0.0f;
        f4 o[DT];
        float ref = 0x1p-126f;  // the values' scales are taken relative to this power of two: probabilities fit f16
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};

        for (int t = t_first, it = 1; t < t_end; t += turns, it++) {
            const int t0 = t * KV_TILE;
            // s^T = k q^T: lane (col, g) gets row `col` of tokens 16 sub + 4 g + i
            f4 x[4];
#pragma unroll
            for (int sub = 0; sub < 4; sub++) x[sub] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; c++) {
                const h8 q0 = sh.in.q[rt][c][0][lane], q1 = sh.in.q[rt][c][1][lane];
#pragma unroll
                for (int sub = 0; sub < 4; sub++) {
                    const h8 k0 = operands<FMT>(kc[sub][c].x, kc[sub][c].y), k1 = operands<FMT>(kc[sub][c].z, kc[sub][c].w);
                    x[sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q0, x[sub], 0, 0, 0);
                    x[sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q1, x[sub], 0, 0, 0);
                }
                HOLD();
            }

            // the values' scales relative to ref; ref grows to the largest finite one's power of two
            float grow = 1.0f;
            if (__any(sv > ref && sv < INFINITY)) {
                float m = sv < INFINITY ? sv : 0.0f;
                for (int of = 32; of; of >>= 1) m = fmaxf(m, __shfl_xor(m, of));
                const float next = __builtin_ldexpf(1.0f, min(__builtin_amdgcn_frexp_expf(m), 127));
                grow = ref * (1.0f / next);
                ref = next;
            }
            float(&ts)[2][KV_TILE] = sh.in.tile_scale[wave];
            ts[0][lane] = sk;
            ts[1][lane] = sv * (1.0f / ref);
            const bool more = t + turns < t_end;
            if (more) {
                if ((it & 63) == 0) load_pages(t + turns);
                find(t + turns, it);
                load_keys(t + turns);
            }
            HOLD();
            __builtin_amdgcn_wave_barrier();

            h8 p[2];
            const bool whole = t0 + KV_TILE <= old;  // every row sees every token
            uint64_t seen = 0;                       // bit i: the row sees token t0 + i
            if (!whole) {
                const int node = t0 - old;  // above -64
                seen = node >= 64 ? 0 : node >= 0 ? sees >> node : sees << -node | ((1ull << -node) - 1);
            }
            float mx = -INFINITY;
#pragma unroll
            for (int sub = 0; sub < 4; sub++) {
                x[sub] *= *(const f4*)&ts[0][sub * 16 + g * 4];
                if (!whole) {
                    const uint32_t bits = (uint32_t)(seen >> (sub * 16 + g * 4));
#pragma unroll
                    for (int i = 0; i < 4; i++) x[sub][i] = bits & (1u << i) ? x[sub][i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, x[sub][i]);
            }
            // the maximum is followed only where it has grown by more than 2^8 (the sums and f16 hold that)
            const float next = fmaxf(top, row_max(mx));
            float by = grow;
            if (__any((next - top) * factor > 8.0f)) {
                const float al = next > top ? __builtin_amdgcn_exp2f((top - next) * factor) : 1.0f;
                sum *= al;
                top = next;
                by *= al;
            }
            if (t != t_first && __any(by != 1.0f))
#pragma unroll
                for (int i = 0; i < DT; i++) o[i] *= by;
            const float off = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int sub = 0; sub < 4; sub++) {
                const f4 vs = *(const f4*)&ts[1][sub * 16 + g * 4];
                float pv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float pr = __builtin_amdgcn_exp2f((x[sub][i] - off) * factor);
                    pv[i] = pr * vs[i];
                    if (!whole) pv[i] = x[sub][i] == -INFINITY ? 0.0f : pv[i];
                    sum += pr;
                }
                const h2 a0 = __builtin_convertvector((f2{pv[0], pv[1]}), h2);
                const h2 a1 = __builtin_convertvector((f2{pv[2], pv[3]}), h2);
                h8& to = p[sub >> 1];
                const int k = (sub & 1) * 4;
                to[k] = a0.x, to[k + 1] = a0.y, to[k + 2] = a1.x, to[k + 3] = a1.y;
            }
            HOLD();
            if (t0 + KV_TILE > total) {  // codes that no token of this sequence wrote may be anything: none are multiplied
                u4 keep;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int have = total - (t0 + k * 16 + g * 4);
                    keep[k] = have >= 4 ? ~0u : have <= 0 ? 0u : (1u << (8 * have)) - 1;
                }
#pragma unroll
                for (int i = 0; i < DT; i++) vc[i] &= keep;
            }
            // o^T += v^T p^T: the k index of both operands runs over tokens 16 w + 4 g + j, as the scores lie
#pragma unroll
            for (int i = 0; i < DT; i++) {
                const h8 v0 = operands<FMT>(vc[i].x, vc[i].y), v1 = operands<FMT>(vc[i].z, vc[i].w);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[0], o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[1], o[i], 0, 0, 0);
                if (i % 4 == 3) HOLD();
            }
            if (more) load_values();
        }

        // the waves' results joined, and written out or as a partial result
        const bool direct = g0 == 0 && g1 == groups;
        const int slot = 2 * w + (at != lo);
        {
            int el = lane;
            asm volatile("" : "+v"(el));  // as in join_parts
            const int col = el & 15, g = el >> 4, r = rt * 16 + col;
            const bool mine = r < live;
            const size_t out_at = row_at(min(r, live - 1));
            const float l = row_sum(sum), m = top == -INFINITY ? -INFINITY : top * factor;
            float best = m, total_sum = l, by = ref;
            auto put = [&](int i, f4 v, b4 gate) {
                const int d = i * 16 + g * 4;
                if (direct) put_out(a, out_at + d, v, total_sum, gate);
                else
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), rsrc, (uint32_t)((slot * rows + r) * D + d) * 4, 0,
                                                           CPOL_SC1);
            };
            if (turns > 1) {
                if (g == 0) sh.wave_ml[wave][col] = f2{m, l};
                __syncthreads();
                f2 ml[WAVES];
#pragma unroll
                for (int k = 0; k < WAVES; k++) ml[k] = sh.wave_ml[(wave & -turns) + (k & (turns - 1))][col];
                best = -INFINITY, total_sum = 0.0f;
#pragma unroll
                for (int k = 0; k < WAVES; k++) best = fmaxf(best, ml[k].x);
#pragma unroll
                for (int k = 0; k < WAVES; k++)  // (without a maximum: 0 or NaN)
                    if (k < turns) total_sum += ml[k].x == -INFINITY ? ml[k].y : ml[k].y * __builtin_amdgcn_exp2f(ml[k].x - best);
                by *= m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - best);
#pragma unroll
                for (int h = 0; h < DT / HALF; h++) {
                    if (h) __syncthreads();
#pragma unroll
                    for (int i = 0; i < HALF; i++)
                        if (mine) sh.joined[wave][i][el] = m == -INFINITY ? f4{0.0f, 0.0f, 0.0f, 0.0f} : o[h * HALF + i] * by;
                    __syncthreads();
                    if (mine)
                        for (int i = turn; i < HALF; i += turns) {
                            const b4 gate = direct ? load_gate(a, out_at + (h * HALF + i) * 16 + g * 4) : b4{};
                            f4 v = {0.0f, 0.0f, 0.0f, 0.0f}, u[WAVES];
#pragma unroll
                            for (int k = 0; k < WAVES; k++) u[k] = sh.joined[(wave & -turns) + (k & (turns - 1))][i][el];
#pragma unroll
                            for (int k = 0; k < WAVES; k++) v += k < turns ? u[k] : f4{0.0f, 0.0f, 0.0f, 0.0f};
                            put(h * HALF + i, v, gate);
                        }
                }
            } else if (mine) {
#pragma unroll
                for (int i = 0; i < DT; i++) {
                    const b4 gate = direct ? load_gate(a, out_at + i * 16 + g * 4) : b4{};
                    put(i, m == -INFINITY ? f4{0.0f, 0.0f, 0.0f, 0.0f} : o[i] * by, gate);
                }
            }
            if (!direct && turn == 0 && g == 0 && mine)
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, (f2{best, total_sum})), rsrc,
                                                      a.ml_at + (uint32_t)(slot * rows + r) * 8, 0, CPOL_SC1);
        }
        if (!direct && a.fuse) {
            const int u0 = at - g0, w0 = group_owner(u0, all, used), parts = group_owner(u0 + groups - 1, all, used) - w0 + 1;
            const Cluster k = cluster(w - w0, parts);
            const int kw = w0 + k.first, k_slot = partial_slot(kw, u0, all, used);
            // the cluster's parts, then the clusters' sums; the last of either to arrive goes on
            int from = kw, first_slot = k_slot, step = 1, count = k.size;
            uint32_t* counter = a.count + k_slot;
            for (bool out = k.of == 1;;) {
                if (count > 1) {
                    if (!last_of(counter, count, &sh.last)) break;
                    join_parts<D>(a, sh, rsrc, first_slot, from, step, count, live, out, row_at);
                }
                if (out) break;
                from = w0, first_slot = partial_slot(w0, u0, all, used), step = k.step, count = k.of;
                counter = a.count + 2 * gridDim.x + w0;
                out = true;
            }
        }
        __syncthreads();
        at += g1 - g0;
    }
}

// The partial results of the rows whose cache several workgroups shared, a workgroup per row: D / 4 threads hold four
// dimensions each, 1024 / D such sets take partials in turn, relative to the largest maximum, and are summed in LDS.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(const Args a, int grid) {
    constexpr int V = D / 4, SETS = 256 / V, DEEP = 8;
    __shared__ f4 sums[SETS][V];
    const int heads = a.kv.heads * a.t.group, rows = 16 << a.row_tiles;
    const int token = blockIdx.x / heads, h = blockIdx.x - token * heads, head = h / a.t.group;
    const int lane = threadIdx.x & 63, v4 = threadIdx.x % V, set = threadIdx.x / V;
    const int all = a.plan[a.t.n_seq], used = min(grid, all);
    const int b = max(0, find_seq(a.t.start, a.t.n_seq, token));  // the last sequence with start <= token
    const Seq s = sequence(a.t, b, rows);
    const int node = token - s.first;
    if (node < 0 || node >= s.news) return;
    const int r = node * a.t.group + h - head * a.t.group;
    const int u0 = a.plan[b] + (head * s.chunks + (r >> (4 + a.row_tiles))) * s.groups, u1 = u0 + s.groups;
    const int w0 = group_owner(u0, all, used), parts = group_owner(u1 - 1, all, used) - w0 + 1;
    if (parts == 1) return;  // one workgroup wrote the row
    const int first_slot = partial_slot(w0, u0, all, used), in = r & (rows - 1);
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
                y[k] = *(const f4*)(a.part + slot(i) * D + v4 * 4);
            }
        }
    };
    load(set);
    const size_t at = (size_t)blockIdx.x * D + v4 * 4;
    const b4 gate = load_gate(a, at);
    f2 mine = lane < parts ? ml[slot(lane)] : f2{-INFINITY, 0.0f};
    for (int i = lane + 64; i < parts; i += 64) {
        const f2 u = ml[slot(i)];
        const float best = fmaxf(mine.x, u.x);
        mine.y = (mine.x == -INFINITY ? mine.y : mine.y * __builtin_amdgcn_exp2f(mine.x - best)) +
                 (u.x == -INFINITY ? u.y : u.y * __builtin_amdgcn_exp2f(u.x - best));
        mine.x = best;
    }
    float best = mine.x;
    for (int o = 32; o; o >>= 1) best = fmaxf(best, __shfl_xor(best, o));
    float total = mine.x == -INFINITY ? mine.y : mine.y * __builtin_amdgcn_exp2f(mine.x - best);
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
    for (int i0 = set; i0 < parts; i0 += SETS * DEEP) {
#pragma unroll
        for (int k = 0; k < DEEP; k++)
            if (i0 + k * SETS < parts) v += (m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - best)) * y[k];
        if (i0 + SETS * DEEP < parts) load(i0 + SETS * DEEP);
    }
    sums[set][v4] = v;
    __syncthreads();
    if (set) return;
    for (int k = 1; k < SETS; k++) v += sums[k][v4];
    put_out(a, at, v, total, gate);
}

template <int D, int FMT>
void launch(hipStream_t stream, const Args& a, int grid, bool join) {
    hipLaunchKernelGGL((tree_attn_kernel<D, FMT>), dim3(grid), dim3(THREADS), 0, stream, a);
    if (join) hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)(a.t.n * a.kv.heads * a.t.group)), dim3(256), 0, stream, a, grid);
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
    const int64_t cap = (int64_t)step->table_ld * kv->page;  // positions that a table can name
    if (step->table_ld < 1 || step->table_ld > ((size_t)1 << 30) / kv->page)
        return fail(QH_EINVAL, "tree_attn: tables of %zu pages of %d tokens (1 to 2^30 positions)", step->table_ld, kv->page);
    const int group = q_heads / kv->heads;
    const int64_t groups = (cap + KV_TILE * GROUP_TILES - 1) / (KV_TILE * GROUP_TILES);  // of the longest sequence there can be
    const int64_t most = (int64_t)(ctx ? ctx_cus(ctx) : 1) * wgs_per_cu(kv->head_dim);
    auto units_of = [&](int rt) { return (int64_t)kv->heads * ((step->max_new * group + (16 << rt) - 1) >> (4 + rt)); };
    // A chunk's rows: all of them, up to 128, while that leaves work for every CU.
    int rt = 0;
    while (rt < 3 && step->max_new * group > 16 << rt && units_of(rt + 1) * step->n_seq * groups >= most) rt++;
    const int rows = 16 << rt;
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
    const int grid = (int)std::min({most, units * step->n_seq * groups, (int64_t)MAX_CLUSTER * MAX_CLUSTER});
    static_assert(3 * MAX_CLUSTER * MAX_CLUSTER <= PF_SK_ITEMS_MAX);
    const size_t part = (size_t)2 * grid * rows * kv->head_dim * 4, ml = (size_t)2 * grid * rows * 8;
    if (part + ml + (TREE_MAX_SEQS + 1) * 4 > PF_SK_PART_BYTES) return fail(QH_EINVAL, "tree_attn: scratch");
    a.row_tiles = rt;
    a.part = (float*)ctx_partials(ctx);
    a.ml_at = (int32_t)part;
    a.plan = (int32_t*)((uint8_t*)ctx_partials(ctx) + part + ml);
    a.count = (uint32_t*)((uint8_t*)ctx_partials(ctx) + PF_SK_PART_BYTES);
    a.fuse = rt == 0;
    const bool join = !a.fuse && groups > 1 && grid > 1;
    auto go = [&](auto d) {
        if (kv->fmt == QH_KV_I8) launch<decltype(d)::value, QH_KV_I8>((hipStream_t)stream, a, grid, join);
        else launch<decltype(d)::value, QH_KV_E4M3>((hipStream_t)stream, a, grid, join);
    };
    if (kv->head_dim == 64) go(std::integral_constant<int, 64>{});
    else if (kv->head_dim == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "tree_attn launch: %s", hipGetErrorString(e));
    return QH_OK;
}
