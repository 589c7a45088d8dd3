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

constexpr int WAVES = GROUP_TILES;  // waves of a workgroup, each with tiles of its own

struct Args {
    const __bf16* q;     // [n][heads][D]
    const __bf16* gate;  // the same, or null
    __bf16* out;
    Kv kv;
    TreeArrays t;
    const int32_t* table;  // [n_seq][table_ld]
    const uint64_t* mask;  // [n], or null: a chain
    float scale;           // softmax scale * log2(e)
    float* part;           // [2 * workgroups][rows of a chunk][D]
    f2* ml;                // [2 * workgroups][rows of a chunk]: maximum (log2) and sum
    int32_t* plan;         // [n_seq + 1]: base of each sequence's groups, then their number
};

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

// The bases of the sequences' groups in LDS: base[b] for b <= n_seq (256 threads, up to four sequences each).
template <int ROWS>
__device__ void plan(const Args& a, int32_t* base, int32_t* wave_sum) {
    int v[TREE_MAX_SEQS / 256], sum = 0;
    const int per = (a.t.n_seq + 255) / 256, b0 = threadIdx.x * per;
#pragma unroll
    for (int i = 0; i < TREE_MAX_SEQS / 256; i++) {
        v[i] = 0;
        if (i < per && b0 + i < a.t.n_seq) {
            const Seq s = sequence(a.t, b0 + i, ROWS);
            v[i] = a.kv.heads * s.chunks * s.groups;
        }
        sum += v[i];
    }
    int run = sum;  // inclusive over the wave
    const int lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(run, o);
        if (lane >= o) run += up;
    }
    if (lane == 63) wave_sum[threadIdx.x >> 6] = run;
    __syncthreads();
    run -= sum;
    for (int w = 0; w < (int)(threadIdx.x >> 6); w++) run += wave_sum[w];
#pragma unroll
    for (int i = 0; i < TREE_MAX_SEQS / 256; i++)
        if (i < per && b0 + i < a.t.n_seq) {
            base[b0 + i] = run;
            run += v[i];
        }
    if (threadIdx.x == 255) base[a.t.n_seq] = run;
    __syncthreads();
}

// The work is a row of groups: for each sequence, kv head and chunk of ROWS rows, the cache in groups of 4 x 64 tokens. The
// workgroups share it in equal parts, across the borders of sequences. In a workgroup each wave takes every fourth tile
// and keeps its own softmax; the four are joined in LDS. What covers a sequence's whole cache is written out, the rest
// as a partial result for join_kernel: at most one at the start of a workgroup's part and one at its end.
template <int D, int FMT, int RT>
__global__ __launch_bounds__(64 * WAVES, RT == 1 ? 2 : 1) void tree_attn_kernel(const Args a) {
    constexpr int C = D / 64, DT = D / 16, ROWS = 16 * RT;
    __shared__ int32_t base[TREE_MAX_SEQS + 1];
    __shared__ int32_t wave_sum[WAVES];
    __shared__ float tile_scale[WAVES][2][KV_TILE];
    __shared__ f2 wave_ml[WAVES][ROWS];
    __shared__ f4 joined[WAVES][DT][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    plan<ROWS>(a, base, wave_sum);
    const int all = base[a.t.n_seq], used = min((int)gridDim.x, all), w = blockIdx.x;
    if (w == 0)
        for (int i = threadIdx.x; i <= a.t.n_seq; i += 64 * WAVES) a.plan[i] = base[i];
    if (w >= used) return;
    const int lo = first_group(w, all, used), hi = first_group(w + 1, all, used);
    const int page = 1 << a.kv.page_shift;
    for (int at = lo; at < hi;) {
        int b = 0;  // the sequence that `at` lies in: the last with base <= at (empty ones share their successor's base)
        for (int step = 512; step; step >>= 1)
            if (b + step < a.t.n_seq && base[b + step] <= at) b += step;
        const Seq s = sequence(a.t, b, ROWS);
        const int unit = (at - base[b]) / s.groups, g0 = (at - base[b]) - unit * s.groups;
        const int g1 = min(s.groups, g0 + hi - at);
        const int head = unit / s.chunks, row0 = (unit - head * s.chunks) * ROWS;
        const int tiles = (s.total + KV_TILE - 1) / KV_TILE, t_end = min(tiles, g1 * WAVES);

        // the rows' queries, scaled by a power of two into f16's range (the factor goes to the scores), and what they see
        h8 qf[RT][C][2];
        float factor[RT];
        uint64_t sees[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const int r = row0 + rt * 16 + col, node = r / a.t.group;
            const bool live = node < s.news;
            const __bf16* qp = a.q + ((size_t)(s.first + (live ? node : 0)) * a.kv.heads * a.t.group + head * a.t.group +
                                      (live ? r - node * a.t.group : 0)) * D;
            float top = 0.0f, odd = 0.0f;
            b8 raw[C][2];
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    raw[c][k] = *(const b8*)(qp + c * 64 + g * 16 + k * 8);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float v = (float)raw[c][k][i];
                        top = fmaxf(top, fabsf(v));
                        odd += v * 0.0f;  // NaN where v is not finite
                    }
                }
            top = row_max(top);
            odd = row_sum(odd);
            int e = 0;
            if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e);
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    qf[rt][c][i >> 3][i & 7] = live ? (_Float16)ldexpf((float)raw[c][i >> 3][i & 7], -e) : (_Float16)0.0f;
            factor[rt] = fmaxf(ldexpf(a.scale, e), 1e-37f) + odd + (s.bad ? NAN : 0.0f);
            sees[rt] = !live ? 0 : a.mask ? a.mask[s.first + node] : ~0ull >> (63 - node);
        }

        f4 o[RT][DT];
        float top[RT], sum[RT];
        float ref = 0x1p-126f;  // the values' scales are taken relative to this power of two: probabilities fit f16
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            top[rt] = -INFINITY, sum[rt] = 0.0f;
#pragma unroll
            for (int i = 0; i < DT; i++) o[rt][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        u4 kc[4][C];
        float sk, sv;
        const uint8_t* vp;
        // a tile's keys and scales (lane l: token l's), and where its values lie; a page that the cache has not gives NaN
        auto load_keys = [&](int t) {
            const int t0 = t * KV_TILE;
            int64_t pg = a.table[(size_t)b * a.t.table_ld + (t0 >> a.kv.page_shift)];
            const bool none = pg < 0 || (pg << a.kv.page_shift) >= a.kv.slots;
            if (none) pg = 0;
            const int in = t0 & (page - 1);
            const uint8_t* kp = a.kv.codes + kv_block<D>(a.kv, pg, head, 0) + (size_t)in * D + col * 64 + g * 16;
            vp = kp + ((size_t)D << a.kv.page_shift);
#pragma unroll
            for (int sub = 0; sub < 4; sub++)
#pragma unroll
                for (int c = 0; c < C; c++) kc[sub][c] = *(const u4*)(kp + sub * 16 * D + c * 1024);
            const float* sp = a.kv.scales + kv_scale(a.kv, pg, head, 0) + in + lane;
            sk = none ? NAN : sp[0];
            sv = t0 + lane < s.total ? sp[page] : 0.0f;
        };
        int t = g0 * WAVES + wave;
        if (t < t_end) load_keys(t);
        for (; t < t_end; t += WAVES) {
            const int t0 = t * KV_TILE;
            u4 vc[DT];
#pragma unroll
            for (int i = 0; i < DT; i++) vc[i] = *(const u4*)(vp + i * 1024);

            // s^T = k q^T: lane (col, g) gets row `col` of tokens 16 sub + 4 g + i
            f4 x[RT][4];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int sub = 0; sub < 4; sub++) x[rt][sub] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int sub = 0; sub < 4; sub++) {
                    const h8 k0 = operands<FMT>(kc[sub][c].x, kc[sub][c].y), k1 = operands<FMT>(kc[sub][c].z, kc[sub][c].w);
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        x[rt][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[rt][c][0], x[rt][sub], 0, 0, 0);
                        x[rt][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[rt][c][1], x[rt][sub], 0, 0, 0);
                    }
                }

            // the values' scales relative to ref; ref grows to the largest finite one's power of two
            float grow = 1.0f;
            if (__any(sv > ref && sv < INFINITY)) {
                float m = sv < INFINITY ? sv : 0.0f;
                for (int of = 32; of; of >>= 1) m = fmaxf(m, __shfl_xor(m, of));
                int e;
                (void)frexpf(m, &e);
                const float next = ldexpf(1.0f, min(e, 127));
                grow = ref / next;
                ref = next;
            }
            tile_scale[wave][0][lane] = sk;
            tile_scale[wave][1][lane] = sv / ref;
            if (t + WAVES < t_end) load_keys(t + WAVES);
            __builtin_amdgcn_wave_barrier();
            f4 ks[4], vs[4];
#pragma unroll
            for (int sub = 0; sub < 4; sub++) {
                ks[sub] = *(const f4*)&tile_scale[wave][0][sub * 16 + g * 4];
                vs[sub] = *(const f4*)&tile_scale[wave][1][sub * 16 + g * 4];
            }
            __builtin_amdgcn_wave_barrier();

            h8 p[RT][2];
            const bool whole = t0 + KV_TILE <= s.old;  // every row sees every token
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                float mx = -INFINITY;
#pragma unroll
                for (int sub = 0; sub < 4; sub++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float v = x[rt][sub][i] * ks[sub][i];
                        if (!whole) {
                            const int node = t0 + sub * 16 + g * 4 + i - s.old;
                            const bool seen = node < 0 || (node < s.news && (sees[rt] >> (node & 63) & 1));
                            v = seen ? v : -INFINITY;
                        }
                        x[rt][sub][i] = v;
                        mx = fmaxf(mx, v);
                    }
                const float next = fmaxf(top[rt], row_max(mx));
                if (grow != 1.0f || __any(next > top[rt])) {
                    const float al = next > top[rt] ? __builtin_amdgcn_exp2f((top[rt] - next) * factor[rt]) : 1.0f;
                    sum[rt] *= al;
                    top[rt] = next;
                    const float by = al * grow;
#pragma unroll
                    for (int i = 0; i < DT; i++) o[rt][i] *= by;
                }
                const float off = top[rt] == -INFINITY ? 0.0f : top[rt];
#pragma unroll
                for (int sub = 0; sub < 4; sub++) {
                    float pr[4], pv[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        pr[i] = __builtin_amdgcn_exp2f((x[rt][sub][i] - off) * factor[rt]);
                        pv[i] = pr[i] * vs[sub][i];
                        if (!whole) pv[i] = x[rt][sub][i] == -INFINITY ? 0.0f : pv[i];
                        sum[rt] += pr[i];
                    }
                    const h2 a0 = __builtin_convertvector((f2{pv[0], pv[1]}), h2);
                    const h2 a1 = __builtin_convertvector((f2{pv[2], pv[3]}), h2);
                    h8& to = p[rt][sub >> 1];
                    const int k = (sub & 1) * 4;
                    to[k] = a0.x, to[k + 1] = a0.y, to[k + 2] = a1.x, to[k + 3] = a1.y;
                }
            }
            if (t0 + KV_TILE > s.total) {  // codes that no token of this sequence wrote may be anything: none are multiplied
                u4 keep;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int have = s.total - (t0 + k * 16 + g * 4);
                    keep[k] = have >= 4 ? ~0u : have <= 0 ? 0u : (1u << (8 * have)) - 1;
                }
#pragma unroll
                for (int i = 0; i < DT; i++) vc[i] &= keep;
            }
            // o^T += v^T p^T: the k index of both operands runs over tokens 16 w + 4 g + j, as the scores lie
#pragma unroll
            for (int i = 0; i < DT; i++) {
                const h8 v0 = operands<FMT>(vc[i].x, vc[i].y), v1 = operands<FMT>(vc[i].z, vc[i].w);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[rt][0], o[rt][i], 0, 0, 0);
                    o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[rt][1], o[rt][i], 0, 0, 0);
                }
            }
        }

        // the four waves' results joined
        const bool direct = g0 == 0 && g1 == s.groups;
        const int slot = 2 * w + (at != lo);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float l = row_sum(sum[rt]), m = top[rt] == -INFINITY ? -INFINITY : top[rt] * factor[rt];
            if (g == 0) wave_ml[wave][rt * 16 + col] = f2{m, l};
            __syncthreads();
            float best = -INFINITY, total = 0.0f;
#pragma unroll
            for (int k = 0; k < WAVES; k++) best = fmaxf(best, wave_ml[k][rt * 16 + col].x);
#pragma unroll
            for (int k = 0; k < WAVES; k++) {
                const f2 v = wave_ml[k][rt * 16 + col];
                total += v.x == -INFINITY ? v.y : v.y * __builtin_amdgcn_exp2f(v.x - best);  // (without a maximum: 0 or NaN)
            }
            const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - best) * ref;
#pragma unroll
            for (int i = 0; i < DT; i++) joined[wave][i][lane] = m == -INFINITY ? f4{0.0f, 0.0f, 0.0f, 0.0f} : o[rt][i] * by;
            __syncthreads();
            const int r = row0 + rt * 16 + col, node = r / a.t.group;
            const size_t token_head = (size_t)(s.first + node) * a.kv.heads * a.t.group + head * a.t.group + (r - node * a.t.group);
            const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
#pragma unroll
            for (int k = 0; k < DT / WAVES; k++) {
                const int i = wave * (DT / WAVES) + k;
                f4 v = joined[0][i][lane];
#pragma unroll
                for (int u = 1; u < WAVES; u++) v += joined[u][i][lane];
                const int d = i * 16 + g * 4;
                if (!direct) {
                    *(f4*)(a.part + ((size_t)slot * ROWS + rt * 16 + col) * D + d) = v;
                } else if (node < s.news) {
                    v *= inv;
                    if (a.gate) {
                        const b4 gt = *(const b4*)(a.gate + token_head * D + d);
#pragma unroll
                        for (int u = 0; u < 4; u++) v[u] *= sigmoid((float)gt[u]);
                    }
                    *(b4*)(a.out + token_head * D + d) = __builtin_convertvector(v, b4);
                }
            }
            if (!direct && wave == 0 && g == 0) a.ml[(size_t)slot * ROWS + rt * 16 + col] = f2{best, total};
        }
        __syncthreads();
        at += g1 - g0;
    }
}

// The partial results of the rows whose cache several workgroups shared, a workgroup per row: its waves take partials in
// turn, relative to the largest maximum, and are summed in LDS.
template <int D, int ROWS>
__global__ __launch_bounds__(512) void join_kernel(const Args a, int grid) {
    constexpr int W = 8, V = D / 64;
    __shared__ float sums[W][D];
    const int heads = a.kv.heads * a.t.group;
    const int token = blockIdx.x / heads, h = blockIdx.x - token * heads, head = h / a.t.group;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int b = 0;  // the last sequence with start <= token and tokens of its own
    for (int step = 512; step; step >>= 1)
        if (b + step < a.t.n_seq && a.t.start[b + step] <= token) b += step;
    const Seq s = sequence(a.t, b, ROWS);
    const int node = token - s.first;
    if (node < 0 || node >= s.news) return;
    const int all = a.plan[a.t.n_seq], used = min(grid, all);
    const int r = node * a.t.group + h - head * a.t.group;
    const int u0 = a.plan[b] + (head * s.chunks + r / ROWS) * s.groups, u1 = u0 + s.groups;
    const int w0 = group_owner(u0, all, used), w1 = group_owner(u1 - 1, all, used);
    if (w0 == w1) return;  // one workgroup wrote the row
    auto slot = [&](int w) { return (size_t)partial_slot(w, u0, all, used) * ROWS + r % ROWS; };
    float best = -INFINITY;
    for (int w = w0 + lane; w <= w1; w += 64) best = fmaxf(best, a.ml[slot(w)].x);
    for (int o = 32; o; o >>= 1) best = fmaxf(best, __shfl_xor(best, o));
    float total = 0.0f;
    for (int w = w0 + lane; w <= w1; w += 64) {
        const f2 v = a.ml[slot(w)];
        total += v.x == -INFINITY ? v.y : v.y * __builtin_amdgcn_exp2f(v.x - best);
    }
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
    float v[V] = {};
    for (int w = w0 + wave; w <= w1; w += W) {
        const size_t at = slot(w);
        const float m = a.ml[at].x, by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - best);
#pragma unroll
        for (int k = 0; k < V; k++) v[k] += by * a.part[at * D + k * 64 + lane];
    }
#pragma unroll
    for (int k = 0; k < V; k++) sums[wave][k * 64 + lane] = v[k];
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < W; k++) y += sums[k][d];
    y = total > 0.0f || total != total ? y / total : 0.0f;
    const size_t at = (size_t)blockIdx.x * D + d;
    if (a.gate) y *= sigmoid((float)a.gate[at]);
    a.out[at] = (__bf16)y;
}

template <int D, int FMT, int RT>
void launch(hipStream_t stream, const Args& a, int grid, bool join) {
    hipLaunchKernelGGL((tree_attn_kernel<D, FMT, RT>), dim3(grid), dim3(64 * WAVES), 0, stream, a);
    if (join)
        hipLaunchKernelGGL((join_kernel<D, 16 * RT>), dim3((unsigned)(a.t.n * a.kv.heads * a.t.group)), dim3(512), 0, stream, a, grid);
}

template <int D, int FMT>
void launch_rows(hipStream_t stream, const Args& a, int rt, int grid, bool join) {
    if (rt == 1) launch<D, FMT, 1>(stream, a, grid, join);
    else launch<D, FMT, 2>(stream, a, grid, join);
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
    const int group = q_heads / kv->heads, rt = step->max_new * group > 16 ? 2 : 1, rows = 16 * rt;
    const int64_t groups = (cap + KV_TILE * WAVES - 1) / (KV_TILE * WAVES);  // of the longest sequence there can be
    const int64_t units = (int64_t)kv->heads * ((step->max_new * group + rows - 1) / rows);
    if (units * step->n_seq > 0x7fffffff / groups)
        return fail(QH_EINVAL, "tree_attn: %d sequences of up to %lld positions are too many for one call", step->n_seq, (long long)cap);
    if (!ctx) return fail(QH_EINVAL, "tree_attn: null context");
    a.q = (const __bf16*)q, a.gate = (const __bf16*)gate, a.out = (__bf16*)out;
    a.t = TreeArrays{step->start, step->len, (int64_t)step->table_ld, a.kv.page_shift, (int)step->n, step->n_seq, step->max_new,
                     group};
    a.table = step->table;
    a.mask = step->mask;
    a.scale = scale * 1.4426950408889634f;
    const int64_t most = (int64_t)ctx_cus(ctx) * (rt == 1 ? 2 : 1);
    const int grid = (int)std::min(most, units * step->n_seq * groups);
    void* const scratch = ctx_partials(ctx);
    const size_t part = (size_t)2 * grid * rows * kv->head_dim * 4, ml = (size_t)2 * grid * rows * 8;
    if (part + ml + (TREE_MAX_SEQS + 1) * 4 > PF_SK_PART_BYTES) return fail(QH_EINVAL, "tree_attn: scratch");
    a.part = (float*)scratch;
    a.ml = (f2*)((uint8_t*)scratch + part);
    a.plan = (int32_t*)((uint8_t*)scratch + part + ml);
    const bool join = groups > 1 && grid > 1;
    auto go = [&](auto d) {
        if (kv->fmt == QH_KV_I8) launch_rows<decltype(d)::value, QH_KV_I8>((hipStream_t)stream, a, rt, grid, join);
        else launch_rows<decltype(d)::value, QH_KV_E4M3>((hipStream_t)stream, a, rt, grid, join);
    };
    if (kv->head_dim == 64) go(std::integral_constant<int, 64>{});
    else if (kv->head_dim == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "tree_attn launch: %s", hipGetErrorString(e));
    return QH_OK;
}
