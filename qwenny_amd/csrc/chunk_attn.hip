// Attention of a prompt's chunk (and of batches of chunks) over the paged, quantised KV cache (qh_chunk_attn).
//
// For each row (a token and one of its query heads) over the positions t up to its token's own:
//   s_t = c q.k_t,  o = sum_t exp(s_t) v_t / sum_t exp(s_t),  then o * sigmoid(gate) where a gate is given,
// with k_t = sk_t * (codes), v_t = sv_t * (codes). One pass over the cache for each 256 rows of a kv head: the running maximum
// and sum of the softmax beside the unnormalised o, rescaled when the maximum grows.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

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

constexpr int WAVES = 8, THREADS = 64 * WAVES, ROWS = 32 * WAVES;

struct Args {
    const __bf16* q;     // [n][heads][D]
    const __bf16* gate;  // the same, or null
    __bf16* out;
    Kv kv;
    TreeArrays t;
    const int32_t* table;  // [n_seq][table_ld]
    float scale;           // softmax scale * log2(e)
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

// The least e >= NO_EXP for which a scale is below 2^e (to 2^126; such powers of two have exact reciprocals).
constexpr int NO_EXP = -126;
__device__ __forceinline__ int scale_exp(float s) { return s > 0.0f ? max(min(__builtin_amdgcn_frexp_expf(s), 126), NO_EXP) : NO_EXP; }

// The sequences' places: first unit (of 256 rows of a kv head), first token and tokens.
struct Plan {
    int32_t base[TREE_MAX_SEQS], first[TREE_MAX_SEQS], news[TREE_MAX_SEQS];
    int32_t sums[2][WAVES];
};
constexpr int REST_DISORDER = 1, REST_SOME = 2;  // starts are not in order; some tokens are in no sequence that has work

// Fills the plan and returns the units in all. Starts that are not in order are found on the way; the plan is then made anew, each
// sequence against all starts before it.
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
__device__ __forceinline__ int find_seq(const int32_t* begin, int n_seq, int at) {
    int lo = -1, hi = n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (begin[mid] <= at ? lo : hi) = mid;
    }
    return __builtin_amdgcn_readfirstlane(lo);
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
struct Shared {
    h8 k[D / 8][KV_TILE];
    h8 v[4][2][D];
    float scale[2][KV_TILE];
    Plan plan;
};

template <int D, int FMT>
__global__ __launch_bounds__(THREADS, 2) void chunk_attn_kernel(const Args a) {
    __shared__ Shared<D> sh;
    int rest;
    const int units = make_plan(a, sh.plan, &rest);
    if (rest) put_rest<D>(a, sh.plan, rest);
    if ((int)blockIdx.x >= units) return;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
    const int b = find_seq(sh.plan.base, a.t.n_seq, blockIdx.x);
    const int first = __builtin_amdgcn_readfirstlane(sh.plan.first[b]), news = __builtin_amdgcn_readfirstlane(sh.plan.news[b]);
    const int old = a.t.len[b], group = a.t.group, rows = news * group, chunks = (rows + ROWS - 1) / ROWS;
    // the longest first
    const int past = blockIdx.x - __builtin_amdgcn_readfirstlane(sh.plan.base[b]);
    const int head = past % a.kv.heads, row0 = (chunks - 1 - past / a.kv.heads) * ROWS;
    const int last = min(row0 + ROWS, rows) - 1;  // the last row of the workgroup
    const int all_see = old + row0 / group + 1;   // positions that all its rows see
    const int t_end = (old + last / group + 1 + KV_TILE - 1) / KV_TILE;

    const int row = min(row0 + wave * 32 + col, last), node = row / group;
    const int sees = old + node + 1;
    const size_t at = ((size_t)(first + node) * a.kv.heads * group + head * group + (row - node * group)) * D;

    // the lane's queries: dimensions 16 i + 8 half .. + 7, scaled by a power of two into f16's range (the factor goes to the scores)
    h8 q[D / 16];
    float factor;
    {
        b8 raw[D / 16];
        uint32_t top = 0;  // bf16 with the sign taken off compares as a whole number; from 0x7f80 on it is not finite
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            raw[i] = *(const b8*)(a.q + at + i * 16 + half * 8);
            const u4 bits = __builtin_bit_cast(u4, raw[i]);
#pragma unroll
            for (int k = 0; k < 4; k++) top = max(top, max(bits[k] & 0x7fffu, bits[k] >> 16 & 0x7fffu));
        }
        const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
        top = max(both[0], both[1]);
        const int e = top < 0x7f80 ? __builtin_amdgcn_frexp_expf(__uint_as_float(top << 16)) - 15 : 0;
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) q[i][k] = (_Float16)__builtin_ldexpf((float)raw[i][k], -e);
        factor = top >= 0x7f80 ? NAN : fminf(fmaxf(__builtin_ldexpf(a.scale, e), 1e-37f), 3e38f);
    }

    f16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
        for (int k = 0; k < 16; k++) o[i][k] = 0.0f;
    float top = -INFINITY, sum = 0.0f;
    int exp = NO_EXP;  // values' scales are taken relative to 2^exp, the largest that the row sees: probabilities fit f16
    const int page_tiles = 1 << (a.kv.page_shift - 6);

    for (int t = 0; t < t_end; t++) {
        const int page = a.table[(size_t)b * a.t.table_ld + (t >> (a.kv.page_shift - 6))];
        const bool none = page < 0 || ((int64_t)page << a.kv.page_shift) >= a.kv.slots;
        const size_t place = none ? 0 : ((size_t)page * a.kv.heads + head) * 2 * page_tiles + (t & (page_tiles - 1));
        const int there = none ? 0 : min(old + news - t * KV_TILE, KV_TILE);  // tokens of the tile that were written
        __syncthreads();
        for (int p = tid; p < KV_TILE * D / 16; p += THREADS) {
            const int u = p >> 6, l = p & 63, c = l >> 4;
            const uint8_t* const codes = a.kv.codes + place * (KV_TILE * D) + u * 1024 + (l & 15) * 64;
            const u4 k = *(const u4*)(codes + c * 16);
            const int token = u / (D / 64) * 16 + (l & 15), chunk = u % (D / 64) * 8 + c * 2;
            const h4 k0 = operands<FMT>(k.x), k1 = operands<FMT>(k.y), k2 = operands<FMT>(k.z), k3 = operands<FMT>(k.w);
            sh.k[chunk][token] = __builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7);
            sh.k[chunk + 1][token] = __builtin_shufflevector(k2, k3, 0, 1, 2, 3, 4, 5, 6, 7);
            const int g = (c & 1) * 2 + (c >> 1);
            u4 v = *(const u4*)(codes + (size_t)page_tiles * (KV_TILE * D) + g * 16);
            if (FMT == QH_KV_E4M3 && there < KV_TILE) {  // what was not written may be NaN codes, which no probability takes away
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const int keep = max(there - (s * 16 + g * 4), 0);
                    v[s] = keep < 4 ? v[s] & ((1u << 8 * keep) - 1) : v[s];
                }
            }
#pragma unroll
            for (int s = 0; s < 4; s++) ((h4*)&sh.v[s][g & 1][u * 16 + (l & 15)])[g >> 1] = operands<FMT>(v[s]);
        }
        if (tid < 2 * KV_TILE) {
            const int which = tid >> 6;
            sh.scale[which][lane] = none ? NAN : a.kv.scales[(place + which * page_tiles) * KV_TILE + lane];
        }
        __syncthreads();
        const bool whole = (t + 1) * KV_TILE <= all_see;
#pragma unroll 1
        for (int tb = 0; tb < 2; tb++) {
            // s^T = k q^T: the lane gets its row's scores of tokens 8 (i / 4) + 4 half + i % 4
            f16 x;
#pragma unroll
            for (int k = 0; k < 16; k++) x[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(sh.k[2 * i + half][tb * 32 + col], q[i], x, 0, 0, 0);
            const int t0 = t * KV_TILE + tb * 32 + half * 4;
            float mx = -INFINITY, largest = 0.0f;
            f4 vs[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f4 ks = *(const f4*)&sh.scale[0][tb * 32 + j * 8 + half * 4];
                vs[j] = *(const f4*)&sh.scale[1][tb * 32 + j * 8 + half * 4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool seen = whole || t0 + 8 * j + i < sees;
                    const float s = seen ? x[4 * j + i] * ks[i] : -INFINITY;
                    x[4 * j + i] = s;
                    mx = fmaxf(mx, s);
                    largest = fmaxf(largest, seen && vs[j][i] < INFINITY ? vs[j][i] : 0.0f);
                }
            }
            mx = both_max(mx), largest = both_max(largest);
            const int exp_was = exp;
            exp = max(exp, scale_exp(largest));
            float by = __builtin_ldexpf(1.0f, exp_was - exp);
            const float next = fmaxf(top, mx);
            // the maximum is followed only where it has grown by more than 2^8 (the sums and f16 hold that)
            if (__any((next - top) * factor > 8.0f)) {
                const float al = next > top ? __builtin_amdgcn_exp2f((top - next) * factor) : 1.0f;
                sum *= al;
                top = next;
                by *= al;
            }
            if (__any(by != 1.0f)) {
#pragma unroll
                for (int i = 0; i < D / 32; i++) o[i] *= by;
            }
            const float off = top == -INFINITY ? 0.0f : top, inv = __builtin_ldexpf(1.0f, -exp);
            h8 p[2];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float pv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float s = x[4 * j + i], pr = __builtin_amdgcn_exp2f((s - off) * factor);
                    pv[i] = s == -INFINITY ? 0.0f : pr * (vs[j][i] * inv);
                    sum += pr;
                }
                const h2 p0 = __builtin_convertvector((f2{pv[0], pv[1]}), h2), p1 = __builtin_convertvector((f2{pv[2], pv[3]}), h2);
                const int k = (j & 1) * 4;
                p[j >> 1][k] = p0.x, p[j >> 1][k + 1] = p0.y, p[j >> 1][k + 2] = p1.x, p[j >> 1][k + 3] = p1.y;
            }
            // o^T += v^T p^T: the lane has its row's dimensions 32 i + 8 (k / 4) + 4 half + k % 4
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < D / 32; i++)
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(sh.v[tb * 2 + s][half][i * 32 + col], p[s], o[i], 0, 0, 0);
        }
    }

    if (row0 + wave * 32 + col > last) return;
    sum = both_sum(sum);
    const float total = __builtin_ldexpf(__builtin_amdgcn_rcpf(sum), exp);
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const size_t d = at + i * 32 + j * 8 + half * 4;
            f4 v = f4{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]} * total;
            if (a.gate) {
                const b4 g = *(const b4*)(a.gate + d);
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] *= sigmoid((float)g[k]);
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
    const int group = q_heads / kv->heads;
    const uint64_t units = ((uint64_t)step->n * group / ROWS + step->n_seq) * kv->heads;  // as many as there can be
    if (units > 0x7fffffffu) return fail(QH_EINVAL, "chunk_attn: %zu tokens of %d heads are too many for one call", step->n, q_heads);
    if (!ctx) return fail(QH_EINVAL, "chunk_attn: null context");
    a.q = (const __bf16*)q, a.gate = (const __bf16*)gate, a.out = (__bf16*)out;
    a.t = TreeArrays{step->start, step->len, (int64_t)step->table_ld, a.kv.page_shift, (int)step->n, step->n_seq, step->max_new,
                     group};
    a.table = step->table;
    a.scale = scale * 1.4426950408889634f;
    auto go = [&](auto d, auto fmt) {
        constexpr int D = decltype(d)::value;
        launch_kernel(chunk_attn_kernel<D, decltype(fmt)::value>, dim3((unsigned)units), dim3(THREADS), (hipStream_t)stream, a);
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
