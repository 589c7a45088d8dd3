// The KV cache's own operators (qh_kv_write, qh_kv_read, qh_kv_move) and the consumer of the attention in-projection that
// fills it (qh_attn_prep). All are bound by the bytes they move.
//
// A vector's scale is max|v| / 127 (int8) or / 448 (e4m3); a code is v / scale rounded once: the quotient is first rounded
// to odd in 24 bits, so that rounding it again to a code's few bits gives the nearest code to the true quotient (a quotient
// rounded to nearest may land on the border between two codes and go the wrong way).
#include <hip/hip_runtime.h>

#include <math.h>

#include <type_traits>

#include "internal.h"
#include "kv.h"

using namespace qh;

namespace {

constexpr int WAVES = 4;

__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

__device__ __forceinline__ float quotient_to_odd(float x, float s) {
    const float y = x / s, r = fmaf(-y, s, x);
    uint32_t u = __float_as_uint(y);
    if (r != 0.0f && y != 0.0f && !(u & 1)) u += (r < 0.0f) == (y < 0.0f) ? 1 : -1;
    return __uint_as_float(u);
}

// The codes of a wave's vector (V values a lane) and its scale; not finite: scale NaN, codes of zero.
template <int FMT, int V>
__device__ __forceinline__ float quantise(const float (&x)[V], uint8_t (&code)[V]) {
    float top = 0.0f, odd = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) top = fmaxf(top, fabsf(x[i])), odd += x[i] * 0.0f;
    top = wave_max(top);
    odd = wave_sum(odd);
    constexpr float most = FMT == QH_KV_I8 ? 127.0f : 448.0f;
    float s = top / most;
    if (!(odd == 0.0f)) s = NAN;
#pragma unroll
    for (int i = 0; i < V; i++) {
        float y = s > 0.0f ? quotient_to_odd(x[i], s) : 0.0f;
        y = fminf(fmaxf(y, -most), most);
        if constexpr (FMT == QH_KV_I8) code[i] = (uint8_t)((int)rintf(y) + 128);
        else code[i] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
    }
    return s;
}

template <int FMT>
__device__ __forceinline__ float code_value(uint32_t code) {
    if constexpr (FMT == QH_KV_I8) return (float)((int)code - 128);
    else return __builtin_amdgcn_cvt_f32_fp8(code, 0);
}

// A wave's vector (lane l holds dimensions V l ..) into one slot as a key (which = 0) or value (1).
template <int D, int FMT, int V>
__device__ __forceinline__ void store(const Kv& kv, int64_t slot, int head, int which, const float (&x)[V], int lane) {
    if (slot < 0 || slot >= kv.slots) return;
    uint8_t code[V];
    const float s = quantise<FMT>(x, code);
    const int64_t page = slot >> kv.page_shift;
    const uint32_t t = (uint32_t)slot & ((1u << kv.page_shift) - 1), d = lane * V;
    uint8_t* const to = kv.codes + kv_block<D>(kv, page, head, which);
    if (which == 0) {
        typedef uint8_t bytes __attribute__((ext_vector_type(V)));
        bytes c;
#pragma unroll
        for (int i = 0; i < V; i++) c[i] = code[i];
        *(bytes*)(to + k_byte<D>(t, d)) = c;
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) to[v_byte<D>(t, d + i)] = code[i];
    }
    if (lane == 0) kv.scales[kv_scale(kv, page, head, which) + t] = s;
}

template <int V>
struct Vec {
    typedef float f __attribute__((ext_vector_type(V)));
    typedef __bf16 b __attribute__((ext_vector_type(V)));
};
template <>
struct Vec<1> {
    typedef float f __attribute__((ext_vector_type(1)));
    typedef __bf16 b __attribute__((ext_vector_type(1)));
};

// a wave for each (token, kv head, keys or values)
template <int D, int FMT>
__global__ __launch_bounds__(64 * WAVES) void kv_write_kernel(Kv kv, const __bf16* __restrict__ k, const __bf16* __restrict__ v,
                                                              const int32_t* __restrict__ slots, int64_t vectors) {
    constexpr int V = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (i >= vectors) return;
    const int which = (int)(i & 1);
    const int64_t th = i >> 1, t = th / kv.heads;
    const auto in = *(const typename Vec<V>::b*)((which ? v : k) + th * D + lane * V);
    float x[V];
#pragma unroll
    for (int j = 0; j < V; j++) x[j] = (float)in[j];
    store<D, FMT, V>(kv, slots[t], (int)(th - t * kv.heads), which, x, lane);
}

template <int D, int FMT>
__global__ __launch_bounds__(64 * WAVES) void kv_read_kernel(Kv kv, const int32_t* __restrict__ slots, int64_t vectors,
                                                             __bf16* __restrict__ k, __bf16* __restrict__ v) {
    constexpr int V = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (i >= vectors) return;
    const int which = (int)(i & 1);
    const int64_t th = i >> 1, tok = th / kv.heads;
    const int head = (int)(th - tok * kv.heads);
    const int64_t slot = slots[tok];
    typename Vec<V>::b y;
#pragma unroll
    for (int j = 0; j < V; j++) y[j] = (__bf16)0.0f;
    if (slot >= 0 && slot < kv.slots) {
        const int64_t page = slot >> kv.page_shift;
        const uint32_t t = (uint32_t)slot & ((1u << kv.page_shift) - 1), d = lane * V;
        const uint8_t* const from = kv.codes + kv_block<D>(kv, page, head, which);
        const float s = kv.scales[kv_scale(kv, page, head, which) + t];
#pragma unroll
        for (int j = 0; j < V; j++) y[j] = (__bf16)(code_value<FMT>(from[which ? v_byte<D>(t, d + j) : k_byte<D>(t, d + j)]) * s);
    }
    *(typename Vec<V>::b*)((which ? v : k) + th * D + lane * V) = y;
}

// a workgroup for each (sequence, kv head, keys or values): 64 moves at a time read into LDS, then written
template <int D>
__global__ __launch_bounds__(256) void kv_move_kernel(Kv kv, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int n,
                                                      const int32_t* __restrict__ start) {
    __shared__ uint8_t held[64][D];
    __shared__ float scale[64];
    __shared__ int32_t from[64], to[64];
    const int which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const int i0 = min(max(start[blockIdx.x], 0), n), i1 = min(max(start[blockIdx.x + 1], i0), n);
    const uint32_t in_page = (1u << kv.page_shift) - 1;
    for (int i = i0; i < i1; i += 64) {
        const int m = min(64, i1 - i);
        if ((int)threadIdx.x < m) {
            int a = src[i + threadIdx.x], b = dst[i + threadIdx.x];
            if (a < 0 || a >= kv.slots || b < 0 || b >= kv.slots || a == b) a = -1;  // nothing to move
            from[threadIdx.x] = a, to[threadIdx.x] = b;
            if (a >= 0) scale[threadIdx.x] = kv.scales[kv_scale(kv, a >> kv.page_shift, head, which) + (a & in_page)];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < m * D; e += 256) {
            const int u = e / D, d = e % D, a = from[u];
            if (a >= 0)
                held[u][d] = kv.codes[kv_block<D>(kv, a >> kv.page_shift, head, which) +
                                      (which ? v_byte<D>(a & in_page, d) : k_byte<D>(a & in_page, d))];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < m * D; e += 256) {
            const int u = e / D, d = e % D, b = to[u];
            if (from[u] >= 0)
                kv.codes[kv_block<D>(kv, b >> kv.page_shift, head, which) +
                         (which ? v_byte<D>(b & in_page, d) : k_byte<D>(b & in_page, d))] = held[u][d];
        }
        if ((int)threadIdx.x < m && from[threadIdx.x] >= 0) {
            const int b = to[threadIdx.x];
            kv.scales[kv_scale(kv, b >> kv.page_shift, head, which) + (b & in_page)] = scale[threadIdx.x];
        }
        __syncthreads();
    }
}

struct Prep {
    const float* x;
    int splits;
    int64_t n;
    int q_heads, kv_heads, rot, gated;
    const float *q_w, *k_w, *inv_freq;
    float eps;
    const int32_t* pos;
    __bf16 *q, *gate, *k, *v;
    Kv kv;
    const int32_t* slots;
};

// One head of one token's partials, summed in their order: V values a lane, up to eight partials in flight.
template <int V>
__device__ __forceinline__ void head_sum(const float* __restrict__ x, int splits, int64_t stride, int lane, float (&y)[V]) {
    typedef typename Vec<V>::f vec;
    vec sum = *(const vec*)(x + lane * V);
    for (int s0 = 1; s0 < splits; s0 += 8) {
        vec p[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (s0 + j < splits) p[j] = *(const vec*)(x + (s0 + j) * stride + lane * V);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (s0 + j < splits) sum += p[j];
    }
#pragma unroll
    for (int i = 0; i < V; i++) y[i] = sum[i];
}

template <int V>
__device__ __forceinline__ void put(__bf16* to, const float (&y)[V], int lane) {
    typename Vec<V>::b o;
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = (__bf16)y[i];
    *(typename Vec<V>::b*)(to + lane * V) = o;
}

// A workgroup takes some heads (blockIdx.y's share) of one token, a wave a head at a time: queries (with their gates),
// keys, values. The angles' sines and cosines are made once per workgroup: pos * inv_freq in turns in f64, whose fraction
// is exact to f32 at any position.
template <int D, int FMT>
__global__ __launch_bounds__(64 * WAVES) void attn_prep_kernel(const Prep a) {
    constexpr int V = D / 64;
    __shared__ float cs[D / 2], sn[D / 2];
    __shared__ float rows[WAVES][D];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = a.rot / 2;
    const int64_t t = blockIdx.x;
    if ((int)threadIdx.x < half) {
        const double turns = (double)a.pos[t] * (double)a.inv_freq[threadIdx.x] * 0.15915494309189535;
        const float part = (float)(turns - rint(turns));
        sincospif(2.0f * part, &sn[threadIdx.x], &cs[threadIdx.x]);
    }
    __syncthreads();
    const int per = a.gated ? 2 : 1, heads = a.q_heads + 2 * a.kv_heads;
    const int64_t ld = (int64_t)(a.q_heads * per + 2 * a.kv_heads) * D, stride = a.n * ld;
    const int share = (heads + gridDim.y - 1) / gridDim.y, h1 = min(heads, (int)(blockIdx.y + 1) * share);
    for (int h = blockIdx.y * share + wave; h < h1; h += WAVES) {
        const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
        const int col = is_q ? h * per : h - a.q_heads + a.q_heads * per;
        const float* const x = a.x + t * ld + (int64_t)col * D;
        float y[V];
        head_sum<V>(x, a.splits, stride, lane, y);
        const float* const w = is_q ? a.q_w : is_k ? a.k_w : nullptr;
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) ss += y[i] * y[i];
            const float r = 1.0f / sqrtf(wave_sum(ss) / (float)D + a.eps);
#pragma unroll
            for (int i = 0; i < V; i++) y[i] = w[lane * V + i] * (y[i] * r);
        }
        if (half && (is_q || is_k)) {
#pragma unroll
            for (int i = 0; i < V; i++) rows[wave][lane * V + i] = y[i];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int d = lane * V + i;
                if (d < half) y[i] = y[i] * cs[d] - rows[wave][d + half] * sn[d];
                else if (d < a.rot) y[i] = y[i] * cs[d - half] + rows[wave][d - half] * sn[d - half];
            }
            __builtin_amdgcn_wave_barrier();
        }
        if (is_q) {
            put<V>(a.q + (t * a.q_heads + h) * D, y, lane);
            if (a.gated) {
                head_sum<V>(x + D, a.splits, stride, lane, y);
                put<V>(a.gate + (t * a.q_heads + h) * D, y, lane);
            }
            continue;
        }
        const int head = h - a.q_heads - (is_k ? 0 : a.kv_heads);
        if constexpr (FMT == 0) put<V>((is_k ? a.k : a.v) + (t * a.kv_heads + head) * D, y, lane);
        else store<D, FMT, V>(a.kv, a.slots[t], head, is_k ? 0 : 1, y, lane);
    }
}

template <class F>
void by_dim(int d, F&& f) {
    if (d == 64) f(std::integral_constant<int, 64>{});
    else if (d == 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
}

int launched(const char* who) {
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "%s launch: %s", who, hipGetErrorString(e));
    return QH_OK;
}

constexpr size_t MAX_TOKENS = (size_t)1 << 20;  // of one call

}  // namespace

extern "C" int qh_kv_sizes(const qh_kv* kv, size_t* code_bytes, size_t* scale_bytes) {
    if (!kv || !code_bytes || !scale_bytes) return fail(QH_EINVAL, "kv_sizes: null");
    qh_kv shape = *kv;
    shape.codes = shape.scales = (float*)16;  // (any: the shape alone is checked)
    Kv c;
    if (int e = kv_check("kv_sizes", &shape, &c)) return e;
    *code_bytes = (size_t)c.slots * kv->heads * 2 * kv->head_dim;
    *scale_bytes = (size_t)c.slots * kv->heads * 2 * sizeof(float);
    return QH_OK;
}

extern "C" int qh_kv_write(void* stream, const qh_kv* kv, const void* k_bf16, const void* v_bf16, const int32_t* slots, size_t n) {
    Kv c;
    if (int e = kv_check("kv_write", kv, &c)) return e;
    if (n == 0) return QH_OK;
    if (!k_bf16 || !v_bf16 || !slots) return fail(QH_EINVAL, "kv_write: null");
    if (n > MAX_TOKENS || (uintptr_t)k_bf16 % 16 || (uintptr_t)v_bf16 % 16)
        return fail(QH_EINVAL, "kv_write: %zu tokens (up to 2^20), buffers 16-byte aligned", n);
    const int64_t vectors = (int64_t)n * c.heads * 2;
    const dim3 grid((unsigned)((vectors + WAVES - 1) / WAVES));
    by_dim(kv->head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto* f = kv->fmt == QH_KV_I8 ? kv_write_kernel<D, QH_KV_I8> : kv_write_kernel<D, QH_KV_E4M3>;
        hipLaunchKernelGGL(f, grid, dim3(64 * WAVES), 0, (hipStream_t)stream, c, (const __bf16*)k_bf16, (const __bf16*)v_bf16,
                           slots, vectors);
    });
    return launched("kv_write");
}

extern "C" int qh_kv_read(void* stream, const qh_kv* kv, const int32_t* slots, size_t n, void* k_bf16, void* v_bf16) {
    Kv c;
    if (int e = kv_check("kv_read", kv, &c)) return e;
    if (n == 0) return QH_OK;
    if (!k_bf16 || !v_bf16 || !slots) return fail(QH_EINVAL, "kv_read: null");
    if (n > MAX_TOKENS || (uintptr_t)k_bf16 % 16 || (uintptr_t)v_bf16 % 16)
        return fail(QH_EINVAL, "kv_read: %zu tokens (up to 2^20), buffers 16-byte aligned", n);
    const int64_t vectors = (int64_t)n * c.heads * 2;
    const dim3 grid((unsigned)((vectors + WAVES - 1) / WAVES));
    by_dim(kv->head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto* f = kv->fmt == QH_KV_I8 ? kv_read_kernel<D, QH_KV_I8> : kv_read_kernel<D, QH_KV_E4M3>;
        hipLaunchKernelGGL(f, grid, dim3(64 * WAVES), 0, (hipStream_t)stream, c, slots, vectors, (__bf16*)k_bf16, (__bf16*)v_bf16);
    });
    return launched("kv_read");
}

extern "C" int qh_kv_move(void* stream, const qh_kv* kv, const int32_t* src, const int32_t* dst, size_t n, const int32_t* start,
                          int n_seq) {
    Kv c;
    if (int e = kv_check("kv_move", kv, &c)) return e;
    if (n_seq < 0 || n_seq > 65535 || n > MAX_TOKENS)
        return fail(QH_EINVAL, "kv_move: %zu moves (up to 2^20) of %d sequences (up to 65535)", n, n_seq);
    if (n == 0 || n_seq == 0) return QH_OK;
    if (!src || !dst || !start) return fail(QH_EINVAL, "kv_move: null");
    by_dim(kv->head_dim, [&](auto d) {
        hipLaunchKernelGGL((kv_move_kernel<decltype(d)::value>), dim3(n_seq, c.heads * 2), dim3(256), 0, (hipStream_t)stream, c, src,
                           dst, (int)n, start);
    });
    return launched("kv_move");
}

extern "C" int qh_attn_prep(void* stream, const float* x, int splits, size_t n, const qh_attn_rows* rows, const float* q_w,
                            const float* k_w, float eps, const float* inv_freq, const int32_t* pos, void* q, void* gate,
                            const qh_kv* kv, const int32_t* slots, void* k, void* v) {
    if (!rows) return fail(QH_EINVAL, "attn_prep: null");
    const int D = rows->head_dim;
    if (D != 64 && D != 128 && D != 256) return fail(QH_EINVAL, "attn_prep: heads of %d dimensions (64, 128 or 256)", D);
    if (rows->q_heads < 1 || rows->kv_heads < 1 || rows->q_heads > 4096 || rows->kv_heads > 1024)
        return fail(QH_EINVAL, "attn_prep: %d query heads, %d kv heads", rows->q_heads, rows->kv_heads);
    if (rows->rot < 0 || rows->rot > D || rows->rot % 2)
        return fail(QH_EINVAL, "attn_prep: %d rotated dimensions of %d (an even number)", rows->rot, D);
    if (splits < 1) return fail(QH_EINVAL, "attn_prep: %d splits", splits);
    Prep a = {};
    if (kv) {
        if (int e = kv_check("attn_prep", kv, &a.kv)) return e;
        if (kv->heads != rows->kv_heads || kv->head_dim != D)
            return fail(QH_EINVAL, "attn_prep: a cache of %d heads of %d for %d heads of %d", kv->heads, kv->head_dim, rows->kv_heads, D);
    }
    if (n == 0) return QH_OK;
    if (!x || !q || (kv ? !slots : !k || !v) || (rows->gated && !gate) || (rows->rot && (!inv_freq || !pos)))
        return fail(QH_EINVAL, "attn_prep: null");
    if (n > MAX_TOKENS || (uintptr_t)x % 16 || (uintptr_t)q % 16 || (uintptr_t)gate % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16)
        return fail(QH_EINVAL, "attn_prep: %zu tokens (up to 2^20), buffers 16-byte aligned", n);
    a.x = x, a.splits = splits, a.n = (int64_t)n, a.q_heads = rows->q_heads, a.kv_heads = rows->kv_heads, a.rot = rows->rot;
    a.gated = rows->gated != 0, a.q_w = q_w, a.k_w = k_w, a.inv_freq = inv_freq, a.eps = eps, a.pos = pos, a.slots = slots;
    a.q = (__bf16*)q, a.gate = (__bf16*)gate, a.k = (__bf16*)k, a.v = (__bf16*)v;
    const int heads = rows->q_heads + 2 * rows->kv_heads;
    const unsigned shares = n >= 512 ? 1 : (heads + WAVES - 1) / WAVES;
    by_dim(D, [&](auto d) {
        constexpr int DD = decltype(d)::value;
        auto* f = !kv ? attn_prep_kernel<DD, 0> : kv->fmt == QH_KV_I8 ? attn_prep_kernel<DD, QH_KV_I8> : attn_prep_kernel<DD, QH_KV_E4M3>;
        hipLaunchKernelGGL(f, dim3((unsigned)n, shares), dim3(64 * WAVES), 0, (hipStream_t)stream, a);
    });
    return launched("attn_prep");
}
