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

// buffer resource word 3 (32-bit data format, no swizzle), and the cache policy of loads past the caches
constexpr int BUF_RSRC_WORD3 = 0x00020000;
constexpr int CPOL_NT = 2;

constexpr int BATCH = 64, BATCH_WAVES = 16;  // tokens of a workgroup that turns values over in LDS, and its waves

// A barrier for what the workgroup's waves wrote to LDS; loads and stores to memory stay in flight over it.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// f over the wave's 64 lanes, or over 16 neighbouring ones: within rows of 16 by DPP, then over the rows
template <int LANES = 64, class F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, F&& f) {
    auto step = [&](auto ctrl) { v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(ctrl)::value, 15, 15, false)); };
    step(std::integral_constant<int, 0xb1>{});   // quad_perm 1 0 3 2
    step(std::integral_constant<int, 0x4e>{});   // quad_perm 2 3 0 1
    step(std::integral_constant<int, 0x141>{});  // row_half_mirror
    step(std::integral_constant<int, 0x140>{});  // row_mirror
    if constexpr (LANES == 16) return v;
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(a[0], a[1]);
    a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(a[0], a[1]);
}
__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float(
        over_lanes(__float_as_uint(v), [](uint32_t x, uint32_t y) { return __float_as_uint(__uint_as_float(x) + __uint_as_float(y)); }));
}

// x / s rounded to odd: of the two neighbours of the quotient the one with its last bit set, unless it is exact. `r`: 1 / s to
// a unit in the last place; the quotient made with it is one of the neighbours.
__device__ __forceinline__ float quotient_to_odd(float x, float s, float r) {
    float y = x * r;
    y = fmaf(fmaf(-y, s, x), r, y);
    const float left = fmaf(-y, s, x);
    const uint32_t u = __float_as_uint(y);
    const int back = (int)(u ^ __float_as_uint(left)) >> 31;  // -1: the quotient's magnitude is below y's
    return left == 0.0f ? y : __uint_as_float((u + back) | 1);
}

// x / s rounded to the nearest whole number, ties to even: the last byte of the result's bits is the number + 128. The first
// whole number is off by one at most; what is left of x beside it is exact where it is near half of s, and says whether to
// take the next one.
__device__ __forceinline__ float whole_quotient(float x, float s, float r) {
    constexpr float up = 0x1.8p23f + 128.0f;  // whole numbers from here on
    const float y = fmaf(x, r, up), left = fmaf(up - y, s, x);
    const uint32_t half = __float_as_uint(0.5f * s) - (__float_as_uint(y) & 1);  // an odd number gives way at half a step, too
    return y + (fabsf(left) > __uint_as_float(half) ? copysignf(1.0f, left) : 0.0f);
}

// The codes of a vector, V values a lane of LANES, and its scale; not finite: scale NaN, codes of zero.
template <int FMT, int LANES, int V>
__device__ __forceinline__ void quantise(const float (&x)[V], uint8_t (&code)[V], float& s) {
    constexpr float most = FMT == QH_KV_I8 ? 127.0f : 448.0f;
    uint32_t bits = 0;  // magnitudes compare as whole numbers; from 0x7f800000 on they are not finite
#pragma unroll
    for (int i = 0; i < V; i++) bits = max(bits, __float_as_uint(x[i]) & 0x7fffffffu);
    bits = over_lanes<LANES>(bits, [](uint32_t x, uint32_t y) { return max(x, y); });
    s = bits >= 0x7f800000u ? NAN : __uint_as_float(bits) / most;
    const float r = __builtin_amdgcn_rcpf(s);
    if (__all(s >= 0x1p-100f)) {  // (not NaN; its reciprocal, its half and what is left of a value are normal numbers)
        float y[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            y[i] = FMT == QH_KV_I8 ? whole_quotient(x[i], s, r) : quotient_to_odd(x[i], s, r);
            if (FMT == QH_KV_I8) code[i] = (uint8_t)__float_as_uint(y[i]);
        }
#pragma unroll
        for (int i = 0; FMT == QH_KV_E4M3 && i < V; i += 2) {
            const int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[i], y[i + 1 < V ? i + 1 : i], 0, false);
            code[i] = (uint8_t)c;
            if (i + 1 < V) code[i + 1] = (uint8_t)(c >> 8);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        float y = !(s > 0.0f) ? 0.0f : s >= 0x1p-126f ? quotient_to_odd(x[i], s, r) : x[i] / s;
        y = fminf(fmaxf(y, -most), most);
        if constexpr (FMT == QH_KV_I8) code[i] = (uint8_t)((int)rintf(y) + 128);
        else code[i] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
    }
}

template <int FMT>
__device__ __forceinline__ float code_value(uint32_t code) {
    if constexpr (FMT == QH_KV_I8) return (float)((int)code - 128);
    else return __builtin_amdgcn_cvt_f32_fp8(code, 0);
}

// A wave's vector's codes (lane l holds dimensions V l ..) and scale into one slot as a key (which = 0) or value (1).
template <int D, int V>
__device__ __forceinline__ void store(const Kv& kv, int64_t slot, int head, int which, const uint8_t (&code)[V], float s, int lane) {
    if (slot < 0 || slot >= kv.slots) return;
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
template <int D, int FMT, int V>
__device__ __forceinline__ void quantise_into(const Kv& kv, int64_t slot, int head, int which, const float (&x)[V], int lane) {
    uint8_t code[V];
    float s;
    quantise<FMT, 64>(x, code, s);
    store<D, V>(kv, slot, head, which, code, s, lane);
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

// Partials s0 .. of one head of one token added to `sum` in their order: V values a lane, up to eight partials in flight.
template <int V>
__device__ __forceinline__ void add_partials(const float* __restrict__ x, int s0, int splits, int64_t stride, int lane,
                                             typename Vec<V>::f& sum) {
    typedef typename Vec<V>::f vec;
    for (; s0 < splits; s0 += 8) {
        vec p[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (s0 + j < splits) p[j] = __builtin_nontemporal_load((const vec*)(x + (s0 + j) * stride + lane * V));
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (s0 + j < splits) sum += p[j];
    }
}
template <int V>
__device__ __forceinline__ void head_sum(const float* __restrict__ x, int splits, int64_t stride, int lane, float (&y)[V]) {
    typename Vec<V>::f sum = __builtin_nontemporal_load((const typename Vec<V>::f*)(x + lane * V));
    add_partials<V>(x, 1, splits, stride, lane, sum);
#pragma unroll
    for (int i = 0; i < V; i++) y[i] = sum[i];
}

// The same in two halves, so that the first P partials are in flight over other work: buffer loads, which read nothing where
// there is none (a branch around a load would have its wait cover all loads).
template <int V, int P>
struct Ahead {
    typename Vec<V>::f p[P];
    const float* x;
    __device__ __forceinline__ void read(const float* from, int splits, int64_t stride, int lane) {
        x = from;
#pragma unroll
        for (int j = 0; j < P; j++) {
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(from + j * stride), 0, j < splits ? 64 * V * 4 : 0, BUF_RSRC_WORD3);
            if constexpr (V == 1) p[j][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, lane * 4, 0, CPOL_NT));
            else if constexpr (V == 2) p[j] = __builtin_bit_cast(typename Vec<V>::f, __builtin_amdgcn_raw_buffer_load_b64(rsrc, lane * 8, 0, CPOL_NT));
            else p[j] = __builtin_bit_cast(typename Vec<V>::f, __builtin_amdgcn_raw_buffer_load_b128(rsrc, lane * 16, 0, CPOL_NT));
        }
    }
    __device__ __forceinline__ void sum(int splits, int64_t stride, int lane, float (&y)[V]) {
        auto v = p[0];
#pragma unroll
        for (int j = 1; j < P; j++)
            if (j < splits) v += p[j];
        add_partials<V>(x, P, splits, stride, lane, v);
#pragma unroll
        for (int i = 0; i < V; i++) y[i] = v[i];
    }
};

// A wave for each (token, kv head, keys or values), for few tokens: bound by its trips to memory, the slot's and the vector's, then
// out (9 tokens of 8 x 128: 2.4 us).
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
    quantise_into<D, FMT, V>(kv, slots[t], (int)(th - t * kv.heads), which, x, lane);
}

// The same back: a trip for the slot, one for codes and scale (9 tokens of 8 x 128: 2.5 us).
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

// Where a batch kernel's values come from: bf16, or the in-projection's partials (f32, summed in their order).
struct Source {
    const __bf16* bf16;
    const float* x;
    int splits;
    int64_t stride, ld;  // of a partial, of a token
    int col;             // of the first head's values
};

// 64 tokens of one kv head, keys (which = 0) or values, for many tokens at a time (prompts); 16 lanes have a token's vector. A
// value's codes lie 64 bytes from dimension to dimension, four tokens side by side: written vector by vector they are single
// bytes, 16.0 us for 2048 tokens of 4 x 256. Here the codes of 64 tokens are put into LDS and turned over: a thread writes four
// tokens' codes of four dimensions, 16 threads the 64 bytes of a dimension; what does not fill four
// tokens' places, at a run's ends, is written apart (by every thread that meets it, and with a wave for each vector: 9.4 us
// against 7.0).
// `which0`: 0 for keys and values, 1 for values alone.
template <int D, int FMT, bool PARTIALS>
__global__ __launch_bounds__(64 * BATCH_WAVES) void kv_write_batch_kernel(Kv kv, Source keys, Source values,
                                                                          const int32_t* __restrict__ slots, int n, int which0) {
    constexpr int V = D / 16, C = V < 8 ? V : 8, ROW = D / 4 + 1;  // C: a lane's values in a row
    __shared__ uint32_t codes[BATCH][ROW];
    __shared__ __align__(4) uint8_t from[BATCH_WAVES][BATCH];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane & 15, t0 = blockIdx.x * BATCH;
    const int which = which0 | (blockIdx.y & (1 - which0)), head = blockIdx.y >> (1 - which0);
    const Source& src = which ? values : keys;
    const int e = threadIdx.x >> 4, t = min(t0 + e, n - 1);
    const int mine = t0 + lane < n ? slots[t0 + lane] : -1;  // lane l: the l-th token's slot
    const int slot = t0 + e < n ? slots[t] : -1;
    float x[V];
#pragma unroll
    for (int c = 0; c < V / C; c++) {
        float y[C];
        if constexpr (PARTIALS) {
            head_sum<C>(src.x + t * src.ld + src.col + head * D + c * 16 * C, src.splits, src.stride, l, y);
        } else {
            const auto in = *(const typename Vec<C>::b*)(src.bf16 + ((int64_t)t * kv.heads + head) * D + (c * 16 + l) * C);
#pragma unroll
            for (int j = 0; j < C; j++) y[j] = (float)in[j];
        }
#pragma unroll
        for (int j = 0; j < C; j++) x[c * C + j] = y[j];
    }
    const bool in_cache = mine >= 0 && mine < kv.slots, slot_in_cache = slot >= 0 && slot < kv.slots;
    uint8_t code[V];
    float s;
    quantise<FMT, 16>(x, code, s);
    uint32_t words[V / 4];
#pragma unroll
    for (int w = 0; w < V / 4; w++) words[w] = code[4 * w] | code[4 * w + 1] << 8 | code[4 * w + 2] << 16 | (uint32_t)code[4 * w + 3] << 24;
    if (slot_in_cache) {
        const uint32_t in_page = (uint32_t)slot & ((1u << kv.page_shift) - 1);
        if (l == 0) kv.scales[kv_scale(kv, slot >> kv.page_shift, head, which) + in_page] = s;
        if (which == 0) {
            uint8_t* const to = kv.codes + kv_block<D>(kv, slot >> kv.page_shift, head, 0);
#pragma unroll
            for (int c = 0; c < V / C; c++) {
                typedef uint32_t bytes __attribute__((ext_vector_type(C / 4)));
                bytes b;
#pragma unroll
                for (int w = 0; w < C / 4; w++) b[w] = words[c * (C / 4) + w];
                *(bytes*)(to + k_byte<D>(in_page, (c * 16 + l) * C)) = b;
            }
        }
    }
    if (which == 0) return;
#pragma unroll
    for (int c = 0; c < V / C; c++)
#pragma unroll
        for (int w = 0; w < C / 4; w++) codes[e][(c * 16 + l) * (C / 4) + w] = words[c * (C / 4) + w];
    __syncthreads();
    // one of the cache's tiles after the other, that of the first token left
    for (uint64_t left = __ballot(in_cache); left;) {
        const int tile = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)left) - 1) >> 6;
        const bool here = in_cache && mine >> 6 == tile;
        left &= ~__ballot(here);
        from[wave][lane] = 255;
        __builtin_amdgcn_wave_barrier();
        if (here) from[wave][mine & 63] = (uint8_t)lane;
        __builtin_amdgcn_wave_barrier();
        const int slot0 = tile << 6;
        uint8_t* const to = kv.codes + kv_block<D>(kv, slot0 >> kv.page_shift, head, 1) + (size_t)(slot0 & ((1 << kv.page_shift) - 1)) * D;
        // bytes 4 l .. of a dimension: tokens 16 (l % 4) + 4 (l / 4) ..
        const uint32_t who = *(const uint32_t*)&from[wave][(l & 3) * 16 + (l >> 2) * 4];
        const bool all = !(who & 0x80808080u);
        if (all) {
            for (int dg = threadIdx.x >> 4; dg < D / 4; dg += 4 * BATCH_WAVES) {
                uint32_t c[4];
#pragma unroll
                for (int j = 0; j < 4; j++) c[j] = codes[who >> (8 * j) & 63][dg];
                // bytes turned over: o[d] = the four tokens' byte d
                const uint32_t a0 = __builtin_amdgcn_perm(c[1], c[0], 0x05010400u), a1 = __builtin_amdgcn_perm(c[1], c[0], 0x07030602u);
                const uint32_t b0 = __builtin_amdgcn_perm(c[3], c[2], 0x05010400u), b1 = __builtin_amdgcn_perm(c[3], c[2], 0x07030602u);
                uint32_t* const at = (uint32_t*)(to + dg * 256 + l * 4);
                at[0] = __builtin_amdgcn_perm(b0, a0, 0x05040100u), at[16] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
                at[32] = __builtin_amdgcn_perm(b1, a1, 0x05040100u), at[48] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
            }
        }
        // four tokens that are not all there (at the ends of a run of slots): byte by byte, a thread each
        for (uint32_t part = (uint32_t)__ballot(!all && who != ~0u) & 0xffffu; part; part &= part - 1) {
            const int q = __ffs(part) - 1;
            const uint32_t some = __builtin_amdgcn_readlane(who, q);
            for (int i = threadIdx.x; i < 4 * D; i += 64 * BATCH_WAVES) {
                const int d = i % D, j = i / D;
                const uint32_t token = some >> (8 * j) & 255;
                if (token < BATCH) to[d * 64 + q * 4 + j] = ((const uint8_t*)codes[token])[d];
            }
        }
    }
}

// The same tokens read back: a tile's values go into LDS whole, each wave then takes its tokens' bytes out of them. 2048 tokens of
// 4 x 256: 12.6 MB in 5.7 us (4.7 at best), 2.2 TB/s, one workgroup to a CU whose trips in and out do not overlap.
template <int D, int FMT>
__global__ __launch_bounds__(64 * BATCH_WAVES) void kv_read_batch_kernel(Kv kv, const int32_t* __restrict__ slots, int n,
                                                                         __bf16* __restrict__ k, __bf16* __restrict__ v) {
    constexpr int V = D / 64, EACH = BATCH / BATCH_WAVES;
    static_assert(D * 4 <= 64 * BATCH_WAVES);
    // where a dimension's 64 bytes lie in LDS, in words: the 64 lanes, V dimensions apart, reach different banks
    auto row = [](int d) { return d * 17 + (d >> 6); };
    __shared__ uint32_t tile_codes[D * 17 + V];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t0 = blockIdx.x * BATCH, which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const uint32_t in_page = (1u << kv.page_shift) - 1;
    const int mine = t0 + lane < n ? slots[t0 + lane] : -1;
    const bool in_cache = mine >= 0 && mine < kv.slots;
    const float scale = in_cache ? kv.scales[kv_scale(kv, mine >> kv.page_shift, head, which) + (mine & in_page)] : 0.0f;
    __bf16* const out = (which ? v : k) + ((int64_t)t0 * kv.heads + head) * D + lane * V;
    auto put = [&](int e, const uint8_t (&c)[V]) {
        const float s = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scale), e));
        typename Vec<V>::b y;
#pragma unroll
        for (int j = 0; j < V; j++) y[j] = (__bf16)(code_value<FMT>(c[j]) * s);
        *(typename Vec<V>::b*)(out + (int64_t)e * kv.heads * D) = y;
    };
    typename Vec<V>::b zero;
#pragma unroll
    for (int j = 0; j < V; j++) zero[j] = (__bf16)0.0f;
    const uint64_t there = __ballot(in_cache);
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = wave * EACH + i;
        if (t0 + e < n && !(there >> e & 1)) *(typename Vec<V>::b*)(out + (int64_t)e * kv.heads * D) = zero;
    }
    if (which == 0) {
        uint8_t c[EACH][V];
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int slot = __builtin_amdgcn_readlane(in_cache ? mine : 0, wave * EACH + i);
            const uint8_t* const at = kv.codes + kv_block<D>(kv, slot >> kv.page_shift, head, 0) + k_byte<D>(slot & in_page, lane * V);
            typedef uint8_t bytes __attribute__((ext_vector_type(V)));
            const bytes b = *(const bytes*)at;
#pragma unroll
            for (int j = 0; j < V; j++) c[i][j] = b[j];
        }
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (there >> (wave * EACH + i) & 1) put(wave * EACH + i, c[i]);
        return;
    }
    // one tile after the other; the next one's values are on their way while the first's are taken out
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    uint64_t left = there, here = 0;
    u4 next = {};
    const int at = min((int)threadIdx.x, D * 4 - 1);
    auto load = [&] {
        const int tile = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)left) - 1) >> 6, slot0 = tile << 6;
        here = __ballot(in_cache && mine >> 6 == tile);
        left &= ~here;
        next = *(const u4*)(kv.codes + kv_block<D>(kv, slot0 >> kv.page_shift, head, 1) + (size_t)(slot0 & in_page) * D + at * 16);
    };
    if (left) load();
    while (here) {
        if ((int)threadIdx.x < D * 4) {
            uint32_t* const to = tile_codes + row(at >> 2) + (at & 3) * 4;
            to[0] = next.x, to[1] = next.y, to[2] = next.z, to[3] = next.w;
        }
        const uint64_t now = here;
        here = 0;
        if (left) load();
        lds_barrier();
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int e = wave * EACH + i;
            if (!(now >> e & 1)) continue;
            const uint32_t t = __builtin_amdgcn_readlane(mine, e) & 63, byte = v_byte<D>(t, 0);
            uint8_t c[V];
#pragma unroll
            for (int j = 0; j < V; j++) c[j] = ((const uint8_t*)(tile_codes + row(lane * V + j)))[byte];
            put(e, c);
        }
        if (here) lds_barrier();
    }
}

// A workgroup for each (sequence, kv head, keys or values): 64 moves at a time read into LDS, then written. Bound by its trips to
// memory: starts, slots, codes, out (a path of three, 4 x 256: 2.1 us).
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
    int heads;  // heads of a token that the kernel takes: the values' last, or without them
};

template <int V>
__device__ __forceinline__ void put(__bf16* to, const float (&y)[V], int lane) {
    typename Vec<V>::b o;
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = (__bf16)y[i];
    *(typename Vec<V>::b*)(to + lane * V) = o;
}

// A workgroup takes some heads (blockIdx.y's share) of one token, a wave a head at a time: queries (with their gates),
// keys, values. The angles' sines and cosines are made once per workgroup, while the first heads' partials are on their way:
// pos * inv_freq in turns in f64, whose fraction is exact to f32 at any position. P: partials of a head in
// flight at once (summed as they come instead: a token of 16 x 256, 8 partials 4.4 us against 3.4, 5 of 24 x 256, 4 partials
// into the cache 5.6 against 4.2, 2048 dense ones, one partial 33.9 against 29.9, which is 5.9 TB/s).
template <int D, int FMT, int P>
__global__ __launch_bounds__(64 * WAVES) void attn_prep_kernel(const Prep a) {
    constexpr int V = D / 64;
    typedef typename Vec<V>::f vec;
    __shared__ __align__(16) float angle[2][D];  // what a dimension and its partner are multiplied by
    __shared__ __align__(16) float rows[WAVES][D];
    // all lines of the arguments are fetched at once, and what does not depend on the sums is read ahead of them: each would be
    // a trip to memory of its own when first touched (2048 tokens of 24 x 256: 33.9 us against 36.8)
    const auto* const line = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" ::"s"(line[0]), "s"(line[16]), "s"(line[32]));
    static_assert(sizeof(Prep) > 128);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = a.rot / 2;
    const int64_t t = blockIdx.x;
    const int per = a.gated ? 2 : 1, heads = a.heads;
    const int64_t ld = (int64_t)(a.q_heads * per + 2 * a.kv_heads) * D, stride = a.n * ld;
    const int share = (heads + gridDim.y - 1) / gridDim.y, h1 = min(heads, (int)(blockIdx.y + 1) * share);
    const int slot = FMT ? a.slots[t] : 0, pos = half ? a.pos[t] : 0;
    const int i_freq = (int)threadIdx.x < half ? threadIdx.x : threadIdx.x - half;
    float freq = 0.0f;
    if ((int)threadIdx.x < a.rot) freq = a.inv_freq[i_freq];
    vec norm[2] = {};
    if (a.q_w) norm[0] = ((const vec*)a.q_w)[lane];
    if (a.k_w) norm[1] = ((const vec*)a.k_w)[lane];
    // a head's partials, with a query's those of its gate, are read while the head before is worked on
    Ahead<V, P> next, next_gate;
    auto read = [&](int h) {
        const bool is_q = h < a.q_heads;
        const float* const x = a.x + t * ld + (int64_t)(is_q ? h * per : h - a.q_heads + a.q_heads * per) * D;
        const int splits = P == 1 && h >= h1 ? 0 : a.splits;  // (of one partial each, without a branch: 29.9 us against 34.3)
        next.read(x, splits, stride, lane);
        next_gate.read(x + D, is_q && a.gated ? splits : 0, stride, lane);
    };
    const int h0 = blockIdx.y * share + wave;
    if (P == 1 || h0 < h1) read(h0);
    if ((int)threadIdx.x < a.rot) {
        const double turns = (double)pos * (double)freq * 0.15915494309189535;
        const float part = (float)(turns - rint(turns));
        float sn, cs;
        sincospif(2.0f * part, &sn, &cs);
        angle[0][threadIdx.x] = cs, angle[1][threadIdx.x] = (int)threadIdx.x < half ? -sn : sn;
    }
    lds_barrier();
    const vec own = *(const vec*)&angle[0][lane * V], other = *(const vec*)&angle[1][lane * V];
    for (int h = h0; h < h1; h += WAVES) {
        const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
        float y[V], gate[V];
        next.sum(a.splits, stride, lane, y);
        if (is_q && a.gated) next_gate.sum(a.splits, stride, lane, gate);
        if (P == 1 || h + WAVES < h1) read(h + WAVES);
        if (is_q ? a.q_w != nullptr : is_k && a.k_w) {
            const vec w = is_q ? norm[0] : norm[1];
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) ss += y[i] * y[i];
            // (rsqrt to a unit in the last place: below the rounding of the mean's own sum)
            const float r = __builtin_amdgcn_rsqf(wave_sum(ss) * (1.0f / D) + a.eps);
#pragma unroll
            for (int i = 0; i < V; i++) y[i] = w[i] * (y[i] * r);
        }
        if (half && (is_q || is_k)) {
            vec u;
#pragma unroll
            for (int i = 0; i < V; i++) u[i] = y[i];
            *(vec*)&rows[wave][lane * V] = u;
            __builtin_amdgcn_wave_barrier();
            float partner[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int d = lane * V + i;
                partner[i] = rows[wave][d < half ? d + half : d < a.rot ? d - half : d];
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float turned = y[i] * own[i] + partner[i] * other[i];
                y[i] = lane * V + i < a.rot ? turned : y[i];
            }
            __builtin_amdgcn_wave_barrier();
        }
        if (is_q) {
            put<V>(a.q + (t * a.q_heads + h) * D, y, lane);
            if (a.gated) put<V>(a.gate + (t * a.q_heads + h) * D, gate, lane);
            continue;
        }
        const int head = h - a.q_heads - (is_k ? 0 : a.kv_heads);
        if constexpr (FMT == 0) put<V>((is_k ? a.k : a.v) + (t * a.kv_heads + head) * D, y, lane);
        else quantise_into<D, FMT, V>(a.kv, slot, head, is_k ? 0 : 1, y, lane);
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
constexpr size_t BATCH_FROM = 64;               // tokens from which the batch kernels take over: a whole batch

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
        if (n >= BATCH_FROM) {
            const Source ks = {(const __bf16*)k_bf16}, vs = {(const __bf16*)v_bf16};
            auto* f = kv->fmt == QH_KV_I8 ? kv_write_batch_kernel<D, QH_KV_I8, false> : kv_write_batch_kernel<D, QH_KV_E4M3, false>;
            launch_kernel(f, dim3((unsigned)((n + BATCH - 1) / BATCH), c.heads * 2), dim3(64 * BATCH_WAVES), (hipStream_t)stream, c, ks, vs, slots, (int)n, 0);
            return;
        }
        auto* f = kv->fmt == QH_KV_I8 ? kv_write_kernel<D, QH_KV_I8> : kv_write_kernel<D, QH_KV_E4M3>;
        launch_kernel(f, grid, dim3(64 * WAVES), (hipStream_t)stream, c, (const __bf16*)k_bf16, (const __bf16*)v_bf16, slots, vectors);
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
        if (n >= BATCH_FROM) {
            auto* f = kv->fmt == QH_KV_I8 ? kv_read_batch_kernel<D, QH_KV_I8> : kv_read_batch_kernel<D, QH_KV_E4M3>;
            launch_kernel(f, dim3((unsigned)((n + BATCH - 1) / BATCH), c.heads * 2), dim3(64 * BATCH_WAVES), (hipStream_t)stream, c, slots, (int)n, (__bf16*)k_bf16, (__bf16*)v_bf16);
            return;
        }
        auto* f = kv->fmt == QH_KV_I8 ? kv_read_kernel<D, QH_KV_I8> : kv_read_kernel<D, QH_KV_E4M3>;
        launch_kernel(f, grid, dim3(64 * WAVES), (hipStream_t)stream, c, slots, vectors, (__bf16*)k_bf16, (__bf16*)v_bf16);
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
        launch_kernel(kv_move_kernel<decltype(d)::value>, dim3(n_seq, c.heads * 2), dim3(256), (hipStream_t)stream, c, src, dst, (int)n, start);
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
    if (n > MAX_TOKENS || ((uintptr_t)x | (uintptr_t)q_w | (uintptr_t)k_w | (uintptr_t)q | (uintptr_t)gate | (uintptr_t)k | (uintptr_t)v) % 16)
        return fail(QH_EINVAL, "attn_prep: %zu tokens (up to 2^20), buffers 16-byte aligned", n);
    a.x = x, a.splits = splits, a.n = (int64_t)n, a.q_heads = rows->q_heads, a.kv_heads = rows->kv_heads, a.rot = rows->rot;
    a.gated = rows->gated != 0, a.q_w = q_w, a.k_w = k_w, a.inv_freq = inv_freq, a.eps = eps, a.pos = pos, a.slots = slots;
    a.q = (__bf16*)q, a.gate = (__bf16*)gate, a.k = (__bf16*)k, a.v = (__bf16*)v;
    // into the cache, many tokens' values are turned over by the batch kernel
    const bool batch = kv && n >= BATCH_FROM;
    const int heads = a.heads = rows->q_heads + (batch ? 1 : 2) * rows->kv_heads;
    const unsigned shares = n >= 512 ? 1 : (heads + WAVES - 1) / WAVES;
    by_dim(D, [&](auto d) {
        constexpr int DD = decltype(d)::value;
        auto kernel = [&](auto p) {
            constexpr int P = decltype(p)::value;
            return !kv ? attn_prep_kernel<DD, 0, P> : kv->fmt == QH_KV_I8 ? attn_prep_kernel<DD, QH_KV_I8, P> : attn_prep_kernel<DD, QH_KV_E4M3, P>;
        };
        auto* f = splits == 1 ? kernel(std::integral_constant<int, 1>{}) : splits <= 4 ? kernel(std::integral_constant<int, 4>{}) : kernel(std::integral_constant<int, 8>{});
        launch_kernel(f, dim3((unsigned)n, shares), dim3(64 * WAVES), (hipStream_t)stream, a);
        if (!batch) return;
        const int64_t ld = (int64_t)(rows->q_heads * (a.gated ? 2 : 1) + 2 * rows->kv_heads) * D;
        const Source vs = {nullptr, x, splits, (int64_t)n * ld, ld, (int)(ld - (int64_t)rows->kv_heads * D)};
        auto* fv = kv->fmt == QH_KV_I8 ? kv_write_batch_kernel<DD, QH_KV_I8, true> : kv_write_batch_kernel<DD, QH_KV_E4M3, true>;
        launch_kernel(fv, dim3((unsigned)((n + BATCH - 1) / BATCH), rows->kv_heads), dim3(64 * BATCH_WAVES), (hipStream_t)stream, a.kv, vs, vs, slots, (int)n, 1);
    });
    return launched("attn_prep");
}
