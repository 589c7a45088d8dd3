// The paged, quantised KV cache (qh_kv of include/qwenny_hip.h): where a token's codes and scales lie, and the checks of
// its description. A (page, kv head) is one block of keys and one of values of page * head_dim bytes each, laid out as the
// attention's matrix instructions read them, so that every load of a wave is 1 KiB in a row and no code is moved between
// lanes:
//   keys: 16 tokens x 64 dimensions in a row ([page / 16][head_dim / 64][16][64]); a lane's 16 bytes are one token's;
//   values: 64 tokens side by side ([page / 64][head_dim][64]), token 16 w + 4 g + j at byte 16 g + 4 w + j: a lane's 16
//   bytes are the tokens whose probabilities the product of queries and keys left in that lane.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/qwenny_hip.h"
#include "attn_plan.h"
#include "internal.h"

namespace qh {

struct Kv {
    uint8_t* codes;
    float* scales;
    int heads, page_shift;
    int64_t slots;  // pages << page_shift
};

// first byte of the keys' (which = 0) or values' (1) block of (page, head)
template <int D>
__device__ __forceinline__ size_t kv_block(const Kv& kv, int64_t page, int head, int which) {
    return ((size_t)(page * kv.heads + head) * 2 + which) * D << kv.page_shift;
}
__device__ __forceinline__ size_t kv_scale(const Kv& kv, int64_t page, int head, int which) {
    return ((size_t)(page * kv.heads + head) * 2 + which) << kv.page_shift;
}
// dimension d of token t of a page, within its block
template <int D>
__device__ __forceinline__ uint32_t k_byte(uint32_t t, uint32_t d) {
    return (t >> 4) * (16 * D) + (d >> 6) * 1024 + (t & 15) * 64 + (d & 63);
}
template <int D>
__device__ __forceinline__ uint32_t v_byte(uint32_t t, uint32_t d) {
    return (t >> 6) * (64 * D) + d * 64 + ((t >> 2) & 3) * 16 + ((t >> 4) & 3) * 4 + (t & 3);
}

// A launch past the stack of call configurations that hipLaunchKernelGGL goes through: 0.2 us less of the host's time.
template <class T>
struct Same {
    typedef T type;
};
template <class... P>
inline void launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, typename Same<P>::type... a) {
    void* args[] = {&a...};
    (void)hipLaunchKernel((const void*)kernel, grid, block, args, 0, stream);  // (its error is read by hipGetLastError)
}

// The cache's description checked; QH_OK and the kernels' form of it in *out, or QH_EINVAL.
inline int kv_check(const char* who, const qh_kv* kv, Kv* out) {
    if (!kv || !kv->codes || !kv->scales) return fail(QH_EINVAL, "%s: null cache", who);
    if (kv->fmt != QH_KV_I8 && kv->fmt != QH_KV_E4M3) return fail(QH_EINVAL, "%s: cache format %d", who, kv->fmt);
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return fail(QH_EINVAL, "%s: heads of %d dimensions (64, 128 or 256)", who, kv->head_dim);
    if (kv->page < KV_TILE || kv->page > 1024 || (kv->page & (kv->page - 1)))
        return fail(QH_EINVAL, "%s: pages of %d tokens (a power of two from 64 to 1024)", who, kv->page);
    if (kv->heads < 1 || kv->heads > 1024) return fail(QH_EINVAL, "%s: %d kv heads (1 to 1024)", who, kv->heads);
    if (kv->pages < 1 || kv->pages > 0x7fffffffu / (size_t)kv->page)
        return fail(QH_EINVAL, "%s: %zu pages of %d tokens (slots are 31-bit)", who, kv->pages, kv->page);
    if ((uintptr_t)kv->codes % 16 || (uintptr_t)kv->scales % 16)
        return fail(QH_EINVAL, "%s: cache buffers must be 16-byte aligned", who);
    out->codes = (uint8_t*)kv->codes;
    out->scales = kv->scales;
    out->heads = kv->heads;
    out->page_shift = __builtin_ctz((unsigned)kv->page);
    out->slots = (int64_t)kv->pages * kv->page;
    return QH_OK;
}

}  // namespace qh
