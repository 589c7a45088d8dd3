// The cache's pages among the requests of a server (qh_kv_plan, qh_kv_release): page tables, and the starts, slots and
// positions of a step, made from the requests' lengths on the device.
//
// With k_b = ceil(len_b / page) pages kept, a release gives the pages k_b .. held_b back, and a plan takes
//   need_b = max(0, ceil((len_b + add_b) / page) - held_b), for the sequences in turn while c_b = sum_{b' <= b} need_b' does
// not pass the free pages. The list of free pages is a stack: a plan takes from its end, a release puts the same pages back
// in the places that a plan took them from. Prefix sums over the sequences say where each one's part begins; which sequence
// a page or a token belongs to is found in them by halving. Bound by the launch and a few trips to memory one after the other:
// a step's arrays are small, and one workgroup has the sums in its LDS. (Kernel times, medians of a trace: one sequence 2.7 us and
// its release 1.9; 1,000 sequences of up to 8 tokens 9.6 and 3.7; 16 prompts 7.0 and 2.4.)
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_plan.h"
#include "internal.h"
#include "kv.h"

using namespace qh;

namespace {

constexpr int THREADS = 1024;  // a thread for each sequence that a step can have
constexpr int RELEASED = 256;  // threads that give back a finished sequence's pages, however few sequences there are
static_assert(THREADS >= TREE_MAX_SEQS);

struct Args {
    int32_t* free;
    int32_t* n_free;
    int32_t* table;
    int32_t* held;
    const int32_t* len;
    const int32_t* add;
    const uint64_t* mask;
    int32_t* start;
    int32_t* slots;
    int32_t* pos;
    int32_t* granted;
    int64_t pages, table_ld;
    int32_t page_shift, n_seq, n;
};

// Sums of N numbers over the threads before this one, and over all; `sums`: LDS.
template <int N>
__device__ __forceinline__ void scan(const int64_t (&v)[N], int64_t (&sums)[N][THREADS / 64], int64_t (&before)[N], int64_t (&all)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int k = 0; k < N; k++) {
        int64_t run = v[k];
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t left = __shfl_up(run, d);
            run += lane >= d ? left : 0;
        }
        if (lane == 63) sums[k][wave] = run;
        before[k] = run - v[k];
        all[k] = 0;
    }
    __syncthreads();
    for (int w = 0; w < waves; w++) {
#pragma unroll
        for (int k = 0; k < N; k++) {
            before[k] += w < wave ? sums[k][w] : 0;
            all[k] += sums[k][w];
        }
    }
}

// The last sequence whose part begins at or before `at`, where parts of nothing lie before their successor's.
__device__ __forceinline__ int find(const int64_t* begin, int n_seq, int64_t at) {
    int lo = 0, hi = n_seq;  // begin[lo] <= at < begin[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (begin[mid] <= at ? lo : hi) = mid;
    }
    return lo;
}

__device__ __forceinline__ int held_of(const Args& a, int b) { return (int)min((int64_t)max(a.held[b], 0), a.table_ld); }
__device__ __forceinline__ int64_t free_of(const Args& a) { return min((int64_t)max(*a.n_free, 0), a.pages); }
__device__ __forceinline__ int64_t pages_of(const Args& a, int64_t tokens) { return (tokens + (1 << a.page_shift) - 1) >> a.page_shift; }

__global__ __launch_bounds__(THREADS) void kv_release_kernel(const Args a) {
    __shared__ int64_t sums[1][THREADS / 64], begin[THREADS];
    __shared__ int32_t kept[THREADS];
    const int b = threadIdx.x;
    int64_t gone = 0;
    const int64_t had = free_of(a);
    if (b < a.n_seq) {
        const int held = held_of(a, b), len = a.len[b];
        const int keep = len < 0 ? held : (int)min(pages_of(a, len), (int64_t)held);
        gone = held - keep;
        kept[b] = keep;
    }
    int64_t before[1], total[1];
    scan<1>({gone}, sums, before, total);
    const int64_t all = total[0];
    begin[b] = before[0];
    __syncthreads();
    // (a pool that says to hold more pages than there are keeps within its list)
    for (int64_t i = b; i < all; i += blockDim.x) {
        const int s = find(begin, a.n_seq, i);
        int32_t* const from = a.table + s * a.table_ld + kept[s] + (i - begin[s]);
        const int64_t to = had + all - 1 - i;
        if (to < a.pages) a.free[to] = *from;
        *from = -1;
    }
    if (b < a.n_seq) a.held[b] = kept[b];
    if (b == 0) *a.n_free = (int32_t)min(had + all, a.pages);
}

// A token's slot and position: token `node` of a sequence of `len` cached ones, its position's page given.
__device__ __forceinline__ void put_token(const Args& a, int i, int node, int64_t len, int64_t page, bool granted) {
    const int64_t at = len + node;
    const int64_t slot = (page << a.page_shift) + (at & ((1 << a.page_shift) - 1));
    a.slots[i] = granted && page >= 0 && page < a.pages ? (int32_t)slot : -1;
    int depth = node;
    if (a.mask && node < 64) depth = (int)__popcll(a.mask[i] & ((1ull << node) - 1));  // (whether it sees itself or not)
    a.pos[i] = (int32_t)min(len + depth, (int64_t)0x7fffffff);
}

// FILL: the tokens' slots and positions too, otherwise kv_fill_kernel makes them.
template <bool FILL>
__global__ __launch_bounds__(THREADS) void kv_plan_kernel(const Args a) {
    __shared__ int64_t sums[2][THREADS / 64], granted_sums[1][THREADS / 64], begin[THREADS], first[THREADS];
    __shared__ int32_t had[THREADS], ok[THREADS], lens[THREADS];
    const int b = threadIdx.x;
    int64_t need = 0, add = 0;
    const int64_t there = free_of(a);
    bool fits = false;
    if (b < a.n_seq) {
        const int held = held_of(a, b);
        const int64_t len = a.len[b], more = a.add[b];
        add = max(more, (int64_t)0);
        fits = len >= 0 && more >= 0 && len + add <= a.table_ld << a.page_shift;
        need = fits && add > 0 ? max(pages_of(a, len + add) - held, (int64_t)0) : 0;
        had[b] = held;
        lens[b] = (int)len;
    }
    int64_t upto[2], all[2];
    scan<2>({need, add}, sums, upto, all);
    const int64_t before = upto[0], token = upto[1], tokens = all[1];
    const bool granted = fits && (need == 0 || before + need <= there);
    begin[b] = before;
    first[b] = token;
    ok[b] = granted;
    if (b < a.n_seq) {
        a.start[b] = (int32_t)min(token, (int64_t)a.n);
        a.granted[b] = granted;
    }
    if (b == 0) a.start[a.n_seq] = (int32_t)min(tokens, (int64_t)a.n);
    // what is granted is the first of all that is asked for
    int64_t taken = all[0];
    if (taken > there) {
        int64_t rest[1], total[1];
        scan<1>({granted ? need : 0}, granted_sums, rest, total);
        taken = total[0];
    }
    __syncthreads();
    for (int64_t i = b; i < taken; i += blockDim.x) {
        const int s = find(begin, a.n_seq, i);
        a.table[s * a.table_ld + had[s] + (i - begin[s])] = a.free[there - 1 - i];
    }
    if (FILL) {
        for (int i = b; i < a.n; i += blockDim.x) {
            if (i >= tokens) {
                a.slots[i] = -1;
                a.pos[i] = 0;
                continue;
            }
            const int s = find(first, a.n_seq, i), node = (int)(i - first[s]);
            const int64_t k = ((int64_t)lens[s] + node) >> a.page_shift;
            int64_t page = -1;  // (from where the table's new pages come from: nothing is read that was written here)
            if (ok[s]) page = k < had[s] ? a.table[s * a.table_ld + k] : a.free[there - 1 - (begin[s] + k - had[s])];
            put_token(a, i, node, lens[s], page, ok[s]);
        }
    }
    if (b < a.n_seq && granted) a.held[b] = (int32_t)(had[b] + need);
    if (b == 0) *a.n_free = (int32_t)(there - taken);
}

// The tokens of a large step, after kv_plan_kernel.
__global__ __launch_bounds__(256) void kv_fill_kernel(const Args a) {
    __shared__ int64_t first[TREE_MAX_SEQS];
    for (int b = threadIdx.x; b < a.n_seq; b += 256) first[b] = a.start[b];
    __syncthreads();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.n) return;
    if (i >= a.start[a.n_seq]) {
        a.slots[i] = -1;
        a.pos[i] = 0;
        return;
    }
    const int s = find(first, a.n_seq, i), node = (int)(i - first[s]);
    const int64_t len = a.len[s];
    const bool ok = a.granted[s];
    put_token(a, i, node, len, ok ? a.table[s * a.table_ld + ((len + node) >> a.page_shift)] : -1, ok);
}

// A workgroup's threads: one for each sequence, and for each of `work` pages or tokens up to THREADS. A single sequence's plan and
// release take 2.7 + 1.9 us so, 4.9 + 2.9 with 1,024 always.
dim3 threads_for(const Args& a, size_t work) { return dim3((unsigned)std::min<size_t>(THREADS, (std::max<size_t>(a.n_seq, work) + 63) / 64 * 64)); }

int pool_check(const char* who, const qh_kv_pool* p, Args* a) {
    if (!p || !p->free || !p->n_free || !p->table || !p->held) return fail(QH_EINVAL, "%s: null pool", who);
    if (p->page < KV_TILE || p->page > 1024 || (p->page & (p->page - 1)))
        return fail(QH_EINVAL, "%s: pages of %d tokens (a power of two from 64 to 1024)", who, p->page);
    if (p->pages < 1 || p->pages > 0x7fffffffu / (size_t)p->page)
        return fail(QH_EINVAL, "%s: %zu pages of %d tokens (slots are 31-bit)", who, p->pages, p->page);
    if (p->n_seq < 1 || p->n_seq > TREE_MAX_SEQS) return fail(QH_EINVAL, "%s: %d sequences (1 to %d)", who, p->n_seq, TREE_MAX_SEQS);
    if (p->table_ld < 1 || p->table_ld > ((size_t)1 << 30) / p->page)
        return fail(QH_EINVAL, "%s: tables of %zu pages of %d tokens (1 to 2^30 positions)", who, p->table_ld, p->page);
    a->free = p->free, a->n_free = p->n_free, a->table = p->table, a->held = p->held;
    a->pages = (int64_t)p->pages, a->table_ld = (int64_t)p->table_ld;
    a->page_shift = __builtin_ctz((unsigned)p->page), a->n_seq = p->n_seq;
    return QH_OK;
}

}  // namespace

extern "C" int qh_kv_release(void* stream, const qh_kv_pool* pool, const int32_t* len) {
    Args a = {};
    if (int e = pool_check("kv_release", pool, &a)) return e;
    if (!len) return fail(QH_EINVAL, "kv_release: null");
    a.len = len;
    launch_kernel(kv_release_kernel, dim3(1), threads_for(a, RELEASED), (hipStream_t)stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "kv_release launch: %s", hipGetErrorString(e));
    return QH_OK;
}

extern "C" int qh_kv_plan(void* stream, const qh_kv_pool* pool, const int32_t* len, const int32_t* add, const uint64_t* mask, size_t n,
                          int32_t* start, int32_t* slots, int32_t* pos, int32_t* granted) {
    Args a = {};
    if (int e = pool_check("kv_plan", pool, &a)) return e;
    if (!len || !add || !start || !granted || (n && (!slots || !pos))) return fail(QH_EINVAL, "kv_plan: null");
    if (n > (size_t)1 << 30) return fail(QH_EINVAL, "kv_plan: %zu tokens (up to 2^30)", n);
    a.len = len, a.add = add, a.mask = mask, a.n = (int32_t)n;
    a.start = start, a.slots = slots, a.pos = pos, a.granted = granted;
    if (n <= 4 * THREADS) {
        launch_kernel(kv_plan_kernel<true>, dim3(1), threads_for(a, n), (hipStream_t)stream, a);
    } else {
        launch_kernel(kv_plan_kernel<false>, dim3(1), dim3(THREADS), (hipStream_t)stream, a);
        launch_kernel(kv_fill_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), (hipStream_t)stream, a);
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return fail(QH_EHIP, "kv_plan launch: %s", hipGetErrorString(e));
    return QH_OK;
}
