// l3_cache.hip -- page tables and slot maps of a paged cache, built from the lengths of a batch of requests.
//
// Request i has len[i] tokens in the cache, on held[i] pages named by table[i][0 .. held[i]); off[i+1] - off[i] tokens are new.
// Token t of the step, the j-th new one of request i, is at position p = len[i] + j and goes to the slot
// table[i][p / page] * page + p % page.  Pages that are missing come off the end of the free list, in order of the requests.
//
// Two launches, because a request's pages depend on those of all requests before it:
//   plan   a thread per request: how many pages it asks for, and their sum over the requests before it in its workgroup; the
//          sums of the workgroups.  What a request was is copied to the workspace, so that its new state may replace the old.
//   apply  adds up the workgroups' sums, decides who is served, writes table, slots, positions and the new state.
#include "l3_token_kernels.h"

#include "l3_dev.h"

namespace l3 {

namespace {

struct CacheHead { uint64_t left; uint32_t bad, pad; };

__device__ __forceinline__ u64 block_escan64(u64 v, u64* tmp, u64* total) {   // kPlanThreads threads; tmp: one word per wave
    const u64 inc = wave_iscan64(v);
    if (lane_id() == 63) tmp[wave_id()] = inc;
    __syncthreads();
    u64 base = 0, tot = 0;
    for (int i = 0; i < kPlanThreads / 64; i++) {
        if (i < wave_id()) base += tmp[i];
        tot += tmp[i];
    }
    __syncthreads();
    *total = tot;
    return base + inc - v;
}

template <bool TRIM>
__global__ __launch_bounds__(kPlanThreads) void cache_plan_kernel(CacheArgs A, PlanRec* recs, u64* blocks, CacheHead* head) {
    __shared__ u64 tmp[kPlanThreads / 64];
    const uint64_t i = (uint64_t)blockIdx.x * kPlanThreads + threadIdx.x;
    PlanRec r{};
    if (i < A.n)
        r = TRIM ? plan_trim(A.len[i], A.held[i], A.keep[i], A.page, A.max_pages)
                 : plan_slots(A.len[i], A.held[i], A.off[i], A.off[i + 1], A.cap, A.page, A.max_pages);
    u64 total;
    r.before = block_escan64((u64)r.delta, tmp, &total);
    if (i < A.n) recs[i] = r;
    if (threadIdx.x == 0) {
        if (blockIdx.x * (uint64_t)kPlanThreads < A.n) blocks[blockIdx.x] = total;
        if (blockIdx.x == 0) {
            const int32_t left = *A.n_free;
            const bool bad = left < 0 || (uint32_t)left > A.n_pages;
            // an unusable count: nothing can be taken from the pool and nothing put back
            head->left = bad ? (TRIM ? A.n_pages : 0) : (uint64_t)left;
            head->bad = bad;
            *A.status = bad ? (uint32_t)kCacheBad : 0u;   // the next kernel adds what it finds
        }
    }
}

// pages that the requests in the workgroups before block `b` ask for; b <= n_blocks <= 1,024
__device__ __forceinline__ u64 pages_before(const u64* blocks, uint64_t b) {
    u64 s = 0;
    for (uint64_t k = 0; k < b; k++) s += blocks[k];
    return s;
}

constexpr int kApplyThreads = 256;

__global__ __launch_bounds__(kApplyThreads) void cache_slots_kernel(CacheArgs A, const PlanRec* recs, const u64* blocks,
                                                                    const CacheHead* head, uint64_t request_blocks) {
    const uint64_t left = head->left;
    uint32_t bits = 0;
    if (blockIdx.x < request_blocks) {   // a thread per request: its new state
        const uint64_t i = (uint64_t)blockIdx.x * kApplyThreads + threadIdx.x;
        if (i < A.n) {
            const PlanRec r = recs[i];
            const u64 before = pages_before(blocks, i / kPlanThreads) + r.before;
            const bool served = slots_served(r, before, left);
            A.len_out[i] = served ? r.new_len : r.len;
            A.held_out[i] = served ? r.held + r.delta : r.held;
            bits = served ? 0u : r.flags ? r.flags : (uint32_t)kCachePool;
        }
    } else {                             // a thread per token
        const uint64_t total = A.n ? A.off[A.n] : 0;
        const uint64_t t = (uint64_t)(blockIdx.x - request_blocks) * kApplyThreads + threadIdx.x;
        if (t < A.cap && t < total) {
            uint64_t a = 0, b = A.n;     // the last request that starts at or before t
            while (b - a > 1) { const uint64_t m = (a + b) / 2; if (A.off[m] <= t) a = m; else b = m; }
            int64_t slot = -1;
            int32_t pos = -1;
            const uint64_t first = A.off[a];
            const PlanRec r = recs[a];
            const u64 before = pages_before(blocks, a / kPlanThreads) + r.before;
            if (first <= t && t < A.off[a + 1] && slots_served(r, before, left)) {
                pos = r.len + (int32_t)(t - first);
                const uint32_t p = (uint32_t)pos / A.page, in = (uint32_t)pos % A.page;
                int32_t id;
                if (p < (uint32_t)r.held) {
                    id = A.table[a * A.table_stride + p];
                } else {
                    id = A.free_pages[left - 1 - before - (p - (uint32_t)r.held)];
                    if (in == 0) A.table[a * A.table_stride + p] = id;   // a new page's first slot is always a new token's
                }
                slot = slot_of(id, in, A.page, A.n_pages);
                if (slot < 0) bits = kCachePage;
            }
            A.slots[t] = slot;
            A.pos[t] = pos;
        }
    }
    if (bits) atomicOr(A.status, bits);
}

// The new count of the pool: pages of all requests that are served.
template <bool TRIM>
__global__ __launch_bounds__(kPlanThreads) void cache_count_kernel(CacheArgs A, const PlanRec* recs, const u64* blocks, const CacheHead* head) {
    __shared__ u64 tmp[kPlanThreads / 64];
    u64 mine = 0;
    const uint64_t left = head->left;
    u64 base = 0;
    for (uint64_t b = 0; b * kPlanThreads < A.n; b++) {
        const uint64_t i = b * kPlanThreads + threadIdx.x;
        if (i < A.n) {
            const PlanRec r = recs[i];
            if (TRIM ? trim_served(r, base + r.before, left, A.n_pages) : slots_served(r, base + r.before, left)) mine += (u64)r.delta;
        }
        base += blocks[b];
    }
    u64 total;
    (void)block_escan64(mine, tmp, &total);
    if (threadIdx.x == 0) {
        const int32_t n = *A.n_free;
        *A.n_free_out = head->bad ? n : TRIM ? n + (int32_t)total : n - (int32_t)total;
    }
}

// A wave per request: its new state, and the pages it gives back to the end of the free list.
__global__ __launch_bounds__(kApplyThreads) void cache_trim_kernel(CacheArgs A, const PlanRec* recs, const u64* blocks, const CacheHead* head) {
    const uint64_t left = head->left;
    for (uint64_t i = (uint64_t)blockIdx.x * (kApplyThreads / 64) + wave_id(); i < A.n; i += (uint64_t)gridDim.x * (kApplyThreads / 64)) {
        const PlanRec r = recs[i];
        const u64 before = pages_before(blocks, i / kPlanThreads) + r.before;
        const bool served = trim_served(r, before, left, A.n_pages);
        if (lane_id() == 0) {
            A.len_out[i] = served ? r.new_len : r.len;
            A.held_out[i] = served ? r.held - r.delta : r.held;
            if (!served) atomicOr(A.status, r.flags ? r.flags : (uint32_t)kCachePool);
        }
        if (!served) continue;
        const int32_t* from = A.table + i * A.table_stride + (r.held - r.delta);
        int32_t* to = A.free_pages + left + before;
        for (int32_t j = lane_id(); j < r.delta; j += 64) to[j] = from[j];
    }
}

struct Parts { PlanRec* recs; u64* blocks; CacheHead* head; uint64_t plan_blocks; };
Parts parts_of(const CacheArgs& A) {
    const CacheWork W = cache_work(A.n);
    uint8_t* base = (uint8_t*)A.work;
    return {(PlanRec*)(base + W.recs), (u64*)(base + W.blocks), (CacheHead*)(base + W.head), A.n ? (A.n + kPlanThreads - 1) / kPlanThreads : 1};
}

}  // namespace

hipError_t launch_cache_slots(const CacheArgs& A, hipStream_t stream) {
    const Parts P = parts_of(A);
    hipError_t e = launch(cache_plan_kernel<false>, P.plan_blocks, kPlanThreads, stream, A, P.recs, P.blocks, P.head);
    if (e != hipSuccess) return e;
    const uint64_t request_blocks = (A.n + kApplyThreads - 1) / kApplyThreads, token_blocks = (A.cap + kApplyThreads - 1) / kApplyThreads;
    if (request_blocks + token_blocks)
        e = launch(cache_slots_kernel, request_blocks + token_blocks, kApplyThreads, stream, A, (const PlanRec*)P.recs, (const u64*)P.blocks, (const CacheHead*)P.head,
                   request_blocks);
    if (e != hipSuccess) return e;
    return launch(cache_count_kernel<false>, 1, kPlanThreads, stream, A, (const PlanRec*)P.recs, (const u64*)P.blocks, (const CacheHead*)P.head);
}

hipError_t launch_cache_trim(const CacheArgs& A, hipStream_t stream) {
    const Parts P = parts_of(A);
    hipError_t e = launch(cache_plan_kernel<true>, P.plan_blocks, kPlanThreads, stream, A, P.recs, P.blocks, P.head);
    if (e != hipSuccess) return e;
    if (A.n) e = launch(cache_trim_kernel, (A.n + kApplyThreads / 64 - 1) / (kApplyThreads / 64), kApplyThreads, stream, A, (const PlanRec*)P.recs, (const u64*)P.blocks, (const CacheHead*)P.head);
    if (e != hipSuccess) return e;
    return launch(cache_count_kernel<true>, 1, kPlanThreads, stream, A, (const PlanRec*)P.recs, (const u64*)P.blocks, (const CacheHead*)P.head);
}

}  // namespace l3
