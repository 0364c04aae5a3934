// l3_cache.hip -- page tables and slot maps of a paged cache, built from the lengths of a batch of requests.
//
// Request i has len[i] tokens in the cache, on held[i] pages named by table[i][0 .. held[i]); off[i+1] - off[i] tokens are new.
// Token t of the step, the j-th new one of request i, is at position p = len[i] + j and goes to the slot
// table[i][p / page] * page + p % page.  Pages that are missing come off the end of the free list, in order of the requests.
//
// A request's pages depend on those of all requests before it, and its state may be replaced in place, so there are two launches:
//   plan   a thread per request: how many pages it asks for, and their sum over the requests before it in its workgroup; the
//          sums of the workgroups.  What a request was is copied to the workspace.
//   apply  adds up the workgroups' sums, decides who is served, writes table, slots, positions and the new state.
// A step that one workgroup has through in the time of a launch does both in one (cache_slots_one_kernel, cache_trim_one_kernel).
// All of it is bound by latency: chains of dependent loads, and launches.  Measured, us a call among others: 256 requests of one
// token 5.4 (one launch; 4.4 on the GPU), 2,048 prompts with a million tokens 12.5 (4.0 + 9.1 on the GPU; 12.6 MB written, 2.5 us at a
// copy's rate), a trim of 256 requests after drafts 5.1 (3.3 on the GPU), of 2,048 requests 8.3 (4.0 + 3.1).
#include "l3_token_kernels.h"

#include "l3_dev.h"

namespace l3 {

namespace {

struct CacheHead { uint64_t left; uint32_t bad, pad; };

template <int THREADS>
__device__ __forceinline__ u64 block_escan64(u64 v, u64* tmp, u64* total) {   // tmp: one word per wave
    const u64 inc = wave_iscan64(v);
    if (lane_id() == 63) tmp[wave_id()] = inc;
    __syncthreads();
    u64 base = 0, tot = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; i++) {
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
    r.before = block_escan64<kPlanThreads>((u64)r.delta, tmp, &total);
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

constexpr int kApplyThreads = 256, kApplyWaves = kApplyThreads / 64;

template <class V>
__device__ __forceinline__ V apply_sum64(V v, u64* tmp) { return block_sum64<kApplyThreads / 64>(v, tmp); }

// pages that the requests in the plan's workgroups before `b` ask for (give back); by a whole workgroup
__device__ __forceinline__ u64 pages_before(const u64* blocks, uint64_t b, u64* tmp) {
    u64 s = 0;
    for (uint64_t k = threadIdx.x; k < b; k += kApplyThreads) s += blocks[k];
    return apply_sum64(s, tmp);
}

// The pages of all requests that are served: who asks for pages is served as long as the sum up to and with it is at most
// `most`, so it is the largest such sum.  One workgroup.
__device__ u64 pages_served(const PlanRec* recs, const u64* blocks, uint64_t n, u64 most, u64* tmp) {
    const uint64_t n_blocks = (n + kPlanThreads - 1) / kPlanThreads;   // at most 1,024
    constexpr int kPer = (int)(kMaxSeqs / kPlanThreads / kApplyThreads);
    u64 mine[kPer], sum = 0;
#pragma unroll
    for (int k = 0; k < kPer; k++) {
        const uint64_t b = (uint64_t)threadIdx.x * kPer + k;
        mine[k] = b < n_blocks ? blocks[b] : 0;
        sum += mine[k];
    }
    const u64 inc = wave_iscan64(sum);
    __syncthreads();
    if (lane_id() == 63) tmp[wave_id()] = inc;
    __syncthreads();
    u64 run = inc - sum, total = 0;
    for (int w = 0; w < kApplyThreads / 64; w++) { if (w < wave_id()) run += tmp[w]; total += tmp[w]; }
    __syncthreads();
    if (total <= most) return total;
    // the workgroup of the plan in which the sum passes `most`: all before it are served, its own requests one by one
    u64 here = ~0ull, before = 0;
#pragma unroll
    for (int k = 0; k < kPer; k++) {
        if (here == ~0ull && run + mine[k] > most) { here = (u64)threadIdx.x * kPer + k; before = run; }
        run += mine[k];
    }
    const u64 at = block_min64<kApplyThreads / 64>(here, tmp);
    const u64 base = apply_sum64(here == at ? before : 0ull, tmp);
    u64 best = base;
    for (uint64_t i = at * kPlanThreads + threadIdx.x; i < n && i < (at + 1) * kPlanThreads; i += kApplyThreads) {
        const u64 e = base + recs[i].before + (u64)recs[i].delta;
        if (e <= most && e > best) best = e;
    }
    __syncthreads();
    return ~block_min64<kApplyThreads / 64>(~best, tmp);
}

// The last i < n with off[i] <= t, 64 places at a time, by a whole wave (for offsets that are not in order: some i < n).  The first
// 64 places are the same for every t: what stands there is loaded by request_probe, before t is known.
__device__ __forceinline__ uint64_t request_probe(const uint64_t* off, uint64_t n) {
    const uint64_t at = (uint64_t)lane_id() * ((n + 63) / 64);
    return at < n ? off[at] : ~0ull;
}
__device__ __forceinline__ uint64_t first_lane64(uint64_t v) {
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)), lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t request_of(const uint64_t* off, uint64_t n, uint64_t t, uint64_t probe) {
    uint64_t lo = 0, len = n, step = (n + 63) / 64;
    u64 m = __ballot(probe <= t && (uint64_t)lane_id() * step < n);
    for (;;) {
        const uint64_t k = m ? 63 - __builtin_clzll(m) : 0;
        lo += k * step;
        len = len - k * step < step ? len - k * step : step;
        if (len <= 1) return lo;
        step = (len + 63) / 64;
        const uint64_t at = (uint64_t)lane_id() * step;
        m = __ballot(at < len && off[lo + (at < len ? at : 0)] <= t);
    }
}

constexpr int32_t kFirstPages = 2, kPageLanes = 16, kGroupPages = 512;

// Slot and position of token t of request i.  ENTER: it enters its page, if that is beyond the first kGroupPages new ones.
template <bool ENTER>
__device__ __forceinline__ uint32_t place_token(const CacheArgs& A, PageDiv D, const Owner& w, uint64_t i, uint64_t t, int64_t* slot, int32_t* pos) {
    *slot = -1;
    *pos = -1;
    if (w.held < 0 || !owns(w, t)) return 0;
    const uint32_t q = (uint32_t)w.len + (uint32_t)(t - w.first), p = D.of(q), in = q - p * A.page;
    // (pages that are new may not be in the table yet)
    int32_t* entry = A.table + i * A.table_stride + p;
    const int32_t id = p < (uint32_t)w.held ? *entry : A.free_pages[w.next - 1 - (p - (uint32_t)w.held)];
    if (ENTER && in == 0 && p >= (uint32_t)w.held + kGroupPages) *entry = id;
    *pos = (int32_t)q;
    *slot = slot_of(id, in, A.page, A.n_pages);
    return *slot < 0 ? (uint32_t)kCachePage : 0u;
}

// A token in front of the first offset is no request's, and what stands there is not the call's (a step that has a slice of a larger
// batch's offsets).  Unless it is one's after all: offsets that descend may have a request below the first one.
__device__ __forceinline__ bool not_the_calls(uint64_t first, const Owner& w, uint64_t t) { return t < first && !owns(w, t); }

// Tokens in blocks of 256 PER, PER neighbours a thread; the requests of a block are found once and kept in LDS (more than there are
// tokens in a block only where many requests have no new token: then every token looks for its own).  Two tokens a thread / four,
// us: 65,536 requests of one token 11.6 / 13.5, a million tokens of 2,048 prompts 13.0 / 12.5, 4 million of 8,192 27.9 / 25.2, 14 million of
// 65,536 74 / 63 (eight: 67): four from kManyTokens on.
//
// The state of a request is a thread's: 16 requests a workgroup, 256 where there are 16,384 and more.  It enters the first new pages
// itself, sixteen lanes together the next up to kGroupPages, the tokens those behind: a new page's first slot is always a new token's.
// (With a wave for all pages of a request one of a million tokens took 110 us, now 10.5; 2^20 requests of one token 205, now 40.)
constexpr uint64_t kManyTokens = 1u << 20;
constexpr int kMaxPlans = (int)(kMaxSeqs / kPlanThreads);
constexpr uint64_t kManyRequests = 16384;

// n entries of `from`, in steps of `step` (1 or -1), to `to`, by LANES neighbouring threads with eight in flight.
template <int32_t LANES = kPageLanes>
__device__ __forceinline__ void copy_pages(int32_t* to, const int32_t* from, int step, int32_t n) {
    for (int32_t j0 = threadIdx.x % LANES; j0 < n; j0 += 8 * LANES) {
        int32_t page[8];
#pragma unroll
        for (int k = 0; k < 8; k++) page[k] = from[step * (j0 + LANES * k < n ? j0 + LANES * k : j0)];
#pragma unroll
        for (int k = 0; k < 8; k++) if (j0 + LANES * k < n) to[j0 + LANES * k] = page[k];
    }
}
// Places in a list for the lanes that want one; called by whole waves.
__device__ __forceinline__ uint32_t list_place(bool want, uint32_t* count) {
    const u64 m = __ballot(want);
    uint32_t at = 0;
    if (m && lane_id() == 0) at = atomicAdd(count, (uint32_t)__popcll(m));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + (uint32_t)__popcll(m & ((1ull << lane_id()) - 1));
}

template <int PER>
__global__ __launch_bounds__(kApplyThreads) void cache_slots_kernel(CacheArgs A, PageDiv D, const PlanRec* recs, const u64* blocks,
                                                                    const CacheHead* head, uint64_t request_blocks, uint32_t per_request_block) {
    constexpr int kTokenBlock = kApplyThreads * PER, kOwners = kTokenBlock;
    __shared__ u64 tmp[kApplyWaves];
    __shared__ Owner owners[kOwners];
    __shared__ uint64_t ends[2];
    __shared__ uint32_t s_many, many_of[kApplyThreads];
    static_assert(kOwners >= kApplyThreads, "the list of requests with many pages lies there too");
    const uint64_t left = head->left;
    uint32_t bits = 0;
    if (blockIdx.x == 0) {
        const u64 taken = pages_served(recs, blocks, A.n, left, tmp);
        if (threadIdx.x == 0) { const int32_t n = *A.n_free; *A.n_free_out = head->bad ? n : n - (int32_t)taken; }
        return;
    }
    if (blockIdx.x <= request_blocks) {  // a thread per request: its new state, and its new pages into the table
        const uint64_t i0 = (uint64_t)(blockIdx.x - 1) * per_request_block, i = i0 + threadIdx.x;   // (it divides kPlanThreads)
        if (threadIdx.x == 0) s_many = 0;
        const bool mine = threadIdx.x < per_request_block && i < A.n;
        const PlanRec r = recs[mine ? i : i0];
        const u64 before = pages_before(blocks, i0 / kPlanThreads, tmp) + r.before;   // (barriers inside)
        const bool served = mine && slots_served_within(A, r, before, left);
        if (mine) {
            A.len_out[i] = served ? r.new_len : r.len;
            A.held_out[i] = served ? r.held + r.delta : r.held;
            bits = served ? 0u : r.flags ? r.flags : (uint32_t)kCachePool;
        }
        if (served && r.delta) {
            int32_t* to = A.table + i * A.table_stride + r.held;
            const int32_t* from = A.free_pages + (left - before) - 1;
            int32_t page[kFirstPages];
#pragma unroll
            for (int32_t j = 0; j < kFirstPages; j++) page[j] = *(from - (j < r.delta ? j : 0));
#pragma unroll
            for (int32_t j = 0; j < kFirstPages; j++) if (j < r.delta) to[j] = page[j];
        }
        const bool more = served && r.delta > kFirstPages;
        const uint32_t at = list_place(more, &s_many);
        if (more) {
            owners[at].next = (uint32_t)(left - before);
            owners[at].held = r.held;
            owners[at].len = r.delta;
            many_of[at] = threadIdx.x;
        }
        __syncthreads();
        for (uint32_t x = threadIdx.x / kPageLanes; x < s_many; x += kApplyThreads / kPageLanes) {
            const int32_t n = owners[x].len < kGroupPages ? owners[x].len : kGroupPages;
            copy_pages(A.table + (i0 + many_of[x]) * A.table_stride + owners[x].held + kFirstPages, A.free_pages + owners[x].next - 1 - kFirstPages, -1, n - kFirstPages);
        }
    } else {
        const uint64_t t0 = (uint64_t)(blockIdx.x - 1 - request_blocks) * kTokenBlock;
        uint64_t total = A.off[A.n];
        const uint64_t probe = request_probe(A.off, A.n), first = first_lane64(probe);   // (lane 0 has loaded off[0])
        if (total > A.cap) total = A.cap;
        if (t0 >= total) return;
        const uint64_t last = (t0 + kTokenBlock < total ? t0 + kTokenBlock : total) - 1;
        constexpr int kPer = kMaxPlans / kApplyThreads;
        const uint64_t n_plans = (A.n + kPlanThreads - 1) / kPlanThreads;
        u64 sums[kPer], base = 0;              // (on their way while the requests are looked for)
#pragma unroll
        for (int k = 0; k < kPer; k++) {
            const uint64_t b = (uint64_t)k * kApplyThreads + threadIdx.x;
            sums[k] = b < n_plans ? blocks[b] : 0;
        }
        // the first two waves find the first and the last request of the block
        if (wave_id() < 2) ends[wave_id()] = request_of(A.off, A.n, wave_id() ? last : t0, probe);
        __syncthreads();
        const uint64_t a0 = ends[0], a1 = ends[1], many = a1 >= a0 ? a1 - a0 + 1 : kOwners + 1;
        const uint64_t b0 = many <= kOwners ? a0 / kPlanThreads : 0;
#pragma unroll
        for (int k = 0; k < kPer; k++) if ((uint64_t)k * kApplyThreads + threadIdx.x < b0) base += sums[k];
        if (b0) base = apply_sum64(base, tmp);
        auto load_owner = [&](uint64_t i) {
            u64 before = base;
            for (uint64_t b = b0; b < i / kPlanThreads; b++) before += blocks[b];
            const PlanRec r = recs[i];
            return owner_of(A, r, A.off[i], A.off[i + 1], before + r.before, left);
        };
        const uint64_t t = t0 + (uint64_t)threadIdx.x * PER;
        int64_t slot[PER];
        int32_t pos[PER];
        bool stays[PER];
        if (many <= kOwners) {
            for (uint64_t k = threadIdx.x; k < many; k += kApplyThreads) owners[k] = load_owner(a0 + k);
            __syncthreads();
            uint32_t k = 0, e = (uint32_t)many;
            while (e - k > 1) { const uint32_t m = (k + e) / 2; if (owners[m].first <= t) k = m; else e = m; }
#pragma unroll
            for (int j = 0; j < PER; j++) {
                while (k + 1 < (uint32_t)many && owners[k + 1].first <= t + j) k++;
                stays[j] = not_the_calls(first, owners[k], t + j);
                if (t + j <= last) bits |= place_token<true>(A, D, owners[k], a0 + k, t + j, &slot[j], &pos[j]);
            }
        } else {
            for (int j = 0; j < PER; j++) {
                uint64_t a = 0, b = A.n;
                while (b - a > 1) { const uint64_t m = (a + b) / 2; if (A.off[m] <= t + j) a = m; else b = m; }
                const Owner w = load_owner(a);
                stays[j] = not_the_calls(first, w, t + j);
                if (t + j <= last) bits |= place_token<true>(A, D, w, a, t + j, &slot[j], &pos[j]);
            }
        }
        if (t >= first && t + PER <= last + 1) {
            __builtin_memcpy(A.slots + t, slot, sizeof slot);
            __builtin_memcpy(A.pos + t, pos, sizeof pos);
        } else {
            for (int j = 0; j < PER; j++) if (t + j <= last && !stays[j]) { A.slots[t + j] = slot[j]; A.pos[t + j] = pos[j]; }
        }
    }
    if (bits) atomicOr(A.status, bits);
}

// The request that page g of a call belongs to: the last one with before <= g.  (Requests in front of it that take no page share
// its `before`, those behind it have at least g + 1.  g is smaller than the pages of those that are served, and up to there
// `before` ascends.)
__device__ __forceinline__ uint32_t request_of_page(const uint32_t* before, uint32_t n, uint32_t g) {
    uint32_t k = 0, e = n;
    while (e - k > 1) { const uint32_t m = (k + e) / 2; if (before[m] <= g) k = m; else e = m; }
    return k;
}

// The sums up to and with each request ascend: the wave's last request that is served has its largest.  (One atomic a wave: with one
// from every lane on the same word the compiler walks through the lanes.)
__device__ __forceinline__ void pages_of_wave(bool served, u64 upto, uint32_t* most) {
    const u64 m = __ballot(served);
    if (m && lane_id() == 63 - __builtin_clzll(m)) atomicMax(most, (uint32_t)upto);
}

// The whole step in one workgroup: a thread for each request, and at most kOneTokens tokens.  What bounds it is
// latency -- three dependent loads and two barriers -- so no more waves are started than the requests need.
constexpr uint64_t kOneTokens = 4096;   // (a workgroup of 1,024 has them in four turns, which take less than a second launch)
constexpr int kOneSmall = 256;

template <int THREADS>
__global__ __launch_bounds__(THREADS) void cache_slots_one_kernel(CacheArgs A, PageDiv D) {
    __shared__ u64 tmp[THREADS / 64];
    __shared__ Owner owners[THREADS];
    __shared__ uint32_t s_before[THREADS], s_status, s_taken;
    const uint64_t i = threadIdx.x;
    const int32_t n_free = *A.n_free;
    const bool bad = n_free < 0 || (uint32_t)n_free > A.n_pages;
    const u64 left = bad ? 0 : (u64)n_free;
    if (threadIdx.x == 0) { s_status = bad ? (uint32_t)kCacheBad : 0u; s_taken = 0; }
    PlanRec r{};
    uint64_t first = 0, end = 0, total = 0;
    if (A.n) total = A.off[A.n];
    if (i < A.n) {
        first = A.off[i];
        end = A.off[i + 1];
        r = plan_slots(A.len[i], A.held[i], first, end, A.cap, A.page, A.max_pages);
    }
    u64 all;
    const u64 before = block_escan64<THREADS>((u64)r.delta, tmp, &all);   // (barriers inside: nobody's state is read behind it)
    bool takes = false;
    if (i < A.n) {
        const bool served = slots_served(r, before, left);
        takes = served && r.delta;
        owners[i] = owner_of(A, r, first, end, before, left);
        s_before[i] = (uint32_t)before;   // (a request asks for at most kOneTokens pages)
        A.len_out[i] = served ? r.new_len : r.len;
        A.held_out[i] = served ? r.held + r.delta : r.held;
        if (!served) atomicOr(&s_status, r.flags ? r.flags : (uint32_t)kCachePool);
    }
    pages_of_wave(takes, before + (u64)r.delta, &s_taken);
    __syncthreads();
    const uint32_t taken = s_taken;
    for (uint32_t g = threadIdx.x; g < taken; g += THREADS) {   // new pages into the table
        const uint32_t k = request_of_page(s_before, (uint32_t)A.n, g);
        A.table[k * A.table_stride + (uint32_t)owners[k].held + (g - s_before[k])] = A.free_pages[left - 1 - g];
    }
    if (total > A.cap) total = A.cap;
    for (uint64_t t = threadIdx.x; t < total; t += THREADS) {
        uint32_t k = 0, e = (uint32_t)A.n;
        while (e - k > 1) { const uint32_t m = (k + e) / 2; if (owners[m].first <= t) k = m; else e = m; }
        int64_t slot;
        int32_t pos;
        const uint32_t bits = place_token<false>(A, D, owners[k], k, t, &slot, &pos);
        if (not_the_calls(owners[0].first, owners[k], t)) continue;
        A.slots[t] = slot;
        A.pos[t] = pos;
        if (bits) atomicOr(&s_status, bits);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        *A.n_free_out = bad ? n_free : n_free - (int32_t)taken;
        *A.status = s_status;
    }
}

// A wave per request: its new state, and the pages it gives back to the end of the free list.
__global__ __launch_bounds__(kApplyThreads) void cache_trim_kernel(CacheArgs A, const PlanRec* recs, const u64* blocks, const CacheHead* head) {
    __shared__ u64 tmp[kApplyThreads / 64];
    const uint64_t left = head->left;
    if (blockIdx.x == 0) {
        const u64 given = pages_served(recs, blocks, A.n, A.n_pages - left, tmp);
        if (threadIdx.x == 0) { const int32_t n = *A.n_free; *A.n_free_out = head->bad ? n : n + (int32_t)given; }
        return;
    }
    const uint64_t i0 = (uint64_t)(blockIdx.x - 1) * kApplyWaves, i = i0 + wave_id();   // (kApplyWaves divides kPlanThreads)
    const u64 base = pages_before(blocks, i0 / kPlanThreads, tmp);
    if (i >= A.n) return;
    const PlanRec r = recs[i];
    const u64 before = base + r.before;
    const bool served = trim_served_within(A, r, before, left);
    if (lane_id() == 0) {
        A.len_out[i] = served ? r.new_len : r.len;
        A.held_out[i] = served ? r.held - r.delta : r.held;
        if (!served) atomicOr(A.status, r.flags ? r.flags : (uint32_t)kCachePool);
    }
    if (!served) return;
    const int32_t* from = A.table + i * A.table_stride + (r.held - r.delta);
    int32_t* to = A.free_pages + left + before;
    for (int32_t j = lane_id(); j < r.delta; j += 64) to[j] = from[j];
}

// The whole call in one workgroup: a thread for each request, which moves the first pages the request gives back itself -- after
// drafts that were not accepted there are no more --, then sixteen lanes for each request that gives more, eight pages each in flight,
// and all threads for one that gives more than kLongPages.  By sixteen lanes / by all threads, us: one request of 131,072 pages 410 /
// 14.5, 16 of 8,192 33 / 16, but 64 of 2,048 17 / 37 (most of the threads have nothing to do).
//
// In one workgroup / in two launches, us on the GPU (and 4 us less for the caller, who makes one launch): 256 requests that give
// nothing 3.4 / 5.2, of which a tenth gives 512 pages 5.9 / 6.2, of which all do 17.4 / 6.3; 1,024 requests 3.8 / 5.9, a tenth of which
// give 128 pages 5.7 / 6.3, all 20.7 / 6.5; 1,000 that all give 131 pages 23.4 / 6.5; 64 that all give 2,048 16.9 / 8.8; one that gives
// 131,072 14.5 / 218.  A step after drafts is the first of these, and a batch that ends at once is rare and costs 17 us at most.
constexpr uint64_t kOnePages = 131072, kOnePagesSmall = 1024;   // pages that the requests hold at the very most
constexpr int32_t kLongPages = 4096;                             // (at most 31 requests of a call give more)

template <int THREADS>
__global__ __launch_bounds__(THREADS) void cache_trim_one_kernel(CacheArgs A) {
    __shared__ u64 tmp[THREADS / 64];
    __shared__ uint32_t s_before[THREADS], s_many[THREADS], s_status, s_given, s_n_many, s_n_long;
    __shared__ int32_t s_first[THREADS], s_delta[THREADS];
    const uint64_t i = threadIdx.x;
    const int32_t n_free = *A.n_free;
    const bool bad = n_free < 0 || (uint32_t)n_free > A.n_pages;
    const u64 left = bad ? A.n_pages : (u64)n_free;
    if (threadIdx.x == 0) { s_status = bad ? (uint32_t)kCacheBad : 0u; s_given = 0; s_n_many = 0; s_n_long = 0; }
    PlanRec r{};
    if (i < A.n) r = plan_trim(A.len[i], A.held[i], A.keep[i], A.page, A.max_pages);
    u64 all;
    const u64 before = block_escan64<THREADS>((u64)r.delta, tmp, &all);   // (at most kOnePages pages)
    bool gives = false;
    if (i < A.n) {
        const bool served = trim_served(r, before, left, A.n_pages);
        gives = served && r.delta;
        A.len_out[i] = served ? r.new_len : r.len;
        A.held_out[i] = served ? r.held - r.delta : r.held;
        if (!served) atomicOr(&s_status, r.flags ? r.flags : (uint32_t)kCachePool);
    }
    pages_of_wave(gives, before + (u64)r.delta, &s_given);
    const int32_t stay = r.held - r.delta;
    if (gives) {
        const int32_t* from = A.table + i * A.table_stride + stay;
        int32_t* to = A.free_pages + left + before;
        int32_t page[kFirstPages];
#pragma unroll
        for (int32_t j = 0; j < kFirstPages; j++) page[j] = from[j < r.delta ? j : 0];
#pragma unroll
        for (int32_t j = 0; j < kFirstPages; j++) if (j < r.delta) to[j] = page[j];
    }
    const bool many = gives && r.delta > kFirstPages, longer = gives && r.delta > kLongPages;   // (the longer ones from the list's end)
    const uint32_t place = list_place(many && !longer, &s_n_many), from_end = list_place(longer, &s_n_long);
    if (many) {
        const uint32_t at = longer ? THREADS - 1 - from_end : place;
        s_many[at] = (uint32_t)i;
        s_before[at] = (uint32_t)before + kFirstPages;
        s_first[at] = stay + kFirstPages;
        s_delta[at] = r.delta - kFirstPages;
    }
    __syncthreads();
    for (uint32_t x = threadIdx.x / kPageLanes; x < s_n_many; x += THREADS / kPageLanes)
        copy_pages(A.free_pages + left + s_before[x], A.table + (uint64_t)s_many[x] * A.table_stride + s_first[x], 1, s_delta[x]);
    for (uint32_t x = THREADS - s_n_long; x < THREADS; x++)
        copy_pages<THREADS>(A.free_pages + left + s_before[x], A.table + (uint64_t)s_many[x] * A.table_stride + s_first[x], 1, s_delta[x]);
    if (threadIdx.x == 0) {
        *A.n_free_out = bad ? n_free : n_free + (int32_t)s_given;
        *A.status = s_status;
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
    const PageDiv D = page_div(A.page);
    if (A.n <= kOneSmall && A.cap <= kOneTokens / 4) return launch(cache_slots_one_kernel<kOneSmall>, 1, kOneSmall, stream, A, D);
    if (A.n <= kPlanThreads && A.cap <= kOneTokens) return launch(cache_slots_one_kernel<kPlanThreads>, 1, kPlanThreads, stream, A, D);
    const Parts P = parts_of(A);
    hipError_t e = launch(cache_plan_kernel<false>, P.plan_blocks, kPlanThreads, stream, A, P.recs, P.blocks, P.head);
    if (e != hipSuccess) return e;
    const uint32_t per_request_block = A.n < kManyRequests ? 16 : kApplyThreads;
    const bool many = A.cap >= kManyTokens;
    const uint64_t request_blocks = (A.n + per_request_block - 1) / per_request_block, token_block = (uint64_t)kApplyThreads * (many ? 4 : 2);
    const uint64_t token_blocks = A.n ? (A.cap + token_block - 1) / token_block : 0;
    return launch(many ? cache_slots_kernel<4> : cache_slots_kernel<2>, 1 + request_blocks + token_blocks, kApplyThreads, stream, A, D, (const PlanRec*)P.recs,
                  (const u64*)P.blocks, (const CacheHead*)P.head, request_blocks, per_request_block);
}

hipError_t launch_cache_trim(const CacheArgs& A, hipStream_t stream) {
    if (A.n <= kOneSmall && A.n * A.max_pages <= kOnePagesSmall) return launch(cache_trim_one_kernel<kOneSmall>, 1, kOneSmall, stream, A);
    if (A.n <= kPlanThreads && A.n * A.max_pages <= kOnePages) return launch(cache_trim_one_kernel<kPlanThreads>, 1, kPlanThreads, stream, A);
    const Parts P = parts_of(A);
    hipError_t e = launch(cache_plan_kernel<true>, P.plan_blocks, kPlanThreads, stream, A, P.recs, P.blocks, P.head);
    if (e != hipSuccess) return e;
    return launch(cache_trim_kernel, 1 + (A.n + kApplyWaves - 1) / kApplyWaves, kApplyThreads, stream, A, (const PlanRec*)P.recs, (const u64*)P.blocks, (const CacheHead*)P.head);
}

}  // namespace l3
