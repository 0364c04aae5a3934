// l3_token_ops.h -- the operators on token ids that stand on either side of a model (l3_embed.hip, l3_cache.hip,
// l3_verify.hip): their arguments, the checks the C ABI makes of them, the sizes of their workspaces and the arithmetic of
// one request.  Plain C++ (the CPU test-suite compiles it too, l3_token_hosttest.cpp).
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "l3_common.h"

namespace l3 {

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };   // L3_F32, L3_F16, L3_BF16
L3_HD int dtype_size(int t) { return t == kF32 ? 4 : 2; }

constexpr uint64_t kMaxCount = 0x7FFFFFFFull;    // ids, rows, tokens, pages: 31 bits
constexpr uint64_t kMaxDim = 1ull << 24;
// Ids sorted in one call.  Every tile adds up the counts of all tiles before it, which is cheap up to about 2^20 ids and grows with
// their square: 64 columns in 16 bits, us: 2^18 ids 85, 2^20 178, 2^22 709, 2^24 4,926.
constexpr uint64_t kMaxGradIds = 1ull << 24;
constexpr uint64_t kMaxGradRows = 1ull << 28;    // rows of a gradient: one workgroup for 32 of them
constexpr uint64_t kMaxSeqs = 1ull << 20;
constexpr uint64_t kMaxStride = kMaxCount;       // elements: (2^31 - 1) rows of (2^31 - 1) elements of 4 bytes stay inside 64 bits

struct EmbedArgs {
    const int32_t* ids; uint64_t n; const uint64_t* n_dev;   // n_dev (optional): only the first *n_dev ids count
    const void* table; int dtype; uint64_t rows, dim, stride;
    void* out; int out_dtype; uint64_t out_stride;
    float scale;
};

struct EmbedGradArgs {
    const int32_t* ids; uint64_t n; const uint64_t* n_dev;
    const void* grad; int dtype; uint64_t grad_stride;
    uint64_t rows, dim;
    void* table; int table_dtype; uint64_t table_stride;
    float scale; int accumulate;
    void* work; uint64_t work_bytes;
};

struct CacheArgs {
    const uint64_t* off;       // slots: n + 1 offsets of the new tokens; trim: null
    const int32_t* keep;       // trim: n lengths; slots: null
    uint64_t n;
    const int32_t* len; const int32_t* held;
    uint32_t page, n_pages;
    int32_t* table; uint64_t table_stride, max_pages;
    int32_t* free_pages;       // trim writes it
    const int32_t* n_free;
    int32_t* len_out; int32_t* held_out; int32_t* n_free_out;
    int64_t* slots; int32_t* pos; uint64_t cap;
    uint32_t* status;
    void* work; uint64_t work_bytes;
};

struct VerifyArgs {
    const int32_t* draft; const uint64_t* off; uint64_t n, n_draft; uint32_t max_draft;
    const void* target; int dtype; uint64_t target_stride;
    const void* q; uint64_t q_stride;                        // null: the drafted tokens were certain
    uint64_t vocab;
    const float* u_accept; const float* u_draw;
    int32_t* out; int32_t* accepted;
    void* work; uint64_t work_bytes;
};

// ---- workspaces ---------------------------------------------------------------------------------------------------
constexpr uint64_t align256(uint64_t b) { return (b + 255) & ~255ull; }

// Ids are sorted by digits of at most kSortBits bits, in tiles of kSortThreads times 1, 2 or 4: small tiles are more workgroups,
// but each adds up the counts of all of them.  Whole gradients of 64 columns by tile (us): 16,384 ids 26 / 30 / 38, 65,536 40 / 42 /
// 50, 262,144 90 / 83 / 86, 2^20 353 / 207 / 173.
constexpr int kSortThreads = 1024, kSortBits = 9, kSortBins = 1 << kSortBits;
inline int sort_rounds(uint64_t n) { return n <= 65536 ? 1 : n <= 262144 ? 2 : 4; }
inline uint64_t sort_tiles(uint64_t n) { const uint64_t t = (uint64_t)kSortThreads * sort_rounds(n); return (n + t - 1) / t; }
// Few ids are not sorted: every position looks for the others of its id by itself, a workgroup for each and 512 columns.  On the GPU,
// us, so / sorted (which is two launches more): 512 ids of 2,048 columns 5 / 16, 1,500 of 2,048 13.1 / 15.8, 768 of 4,096 13.7 / 15.0,
// 1,024 of 4,096 16.9 / 15.6.  The limit on the ids is for batches that are one id throughout, whose rows one workgroup adds up: 2,048
// ids 57 / 16, 4,096 117 / 17.  Up to kRankIds ids are sorted in one launch by counting, more digit by digit (l3_embed.hip has the
// times of both).
constexpr uint64_t kDirectIds = 2048, kDirectBlocks = 6144, kRankIds = 8192;
inline bool grad_direct(uint64_t n, uint64_t dim) { return n <= kDirectIds && n * ((dim + 511) / 512) <= kDirectBlocks; }
// Sorted positions one wave adds up: few enough that there are about kGradWalkers waves, and 8 .. 64.  By kGradWalkers = 1,024 / 2,048 /
// 4,096 / 8,192, us: 65,536 ids of 64 columns 52 / 40 / 39 / 40, of 2,048 168 / 169 / 167 / 160, 16,384 of 2,048 57 / 50 / 51 / 53 (fewer waves
// leave the GPU idle, more leave more parts).
constexpr uint64_t kGradWalkers = 4096;
constexpr int kGradWaves = 4;        // waves of a workgroup
inline uint32_t grad_chunk(uint64_t n, uint64_t dim) {
    const uint64_t want = n * ((dim + 511) / 512) / kGradWalkers;
    uint32_t c = 8;
    while (c < 64 && c < want) c *= 2;
    return c;
}
// The tiles and the parts take up what the largest of all calls of at most n ids and dim columns needs, so that a workspace for the largest
// batch is enough for every smaller one: tiles and chunks double in size where n passes a limit, and what they leave halves.
//   tiles   those of n, or of the limits that n has passed.
//   parts   2 blocks dim8, blocks = ceil(n / (4 chunk)): with the smallest chunk at most 2 ceil(n / 32) dim8.  The largest chunk's grow with
//           n and dim.  A chunk c below it means want <= c, that is n ceil(dim / 512) < (c + 1) kGradWalkers, so n dim8 <= 512 (c + 1)
//           kGradWalkers and blocks dim8 <= n dim8 / (4 c) + dim8 <= 128 (1 + 1 / 8) kGradWalkers + dim8.
inline uint64_t sort_tiles_most(uint64_t n) {
    const uint64_t limits[] = {65536, 262144};
    uint64_t most = sort_tiles(n);
    for (const uint64_t limit : limits) if (n > limit && sort_tiles(limit) > most) most = sort_tiles(limit);
    return most;
}
inline uint64_t grad_parts_most(uint64_t n, uint64_t dim8) {
    const uint64_t few = (n + 8 * kGradWaves - 1) / (8 * kGradWaves) * dim8, many = (n + 64 * kGradWaves - 1) / (64 * kGradWaves) * dim8;
    const uint64_t between = 144 * kGradWalkers + dim8, most = many > between ? many : between;
    return 2 * (few < most ? few : most);
}
struct GradWork { uint64_t keys0, pos0, keys1, pos1, hist, part, total; uint32_t chunk; uint64_t blocks, dim8; };
inline GradWork grad_work(uint64_t n, uint64_t dim) {
    GradWork w;
    w.chunk = grad_chunk(n, dim);
    w.blocks = (n + kGradWaves * w.chunk - 1) / (kGradWaves * w.chunk);
    w.dim8 = (dim + 7) & ~7ull;
    uint64_t at = 0;
    auto take = [&](uint64_t b) { const uint64_t p = at; at += align256(b); return p; };
    w.keys0 = take(4 * n); w.pos0 = take(4 * n); w.keys1 = take(4 * n); w.pos1 = take(4 * n);
    w.hist = take(sort_tiles_most(n) * kSortBins * 4);
    w.part = take(grad_parts_most(n, w.dim8) * 4);
    w.total = at ? at : 256;
    return w;
}

constexpr int kPlanThreads = 1024;
struct PlanRec {
    uint64_t before;         // pages that the requests before it in its block of kPlanThreads ask for (or give back)
    int32_t len, held;       // as they were
    int32_t delta;           // pages it asks for (or gives back)
    int32_t new_len;
    uint32_t flags, pad;     // kCache* bits that keep it from being served
};
struct CacheWork { uint64_t recs, blocks, head, total; };
inline CacheWork cache_work(uint64_t n) {
    CacheWork w;
    uint64_t at = 0;
    auto take = [&](uint64_t b) { const uint64_t p = at; at += align256(b); return p; };
    w.head = take(16);
    w.recs = take(n * sizeof(PlanRec));
    w.blocks = take(((n + kPlanThreads - 1) / kPlanThreads) * 8);
    w.total = at;
    return w;
}

constexpr int kVerifyChunk = 2048;   // entries of a row one workgroup adds up
// What became of a request's drafted tokens: all accepted, or token `a` rejected.
enum : int { kBadRequest = 0, kDrawTarget = 1, kDrawRest = 2 };
struct VerifyVerdict { int32_t state; uint32_t a; uint64_t p_row, q_row; int32_t token; int32_t pad; };
struct VerifyWork { uint64_t sums, verdicts, total, chunks; };
inline VerifyWork verify_work(uint64_t n, uint64_t vocab) {
    VerifyWork w;
    w.chunks = (vocab + kVerifyChunk - 1) / kVerifyChunk;
    w.sums = 0;
    w.verdicts = align256(n * w.chunks * 16);
    w.total = w.verdicts + align256((n ? n : 1) * sizeof(VerifyVerdict));
    return w;
}

// ---- checks: null, or what is wrong -------------------------------------------------------------------------------
inline bool bad_dtype(int t) { return t != kF32 && t != kF16 && t != kBF16; }
inline bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

inline const char* check_embed(const EmbedArgs& A) {
    if (bad_dtype(A.dtype) || bad_dtype(A.out_dtype)) return "unknown element type";
    if (A.n > kMaxCount) return "more than 2^31 - 1 ids: split the call";
    if (A.rows == 0 || A.rows > kMaxCount) return "n_rows must be 1 .. 2^31 - 1";
    if (A.dim == 0 || A.dim > kMaxDim) return "dim must be 1 .. 2^24";
    if (A.stride < A.dim || A.out_stride < A.dim || A.stride > kMaxStride || A.out_stride > kMaxStride) return "a row stride is smaller than dim or above 2^31 - 1";
    if (A.n == 0) return nullptr;
    if (!A.ids || !A.table || !A.out) return "null pointer argument";
    if (misaligned(A.ids, 4) || misaligned(A.n_dev, 8) || misaligned(A.table, dtype_size(A.dtype)) || misaligned(A.out, dtype_size(A.out_dtype)))
        return "a pointer is not aligned to its element";
    return nullptr;
}

inline const char* check_embed_grad(const EmbedGradArgs& A) {
    if (bad_dtype(A.dtype) || bad_dtype(A.table_dtype)) return "unknown element type";
    if (A.n > kMaxGradIds) return "more than 2^24 ids: split the call";
    if (A.rows == 0 || A.rows > kMaxGradRows) return "n_rows must be 1 .. 2^28";
    if (A.dim == 0 || A.dim > kMaxDim) return "dim must be 1 .. 2^24";
    if (A.grad_stride < A.dim || A.table_stride < A.dim || A.grad_stride > kMaxStride || A.table_stride > kMaxStride)
        return "a row stride is smaller than dim or above 2^31 - 1";
    if (A.accumulate != 0 && A.accumulate != 1) return "accumulate must be 0 or 1";
    if (!A.table) return "null pointer argument";
    if (misaligned(A.table, dtype_size(A.table_dtype)) || misaligned(A.n_dev, 8)) return "a pointer is not aligned to its element";
    if (A.n == 0) return nullptr;
    if (!A.ids || !A.grad || !A.work) return "null pointer argument";
    if (misaligned(A.ids, 4) || misaligned(A.grad, dtype_size(A.dtype))) return "a pointer is not aligned to its element";
    if (misaligned(A.work, 16)) return "the workspace must be aligned to 16 bytes";
    if (A.work_bytes < grad_work(A.n, A.dim).total) return "workspace too small (l3_embed_grad_workspace)";
    return nullptr;
}

inline const char* check_cache(const CacheArgs& A, bool trim) {
    if (A.n > kMaxSeqs) return "more than 2^20 requests: split the call";
    if (A.page == 0 || A.page > (1u << 20)) return "page_size must be 1 .. 2^20";
    if (A.n_pages == 0 || A.n_pages > kMaxCount) return "n_pages must be 1 .. 2^31 - 1";
    if (A.max_pages == 0 || A.max_pages > kMaxCount) return "max_pages must be 1 .. 2^31 - 1";
    if (A.table_stride < A.max_pages || A.table_stride > kMaxStride) return "table_stride is smaller than max_pages or above 2^31 - 1";
    if (A.cap > kMaxCount) return "cap must be at most 2^31 - 1";
    if (!A.n_free || !A.n_free_out || !A.status) return "null pointer argument";
    if (misaligned(A.n_free, 4) || misaligned(A.n_free_out, 4) || misaligned(A.status, 4)) return "a pointer is not aligned to its element";
    if (!A.free_pages || misaligned(A.free_pages, 4)) return A.free_pages ? "a pointer is not aligned to its element" : "null pointer argument";
    if (!A.work) return "null pointer argument";
    if (misaligned(A.work, 16)) return "the workspace must be aligned to 16 bytes";
    if (A.work_bytes < cache_work(A.n).total) return "workspace too small (l3_cache_workspace)";
    if (!trim && (!A.off || misaligned(A.off, 8))) return A.off ? "a pointer is not aligned to its element" : "null pointer argument";
    if (!trim && A.cap && (!A.slots || !A.pos)) return "null pointer argument";
    if (!trim && (misaligned(A.slots, 8) || misaligned(A.pos, 4))) return "a pointer is not aligned to its element";
    if (A.n == 0) return nullptr;
    if (!A.len || !A.held || !A.table || !A.len_out || !A.held_out || (trim && !A.keep)) return "null pointer argument";
    if (misaligned(A.len, 4) || misaligned(A.held, 4) || misaligned(A.table, 4) || misaligned(A.len_out, 4) || misaligned(A.held_out, 4) || misaligned(A.keep, 4))
        return "a pointer is not aligned to its element";
    return nullptr;
}

inline const char* check_verify(const VerifyArgs& A) {
    if (bad_dtype(A.dtype)) return "unknown element type";
    if (A.n > kMaxSeqs) return "more than 2^20 requests: split the call";
    if (A.n_draft > kMaxCount) return "more than 2^31 - 1 drafted tokens: split the call";
    if (A.max_draft > 65535) return "max_draft must be at most 65,535";
    if (A.vocab == 0 || A.vocab > kMaxCount) return "vocab must be 1 .. 2^31 - 1";
    if (A.target_stride < A.vocab || A.target_stride > kMaxStride || (A.q && (A.q_stride < A.vocab || A.q_stride > kMaxStride)))
        return "a row stride is smaller than vocab or above 2^31 - 1";
    if (A.n == 0) return nullptr;
    if (!A.off || !A.target || !A.u_draw || !A.out || !A.accepted || !A.work) return "null pointer argument";
    if (A.n_draft && (!A.draft || !A.u_accept)) return "null pointer argument";
    if (misaligned(A.off, 8) || misaligned(A.draft, 4) || misaligned(A.u_accept, 4) || misaligned(A.u_draw, 4) || misaligned(A.out, 4) ||
        misaligned(A.accepted, 4) || misaligned(A.target, dtype_size(A.dtype)) || misaligned(A.q, dtype_size(A.dtype)))
        return "a pointer is not aligned to its element";
    if (misaligned(A.work, 16)) return "the workspace must be aligned to 16 bytes";
    if (A.work_bytes < verify_work(A.n, A.vocab).total) return "workspace too small (l3_verify_workspace)";
    return nullptr;
}

// ---- one request of the paged cache -------------------------------------------------------------------------------
enum : uint32_t {
    kCachePool = 1,   // L3_CACHE_POOL: the pool ran short (trim: it would hold more pages than there are)
    kCacheRow = 2,    // L3_CACHE_ROW: more tokens than max_pages pages hold
    kCacheBad = 4,    // L3_CACHE_BAD: offsets, lengths or counts that cannot be
    kCachePage = 8,   // L3_CACHE_PAGE: a page outside the pool
};

L3_HD bool sane_request(int32_t len, int32_t held, uint32_t page, uint64_t max_pages) {
    return len >= 0 && held >= 0 && (uint64_t)held <= max_pages && (uint64_t)len <= (uint64_t)held * page;
}
// Tokens [a, b) are new: pages it needs beyond those it holds.
L3_HD PlanRec plan_slots(int32_t len, int32_t held, uint64_t a, uint64_t b, uint64_t cap, uint32_t page, uint64_t max_pages) {
    PlanRec r;
    r.before = 0; r.len = len; r.held = held; r.delta = 0; r.new_len = len; r.flags = 0; r.pad = 0;
    if (a > b || b > cap || !sane_request(len, held, page, max_pages)) { r.flags = kCacheBad; return r; }
    const uint64_t end = (uint64_t)len + (b - a);
    if (b == a) return r;
    if (end > max_pages * page || end > kMaxCount) { r.flags = kCacheRow; return r; }
    const uint32_t pages = ((uint32_t)end + page - 1) / page;   // (below 2^31 + 2^20)
    r.delta = pages > (uint32_t)held ? (int32_t)(pages - (uint32_t)held) : 0;
    r.new_len = (int32_t)end;
    return r;
}
// keep < 0: left as it is; else it keeps min(keep, len) tokens and the pages these need.
L3_HD PlanRec plan_trim(int32_t len, int32_t held, int32_t keep, uint32_t page, uint64_t max_pages) {
    PlanRec r;
    r.before = 0; r.len = len; r.held = held; r.delta = 0; r.new_len = len; r.flags = 0; r.pad = 0;
    if (keep < 0) return r;
    if (!sane_request(len, held, page, max_pages)) { r.flags = kCacheBad; return r; }
    r.new_len = keep < len ? keep : len;
    r.delta = held - (int32_t)(((uint32_t)r.new_len + page - 1) / page);
    return r;
}
// Is it served?  `before`: pages the requests before it ask for / give back; `left`: pages in the pool.
L3_HD bool slots_served(const PlanRec& r, uint64_t before, uint64_t left) {
    return r.flags == 0 && (r.delta == 0 || before + (uint64_t)r.delta <= left);
}
L3_HD bool trim_served(const PlanRec& r, uint64_t before, uint64_t left, uint64_t n_pages) {
    return r.flags == 0 && (r.delta == 0 || left + before + (uint64_t)r.delta <= n_pages);
}
// A record of the plan that would lead outside the table or the pool is not served.  The plan makes none; a workspace that two
// calls share by mistake may hold anything.
L3_HD bool kept_within(const CacheArgs& A, const PlanRec& r, bool trim, uint64_t before, uint64_t left) {
    if (r.held < 0 || r.delta < 0 || left > A.n_pages || (uint64_t)r.held + (trim ? 0u : (uint32_t)r.delta) > A.max_pages) return false;
    const uint64_t most = trim ? A.n_pages - left : left;
    return r.delta == 0 || ((!trim || r.delta <= r.held) && before <= most && (uint64_t)r.delta <= most - before);
}
L3_HD bool slots_served_within(const CacheArgs& A, const PlanRec& r, uint64_t before, uint64_t left) {
    return slots_served(r, before, left) && kept_within(A, r, false, before, left);
}
L3_HD bool trim_served_within(const CacheArgs& A, const PlanRec& r, uint64_t before, uint64_t left) {
    return trim_served(r, before, left, A.n_pages) && (r.delta == 0 || kept_within(A, r, true, before, left));   // (one left alone may hold anything)
}
// What a token needs of its request (tokens and pages are below 2^31; an offset that is not is the largest number instead).
struct Owner {
    uint32_t first, end;     // its new tokens
    uint32_t next;           // free list: its first new page is at next - 1
    int32_t len, held;       // held < 0: not served
};
L3_HD Owner owner_of(const CacheArgs& A, const PlanRec& r, uint64_t first, uint64_t end, uint64_t before, uint64_t left) {
    // (its tokens end within its pages, so that none of them need be looked at by itself)
    const uint64_t count = end - first, upto = (uint64_t)r.len + count;
    const bool served = slots_served_within(A, r, before, left) && r.len >= 0 && end >= first && count <= kMaxCount && upto <= kMaxCount &&
                        upto <= ((uint64_t)r.held + (uint64_t)r.delta) * A.page;
    Owner w;
    w.first = first < ~0u ? (uint32_t)first : ~0u;
    w.end = end < ~0u ? (uint32_t)end : ~0u;
    w.next = served ? (uint32_t)(left - before) : 0;
    w.len = r.len;
    w.held = served ? r.held : -1;
    return w;
}
L3_HD bool owns(const Owner& w, uint64_t t) { return t >= w.first && t < w.end; }
// The same for the verification: a verdict is held to the rows there are.
L3_HD bool verdict_within(const VerifyArgs& A, const VerifyVerdict& R) {
    return R.a <= A.max_draft && R.p_row < A.n_draft + A.n && (R.state != kDrawRest || R.q_row < A.n_draft);
}
// x / page for x < 2^31 by a product: with 2^s the first power of two that is not below page, m = floor(2^(31 + s) / page) + 1 is
// 2^(31 + s) / page + e, 0 < e <= 1, so x m / 2^(31 + s) is x / page + x e / 2^(31 + s), too large by less than 2^-s <= 1 / page.
struct PageDiv {
    uint32_t m, shift;
    L3_HD uint32_t of(uint32_t x) const { return (uint32_t)(((uint64_t)x * m) >> shift); }
};
inline PageDiv page_div(uint32_t page) {
    uint32_t s = 0;
    while ((1u << s) < page) s++;
    return {(uint32_t)((1ull << (31 + s)) / page + 1), 31 + s};
}
L3_HD int64_t slot_of(int32_t page_id, uint32_t in_page, uint32_t page, uint32_t n_pages) {
    if (page_id < 0 || (uint32_t)page_id >= n_pages) return -1;
    return (int64_t)page_id * page + in_page;
}

}  // namespace l3
