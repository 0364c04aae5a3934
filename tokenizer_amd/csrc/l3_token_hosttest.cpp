// l3_token_hosttest.cpp -- host build of l3_token_ops.h and l3_errtext.h for the CPU test-suite (tests/test_token_ops_host.py): the
// checks the C ABI makes of its arguments, the workspace sizes, the error texts, and the paged cache one request after the other
// with the arithmetic the kernels use.  A unit-test shim: nothing in the product calls it.
#include "l3_errtext.h"
#include "l3_token_ops.h"

using namespace l3;

extern "C" {

const char* l3t_check_embed(const EmbedArgs* A) { return check_embed(*A); }
const char* l3t_check_embed_grad(const EmbedGradArgs* A) { return check_embed_grad(*A); }
const char* l3t_check_cache(const CacheArgs* A, int trim) { return check_cache(*A, trim != 0); }
const char* l3t_check_verify(const VerifyArgs* A) { return check_verify(*A); }
uint64_t l3t_grad_work(uint64_t n, uint64_t dim) { return grad_work(n, dim).total; }
// where the counts and the parts of a gradient's workspace end, and where the next piece begins
void l3t_grad_pieces(uint64_t n, uint64_t dim, uint64_t* out) {
    const GradWork w = grad_work(n, dim);
    out[0] = w.hist + sort_tiles(n) * kSortBins * 4;
    out[1] = w.part;
    out[2] = w.part + 2 * w.blocks * w.dim8 * 4;
    out[3] = w.total;
}
uint64_t l3t_cache_work(uint64_t n) { return cache_work(n).total; }
uint64_t l3t_verify_work(uint64_t n, uint64_t vocab) { return verify_work(n, vocab).total; }

ErrText* l3t_err_new() { return new ErrText(); }
void l3t_err_delete(ErrText* e) { delete e; }
void l3t_err_assign(ErrText* e, const char* text) { *e = text; }
void l3t_err_leave(ErrText* e, const char* what, const char* more) { e->leave_for_this_thread(what, more); }
const char* l3t_err_text(const ErrText* e) { return e->c_str(); }

uint32_t l3t_page_div(uint32_t x, uint32_t page) { return page_div(page).of(x); }

// the checks of what a kernel finds in a workspace
int l3t_slots_served_within(const CacheArgs* A, const PlanRec* r, uint64_t before, uint64_t left) { return slots_served_within(*A, *r, before, left); }
int l3t_trim_served_within(const CacheArgs* A, const PlanRec* r, uint64_t before, uint64_t left) { return trim_served_within(*A, *r, before, left); }
void l3t_owner_of(const CacheArgs* A, const PlanRec* r, uint64_t first, uint64_t end, uint64_t before, uint64_t left, Owner* out) {
    *out = owner_of(*A, *r, first, end, before, left);
}
int l3t_verdict_within(const VerifyArgs* A, const VerifyVerdict* R) { return verdict_within(*A, *R); }

void l3t_cache_slots(const CacheArgs* P) {
    const CacheArgs& A = *P;
    const int32_t n_free = *A.n_free;
    const bool bad = n_free < 0 || (uint32_t)n_free > A.n_pages;
    const uint64_t left = bad ? 0 : (uint64_t)n_free;
    uint32_t status = bad ? (uint32_t)kCacheBad : 0u;
    uint64_t before = 0, taken = 0;
    for (uint64_t i = 0; i < A.n; i++) {
        const uint64_t a = A.off[i], b = A.off[i + 1];
        const PlanRec r = plan_slots(A.len[i], A.held[i], a, b, A.cap, A.page, A.max_pages);
        const bool served = slots_served(r, before, left);
        if (!served) status |= r.flags ? r.flags : (uint32_t)kCachePool;
        for (uint64_t t = a; t < b && t < A.cap; t++) {
            A.slots[t] = -1;
            A.pos[t] = -1;
            if (!served) continue;
            const uint32_t pos = (uint32_t)r.len + (uint32_t)(t - a), p = pos / A.page, in = pos % A.page;
            int32_t* entry = A.table + i * A.table_stride + p;
            if (p >= (uint32_t)r.held && in == 0) *entry = A.free_pages[left - 1 - before - (p - (uint32_t)r.held)];
            A.pos[t] = (int32_t)pos;
            A.slots[t] = slot_of(*entry, in, A.page, A.n_pages);
            if (A.slots[t] < 0) status |= kCachePage;
        }
        A.len_out[i] = served ? r.new_len : r.len;
        A.held_out[i] = served ? r.held + r.delta : r.held;
        if (served) taken += (uint64_t)r.delta;
        before += (uint64_t)r.delta;
    }
    *A.n_free_out = bad ? n_free : n_free - (int32_t)taken;
    *A.status = status;
}

void l3t_cache_trim(const CacheArgs* P) {
    const CacheArgs& A = *P;
    const int32_t n_free = *A.n_free;
    const bool bad = n_free < 0 || (uint32_t)n_free > A.n_pages;
    const uint64_t left = bad ? A.n_pages : (uint64_t)n_free;
    uint32_t status = bad ? (uint32_t)kCacheBad : 0u;
    uint64_t before = 0, given = 0;
    for (uint64_t i = 0; i < A.n; i++) {
        const PlanRec r = plan_trim(A.len[i], A.held[i], A.keep[i], A.page, A.max_pages);
        const bool served = trim_served(r, before, left, A.n_pages);
        if (!served) status |= r.flags ? r.flags : (uint32_t)kCachePool;
        if (served) {
            for (int32_t j = 0; j < r.delta; j++) A.free_pages[left + before + (uint64_t)j] = A.table[i * A.table_stride + (uint64_t)(r.held - r.delta + j)];
            given += (uint64_t)r.delta;
        }
        A.len_out[i] = served ? r.new_len : r.len;
        A.held_out[i] = served ? r.held - r.delta : r.held;
        before += (uint64_t)r.delta;
    }
    *A.n_free_out = bad ? n_free : n_free + (int32_t)given;
    *A.status = status;
}

}  // extern "C"
