// paged.cuh -- what the operators on a paged key/value cache share: the device view of
// the cache, its checks, and the lookup of a packed token's sequence.
#pragma once
#include "common.cuh"

namespace gdn {

// gdn_paged_cache as the kernels take it
struct PagedView {
    uint16_t* k;
    uint16_t* v;
    const int* table;
    long table_ld, page_stride, token_stride, head_stride;
    int num_pages, page_shift, max_pages, n_kv;
};

inline int check_cache(const char* name, const gdn_paged_cache* c, PagedView* v) {
    if (!c || !c->k || !c->v || !c->block_table)
        return fail(GDN_ERR_NULL, "%s: the cache's k, v and block_table are required", name);
    if (c->num_pages < 1 || c->max_pages < 1 || c->n_kv < 1 || c->table_ld < c->max_pages)
        return fail(GDN_ERR_SHAPE, "%s: the cache needs pages, table entries and kv heads (num_pages=%d max_pages=%d "
                                   "table_ld=%ld n_kv=%d)", name, c->num_pages, c->max_pages, c->table_ld, c->n_kv);
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) != 0)
        return fail(GDN_ERR_SHAPE, "%s: page_size must be a power of two, at least 16 (got %d)", name, c->page_size);
    if (c->max_pages > 0x7fffffff / c->page_size)
        return fail(GDN_ERR_SHAPE, "%s: max_pages x page_size exceeds 2^31 positions", name);
    for (long s : {c->page_stride, c->token_stride, c->head_stride})
        if (s <= 0 || s % 8 != 0)
            return fail(GDN_ERR_ALIGN, "%s: cache strides must be positive multiples of 8 elements", name);
    if (!aligned16(c->k) || !aligned16(c->v)) return fail(GDN_ERR_ALIGN, "%s: the cache must be 16-byte aligned", name);
    v->k = static_cast<uint16_t*>(c->k);
    v->v = static_cast<uint16_t*>(c->v);
    v->table = c->block_table;
    v->table_ld = c->table_ld;
    v->page_stride = c->page_stride;
    v->token_stride = c->token_stride;
    v->head_stride = c->head_stride;
    v->num_pages = c->num_pages;
    v->page_shift = 0;
    while ((1 << v->page_shift) < c->page_size) ++v->page_shift;
    v->max_pages = c->max_pages;
    v->n_kv = c->n_kv;
    return GDN_OK;
}

// The sequence of packed token t: the last b in [0, B) with cu[b] <= t (cu[0] taken as 0).
// A warp narrows the range 32-fold per step.
__device__ __forceinline__ int sequence_of(const int* __restrict__ cu, int B, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = B;                         // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) >> 5;
        const int probe = lo + lane * step;
        const bool le = lane == 0 || (lane * step < n && cu[probe] <= t);
        const int hits = __popc(__ballot_sync(0xffffffffu, le));
        lo += (hits - 1) * step;
        n = min(step, B - lo);
    }
    return lo;
}

}  // namespace gdn
