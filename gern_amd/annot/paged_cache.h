// Host mirrors of the aggregates of the gernels over a paged 8-bit cache of keys
// and values (gernels/serving/paged_cache.h, page_table.h, cache_write.h,
// cache_attention.h); the annotations are the general ones of annot/pieces.h.
#pragma once

#include "annot/pieces.h"

#include <cstddef>

namespace gern {
namespace hip {

// Host mirrors (same layout) of the aggregates of the same names in gernels::.
struct PagedCache {
    void *k, *v;
    float *k_scales, *v_scales;
    int64_t pages, heads;
    uint32_t *faults;
};
struct WritableCache : PagedCache {
    int64_t pieces, stretch;
};
struct NewTokens {
    const void *k, *v;
    int64_t k_pitch, v_pitch;
    const int32_t *slots;
    int64_t tokens;
};
struct RequestLengths {
    const int32_t *cached, *added;
    int64_t requests;
};
struct FreePages {
    const int32_t *list, *count;
    int64_t capacity;
};
struct PageTableOut {
    int32_t *table, *lengths, *starts, *slots, *counts;
    int64_t width, tokens, shares;
};

struct AttentionBatch {
    const void *q;
    int64_t q_pitch;
    const int32_t *table, *lengths, *starts;
    int64_t width, tokens, group;
    float scale;
};
struct AttentionOut {
    void *out;
    int64_t out_pitch;
    float *partial, *stats;
    int64_t splits, chunk, pieces, heads, requests;
};
struct JoinRows {
    void *out;
    int64_t out_pitch;
    const float *partial, *stats;
    const int32_t *starts;
    int64_t splits, requests, q_heads, rows, blocks;
};

// The sizes and last members' places that csrc/gernel_check.hip asks of gernels::.
static_assert(sizeof(PagedCache) == 56 && offsetof(PagedCache, faults) == 48);
static_assert(sizeof(WritableCache) == 72);
static_assert(sizeof(NewTokens) == 48 && offsetof(NewTokens, tokens) == 40);
static_assert(sizeof(RequestLengths) == 24 && offsetof(RequestLengths, requests) == 16);
static_assert(sizeof(FreePages) == 24 && offsetof(FreePages, capacity) == 16);
static_assert(sizeof(PageTableOut) == 64 && offsetof(PageTableOut, shares) == 56);
static_assert(sizeof(AttentionBatch) == 72 && offsetof(AttentionBatch, scale) == 64);
static_assert(sizeof(AttentionOut) == 72 && offsetof(AttentionOut, requests) == 64);
static_assert(sizeof(JoinRows) == 80 && offsetof(JoinRows, blocks) == 72);

}  // namespace hip

}  // namespace gern
