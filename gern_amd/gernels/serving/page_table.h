// Block tables and slot maps of a batch of requests over a paged cache.
//
// Request b holds cached[b] tokens and adds added[b]; a page holds P tokens:
//
//   length[b] = cached[b] + added[b]
//   need[b]   = ceil(length[b] / P) - ceil(cached[b] / P)      new pages
//   first[b]  = sum of need[c], starts[b] = sum of added[c], c < b
//   table[b, ceil(cached[b] / P) + j] = free[count - 1 - first[b] - j], j < need[b]
//   slot[starts[b] + i] = table[b, p / P] * P + p % P, p = cached[b] + i
//
// A page that the free list no longer has is -1 in the table and its tokens'
// slots are -1, as are the slots behind the last token.
//
// Bound by latency: a decoding step of 256 requests moves 5 KB.  So it is ONE
// launch: every workgroup takes the prefix sums of the whole batch itself
// (8 bytes a request, from L2) instead of waiting for another workgroup's, and
// finds a token's request by bisection in LDS; page numbers of new pages come
// from the free list, not from the table entry that another workgroup may be
// writing.
#pragma once

#include "gernels/serving/paged_cache.h"

namespace gernels {

struct RequestLengths {
    const int32_t *cached, *added;
    int64_t requests;

    __device__ __forceinline__ const RequestLengths &whole() const {
        return *this;
    }
};

struct FreePages {
    const int32_t *list;   // `capacity` page numbers
    const int32_t *count;  // how many of them are free: list[0 .. count)
    int64_t capacity;

    __device__ __forceinline__ const FreePages &whole() const {
        return *this;
    }
};

// What is built.  A subset is the share of one workgroup.
struct PageTableShare;
struct PageTableOut {
    int32_t *table;    // [requests, width]
    int32_t *lengths;  // [requests]
    int32_t *starts;   // [requests + 1]
    int32_t *slots;    // [tokens]
    int32_t *counts;   // pages left in the free list, pages that were missing
    int64_t width;
    int64_t tokens;
    int64_t shares;    // workgroups

    __device__ __forceinline__ PageTableShare share(int64_t x) const;
};
struct PageTableShare {
    const PageTableOut &out;
    int64_t x;
};
__device__ __forceinline__ PageTableShare PageTableOut::share(int64_t x) const {
    return {*this, x};
}

namespace detail {

// Sum over the lanes below this one, and the wavefront's total in lane 63's
// inclusive value.
__device__ __forceinline__ int wave_inclusive_sum(int x) {
    const int lane = lane_id();
    for (int d = 1; d < kWaveSize; d *= 2) {
        const int y = __shfl_up(x, d);
        x += lane >= d ? y : 0;
    }
    return x;
}

// Largest i in [0, n) with sums[i] <= x, for sums that ascend from 0.
__device__ __forceinline__ int last_not_above(const int *sums, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] <= x) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

}  // namespace detail

// THREADS threads, at most THREADS * PER requests.
template<int64_t PAGE, int64_t THREADS, int64_t PER>
__device__ __forceinline__ void extend_page_table(const RequestLengths &batch, const FreePages &free_pages, const PageTableShare &share) {
    constexpr int kWaves = THREADS / kWaveSize;
    __shared__ int starts[THREADS * PER], first[THREADS * PER], held[THREADS * PER];
    __shared__ int wave_added[kWaves], wave_need[kWaves], wave_lack[kWaves];
    const PageTableOut &out = share.out;
    const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWaveSize;
    const int n = (int)batch.requests;

    // Consecutive requests per thread, so that one scan over threads is enough.
    int cached[PER], added[PER], need[PER];
    int sum_added = 0, sum_need = 0, lack = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int b = tid * (int)PER + j;
        // negative lengths count as zero
        cached[j] = b < n ? max(batch.cached[b], 0) : 0;
        added[j] = b < n ? max(batch.added[b], 0) : 0;
        const int64_t before = (cached[j] + PAGE - 1) / PAGE, after = ((int64_t)cached[j] + added[j] + PAGE - 1) / PAGE;
        // pages the table has no room for are missing, too
        const int64_t fits = min(after, max(out.width, before));
        need[j] = (int)(fits - before);
        lack += (int)(after - fits);
        sum_added += added[j];
        sum_need += need[j];
    }
    const int upto_added = detail::wave_inclusive_sum(sum_added), upto_need = detail::wave_inclusive_sum(sum_need);
    const int upto_lack = detail::wave_inclusive_sum(lack);
    if (lane == kWaveSize - 1) {
        wave_added[wave] = upto_added;
        wave_need[wave] = upto_need;
        wave_lack[wave] = upto_lack;
    }
    __syncthreads();
    int at_added = upto_added - sum_added, at_need = upto_need - sum_need;
    int total_added = 0, total_need = 0, total_lack = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        at_added += w < wave ? wave_added[w] : 0;
        at_need += w < wave ? wave_need[w] : 0;
        total_added += wave_added[w];
        total_need += wave_need[w];
        total_lack += wave_lack[w];
    }
    const int count = min(max(*free_pages.count, 0), (int)min(free_pages.capacity, (int64_t)0x7fffffff));
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int b = tid * (int)PER + j;
        if (b < n) {
            starts[b] = at_added;
            first[b] = at_need;
            held[b] = cached[j];
            if (share.x == 0) {
                out.starts[b] = at_added;
                out.lengths[b] = cached[j] + added[j];
            }
        }
        at_added += added[j];
        at_need += need[j];
    }
    if (share.x == 0 && tid == 0) {
        out.starts[n] = total_added;
        out.counts[0] = max(count - total_need, 0);
        out.counts[1] = max(total_need - count, 0) + total_lack;
    }
    __syncthreads();

    const int64_t step = out.shares * THREADS;
    for (int64_t i = share.x * THREADS + tid; i < total_need; i += step) {
        const int b = detail::last_not_above(first, n, (int)i);
        const int64_t j = (held[b] + PAGE - 1) / PAGE + (i - first[b]);
        const int64_t at = count - 1 - i;
        if (j < out.width) {
            out.table[b * out.width + j] = at >= 0 ? free_pages.list[at] : -1;
        }
    }
    for (int64_t t = share.x * THREADS + tid; t < out.tokens; t += step) {
        int64_t slot = -1;
        if (t < total_added) {
            const int b = detail::last_not_above(starts, n, (int)t);
            const int64_t pos = held[b] + (t - starts[b]);
            const int64_t p = pos / PAGE, before = (held[b] + PAGE - 1) / PAGE;
            int page = -1;
            if (p < out.width) {
                if (p < before) {
                    page = out.table[b * out.width + p];
                } else {
                    const int64_t at = count - 1 - (first[b] + (p - before));
                    page = at >= 0 ? free_pages.list[at] : -1;
                }
            }
            slot = page >= 0 ? (int64_t)page * PAGE + pos % PAGE : -1;
            slot = slot <= 0x7fffffff ? slot : -1;
        }
        out.slots[t] = (int)slot;
    }
}

}  // namespace gernels
