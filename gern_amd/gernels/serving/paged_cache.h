// A paged cache of keys and values in 8 bits, and what the gernels over it
// share.
//
//   codes   [pages, heads, page size, head dim] bytes (e4m3: 4 exponent bits,
//           3 mantissa bits, largest value 448, no infinities), one array for
//           keys and one for values
//   scales  [pages, heads] fp32, for each of the two; a value is code * scale
//
// One page of one head is contiguous (page size x head dim bytes): attention
// for a head reads whole lines, and the scale changes only from page to page.
#pragma once

#include "gernels/prelude.h"

namespace gernels {

struct PagedCache {
    uint32_t *k, *v;         // four codes a word
    float *k_scales, *v_scales;
    int64_t pages;
    int64_t heads;
    uint32_t *faults;        // counts pages and slots that are not in the cache

    __device__ __forceinline__ const PagedCache &whole() const {
        return *this;
    }
};

}  // namespace gernels
