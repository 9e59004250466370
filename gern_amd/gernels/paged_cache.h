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

// Element types of keys, values and queries outside the cache.
struct Bf16 {
    static constexpr bool kBf16 = true;
};
struct F16 {
    static constexpr bool kBf16 = false;
};

template<class T>
__device__ __forceinline__ float half_to_float(uint32_t bits16) {
    if constexpr (T::kBf16) {
        return __builtin_bit_cast(float, bits16 << 16);
    } else {
        return (float)__builtin_bit_cast(_Float16, (unsigned short)bits16);
    }
}

// Two values rounded to T (nearest even), the first in the low half.
template<class T>
__device__ __forceinline__ uint32_t pack_halves(float a, float b) {
    if constexpr (T::kBf16) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        const pair p = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, p);
    } else {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        const pair p = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, p);
    }
}

struct alignas(16) Words4 {
    uint32_t w[4];
};
struct alignas(8) Words2 {
    uint32_t w[2];
};

}  // namespace gernels
