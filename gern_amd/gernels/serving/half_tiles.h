// 16-bit floats in words, and the 16 x 16 x 32 matrix instruction on them: what
// the gernels with bf16 or fp16 operands beside 8- or 4-bit codes share.
#pragma once

#include "gernels/prelude.h"

namespace gernels {

// Element types of 16-bit operands and results.
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

namespace detail {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Frag {
    uint32_t w[4];
};

// C += A B on 16 x 16 x 32: lane (g, c) holds row / column c of A / B at k = 8g .. 8g+7,
// and rows 4g .. 4g+3 of column c of C.
template<bool BF16>
__device__ __forceinline__ f32x4 mfma_16x16x32(const Frag &a, const Frag &b, f32x4 c) {
    if constexpr (BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

// N words from memory in as few loads as their alignment allows (N = 1 .. 4).
template<int N>
__device__ __forceinline__ void load_words(uint32_t *to, const uint32_t *from) {
    if constexpr (N == 4) {
        const Words4 x = *reinterpret_cast<const Words4 *>(from);
        to[0] = x.w[0], to[1] = x.w[1], to[2] = x.w[2], to[3] = x.w[3];
    } else if constexpr (N == 2) {
        const Words2 x = *reinterpret_cast<const Words2 *>(from);
        to[0] = x.w[0], to[1] = x.w[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            to[i] = from[i];
        }
    }
}

}  // namespace detail

}  // namespace gernels
