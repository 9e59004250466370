// New keys and values into a paged cache (gernels/paged_cache.h).
//
// Token t goes to slot[t] = page * P + place (-1: nowhere).  For every page and
// head, over what the page holds in front of the new tokens and what is added:
//
//   need  = the smallest power of two with amax(new) <= 448 need, at least 2^-64
//   scale = need, or max(old scale, need) where the page holds earlier tokens
//   code  = e4m3(x / scale), rounded to nearest even, saturated; a NaN stays one
//   earlier codes move along: code = e4m3(code * (old scale / scale))
//
// The scales are powers of two so that x / scale and old / scale are exact in
// fp32: a code is one rounding away from the value it stands for, a page whose
// scale grows loses only what drops under the smallest step (2^-9 of the new
// scale), and writing the same tokens again changes nothing.  e4m3 keeps its
// three mantissa bits at any scale, so the power of two costs no precision.
//
// Bound by memory: 2 bytes read and 1 written a value, plus the earlier codes of
// a page whose scale grows.  One workgroup takes a stretch of tokens of one head
// of the keys or of the values and looks for the runs in it: consecutive tokens
// in consecutive slots of one page.  A run is the first token's workgroup's.
#pragma once

#include "gernels/half_tiles.h"
#include "gernels/paged_cache.h"

namespace gernels {

template<class T>
struct NewTokensOf {
    const uint32_t *k, *v;     // two values a word; heads of a token are contiguous
    int64_t k_pitch, v_pitch;  // words from token to token
    const int32_t *slots;
    int64_t tokens;

    __device__ __forceinline__ const NewTokensOf &whole() const {
        return *this;
    }
};

// The cache as something that is written: a subset is a stretch of tokens, one
// head, keys (0) or values (1).
struct CacheStretch {
    const PagedCache &cache;
    int64_t begin, end, head, side;
};
struct WritableCache : PagedCache {
    int64_t stretches, stretch, sides;  // how many, tokens in each, 2

    __device__ __forceinline__ CacheStretch at(int64_t x, int64_t head, int64_t side) const {
        return {*this, x * stretch, (x + 1) * stretch, head, side};
    }
};

namespace detail {

constexpr float kE4m3Max = 448.0f;

// The smallest power of two 2^e, e >= -64, with amax <= 448 * 2^e.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
    // 448 = 1.75 * 2^8
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, -64);
    return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// Saturates; a NaN passes.
__device__ __forceinline__ float to_e4m3_range(float x) {
    const float c = __builtin_amdgcn_fmed3f(x, -kE4m3Max, kE4m3Max);
    return x != x ? x : c;
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(to_e4m3_range(a), to_e4m3_range(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(to_e4m3_range(c), to_e4m3_range(d), w, true);
    return (uint32_t)w;
}

__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = __builtin_fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}

template<int THREADS>
__device__ __forceinline__ float block_max(float x) {
    for (int d = 1; d < kWaveSize; d *= 2) {
        x = __builtin_fmaxf(x, __shfl_xor(x, d));
    }
    if constexpr (THREADS > kWaveSize) {
        __shared__ float of_wave[THREADS / kWaveSize];
        __syncthreads();  // the previous run's values have been read
        if (lane_id() == 0) {
            of_wave[threadIdx.x / kWaveSize] = x;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / kWaveSize; w++) {
            x = __builtin_fmaxf(x, of_wave[w]);
        }
    }
    return x;
}

}  // namespace detail

template<int64_t D, int64_t PAGE, int64_t THREADS, class T>
__device__ __forceinline__ void write_cache(const NewTokensOf<T> &tokens, const CacheStretch &to) {
    const PagedCache &cache = to.cache;
    const int lane = lane_id(), tid = threadIdx.x;
    constexpr int kPieces = D / 8;  // 16-byte pieces of a new row
    const int64_t end = min(to.end, tokens.tokens);
    const uint32_t *src = (to.side == 0 ? tokens.k : tokens.v) + to.head * (D / 2);
    const int64_t pitch = to.side == 0 ? tokens.k_pitch : tokens.v_pitch;
    float *scales = to.side == 0 ? cache.k_scales : cache.v_scales;
    uint32_t *codes = to.side == 0 ? cache.k : cache.v;

    for (int64_t t = to.begin; t < end;) {
        // the run from t on: lane i looks at token t + i
        const int slot = tokens.slots[t];
        const int place = slot >= 0 ? slot % (int)PAGE : 0;
        const int64_t page = slot / (int)PAGE;
        int n = 1;
        if (slot >= 0) {
            for (int base = 0; base < PAGE; base += kWaveSize) {
                const int64_t i = base + lane;
                const bool in = place + i < PAGE && t + i < tokens.tokens && tokens.slots[min(t + i, tokens.tokens - 1)] == slot + (int)i;
                const uint64_t out = ~__ballot(in);
                if (out != 0) {
                    n = base + __builtin_ctzll(out);
                    break;
                }
                n = base + kWaveSize;
            }
        }
        // the tail of a run that began in an earlier stretch is that workgroup's
        const bool mine = slot >= 0 && (place == 0 || t == 0 || tokens.slots[t - 1] != slot - 1);
        const bool there = page < cache.pages;
        if (slot >= 0 && !there && mine && to.head == 0 && to.side == 0 && tid == 0) {
            atomicAdd(cache.faults, 1u);
        }
        if (mine && there) {
            const uint32_t *rows = src + t * pitch;
            float amax = 0.0f;
            for (int i = tid; i < n * kPieces; i += THREADS) {
                const Words4 x = *reinterpret_cast<const Words4 *>(rows + (i / kPieces) * pitch + (i % kPieces) * 4);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    amax = __builtin_fmaxf(amax, detail::finite_magnitude(half_to_float<T>(x.w[j] & 0xffffu)));
                    amax = __builtin_fmaxf(amax, detail::finite_magnitude(half_to_float<T>(x.w[j] >> 16)));
                }
            }
            amax = detail::block_max<THREADS>(amax);
            const int64_t at = page * cache.heads + to.head;
            const float need = detail::scale_for(amax), old = scales[at];
            const float scale = place > 0 && old > need ? old : need;
            if constexpr (THREADS > kWaveSize) {
                __syncthreads();  // every thread has the old scale
            }
            uint32_t *page_codes = codes + at * (PAGE * D / 4);
            if (place > 0 && scale != old) {
                const float ratio = old / scale;
                for (int i = tid; i < place * (int)(D / 16); i += THREADS) {
                    Words4 c = *reinterpret_cast<const Words4 *>(page_codes + i * 4);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        typedef float f32x2 __attribute__((ext_vector_type(2)));
                        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.w[j], false);
                        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.w[j], true);
                        c.w[j] = detail::pack_e4m3(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
                    }
                    *reinterpret_cast<Words4 *>(page_codes + i * 4) = c;
                }
            }
            if (tid == 0 && scale != old) {
                scales[at] = scale;
            }
            // a power of two but for an older scale that the caller made
            const bool exact = (__builtin_bit_cast(uint32_t, scale) & 0x7fffffu) == 0;
            const float inverse = 1.0f / scale;
            for (int i = tid; i < n * kPieces; i += THREADS) {
                const int row = i / kPieces, piece = i % kPieces;
                const Words4 x = *reinterpret_cast<const Words4 *>(rows + row * pitch + piece * 4);
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    f[2 * j] = half_to_float<T>(x.w[j] & 0xffffu);
                    f[2 * j + 1] = half_to_float<T>(x.w[j] >> 16);
                }
                if (exact) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        f[j] *= inverse;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        f[j] /= scale;
                    }
                }
                const Words2 c = {{detail::pack_e4m3(f[0], f[1], f[2], f[3]), detail::pack_e4m3(f[4], f[5], f[6], f[7])}};
                *reinterpret_cast<Words2 *>(page_codes + (place + row) * (D / 4) + piece * 2) = c;
            }
        }
        t += n;
    }
}

}  // namespace gernels
