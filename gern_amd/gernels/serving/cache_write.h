// New keys and values into a paged cache (gernels/serving/paged_cache.h).
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
// Measured: 8 prompts, 8 heads of 64 (59 MB) in 15.7 us, of which loads that
// depend on one another (slots, values and scale, codes) are most; 256 tokens, 8
// heads of 128 in 5.1 us on the GPU.
#pragma once

#include "gernels/serving/half_tiles.h"
#include "gernels/serving/paged_cache.h"

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

// The cache as something that is written: a piece is a stretch of tokens of one
// head of the keys (side 0) or of the values (1).  Heads and sides run fastest, so
// that the workgroups that run together read whole rows of new tokens between them
// (8192 to 16384 tokens, 8 heads of 64: 20 us with the stretches fastest).
struct CacheStretch {
    const PagedCache &cache;
    int64_t begin, end, head, side;
};
struct WritableCache : PagedCache {
    int64_t pieces, stretch;  // workgroups, and tokens in a stretch

    __device__ __forceinline__ CacheStretch at(int64_t x) const {
        const uint32_t per = 2 * (uint32_t)heads, piece = (uint32_t)x, i = piece % per;
        const int64_t begin = (int64_t)(piece / per) * stretch;
        return {*this, begin, begin + stretch, i % (uint32_t)heads, i / (uint32_t)heads};
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

// Four codes.  Values beyond the range have to be brought into it first (`saturate`); NaN stays NaN either way.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d, bool saturate) {
    if (saturate) {
        a = to_e4m3_range(a), b = to_e4m3_range(b), c = to_e4m3_range(c), d = to_e4m3_range(d);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (uint32_t)w;
}

// Magnitudes of 16-bit floats compare like their bits, two to an instruction.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
constexpr uint32_t kMagnitude = 0x7fff7fffu;
template<class T>
struct Infinity {
    static constexpr uint32_t bits = T::kBf16 ? 0x7f80u : 0x7c00u;
};
__device__ __forceinline__ uint32_t larger_halves(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t largest_magnitudes(const Words4 &x) {
    return larger_halves(larger_halves(x.w[0] & kMagnitude, x.w[1] & kMagnitude), larger_halves(x.w[2] & kMagnitude, x.w[3] & kMagnitude));
}
// The same, infinities and NaN left out.
template<class T>
__device__ __forceinline__ uint32_t largest_finite_magnitude(const Words4 &x) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t low = x.w[j] & 0x7fffu, high = x.w[j] >> 16 & 0x7fffu;
        most = max(most, low < Infinity<T>::bits ? low : 0u);
        most = max(most, high < Infinity<T>::bits ? high : 0u);
    }
    return most;
}

template<int THREADS>
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    for (int d = 1; d < kWaveSize; d *= 2) {
        x = max(x, (uint32_t)__shfl_xor((int)x, d));
    }
    if constexpr (THREADS > kWaveSize) {
        __shared__ uint32_t of_wave[THREADS / kWaveSize];
        __syncthreads();  // the previous run's values have been read
        if (lane_id() == 0) {
            of_wave[threadIdx.x / kWaveSize] = x;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / kWaveSize; w++) {
            x = max(x, of_wave[w]);
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
    constexpr int kWhole = (int)((PAGE * kPieces + THREADS - 1) / THREADS), kHeld = THREADS > kWaveSize ? kWhole : kWhole < 2 ? kWhole : 2;
    // tokens of a stretch (the caller's, at most this many) and of a run that begins in it
    constexpr int kStretch = THREADS > kWaveSize ? (int)PAGE : 1, kWords = (kStretch + (int)PAGE + 63) / 64;
    const int64_t end = min(min(to.end, to.begin + kStretch), tokens.tokens);
    const uint32_t *src = (to.side == 0 ? tokens.k : tokens.v) + to.head * (D / 2);
    const int64_t pitch = to.side == 0 ? tokens.k_pitch : tokens.v_pitch;
    float *scales = to.side == 0 ? cache.k_scales : cache.v_scales;
    uint32_t *codes = to.side == 0 ? cache.k : cache.v;

    // One load tells all runs of the stretch, to their ends: lane i of word w looks at token begin + 64 w + i.  A token
    // that continues the run of the one before it is a set bit.
    int slot_of[kWords];
    uint64_t goes_on[kWords];
#pragma unroll
    for (int w = 0; w < kWords; w++) {
        const int64_t t = to.begin + 64 * w + lane;
        const int slot = tokens.slots[min(t, tokens.tokens - 1)], before = tokens.slots[max(min(t, tokens.tokens - 1) - 1, (int64_t)0)];
        slot_of[w] = slot;
        goes_on[w] = __ballot(t > 0 && t < tokens.tokens && slot > 0 && slot % (int)PAGE != 0 && slot == before + 1);
    }
    const int count = (int)(end - to.begin);
    for (int at_token = 0; at_token < count;) {
        // first token and length of the next run; both may be in a later word
        int slot = 0, n = 1;
        bool first = false;
#pragma unroll
        for (int w = 0; w < kWords; w++) {
            if (at_token / 64 == w) {
                slot = __builtin_amdgcn_readlane(slot_of[w], at_token % 64);
                first = !(goes_on[w] >> (at_token % 64) & 1);
            }
        }
        bool open = true;
#pragma unroll
        for (int w = 0; w < kWords; w++) {
            const int from = max(at_token + 1 - 64 * w, 0);
            if (open && from < 64) {
                const uint64_t ends = ~goes_on[w] >> from << from;
                open = ends == 0;
                n = 64 * w + (open ? 64 : __builtin_ctzll(ends)) - at_token;
            }
        }
        // the tail of a run that began in an earlier stretch is that workgroup's
        const bool mine = first && slot >= 0;
        const int64_t t = to.begin + at_token, page = slot / (int)PAGE;
        const int place = slot % (int)PAGE;
        const bool there = page < cache.pages;
        at_token += n;
        if (mine && !there && to.head == 0 && to.side == 0 && tid == 0) {
            atomicAdd(cache.faults, 1u);
        }
        if (mine && there) {
            const int64_t at = page * cache.heads + to.head;
            const float old = scales[at];
            // The run's values stay in registers between the scale and the codes; what does not fit (a run of more than a
            // few tokens on one wavefront) is read again.
            const uint32_t *rows = src + t * pitch;
            const int pieces = n * kPieces;
            Words4 held[kHeld];
            auto value = [&](int i) { return *reinterpret_cast<const Words4 *>(rows + (i / kPieces) * pitch + (i % kPieces) * 4); };
#pragma unroll
            for (int j = 0; j < kHeld; j++) {
                held[j] = value(min(tid + j * (int)THREADS, pieces - 1));
            }
            uint32_t halves = 0;
#pragma unroll
            for (int j = 0; j < kHeld; j++) {
                halves = detail::larger_halves(halves, detail::largest_magnitudes(held[j]));
            }
            for (int i = tid + kHeld * (int)THREADS; i < pieces; i += THREADS) {
                halves = detail::larger_halves(halves, detail::largest_magnitudes(value(i)));
            }
            uint32_t most = detail::block_max<THREADS>(max(halves & 0xffffu, halves >> 16));
            const bool all_finite = most < detail::Infinity<T>::bits;
            if (!all_finite) {
                most = 0;
                for (int i = tid; i < pieces; i += THREADS) {
                    most = max(most, detail::largest_finite_magnitude<T>(value(i)));
                }
                most = detail::block_max<THREADS>(most);
            }
            const float need = detail::scale_for(half_to_float<T>(most));
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
                        c.w[j] = detail::pack_e4m3(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio, true);
                    }
                    *reinterpret_cast<Words4 *>(page_codes + i * 4) = c;
                }
            }
            if (tid == 0 && scale != old) {
                scales[at] = scale;
            }
            // a power of two but for an older scale that the caller made; finite values are within its range
            const bool exact = (__builtin_bit_cast(uint32_t, scale) & 0x7fffffu) == 0;
            const float inverse = 1.0f / scale;
            auto store = [&](int i, const Words4 &x) {
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
                const Words2 c = {{detail::pack_e4m3(f[0], f[1], f[2], f[3], !all_finite), detail::pack_e4m3(f[4], f[5], f[6], f[7], !all_finite)}};
                *reinterpret_cast<Words2 *>(page_codes + (place + i / kPieces) * (D / 4) + (i % kPieces) * 2) = c;
            };
#pragma unroll
            for (int j = 0; j < kHeld; j++) {
                if (tid + j * (int)THREADS < pieces) {
                    store(tid + j * (int)THREADS, held[j]);
                }
            }
            for (int i = tid + kHeld * (int)THREADS; i < pieces; i += THREADS) {
                store(i, value(i));
            }
        }
    }
}

}  // namespace gernels
