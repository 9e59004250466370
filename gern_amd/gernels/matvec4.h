// y = x W^T for a few rows of x and a matrix W in 4 bits.
//
//   W[n, k] = s[k / G, n] * (q[n, k] - z[k / G, n])     q in 0 .. 15, groups of G columns
//   y[m, n] = sum_g s[g, n] * (sum_{k in g} x[m, k] q[n, k] - z[g, n] * sum_{k in g} x[m, k])
//
// Bound by memory: N K / 2 bytes of codes, read once, for 2 M N K operations.  The
// matrix cores do them for up to 16 rows at the price of one.  A wavefront takes
// 16 columns n per tile and blocks of 128 k: lane (g, c), c = lane mod 16,
// g = lane / 16, reads 16 bytes (32 codes) of row c, and four lane exchanges
// transpose the 4 x 4 words of lane groups and registers so that a step of
// v_mfma_16x16x32 covers 32 consecutive k: any group of 32, 64 or 128 columns is
// then a whole number of steps, and its scale multiplies fp32 sums, not weights.
//
// A code becomes a 16-bit float without arithmetic: or'ed into the mantissa of
// 128 (bf16, lowest bits) or 64 (fp16, bits 4 - 7) it stands for 128 + q or 64 + q
// exactly, two codes (nibbles i and i + 4) an instruction.  x is laid out in pairs
// (i, i + 4) to match, and the offset leaves with the zero point:
// sum x (128 + q) - (128 + z) sum x.  The sum of x comes from one more matrix
// instruction, against ones, for all columns.  The offset costs fp32 rounding of a
// sum 128 / 4.6 (the spread of q - z) times larger: 2^-24 * 28, 2^-19.2 of the
// result's size against the 2^-9 (bf16) or 2^-12 (fp16) of its last rounding.
//
// The wavefronts of a workgroup divide K and add their sums in LDS, in a fixed
// order.
#pragma once

#include "gernels/half_tiles.h"

namespace gernels {

template<class T>
struct ActivationsOf {
    const uint32_t *x;   // two values a word
    int64_t pitch;       // words from row to row
    int64_t rows;        // M

    __device__ __forceinline__ const ActivationsOf &whole() const {
        return *this;
    }
};

struct Weights4 {
    const uint32_t *codes;          // [n, k / 8]: eight codes a word, lowest bits first
    const unsigned short *scales;   // [k / G, n]
    const unsigned char *zeros;     // [k / G, n], or null: 8
    int64_t n, k;

    __device__ __forceinline__ const Weights4 &whole() const {
        return *this;
    }
};

struct MatvecColumns;
struct MatvecOut {
    unsigned short *y;
    int64_t pitch;    // elements from row to row
    int64_t columns;  // workgroups

    __device__ __forceinline__ MatvecColumns at(int64_t x) const;
};
struct MatvecColumns {
    const MatvecOut &to;
    int64_t x;
};
__device__ __forceinline__ MatvecColumns MatvecOut::at(int64_t x) const {
    return {*this, x};
}

namespace detail {

// Words of lane group g, register s <-> lane group s, register g.
__device__ __forceinline__ void transpose_lane_groups(uint32_t w[4]) {
#pragma unroll
    for (int s = 0; s < 2; s++) {
        const auto r = __builtin_amdgcn_permlane32_swap(w[s], w[2 + s], false, false);
        w[s] = r[0], w[2 + s] = r[1];
    }
#pragma unroll
    for (int s = 0; s < 4; s += 2) {
        const auto r = __builtin_amdgcn_permlane16_swap(w[s], w[s + 1], false, false);
        w[s] = r[0], w[s + 1] = r[1];
    }
}

// offset + code for the eight codes of a word, in pairs (i, i + 4).
template<bool BF16>
struct CodeOffset {
    static constexpr float value = BF16 ? 128.0f : 64.0f;
};
template<bool BF16>
__device__ __forceinline__ Frag offset_codes(uint32_t w) {
    if constexpr (BF16) {
        return {{(w & 0x000f000fu) | 0x43004300u, ((w >> 4) & 0x000f000fu) | 0x43004300u, ((w >> 8) & 0x000f000fu) | 0x43004300u,
                 ((w >> 12) & 0x000f000fu) | 0x43004300u}};
    } else {
        return {{((w << 4) & 0x00f000f0u) | 0x54005400u, (w & 0x00f000f0u) | 0x54005400u, ((w >> 4) & 0x00f000f0u) | 0x54005400u,
                 ((w >> 8) & 0x00f000f0u) | 0x54005400u}};
    }
}

// (0, 1) (2, 3) (4, 5) (6, 7) -> (0, 4) (1, 5) (2, 6) (3, 7)
__device__ __forceinline__ Frag pair_with_fourth(const Frag &x) {
    return {{__builtin_amdgcn_perm(x.w[2], x.w[0], 0x05040100u), __builtin_amdgcn_perm(x.w[2], x.w[0], 0x07060302u),
             __builtin_amdgcn_perm(x.w[3], x.w[1], 0x05040100u), __builtin_amdgcn_perm(x.w[3], x.w[1], 0x07060302u)}};
}

// One block of 128 k: codes, activations, scales and zero points.
template<int G, int MT, int NT>
struct MatvecBlock {
    uint32_t codes[NT][4];
    Frag x[MT][4];
    uint32_t scale[NT][128 / G], zero[NT][128 / G];
};

}  // namespace detail

// MT tiles of 16 rows against NT tiles of 16 columns on WAVES wavefronts.
template<int64_t G, int64_t MT, int64_t NT, int64_t WAVES, class T>
__device__ __forceinline__ void multiply_4bit(const ActivationsOf<T> &a, const Weights4 &weights, const MatvecColumns &columns) {
    constexpr bool kBf16 = T::kBf16;
    constexpr int kGroups = 128 / G;  // of a block
    constexpr int kSteps = G / 32;    // of a group
    const int lane = lane_id(), g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int64_t n0 = columns.x * (16 * NT);
    const int blocks = (int)((weights.k + 127) / 128);
    const int groups = (int)(weights.k / G);

    // rows and columns behind the last one read it again; their sums are not stored
    const uint32_t *code_row[NT];
    int64_t column[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        column[t] = min(n0 + 16 * t + c, weights.n - 1);
        code_row[t] = weights.codes + column[t] * (weights.k / 8) + 4 * g;
    }
    auto load = [&](detail::MatvecBlock<G, MT, NT> &b, int block) {
        // a last block may be 32, 64 or 96 wide: its missing x are zero, and its missing codes are the row's first
        const int64_t k0 = (int64_t)block * 128;
        const int64_t word = k0 + 32 * g < weights.k ? k0 / 8 : -4 * g;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            detail::load_words<4>(b.codes[t], code_row[t] + word);
#pragma unroll
            for (int j = 0; j < kGroups; j++) {
                const int64_t at = min((int)(block * kGroups) + j, groups - 1) * weights.n + column[t];
                b.scale[t][j] = weights.scales[at];
                b.zero[t][j] = weights.zeros != nullptr ? weights.zeros[at] : 8;
            }
        }
#pragma unroll
        for (int r = 0; r < MT; r++) {
#pragma unroll
            for (int s = 0; s < 4; s++) {
                b.x[r][s] = detail::Frag{{0u, 0u, 0u, 0u}};
                if (16 * r + c < a.rows && k0 + 32 * s < weights.k) {
                    detail::load_words<4>(b.x[r][s].w, a.x + (16 * r + c) * a.pitch + (k0 + 32 * s + 8 * g) / 2);
                }
            }
        }
    };

    detail::f32x4 total[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int r = 0; r < MT; r++) {
            total[t][r] = detail::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    constexpr uint32_t kOnes = kBf16 ? 0x3f803f80u : 0x3c003c00u;
    const detail::Frag ones = {{kOnes, kOnes, kOnes, kOnes}};
    auto add = [&](detail::MatvecBlock<G, MT, NT> &b) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            detail::transpose_lane_groups(b.codes[t]);
        }
#pragma unroll
        for (int j = 0; j < kGroups; j++) {
            detail::f32x4 dot[NT][MT], sum[MT];
#pragma unroll
            for (int r = 0; r < MT; r++) {
                sum[r] = detail::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    dot[t][r] = sum[r];
                }
            }
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                const int s = j * kSteps + i;
                detail::Frag x[MT];
#pragma unroll
                for (int r = 0; r < MT; r++) {
                    x[r] = detail::pair_with_fourth(b.x[r][s]);
                    sum[r] = detail::mfma_16x16x32<kBf16>(x[r], ones, sum[r]);
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const detail::Frag w = detail::offset_codes<kBf16>(b.codes[t][s]);
#pragma unroll
                    for (int r = 0; r < MT; r++) {
                        dot[t][r] = detail::mfma_16x16x32<kBf16>(x[r], w, dot[t][r]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float scale = half_to_float<T>(b.scale[t][j]);
                const float zero = -((float)b.zero[t][j] + detail::CodeOffset<kBf16>::value);
#pragma unroll
                for (int r = 0; r < MT; r++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        total[t][r][e] = __builtin_fmaf(scale, __builtin_fmaf(zero, sum[r][e], dot[t][r][e]), total[t][r][e]);
                    }
                }
            }
        }
    };

    int block = wave;
    if (block < blocks) {
        detail::MatvecBlock<G, MT, NT> even, odd;
        load(even, block);
        while (true) {
            if (block + WAVES < blocks) {
                load(odd, block + WAVES);
            }
            add(even);
            block += WAVES;
            if (block >= blocks) {
                break;
            }
            if (block + WAVES < blocks) {
                load(even, block + WAVES);
            }
            add(odd);
            block += WAVES;
            if (block >= blocks) {
                break;
            }
        }
    }

    // [wavefront][tile][row of four][lane]
    constexpr int kTiles = NT * MT;
    __shared__ float parts[WAVES][kTiles * 4][kWaveSize];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int r = 0; r < MT; r++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                parts[wave][(t * MT + r) * 4 + e][lane] = total[t][r][e];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kTiles * 4 * kWaveSize; i += WAVES * kWaveSize) {
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            y += parts[w][i / kWaveSize][i % kWaveSize];
        }
        const int from = i % kWaveSize, tile = i / kWaveSize / 4, e = i / kWaveSize % 4;
        const int64_t m = 16 * (tile % MT) + 4 * (from / 16) + e, n = n0 + 16 * (tile / MT) + from % 16;
        if (m < a.rows && n < weights.n) {
            columns.to.y[m * columns.to.pitch + n] = (unsigned short)(pack_halves<T>(y, 0.0f) & 0xffffu);
        }
    }
}

}  // namespace gernels
