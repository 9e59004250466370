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
// a power of two (bf16: 2^-9, lowest bits, fp16: 64, bits 4 - 7) it stands for
// 2^-16 (128 + q) or 64 + q exactly, two codes (nibbles i and i + 4) an
// instruction.  The 2^-16, taken back at the end, keeps a group's sums of bf16
// activations finite whatever these are (128 of them times 128 + 255 at most).  x is laid out in pairs
// (i, i + 4) to match, and the offset leaves with the zero point:
// sum x (128 + q) - (128 + z) sum x.  The sum of x comes from one more matrix
// instruction, against ones (2^-9 again), for all columns.  The offset costs fp32 rounding of a
// sum 128 / 4.6 (the spread of q - z) times larger: 2^-24 * 28, 2^-19.2 of the
// result's size against the 2^-8 (bf16) or 2^-11 (fp16) of its last rounding.
//
// The wavefronts of a workgroup divide K and add their sums in LDS, in a fixed
// order.  Measured: 1 row, 28672 columns, K = 8192, G = 128 in 27.5 us (4.5 TB/s of
// codes, scales and zero points; a copy of 1 GiB moves 5.2 on the same GPU); 13
// rows, 10001 columns, K = 8192, G = 64 in 15.6 us (2.9 TB/s: bound by the latency
// of its loads, a block ahead for one wavefront a SIMD on 209 CUs; the vector ALU is
// busy for 24 % of the time, the matrix cores for 6 %).
#pragma once

#include "gernels/serving/half_tiles.h"

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

// unit * (offset + code) for the eight codes of a word, in pairs (i, i + 4); `one` stands for one in the sum of x, and is a
// power of two (bits `ones`, twice).
template<bool BF16>
struct CodeOffset {
    static constexpr float value = BF16 ? 128.0f : 64.0f;
    static constexpr float unit = BF16 ? 0x1p-16f : 1.0f, one = BF16 ? 0x1p-9f : 1.0f;
    static constexpr uint32_t ones = BF16 ? 0x3b003b00u : 0x3c003c00u;
};
// `offsets` is code_offsets<BF16>(): in a register, so that `and` and `or` are one instruction (two literals do not fit).
template<bool BF16>
__device__ __forceinline__ uint32_t code_offsets() {
    uint32_t two = BF16 ? 0x3b003b00u : 0x54005400u;
    asm volatile("" : "+v"(two));
    return two;
}
template<bool BF16>
__device__ __forceinline__ Frag offset_codes(uint32_t w, uint32_t offsets) {
    if constexpr (BF16) {
        return {{(w & 0x000f000fu) | offsets, ((w >> 4) & 0x000f000fu) | offsets, ((w >> 8) & 0x000f000fu) | offsets, ((w >> 12) & 0x000f000fu) | offsets}};
    } else {
        return {{((w << 4) & 0x00f000f0u) | offsets, (w & 0x00f000f0u) | offsets, ((w >> 4) & 0x00f000f0u) | offsets, ((w >> 8) & 0x00f000f0u) | offsets}};
    }
}

// (0, 1) (2, 3) (4, 5) (6, 7) -> (0, 4) (1, 5) (2, 6) (3, 7)
__device__ __forceinline__ Frag pair_with_fourth(const Frag &x) {
    return {{__builtin_amdgcn_perm(x.w[2], x.w[0], 0x05040100u), __builtin_amdgcn_perm(x.w[2], x.w[0], 0x07060302u),
             __builtin_amdgcn_perm(x.w[3], x.w[1], 0x05040100u), __builtin_amdgcn_perm(x.w[3], x.w[1], 0x07060302u)}};
}

// All four lane groups get, in register t, what lane group t has in w: the transposition of four equal registers.
__device__ __forceinline__ void spread_lane_groups(uint32_t w, uint32_t to[4]) {
    to[0] = to[1] = to[2] = to[3] = w;
    transpose_lane_groups(to);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// One block of 128 k as it is loaded: codes, activations, scales and zero points.  Vectors, not arrays: a loaded vector
// that is carried to the next iteration as four words is copied word by word, and waited for, where it is loaded.
// With three or four tiles of columns, lane group t holds the scales and zero points of tile t, one load for all;
// otherwise each tile's are in every lane group.
template<int G, int MT, int NT>
struct MatvecBlock {
    static constexpr int kXTiles = MT == 0 ? 1 : MT, kXSteps = MT == 0 ? 1 : 4, kScaleTiles = NT >= 3 ? 1 : NT;
    u32x4 codes[NT];
    u32x4 x[kXTiles][kXSteps];
    uint32_t scale[kScaleTiles][128 / G], zero[kScaleTiles][128 / G];
};

}  // namespace detail

// NT (1 to 4) tiles of 16 columns on WAVES wavefronts, for up to 16 MT rows of x; MT = 0: up to 4 rows.
//
// With up to 4 rows the 16 rows of a matrix instruction hold them four times over, shifted: row 4 i + s is row i at
// step s of a block (k = 32 s ..).  One load brings x for all four steps, and step s's products stand in row 4 i + s of
// an accumulator of its own, element s of lane group i: four times less x to load and to arrange.
template<int64_t G, int64_t MT, int64_t NT, int64_t WAVES, class T>
__device__ __forceinline__ void multiply_4bit(const ActivationsOf<T> &a, const Weights4 &weights, const MatvecColumns &columns) {
    constexpr bool kBf16 = T::kBf16, kFew = MT == 0;
    constexpr int kGroups = 128 / G;  // of a block
    constexpr int kSteps = G / 32;    // of a group
    constexpr int kRowTiles = kFew ? 1 : MT, kSums = kFew ? 1 : 4;  // sums a lane holds of a tile
    using Block = detail::MatvecBlock<G, MT, NT>;
    const int lane = lane_id(), g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int64_t n0 = columns.x * (16 * NT);
    const int words = (int)(weights.k / 8), blocks = (words + 15) / 16;

    // Addresses are a uniform base, which the scalar unit advances, and a lane's offset, which stays.  Rows and columns
    // behind the last one read it again; their sums are not stored.  A last block that is not whole is read as the
    // LAST 128 columns (fewer, where there are not that many), and x is zero in those that an earlier block had.  No load
    // stands behind a branch: what a branch may leave unloaded is waited for where the paths meet, and loads are to run
    // ahead of their use.
    const int last_column = (int)min(weights.n - 1 - n0, (int64_t)(16 * NT - 1));
    uint32_t code_offset[NT], x_offset[kRowTiles], scale_offset[Block::kScaleTiles];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        code_offset[t] = (uint32_t)min(16 * t + c, last_column) * (uint32_t)words + (uint32_t)min(4 * g, words - 4);
    }
#pragma unroll
    for (int t = 0; t < Block::kScaleTiles; t++) {
        scale_offset[t] = (uint32_t)min(16 * (NT >= 3 ? g : t) + c, last_column);
    }
    const int last_row = (int)a.rows - 1;
#pragma unroll
    for (int r = 0; r < kRowTiles; r++) {
        const int row = min(kFew ? c / 4 : 16 * r + c, last_row);
        x_offset[r] = (uint32_t)(row * (int)a.pitch + 4 * g + (kFew ? min(16 * (c % 4), 4 * words - 16) : 0));
    }
    const bool with_zeros = weights.zeros != nullptr;
    const uint32_t *codes = weights.codes + n0 * words;
    const unsigned short *scales = weights.scales + n0;
    const unsigned char *zeros = with_zeros ? weights.zeros + n0 : reinterpret_cast<const unsigned char *>(weights.scales);

    auto load = [&](Block &b, int block) {
        const int first = max(min(16 * block, words - 16), 0);  // in words of codes
        const uint32_t *block_codes = codes + first;
        const uint32_t *block_x = a.x + 4 * first;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            b.codes[t] = *reinterpret_cast<const detail::u32x4 *>(block_codes + code_offset[t]);
        }
#pragma unroll
        for (int r = 0; r < kRowTiles; r++) {
#pragma unroll
            for (int s = 0; s < Block::kXSteps; s++) {
                b.x[r][s] = *reinterpret_cast<const detail::u32x4 *>(block_x + (kFew ? 0 : min(16 * s, 4 * words - 16)) + x_offset[r]);
            }
        }
#pragma unroll
        for (int j = 0; j < kGroups; j++) {
            // a block of fewer than 128 columns has fewer groups: the last one again
            const int64_t group_row = (int64_t)min(first * 8 / (int)G + j, words * 8 / (int)G - 1) * weights.n;
#pragma unroll
            for (int t = 0; t < Block::kScaleTiles; t++) {
                b.scale[t][j] = (scales + group_row)[scale_offset[t]];
                b.zero[t][j] = (zeros + group_row)[scale_offset[t]];
            }
        }
    };

    float total[NT][kRowTiles][kSums];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int r = 0; r < kRowTiles; r++) {
#pragma unroll
            for (int e = 0; e < kSums; e++) {
                total[t][r][e] = 0.0f;
            }
        }
    }
    using Offset = detail::CodeOffset<kBf16>;
    constexpr uint32_t kOnes = Offset::ones;
    const detail::Frag ones = {{kOnes, kOnes, kOnes, kOnes}};
    const detail::f32x4 nothing = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t offsets = detail::code_offsets<kBf16>();
    auto add = [&](Block &b, int block, bool may_be_last) {
        if (may_be_last && 16 * block + 16 > words) {
            // x is zero in front of this block's columns and behind the last one
            const int first = max(min(16 * block, words - 16), 0);
#pragma unroll
            for (int r = 0; r < kRowTiles; r++) {
#pragma unroll
                for (int s = 0; s < Block::kXSteps; s++) {
                    const int word = first + 4 * (kFew ? c % 4 : s);
                    if (word < 16 * block || word >= words) {
                        b.x[r][s] = detail::u32x4{0u, 0u, 0u, 0u};
                    }
                }
            }
        }
        detail::Frag x[kRowTiles][Block::kXSteps];
#pragma unroll
        for (int r = 0; r < kRowTiles; r++) {
#pragma unroll
            for (int s = 0; s < Block::kXSteps; s++) {
                x[r][s] = detail::pair_with_fourth(__builtin_bit_cast(detail::Frag, b.x[r][s]));
            }
        }
        uint32_t block_codes[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int s = 0; s < 4; s++) {
                block_codes[t][s] = b.codes[t][s];
            }
            detail::transpose_lane_groups(block_codes[t]);
        }
        const detail::f32x4 sum_of_steps = kFew ? detail::mfma_16x16x32<kBf16>(x[0][0], ones, nothing) : nothing;
#pragma unroll
        for (int j = 0; j < kGroups; j++) {
            uint32_t scale_zero[4];  // scale in the low half, zero point above it
            if constexpr (NT >= 3) {
                detail::spread_lane_groups(b.scale[0][j] | b.zero[0][j] << 16, scale_zero);
            } else {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    scale_zero[t] = b.scale[t][j] | b.zero[t][j] << 16;
                }
            }
            float sum[kRowTiles][kSums];
#pragma unroll
            for (int r = 0; r < kRowTiles; r++) {
                if constexpr (kFew) {
                    sum[0][0] = sum_of_steps[j * kSteps];
#pragma unroll
                    for (int i = 1; i < kSteps; i++) {
                        sum[0][0] += sum_of_steps[j * kSteps + i];
                    }
                } else {
                    detail::f32x4 of_group = nothing;
#pragma unroll
                    for (int i = 0; i < kSteps; i++) {
                        of_group = detail::mfma_16x16x32<kBf16>(x[r][j * kSteps + i], ones, of_group);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sum[r][e] = of_group[e];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float dot[kRowTiles][kSums];
                if constexpr (kFew) {
                    detail::f32x4 of_step[kSteps];
#pragma unroll
                    for (int i = 0; i < kSteps; i++) {
                        of_step[i] = detail::mfma_16x16x32<kBf16>(x[0][0], detail::offset_codes<kBf16>(block_codes[t][j * kSteps + i], offsets), nothing);
                    }
                    dot[0][0] = of_step[0][j * kSteps];
#pragma unroll
                    for (int i = 1; i < kSteps; i++) {
                        dot[0][0] += of_step[i][j * kSteps + i];
                    }
                } else {
                    detail::f32x4 of_group[kRowTiles];
#pragma unroll
                    for (int r = 0; r < kRowTiles; r++) {
                        of_group[r] = nothing;
                    }
#pragma unroll
                    for (int i = 0; i < kSteps; i++) {
                        const int s = j * kSteps + i;
                        const detail::Frag w = detail::offset_codes<kBf16>(block_codes[t][s], offsets);
#pragma unroll
                        for (int r = 0; r < kRowTiles; r++) {
                            of_group[r] = detail::mfma_16x16x32<kBf16>(x[r][s], w, of_group[r]);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < kRowTiles; r++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            dot[r][e] = of_group[r][e];
                        }
                    }
                }
                const float scale = half_to_float<T>(scale_zero[t] & 0xffffu);
                constexpr float kPerOne = Offset::unit / Offset::one;
                const float zero = __builtin_fmaf(with_zeros ? (float)(scale_zero[t] >> 16) : 8.0f, -kPerOne, -kPerOne * Offset::value);
#pragma unroll
                for (int r = 0; r < kRowTiles; r++) {
#pragma unroll
                    for (int e = 0; e < kSums; e++) {
                        total[t][r][e] = __builtin_fmaf(scale, __builtin_fmaf(zero, sum[r][e], dot[r][e]), total[t][r][e]);
                    }
                }
            }
        }
    };

    int block = wave;
    if constexpr (MT <= 1 || NT == 1) {
        // The next block's loads are issued in front of this one's products, and the barriers keep them there.
        if (block < blocks) {
            Block even, odd;
            load(even, block);
            for (; block + 2 * WAVES < blocks; block += 2 * WAVES) {
                load(odd, block + WAVES);
                __builtin_amdgcn_sched_barrier(0);
                add(even, block, false);
                __builtin_amdgcn_sched_barrier(0);
                load(even, block + 2 * WAVES);
                __builtin_amdgcn_sched_barrier(0);
                add(odd, block + WAVES, false);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (block + WAVES < blocks) {
                load(odd, block + WAVES);
                __builtin_amdgcn_sched_barrier(0);
                add(even, block, true);
                add(odd, block + WAVES, true);
            } else {
                add(even, block, true);
            }
        }
    } else {
        // two blocks of x do not fit beside the sums
        for (; block < blocks; block += WAVES) {
            Block b;
            load(b, block);
            add(b, block, true);
        }
    }

    // [wavefront][tile and sum][lane]
    constexpr int kParts = NT * kRowTiles * kSums;
    __shared__ float parts[WAVES][kParts][kWaveSize];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int r = 0; r < kRowTiles; r++) {
#pragma unroll
            for (int e = 0; e < kSums; e++) {
                parts[wave][(t * kRowTiles + r) * kSums + e][lane] = total[t][r][e];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kParts * kWaveSize; i += WAVES * kWaveSize) {
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            y += parts[w][i / kWaveSize][i % kWaveSize];
        }
        y *= 1.0f / Offset::unit;
        const int from = i % kWaveSize, tile = i / kWaveSize / kSums, e = i / kWaveSize % kSums;
        const int64_t m = kFew ? from / 16 : 16 * (tile % kRowTiles) + 4 * (from / 16) + e, n = n0 + 16 * (tile / kRowTiles) + from % 16;
        if (m < a.rows && n < weights.n) {
            columns.to.y[m * columns.to.pitch + n] = (unsigned short)(pack_halves<T>(y, 0.0f) & 0xffffu);
        }
    }
}

}  // namespace gernels
