// Attention of queries over a paged 8-bit cache (gernels/paged_cache.h).
//
// Request r has n queries (consecutive tokens) and holds `length` keys; with
// G query heads to a head of the cache, query i of head h' = h G + u sees the
// keys j <= length - n + i:
//
//   z_j = scale * ks(j) * (q . kc_j)        ks, vs: scales of key j's page
//   o   = sum_j softmax(z)_j * vs(j) * vc_j         0 where nothing is seen
//
// One pass over the keys with the running maximum and sum of the softmax, in
// fp32.  The value scale goes into the exponent: with
//   y_j = z_j + log2 vs(j) (base 2) and m = max y,
//   w_j = 2^(y_j - m) = p_j vs(j) / max(...) <= 1,
// o = sum w_j vc_j / sum (w_j / vs(j)): the weights of the second product are at
// most 1 whatever the scales are, and no product is scaled twice.
//
// On the matrix cores, transposed so that nothing crosses lanes:
//   S^T = K Q^T: 16 keys x 16 query rows a v_mfma_16x16x32; lane (g, c), c = lane
//         mod 16, g = lane / 16, holds keys 4g .. 4g+3 of query row c
//   O^T = V^T P^T: exactly those four keys (of two 16-key tiles) are what lane
//         (g, c) supplies of P^T, so P stays in the registers it was computed in;
//         the k index of the product runs over the keys in that order
//   the row statistics of query row c live in the lanes with that c; their
//         maximum takes two lane exchanges
// The head dimension's order inside K Q^T is free as long as both agree: lane
// group g takes the g-th quarter of the row, 16 bytes at a time.
// V arrives as rows of D bytes; lane c takes bytes [c D/16, (c+1) D/16) of eight
// rows and transposes 4 x 4 bytes in registers (two v_perm a word), so O^T's tile
// i holds dimension c D/16 + i and a lane ends up with D/4 consecutive values.
//
// Precision: codes go to bf16 / fp16 exactly.  Q.K is exact products in the
// queries' type, summed in fp32.  The weights are rounded to fp16 (half a step is
// 2^-11 of a weight) because fp16 holds every e4m3 code exactly, and their sum is
// taken before rounding; bf16 weights would cost eight times that error.
//
// Bound by memory for few queries: 2 D bytes a key and head, read once.  Codes
// are loaded one 32-key step ahead, page numbers two.
#pragma once

#include "gernels/half_tiles.h"
#include "gernels/paged_cache.h"

namespace gernels {

template<class T>
struct AttentionBatchOf {
    const uint32_t *q;        // two values a word; heads of a token are contiguous
    int64_t q_pitch;          // words from token to token
    const int32_t *table;     // [requests, width]
    const int32_t *lengths;   // [requests]
    const int32_t *starts;    // [requests + 1]
    int64_t width;
    int64_t tokens;           // rows of q
    int64_t group;            // query heads per head of the cache
    float scale;              // times log2(e)

    __device__ __forceinline__ const AttentionBatchOf &whole() const {
        return *this;
    }
};

struct AttentionPiece;
struct AttentionOut {
    uint32_t *out;       // two values a word
    int64_t out_pitch;   // words
    float *partial;      // [splits, tokens * query heads, D], with splits > 1
    float *stats;        // [splits, tokens * query heads, 2]: maximum, sum
    int64_t splits;      // of the keys, `chunk` each (the last one takes the rest)
    int64_t chunk;
    int64_t pieces;      // workgroups per request and head: row tiles * splits
    int64_t heads;
    int64_t requests;

    __device__ __forceinline__ AttentionPiece piece(int64_t x, int64_t head, int64_t request) const;
};
struct AttentionPiece {
    const AttentionOut &to;
    int64_t x, head, request;
};
__device__ __forceinline__ AttentionPiece AttentionOut::piece(int64_t x, int64_t head, int64_t request) const {
    return {*this, x, head, request};
}

namespace detail {

// Two e4m3 codes (the low or the high two of a word) as bf16 or fp16; exact.
template<bool BF16, bool HIGH>
__device__ __forceinline__ uint32_t codes_to_halves(uint32_t w) {
    if constexpr (BF16) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
    } else {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
    }
}

// Maximum / sum over the four lanes with the same lane mod 16.
template<class F>
__device__ __forceinline__ float over_lane_groups(float x, F combine) {
    const auto a = __builtin_amdgcn_permlane32_swap(as_int(x), as_int(x), false, false);
    x = combine(as_float((int)a[0]), as_float((int)a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(as_int(x), as_int(x), false, false);
    return combine(as_float((int)b[0]), as_float((int)b[1]));
}
__device__ __forceinline__ float max_over_lane_groups(float x) {
    return over_lane_groups(x, [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_lane_groups(float x) {
    return over_lane_groups(x, [](float a, float b) { return a + b; });
}

// Below every score; finite, so that a row that has seen nothing yet gives 2^(-inf - m) = 0.
constexpr float kLowest = -1.0e30f;

// 32 keys of one head of the cache: two tiles of 16, each inside a page.
template<int D>
struct KeyTile {
    uint32_t k[2][D / 16];  // lane (g, c): key c of tile t, dimensions [g D/4, (g+1) D/4)
    uint32_t v[8][D / 64];  // lane (g, c): key 4g + j of tile j / 4, dimensions [c D/16, (c+1) D/16)
    float k_scale[2], v_scale[2];
    bool there[2];          // the tile's page is in the cache
};

// What a wavefront needs to walk the keys of one request and head.
template<int D, int PAGE>
struct KeyWalk {
    const PagedCache &cache;
    const int32_t *pages;  // the request's row of the block table
    int64_t head;
    int length;            // keys in the cache

    // Page numbers of the two tiles at key `base` (uniform); -1 behind the last key.
    __device__ __forceinline__ void look_up(int base, int id[2]) const {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            id[t] = base + 16 * t < length ? pages[(base + 16 * t) / PAGE] : -1;
        }
    }
    // Every address is inside a whole page of the cache: what is not there is read from page 0.
    __device__ __forceinline__ void load(KeyTile<D> &tile, int base, const int id[2]) const {
        const int lane = lane_id(), g = lane / 16, c = lane % 16;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            tile.there[t] = id[t] >= 0 && id[t] < cache.pages;
            const int64_t at = (int64_t)(tile.there[t] ? id[t] : 0) * cache.heads + head;
            const int place = (base + 16 * t) % PAGE;
            const uint32_t *k = cache.k + at * (PAGE * D / 4) + (place + c) * (D / 4) + g * (D / 16);
            const uint32_t *v = cache.v + at * (PAGE * D / 4) + (place + 4 * g) * (D / 4) + c * (D / 64);
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
                load_words<4>(&tile.k[t][4 * i], k + 4 * i);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                load_words<D / 64>(tile.v[4 * t + j], v + j * (D / 4));
            }
            tile.k_scale[t] = cache.k_scales[at];
            tile.v_scale[t] = cache.v_scales[at];
        }
    }
};

// The running softmax of R tiles of 16 query rows.
template<int D, int R, bool BF16>
struct RowState {
    Frag q[R][D / 32];     // lane (g, c): row c, dimensions g D/4 + 8 s ..
    f32x4 o[R][D / 16];    // lane (g, c): row c, o[.][i][e] is dimension (4 g + e) D/16 + i
    float m[R], l[R];      // maximum over the row, sum over this lane's keys
    int limit[R];          // keys that row c sees

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; r++) {
            m[r] = kLowest;
            l[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                o[r][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
    }

    // Adds the keys [base, base + 32).  `whole`: every row sees all of them.
    __device__ __forceinline__ void add(KeyTile<D> &tile, int base, int length, bool whole, float scale) {
        const int lane = lane_id(), g = lane / 16;
        f32x4 s[R][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                s[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const uint32_t a = tile.k[t][2 * i], b = tile.k[t][2 * i + 1];
                const Frag k = {{codes_to_halves<BF16, false>(a), codes_to_halves<BF16, true>(a), codes_to_halves<BF16, false>(b),
                                 codes_to_halves<BF16, true>(b)}};
#pragma unroll
                for (int r = 0; r < R; r++) {
                    s[r][t] = mfma_16x16x32<BF16>(k, q[r][i], s[r][t]);
                }
            }
        }
        float up[2], per_v[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            // a scale under 2^-64 counts as that (its codes are zero, or too small to matter)
            float vs = tile.v_scale[t] < 5.421010862e-20f ? 5.421010862e-20f : tile.v_scale[t];
            vs = whole || (tile.there[t] && base + 16 * t < length) ? vs : 1.0f;
            up[t] = __builtin_amdgcn_logf(vs);  // base 2
            per_v[t] = __builtin_amdgcn_rcpf(vs);
        }
        Frag p[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            float y[8];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const float ks = tile.k_scale[t] * scale;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    y[4 * t + e] = __builtin_fmaf(s[r][t][e], ks, up[t]);
                }
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const bool seen = tile.there[j / 4] && base + 16 * (j / 4) + 4 * g + j % 4 < limit[r];
                    y[j] = seen ? y[j] : -__builtin_inff();
                }
            }
            float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(y[0], y[1]), __builtin_fmaxf(y[2], y[3])),
                                        __builtin_fmaxf(__builtin_fmaxf(y[4], y[5]), __builtin_fmaxf(y[6], y[7])));
            top = max_over_lane_groups(top);
            if (__ballot(top > m[r]) != 0) {
                const float now = __builtin_fmaxf(top, m[r]);
                const float shrink = __builtin_amdgcn_exp2f(m[r] - now);
                m[r] = now;
                l[r] *= shrink;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    o[r][i] *= shrink;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                y[j] = __builtin_amdgcn_exp2f(y[j] - m[r]);
                l[r] = __builtin_fmaf(y[j], per_v[j / 4], l[r]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                p[r].w[j] = pack_halves<F16>(y[2 * j], y[2 * j + 1]);
            }
        }
        if (!whole) {
            // what stands behind the last key may be anything, NaN too: 0 * NaN must not reach the sum
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool keep = tile.there[j / 4] && base + 16 * (j / 4) + 4 * g + j % 4 < length;
#pragma unroll
                for (int w = 0; w < D / 64; w++) {
                    tile.v[j][w] = keep ? tile.v[j][w] : 0u;
                }
            }
        }
#pragma unroll
        for (int w = 0; w < D / 64; w++) {
            uint32_t column[2][4];  // [tile][byte of the word]: four keys of one dimension
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t a = tile.v[4 * t][w], b = tile.v[4 * t + 1][w], c = tile.v[4 * t + 2][w], d = tile.v[4 * t + 3][w];
                // v_perm_b32: selector bytes 0-3 pick from the second operand, 4-7 from the first
                const uint32_t ab_low = __builtin_amdgcn_perm(b, a, 0x05010400u), ab_high = __builtin_amdgcn_perm(b, a, 0x07030602u);
                const uint32_t cd_low = __builtin_amdgcn_perm(d, c, 0x05010400u), cd_high = __builtin_amdgcn_perm(d, c, 0x07030602u);
                column[t][0] = __builtin_amdgcn_perm(cd_low, ab_low, 0x05040100u);
                column[t][1] = __builtin_amdgcn_perm(cd_low, ab_low, 0x07060302u);
                column[t][2] = __builtin_amdgcn_perm(cd_high, ab_high, 0x05040100u);
                column[t][3] = __builtin_amdgcn_perm(cd_high, ab_high, 0x07060302u);
            }
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const Frag v = {{codes_to_halves<false, false>(column[0][b]), codes_to_halves<false, true>(column[0][b]),
                                 codes_to_halves<false, false>(column[1][b]), codes_to_halves<false, true>(column[1][b])}};
#pragma unroll
                for (int r = 0; r < R; r++) {
                    o[r][4 * w + b] = mfma_16x16x32<false>(v, p[r], o[r][4 * w + b]);
                }
            }
        }
    }
};

// N values of a row of the result, from element d on.
template<class T, int N>
__device__ __forceinline__ void store_halves(uint32_t *row, int d, const float (&x)[N]) {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        w[i] = pack_halves<T>(x[2 * i], x[2 * i + 1]);
    }
    uint32_t *to = row + d / 2;
    if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            *reinterpret_cast<Words4 *>(to + 4 * i) = Words4{{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]}};
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            *reinterpret_cast<Words2 *>(to + 2 * i) = Words2{{w[2 * i], w[2 * i + 1]}};
        }
    }
}

template<int N>
__device__ __forceinline__ void store_floats(float *to, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        *reinterpret_cast<Words4 *>(to + 4 * i) =
            Words4{{(uint32_t)as_int(x[4 * i]), (uint32_t)as_int(x[4 * i + 1]), (uint32_t)as_int(x[4 * i + 2]), (uint32_t)as_int(x[4 * i + 3])}};
    }
}

}  // namespace detail

// One piece: R tiles of 16 query rows (a row is a query and one of the G heads
// that share a head of the cache) against one split of the keys, on WAVES
// wavefronts.  KEYS: the wavefronts take the 32-key tiles in turn and meet in LDS
// at the end; otherwise each takes R row tiles of its own and all walk the same
// keys, which then come from the CU's cache for all but the first.
template<int64_t D, int64_t PAGE, int64_t R, int64_t WAVES, int64_t KEYS, class T>
__device__ __forceinline__ void attend(const AttentionBatchOf<T> &batch, const PagedCache &cache, const AttentionPiece &piece) {
    constexpr int kRows = 16 * R;                            // of a wavefront
    constexpr int kTileRows = KEYS ? kRows : kRows * WAVES;  // of a workgroup
    constexpr bool kBf16 = T::kBf16;
    const AttentionOut &to = piece.to;
    const int lane = lane_id(), g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int splits = (int)to.splits, split = (int)piece.x % splits, tiles = (int)to.pieces / splits;
    const int group = (int)batch.group;

    const int tokens = (int)batch.tokens;
    const int first = min(max(batch.starts[piece.request], 0), tokens);
    const int queries = min(max(batch.starts[piece.request + 1], first), tokens) - first;
    const int64_t room = batch.width * PAGE;
    const int asked = batch.lengths[piece.request];
    const int length = (int)min((int64_t)max(asked, 0), room);
    const int rows = queries * group;
    if (asked > room && piece.x == 0 && piece.head == 0 && threadIdx.x == 0) {
        atomicAdd(cache.faults, 1u);
    }
    const detail::KeyWalk<D, PAGE> walk = {cache, batch.table + piece.request * batch.width, piece.head, length};
    const int64_t all_rows = batch.tokens * to.heads * group;

    for (int tile = (int)piece.x / splits; tile * kTileRows < rows; tile += tiles) {
        const int row0 = tile * kTileRows + (KEYS ? 0 : wave * kRows);
        detail::RowState<D, R, kBf16> state;
        state.clear();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int row = row0 + 16 * r + c;
            const int i = row / group, u = row % group;
            state.limit[r] = row < rows ? min(max(length - queries + i + 1, 0), length) : 0;
            const uint32_t *q = batch.q + (first + (row < rows ? i : 0)) * batch.q_pitch + (piece.head * group + (row < rows ? u : 0)) * (D / 2) + g * (D / 8);
#pragma unroll
            for (int s = 0; s < D / 32; s++) {
                detail::load_words<4>(state.q[r][s].w, q + 4 * s);
                if (row >= rows) {
                    state.q[r][s] = detail::Frag{{0u, 0u, 0u, 0u}};
                }
            }
        }
        // keys that any / every row of this wavefront sees
        const int last_row = min(row0 + kRows, rows) - 1;
        const int most = row0 < rows ? min(max(length - queries + last_row / group + 1, 0), length) : 0;
        const int least = row0 + kRows <= rows ? min(max(length - queries + row0 / group + 1, 0), length)
                                               : min(most, max(length - queries + row0 / group + 1, 0));
        const int64_t begin64 = (int64_t)split * to.chunk;
        const int begin = (int)min(begin64, (int64_t)most);
        const int end = split + 1 < splits ? (int)min(begin64 + to.chunk, (int64_t)most) : most;
        constexpr int kStep = KEYS ? 32 * WAVES : 32;
        bool missing = false;

        auto add = [&](detail::KeyTile<D> &keys, int base) {
            // `end` cuts a tile only where no row sees further: splits are whole tiles
            const bool whole = base + 32 <= least && keys.there[0] && keys.there[1];
            missing = missing || (!keys.there[0] && base < end) || (!keys.there[1] && base + 16 < end);
            state.add(keys, base, length, whole, batch.scale);
        };
        int base = begin + (KEYS ? 32 * wave : 0);
        if (base < end) {
            detail::KeyTile<D> even, odd;
            int id[2], next_id[2];
            walk.look_up(base, id);
            walk.look_up(base + kStep, next_id);
            walk.load(even, base, id);
            while (true) {
                if (base + kStep < end) {
                    walk.load(odd, base + kStep, next_id);
                    walk.look_up(base + 2 * kStep, next_id);
                }
                add(even, base);
                base += kStep;
                if (base >= end) {
                    break;
                }
                if (base + kStep < end) {
                    walk.load(even, base + kStep, next_id);
                    walk.look_up(base + 2 * kStep, next_id);
                }
                add(odd, base);
                base += kStep;
                if (base >= end) {
                    break;
                }
            }
        }
        if (missing && lane == 0) {
            atomicAdd(cache.faults, 1u);
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            state.l[r] = detail::sum_over_lane_groups(state.l[r]);
        }

        if constexpr (KEYS != 0) {
            // The wavefronts' parts meet in LDS; thread t then takes D / 16 values of row t / 16.
            constexpr int kPitch = D + 4;
            constexpr int kPart = D / 16;
            __shared__ __attribute__((aligned(16))) float parts[WAVES][16][kPitch];
            __shared__ float part_m[WAVES][16], part_l[WAVES][16];
            static_assert(WAVES == 4, "256 threads share 16 rows");
#pragma unroll
            for (int r = 0; r < R; r++) {
                __syncthreads();  // the previous rows have been read
#pragma unroll
                for (int e = 0; e < 4; e++) {
#pragma unroll
                    for (int i = 0; i < D / 16; i += 4) {
                        const float x[4] = {state.o[r][i][e], state.o[r][i + 1][e], state.o[r][i + 2][e], state.o[r][i + 3][e]};
                        detail::store_floats(&parts[wave][c][g * (D / 4) + e * (D / 16) + i], x);
                    }
                }
                if (g == 0) {
                    part_m[wave][c] = state.m[r];
                    part_l[wave][c] = state.l[r];
                }
                __syncthreads();
                const int at = threadIdx.x / 16, d = (threadIdx.x % 16) * kPart;
                const int row = row0 + 16 * r + at;
                float m = part_m[0][at];
#pragma unroll
                for (int w = 1; w < WAVES; w++) {
                    m = __builtin_fmaxf(m, part_m[w][at]);
                }
                float sum = 0.0f, x[kPart];
#pragma unroll
                for (int i = 0; i < kPart; i++) {
                    x[i] = 0.0f;
                }
#pragma unroll
                for (int w = 0; w < WAVES; w++) {
                    const float weight = __builtin_amdgcn_exp2f(part_m[w][at] - m);
                    sum = __builtin_fmaf(part_l[w][at], weight, sum);
#pragma unroll
                    for (int i = 0; i < kPart; i++) {
                        x[i] = __builtin_fmaf(parts[w][at][d + i], weight, x[i]);
                    }
                }
                if (row < rows) {
                    const int64_t token = first + row / group, head = piece.head * group + row % group;
                    if (splits == 1) {
                        const float per_sum = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                        for (int i = 0; i < kPart; i++) {
                            x[i] *= per_sum;
                        }
                        detail::store_halves<T>(to.out + token * to.out_pitch + head * (D / 2), d, x);
                    } else {
                        const int64_t slot = split * all_rows + token * (to.heads * group) + head;
                        detail::store_floats(to.partial + slot * D + d, x);
                        if (d == 0) {
                            to.stats[2 * slot] = m;
                            to.stats[2 * slot + 1] = sum;
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int row = row0 + 16 * r + c;
                if (row < rows) {
                    const int64_t token = first + row / group, head = piece.head * group + row % group;
                    const float per_sum = splits > 1 ? 1.0f : state.l[r] != 0.0f ? 1.0f / state.l[r] : 0.0f;
                    const int64_t slot = split * all_rows + token * (to.heads * group) + head;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x[D / 16];
#pragma unroll
                        for (int i = 0; i < D / 16; i++) {
                            x[i] = state.o[r][i][e] * per_sum;
                        }
                        const int d = g * (D / 4) + e * (D / 16);
                        if (splits == 1) {
                            detail::store_halves<T>(to.out + token * to.out_pitch + head * (D / 2), d, x);
                        } else {
                            detail::store_floats(to.partial + slot * D + d, x);
                        }
                    }
                    if (splits > 1 && g == 0) {
                        to.stats[2 * slot] = state.m[r];
                        to.stats[2 * slot + 1] = state.l[r];
                    }
                }
            }
        }
    }
}

// Rows of the result from the splits' parts, in the order of the splits (at most
// 64): one wavefront a row, lane s first holds the statistics of split s.
struct JoinRows {
    uint32_t *out;
    int64_t out_pitch;
    const float *partial, *stats;
    const int32_t *starts;
    int64_t splits, requests, q_heads, rows;
    int64_t blocks;  // workgroups

    __device__ __forceinline__ struct JoinBlock block(int64_t x) const;
};
struct JoinBlock {
    const JoinRows &to;
    int64_t x;
};
__device__ __forceinline__ JoinBlock JoinRows::block(int64_t x) const {
    return {*this, x};
}

template<int64_t D, int64_t WAVES, class T>
__device__ __forceinline__ void join_splits(const AttentionBatchOf<T> &, const JoinBlock &block) {
    constexpr int kPart = D / 64;  // values a lane
    const JoinRows &to = block.to;
    const int lane = lane_id();
    const int64_t row = block.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int64_t token = row / to.q_heads;
    if (row >= to.rows || token < to.starts[0] || token >= to.starts[to.requests]) {
        return;
    }
    float m = detail::kLowest, l = 0.0f;
    if (lane < to.splits) {
        m = to.stats[2 * (lane * to.rows + row)];
        l = to.stats[2 * (lane * to.rows + row) + 1];
    }
    float top = m;
    for (int d = 1; d < kWaveSize; d *= 2) {
        top = __builtin_fmaxf(top, __shfl_xor(top, d));
    }
    const float weight = l != 0.0f ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
    float sum = l * weight;
    for (int d = 1; d < kWaveSize; d *= 2) {
        sum += __shfl_xor(sum, d);
    }
    float x[kPart];
#pragma unroll
    for (int i = 0; i < kPart; i++) {
        x[i] = 0.0f;
    }
    for (int s = 0; s < to.splits; s++) {
        const float w = as_float(__builtin_amdgcn_readlane(as_int(weight), s));
        // a split that saw none of the row's keys left its part unwritten or zero
        if (w != 0.0f) {
            const float *part = to.partial + (s * to.rows + row) * D + lane * kPart;
#pragma unroll
            for (int i = 0; i < kPart; i++) {
                x[i] = __builtin_fmaf(part[i], w, x[i]);
            }
        }
    }
    const float per_sum = sum != 0.0f ? 1.0f / sum : 0.0f;
    unsigned short *out = reinterpret_cast<unsigned short *>(to.out + token * to.out_pitch + (row % to.q_heads) * (D / 2)) + lane * kPart;
#pragma unroll
    for (int i = 0; i < kPart; i++) {
        out[i] = (unsigned short)(pack_halves<T>(x[i] * per_sum, 0.0f) & 0xffffu);
    }
}

}  // namespace gernels
