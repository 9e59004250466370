// Attention of queries over a paged 8-bit cache (gernels/serving/paged_cache.h).
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
//   y_j = z_j + log2 vs(j) (base 2) and m = max y - 15,
//   w_j = 2^(y_j - m) = 2^15 p_j vs(j) / max(...) <= 2^15,
// o = sum w_j vc_j / sum (w_j / vs(j)): the weights of the second product are at
// most 2^15 whatever the scales are, and no product is scaled twice.
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
// queries' type, summed in fp32.  The weights are rounded to fp16 because fp16
// holds every e4m3 code exactly, and their sum is taken before rounding; bf16
// weights would cost eight times that error.  Half a step is 2^-11 of a weight down
// to 2^-14, which is 2^-29 of the row's largest because that is 2^15; what is under
// that is off by 2^-40 of the largest.  (With the largest at 1, 131072 keys that are
// 13 under one whose page of values has 64 times their scale lost two thirds of what
// they add up to.)  o <= 2^15 * 448 * 2^30 keys is far from the end of fp32.
//
// Bound by memory for few queries: 2 D bytes a key and head, read once (64 requests of
// 4096 to 8192 keys, 8 heads of 128: 788 MB in 154 us, 5.1 TB/s; a copy of 1 GiB
// moves 5.2 on the same GPU).
#pragma once

#include "gernels/serving/half_tiles.h"
#include "gernels/serving/paged_cache.h"

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
    float *stats;        // [splits, tokens * query heads, 2]: taken off the exponents, sum
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

// The larger of two numbers that are not NaN.  fmaxf first quiets operands that it does not know to be results of
// arithmetic (products of the matrix cores, lanes exchanged), an instruction each; the median with infinity does not.
__device__ __forceinline__ float larger(float a, float b) {
    float infinity = __builtin_inff();
    asm("" : "+s"(infinity));  // or the compiler makes it fmaxf again
    return __builtin_amdgcn_fmed3f(a, b, infinity);
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
    return over_lane_groups(x, [](float a, float b) { return larger(a, b); });
}
__device__ __forceinline__ float sum_over_lane_groups(float x) {
    return over_lane_groups(x, [](float a, float b) { return a + b; });
}

// 0, as a value that may differ from lane to lane for all the compiler knows.
__device__ __forceinline__ int opaque_zero() {
    int zero = 0;
    asm volatile("" : "+v"(zero));
    return zero;
}

// Below every score; finite, so that a row that has seen nothing yet gives 2^(-inf - m) = 0.
constexpr float kLowest = -1.0e30f;

// log2 of a row's largest weight: the largest power of two of fp16.
constexpr float kWeightBits = 15.0f;
// What is taken off the exponents of a row with this maximum: the maximum less kWeightBits, so that its own weight is a
// power of two and not rounded; or the maximum itself where (from 2^24 on) the difference is rounded down and a weight would
// leave fp16.  (Differences of ordinary scores are off by 2^-20: that is not more.)
constexpr float kMoreThanWeightBits = 15.001f;
__device__ __forceinline__ float less_weight_bits(float most) {
    const float less = most - kWeightBits;
    return most - less > kMoreThanWeightBits ? most : less;
}

// The least scale of values, 2^-80: 2^30 weights of 2^15, each over it, add up to less than 2^126.  What is under it
// counts as 0: the softmax takes it as this, and the values are 0.
constexpr float kLeastValueScale = 8.271806125530277e-25f;

// 16 keys of one head of the cache, as they are in memory.
template<int D>
struct RawKeys {
    uint32_t k[D / 16];     // lane (g, c): key c, dimensions [g D/4, (g+1) D/4)
    uint32_t v[4][D / 64];  // lane (g, c): keys 4g .. 4g+3, dimensions [c D/16, (c+1) D/16)
    float k_scale, v_scale;
    int64_t at;             // its page and head
    bool there;             // it has keys, and their page is in the cache

    // Fragment i of K: dimensions [32 i, 32 i + 32) in the order described above.
    template<bool BF16>
    __device__ __forceinline__ Frag key_frag(int i) const {
        const uint32_t a = k[2 * i], b = k[2 * i + 1];
        return {{codes_to_halves<BF16, false>(a), codes_to_halves<BF16, true>(a), codes_to_halves<BF16, false>(b), codes_to_halves<BF16, true>(b)}};
    }
    // Half of fragment i of V^T: dimension c D/16 + i of keys 4g .. 4g+3.
    __device__ __forceinline__ Words2 value_half(int i) const {
        const uint32_t a = v[0][i / 4], b = v[1][i / 4], c = v[2][i / 4], d = v[3][i / 4];
        // v_perm_b32: selector bytes 0-3 pick from the second operand, 4-7 from the first
        const uint32_t pick = i % 4 < 2 ? 0x05010400u : 0x07030602u;
        const uint32_t ab = __builtin_amdgcn_perm(b, a, pick), cd = __builtin_amdgcn_perm(d, c, pick);
        const uint32_t column = __builtin_amdgcn_perm(cd, ab, i % 2 == 0 ? 0x05040100u : 0x07060302u);
        return {{codes_to_halves<false, false>(column), codes_to_halves<false, true>(column)}};
    }
    // What stands behind the last key may be anything, NaN too, and 0 * NaN must not reach a sum.
    __device__ __forceinline__ void clear_values_behind(int base, int length) {
        const int g = lane_id() / 16;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool keep = there && base + 4 * g + j < length;
#pragma unroll
            for (int w = 0; w < D / 64; w++) {
                v[j][w] = keep ? v[j][w] : 0u;
            }
        }
    }
    // Whether the values' scale counts as 0.
    __device__ __forceinline__ bool without_scale() const {
        return as_float(__builtin_amdgcn_readfirstlane(as_int(v_scale))) < kLeastValueScale;
    }
    __device__ __forceinline__ void clear_values_without_scale() {
        const uint32_t keep = without_scale() ? 0u : 0xffffffffu;
#pragma unroll
        for (int j = 0; j < 4; j++) {
#pragma unroll
            for (int w = 0; w < D / 64; w++) {
                v[j][w] &= keep;
            }
        }
    }
    // Makes 0 of the values that are NaN (codes 127 and 255); whether there were any.
    __device__ __forceinline__ bool take_nan() {
        uint32_t found = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
#pragma unroll
            for (int w = 0; w < D / 64; w++) {
                const uint32_t nan = ((v[j][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                v[j][w] &= ~((nan >> 7) * 0xffu);
                found |= nan;
            }
        }
        return __ballot(found != 0) != 0;
    }
};

// The scales of a tile as the softmax takes them.
struct TileScales {
    float k;      // of the scores, with the attention's own scale
    float up;     // log2 of the values' scale
    float per_v;  // one over it
    bool there;
};
template<int D>
__device__ __forceinline__ TileScales scales_of(const RawKeys<D> &tile, float scale) {
    const float v = tile.v_scale;
    const float vs = !tile.there ? 1.0f : v < kLeastValueScale ? kLeastValueScale : v;
    return {tile.k_scale * scale, __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs), tile.there};
}

// What a wavefront needs to walk the keys of one request and head.
template<int D, int PAGE>
struct KeyWalk {
    const PagedCache &cache;
    const int32_t *pages;  // the request's row of the block table
    int64_t head;
    int width;             // of the table
    int length;            // keys in the cache
    int zero;

    // The page number at key `base` (uniform; behind the table the last one).  Does not wait for `length`.  The load is a vector
    // load (`zero` is a 0 that the compiler does not see through), in order with those of the codes: a scalar load is
    // put where its value is needed and waited for there.
    __device__ __forceinline__ int look_up(int base) const {
        return pages[min(base / PAGE, width - 1) + zero];
    }
    // The 16 keys at `base`, a multiple of 16, in two halves.  Every address is inside a whole page of the cache: what
    // is not there is read from page 0.
    __device__ __forceinline__ void load_keys(RawKeys<D> &tile, int base, int looked_up) const {
        const int lane = lane_id(), g = lane / 16, c = lane % 16;
        const int id = __builtin_amdgcn_readfirstlane(looked_up);
        tile.there = id >= 0 && id < cache.pages && base < length;
        tile.at = (int64_t)(tile.there ? id : 0) * cache.heads + head;
        tile.k_scale = cache.k_scales[tile.at + zero];
        tile.v_scale = cache.v_scales[tile.at + zero];
        const uint32_t *k = cache.k + tile.at * (PAGE * D / 4) + (base % PAGE + c) * (D / 4) + g * (D / 16);
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            load_words<4>(&tile.k[4 * i], k + 4 * i);
        }
    }
    __device__ __forceinline__ void load_values(RawKeys<D> &tile, int base) const {
        const int lane = lane_id(), g = lane / 16, c = lane % 16;
        const uint32_t *v = cache.v + tile.at * (PAGE * D / 4) + (base % PAGE + 4 * g) * (D / 4) + c * (D / 64);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            load_words<D / 64>(tile.v[j], v + j * (D / 4));
        }
    }
};

// The running softmax of R tiles of 16 query rows.
template<int D, int R, bool BF16>
struct RowState {
    Frag q[R][D / 32];     // lane (g, c): row c, dimensions g D/4 + 8 s ..
    f32x4 o[R][D / 16];    // lane (g, c): row c, o[.][i][e] is dimension (4 g + e) D/16 + i
    float m[R], l[R];      // taken off the row's exponents (less_weight_bits), sum over this lane's keys
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

    // Adds the keys [base, base + 32 PAIRS): fragment i of 16-key tile t is key_frag(t, i), of V^T of the p-th pair of
    // tiles value_frag(p, i).  `whole`: every row sees all of them.  after_keys() is called when the keys' fragments have
    // been used.
    template<int PAIRS, class KeyFrag, class Scales, class AfterKeys, class ValueFrag>
    __device__ __forceinline__ void add(int base, bool whole, KeyFrag key_frag, Scales scales_of_tile, AfterKeys after_keys, ValueFrag value_frag) {
        constexpr int kTiles = 2 * PAIRS;
        const int g = lane_id() / 16;
        f32x4 s[R][kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                s[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const Frag k = key_frag(t, i);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    s[r][t] = mfma_16x16x32<BF16>(k, q[r][i], s[r][t]);
                }
            }
        }
        TileScales scales[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
            scales[t] = scales_of_tile(t);
        }
        after_keys();
        // Many rows one after the other: of 64 dimensions 32 bytes a lane are spilled otherwise (prompt pieces 101.5 us, 115.8
        // without), of 128 and 192 it is faster (300 queries 117 / 120, 161 / 175 us); of 256 it is not (199 / 188), nor with few rows.
        constexpr bool kInTurn = PAIRS > 1 && D <= 192;
        if constexpr (kInTurn) {
            __builtin_amdgcn_sched_barrier(0);
        }
        Frag p[R][PAIRS];
#pragma unroll
        for (int r = 0; r < R; r++) {
            // A score is rounded once, before the maximum is taken and before it is subtracted: however large scores are, the
            // largest one's weight is what it should be.  (In one step, s k + (up - m), it would be off by m's rounding.)
#pragma unroll
            for (int t = 0; t < kTiles; t++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[r][t][e] = __builtin_fmaf(s[r][t][e], scales[t].k, scales[t].up);
                }
            }
            if (!whole) {
#pragma unroll
                for (int t = 0; t < kTiles; t++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool seen = scales[t].there && base + 16 * t + 4 * g + e < limit[r];
                        s[r][t][e] = seen ? s[r][t][e] : -__builtin_inff();
                    }
                }
            }
            float top = kLowest;
#pragma unroll
            for (int t = 0; t < kTiles; t++) {
                const float score = larger(larger(s[r][t][0], s[r][t][1]), larger(s[r][t][2], s[r][t][3]));
                top = t == 0 ? score : larger(top, score);
            }
            top = max_over_lane_groups(top);
            const bool more = top - m[r] > kMoreThanWeightBits;
            if (__ballot(more) != 0) {
                const float now = more ? less_weight_bits(top) : m[r];
                const float shrink = __builtin_amdgcn_exp2f(m[r] - now);
                m[r] = now;
                l[r] *= shrink;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    o[r][i] *= shrink;
                }
            }
#pragma unroll
            for (int t = 0; t < kTiles; t++) {
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    y[e] = __builtin_amdgcn_exp2f(s[r][t][e] - m[r]);
                    l[r] = __builtin_fmaf(y[e], scales[t].per_v, l[r]);
                }
                p[r][t / 2].w[2 * (t % 2)] = pack_halves<F16>(y[0], y[1]);
                p[r][t / 2].w[2 * (t % 2) + 1] = pack_halves<F16>(y[2], y[3]);
            }
            if constexpr (kInTurn) {
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int pair = 0; pair < PAIRS; pair++) {
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                const Frag v = value_frag(pair, i);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    o[r][i] = mfma_16x16x32<false>(v, p[r][pair], o[r][i]);
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

// What a workgroup knows of its request, and the rows and keys of its piece.
template<int D, int PAGE, class T>
struct AttentionRequest {
    int first, queries, length;  // first row of q, rows, keys
    int group, rows;             // rows * group: rows of this head of the cache
    int split, splits;
    int64_t all_rows;

    __device__ __forceinline__ AttentionRequest(const AttentionBatchOf<T> &batch, const PagedCache &cache, const AttentionPiece &piece) {
        const int tokens = (int)batch.tokens;
        first = min(max(batch.starts[piece.request], 0), tokens);
        queries = min(max(batch.starts[piece.request + 1], first), tokens) - first;
        const int64_t room = batch.width * PAGE;
        const int asked = batch.lengths[piece.request];
        length = (int)min((int64_t)max(asked, 0), room);
        group = (int)batch.group;
        rows = queries * group;
        splits = (int)piece.to.splits;
        split = (int)piece.x % splits;
        all_rows = batch.tokens * piece.to.heads * group;
        if (asked > room && piece.x == 0 && piece.head == 0 && threadIdx.x == 0) {
            atomicAdd(cache.faults, 1u);
        }
    }
    // Keys that a row sees.
    __device__ __forceinline__ int limit(int row) const {
        return min(max(length - queries + row / group + 1, 0), length);
    }
    // Where a row's result, or its part of split `split`, is.
    __device__ __forceinline__ int64_t token(int row) const {
        return first + row / group;
    }
    __device__ __forceinline__ int64_t head(int row, const AttentionPiece &piece) const {
        return piece.head * group + row % group;
    }
    __device__ __forceinline__ int64_t part(int row, const AttentionPiece &piece) const {
        return split * all_rows + token(row) * (piece.to.heads * group) + head(row, piece);
    }
    // Where a dimension of a row's result, or of its part, is; set to NaN.
    __device__ __forceinline__ void put_nan(int row, int d, const AttentionPiece &piece) const {
        if (splits == 1) {
            reinterpret_cast<unsigned short *>(piece.to.out + token(row) * piece.to.out_pitch + head(row, piece) * (D / 2))[d] = 0x7fff;
        } else {
            piece.to.partial[part(row, piece) * D + d] = __builtin_nanf("");
        }
    }
};

// NaN among the values of keys that some rows of a workgroup see and others do not is taken out (0 * NaN must not reach a
// row that does not see the key) and put into the results of the rows that do when all are stored.  This does so for the rows
// [row, end) and the `count` keys at begin + offset, + step ... of their split: with `all` for all of them, which does no harm,
// or for those that the first row does not see.  It is rare, and reads the codes again: noted in the loop over the keys, or
// done right behind it, it would cost every call of few rows (64 requests: 177 and 160 us for 154).
template<int D, int PAGE, class T>
__device__ __forceinline__ void return_nan(const AttentionRequest<D, PAGE, T> &request, const AttentionPiece &piece, const KeyWalk<D, PAGE> &walk, int row,
                                           int end, int offset, int count, int step, bool all) {
    const int most = row < end ? request.limit(end - 1) : 0, least = all ? 0 : request.limit(row);
    const int64_t begin = (int64_t)request.split * piece.to.chunk;
    const int last = request.split + 1 < request.splits ? (int)min(begin + piece.to.chunk, (int64_t)most) : most;
    const int lane = lane_id() + opaque_zero(), quarter = lane % 4;
#pragma unroll 1
    for (int at = (int)min(begin, (int64_t)most) + offset; at < last; at += step) {
#pragma unroll 1
        for (int key = at + lane / 4; key < at + count && at + count > least; key += 16) {
            const int id = walk.pages[min(key / PAGE, walk.width - 1)];
            if (id < 0 || id >= walk.cache.pages || key >= most) {
                continue;
            }
            const uint32_t *v = walk.cache.v + ((int64_t)id * walk.cache.heads + walk.head) * (PAGE * D / 4);
            const unsigned char *codes = reinterpret_cast<const unsigned char *>(v) + key % PAGE * D;
#pragma unroll 1
            for (int d = quarter * (D / 4); d < (quarter + 1) * (D / 4); d++) {
                if ((codes[d] & 127) == 127) {
#pragma unroll 1
                    for (int r = row; r < end; r++) {
                        if (key < request.limit(r)) {
                            request.put_nan(r, d, piece);
                        }
                    }
                }
            }
        }
    }
}

// Queries and limits of the R tiles of rows from row0 on.
template<int D, int PAGE, int R, class T>
__device__ __forceinline__ void load_queries(RowState<D, R, T::kBf16> &state, const AttentionRequest<D, PAGE, T> &request, const AttentionBatchOf<T> &batch,
                                             const AttentionPiece &piece, int row0) {
    const int lane = lane_id(), g = lane / 16, c = lane % 16;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = row0 + 16 * r + c;
        const bool mine = row < request.rows;
        state.limit[r] = mine ? request.limit(row) : 0;
        const uint32_t *q = batch.q + request.token(mine ? row : 0) * batch.q_pitch + request.head(mine ? row : 0, piece) * (D / 2) + g * (D / 8);
#pragma unroll
        for (int s = 0; s < D / 32; s++) {
            load_words<4>(state.q[r][s].w, q + 4 * s);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                // the scale's sign goes to the queries
                state.q[r][s].w[w] = mine ? state.q[r][s].w[w] ^ (batch.scale < 0.0f ? 0x80008000u : 0u) : 0u;
            }
        }
    }
}

}  // namespace detail

// One piece for FEW rows (a row is a query and one of the G heads that share a head
// of the cache): 16 of them against one split of the keys.  The WAVES wavefronts
// take the 32-key tiles in turn, each from memory to its registers, and meet in
// LDS at the end.
template<int64_t D, int64_t PAGE, int64_t WAVES, class T>
__device__ __forceinline__ void attend_few_rows(const AttentionBatchOf<T> &batch, const PagedCache &cache, const AttentionPiece &piece) {
    const AttentionOut &to = piece.to;
    const int lane = lane_id(), g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const detail::AttentionRequest<D, PAGE, T> request(batch, cache, piece);
    const detail::KeyWalk<D, PAGE> walk = {cache, batch.table + piece.request * batch.width, piece.head, (int)batch.width, request.length, detail::opaque_zero()};
    const int tiles = (int)to.pieces / request.splits;

    int notes = 0;  // 1: NaN was taken, 2: keys that all rows see were not taken whole

    for (int tile = (int)piece.x / request.splits; tile * 16 < request.rows; tile += tiles) {
        const int row0 = tile * 16;
        detail::RowState<D, 1, T::kBf16> state;
        state.clear();
        detail::load_queries(state, request, batch, piece, row0);
        // keys that any / every row sees (rows behind the last one are not stored)
        const int most = request.limit(min(row0 + 16, request.rows) - 1), least = request.limit(row0);
        const int64_t begin = (int64_t)request.split * to.chunk;
        // `end` cuts a tile only where no row sees further: splits are whole tiles
        const int end = request.split + 1 < request.splits ? (int)min(begin + to.chunk, (int64_t)most) : most;
        constexpr int kStep = 32 * WAVES;
        bool missing = false;
        // Keys of the next step are loaded when this step's have been multiplied, values likewise, page numbers a step
        // before: no register is held for a load that waits, and none of the loads is waited for where it is issued.
        int base = (int)min(begin, (int64_t)most) + 32 * wave;
        detail::RawKeys<D> keys[2];
        int id[2] = {walk.look_up(base), walk.look_up(base + 16)};
        if (base < end) {
            walk.load_keys(keys[0], base, id[0]);
            walk.load_keys(keys[1], base + 16, id[1]);
            id[0] = walk.look_up(base + kStep);
            id[1] = walk.look_up(base + kStep + 16);
            walk.load_values(keys[0], base);
            walk.load_values(keys[1], base + 16);
        }
        while (base < end) {
            const bool there[2] = {keys[0].there, keys[1].there};
            const bool all_see = base + 32 <= least, whole = all_see && there[0] && there[1] && !keys[0].without_scale() && !keys[1].without_scale();
            missing = missing || !there[0] || (!there[1] && base + 16 < end);
            notes |= all_see && !whole ? 2 : 0;
            const bool more = base + kStep < end;
            state.template add<1>(
                base, whole, [&](int t, int i) { return keys[t].template key_frag<T::kBf16>(i); },
                [&](int t) { return detail::scales_of(keys[t], __builtin_fabsf(batch.scale)); },
                [&]() {
                    if (!whole) {
                        keys[0].clear_values_behind(base, request.length);
                        keys[1].clear_values_behind(base + 16, request.length);
                        notes |= keys[0].take_nan() ? 1 : 0;
                        notes |= keys[1].take_nan() ? 1 : 0;
                        keys[0].clear_values_without_scale();
                        keys[1].clear_values_without_scale();
                    }
                    if (more) {
                        walk.load_keys(keys[0], base + kStep, id[0]);
                        walk.load_keys(keys[1], base + kStep + 16, id[1]);
                        id[0] = walk.look_up(base + 2 * kStep);
                        id[1] = walk.look_up(base + 2 * kStep + 16);
                    }
                },
                [&](int, int i) {
                    const Words2 a = keys[0].value_half(i), b = keys[1].value_half(i);
                    return detail::Frag{{a.w[0], a.w[1], b.w[0], b.w[1]}};
                });
            if (more) {
                walk.load_values(keys[0], base + kStep);
                walk.load_values(keys[1], base + kStep + 16);
            }
            base += kStep;
        }
        if (missing && lane == 0) {
            atomicAdd(cache.faults, 1u);
        }
        state.l[0] = detail::sum_over_lane_groups(state.l[0]);

        // The wavefronts' parts meet in LDS; thread t then takes D / 16 values of row t / 16.
        constexpr int kPitch = D + 4;
        constexpr int kPart = D / 16;
        __shared__ __attribute__((aligned(16))) float parts[WAVES][16][kPitch];
        __shared__ float part_m[WAVES][16], part_l[WAVES][16];
        static_assert(WAVES >= 4, "256 threads share 16 rows");
        __syncthreads();  // the previous rows have been read
#pragma unroll
        for (int e = 0; e < 4; e++) {
#pragma unroll
            for (int i = 0; i < D / 16; i += 4) {
                const float x[4] = {state.o[0][i][e], state.o[0][i + 1][e], state.o[0][i + 2][e], state.o[0][i + 3][e]};
                detail::store_floats(&parts[wave][c][g * (D / 4) + e * (D / 16) + i], x);
            }
        }
        if (g == 0) {
            part_m[wave][c] = state.m[0];
            part_l[wave][c] = state.l[0];
        }
        __syncthreads();
        const int at = threadIdx.x / 16, d = (threadIdx.x % 16) * kPart, row = row0 + at;
        if (threadIdx.x < 256 && row < request.rows) {
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
            if (request.splits == 1) {
                const float per_sum = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                for (int i = 0; i < kPart; i++) {
                    x[i] *= per_sum;
                }
                detail::store_halves<T>(to.out + request.token(row) * to.out_pitch + request.head(row, piece) * (D / 2), d, x);
            } else {
                const int64_t part = request.part(row, piece);
                detail::store_floats(to.partial + part * D + d, x);
                if (d == 0) {
                    to.stats[2 * part] = m;
                    to.stats[2 * part + 1] = sum;
                }
            }
        }
    }
    __syncthreads();  // the results are stored
    if ((notes & 1) != 0) {
        for (int tile = (int)piece.x / request.splits; tile * 16 < request.rows; tile += tiles) {
            detail::return_nan(request, piece, walk, tile * 16, min(request.rows, tile * 16 + 16), 32 * wave, 32, 32 * WAVES, (notes & 2) != 0);
        }
    }
}

// One piece for MANY rows: 16 R for each of WAVES wavefronts, all against the same
// keys.  Blocks of 16 WAVES keys are staged in LDS as the fragments that the matrix
// instructions take, a 16-key tile by each wavefront: codes are converted and
// values transposed once for the whole workgroup, and fragments are read 16 bytes
// a lane without bank conflicts.  The next block's codes are loaded while this one
// is multiplied.  Per 16 rows and 32 keys a softmax of 8 scores a lane (8
// exponentials at a quarter of the rate) stands against D / 8 matrix instructions, but
// what bounds it are waits: 1.6 wavefronts a SIMD between barriers, a third of whose time
// is waiting, keep the vector ALU busy for 47 % of the time and the matrix cores for
// 13 %.  6 requests of 113 to 447 queries and 4032 to 5915 keys, 16 heads of
// 64 on 4: 30.6 GFLOP in 101 us, 15 of them the join of six splits (213 us with keys
// from memory for every wavefront).
template<int64_t D, int64_t PAGE, int64_t R, int64_t WAVES, class T>
__device__ __forceinline__ void attend_many_rows(const AttentionBatchOf<T> &batch, const PagedCache &cache, const AttentionPiece &piece) {
    constexpr int kRows = 16 * R, kTileRows = kRows * WAVES, kBlock = 16 * WAVES;
    const AttentionOut &to = piece.to;
    const int lane = lane_id(), g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const detail::AttentionRequest<D, PAGE, T> request(batch, cache, piece);
    const detail::KeyWalk<D, PAGE> walk = {cache, batch.table + piece.request * batch.width, piece.head, (int)batch.width, request.length, detail::opaque_zero()};
    const int tiles = (int)to.pieces / request.splits;
    const float scale = __builtin_fabsf(batch.scale);

    // Two buffers and one barrier a block; one and two where two would leave no room in LDS for a second workgroup.
    constexpr int kBuffers = D <= 128 ? 2 : 1;
    __shared__ __attribute__((aligned(16))) uint32_t k_frags[kBuffers][WAVES][D / 32][kWaveSize][4];
    __shared__ __attribute__((aligned(16))) uint32_t v_frags[kBuffers][WAVES / 2][D / 16][kWaveSize][4];
    __shared__ __attribute__((aligned(16))) float tile_scales[kBuffers][WAVES][4];  // k, up, per_v, 1 there | 2 NaN taken

    for (int tile = (int)piece.x / request.splits; tile * kTileRows < request.rows; tile += tiles) {
        const int row0 = tile * kTileRows + wave * kRows;
        detail::RowState<D, R, T::kBf16> state;
        state.clear();
        detail::load_queries(state, request, batch, piece, row0);
        // keys that any / every row of the workgroup, and any / every row of this wavefront sees
        const int all = request.limit(min((tile + 1) * kTileRows, request.rows) - 1), least_of_all = request.limit(tile * kTileRows);
        const int most = row0 < request.rows ? request.limit(min(row0 + kRows, request.rows) - 1) : 0;
        const int least = row0 < request.rows ? request.limit(row0) : 0;
        const int64_t begin64 = (int64_t)request.split * to.chunk;
        const int begin = (int)min(begin64, (int64_t)all);
        const int end = request.split + 1 < request.splits ? (int)min(begin64 + to.chunk, (int64_t)all) : all;
        bool missing = false, nan = false;

        detail::RawKeys<D> keys;
        auto stage = [&](int buffer, int base) {
            bool taken = false;
            if (!keys.there || keys.without_scale() || base + 16 > least_of_all) {
                keys.clear_values_behind(base, request.length);
                taken = keys.take_nan();
                keys.clear_values_without_scale();
            }
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const detail::Frag k = keys.template key_frag<T::kBf16>(i);
                *reinterpret_cast<Words4 *>(k_frags[buffer][wave][i][lane]) = Words4{{k.w[0], k.w[1], k.w[2], k.w[3]}};
            }
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                *reinterpret_cast<Words2 *>(&v_frags[buffer][wave / 2][i][lane][2 * (wave % 2)]) = keys.value_half(i);
            }
            const detail::TileScales scales = detail::scales_of(keys, scale);
            if (lane == 0) {
                const float x[4] = {scales.k, scales.up, scales.per_v, as_float((scales.there ? 1 : 0) | (taken ? 2 : 0))};
                detail::store_floats(tile_scales[buffer][wave], x);
            }
            missing = missing || (!keys.there && base < end);
        };

        __syncthreads();  // the previous rows' last block has been read
        int base = begin;
        int id = walk.look_up(base + 16 * wave);
        if (base < end) {
            walk.load_keys(keys, base + 16 * wave, id);
            id = walk.look_up(base + kBlock + 16 * wave);
            walk.load_values(keys, base + 16 * wave);
            stage(0, base + 16 * wave);
        }
        __syncthreads();
        for (int buffer = 0; base < end; buffer ^= kBuffers - 1) {
            const bool more = base + kBlock < end;
            if (more) {
                walk.load_keys(keys, base + kBlock + 16 * wave, id);
                id = walk.look_up(base + 2 * kBlock + 16 * wave);
                walk.load_values(keys, base + kBlock + 16 * wave);
            }
            if (base < min(most, end)) {
                detail::TileScales scales[WAVES];
                bool there = true;
#pragma unroll
                for (int t = 0; t < WAVES; t++) {
                    uint32_t x[4];
                    detail::load_words<4>(x, reinterpret_cast<const uint32_t *>(tile_scales[buffer][t]));
                    scales[t] = {as_float((int)x[0]), as_float((int)x[1]), as_float((int)x[2]), false};
                    const int flags = __builtin_amdgcn_readfirstlane((int)x[3]);
                    scales[t].there = (flags & 1) != 0;
                    there = there && scales[t].there;
                    nan = nan || (flags & 2) != 0;
                }
                // the whole block at once: fewer lane exchanges a key
                state.template add<WAVES / 2>(
                    base, base + kBlock <= least && there,
                    [&](int t, int i) {
                        detail::Frag k;
                        detail::load_words<4>(k.w, k_frags[buffer][t][i][lane]);
                        return k;
                    },
                    [&](int t) { return scales[t]; }, [] {},
                    [&](int pair, int i) {
                        detail::Frag v;
                        detail::load_words<4>(v.w, v_frags[buffer][pair][i][lane]);
                        return v;
                    });
            }
            if (kBuffers == 1) {
                __syncthreads();  // this block has been read
            }
            if (more) {
                stage(buffer ^ (kBuffers - 1), base + kBlock + 16 * wave);
            }
            __syncthreads();
            base += kBlock;
        }
        if (missing && lane == 0) {
            atomicAdd(cache.faults, 1u);
        }

#pragma unroll
        for (int r = 0; r < R; r++) {
            const float sum = detail::sum_over_lane_groups(state.l[r]);
            const int row = row0 + 16 * r + c;
            if (row < request.rows) {
                const float per_sum = request.splits > 1 ? 1.0f : sum != 0.0f ? 1.0f / sum : 0.0f;
                const int64_t part = request.part(row, piece);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x[D / 16];
#pragma unroll
                    for (int i = 0; i < D / 16; i++) {
                        x[i] = state.o[r][i][e] * per_sum;
                    }
                    const int d = g * (D / 4) + e * (D / 16);
                    if (request.splits == 1) {
                        detail::store_halves<T>(to.out + request.token(row) * to.out_pitch + request.head(row, piece) * (D / 2), d, x);
                    } else {
                        detail::store_floats(to.partial + part * D + d, x);
                    }
                }
                if (request.splits > 1 && g == 0) {
                    to.stats[2 * part] = state.m[r];
                    to.stats[2 * part + 1] = sum;
                }
            }
        }
        if (nan) {
            __threadfence_block();  // this wavefront's results are stored
            detail::return_nan(request, piece, walk, row0, min(request.rows, row0 + kRows), 0, 16, 16, true);
        }
    }
}

// Rows of the result from the splits' parts: PER_ROW wavefronts a row take the
// splits (at most 64 for one wavefront, 256 for a workgroup) in turn and meet in LDS,
// always in the same order.  A lane first holds the statistics of splits lane,
// lane + 64 ...  One wavefront a row pays for many rows of few splits (25472 rows, 6
// splits, 64 dimensions: 35 us with four), four for few rows of many.
constexpr int kSplitsPerLane = 4;
struct JoinRows {
    uint32_t *out;
    int64_t out_pitch;
    const float *partial, *stats;
    const int32_t *starts;
    int64_t splits, requests, q_heads;
    int64_t rows;    // tokens * query heads
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

template<int64_t D, int64_t WAVES, int64_t PER_ROW, class T>
__device__ __forceinline__ void join_splits(const AttentionBatchOf<T> &, const JoinBlock &block) {
    constexpr int kPart = D / 64;  // values a lane
    constexpr int kHeld = PER_ROW == 1 ? 1 : kSplitsPerLane;
    static_assert(PER_ROW == 1 || PER_ROW == WAVES, "a row is a wavefront's or the workgroup's");
    const JoinRows &to = block.to;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int row = (int)(block.x * (WAVES / PER_ROW)) + (PER_ROW == 1 ? wave : 0), token = row / (int)to.q_heads;
    // a row of no request has no parts
    if (row >= (int)to.rows || token < to.starts[0] || token >= to.starts[to.requests]) {
        return;
    }
    const int splits = (int)to.splits;
    float m[kHeld], l[kHeld], top = detail::kLowest;
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
        const int s = j * kWaveSize + lane;
        m[j] = detail::kLowest, l[j] = 0.0f;
        if (s < splits) {
            m[j] = to.stats[2 * (s * to.rows + row)];
            l[j] = to.stats[2 * (s * to.rows + row) + 1];
        }
        top = __builtin_fmaxf(top, m[j]);
    }
    for (int d = 1; d < kWaveSize; d *= 2) {
        top = __builtin_fmaxf(top, __shfl_xor(top, d));
    }
    float weight[kHeld], sum = 0.0f;
    int used = 0;  // splits up to the last one that saw any of the row's keys
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
        weight[j] = l[j] != 0.0f ? __builtin_amdgcn_exp2f(m[j] - top) : 0.0f;
        sum = __builtin_fmaf(l[j], weight[j], sum);
        const uint64_t some = __ballot(l[j] != 0.0f);
        used = some != 0 ? j * kWaveSize + 64 - __builtin_clzll(some) : used;
    }
    for (int d = 1; d < kWaveSize; d *= 2) {
        sum += __shfl_xor(sum, d);
    }
    const float per_sum = sum != 0.0f ? 1.0f / sum : 0.0f;
    float x[kPart];
#pragma unroll
    for (int i = 0; i < kPart; i++) {
        x[i] = 0.0f;
    }
    const float *part = to.partial + (int64_t)row * D + lane * kPart;
    uint32_t *out = to.out + token * to.out_pitch + (row % (int)to.q_heads) * (D / 2);
    auto add = [&](int s, float w) {
#pragma unroll
        for (int i = 0; i < kPart; i++) {
            // a weight of 0 as well: every split wrote its part, zeros where it saw nothing, and NaN is to stay
            x[i] = __builtin_fmaf(part[s * to.rows * D + i], w, x[i]);
        }
    };
    if constexpr (PER_ROW == 1) {
        // through LDS and not from lane to lane, so that the loop unrolls and its loads overlap; only this wavefront reads
        __shared__ float weights[WAVES][kWaveSize];
        weights[wave][lane] = weight[0];
#pragma unroll 8
        for (int s = 0; s < used; s++) {
            add(s, weights[wave][s]);
        }
        unsigned short *to_lane = reinterpret_cast<unsigned short *>(out) + lane * kPart;
#pragma unroll
        for (int i = 0; i < kPart; i++) {
            to_lane[i] = (unsigned short)(pack_halves<T>(x[i] * per_sum, 0.0f) & 0xffffu);
        }
    } else {
        __shared__ float weights[kHeld * kWaveSize];
        __shared__ float parts[WAVES][D];
#pragma unroll
        for (int j = 0; j < kHeld; j++) {
            weights[j * kWaveSize + lane] = weight[j];  // every wavefront writes the same
        }
        __syncthreads();
#pragma unroll 8
        for (int s = wave; s < used; s += WAVES) {
            add(s, weights[s]);
        }
#pragma unroll
        for (int i = 0; i < kPart; i++) {
            parts[wave][lane * kPart + i] = x[i];
        }
        __syncthreads();
        if (threadIdx.x < D / 2) {
            float a = 0.0f, b = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                a += parts[w][2 * threadIdx.x];
                b += parts[w][2 * threadIdx.x + 1];
            }
            out[threadIdx.x] = pack_halves<T>(a * per_sum, b * per_sum);
        }
    }
}

}  // namespace gernels
