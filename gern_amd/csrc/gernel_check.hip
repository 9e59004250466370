// Ahead-of-time instantiation of every gernel for gfx950: the build check.
// The kernels that run are instantiated by hiprtc from generated code; this
// file only proves that the library compiles with hipcc as well.
#include "gernels/blur.h"
#include "gernels/softmax.h"

template<int64_t col, int64_t row, int64_t stride>
__global__ void __launch_bounds__(64) check_blur_xyx(gernels::MatrixF32 input, gernels::MatrixF32 output) {
    const int64_t y = blockIdx.x * col;
    const int64_t x = blockIdx.y * row;
    auto out_tile = output.template view_wave<row, col>(x, y);
    auto t2 = gernels::allocate_wave_tile<row, col + stride - 1>();
    auto t1 = gernels::allocate_wave_tile<row + stride - 1, col + stride - 1>();
    auto in_tile = input.template load_wave<row + stride - 1, col + 2 * (stride - 1)>(x, y);
    gernels::blur_x<stride>(in_tile, t1);
    gernels::blur_y<stride>(t1, t2);
    gernels::blur_x<stride>(t2, out_tile);
    output.store_wave(x, y, out_tile);
}
template __global__ void check_blur_xyx<252, 8, 3>(gernels::MatrixF32, gernels::MatrixF32);
template __global__ void check_blur_xyx<248, 4, 5>(gernels::MatrixF32, gernels::MatrixF32);

template<int64_t ncol, int64_t row>
__global__ void __launch_bounds__(64) check_softmax(gernels::MatrixF32 input, gernels::MatrixF32 output) {
    const int64_t x = blockIdx.x * row;
    auto in_tile = input.template load_wave<row, ncol>(x, 0);
    auto vec = gernels::allocate_wave_vec<row>();
    gernels::max_row(vec, in_tile);
    auto t = gernels::allocate_wave_tile<row, ncol>();
    gernels::subtract_vec(vec, in_tile, t);
    auto e = gernels::allocate_wave_tile<row, ncol>();
    gernels::exp_matrix(t, e);
    gernels::sum_row(vec, e);
    auto out_tile = output.template view_wave<row, ncol>(x, 0);
    gernels::divide_vec(vec, e, out_tile);
    output.store_wave(x, 0, out_tile);
}
template __global__ void check_softmax<4096, 1>(gernels::MatrixF32, gernels::MatrixF32);
template __global__ void check_softmax<1000, 2>(gernels::MatrixF32, gernels::MatrixF32);

#include "gernels/mm.h"

template<int64_t BM, int64_t BN, int64_t KC>
__global__ void __launch_bounds__(256) check_gemm_bf16(gernels::MatrixBF16 A, gernels::MatrixBF16 B, gernels::MatrixF32 C) {
    const int64_t i = blockIdx.y * BM, j = blockIdx.x * BN;
    auto acc = C.template load_acc_mfma<BM, BN>(i, j);
    for (int64_t k = 0; k < A.col; k += KC) {
        auto a = A.template view<BM, KC>(i, k);
        auto b = B.template view<KC, BN>(k, j);
        gernels::matrix_multiply(a, b, acc);
    }
    C.add_acc(i, j, acc);
}
template __global__ void check_gemm_bf16<256, 256, 4096>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32);
template __global__ void check_gemm_bf16<128, 128, 4096>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32);

template<int64_t BM, int64_t BN, int64_t KC>
__global__ void __launch_bounds__(512) check_gemm_bf16_8waves(gernels::MatrixBF16 A, gernels::MatrixBF16 B, gernels::MatrixF32 C) {
    const int64_t i = blockIdx.y * BM, j = blockIdx.x * BN;
    auto acc = C.template load_acc_mfma8<BM, BN>(i, j);
    for (int64_t k = 0; k < A.col; k += KC) {
        auto a = A.template view_exact<BM, KC>(i, k);
        auto b = B.template view_exact<KC, BN>(k, j);
        gernels::matrix_multiply(a, b, acc);
    }
    C.store_acc(i, j, acc);
}
template __global__ void check_gemm_bf16_8waves<256, 256, 4096>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32);

template<int64_t BM, int64_t BN, int64_t KC, bool ADD>
__global__ void __launch_bounds__(512) check_gemm_bf16_16x16x32(gernels::MatrixBF16 A, gernels::MatrixBF16 B, gernels::MatrixF32 C) {
    const int64_t i = blockIdx.y * BM, j = blockIdx.x * BN;
    auto acc = C.template load_acc_mfma16<BM, BN>(i, j);
    for (int64_t k = 0; k < A.col; k += KC) {
        auto a = A.template view_exact<BM, KC>(i, k);
        auto b = B.template view_exact<KC, BN>(k, j);
        gernels::matrix_multiply(a, b, acc);
    }
    if (ADD) {
        C.add_acc(i, j, acc);
    } else {
        C.store_acc(i, j, acc);
    }
}
template __global__ void check_gemm_bf16_16x16x32<256, 256, 4096, false>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32);
template __global__ void check_gemm_bf16_16x16x32<256, 256, 4096, true>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32);

template<int64_t BM, int64_t BN, int64_t KC>
__global__ void __launch_bounds__(256) check_gemm_f32(gernels::MatrixF32 A, gernels::MatrixF32 B, gernels::MatrixF32 C) {
    const int64_t i = blockIdx.y * BM, j = blockIdx.x * BN;
    auto acc = C.template load_acc_fma<BM, BN>(i, j);
    for (int64_t k = 0; k < A.col; k += KC) {
        auto a = A.template view<BM, KC>(i, k);
        auto b = B.template view<KC, BN>(k, j);
        gernels::matrix_multiply(a, b, acc);
    }
    C.store_acc(i, j, acc);
}
template __global__ void check_gemm_f32<128, 128, 4096>(gernels::MatrixF32, gernels::MatrixF32, gernels::MatrixF32);

template<int64_t BM, int64_t BN, int64_t KC>
__global__ void __launch_bounds__(512) check_gemm_f32_mfma(gernels::MatrixF32 A, gernels::MatrixF32 B, gernels::MatrixF32 C) {
    const int64_t i = blockIdx.y * BM, j = blockIdx.x * BN;
    auto acc = C.template load_acc_mfma8_f32<BM, BN>(i, j);
    for (int64_t k = 0; k < A.col; k += KC) {
        auto a = A.template view_exact<BM, KC>(i, k);
        auto b = B.template view_exact<KC, BN>(k, j);
        gernels::matrix_multiply(a, b, acc);
    }
    C.add_acc(i, j, acc);
}
template __global__ void check_gemm_f32_mfma<256, 256, 4096>(gernels::MatrixF32, gernels::MatrixF32, gernels::MatrixF32);

#include "gernels/qk_softmax.h"

template<int64_t N, int64_t D>
__global__ void __launch_bounds__(64 * gernels::qk_waves(N)) check_qk_softmax(gernels::MatrixBF16 Q, gernels::MatrixBF16 K, gernels::MatrixF32 S,
                                                        float scale) {
    const int64_t x = blockIdx.x * 16;
    auto q = Q.template view<16, D>(x, 0);
    auto k = K.template view<N, D>(0, 0);
    auto logits = gernels::allocate_row_block<16, N>();
    gernels::qk_scaled(q, k, logits, scale);
    auto stat = gernels::allocate_row_stat<16>();
    gernels::max_row(stat, logits);
    auto shifted = gernels::allocate_row_block<16, N>();
    gernels::subtract_vec(stat, logits, shifted);
    auto expd = gernels::allocate_row_block<16, N>();
    gernels::exp_matrix(shifted, expd);
    gernels::sum_row(stat, expd);
    auto out = S.template view_row_block<16, N>(x, 0);
    gernels::divide_vec(stat, expd, out);
    S.store_row_block(x, 0, out);
}
template __global__ void check_qk_softmax<4096, 128>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32, float);
template __global__ void check_qk_softmax<1024, 64>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32, float);

#include "gernels/qk_tiles.h"

// The tile program of the fused QK^T softmax: one workgroup per 256 x 256 tile of S.
template<int64_t D>
__global__ void __launch_bounds__(512) check_qk_softmax_tiles(gernels::MatrixBF16 Q, gernels::MatrixBF16 K, gernels::MatrixF32 S,
                                                             gernels::RowStatsExchange exchange, float scale) {
    const int64_t x = (int64_t)blockIdx.y * 256, y = (int64_t)blockIdx.x * 256;
    auto session = exchange.open();
    auto out = S.template view_score_tile<256, 256>(x, y);
    auto logits = gernels::allocate_score_tile<256, 256>();
    auto q = Q.template view<256, D>(x, 0);
    auto k = K.template view<256, D>(y, 0);
    gernels::qk_scaled(q, k, logits, scale);
    gernels::softmax_rows_across_tiles(logits, session, out);
    S.store_score_tile(x, y, out);
}
template __global__ void check_qk_softmax_tiles<128>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32, gernels::RowStatsExchange, float);
template __global__ void check_qk_softmax_tiles<192>(gernels::MatrixBF16, gernels::MatrixBF16, gernels::MatrixF32, gernels::RowStatsExchange, float);

#include "gernels/serving/cache_attention.h"
#include "gernels/serving/cache_write.h"
#include "gernels/serving/page_table.h"

template<int64_t PER>
__global__ void __launch_bounds__(1024) check_page_table(gernels::RequestLengths batch, gernels::FreePages free_pages, gernels::PageTableOut table) {
    auto share = table.share(blockIdx.x);
    gernels::extend_page_table<16, 1024, PER>(batch.whole(), free_pages.whole(), share);
}
template __global__ void check_page_table<1>(gernels::RequestLengths, gernels::FreePages, gernels::PageTableOut);
template __global__ void check_page_table<8>(gernels::RequestLengths, gernels::FreePages, gernels::PageTableOut);

template<int64_t D, int64_t PAGE, int64_t THREADS, class T>
__global__ void __launch_bounds__(THREADS) check_write_cache(gernels::NewTokensOf<T> tokens, gernels::WritableCache cache) {
    auto stretch = cache.at(blockIdx.x);
    gernels::write_cache<D, PAGE, THREADS>(tokens.whole(), stretch);
}
template __global__ void check_write_cache<128, 16, 64, gernels::Bf16>(gernels::NewTokensOf<gernels::Bf16>, gernels::WritableCache);
template __global__ void check_write_cache<64, 128, 256, gernels::F16>(gernels::NewTokensOf<gernels::F16>, gernels::WritableCache);

template<int64_t D, int64_t PAGE, class T>
__global__ void __launch_bounds__(256, D <= 64 ? 4 : D <= 128 ? 3 : 2) check_attend_few(gernels::AttentionBatchOf<T> batch, gernels::PagedCache cache, gernels::AttentionOut result) {
    auto piece = result.piece(blockIdx.x, blockIdx.y, blockIdx.z);
    gernels::attend_few_rows<D, PAGE, 4>(batch.whole(), cache.whole(), piece);
}
template<int64_t D, int64_t PAGE, int64_t R, class T>
__global__ void __launch_bounds__(256, 2) check_attend_many(gernels::AttentionBatchOf<T> batch, gernels::PagedCache cache, gernels::AttentionOut result) {
    auto piece = result.piece(blockIdx.x, blockIdx.y, blockIdx.z);
    gernels::attend_many_rows<D, PAGE, R, 4>(batch.whole(), cache.whole(), piece);
}
template __global__ void check_attend_few<64, 32, gernels::Bf16>(gernels::AttentionBatchOf<gernels::Bf16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_few<128, 64, gernels::Bf16>(gernels::AttentionBatchOf<gernels::Bf16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_few<128, 16, gernels::F16>(gernels::AttentionBatchOf<gernels::F16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_few<192, 16, gernels::F16>(gernels::AttentionBatchOf<gernels::F16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_few<256, 16, gernels::F16>(gernels::AttentionBatchOf<gernels::F16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_many<64, 32, 2, gernels::Bf16>(gernels::AttentionBatchOf<gernels::Bf16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_many<128, 16, 2, gernels::F16>(gernels::AttentionBatchOf<gernels::F16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_many<192, 64, 1, gernels::Bf16>(gernels::AttentionBatchOf<gernels::Bf16>, gernels::PagedCache, gernels::AttentionOut);
template __global__ void check_attend_many<256, 16, 1, gernels::F16>(gernels::AttentionBatchOf<gernels::F16>, gernels::PagedCache, gernels::AttentionOut);

template<int64_t D, int64_t PER_ROW, class T>
__global__ void __launch_bounds__(256) check_join_splits(gernels::AttentionBatchOf<T> batch, gernels::JoinRows rows) {
    auto block = rows.block(blockIdx.x);
    gernels::join_splits<D, 4, PER_ROW>(batch.whole(), block);
}
template __global__ void check_join_splits<192, 4, gernels::Bf16>(gernels::AttentionBatchOf<gernels::Bf16>, gernels::JoinRows);
template __global__ void check_join_splits<64, 1, gernels::F16>(gernels::AttentionBatchOf<gernels::F16>, gernels::JoinRows);

#include "gernels/serving/matvec4.h"

template<int64_t G, int64_t MT, int64_t NT, class T>
__global__ void __launch_bounds__(512) check_matvec4(gernels::ActivationsOf<T> x, gernels::Weights4 weights, gernels::MatvecOut y) {
    auto columns = y.at(blockIdx.x);
    gernels::multiply_4bit<G, MT, NT, 8>(x.whole(), weights.whole(), columns);
}
template __global__ void check_matvec4<128, 0, 1, gernels::Bf16>(gernels::ActivationsOf<gernels::Bf16>, gernels::Weights4, gernels::MatvecOut);
template __global__ void check_matvec4<128, 0, 4, gernels::Bf16>(gernels::ActivationsOf<gernels::Bf16>, gernels::Weights4, gernels::MatvecOut);
template __global__ void check_matvec4<32, 0, 4, gernels::F16>(gernels::ActivationsOf<gernels::F16>, gernels::Weights4, gernels::MatvecOut);
template __global__ void check_matvec4<128, 1, 1, gernels::Bf16>(gernels::ActivationsOf<gernels::Bf16>, gernels::Weights4, gernels::MatvecOut);
template __global__ void check_matvec4<64, 1, 4, gernels::F16>(gernels::ActivationsOf<gernels::F16>, gernels::Weights4, gernels::MatvecOut);
template __global__ void check_matvec4<64, 2, 4, gernels::F16>(gernels::ActivationsOf<gernels::F16>, gernels::Weights4, gernels::MatvecOut);
template __global__ void check_matvec4<32, 4, 4, gernels::F16>(gernels::ActivationsOf<gernels::F16>, gernels::Weights4, gernels::MatvecOut);

// The layouts of what the host hands to these gernels (annot/paged_cache.h, annot/matvec4.h ask the same of its mirrors).
namespace gernels {
static_assert(sizeof(PagedCache) == 56 && offsetof(PagedCache, faults) == 48);
static_assert(sizeof(WritableCache) == 72);
static_assert(sizeof(NewTokensOf<Bf16>) == 48 && offsetof(NewTokensOf<Bf16>, tokens) == 40);
static_assert(sizeof(RequestLengths) == 24 && offsetof(RequestLengths, requests) == 16);
static_assert(sizeof(FreePages) == 24 && offsetof(FreePages, capacity) == 16);
static_assert(sizeof(PageTableOut) == 64 && offsetof(PageTableOut, shares) == 56);
static_assert(sizeof(AttentionBatchOf<F16>) == 72 && offsetof(AttentionBatchOf<F16>, scale) == 64);
static_assert(sizeof(AttentionOut) == 72 && offsetof(AttentionOut, requests) == 64);
static_assert(sizeof(JoinRows) == 80 && offsetof(JoinRows, blocks) == 72);
static_assert(sizeof(ActivationsOf<F16>) == 24 && offsetof(ActivationsOf<F16>, rows) == 16);
static_assert(sizeof(Weights4) == 40 && offsetof(Weights4, k) == 32);
static_assert(sizeof(MatvecOut) == 24 && offsetof(MatvecOut, columns) == 16);
}  // namespace gernels
