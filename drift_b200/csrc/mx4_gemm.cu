// mx4_gemm.cu — the product of two packed 4-bit matrices:
//
//   C[i, o] = sum_k a[i, k] b[o, k]  (+ bias[o])
//
// with a and b the values that codes and scales stand for. The tensor cores
// multiply the codes and apply the scales (tcgen05 kind::mxf4, one scale per 32
// elements); sums are fp32 in TMEM and round once on the way out.
#include <algorithm>

#include "epilogue.cuh"
#include "internal.h"
#include "mx4.cuh"
#include "mx4_thin.cuh"
#include "tc.cuh"

namespace drift {

static bool encode_codes(CUtensorMap *map, const drift_mx4 *q, uint32_t rows) {
    const uint64_t bytes = (uint64_t)mx4_row_bytes(q->cols);
    return tc::encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, q->codes, bytes, q->rows, bytes, 128,
                         rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Rows of scale tiles, 256 words (two tiles) a stage; `box` rows at a time.
static bool encode_scales(CUtensorMap *map, const drift_mx4 *q, uint32_t box) {
    const uint64_t words = (uint64_t)mx4_k_tiles(q->cols) * 128;
    return tc::encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, q->scales, words,
                         mx4_row_tiles(q->rows), words * 4, 256, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// K = 0: the sum of nothing.
template <class T>
__global__ void __launch_bounds__(256) fill_bias_kernel(T *C, int64_t stride, int64_t rows,
                                                        int64_t cols, const float *bias) {
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < rows * cols; i += 256LL * gridDim.x)
        C[i / cols * stride + i % cols] = T(bias ? bias[i % cols] : 0.0f);
}

// Estimated hundredths of a microsecond, from products of 129 x 2048 x 2048 to 2048
// x 4096 x 4096 measured both ways (within a tenth of the pairs' times, a fifth of the
// thin ones'): a wave of pair tiles takes 0.41 us a stage and 2.2, a wave of thin CTAs
// 0.5 a stage and 2.2, or 5 where one CTA has a whole contraction and writes alone.
static int64_t pair_cost(int64_t m, int64_t n, int64_t stages, int sms) {
    const int64_t tiles = (m + tc::kTile - 1) / tc::kTile * ((n + tc::kTile - 1) / tc::kTile);
    return (tiles + sms / 2 - 1) / (sms / 2) * (41 * stages + 220);
}
static int64_t thin_cost(int64_t tiles, int64_t stages, int split, int slots) {
    return (tiles * split + slots - 1) / slots * (50 * ((stages + split - 1) / split) + (split > 1 ? 220 : 500));
}
// How many CTAs share a thin tile's contraction: up to four, or a portable
// cluster's eight where tiles are few. (Sixteen clusters of eight did not all fit
// the GPU at once: 64 x 2048 x 2048 took 9.8 us with them and 4.7 with fours.)
static int thin_split(int64_t tiles, int64_t stages, int slots) {
    int best = 1;
    for (int s = 2; s <= (tiles <= 9 ? 8 : 4) && s <= stages; s++)
        if (thin_cost(tiles, stages, s, slots) < thin_cost(tiles, stages, best, slots)) best = s;
    return best;
}

template <int NT, class T>
static int gemm_thin(const drift_mx4 *a, const drift_mx4 *b, const float *bias, T *C,
                     int64_t c_stride, int *d_err, cudaStream_t st) {
    thin::Args args;
    if (!encode_codes(&args.w, b, 128) || !encode_codes(&args.x, a, NT) ||
        !encode_scales(&args.sfw, b, 1) || !encode_scales(&args.sfx, a, 1))
        return DRIFT_ECUDA;
    args.rows = b->rows, args.tokens = a->rows;
    args.w_tiles = (int)((b->rows + 127) / 128);
    args.k_stages = (int)((a->cols + 255) / 256);
    args.bias = bias;
    args.c = C, args.stride = c_stride;
    args.vec = rows_aligned(C, c_stride);
    args.err = d_err;
    const int t_tiles = (int)((a->rows + NT - 1) / NT);
    const int split = thin_split((int64_t)args.w_tiles * t_tiles, args.k_stages,
                                 sm_count() * thin::Shape<NT>::per_sm);
    return thin::launch<NT, T>(args, t_tiles, split, st);
}

template <class T>
static int gemm(const drift_mx4 *a, const drift_mx4 *b, const float *bias, T *C, int64_t c_stride,
                int *d_err, cudaStream_t st) {
    if (a->cols == 0) {
        fill_bias_kernel<<<sm_count() * 2, 256, 0, st>>>(C, c_stride, a->rows, b->rows, bias);
        return cudaGetLastError() == cudaSuccess ? DRIFT_OK : DRIFT_ECUDA;
    }
    // Up to 128 rows the thin kernel wastes no lanes; beyond, few pair tiles leave SMs
    // idle that its smaller tiles and shared contractions reach.
    const int sms = sm_count();
    const int64_t stages = (a->cols + 255) / 256;
    const int64_t thin_tiles = (a->rows + 127) / 128 * ((b->rows + 127) / 128);
    if (a->rows <= 128 || thin_cost(thin_tiles, stages, thin_split(thin_tiles, stages, sms), sms) <
                              pair_cost(a->rows, b->rows, stages, sms)) {
        if (a->rows <= 16) return gemm_thin<16>(a, b, bias, C, c_stride, d_err, st);
        if (a->rows <= 32) return gemm_thin<32>(a, b, bias, C, c_stride, d_err, st);
        if (a->rows <= 64) return gemm_thin<64>(a, b, bias, C, c_stride, d_err, st);
        return gemm_thin<128>(a, b, bias, C, c_stride, d_err, st);
    }
    tc::Args args;
    if (!encode_codes(&args.a, a, 128) || !encode_codes(&args.b, b, 128) ||
        !encode_scales(&args.sfa, a, 1) || !encode_scales(&args.sfb, b, 2))
        return DRIFT_ECUDA;
    args.m_tiles = (int)((a->rows + tc::kTile - 1) / tc::kTile);
    args.n_tiles = (int)((b->rows + tc::kTile - 1) / tc::kTile);
    args.k_stages = (int)((a->cols + 255) / 256);
    args.splits = 1;
    args.err = d_err;
    const StoreEpi<T> epi{C, c_stride, a->rows, b->rows, bias, nullptr, 1.0f,
                          rows_aligned(C, c_stride)};
    return tc::launch<tc::KIND_MX4, false, false, false>(args, epi, sms, st);
}

int launch_mx4_gemm(const drift_mx4 *a, const drift_mx4 *b, const float *bias, int type, void *C,
                    int64_t c_stride, int *d_err, cudaStream_t st) {
    switch (type) {
        case DRIFT_T_F64: return gemm(a, b, bias, (double *)C, c_stride, d_err, st);
        case DRIFT_T_F32: return gemm(a, b, bias, (float *)C, c_stride, d_err, st);
        case DRIFT_T_BF16: return gemm(a, b, bias, (__nv_bfloat16 *)C, c_stride, d_err, st);
        default: return gemm(a, b, bias, (__half *)C, c_stride, d_err, st);
    }
}

}  // namespace drift
