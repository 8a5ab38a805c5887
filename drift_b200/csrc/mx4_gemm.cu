// mx4_gemm.cu — the product of two packed 4-bit matrices:
//
//   C[i, o] = sum_k a[i, k] b[o, k]  (+ bias[o])
//
// with a and b the values that codes and scales stand for and the sum in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "mx4.cuh"

namespace drift {

__device__ __forceinline__ float mx_code_value(unsigned c) {
    const unsigned m = c & 7;
    const float v = m < 2 ? 0.5f * m : (float)((2 + (m & 1)) << (m >> 1)) * 0.25f;
    return c & 8 ? -v : v;
}

__device__ __forceinline__ float mx_scale_value(unsigned s) {
    return s ? __uint_as_float(s << 23) : 0x1p-127f;
}

struct MxOperand {
    const uint8_t *codes, *scales;
    int64_t rows;
};

// 64 x 64 outputs a CTA, 4 x 4 a thread, one block of 32 at a time through
// shared memory.
template <class T>
__global__ void __launch_bounds__(256) mx4_gemm_simple_kernel(MxOperand A, MxOperand B, int64_t K,
                                                              const float *bias, T *C,
                                                              int64_t c_stride) {
    __shared__ float sa[32][65], sb[32][65];
    const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t blocks = mx4_blocks(K), k_tiles = mx4_k_tiles(K);
    float acc[4][4] = {};
    for (int64_t kb = 0; kb < blocks; kb++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const MxOperand &X = h ? B : A;
            float(*s)[65] = h ? sb : sa;
            const int r = tid >> 2, q = tid & 3;  // four threads a row, eight codes each
            const int64_t row = (h ? n0 : m0) + r;
            unsigned w = 0;
            float scale = 0.0f;
            if (row < X.rows) {
                w = *reinterpret_cast<const unsigned *>(X.codes + row * blocks * 16 + kb * 16 +
                                                        q * 4);
                scale = mx_scale_value(X.scales[mx4_scale_offset(row, kb, k_tiles)]);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) s[q * 8 + j][r] = mx_code_value(w >> (4 * j) & 15) * scale;
        }
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < 32; k++) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = sa[k][ty + 16 * i], b[i] = sb[k][tx + 16 * i];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t row = m0 + ty + 16 * i, col = n0 + tx + 16 * j;
            if (row < A.rows && col < B.rows)
                C[row * c_stride + col] = T(acc[i][j] + (bias ? bias[col] : 0.0f));
        }
    }
}

int64_t mx4_gemm_workspace(int64_t M, int64_t N, int64_t K) {
    (void)M, (void)N, (void)K;
    return 0;
}

int launch_mx4_gemm(const drift_mx4 *a, const drift_mx4 *b, const float *bias, int type, void *C,
                    int64_t c_stride, void *ws, int *d_err, cudaStream_t st) {
    (void)ws, (void)d_err;
    const MxOperand A{a->codes, a->scales, a->rows}, B{b->codes, b->scales, b->rows};
    const dim3 grid((unsigned)((a->rows + 63) / 64), (unsigned)((b->rows + 63) / 64));
    switch (type) {
        case DRIFT_T_F64:
            mx4_gemm_simple_kernel<<<grid, 256, 0, st>>>(A, B, a->cols, bias, (double *)C, c_stride);
            break;
        case DRIFT_T_F32:
            mx4_gemm_simple_kernel<<<grid, 256, 0, st>>>(A, B, a->cols, bias, (float *)C, c_stride);
            break;
        case DRIFT_T_BF16:
            mx4_gemm_simple_kernel<<<grid, 256, 0, st>>>(A, B, a->cols, bias, (__nv_bfloat16 *)C,
                                                         c_stride);
            break;
        default:
            mx4_gemm_simple_kernel<<<grid, 256, 0, st>>>(A, B, a->cols, bias, (__half *)C,
                                                         c_stride);
    }
    return cudaGetLastError() == cudaSuccess ? DRIFT_OK : DRIFT_ECUDA;
}

}  // namespace drift
