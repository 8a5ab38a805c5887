// epilogue.cuh — epilogues of tc.cuh's products that write a matrix: a thread
// holds 128 consecutive columns of one row.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc.cuh"

namespace drift {

template <class T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
}

// Whether rows of a matrix start on 16-byte boundaries.
template <class T> inline bool rows_aligned(const T *p, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * (int64_t)sizeof(T) % 16 == 0;
}

// Columns c0 .. c0+7 of a thread's row.
template <class T>
__device__ __forceinline__ void store8(T *p, const float *x, int64_t left, bool vec) {
    if (vec && left >= 8) {
        if constexpr (sizeof(T) == 8) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                reinterpret_cast<double2 *>(p)[j] = make_double2(x[2 * j], x[2 * j + 1]);
        } else if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]),
                                                       pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < left) p[j] = T(x[j]);
    }
}

// C = D * alpha (+ bias), rounded once.
template <class T> struct StoreEpi {
    T *c;
    int64_t stride, rows, cols;
    const float *bias;
    const float *alpha;  // a power of two, or null for 1
    bool vec;
    __device__ __forceinline__ void run(float (&v)[128], int64_t row, int64_t col, const tc::Work &,
                                        int) const {
        if (alpha) {
            const float f = *alpha;
#pragma unroll
            for (int j = 0; j < 128; j++) v[j] *= f;
        }
        if (bias) {
#pragma unroll
            for (int j = 0; j < 128; j++)
                if (col + j < cols) v[j] += __ldg(bias + col + j);
        }
        if (row >= rows) return;
        T *p = c + row * stride + col;
#pragma unroll
        for (int j = 0; j < 128; j += 8) store8(p + j, v + j, cols - col - j, vec);
    }
};

// Part `split` of C, fp32, added to or written. Each element has one writer a
// launch, so the sum's order is the launches'.
struct PartEpi {
    float *c;
    int64_t part, stride, rows, cols;  // stride a multiple of 4, c 16-byte aligned
    bool add;
    __device__ __forceinline__ void run(float (&v)[128], int64_t row, int64_t col,
                                        const tc::Work &w, int) const {
        if (row >= rows) return;
        float *p = c + w.split * part + row * stride + col;
#pragma unroll
        for (int j = 0; j < 128; j += 4) {
            if (col + j >= cols) break;  // the stride's padding columns may be written
            if (add)
                asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + j),
                             "f"(v[j]), "f"(v[j + 1]), "f"(v[j + 2]), "f"(v[j + 3])
                             : "memory");
            else
                *reinterpret_cast<float4 *>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
    }
};

}  // namespace drift
