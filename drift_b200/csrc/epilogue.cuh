// epilogue.cuh — epilogues of tc.cuh's products that write a matrix. A thread
// holds 128 consecutive columns of one row, row0 + lane.
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

// The 16 bytes of columns j .. of a thread's row, in the output's type.
template <class T> __device__ __forceinline__ uint4 pack16(const float *x) {
    if constexpr (sizeof(T) == 8) {
        const double2 d = make_double2(x[0], x[1]);
        return *reinterpret_cast<const uint4 *>(&d);
    } else if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                          __float_as_uint(x[3]));
    } else {
        return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                          pack2<T>(x[6], x[7]));
    }
}

__device__ __forceinline__ void smem_store16(unsigned at, uint4 w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z),
                 "r"(w.w)
                 : "memory");
}
__device__ __forceinline__ uint4 smem_load16(unsigned at) {
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "r"(at)
                 : "memory");
    return w;
}

template <class T> __device__ __forceinline__ T smem_load(unsigned at) {
    if constexpr (sizeof(T) == 8) {
        double x;
        asm volatile("ld.shared.f64 %0, [%1];" : "=d"(x) : "r"(at) : "memory");
        return x;
    } else if constexpr (sizeof(T) == 4) {
        float x;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
        return x;
    } else {
        unsigned short x;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at) : "memory");
        return *reinterpret_cast<const T *>(&x);
    }
}

// Passes a warp's 32 rows x 128 columns (lane = row) through shared memory, 128
// bytes a row at a time, so that eight lanes hold a row's 128 bytes and a store
// instruction covers four whole lines: lane by lane a store of 16 bytes would
// touch 32. The 16-byte units of a row are swizzled by its number against bank
// conflicts. `put(row, column, word)` gets 16 bytes of row row0 + row.
template <class T, class Put>
__device__ __forceinline__ void by_rows(const float (&v)[128], unsigned staging, int lane, Put put) {
    constexpr int kCols = 128 / (int)sizeof(T), kUnit = 16 / (int)sizeof(T);
#pragma unroll
    for (int c = 0; c < 128; c += kCols) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            smem_store16(staging + lane * 128 + ((j ^ (lane & 7)) << 4),
                         pack16<T>(v + c + j * kUnit));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int row = i * 4 + (lane >> 3), j = lane & 7;
            put(row, c + j * kUnit, smem_load16(staging + row * 128 + ((j ^ (row & 7)) << 4)));
        }
        __syncwarp();
    }
}

// The same where rows are not 16-byte aligned: a store instruction takes up to 32
// neighbouring elements of one row. `put(row, column, element)`. (Each lane storing
// its own row, 128 x 2 bytes in 32 lines at a time, took 40 us a tile.)
template <class T, class Put>
__device__ __forceinline__ void by_elements(const float (&v)[128], unsigned staging, int lane,
                                            Put put) {
    constexpr int kCols = 128 / (int)sizeof(T), kUnit = 16 / (int)sizeof(T);
#pragma unroll
    for (int c = 0; c < 128; c += kCols) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            smem_store16(staging + lane * 128 + ((j ^ (lane & 7)) << 4),
                         pack16<T>(v + c + j * kUnit));
        __syncwarp();
#pragma unroll 4
        for (int r = 0; r < 32; r++) {
#pragma unroll
            for (int j0 = 0; j0 < kCols; j0 += 32) {
                const int j = j0 + lane, byte = j * (int)sizeof(T);
                if (j < kCols)
                    put(r, c + j,
                        smem_load<T>(staging + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15)));
            }
        }
        __syncwarp();
    }
}

// Adds bias[col ...] to a thread's columns below `cols` (to others and without one, 0). All
// lanes want the same 128 numbers: each loads four of them, and the warp reads them
// back from shared memory. (128 loads a thread from global memory, in the few
// registers left beside v, took longer than the products of a tile up to 1024 deep:
// cross entropy of 1024 x 50176 x 512 in 88 us with a bias; 58 now, as without.)
struct Bias4 {
    float b[4];
    __device__ __forceinline__ Bias4(const float *bias, int64_t col, int64_t cols, int lane) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t i = col + j * 32 + lane;
            b[j] = bias && i < cols ? bias[i] : 0.0f;
        }
    }
};
__device__ __forceinline__ void add_bias(float (&v)[128], const Bias4 &bias, unsigned staging,
                                         int lane) {
#pragma unroll
    for (int j = 0; j < 4; j++)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(staging + (j * 32 + lane) * 4), "f"(bias.b[j])
                     : "memory");
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 128; j += 4) {
        const uint4 b = smem_load16(staging + j * 4);
        v[j] += __uint_as_float(b.x), v[j + 1] += __uint_as_float(b.y);
        v[j + 2] += __uint_as_float(b.z), v[j + 3] += __uint_as_float(b.w);
        // Here and not where the sums are used, lest both terms wait in registers.
        asm volatile("" : "+f"(v[j]), "+f"(v[j + 1]), "+f"(v[j + 2]), "+f"(v[j + 3]));
    }
    __syncwarp();
}

// C = D * alpha (+ bias), rounded once.
template <class T> struct StoreEpi {
    T *c;
    int64_t stride, rows, cols;
    const float *bias;
    const float *alpha;  // null for 1
    float beta;          // a power of two, 1 without alpha
    bool vec;
    __device__ __forceinline__ int before(int64_t, int64_t, int) const { return 0; }
    __device__ __forceinline__ void run(float (&v)[128], int, int64_t row0, int64_t col,
                                        const tc::Work &, int lane, unsigned staging) const {
        if (col >= cols) return;
        if (alpha) {
            const float f = *alpha * beta;
#pragma unroll
            for (int j = 0; j < 128; j++) v[j] *= f;
        }
        if (bias) add_bias(v, Bias4(bias, col, cols, lane), staging, lane);
        if (vec) {
            T *p = c + row0 * stride + col;
            const int64_t left = cols - col;
            by_rows<T>(v, staging, lane, [&](int r, int j, uint4 w) {
                constexpr int kUnit = 16 / (int)sizeof(T);
                if (row0 + r >= rows || j >= left) return;
                T *to = p + r * stride + j;
                if (j + kUnit <= left) {
                    *reinterpret_cast<uint4 *>(to) = w;
                } else {
                    const T *x = reinterpret_cast<const T *>(&w);
#pragma unroll
                    for (int u = 0; u < kUnit; u++)
                        if (j + u < left) to[u] = x[u];
                }
            });
        } else {
            T *p = c + row0 * stride + col;
            const int rows_left = (int)min((int64_t)32, rows - row0);
            const int left = (int)min((int64_t)128, cols - col);
            by_elements<T>(v, staging, lane, [&](int r, int j, T x) {
                if (r < rows_left && j < left) p[r * stride + j] = x;
            });
        }
    }
};

// Part `split` of C, fp32, added to or written. Each element has one writer a
// launch, so the sum's order is the launches'.
struct PartEpi {
    float *c;
    int64_t part, stride, rows, cols;  // stride a multiple of 4, c 16-byte aligned
    bool add;
    __device__ __forceinline__ int before(int64_t, int64_t, int) const { return 0; }
    __device__ __forceinline__ void run(float (&v)[128], int, int64_t row0, int64_t col,
                                        const tc::Work &w, int lane, unsigned staging) const {
        if (col >= cols) return;
        float *p = c + w.split * part + row0 * stride + col;
        by_rows<float>(v, staging, lane, [&](int r, int j, uint4 x) {
            if (row0 + r >= rows || col + j >= cols) return;  // padding columns may be written
            float *to = p + r * stride + j;
            if (add)
                asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to),
                             "f"(__uint_as_float(x.x)), "f"(__uint_as_float(x.y)),
                             "f"(__uint_as_float(x.z)), "f"(__uint_as_float(x.w))
                             : "memory");
            else
                *reinterpret_cast<uint4 *>(to) = x;
        });
    }
};

}  // namespace drift
