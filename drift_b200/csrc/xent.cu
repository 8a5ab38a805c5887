// xent.cu — a linear layer with softmax cross entropy over its outputs, in
// pieces of the vocabulary, and its gradients; no more logits are held than one
// piece's.
//
//   l = x W^T + b       lse_i = log sum_v exp l_iv       loss_i = lse_i - l_i,t(i)
//   d_iv = (exp(l_iv - lse_i) - [v = t(i)]) g_i
//   dx = d W            dW = d^T x            db_v = sum_i d_iv
//
// x and W are bf16 (or fp16), sums and statistics fp32.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "internal.h"

namespace drift {

template <class T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

// C (+)= A B^T: A(i, k) at A[i*a_r + k*a_k], B(o, k) at B[o*b_r + k*b_k], 64 x 64
// outputs a CTA.
template <class TA, class TB, class TC>
__global__ void __launch_bounds__(256) simple_gemm_kernel(int64_t M, int64_t N, int64_t K,
                                                          const TA *A, int64_t a_r, int64_t a_k,
                                                          const TB *B, int64_t b_r, int64_t b_k,
                                                          TC *C, int64_t c_r, bool add) {
    __shared__ float sa[32][65], sb[32][65];
    const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += 32) {
        for (int i = tid; i < 64 * 32; i += 256) {
            const int ra = a_k == 1 ? i >> 5 : i & 63, ka = a_k == 1 ? i & 31 : i >> 6;
            const int rb = b_k == 1 ? i >> 5 : i & 63, kb = b_k == 1 ? i & 31 : i >> 6;
            sa[ka][ra] = m0 + ra < M && k0 + ka < K
                             ? to_f(A[(m0 + ra) * a_r + (k0 + ka) * a_k]) : 0.0f;
            sb[kb][rb] = n0 + rb < N && k0 + kb < K
                             ? to_f(B[(n0 + rb) * b_r + (k0 + kb) * b_k]) : 0.0f;
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
            if (row < M && col < N) {
                TC *c = C + row * c_r + col;
                *c = TC(add ? to_f(*c) + acc[i][j] : acc[i][j]);
            }
        }
    }
}

struct XentRows {
    const void *targets;
    bool wide;  // int64 targets, else int32
    int64_t ignore, vocab;
    // The target of row i; negative for an ignored row. One outside the
    // vocabulary sets `bad` and counts as ignored.
    __device__ int64_t at(int64_t i, bool &bad) const {
        const int64_t t = wide ? static_cast<const int64_t *>(targets)[i]
                               : (int64_t) static_cast<const int32_t *>(targets)[i];
        if (t == ignore) return -1;
        if (t < 0 || t >= vocab) {
            bad = true;
            return -1;
        }
        return t;
    }
};

// Maximum that keeps a NaN, so that a row with one has a NaN log sum.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Joins a piece's logits to the running maximum, sum and target logit of a row.
__global__ void __launch_bounds__(256) xent_stats_kernel(const float *logits, int64_t n,
                                                         int64_t v0, const float *bias,
                                                         XentRows rows, float *run, int *err) {
    __shared__ float sm[8], ss[8];
    const int64_t i = blockIdx.x;
    const float *l = logits + i * n;
    float m = -INFINITY, s = 0.0f;
    for (int64_t v = threadIdx.x; v < n; v += 256) {
        const float x = l[v] + (bias ? bias[v0 + v] : 0.0f);
        const float top = max_nan(m, x);
        if (top > -INFINITY) s = s * expf(m - top) + expf(x - top);
        m = top;
    }
    for (int o = 16; o; o >>= 1) {
        const float m2 = __shfl_xor_sync(~0u, m, o), s2 = __shfl_xor_sync(~0u, s, o);
        const float top = max_nan(m, m2);
        if (top > -INFINITY) s = s * expf(m - top) + s2 * expf(m2 - top);
        m = top;
    }
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m, ss[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        float *r = run + 3 * i;
        if (v0) m = r[0], s = r[1];
        else m = -INFINITY, s = 0.0f;
        for (int w = 0; w < 8; w++) {
            const float top = max_nan(m, sm[w]);
            if (top > -INFINITY) s = s * expf(m - top) + ss[w] * expf(sm[w] - top);
            m = top;
        }
        r[0] = m, r[1] = s;
        bool bad = false;
        const int64_t t = rows.at(i, bad);
        if (bad) atomicOr(err, DEV_ERR_INDEX);
        if (t >= v0 && t < v0 + n) r[2] = l[t - v0] + (bias ? bias[t] : 0.0f);
    }
}

// Losses and log sums of the rows from their running statistics; one CTA, so
// that the mean over the counted rows is summed in a fixed order.
__global__ void __launch_bounds__(1024) xent_finish_kernel(const float *run, int64_t T,
                                                           XentRows rows, float *loss, float *lse,
                                                           float *mean) {
    __shared__ float sl[1024];
    __shared__ int sc[1024];
    float sum = 0.0f;
    int count = 0;
    for (int64_t i = threadIdx.x; i < T; i += 1024) {
        const float z = run[3 * i] + logf(run[3 * i + 1]);
        bool bad = false;
        const bool on = rows.at(i, bad) >= 0;
        const float l = on ? z - run[3 * i + 2] : 0.0f;
        lse[i] = z;
        if (loss) loss[i] = l;
        sum += l;
        count += on;
    }
    if (!mean) return;
    sl[threadIdx.x] = sum, sc[threadIdx.x] = count;
    __syncthreads();
    for (int o = 512; o; o >>= 1) {
        if (threadIdx.x < o) sl[threadIdx.x] += sl[threadIdx.x + o], sc[threadIdx.x] += sc[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float c = (float)max(sc[0], 1);
        mean[0] = sl[0] / c;
        mean[1] = 1.0f / c;
    }
}

// A piece's logits to its part of d, in place.
__global__ void __launch_bounds__(256) xent_dlogits_kernel(float *logits, int64_t n, int64_t v0,
                                                           const float *bias, XentRows rows,
                                                           const float *lse, const float *g,
                                                           int64_t g_stride) {
    const int64_t i = blockIdx.x;
    bool bad = false;
    const int64_t t = rows.at(i, bad);
    const float z = lse[i], gi = t >= 0 ? g[i * g_stride] : 0.0f;
    for (int64_t v = threadIdx.x; v < n; v += 256) {
        const float p = expf(logits[i * n + v] + (bias ? bias[v0 + v] : 0.0f) - z);
        logits[i * n + v] = t >= 0 ? (p - (v0 + v == t ? 1.0f : 0.0f)) * gi : 0.0f;
    }
}

__global__ void __launch_bounds__(256) xent_colsum_kernel(const float *d, int64_t T, int64_t n,
                                                          float *db) {
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v >= n) return;
    float s = 0.0f;
    for (int64_t i = 0; i < T; i++) s += d[i * n + v];
    db[v] = s;
}

template <class T>
__global__ void __launch_bounds__(256) narrow_kernel(const float *x, T *y, int64_t rows,
                                                     int64_t cols, int64_t stride) {
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < rows * cols; i += 256LL * gridDim.x)
        y[i / cols * stride + i % cols] = T(x[i]);
}

static int64_t xent_piece(const drift_xent *op) {
    const int64_t fit = (256LL << 20) / 4 / std::max<int64_t>(op->tokens, 1);
    return std::max<int64_t>(64, std::min(op->vocab, fit / 64 * 64));
}

int64_t xent_workspace(const drift_xent *op, bool grad) {
    const int64_t run = (op->tokens * 3 * 4 + 255) / 256 * 256;
    return run + op->tokens * xent_piece(op) * 4 + (grad ? op->tokens * op->depth * 4 : 0) + 256;
}

static dim3 tiles(int64_t m, int64_t n) {
    return dim3((unsigned)((m + 63) / 64), (unsigned)((n + 63) / 64));
}

static XentRows rows_of(const drift_xent *op) {
    return XentRows{op->targets, op->target_bits == 64, op->ignore_index, op->vocab};
}

template <class T>
static int xent_forward(const drift_xent *op, float *loss, float *lse, float *mean, char *ws,
                        int *err, cudaStream_t st) {
    const int64_t n_t = op->tokens, piece = xent_piece(op);
    float *run = (float *)ws, *logits = (float *)(ws + (n_t * 12 + 255) / 256 * 256);
    for (int64_t v0 = 0; n_t && v0 < op->vocab; v0 += piece) {
        const int64_t n = std::min(piece, op->vocab - v0);
        simple_gemm_kernel<<<tiles(n_t, n), 256, 0, st>>>(
            n_t, n, op->depth, (const T *)op->x, op->x_stride, 1,
            (const T *)op->w + v0 * op->w_stride, op->w_stride, 1, logits, n, false);
        xent_stats_kernel<<<(unsigned)n_t, 256, 0, st>>>(logits, n, v0, op->bias, rows_of(op), run,
                                                         err);
    }
    xent_finish_kernel<<<1, 1024, 0, st>>>(run, n_t, rows_of(op), loss, lse, mean);
    return cudaGetLastError() == cudaSuccess ? DRIFT_OK : DRIFT_ECUDA;
}

template <class T>
static int xent_backward(const drift_xent *op, const float *lse, const float *g, int64_t g_stride,
                         void *dx, int64_t dx_stride, void *dw, int64_t dw_stride, float *db,
                         char *ws, int *err, cudaStream_t st) {
    (void)err;
    const int64_t n_t = op->tokens, d = op->depth, piece = xent_piece(op);
    if (n_t == 0) {
        if (dw) cudaMemset2DAsync(dw, dw_stride * 2, 0, d * 2, op->vocab, st);
        if (db) cudaMemsetAsync(db, 0, op->vocab * 4, st);
        return cudaGetLastError() == cudaSuccess ? DRIFT_OK : DRIFT_ECUDA;
    }
    float *acc = (float *)ws, *logits = (float *)(ws + (n_t * d * 4 + 255) / 256 * 256);
    for (int64_t v0 = 0; v0 < op->vocab; v0 += piece) {
        const int64_t n = std::min(piece, op->vocab - v0);
        const T *w = (const T *)op->w + v0 * op->w_stride;
        simple_gemm_kernel<<<tiles(n_t, n), 256, 0, st>>>(n_t, n, d, (const T *)op->x,
                                                          op->x_stride, 1, w, op->w_stride, 1,
                                                          logits, n, false);
        xent_dlogits_kernel<<<(unsigned)n_t, 256, 0, st>>>(logits, n, v0, op->bias, rows_of(op),
                                                           lse, g, g_stride);
        if (dx)
            simple_gemm_kernel<<<tiles(n_t, d), 256, 0, st>>>(n_t, d, n, logits, n, 1, w, 1,
                                                              op->w_stride, acc, d, v0 > 0);
        if (dw)
            simple_gemm_kernel<<<tiles(n, d), 256, 0, st>>>(
                n, d, n_t, logits, 1, n, (const T *)op->x, 1, op->x_stride,
                (T *)dw + v0 * dw_stride, dw_stride, false);
        if (db)
            xent_colsum_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(logits, n_t, n,
                                                                            db + v0);
    }
    if (dx) narrow_kernel<<<sm_count() * 4, 256, 0, st>>>(acc, (T *)dx, n_t, d, dx_stride);
    return cudaGetLastError() == cudaSuccess ? DRIFT_OK : DRIFT_ECUDA;
}

int launch_xent(const drift_xent *op, float *loss, float *lse, float *mean, void *ws, int *err,
                cudaStream_t st) {
    return op->type == DRIFT_T_BF16
               ? xent_forward<__nv_bfloat16>(op, loss, lse, mean, (char *)ws, err, st)
               : xent_forward<__half>(op, loss, lse, mean, (char *)ws, err, st);
}

int launch_xent_grad(const drift_xent *op, const float *lse, const float *g, int64_t g_stride,
                     void *dx, int64_t dx_stride, void *dw, int64_t dw_stride, float *db, void *ws,
                     int *err, cudaStream_t st) {
    return op->type == DRIFT_T_BF16
               ? xent_backward<__nv_bfloat16>(op, lse, g, g_stride, dx, dx_stride, dw, dw_stride,
                                              db, (char *)ws, err, st)
               : xent_backward<__half>(op, lse, g, g_stride, dx, dx_stride, dw, dw_stride, db,
                                       (char *)ws, err, st);
}

}  // namespace drift
