// adamw.cu — one AdamW step over a list of tensors in one launch, moments in
// 32 bits or in 8 bits with one scale per 256 elements.
//
// Every element does, in 32 bits, each operation rounded on its own
// (-fmad=false; the order is part of the definition, so a plain evaluation in
// the same order gives the same bits):
//
//   m' = b1 m + (1-b1) g          v' = b2 v + ((1-b2) g) g        r = sqrt(v')
//   p' = (1 - lr wd) p - (lr/(1-b1^t) m') / (r / sqrt(1-b2^t) + eps)
//
// In 8 bits the first moment is held as e4m3 codes of m * (448 / amax) and
// the second as e4m3 codes of its root r, which spans half the binades that v
// does. p' uses the moments before they are rounded to codes.
//
// Bound: HBM bytes. 32-bit moments with fp32 parameters and bf16 gradients
// move 26 bytes an element, 8-bit moments with bf16 parameters and gradients
// 10.1. One warp owns a block of 256 elements, eight a lane, so a block's
// amax is five shuffles and every access is one or two 16-byte loads or
// stores a lane.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "internal.h"

namespace drift {

constexpr int kAdamThreads = 256;
constexpr int kAdamBlock = 256;                     // elements that share a scale
constexpr int kAdamBlocksPerWarp = 2;
constexpr int kAdamChunk = kAdamBlock * (kAdamThreads / 32) * kAdamBlocksPerWarp;
constexpr int kAdamTensors = 128;                   // tensors of one launch

struct AdamTensor {
    void *p;
    const void *g;
    void *m, *v;
    float *ms, *vs;
    void *copy;
    int64_t n;
    uint64_t first_draw;  // stochastic rounding: index of the tensor's first draw
    int8_t pt, gt, ct;    // DRIFT_T_*; ct < 0: no copy
    int8_t vec;           // every array starts on a 16-byte boundary (8 for codes)
};

struct AdamArgs {
    AdamTensor t[kAdamTensors];
    uint32_t first[kAdamTensors + 1];  // first chunk of each tensor
    int count;
    float b1, b2, c1, c2, eps;
    const float *scal;        // lr/(1-b1^t), 1/sqrt(1-b2^t), 1 - lr wd
    const uint64_t *rng;      // Rng state of this step's draws
    const float *grad_scale;  // may be null
};

// The step's scalars, in double and rounded once; advances the step count and
// the Rng state, so that a captured call replays as the next step.
__global__ void adamw_prepare_kernel(int64_t *step, double b1, double b2, double lr,
                                     const float *d_lr, double wd, float *scal, uint64_t *rng,
                                     uint64_t draws, uint64_t *rng_used) {
    const int64_t t = *step + 1;
    *step = t;
    if (d_lr) lr = (double)*d_lr;
    scal[0] = (float)(lr / (1.0 - pow(b1, (double)t)));
    scal[1] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    scal[2] = (float)(1.0 - lr * wd);
    if (rng) {
        *rng_used = *rng;
        *rng += draws * kGolden;
    }
}

__device__ __forceinline__ float half_bits_to_float(uint16_t h, int type) {
    return type == DRIFT_T_BF16 ? __uint_as_float((unsigned)h << 16)
                                : __half2float(__ushort_as_half(h));
}

__device__ __forceinline__ uint16_t float_to_half_bits(float f, int type) {
    return type == DRIFT_T_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f))
                                : __half_as_ushort(__float2half_rn(f));
}

// Eight consecutive elements at `i`; `vec` reads them 16 bytes at a time.
__device__ __forceinline__ void load8(const void *p, int type, int64_t i, int valid, bool vec,
                                      float (&x)[8]) {
    if (type == DRIFT_T_F32) {
        const float *f = static_cast<const float *>(p) + i;
        if (vec && valid == 8) {
            const float4 a = *reinterpret_cast<const float4 *>(f);
            const float4 b = *reinterpret_cast<const float4 *>(f + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
            x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = j < valid ? f[j] : 0.0f;
        }
    } else {
        const uint16_t *h = static_cast<const uint16_t *>(p) + i;
        if (vec && valid == 8) {
            const uint4 a = *reinterpret_cast<const uint4 *>(h);
            const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[2 * j] = half_bits_to_float((uint16_t)w[j], type);
                x[2 * j + 1] = half_bits_to_float((uint16_t)(w[j] >> 16), type);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = j < valid ? half_bits_to_float(h[j], type) : 0.0f;
        }
    }
}

__device__ __forceinline__ void store8(void *p, int type, int64_t i, int valid, bool vec,
                                       const float (&x)[8]) {
    if (type == DRIFT_T_F32) {
        float *f = static_cast<float *>(p) + i;
        if (vec && valid == 8) {
            *reinterpret_cast<float4 *>(f) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(f + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < valid) f[j] = x[j];
        }
    } else {
        uint16_t *h = static_cast<uint16_t *>(p) + i;
        if (vec && valid == 8) {
            unsigned w[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                w[j] = float_to_half_bits(x[2 * j], type) |
                       (unsigned)float_to_half_bits(x[2 * j + 1], type) << 16;
            *reinterpret_cast<uint4 *>(h) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < valid) h[j] = float_to_half_bits(x[j], type);
        }
    }
}

// Eight e4m3 codes and their values times `scale`.
__device__ __forceinline__ void load_codes(const void *p, int64_t i, int valid, bool vec,
                                           float scale, float (&x)[8]) {
    const uint8_t *c = static_cast<const uint8_t *>(p) + i;
    uint64_t w = 0;
    if (vec && valid == 8) {
        w = *reinterpret_cast<const uint64_t *>(c);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < valid) w |= (uint64_t)c[j] << (8 * j);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(
            (__nv_fp8x2_storage_t)(w >> (16 * j)), __NV_E4M3));
        x[2 * j] = __low2float(h) * scale;
        x[2 * j + 1] = __high2float(h) * scale;
    }
}

__device__ __forceinline__ float warp_max_bits(const float (&x)[8]) {
    unsigned a = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) a = max(a, __float_as_uint(x[j]) & 0x7fffffffu);
    return __uint_as_float(__reduce_max_sync(0xffffffffu, a));  // NaN above Inf above all else
}

// Stochastic rounding to e4m3: the code below |y| or the one above, the upper
// with the dropped fraction as its probability (20 random bits). Below 2^-6
// the quantum is 2^-9 throughout, which adding 2^-6 gives.
__device__ __forceinline__ float round_e4m3_sr(float y, unsigned u20) {
    float a = fminf(fabsf(y), 448.0f);
    const bool sub = a < 0x1p-6f;
    if (sub) a += 0x1p-6f;
    a = __uint_as_float((__float_as_uint(a) + u20) & 0xfff00000u);
    if (sub) a -= 0x1p-6f;
    return copysignf(a, y);
}

// Writes a warp's block of 256 values as codes and its scale. A block whose
// values are all below 2^-100 is held as zeros (448 / amax would overflow);
// one with an Inf or NaN reads back as NaN, so that it is not mistaken for
// a state.
template <bool SR>
__device__ __forceinline__ void store_codes(void *p, float *scale, int64_t i, int64_t block,
                                            int valid, bool vec, int lane, const float (&x)[8],
                                            const unsigned (&u)[8]) {
    const float amax = warp_max_bits(x);
    float inv = 0.0f, s = 1.0f;
    if (!(amax <= 3.402823466e38f)) {
        inv = s = __uint_as_float(0x7fffffffu);
    } else if (amax >= 0x1p-100f) {
        inv = 448.0f / amax;
        s = amax / 448.0f;
    }
    if (lane == 0) scale[block] = s;
    uint64_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a = x[2 * j] * inv, b = x[2 * j + 1] * inv;
        if (SR) {
            a = a == a ? round_e4m3_sr(a, u[2 * j]) : a;
            b = b == b ? round_e4m3_sr(b, u[2 * j + 1]) : b;
        }
        w |= (uint64_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)
             << (16 * j);
    }
    uint8_t *c = static_cast<uint8_t *>(p) + i;
    if (vec && valid == 8) {
        *reinterpret_cast<uint64_t *>(c) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < valid) c[j] = (uint8_t)(w >> (8 * j));
    }
}

template <bool EIGHT, bool SR>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamArgs a) {
    // The last tensor whose first chunk is not above this one.
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const AdamTensor &t = a.t[lo];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float a1 = a.scal[0], rc2 = a.scal[1], keep = a.scal[2];
    const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
    const uint64_t state = SR ? *a.rng : 0;
    const bool vec = t.vec;
    const int64_t base = (int64_t)(blockIdx.x - a.first[lo]) * kAdamChunk;
#pragma unroll 1
    for (int b = 0; b < kAdamBlocksPerWarp; b++) {
        const int64_t block = base / kAdamBlock + b * (kAdamThreads / 32) + warp;
        if (block * kAdamBlock >= t.n) break;  // the same for the whole warp
        const int64_t i = block * kAdamBlock + lane * 8;
        const int valid = (int)max((int64_t)0, min((int64_t)8, t.n - i));
        float p[8], g[8], m[8], v[8], r[8];
        load8(t.g, t.gt, i, valid, vec, g);
        load8(t.p, t.pt, i, valid, vec, p);
        if (EIGHT) {
            load_codes(t.m, i, valid, vec, t.ms[block], m);
            load_codes(t.v, i, valid, vec, t.vs[block], r);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = r[j] * r[j];
        } else {
            load8(t.m, DRIFT_T_F32, i, valid, vec, m);
            load8(t.v, DRIFT_T_F32, i, valid, vec, v);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float gj = a.grad_scale ? g[j] * gs : g[j];
            m[j] = a.b1 * m[j] + a.c1 * gj;
            v[j] = a.b2 * v[j] + (a.c2 * gj) * gj;
            r[j] = __fsqrt_rn(v[j]);
            p[j] = keep * p[j] - __fdiv_rn(a1 * m[j], r[j] * rc2 + a.eps);
        }
        store8(t.p, t.pt, i, valid, vec, p);
        if (t.ct >= 0) store8(t.copy, t.ct, i, valid, vec, p);
        if (EIGHT) {
            unsigned um[8] = {}, uv[8] = {};
            if (SR) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint64_t u = splitmix_mix(state + (t.first_draw + i + j + 1) * kGolden);
                    um[j] = (unsigned)(u >> 44);
                    uv[j] = (unsigned)(u >> 24) & 0xfffffu;
                }
            }
            // Lanes past the end hold zeros, which leave the amax as it is.
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j >= valid) m[j] = r[j] = 0.0f;
            store_codes<SR>(t.m, t.ms, i, block, valid, vec, lane, m, um);
            store_codes<SR>(t.v, t.vs, i, block, valid, vec, lane, r, uv);
        } else {
            store8(t.m, DRIFT_T_F32, i, valid, vec, m);
            store8(t.v, DRIFT_T_F32, i, valid, vec, v);
        }
    }
}

static bool aligned(const void *p, unsigned to) {
    return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

int launch_adamw(const drift_adamw *h, const drift_adamw_tensor *tensors, int64_t count,
                 int64_t *d_step, float *d_scalars, const float *d_lr, const float *d_grad_scale,
                 uint64_t *d_rng, cudaStream_t st) {
    const bool eight = h->state_bits == 8;
    const bool sr = eight && h->rounding == DRIFT_STOCHASTIC;
    uint64_t draws = 0;
    for (int64_t i = 0; i < count; i++) draws += (uint64_t)tensors[i].n;
    uint64_t *rng_used = reinterpret_cast<uint64_t *>(d_scalars + 4);
    adamw_prepare_kernel<<<1, 1, 0, st>>>(d_step, h->beta1, h->beta2, h->lr, d_lr,
                                          h->weight_decay, d_scalars, sr ? d_rng : nullptr, draws,
                                          rng_used);
    AdamArgs a;
    a.b1 = (float)h->beta1;
    a.b2 = (float)h->beta2;
    a.c1 = (float)(1.0 - h->beta1);
    a.c2 = (float)(1.0 - h->beta2);
    a.eps = (float)h->eps;
    a.scal = d_scalars;
    a.rng = rng_used;
    a.grad_scale = d_grad_scale;
    a.count = 0;
    uint64_t chunks = 0, drawn = 0;
    auto flush = [&]() {
        if (a.count == 0) return;
        a.first[a.count] = (uint32_t)chunks;
        const unsigned grid = (unsigned)chunks;
        if (!eight) adamw_kernel<false, false><<<grid, kAdamThreads, 0, st>>>(a);
        else if (!sr) adamw_kernel<true, false><<<grid, kAdamThreads, 0, st>>>(a);
        else adamw_kernel<true, true><<<grid, kAdamThreads, 0, st>>>(a);
        a.count = 0;
        chunks = 0;
    };
    for (int64_t i = 0; i < count; i++) {
        const drift_adamw_tensor &t = tensors[i];
        if (t.n == 0) continue;
        const uint64_t c = ((uint64_t)t.n + kAdamChunk - 1) / kAdamChunk;
        if (a.count == kAdamTensors || chunks + c > 0x7fffffffULL) flush();
        AdamTensor &d = a.t[a.count];
        d.p = t.param, d.g = t.grad, d.m = t.m, d.v = t.v;
        d.ms = t.m_scale, d.vs = t.v_scale, d.copy = t.copy;
        d.n = t.n;
        d.first_draw = drawn;
        d.pt = (int8_t)t.param_type, d.gt = (int8_t)t.grad_type;
        d.ct = t.copy ? (int8_t)t.copy_type : (int8_t)-1;
        d.vec = aligned(t.param, 16) && aligned(t.grad, 16) && aligned(t.copy, 16) &&
                aligned(t.m, eight ? 8 : 16) && aligned(t.v, eight ? 8 : 16);
        a.first[a.count++] = (uint32_t)chunks;
        chunks += c;
        drawn += (uint64_t)t.n;
    }
    flush();
    return cudaGetLastError() == cudaSuccess ? DRIFT_OK : DRIFT_ECUDA;
}

}  // namespace drift
