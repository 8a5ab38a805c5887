// adamw.cu — one AdamW step over a list of tensors in one launch, moments in
// 32 bits or in 8 bits with one scale per 256 elements.
//
// Every element does, in 32 bits, the moments' operations each rounded on its own
// (this is their definition, so the same operations elsewhere give the bits of m, v
// and m's codes; a unit's difference now and then would move a code by a whole step,
// and m, which forgets in ten steps, by more in the next):
//
//   m' = b1 m + (1-b1) g          v' = b2 v + ((1-b2) g) g        r = sqrt(v')
//   p' = fma(1 - lr wd, p, -(lr/(1-b1^t) m') / fma(r, 1/sqrt(1-b2^t), eps))
//
// The quotient is a product with a reciprocal, within two units in the last place.
// The root is within one; 8-bit moments, whose state it is, take Newton's step to
// the nearest float (no code of 16M differed from the IEEE root's).
//
// In 8 bits the first moment is held as e4m3 codes of m * (1 / amax * 448) and
// the second as e4m3 codes of its root r, which spans half the binades that v
// does. p' uses the moments before they are rounded to codes.
//
// Bound: HBM bytes. 32-bit moments with fp32 parameters and bf16 gradients
// move 26 bytes an element, 8-bit moments with bf16 parameters and gradients
// 10.1. One warp owns a block of 256 elements, eight a lane, so a block's amax is
// a handful of instructions and every access is one or two 16-byte loads or
// stores a lane.
//
// Measured on one B200: 200M bf16 parameters with 8-bit moments in 346 us (5.8 TB/s, 90 %
// of the copy rate; 366 with a reciprocal that keeps subnormals), 8.6M fp32 ones with
// 32-bit moments in 37 us (6.0 TB/s). With 8-bit moments it is near its instructions
// too (46 an element, 75 % of the issue slots), and is slower on a hot card: 400M take
// 762 to 784 us in turn with other work. Each CTA on a stretch of its own took 60 % longer for
// the first: the CTAs in flight then touch as many stretches of seven arrays, where
// side by side they sweep one of each. Scalar operations, IEEE roots and quotients,
// 68 instructions an element, took 1083 us for 400M.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "internal.h"
#include "pairs.cuh"
#include "pdl.cuh"

namespace drift {

constexpr int kAdamThreads = 256;
constexpr int kAdamBlock = 256;                     // elements that share a scale
constexpr int kAdamMostBlocks = 32;                  // blocks that a warp takes in turn
constexpr int kAdamTensors = 256;                   // tensors of one launch

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
    float b1, b2, c1, c2, eps, one;  // one: 1, for f2_add
    const float *scal;        // lr/(1-b1^t), 1/sqrt(1-b2^t), 1 - lr wd
    const uint64_t *rng;      // Rng state of this step's draws
    const float *grad_scale;  // may be null
};

// The step's scalars, in double and rounded once; advances the step count and
// the Rng state, so that a captured call replays as the next step.
__global__ void adamw_prepare_kernel(int64_t *step, double b1, double b2, double lr,
                                     const float *d_lr, double wd, float *scal, uint64_t *rng,
                                     uint64_t draws, uint64_t *rng_used) {
    pdl_trigger();
    pdl_wait();
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

// Within one unit. The denominators are 0, Inf, NaN or well inside the normal range (a
// root is above 2^-75, and eps is 0 or above 1e-30; a root is below 2^64, its factor
// below 2^27), where flushing subnormals changes nothing.
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float sqrt_fast(float x) {  // within one unit
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rsqrt_fast(float x) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Roots of four pairs, rounded to nearest but for a few in a million that fall a unit
// short: s = v / sqrt(v) from the hardware's reciprocal root, then Newton's step
// s - (s^2 - v) / (2 sqrt(v)) with a fused residual (Markstein 1990). That wants v well
// inside the normal range; a warp with another v anywhere takes IEEE roots (100M bf16
// parameters whose gradients and moments are all 0: 235 us, against 179).
__device__ __forceinline__ void roots(const f2 (&v)[4], f2 (&r)[4]) {
    unsigned out = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a, b;
        f2_split(v[j], a, b);
        // Between 2^-100 and 2^100, read as integers.
        out = max(out, max(__float_as_uint(a) - 0x0d800000u, __float_as_uint(b) - 0x0d800000u));
    }
    if (__any_sync(0xffffffffu, out >= 0x64000000u)) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float a, b;
            f2_split(v[j], a, b);
            r[j] = f2_pack(__fsqrt_rn(a), __fsqrt_rn(b));
        }
        return;
    }
    const f2 minus_one = f2_both(-1.0f), minus_half = f2_both(-0.5f);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a, b;
        f2_split(v[j], a, b);
        const f2 y = f2_pack(rsqrt_fast(a), rsqrt_fast(b));
        const f2 s = f2_mul(v[j], y);
        r[j] = f2_fma(f2_fma(s, s, f2_mul(v[j], minus_one)), f2_mul(y, minus_half), s);
    }
}
// The largest magnitude of three; NaN wins.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// ------------------------------------------------------------------ eight elements

// Eight elements as they lie in memory: 16-bit types use the first word.
struct Raw8 {
    uint4 w[2];
};

__device__ __forceinline__ uint16_t float_to_half_bits(float f, int type) {
    return type == DRIFT_T_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f))
                                : __half_as_ushort(__float2half_rn(f));
}

// `whole`: all eight exist and are aligned for 16-byte accesses.
__device__ __forceinline__ Raw8 load_raw(const void *p, int type, int64_t i, int valid,
                                         bool whole) {
    Raw8 r;
    if (type == DRIFT_T_F32) {
        const float *f = static_cast<const float *>(p) + i;
        if (whole) {
            r.w[0] = *reinterpret_cast<const uint4 *>(f);
            r.w[1] = reinterpret_cast<const uint4 *>(f)[1];
        } else {
            unsigned *u = reinterpret_cast<unsigned *>(r.w);
#pragma unroll
            for (int j = 0; j < 8; j++) u[j] = j < valid ? __float_as_uint(f[j]) : 0u;
        }
    } else {
        const uint16_t *h = static_cast<const uint16_t *>(p) + i;
        if (whole) {
            r.w[0] = *reinterpret_cast<const uint4 *>(h);
        } else {
            unsigned *u = reinterpret_cast<unsigned *>(r.w);
#pragma unroll
            for (int j = 0; j < 4; j++)
                u[j] = (2 * j < valid ? h[2 * j] : 0u) |
                       (2 * j + 1 < valid ? (unsigned)h[2 * j + 1] << 16 : 0u);
        }
    }
    return r;
}

__device__ __forceinline__ void unpack(const Raw8 &r, int type, f2 (&x)[4]) {
    const unsigned *u = reinterpret_cast<const unsigned *>(r.w);
    if (type == DRIFT_T_F32) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            x[j] = f2_pack(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1]));
    } else if (type == DRIFT_T_BF16) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            x[j] = f2_pack(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u));
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
            x[j] = f2_pack(f.x, f.y);
        }
    }
}

__device__ __forceinline__ void store8(void *p, int type, int64_t i, int valid, bool whole,
                                       const f2 (&y)[4]) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; j++) f2_split(y[j], x[2 * j], x[2 * j + 1]);
    if (type == DRIFT_T_F32) {
        float *f = static_cast<float *>(p) + i;
        if (whole) {
            __stcs(reinterpret_cast<float4 *>(f), make_float4(x[0], x[1], x[2], x[3]));
            __stcs(reinterpret_cast<float4 *>(f) + 1, make_float4(x[4], x[5], x[6], x[7]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < valid) f[j] = x[j];
        }
    } else {
        uint16_t *h = static_cast<uint16_t *>(p) + i;
        if (whole) {
            uint4 w;
            unsigned *u = reinterpret_cast<unsigned *>(&w);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (type == DRIFT_T_BF16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
                    u[j] = *reinterpret_cast<const unsigned *>(&b);
                } else {
                    const __half2 b = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
                    u[j] = *reinterpret_cast<const unsigned *>(&b);
                }
            }
            __stcs(reinterpret_cast<uint4 *>(h), w);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < valid) h[j] = float_to_half_bits(x[j], type);
        }
    }
}

__device__ __forceinline__ uint64_t load_codes(const void *p, int64_t i, int valid, bool whole) {
    const uint8_t *c = static_cast<const uint8_t *>(p) + i;
    if (whole) return *reinterpret_cast<const uint64_t *>(c);
    uint64_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < valid) w |= (uint64_t)c[j] << (8 * j);
    return w;
}

// Eight e4m3 codes' values times `scale`.
__device__ __forceinline__ void decode(uint64_t w, float scale, f2 (&x)[4]) {
    const f2 s = f2_both(scale);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(
            (__nv_fp8x2_storage_t)(w >> (16 * j)), __NV_E4M3)));
        x[j] = f2_mul(f2_pack(f.x, f.y), s);
    }
}

__device__ __forceinline__ float warp_amax(const f2 (&x)[4]) {
    float a[8];
#pragma unroll
    for (int j = 0; j < 4; j++) f2_split(x[j], a[2 * j], a[2 * j + 1]);
    const float m = max3_abs(max3_abs(a[0], a[1], a[2]), max3_abs(a[3], a[4], a[5]),
                             max3_abs(a[6], a[7], 0.0f));
    // As bit patterns magnitudes order like integers, NaN above Inf above all else.
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7fffffffu));
}

// Stochastic rounding to e4m3: the code below |y| or the one above, the upper
// with the dropped fraction as its probability (20 random bits). Below 2^-6
// the quantum is 2^-9 throughout, which adding 2^-6 gives.
__device__ __forceinline__ float round_e4m3_sr(float y, unsigned u20) {
    if (y != y) return y;
    float a = fminf(fabsf(y), 448.0f);
    const bool sub = a < 0x1p-6f;
    if (sub) a += 0x1p-6f;
    a = __uint_as_float((__float_as_uint(a) + u20) & 0xfff00000u);
    if (sub) a -= 0x1p-6f;
    return copysignf(a, y);
}

// Codes of a lane's eight values times `inv`.
template <bool SR>
__device__ __forceinline__ void store_codes(void *p, int64_t i, int valid, bool whole, float inv,
                                            const f2 (&x)[4], const unsigned (&u)[8]) {
    const f2 k = f2_both(inv);
    unsigned h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a, b;
        f2_split(f2_mul(x[j], k), a, b);
        if (SR) a = round_e4m3_sr(a, u[2 * j]), b = round_e4m3_sr(b, u[2 * j + 1]);
        h[j] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    }
    const uint2 w = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    uint8_t *c = static_cast<uint8_t *>(p) + i;
    if (whole) {
        __stcs(reinterpret_cast<uint2 *>(c), w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < valid) c[j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
    }
}

// ------------------------------------------------------------------ the step

// What a lane has loaded of one block.
template <bool EIGHT> struct Loaded {
    Raw8 p, g, m, v;  // m, v: 32-bit moments
};
template <> struct Loaded<true> {
    Raw8 p, g;
    uint64_t m, v;
    float ms, vs;
};

// PT, GT: the types of parameter and gradient, or -1 to look them up. WHOLE: all 256
// elements exist and are aligned.
template <bool EIGHT, int PT, int GT, bool WHOLE>
__device__ __forceinline__ void load_block(const AdamTensor &t, int64_t block, int lane,
                                           Loaded<EIGHT> &l) {
    const int64_t i = block * kAdamBlock + lane * 8;
    const int valid = WHOLE ? 8 : (int)max((int64_t)0, min((int64_t)8, t.n - i));
    l.g = load_raw(t.g, GT < 0 ? t.gt : GT, i, valid, WHOLE);
    l.p = load_raw(t.p, PT < 0 ? t.pt : PT, i, valid, WHOLE);
    if constexpr (EIGHT) {
        l.m = load_codes(t.m, i, valid, WHOLE);
        l.v = load_codes(t.v, i, valid, WHOLE);
        l.ms = t.ms[block];
        l.vs = t.vs[block];
    } else {
        l.m = load_raw(t.m, DRIFT_T_F32, i, valid, WHOLE);
        l.v = load_raw(t.v, DRIFT_T_F32, i, valid, WHOLE);
    }
}

struct Scalars {
    f2 b1, b2, c1, c2, eps, neg_a1, rc2, keep, gs, one;
    uint64_t state;
};

template <bool EIGHT, bool SR, int PT, int GT, bool WHOLE>
__device__ __forceinline__ void update_block(const AdamTensor &t, int64_t block, int lane,
                                             const Loaded<EIGHT> &l, const Scalars &k) {
    const int64_t i = block * kAdamBlock + lane * 8;
    const int valid = WHOLE ? 8 : (int)max((int64_t)0, min((int64_t)8, t.n - i));
    const int pt = PT < 0 ? t.pt : PT, gt = GT < 0 ? t.gt : GT;
    f2 p[4], g[4], m[4], v[4], r[4];
    unpack(l.g, gt, g);
    unpack(l.p, pt, p);
    if constexpr (EIGHT) {
        decode(l.m, l.ms, m);
        decode(l.v, l.vs, r);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = f2_mul(r[j], r[j]);
    } else {
        unpack(l.m, DRIFT_T_F32, m);
        unpack(l.v, DRIFT_T_F32, v);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const f2 gj = f2_mul(g[j], k.gs);  // by 1 without a scale
        m[j] = f2_add(f2_mul(k.b1, m[j]), f2_mul(k.c1, gj), k.one);
        v[j] = f2_add(f2_mul(k.b2, v[j]), f2_mul(f2_mul(k.c2, gj), gj), k.one);
    }
    if constexpr (EIGHT) {
        roots(v, r);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float a, b;
            f2_split(v[j], a, b);
            r[j] = f2_pack(sqrt_fast(a), sqrt_fast(b));
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a, b;
        f2_split(f2_fma(r[j], k.rc2, k.eps), a, b);
        const f2 step = f2_mul(f2_mul(k.neg_a1, m[j]), f2_pack(rcp_fast(a), rcp_fast(b)));
        p[j] = f2_fma(k.keep, p[j], step);
    }
    store8(t.p, pt, i, valid, WHOLE, p);
    if (t.ct >= 0) store8(t.copy, t.ct, i, valid, WHOLE, p);
    if constexpr (EIGHT) {
        unsigned um[8] = {}, uv[8] = {};
        if (SR) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint64_t u = splitmix_mix(k.state + (t.first_draw + i + j + 1) * kGolden);
                um[j] = (unsigned)(u >> 44);
                uv[j] = (unsigned)(u >> 24) & 0xfffffu;
            }
        }
        // Elements past the end hold zeros throughout, so they leave an amax as
        // it is. A block whose values are all below 2^-100 is held as zeros
        // (the inverse would overflow); one with an Inf or NaN reads back as NaN, so
        // that it is not mistaken for a state. Half of the warp inverts m's amax,
        // half r's.
        const float am = warp_amax(m), ar = warp_amax(r);
        const float amax = lane < 16 ? am : ar;
        float inv = 0.0f, s = 1.0f;
        if (!(amax <= 3.402823466e38f)) {
            inv = s = __uint_as_float(0x7fffffffu);
        } else if (amax >= 0x1p-100f) {
            inv = __frcp_rn(amax) * 448.0f;
            s = amax * (1.0f / 448.0f);
        }
        if (lane == 0) t.ms[block] = s;
        if (lane == 16) t.vs[block] = s;
        store_codes<SR>(t.m, i, valid, WHOLE, __shfl_sync(0xffffffffu, inv, 0), m, um);
        store_codes<SR>(t.v, i, valid, WHOLE, __shfl_sync(0xffffffffu, inv, 16), r, uv);
    } else {
        store8(t.m, DRIFT_T_F32, i, valid, WHOLE, m);
        store8(t.v, DRIFT_T_F32, i, valid, WHOLE, v);
    }
}

// `n` whole blocks, `step` apart; the next one's loads are in flight while one is
// computed.
template <bool EIGHT, bool SR, int PT, int GT>
__device__ __forceinline__ void run_blocks(const AdamTensor &t, int64_t block, int n, int64_t step,
                                           int lane, const Scalars &k) {
    Loaded<EIGHT> next;
    load_block<EIGHT, PT, GT, true>(t, block, lane, next);
#pragma unroll 1
    for (int b = 0; b < n; b++) {
        const Loaded<EIGHT> now = next;
        if (b + 1 < n)
            load_block<EIGHT, PT, GT, true>(t, block + step, lane, next);
        update_block<EIGHT, SR, PT, GT, true>(t, block, lane, now, k);
        block += step;
    }
}

// 8-bit moments: 64 registers and four CTAs an SM; 32-bit ones hold more in flight
// a thread and run as fast with two.
template <bool EIGHT, bool SR>
__global__ void __launch_bounds__(kAdamThreads, EIGHT && !SR ? 4 : 2) adamw_kernel(const __grid_constant__ AdamArgs a) {
    pdl_trigger();
    pdl_wait();
    // The last tensor whose first chunk is not above this one.
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const AdamTensor &t = a.t[lo];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kWarps = kAdamThreads / 32;
    // This warp's blocks: b0, b0 + step, ..., the tensor's CTAs side by side, so that
    // all that run at a time sweep one stretch of memory.
    const int64_t b0 = (int64_t)(blockIdx.x - a.first[lo]) * kWarps + warp;
    const int64_t step = (int64_t)(a.first[lo + 1] - a.first[lo]) * kWarps;
    const auto count = [&](int64_t blocks) {  // of them below `blocks`
        return blocks > b0 ? (int)((blocks - b0 + step - 1) / step) : 0;
    };
    const int n = count((t.n + kAdamBlock - 1) / kAdamBlock);
    int whole = t.vec ? count(t.n / kAdamBlock) : 0;
    Scalars k;
    k.b1 = f2_both(a.b1), k.b2 = f2_both(a.b2), k.c1 = f2_both(a.c1), k.c2 = f2_both(a.c2);
    k.eps = f2_both(a.eps), k.one = f2_both(a.one);
    k.neg_a1 = f2_both(-a.scal[0]), k.rc2 = f2_both(a.scal[1]), k.keep = f2_both(a.scal[2]);
    k.gs = f2_both(a.grad_scale ? *a.grad_scale : 1.0f);
    k.state = SR ? *a.rng : 0;
    // The usual types have code of their own; fp16, bf16 parameters with fp32 gradients,
    // unaligned tensors and the last, partial block of one take the general form, which
    // loads and stores element by element: 100M in 633 to 654 us with 32-bit moments and
    // 501 to 511 with 8-bit ones, where the usual types take 347 to 428 and 179 to 273.
    if (whole) {
        if (t.pt == DRIFT_T_F32 && t.gt == DRIFT_T_F32)
            run_blocks<EIGHT, SR, DRIFT_T_F32, DRIFT_T_F32>(t, b0, whole, step, lane, k);
        else if (t.pt == DRIFT_T_F32 && t.gt == DRIFT_T_BF16)
            run_blocks<EIGHT, SR, DRIFT_T_F32, DRIFT_T_BF16>(t, b0, whole, step, lane, k);
        else if (t.pt == DRIFT_T_BF16 && t.gt == DRIFT_T_BF16)
            run_blocks<EIGHT, SR, DRIFT_T_BF16, DRIFT_T_BF16>(t, b0, whole, step, lane, k);
        else
            whole = 0;
    }
#pragma unroll 1
    for (int b = whole; b < n; b++) {
        Loaded<EIGHT> now;
        load_block<EIGHT, -1, -1, false>(t, b0 + b * step, lane, now);
        update_block<EIGHT, SR, -1, -1, false>(t, b0 + b * step, lane, now, k);
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
    int64_t blocks = 0;
    for (int64_t i = 0; i < count; i++) {
        draws += (uint64_t)tensors[i].n;
        blocks += (tensors[i].n + kAdamBlock - 1) / kAdamBlock;
    }
    uint64_t *rng_used = reinterpret_cast<uint64_t *>(d_scalars + 4);
    int rc = launch_pdl(adamw_prepare_kernel, dim3(1), 1, 0, st, 0, d_step, h->beta1, h->beta2,
                        h->lr, d_lr, h->weight_decay, d_scalars, sr ? d_rng : nullptr, draws,
                        rng_used);
    AdamArgs a;
    a.b1 = (float)h->beta1;
    a.b2 = (float)h->beta2;
    a.c1 = (float)(1.0 - h->beta1);
    a.c2 = (float)(1.0 - h->beta2);
    a.eps = (float)h->eps;
    a.one = 1.0f;
    a.scal = d_scalars;
    a.rng = rng_used;
    a.grad_scale = d_grad_scale;
    a.count = 0;
    // Warps take several blocks in turn, loading ahead, once that leaves twelve
    // CTAs an SM (three waves or more); few blocks spread over the SMs instead.
    int per_warp = 1;
    while (per_warp < kAdamMostBlocks &&
           blocks >= (int64_t)per_warp * 2 * (kAdamThreads / 32) * 12 * sm_count())
        per_warp *= 2;
    const uint64_t chunk_len = (uint64_t)kAdamBlock * (kAdamThreads / 32) * per_warp;
    uint64_t chunks = 0, drawn = 0;
    auto flush = [&]() {
        if (a.count == 0) return;
        a.first[a.count] = (uint32_t)chunks;
        const auto kernel = !eight ? adamw_kernel<false, false>
                            : !sr  ? adamw_kernel<true, false>
                                   : adamw_kernel<true, true>;
        if (!rc) rc = launch_pdl(kernel, dim3((unsigned)chunks), kAdamThreads, 0, st, 0, a);
        a.count = 0;
        chunks = 0;
    };
    for (int64_t i = 0; i < count; i++) {
        const drift_adamw_tensor &t = tensors[i];
        if (t.n == 0) continue;
        const uint64_t c = ((uint64_t)t.n + chunk_len - 1) / chunk_len;
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
    return rc;
}

}  // namespace drift
