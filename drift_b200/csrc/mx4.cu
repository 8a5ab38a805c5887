// mx4.cu — microscaled 4-bit floating point as the hardware holds it: the cast
// into packed e2m1 codes and power-of-two scales, and back to values.
//
// The numbers are those of Quant.quantize's MX cast with e2m1 elements and
// blocks of 32 (java/src/main/java/io/drift/kernel/Quant.java:95-123): block
// exponent floor(log2 amax) - 2 + headroom within [-127, 127], NaN ignored in
// amax, blocks whose amax is 0 or Inf held as zeros, elements rounded and
// saturated at 6, values above 6 before rounding counted as clamped. Blocks
// start afresh in every row, since a product contracts rows.
//
// Bound: HBM bytes (the source once, 17/32 byte an element out, for each
// direction of blocks). Along rows a lane takes eight elements, so four lanes
// share a block and its amax is two shuffles. Down columns a CTA stages a tile
// of 128 x 128 (64 of the wider types) in shared memory; where both directions are
// wanted they read the same tile, so the source is read once.
//
// Measured on one B200: rows of 8192 x 8192 bf16 in 33 us (5.2 TB/s, 80 % of the copy
// rate), columns in 37 us, both in 68 us (3.0 TB/s); rows of 4096 x 4096 fp32 in 12.3
// us (6.2 TB/s), both axes in 23 us. 16-bit sources take some 11 instructions an
// element and axis: a conversion makes two codes, and each element is widened and
// scaled on the way. Both axes at once fill neither the issue slots (65 %) nor DRAM
// (31 %): a CTA's phases (load, rows, columns, store) wait for one another at barriers,
// and three CTAs an SM overlap only so much of that.
// The other roundings take every element the long way (mx_slow8): truncating 133, 145
// and 276 us for rows, columns and both of that matrix, stochastic 249, 254 and 498,
// with a draw and a comparison in doubles an element.
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "codec.cuh"
#include "internal.h"
#include "mx4.cuh"
#include "pairs.cuh"
#include "pdl.cuh"

namespace drift {

// ------------------------------------------------------------------ one block's arithmetic

// A source type. `key` of an element orders like its magnitude, its NaNs above
// its Inf (kInf) and Inf above the rest, and holds its exponent (of a subnormal of
// the wider types: one below the normal ones', where the scale is at its limit).
template <int TYPE> struct MxSrc;
template <> struct MxSrc<DRIFT_T_F64> {
    using T = double;
    using V = double;
    static constexpr unsigned kInf = 0x7ff00000u;
    __device__ static V get(T x) { return x; }
    // The high word, with one bit for a low word that is not zero.
    __device__ static unsigned key(T x) {
        return ((unsigned)__double2hiint(x) & 0x7fffffffu) | min((unsigned)__double2loint(x), 1u);
    }
    __device__ static int exponent(unsigned key) { return (int)(key >> 20) - 1023; }
};
template <> struct MxSrc<DRIFT_T_F32> {
    using T = float;
    using V = float;
    static constexpr unsigned kInf = 0x7f800000u;
    __device__ static V get(T x) { return x; }
    __device__ static unsigned key(T x) { return __float_as_uint(x) & 0x7fffffffu; }
    __device__ static int exponent(unsigned key) { return (int)(key >> 23) - 127; }
};
template <> struct MxSrc<DRIFT_T_BF16> {
    using T = __nv_bfloat16;
    using V = float;
    static constexpr unsigned kInf = 0x7f80u;
    __device__ static V get(T x) { return __bfloat162float(x); }
    __device__ static V get_bits(unsigned h) { return __uint_as_float(h << 16); }
    // Of each half, the larger magnitude, signs left in place; a NaN stays one.
    __device__ static unsigned max2(unsigned a, unsigned b) {
        unsigned m;
        asm("{\n .reg .b32 x, y;\n abs.bf16x2 x, %1;\n abs.bf16x2 y, %2;\n"
            " max.NaN.bf16x2 %0, x, y;\n}"
            : "=r"(m)
            : "r"(a), "r"(b));
        return m;
    }
    // Both halves times powers of two, exact but for results far below the smallest
    // code: two products an instruction, then widened.
    __device__ static void scaled2(unsigned w, float lo, float hi, float &a, float &b) {
        const unsigned k = __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
        asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(k));
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    }
    __device__ static int exponent(unsigned key) { return (int)(key >> 7) - 127; }
};
template <> struct MxSrc<DRIFT_T_FP16> {
    using T = __half;
    using V = float;
    static constexpr unsigned kInf = 0x7c00u;
    __device__ static V get(T x) { return __half2float(x); }
    __device__ static V get_bits(unsigned h) { return __half2float(__ushort_as_half((uint16_t)h)); }
    __device__ static unsigned max2(unsigned a, unsigned b) {
        return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu);
    }
    __device__ static void scaled2(unsigned w, float lo, float hi, float &a, float &b) {
        a = get_bits(w & 0xffffu) * lo;
        b = get_bits(w >> 16) * hi;
    }
    __device__ static int exponent(unsigned key) {
        return MxSrc<DRIFT_T_F32>::exponent(__float_as_uint(get_bits(key)));
    }
};

// Magnitude for amax: NaN counts as nothing (Quant.java:25-34).
__device__ __forceinline__ float mx_mag(float x) { return x == x ? fabsf(x) : 0.0f; }
__device__ __forceinline__ double mx_mag(double x) { return x == x ? fabs(x) : 0.0; }

// Math.getExponent of the value as a double, so a float subnormal has its own
// exponent.
__device__ __forceinline__ int mx_exponent(float a) {
    const int e = (int)(__float_as_uint(a) >> 23);
    return e ? e - 127 : -118 - __clz(__float_as_uint(a));  // 31 - clz - 149
}
__device__ __forceinline__ int mx_exponent(double a) { return java_get_exponent(a); }

struct MxScale {
    int shared;  // exponent of the block's scale
    bool zero;   // amax 0 or Inf: the block is held as zeros
};

template <class V>
__device__ __forceinline__ MxScale mx_scale(V amax, int headroom) {
    MxScale s;
    s.zero = !(amax > (V)0) || isinf(amax);
    const int e = mx_exponent(amax) - 2 + headroom;
    s.shared = s.zero ? 0 : max(-127, min(127, e));
    return s;
}

// x * 2^-shared: exact, except far below the smallest code.
__device__ __forceinline__ float mx_scaled(float x, int shared) {
    const unsigned up = (unsigned)(127 - shared) << 23;
    return x * (shared < 127 ? __uint_as_float(up) : 0x1p-127f);
}
__device__ __forceinline__ double mx_scaled(double x, int shared) {
    return __dmul_rn(x, pow2(-shared));
}

// A double narrowed to float with its lost bits kept as a sticky lowest bit, so
// that the rounding to e2m1 sees on which side of a midpoint the double was.
__device__ __forceinline__ float mx_narrow(float x) { return x; }
__device__ __forceinline__ float mx_narrow(double x) {
    const float f = __double2float_rz(x);
    return (double)f == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Codes of eight values to nearest, ties to the even code, saturating at 6: value
// j in bits 4j to 4j+3.
__device__ __forceinline__ unsigned mx_rn8(const float (&y)[8]) {
    unsigned w;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}

// The code toward zero of |x| <= 6, and its value.
__device__ __forceinline__ unsigned mx_floor(float a, float &base) {
    if (a < 1.0f) {
        base = a >= 0.5f ? 0.5f : 0.0f;
        return a >= 0.5f;
    }
    const unsigned b = __float_as_uint(a);
    base = __uint_as_float(b & 0xffc00000u);
    return (b >> 22) - (127u * 2 - 2);  // 1 -> 2, 1.5 -> 3, 2 -> 4, ... 6 -> 7
}

// Code of one scaled value under truncation or stochastic rounding (u53: its
// draw). The fraction of the step that truncation drops is exact in V; Java
// rounds up where nextDouble() is below it (MiniFloat.java:264-273).
template <class V>
__device__ __forceinline__ unsigned mx_code(V x, int rm, uint64_t u53) {
    const V a = fmin(fabs(x), (V)6);
    float base;
    unsigned code = mx_floor(sizeof(V) == 8 ? __double2float_rz((double)a) : (float)a, base);
    if (rm == DRIFT_STOCHASTIC) {
        const V frac = (a - (V)base) * (base < 2.0f ? (V)2 : base < 4.0f ? (V)1 : (V)0.5);
        if (u53_to_double(u53) * 0x1p-53 < (double)frac) code++;
    }
    return code | (signbit(x) ? 8u : 0u);
}

// Eight values of one block (or zeros past the end) to 32 bits of codes.
// `draw` is the index of element 0's draw, `step` the distance to the next
// element's.
template <class V>
__device__ __forceinline__ unsigned mx_pack8(const V (&x)[8], const MxScale &s, int rm,
                                             uint64_t state, uint64_t draw, uint64_t step,
                                             int valid, unsigned &clamps, int &err) {
    V y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        V v = j < valid ? x[j] : (V)0;
        if (v != v) {  // the format has no NaN: flagged, held as +0
            if (!s.zero) err |= DEV_ERR_NAN_FINITE;
            v = (V)0;
        }
        y[j] = s.zero ? (V)0 : mx_scaled(v, s.shared);
        clamps += fabs(y[j]) > (V)6;
    }
    unsigned w = 0;
    if (rm == DRIFT_NEAREST_EVEN) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = mx_narrow(y[j]);
        w = mx_rn8(f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint64_t u = rm == DRIFT_STOCHASTIC ? draw_u53(state, draw + j * step) : 0;
            w |= mx_code(y[j], rm, u) << (4 * j);
        }
    }
    return w;
}

// Eight consecutive elements as they lie in memory.
template <int TYPE> struct MxRaw8 {
    using S = MxSrc<TYPE>;
    static constexpr int kVecs = sizeof(typename S::T) * 8 / 16;
    uint4 w[kVecs];
    __device__ const unsigned *words() const { return reinterpret_cast<const unsigned *>(w); }
    __device__ unsigned key() const {  // the largest of the eight
        if constexpr (sizeof(typename S::T) == 2) {
            const unsigned *u = words();
            const unsigned m =
                S::max2(S::max2(u[0], u[1]), S::max2(u[2], u[3])) & 0x7fff7fffu;
            return max(m & 0xffffu, m >> 16);
        } else {
            const typename S::T *x = reinterpret_cast<const typename S::T *>(w);
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) m = max(m, S::key(x[j]));
            return m;
        }
    }
    __device__ void values(typename S::V (&x)[8]) const {
        if constexpr (sizeof(typename S::T) == 2) {
            const unsigned *u = words();
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = S::get_bits(u[j / 2] >> (j & 1) * 16 & 0xffffu);
        } else {
            const typename S::T *t = reinterpret_cast<const typename S::T *>(w);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = t[j];
        }
    }
};

// The scale of a block from its key, and the factor 2^-shared, for a headroom of 1
// at most: then shared is below 127 (but of large doubles), the factor a normal
// number, and subnormals' scales are at the lower limit whatever their exponent.
// Key 0 is a block of zeros, which callers hold as +0 whatever the signs.
template <class V> struct MxFactor {
    int shared;
    V down;
};
template <int TYPE>
__device__ __forceinline__ MxFactor<typename MxSrc<TYPE>::V> mx_factor(unsigned key, int headroom) {
    MxFactor<typename MxSrc<TYPE>::V> f;
    int e = max(MxSrc<TYPE>::exponent(key) + (headroom - 2), -127);
    if constexpr (TYPE == DRIFT_T_F64) {
        e = min(e, 127);
        f.down = __longlong_as_double((long long)(1023 - e) << 52);
    } else {
        f.down = __uint_as_float((unsigned)(127 - e) << 23);
    }
    f.shared = key ? e : 0;
    return f;
}

// Codes to nearest of eight elements of a block without Inf or NaN.
__device__ __forceinline__ unsigned mx_fast8(const float (&x)[8], float down) {
    const f2 k = f2_both(down);
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; j++)
        f2_split(f2_mul(f2_pack(x[2 * j], x[2 * j + 1]), k), y[2 * j], y[2 * j + 1]);
    return mx_rn8(y);
}
__device__ __forceinline__ unsigned mx_fast8(const double (&x)[8], double down) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = mx_narrow(x[j] * down);
    return mx_rn8(y);
}

template <int TYPE>
__device__ __forceinline__ unsigned mx_fast8(const MxRaw8<TYPE> &r,
                                             typename MxSrc<TYPE>::V down) {
    using S = MxSrc<TYPE>;
    if constexpr (sizeof(typename S::T) == 2) {
        const unsigned *u = r.words();
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; j++) S::scaled2(u[j], down, down, y[2 * j], y[2 * j + 1]);
        return mx_rn8(y);
    } else {
        typename S::V x[8];
        r.values(x);
        return mx_fast8(x, down);
    }
}

// ------------------------------------------------------------------ the cast

struct MxCast {
    const void *src;
    int64_t rows, cols, row_stride;
    int headroom, rm;
    bool quick;                        // to nearest, headroom 1 at most
    bool vec, wide;                    // rows start 16-byte, 32-byte aligned
    uint8_t *codes, *scales;           // blocks along rows
    uint8_t *codes_t, *scales_t;       // blocks down columns: the transpose, packed
    uint64_t draw_t;                   // first draw of the transposed cast
    const uint64_t *state;
    unsigned long long *clamped, *clamped_t;
    int *err;
};

// Eight elements at p, 16-byte aligned; `wide`: 32-byte aligned, so that the wider
// types' lanes take whole sectors an instruction.
template <int TYPE>
__device__ __forceinline__ MxRaw8<TYPE> mx_load_whole(const typename MxSrc<TYPE>::T *p, bool wide) {
    MxRaw8<TYPE> r;
    constexpr int kVecs = MxRaw8<TYPE>::kVecs;
    if (kVecs > 1 && wide) {
#pragma unroll
        for (int j = 0; j + 1 < kVecs; j += 2)
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                : "=r"(r.w[j].x), "=r"(r.w[j].y), "=r"(r.w[j].z), "=r"(r.w[j].w),
                  "=r"(r.w[j + 1].x), "=r"(r.w[j + 1].y), "=r"(r.w[j + 1].z), "=r"(r.w[j + 1].w)
                : "l"(reinterpret_cast<const uint4 *>(p) + j));
    } else {
#pragma unroll
        for (int j = 0; j < kVecs; j++) r.w[j] = reinterpret_cast<const uint4 *>(p)[j];
    }
    return r;
}
// `valid` elements at p, the rest zeros; `vec`: p is 16-byte aligned.
template <int TYPE>
__device__ __forceinline__ MxRaw8<TYPE> mx_load8(bool vec, const typename MxSrc<TYPE>::T *p,
                                                 int valid) {
    using T = typename MxSrc<TYPE>::T;
    if (vec && valid == 8) return mx_load_whole<TYPE>(p, false);
    MxRaw8<TYPE> r;
    T *t = reinterpret_cast<T *>(r.w);
#pragma unroll
    for (int j = 0; j < MxRaw8<TYPE>::kVecs; j++) r.w[j] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < valid) t[j] = p[j];
    return r;
}

__device__ __forceinline__ void mx_finish(unsigned clamps, int err, unsigned long long *clamped,
                                          int *d_err) {
    clamps = __reduce_add_sync(0xffffffffu, clamps);
    err = (int)__reduce_or_sync(0xffffffffu, (unsigned)err);
    if ((threadIdx.x & 31) == 0) {
        if (clamped && clamps) atomicAdd(clamped, (unsigned long long)clamps);
        if (err) atomicOr(d_err, err);
    }
}

// Everything the short way leaves: blocks with Inf or NaN, and the other roundings.
// Out of line, since its instructions beside the short way's cost more in fetches
// than the call.
template <int TYPE>
__device__ __noinline__ unsigned mx_slow8(const MxCast &a, const typename MxSrc<TYPE>::V (&x)[8],
                                          typename MxSrc<TYPE>::V amax, int valid, uint64_t state,
                                          uint64_t draw, uint64_t step, int &shared,
                                          unsigned &clamps, int &err) {
    const MxScale s = mx_scale(amax, a.headroom);
    shared = s.shared;
    return mx_pack8(x, s, a.rm, state, draw, step, valid, clamps, err);
}

// Eight elements of a block that four neighbouring lanes share: their codes and
// the block's shared exponent. Elements past the end are zeros and change nothing.
template <int TYPE>
__device__ __forceinline__ unsigned mx_cast8(const MxCast &a, const MxRaw8<TYPE> &r, int valid,
                                             uint64_t state, uint64_t draw, int &shared,
                                             unsigned &clamps, int &err) {
    using S = MxSrc<TYPE>;
    using V = typename S::V;
    unsigned key = r.key();
    key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
    key = max(key, __shfl_xor_sync(0xffffffffu, key, 2));
    V x[8];
    if (__all_sync(0xffffffffu, key < S::kInf) && a.quick) {
        const MxFactor<V> f = mx_factor<TYPE>(key, a.headroom);
        shared = f.shared;
        if (a.clamped) {
            r.values(x);
#pragma unroll
            for (int j = 0; j < 8; j++) clamps += fabs(x[j] * f.down) > (V)6;
        }
        const unsigned w = mx_fast8<TYPE>(r, f.down);
        return key ? w : 0;
    }
    r.values(x);
    V amax = (V)0;
#pragma unroll
    for (int j = 0; j < 8; j++) amax = fmax(amax, mx_mag(x[j]));
    amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // Copies, so that only this path's live in memory.
    V y[8];
    unsigned more = 0;
    int sh = 0, e = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = x[j];
    const unsigned w = mx_slow8<TYPE>(a, y, amax, valid, state, draw, 1, sh, more, e);
    shared = sh;
    clamps += more;
    err |= e;
    return w;
}

// Blocks along rows: a warp takes U chunks of 256 elements of one row (eight
// blocks, two tiles of scales each) at a time, with all their loads in flight.
// Rows past the end up to the tile's 128, and blocks past the row's end, get
// their padding bytes.
template <int TYPE, int U>
__global__ void __launch_bounds__(256) mx4_rows_kernel(const __grid_constant__ MxCast a,
                                                       uint32_t per_row, uint32_t items) {
    using T = typename MxSrc<TYPE>::T;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t blocks = mx4_blocks(a.cols);
    const int chunks = (int)(mx4_k_tiles(a.cols) / 2);
    const uint64_t state = a.rm == DRIFT_STOCHASTIC ? *a.state : 0;
    unsigned clamps = 0;
    int err = 0;
    const uint32_t stride = gridDim.x * 8;
    // A lane's block is 0 to 7 of a chunk; its scale's place in the two tiles.
    const int place = (lane >> 4) * kMxTileBytes + (lane >> 2 & 3);
    for (uint32_t it = blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += stride) {
        const uint32_t row = it / per_row;
        const int first = (int)(it - row * per_row) * U;
        const int64_t col0 = (int64_t)first * 256 + lane * 8;
        const bool in_row = row < a.rows;
        const T *src = static_cast<const T *>(a.src) + row * a.row_stride + col0;
        uint8_t *codes = a.codes + row * (blocks * 16) + col0 / 2;
        uint8_t *scales = a.scales + mx4_scale_offset(row, 0, chunks * 2) +
                          (int64_t)first * 2 * kMxTileBytes + place;
        // What is left of the row from this lane's first element on.
        const int64_t left = in_row ? a.cols - col0 : 0;
        const auto cast = [&](auto is_whole) {
            // Whole: all U chunks are elements of a row, aligned.
            constexpr bool kWhole = decltype(is_whole)::value;
            MxRaw8<TYPE> raw[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                raw[u] = kWhole ? mx_load_whole<TYPE>(src + u * 256, a.wide)
                                : mx_load8<TYPE>(a.vec, src + u * 256,
                                                 (int)max((int64_t)0,
                                                          min((int64_t)8, left - u * 256)));
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (!kWhole && first + u >= chunks) break;  // the same for the whole warp
                int shared;
                const int valid =
                    kWhole ? 8 : (int)max((int64_t)0, min((int64_t)8, left - u * 256));
                const unsigned w =
                    mx_cast8<TYPE>(a, raw[u], valid, state,
                                   (uint64_t)row * a.cols + col0 + u * 256, shared, clamps, err);
                const bool in = kWhole || (in_row && (col0 + u * 256) >> 5 < blocks);
                if (in) *reinterpret_cast<unsigned *>(codes + u * 128) = w;
                if ((lane & 3) == 0)
                    scales[u * 2 * kMxTileBytes] = in ? (uint8_t)(shared + 127) : (uint8_t)127;
            }
        };
        if (a.vec && in_row && (int64_t)(first + U) * 256 <= a.cols) cast(std::true_type{});
        else cast(std::false_type{});
    }
    mx_finish(clamps, err, a.clamped, a.err);
}

// Blocks down columns (and along rows too, where a.codes is given). A CTA takes
// 128 rows of 128 columns (64 of the wider types): the loads' registers give the
// row cast, shared memory the columns, of which a thread casts one 32-bit word
// wide (two 16-bit columns) of 32 rows. Codes go back through shared memory, so
// that a column's 64 bytes leave together.
constexpr int kMxTr = 128;
template <int TYPE> struct MxTile {
    using T = typename MxSrc<TYPE>::T;
    static constexpr int kWide = sizeof(T) == 2 ? 2 : 1;       // columns a thread casts
    static constexpr int kCols = 64 * kWide;
    static constexpr int kLdBytes = kCols * (int)sizeof(T) + 16;
    static constexpr int kStage = kCols * 80;                  // codes: 64 bytes a column, padded
    static constexpr int kSmem = kMxTr * kLdBytes > kStage ? kMxTr * kLdBytes : kStage;
    static constexpr int kLoads = kMxTr * kCols / 8 / 256;     // groups of eight a thread loads
};

// One column's block of 32, the long way: 16 bytes of codes.
template <int TYPE>
__device__ __forceinline__ uint4 mx_slow_col(const MxCast &a,
                                             const typename MxSrc<TYPE>::V (&x)[32],
                                             uint64_t state, uint64_t draw, int &shared,
                                             unsigned &clamps, int &err) {
    using V = typename MxSrc<TYPE>::V;
    uint4 w;
    unsigned *wp = reinterpret_cast<unsigned *>(&w);
    V amax = (V)0;
#pragma unroll
    for (int j = 0; j < 32; j++) amax = fmax(amax, mx_mag(x[j]));
    unsigned more = 0;
    int sh = 0, e = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        V y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = x[q * 8 + j];
        wp[q] = mx_slow8<TYPE>(a, y, amax, 8, state, draw + (uint64_t)q * 8 * a.cols, a.cols, sh,
                               more, e);
    }
    shared = sh;
    clamps += more;
    err |= e;
    return w;
}

template <int TYPE>
__global__ void __launch_bounds__(256, sizeof(typename MxSrc<TYPE>::T) == 8 ? 2 : 3) mx4_cols_kernel(const __grid_constant__ MxCast a,
                                                       uint32_t row_tiles,
                                                       uint32_t col_tiles) {
    using S = MxSrc<TYPE>;
    using T = typename S::T;
    using V = typename S::V;
    using G = MxTile<TYPE>;
    extern __shared__ __align__(16) unsigned char mx_smem[];
    pdl_trigger();
    pdl_wait();
    const uint32_t tile_r = blockIdx.x / col_tiles, tile_c = blockIdx.x - tile_r * col_tiles;
    const int64_t r0 = (int64_t)tile_r * kMxTr, c0 = (int64_t)tile_c * G::kCols;
    const int tid = threadIdx.x, lane = tid & 31;
    const uint64_t state = a.rm == DRIFT_STOCHASTIC ? *a.state : 0;

    constexpr int kGroups = G::kCols / 8;  // groups of eight in a row of the tile
    const bool whole = a.vec && r0 + kMxTr <= a.rows && c0 + G::kCols <= a.cols;
    MxRaw8<TYPE> raw[G::kLoads];
    constexpr int kStep = 256 / kGroups;  // rows from one load to the next
    const int row_t = tid / kGroups, col_t = tid % kGroups * 8;
    {
        const T *p = static_cast<const T *>(a.src) + (r0 + row_t) * a.row_stride + c0 + col_t;
        const int64_t down = kStep * a.row_stride;
        if (whole) {
#pragma unroll
            for (int i = 0; i < G::kLoads; i++, p += down) raw[i] = mx_load_whole<TYPE>(p, a.wide);
        } else {
            const int valid = (int)max((int64_t)0, min((int64_t)8, a.cols - c0 - col_t));
#pragma unroll
            for (int i = 0; i < G::kLoads; i++, p += down)
                raw[i] = mx_load8<TYPE>(a.vec, p, r0 + row_t + i * kStep < a.rows ? valid : 0);
        }
    }
    {
        unsigned char *to = mx_smem + row_t * G::kLdBytes + col_t * sizeof(T);
#pragma unroll
        for (int i = 0; i < G::kLoads; i++)
#pragma unroll
            for (int j = 0; j < MxRaw8<TYPE>::kVecs; j++)
                reinterpret_cast<uint4 *>(to + i * kStep * G::kLdBytes)[j] = raw[i].w[j];
    }

    if (a.codes) {
        unsigned clamps = 0;
        int err = 0;
        const int blocks = (int)mx4_blocks(a.cols), k_tiles = (int)mx4_k_tiles(a.cols);
        const int64_t row_bytes = (int64_t)blocks * 16;
        const int r = row_t, block = (int)(c0 >> 5) + tid % kGroups / 4;
        const bool in_cols = block < blocks;
        uint8_t *codes = a.codes + (r0 + r) * row_bytes + c0 / 2 + tid % kGroups * 4;
        uint8_t *scales = a.scales + ((int64_t)tile_r * k_tiles + block / 4) * kMxTileBytes +
                          block % 4;
        uint64_t draw = (uint64_t)(r0 + r) * a.cols + c0 + tid % kGroups * 8;
#pragma unroll
        for (int i = 0; i < G::kLoads; i++) {
            const int at = r + i * kStep;
            int shared;
            const unsigned w = mx_cast8<TYPE>(a, raw[i], 8, state, draw, shared, clamps, err);
            const bool in = in_cols && r0 + at < a.rows;
            if (in) *reinterpret_cast<unsigned *>(codes) = w;
            codes += kStep * row_bytes;
            draw += (uint64_t)kStep * a.cols;
            if ((lane & 3) == 0 && block < k_tiles * 4) {
                uint8_t *to = scales + at % 32 * 16 + at / 32 * 4;
                *to = in ? (uint8_t)(shared + 127) : (uint8_t)127;
                // The last columns' CTA also writes the pair's remaining blocks.
                if (tile_c + 1 == col_tiles)
                    for (int b = block + G::kCols / 32; b < k_tiles * 4; b += G::kCols / 32)
                        to[(b / 4 - block / 4) * kMxTileBytes + b % 4 - block % 4] = 127;
            }
        }
        mx_finish(clamps, err, a.clamped, a.err);
    }
    __syncthreads();

    // Down columns: thread = (word of columns, block of 32 rows).
    unsigned clamps = 0;
    int err = 0;
    const int word = tid & 63, b = tid >> 6;
    const int64_t row = r0 + b * 32;
    uint4 codes[G::kWide];
    int shared[G::kWide];
    const uint64_t draw = a.draw_t + (uint64_t)row * a.cols + c0 + word * G::kWide;
    if constexpr (G::kWide == 2) {
        unsigned u[32], m = 0;
#pragma unroll
        for (int j = 0; j < 32; j++) {
            u[j] = *reinterpret_cast<const unsigned *>(mx_smem + (b * 32 + j) * G::kLdBytes +
                                                       word * 4);
            m = S::max2(m, u[j]);
        }
        const unsigned key[2] = {m & 0x7fffu, m >> 16 & 0x7fffu};
        if (max(key[0], key[1]) < S::kInf && a.quick) {
            const MxFactor<V> f0 = mx_factor<TYPE>(key[0], a.headroom);
            const MxFactor<V> f1 = mx_factor<TYPE>(key[1], a.headroom);
            shared[0] = f0.shared, shared[1] = f1.shared;
            unsigned *w0 = reinterpret_cast<unsigned *>(&codes[0]);
            unsigned *w1 = reinterpret_cast<unsigned *>(&codes[1]);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float y0[8], y1[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    S::scaled2(u[q * 8 + j], f0.down, f1.down, y0[j], y1[j]);
                if (a.clamped_t) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        clamps += (fabsf(y0[j]) > 6.0f) + (fabsf(y1[j]) > 6.0f);
                }
                w0[q] = key[0] ? mx_rn8(y0) : 0;
                w1[q] = key[1] ? mx_rn8(y1) : 0;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                V x[32];
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] = S::get_bits(u[j] >> h * 16 & 0xffffu);
                codes[h] = mx_slow_col<TYPE>(a, x, state, draw + h, shared[h], clamps, err);
            }
        }
    } else {
        V x[32];
        unsigned key = 0;
#pragma unroll
        for (int j = 0; j < 32; j++) {
            x[j] = *reinterpret_cast<const T *>(mx_smem + (b * 32 + j) * G::kLdBytes +
                                                word * sizeof(T));
            key = max(key, S::key(x[j]));
        }
        if (key < S::kInf && a.quick) {
            const MxFactor<V> f = mx_factor<TYPE>(key, a.headroom);
            shared[0] = f.shared;
            unsigned *wp = reinterpret_cast<unsigned *>(&codes[0]);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                V y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = x[q * 8 + j];
                if (a.clamped_t) {
#pragma unroll
                    for (int j = 0; j < 8; j++) clamps += fabs(y[j] * f.down) > (V)6;
                }
                wp[q] = key ? mx_fast8(y, f.down) : 0;
            }
        } else {
            codes[0] = mx_slow_col<TYPE>(a, x, state, draw, shared[0], clamps, err);
        }
    }
    __syncthreads();
    const int64_t blocks = mx4_blocks(a.rows);
    const int k_tiles = (int)mx4_k_tiles(a.rows);
    // The transpose's tile of scales: its rows are columns here, its blocks rows.
    uint8_t *scales_t =
        a.scales_t + ((c0 / 128) * k_tiles + tile_r) * (int64_t)kMxTileBytes + b;
#pragma unroll
    for (int h = 0; h < G::kWide; h++) {
        const int c = word * G::kWide + h, in_tile = (int)(c0 % 128) + c;
        *reinterpret_cast<uint4 *>(mx_smem + c * 80 + b * 16) = codes[h];
        // With the padding of the last tiles: columns up to the tile's 128 rows (the
        // grid's columns end with them), blocks up to a whole pair of tiles.
        uint8_t *to = scales_t + in_tile % 32 * 16 + in_tile / 32 * 4;
        *to = c0 + c < a.cols && row < a.rows ? (uint8_t)(shared[h] + 127) : (uint8_t)127;
        if (tile_r + 1 == row_tiles && tile_r % 2 == 0) to[kMxTileBytes] = 127;
    }
    mx_finish(clamps, err, a.clamped_t, a.err);
    __syncthreads();
    {
        const int c = tid >> 2, q = tid & 3;
        uint8_t *to = a.codes_t + (c0 + c) * blocks * 16 + (r0 / 32 + q) * 16;
        const bool in = r0 + q * 32 < a.rows;
#pragma unroll
        for (int i = 0; i < G::kCols / 64; i++) {
            if (in && c0 + c + i * 64 < a.cols)
                *reinterpret_cast<uint4 *>(to + i * 64 * blocks * 16) =
                    *reinterpret_cast<const uint4 *>(mx_smem + (c + i * 64) * 80 + q * 16);
        }
    }
}

__global__ void mx4_advance_kernel(uint64_t *state, uint64_t draws) {
    pdl_trigger();
    pdl_wait();
    *state += draws * kGolden;
}

template <int TYPE>
static int launch_cast(const MxCast &a, cudaStream_t st) {
    using T = typename MxSrc<TYPE>::T;
    if (!a.codes_t) {
        const uint32_t chunks = (uint32_t)(mx4_k_tiles(a.cols) / 2);
        const uint32_t rows = (uint32_t)(mx4_row_tiles(a.rows) * 128);
        const uint32_t sms = (uint32_t)sm_count();
        // Four chunks a warp (two of doubles, whose loads fill as many registers), where
        // the rows have them, once that still leaves every SM two CTAs; else a warp a
        // chunk.
        constexpr uint32_t kU = sizeof(T) == 8 ? 2 : 4;
        if (chunks >= kU && rows * (uint64_t)((chunks + kU - 1) / kU) >= sms * 2 * 8) {
            const uint32_t per_row = (chunks + kU - 1) / kU, items = rows * per_row;
            const uint32_t grid = std::min<uint32_t>((items + 7) / 8, sms * 8);
            return launch_pdl(mx4_rows_kernel<TYPE, kU>, dim3(grid), 256, 0, st, 0, a, per_row,
                              items);
        } else {
            const uint32_t items = rows * chunks;
            return launch_pdl(mx4_rows_kernel<TYPE, 1>,
                              dim3(std::min<uint32_t>((items + 7) / 8, sms * 64)), 256, 0, st, 0,
                              a, chunks, items);
        }
    } else {
        using G = MxTile<TYPE>;
        static unsigned long long done = 0;
        if (!allow_smem(mx4_cols_kernel<TYPE>, G::kSmem, done)) return DRIFT_ECUDA;
        // Columns up to the tile's 128, so that every padding byte is written.
        const uint32_t row_tiles = (uint32_t)mx4_row_tiles(a.rows);
        const uint32_t col_tiles = (uint32_t)mx4_row_tiles(a.cols) * (128 / G::kCols);
        return launch_pdl(mx4_cols_kernel<TYPE>, dim3(row_tiles * col_tiles), 256, G::kSmem, st, 0,
                          a, row_tiles, col_tiles);
    }
}

int launch_mx4_quantize(int headroom, int rm, int type, const void *src, int64_t rows,
                        int64_t cols, int64_t row_stride, uint8_t *codes, uint8_t *scales,
                        uint8_t *codes_t, uint8_t *scales_t, uint64_t *d_state,
                        unsigned long long *clamped, unsigned long long *clamped_t, int *d_err,
                        cudaStream_t st) {
    static const int size[4] = {8, 4, 2, 2};
    MxCast a;
    a.src = src;
    a.rows = rows, a.cols = cols, a.row_stride = row_stride;
    a.headroom = headroom, a.rm = rm;
    a.quick = rm == DRIFT_NEAREST_EVEN && headroom <= 1;
    const uintptr_t at = reinterpret_cast<uintptr_t>(src) | (uintptr_t)(row_stride * size[type]);
    a.vec = at % 16 == 0, a.wide = at % 32 == 0;
    a.codes = codes, a.scales = scales, a.codes_t = codes_t, a.scales_t = scales_t;
    a.draw_t = codes ? (uint64_t)rows * cols : 0;
    a.state = d_state;
    a.clamped = clamped, a.clamped_t = clamped_t;
    a.err = d_err;
    int rc;
    switch (type) {
        case DRIFT_T_F64: rc = launch_cast<DRIFT_T_F64>(a, st); break;
        case DRIFT_T_F32: rc = launch_cast<DRIFT_T_F32>(a, st); break;
        case DRIFT_T_BF16: rc = launch_cast<DRIFT_T_BF16>(a, st); break;
        default: rc = launch_cast<DRIFT_T_FP16>(a, st); break;
    }
    if (rc) return rc;
    if (rm == DRIFT_STOCHASTIC)
        return launch_pdl(mx4_advance_kernel, dim3(1), 1, 0, st, 0, d_state,
                          (uint64_t)rows * cols * ((codes != nullptr) + (codes_t != nullptr)));
    return DRIFT_OK;
}

// ------------------------------------------------------------------ back to values

// Two elements' values without their scale.
__device__ __forceinline__ float2 mx_pair(unsigned byte) {
    unsigned h;
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %1;\n cvt.rn.f16x2.e2m1x2 %0, a;\n}"
        : "=r"(h)
        : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// Eight values a thread. A double, float or bf16 holds every value exactly,
// except that 2^127 times 2 or more overflows float and bf16; fp16 rounds. The scale
// byte 255 is E8M0's NaN here as in the tensor cores.
template <class T>
__global__ void __launch_bounds__(256) mx4_values_kernel(const uint8_t *codes,
                                                         const uint8_t *scales, int64_t rows,
                                                         int64_t cols, T *dst, int64_t stride,
                                                         uint32_t groups, bool vec) {
    pdl_trigger();
    pdl_wait();
    const int64_t row_bytes = mx4_row_bytes(cols), k_tiles = mx4_k_tiles(cols);
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        for (uint32_t g = blockIdx.x * 256 + threadIdx.x; g < groups; g += gridDim.x * 256) {
            const int64_t col = (int64_t)g * 8;
            const unsigned w =
                *reinterpret_cast<const unsigned *>(codes + row * row_bytes + col / 2);
            const int shared = (int)scales[mx4_scale_offset(row, col >> 5, k_tiles)] - 127;
            __align__(16) T v[8];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = mx_pair(w >> (8 * j) & 0xffu);
                if constexpr (sizeof(T) == 8) {
                    const double up = shared < 128 ? pow2(shared) : CUDART_NAN;
                    v[2 * j] = f.x * up, v[2 * j + 1] = f.y * up;
                } else {
                    const float up = shared == 128   ? CUDART_NAN_F
                                     : shared > -127 ? __uint_as_float((unsigned)(shared + 127) << 23)
                                                     : 0x1p-127f;
                    v[2 * j] = T(f.x * up), v[2 * j + 1] = T(f.y * up);
                }
            }
            T *p = dst + row * stride + col;
            if (vec && col + 8 <= cols) {
                const uint4 *w = reinterpret_cast<const uint4 *>(v);
                if constexpr (sizeof(T) == 2) {
                    *reinterpret_cast<uint4 *>(p) = w[0];
                } else {
                    // Whole sectors an instruction (vec: 32-byte aligned).
#pragma unroll
                    for (int j = 0; j < (int)sizeof(T) / 4; j++)
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                                         reinterpret_cast<uint4 *>(p) + 2 * j),
                                     "r"(w[2 * j].x), "r"(w[2 * j].y), "r"(w[2 * j].z),
                                     "r"(w[2 * j].w), "r"(w[2 * j + 1].x), "r"(w[2 * j + 1].y),
                                     "r"(w[2 * j + 1].z), "r"(w[2 * j + 1].w)
                                     : "memory");
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (col + j < cols) p[j] = v[j];
            }
        }
    }
}

int launch_mx4_dequantize(const drift_mx4 *q, int type, void *dst, int64_t stride,
                          cudaStream_t st) {
    static const int size[4] = {8, 4, 2, 2};
    const uint32_t groups = (uint32_t)((q->cols + 7) / 8);
    const uintptr_t at = reinterpret_cast<uintptr_t>(dst) | (uintptr_t)(stride * size[type]);
    const bool vec = at % (size[type] == 2 ? 16 : 32) == 0;
    const dim3 grid((groups + 255) / 256, (unsigned)std::min<int64_t>(q->rows, 65535));
    const auto run = [&](auto *p) {
        return launch_pdl(mx4_values_kernel<std::remove_pointer_t<decltype(p)>>, grid, 256, 0, st, 0,
                          q->codes, q->scales, q->rows, q->cols, p, stride, groups, vec);
    };
    switch (type) {
        case DRIFT_T_F64: return run((double *)dst);
        case DRIFT_T_F32: return run((float *)dst);
        case DRIFT_T_BF16: return run((__nv_bfloat16 *)dst);
        default: return run((__half *)dst);
    }
}

}  // namespace drift
