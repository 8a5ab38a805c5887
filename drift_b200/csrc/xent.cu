// xent.cu — a linear layer with softmax cross entropy over its outputs, in
// pieces of the vocabulary, and its gradients; no logits are kept.
//
//   l = x W^T + b       lse_i = log sum_v exp l_iv       loss_i = lse_i - l_i,t(i)
//   d_iv = (exp(l_iv - lse_i) - [v = t(i)]) g_i
//   dx = d W            dW = d^T x            db_v = sum_i d_iv
//
// x and W are bf16 or fp16; sums, statistics and log sums are fp32. All four
// products run on the tensor cores (tc.cuh):
//
//   forward   the logits' tile stays in registers: each thread reduces its 128
//             columns of a row to a maximum, a sum of exponentials and perhaps the
//             target's logit; a second kernel joins the parts of a row.
//             (Where a mean loss is wanted with its gradients and all logits fit in
//             L2, they are kept in the workspace until d has replaced them.)
//   gradient  a piece of the vocabulary at a time: the logits again, whose
//             epilogue writes d in the inputs' type (one rounding, which halves
//             its bytes and feeds the tensor cores; an element's error is half a
//             unit of that type, as the results' own: theirs, relative, grows from
//             1.65e-3 to 1.98e-3 at 64 x 2048 x 96 and stays at 1.7e-3 at 4096 x
//             131072 x 4096), then dx += d W and dW = d^T x from it, reading d and W
//             where they lie (MN-major).
//
// fp16 holds d times a power of two (2^15, or with weights by row one that brings
// the largest finite |g| of the rows that count near 2^15), so that small
// probabilities keep their bits; the products undo it exactly. bf16 has fp32's range
// and needs none.
//
// Bound: the tensor cores for many tokens (8 T D V operations with the
// gradient's second computation of the logits, against 6 T D V if they were
// kept); the bytes of W for few. Measured on one B200: 4096 tokens x 131072 entries
// x 4096 with gradients in 14.2 to 15.3 ms (1.15 to 1.24 PFLOP/s under the power
// cap), the loss of 64 tokens x 131072 x 4096 in 224 us (4.8 TB/s).
#include <algorithm>

#include "epilogue.cuh"
#include "internal.h"
#include "tc.cuh"

namespace drift {

// Stages of 64 summed in TMEM, whose sums truncate: 2^-18 of a logit's magnitude at
// most over 16, which moves an fp32 loss by a few units; the gradients' products
// round to 16 bits, so theirs may be longer. Measured on 1001 log sums, relative: 3.0e-7
// at depths of 1024, 2048 and 4096 (with runs of 64 stages 3.0e-7, 6.6e-7 and 1.3e-6;
// sums rounded to nearest at each step 3e-8).
constexpr int kLogitRun = 16, kGradRun = 64;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Maximum that keeps a NaN, so that a row with one has a NaN log sum.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

struct XentRows {
    const void *targets;
    bool wide;  // int64 targets, else int32
    int64_t ignore, vocab;
    // The target of row i; negative for an ignored row. One outside the
    // vocabulary sets `bad` and counts as ignored.
    __device__ __forceinline__ int64_t at(int64_t i, bool &bad) const {
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

// A maximum and a sum of exponentials relative to it.
struct Stat {
    float m, s;
};
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    Stat r;
    r.m = max_nan(a.m, b.m);
    r.s = r.m > -INFINITY ? a.s * exp2_fast((a.m - r.m) * kLog2e) +
                                b.s * exp2_fast((b.m - r.m) * kLog2e)
                          : 0.0f;
    return r;
}

// ------------------------------------------------------------------ epilogues

// Adds the bias; columns past the piece become -inf.
__device__ __forceinline__ void finish_logits(float (&v)[128], int64_t col, int64_t cols,
                                              const Bias4 &bias, unsigned staging, int lane) {
    add_bias(v, bias, staging, lane);
    if (col + 128 > cols) {
#pragma unroll
        for (int j = 0; j < 128; j++)
            if (col + j >= cols) v[j] = -INFINITY;
    }
}

// Statistics of 128 logits of a row.
struct StatsEpi {
    Stat *parts;   // [column group of 128][row]
    float *target; // target's logit per row
    const float *bias;  // of the piece's first column
    int64_t rows, cols, v0;
    XentRows x;
    // Loaded before the accumulator is awaited, which takes 0.5 to 1.1 us off losses of
    // 20 us and less. (In the other epilogues it costs more in registers.)
    struct Before {
        Bias4 bias;
        int t;  // the target's column of the thread's 128, if there
    };
    __device__ __forceinline__ Before before(int64_t row, int64_t col, int lane) const {
        bool bad = false;
        const int64_t t = row < rows ? x.at(row, bad) - v0 - col : -1;
        return Before{Bias4(bias, col, cols, lane), t < 128 ? (int)max(t, (int64_t)-1) : 128};
    }
    __device__ __forceinline__ void run(float (&v)[128], const Before &b, int64_t row0, int64_t col,
                                        const tc::Work &, int lane, unsigned staging) const {
        if (col >= cols) return;
        const int64_t row = row0 + lane;
        finish_logits(v, col, cols, b.bias, staging, lane);
        float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int j = 4; j < 128; j++) m[j & 3] = max_nan(m[j & 3], v[j]);
        const float top = max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
        float s[4] = {};
        // The difference first: a masked entry may be the type's lowest value, whose
        // product with log2 e overflows.
#pragma unroll
        for (int j = 0; j < 128; j++) s[j & 3] += exp2_fast((v[j] - top) * kLog2e);
        if (row >= rows) return;
        const float sum = (s[0] + s[1]) + (s[2] + s[3]);
        parts[(col >> 7) * rows + row] = Stat{top, top > -INFINITY ? sum : 0.0f};
        if (b.t >= 0 && b.t < 128) {
            float l = 0.0f;
#pragma unroll
            for (int j = 0; j < 128; j++)
                if (j == b.t) l = v[j];
            target[row] = l;
        }
    }
};

// d of 128 logits of a row, in the inputs' type; and, with DB, its column sums
// over the warp's 32 rows.
template <class T, bool DB> struct GradEpi {
    T *d;
    int64_t ld;       // row stride of d, a multiple of 8
    const float *bias;
    int64_t rows, cols, v0;
    XentRows x;
    const float *lse, *g;  // g: null for 1 throughout
    int64_t g_stride;
    const float *scale;    // the power of two that d is held times: device, or null
    float fixed;           // and the host's
    float *sums;           // DB: [row / 32][column], not scaled
    __device__ __forceinline__ int before(int64_t, int64_t, int) const { return 0; }
    __device__ __forceinline__ void run(float (&v)[128], int, int64_t row0, int64_t col,
                                        const tc::Work &, int lane, unsigned staging) const {
        if (col >= cols) return;
        const int64_t row = row0 + lane;
        finish_logits(v, col, cols, Bias4(bias, col, cols, lane), staging, lane);
        bool bad = false;
        const int64_t t = row < rows ? x.at(row, bad) : -1;
        const float gi = t >= 0 ? (g ? g[row * g_stride] : 1.0f) : 0.0f;
        const float z = t >= 0 ? lse[row] : 0.0f;
        const int64_t at = t - v0 - col;
#pragma unroll
        for (int j = 0; j < 128; j++) {
            const float p = exp2_fast((v[j] - z) * kLog2e);
            v[j] = t >= 0 ? ((int64_t)j == at ? p - 1.0f : p) * gi : 0.0f;
        }
        if (DB) {
            // 32 columns over 32 lanes at a time: at each step a lane keeps half of
            // its columns and gets its partner's sums of them, so lane l ends with
            // column l's sum.
#pragma unroll
            for (int c = 0; c < 128; c += 32) {
                float a[32];
#pragma unroll
                for (int j = 0; j < 32; j++) a[j] = v[c + j];
#pragma unroll
                for (int h = 16; h; h >>= 1) {
                    const bool up = lane & h;
#pragma unroll
                    for (int j = 0; j < h; j++) {
                        const float keep = up ? a[j + h] : a[j], give = up ? a[j] : a[j + h];
                        a[j] = keep + __shfl_xor_sync(0xffffffffu, give, h);
                    }
                }
                if (col + c + lane < cols) sums[(row0 >> 5) * cols + col + c + lane] = a[0];
            }
        }
        const float f = scale ? *scale : fixed;
        if (f != 1.0f) {
#pragma unroll
            for (int j = 0; j < 128; j++) v[j] *= f;
        }
        T *p = d + row0 * ld + col;
        by_rows<T>(v, staging, lane, [&](int r, int j, uint4 w) {
            if (row0 + r < rows && col + j < ld)  // padding columns get zeros
                *reinterpret_cast<uint4 *>(p + r * ld + j) = w;
        });
    }
};

// ------------------------------------------------------------------ small kernels

// Joins a row's parts, and the running statistics of the pieces before; the last
// piece gives its log sum and loss. Many rows: a CTA takes 32 of them, 32 threads a
// row, so that a warp reads 32 rows' part i together. Few rows (ROWS 1): a CTA a row.
template <int ROWS>
__global__ void __launch_bounds__(1024) xent_join_kernel(const Stat *parts, int n_parts, int64_t T,
                                                         Stat *run, bool first, bool last,
                                                         const float *target, XentRows x,
                                                         float *loss, float *lse, int *err) {
    pdl_trigger();
    pdl_wait();
    __shared__ Stat sh[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * ROWS + (ROWS == 1 ? 0 : lane);
    Stat r{-INFINITY, 0.0f};
    if (row < T) {
        const int from = ROWS == 1 ? (int)threadIdx.x : warp;
        const int step = ROWS == 1 ? (int)blockDim.x : warps;
#pragma unroll 4
        for (int i = from; i < n_parts; i += step) r = join(r, parts[(int64_t)i * T + row]);
    }
    if (ROWS == 1) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            r = join(r, Stat{__shfl_xor_sync(0xffffffffu, r.m, o),
                             __shfl_xor_sync(0xffffffffu, r.s, o)});
    }
    sh[warp][lane] = r;
    __syncthreads();
    if (warp || row >= T || (ROWS == 1 && lane)) return;
    for (int i = 1; i < warps; i++) r = join(r, sh[i][lane]);
    if (!first) r = join(run[row], r);
    if (!last) {
        run[row] = r;
        return;
    }
    const float z = r.m + logf(r.s);
    bool bad = false;
    const int64_t t = x.at(row, bad);
    if (bad) atomicOr(err, DEV_ERR_INDEX);
    lse[row] = z;
    loss[row] = t >= 0 ? z - target[row] : 0.0f;  // may be target itself
}

// fp16: the power of two that brings the largest finite |g| of a row with a gradient
// into [2^14, 2^15), and its inverse; 1 where all are below 2^-96. An Inf or NaN spoils
// its own row of dx, not the others' scale.
__global__ void __launch_bounds__(1024) xent_scale_kernel(const float *g, int64_t g_stride,
                                                          XentRows x, int64_t n, float *scale) {
    pdl_trigger();
    pdl_wait();
    __shared__ unsigned sm[32];
    unsigned m = 0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        bool bad = false;
        const unsigned w = __float_as_uint(g[i * g_stride]) & 0x7fffffffu;
        m = max(m, w < 0x7f800000u && x.at(i, bad) >= 0 ? w : 0u);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
        m = __reduce_max_sync(0xffffffffu, sm[threadIdx.x]);
        const int e = (int)(m >> 23);  // biased exponent
        const bool use = e > 30;
        const int k = use ? 14 - (e - 127) : 0;
        if (threadIdx.x == 0) {
            scale[0] = exp2f((float)k);
            scale[1] = exp2f((float)-k);
        }
    }
}

// db of a piece: the sum over `groups` rows of `sums` (each the sum of 32 tokens, or
// one token's d), in order.
__global__ void __launch_bounds__(256) xent_colsum_kernel(const float *sums, int64_t groups,
                                                          int64_t n, int64_t ld,
                                                          const float *alpha, float *db) {
    pdl_trigger();
    pdl_wait();
    __shared__ float sh[8][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t v = (int64_t)blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (v < n) {
#pragma unroll 4
        for (int64_t i = slice; i < groups; i += 8) s += sums[i * ld + v];
    }
    sh[slice][lane] = s;
    __syncthreads();
    if (slice || v >= n) return;
    for (int i = 1; i < 8; i++) s += sh[i][lane];
    db[v] = alpha ? s * *alpha : s;
}

// Sums the parts of dx and rounds to its type.
template <class T>
__global__ void __launch_bounds__(256) xent_dx_kernel(const float *acc, int splits, int64_t part,
                                                      int64_t ld, T *dx, int64_t rows,
                                                      int64_t cols, int64_t stride,
                                                      const float *alpha, float beta) {
    pdl_trigger();
    pdl_wait();
    const float f = alpha ? *alpha * beta : beta;
    const int64_t groups = (cols + 3) / 4;
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < rows * groups; i += 256LL * gridDim.x) {
        const int64_t r = i / groups, c = (i - r * groups) * 4;
        float4 s = *reinterpret_cast<const float4 *>(acc + r * ld + c);
        for (int k = 1; k < splits; k++) {
            const float4 y = *reinterpret_cast<const float4 *>(acc + k * part + r * ld + c);
            s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
        }
        const float v[4] = {s.x * f, s.y * f, s.z * f, s.w * f};
        T *p = dx + r * stride + c;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (c + j < cols) p[j] = T(v[j]);
    }
}

// The x that dW = d^T x reads: an ignored row's d is 0, but 0 times an Inf or NaN
// that a padded position may hold is not, so those rows are copied as zeros. The
// copy is 4 bytes an element of x beside 2 V operations.
struct CopyRows {
    const uint4 *from;  // null: no copy
    uint4 *to;
    int64_t from_ld, to_ld, units;  // in units of 16 bytes
    int last;                       // elements of x in a row's last unit
    __device__ __forceinline__ void copy_row(int64_t row, bool on) const {
        if (!from) return;
        const uint4 *f = from + row * from_ld;
        uint4 *t = to + row * to_ld;
        for (int64_t i = threadIdx.x; i < units; i += blockDim.x) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (on && (i + 1 < units || last == 8)) {
                w = f[i];
            } else if (on) {  // the row's memory may end with its last element
                const uint16_t *h = reinterpret_cast<const uint16_t *>(f + i);
                unsigned *u = reinterpret_cast<unsigned *>(&w);
#pragma unroll
                for (int j = 0; j < 7; j++)
                    if (j < last) u[j / 2] |= (unsigned)h[j] << (j & 1) * 16;
            }
            t[i] = w;
        }
    }
};
__global__ void __launch_bounds__(128) xent_copy_kernel(CopyRows xs, XentRows x) {
    pdl_trigger();
    pdl_wait();
    bool bad = false;
    xs.copy_row(blockIdx.x, x.at(blockIdx.x, bad) >= 0);
}

// The mean loss with its gradients where all logits fit the workspace at once: a
// CTA takes a row, sums the parts of its logits, and replaces them by d, both in
// fp32 (for db) and in the inputs' type times `scale`. Its loss goes to `row_loss`.
// With `xs` the CTA also copies its row of x, an ignored one as zeros (copy_row).
template <class T>
__global__ void __launch_bounds__(256) xent_row_kernel(float *logits, int splits, int64_t part,
                                                       int64_t ld, int64_t n, const float *bias,
                                                       XentRows x, T *d, float scale, bool keep,
                                                       float *row_loss, CopyRows xs, int *err) {
    pdl_trigger();
    pdl_wait();
    __shared__ Stat sh[8];
    __shared__ float target;
    const int64_t row = blockIdx.x;
    float *l = logits + row * ld;
    bool bad = false;
    const int64_t t = x.at(row, bad);
    Stat r{-INFINITY, 0.0f};
    for (int64_t v = threadIdx.x; v < n; v += 256) {
        float y = l[v];
        for (int k = 1; k < splits; k++) y += l[k * part + v];
        if (bias) y += bias[v];
        l[v] = y;  // read again by this thread alone
        if (v == t) target = y;
        r = join(r, Stat{y, 1.0f});
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
        r = join(r, Stat{__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = r;
    __syncthreads();
    r = sh[0];
#pragma unroll
    for (int i = 1; i < 8; i++) r = join(r, sh[i]);
    const float z = r.m + logf(r.s);
    for (int64_t v = threadIdx.x; v < n; v += 256) {
        const float p = exp2_fast((l[v] - z) * kLog2e);
        const float g = t >= 0 ? (v == t ? p - 1.0f : p) : 0.0f;
        d[row * ld + v] = T(g * scale);
        if (keep) l[v] = g;
    }
    if (threadIdx.x == 0) {
        if (bad) atomicOr(err, DEV_ERR_INDEX);
        row_loss[row] = t >= 0 ? z - target : 0.0f;
    }
    xs.copy_row(row, t >= 0);
}

// The mean of the rows' losses, and 1 / their number, by one CTA in a fixed order.
// Returns the latter to every thread.
__device__ __forceinline__ float rows_mean(const float *row_loss, int64_t T, const XentRows &x,
                                           float *mean, float *inv) {
    __shared__ float sl[32];
    __shared__ int sc[32];
    float sum = 0.0f;
    int count = 0;
    for (int64_t i = threadIdx.x; i < T; i += blockDim.x) {
        bool bad = false;
        sum += row_loss[i];
        count += x.at(i, bad) >= 0;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    count = (int)__reduce_add_sync(0xffffffffu, count);
    if ((threadIdx.x & 31) == 0) sl[threadIdx.x >> 5] = sum, sc[threadIdx.x >> 5] = count;
    __syncthreads();
    sum = 0.0f, count = 0;
    for (int i = 0; i < (int)blockDim.x / 32; i++) sum += sl[i], count += sc[i];
    const float c = (float)max(count, 1);
    if (threadIdx.x == 0 && mean) {
        *mean = sum / c;
        *inv = 1.0f / c;
    }
    return 1.0f / c;
}
__global__ void __launch_bounds__(1024) xent_mean_kernel(const float *row_loss, int64_t T,
                                                         XentRows x, float *mean, float *inv) {
    pdl_trigger();
    pdl_wait();
    rows_mean(row_loss, T, x, mean, inv);
}

// db of the kept logits' d, and the mean: every CTA counts the rows for itself, the
// first one writes the mean and the inverse count.
__global__ void __launch_bounds__(256) xent_mean_db_kernel(const float *row_loss, int64_t T,
                                                           XentRows x, float *mean, float *inv,
                                                           const float *d, int64_t n, int64_t ld,
                                                           float *db) {
    pdl_trigger();
    pdl_wait();
    __shared__ float sh[8][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t v = (int64_t)blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (v < n) {
#pragma unroll 4
        for (int64_t i = slice; i < T; i += 8) s += d[i * ld + v];
    }
    sh[slice][lane] = s;
    const float k = rows_mean(row_loss, T, x, blockIdx.x == 0 ? mean : nullptr, inv);  // syncs
    if (slice || v >= n) return;
    for (int i = 1; i < 8; i++) s += sh[i][lane];
    db[v] = s * k;
}

// ------------------------------------------------------------------ plans

static int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
static int tiles(int64_t x) { return (int)((x + tc::kTile - 1) / tc::kTile); }
static int stages(int64_t k) { return (int)((k + 63) / 64); }

// Pairs of SMs that the plans cut contractions for: a B200's, and not the current
// device's, which need not be the context's when a workspace's size is asked for. (The
// launches then ask for the device's own.)
constexpr int kPlanPairs = 74;

// The forward pass holds 16 bytes a row and 256 columns; pieces keep that near
// 64 MB.
struct ForwardPlan {
    int64_t piece, parts, target, run, bytes;  // offsets in the workspace
};
static ForwardPlan forward_plan(const drift_xent *op) {
    ForwardPlan p;
    const int64_t t = std::max<int64_t>(op->tokens, 1);
    p.piece = std::min(up(op->vocab, 256), std::max<int64_t>(1, (64LL << 20) / (t * 16)) * 256);
    p.parts = 0;
    p.target = up(t * (p.piece / 128) * 8, 256);
    p.run = p.target + up(t * 4, 256);
    p.bytes = p.run + up(t * 8, 256);
    return p;
}

// A piece of d is near 256 MB: large enough that the pass over the fp32 sums of
// dx that each piece costs (8 bytes an element of dx) is small beside the
// piece's products, small enough to be no burden beside W.
struct GradPlan {
    int64_t piece, ld, d, sums, acc, part, acc_ld, scale, x, x_ld, bytes;
    int pieces, splits;
    bool direct;  // dx in one product, rounded by its epilogue
};
static GradPlan grad_plan(const drift_xent *op) {
    GradPlan p;
    const int64_t t = std::max<int64_t>(op->tokens, 1);
    p.piece = std::min(up(op->vocab, 256), std::max<int64_t>(256, (128LL << 20) / t / 256 * 256));
    p.pieces = (int)((op->vocab + p.piece - 1) / p.piece);
    p.ld = std::min(p.piece, up(op->vocab, 8));
    // dx contracts the vocabulary: with few tokens its tiles are fewer than the
    // pairs of SMs, and the contraction is cut so that they all have work, down
    // to 16 stages (1024 entries) a part.
    const int dx_tiles = tiles(t) * tiles(op->depth);
    const int most = std::max(1, stages(p.ld) / 16);
    p.splits = std::max(1, std::min(most, kPlanPairs / dx_tiles));
    p.direct = p.pieces == 1 && p.splits == 1;
    p.acc_ld = up(op->depth, 4);
    p.part = t * p.acc_ld;
    p.d = 0;
    p.sums = up(t * p.ld * 2, 256);
    // Whether db is wanted is not known here, and a bias does not say. A sixteenth of d for
    // many tokens.
    p.acc = p.sums + up(up(t, 256) / 32 * p.ld * 4, 256);
    p.scale = p.acc + (p.direct ? 0 : up(p.splits * p.part * 4, 256));
    p.x_ld = up(op->depth, 8);
    p.x = p.scale + 256;
    p.bytes = p.x + up(t * p.x_ld * 2, 256);
    return p;
}

// Up to 64 MB of fp32 logits are kept between the loss and its gradient, which
// then costs 6 T D V operations and not 8: writing and reading them back is 8
// bytes an element in L2, computing them again 2 D operations. A CTA takes a row,
// so rows longer than 2^15 (some 20 us) are left to the other way.
struct KeptPlan {
    bool use;
    int64_t ld, part, logits, d, loss, inv, acc, acc_part, acc_ld, x, x_ld, bytes;
    int splits, dx_splits;
};
static KeptPlan kept_plan(const drift_xent *op) {
    KeptPlan p;
    const int64_t t = std::max<int64_t>(op->tokens, 1);
    p.ld = up(op->vocab, 8);
    p.use = op->tokens > 0 && op->vocab <= 32768 && t * p.ld <= (16LL << 20);
    p.part = t * p.ld;
    if (!p.use) return p;
    // Few tiles: the contractions are cut, down to two stages a part here, where a
    // part is a pass over the logits in L2, and 16 for dx.
    const int lt = tiles(t) * tiles(op->vocab), dt = tiles(t) * tiles(op->depth);
    p.splits = std::max(1, std::min({stages(op->depth) / 2, kPlanPairs / lt, 16}));
    p.dx_splits = std::max(1, std::min(stages(op->vocab) / 16, kPlanPairs / dt));
    p.logits = 0;
    p.d = up(p.splits * p.part * 4, 256);
    p.loss = p.d + up(p.part * 2, 256);
    p.acc_ld = up(op->depth, 4);
    p.acc_part = t * p.acc_ld;
    p.inv = p.loss + up(t * 4, 256);
    p.acc = p.inv + 256;
    p.x_ld = up(op->depth, 8);
    p.x = p.acc + (p.dx_splits > 1 ? up(p.dx_splits * p.acc_part * 4, 256) : 0);
    p.bytes = p.x + up(t * p.x_ld * 2, 256);
    return p;
}

int64_t xent_workspace(const drift_xent *op, int mode) {
    if (mode == 2) {
        const KeptPlan k = kept_plan(op);
        if (k.use) return k.bytes;
    }
    const int64_t f = forward_plan(op).bytes;
    return mode ? std::max(f, grad_plan(op).bytes) + (mode == 2 ? up(op->tokens * 4, 256) + 256 : 0) : f;
}

static XentRows rows_of(const drift_xent *op) {
    return XentRows{op->targets, op->target_bits == 64, op->ignore_index, op->vocab};
}

static int launch_mean(const float *row_loss, int64_t n, const XentRows &rows, float *mean,
                       float *inv, cudaStream_t st) {
    return launch_pdl(xent_mean_kernel, dim3(1), n <= 256 ? 256 : 1024, 0, st, 0, row_loss, n, rows,
                      mean, inv);
}

// x's rows start on 16-byte boundaries (its stride is whole units), and so do the copy's.
static CopyRows copy_rows(const drift_xent *op, void *to, int64_t to_ld) {
    return CopyRows{static_cast<const uint4 *>(op->x), static_cast<uint4 *>(to), op->x_stride / 8,
                    to_ld / 8, (op->depth + 7) / 8, (int)((op->depth - 1) % 8) + 1};
}

static int done() { return cudaGetLastError() == cudaSuccess ? DRIFT_OK : DRIFT_ECUDA; }

// The maps and shape of a piece's logits: x (T x D) against rows v0 .. of W.
static bool logit_args(tc::Args &a, const drift_xent *op, int64_t v0, int64_t n, bool bf16,
                       int *err) {
    const char *w = static_cast<const char *>(op->w) + v0 * op->w_stride * 2;
    a.m_tiles = tiles(op->tokens);
    a.n_tiles = tiles(n);
    a.k_stages = stages(op->depth);
    a.splits = 1;
    a.run = kLogitRun;
    a.err = err;
    return tc::encode_16(&a.a, bf16, op->x, op->tokens, op->depth, op->x_stride, true) &&
           tc::encode_16(&a.b, bf16, w, n, op->depth, op->w_stride, true);
}

template <bool BF16>
static int forward(const drift_xent *op, float *loss, float *lse, float *mean, float *inv, char *ws,
                   int *err, cudaStream_t st) {
    const ForwardPlan p = forward_plan(op);
    const int64_t n_t = op->tokens;
    const XentRows rows = rows_of(op);
    Stat *parts = reinterpret_cast<Stat *>(ws + p.parts);
    Stat *run = reinterpret_cast<Stat *>(ws + p.run);
    float *target = reinterpret_cast<float *>(ws + p.target);
    // Where the caller wants no losses but their mean, they take the place of the
    // targets' logits, which the last join reads just before.
    float *row_loss = loss ? loss : target;
    for (int64_t v0 = 0; n_t && v0 < op->vocab; v0 += p.piece) {
        const int64_t n = std::min(p.piece, op->vocab - v0);
        tc::Args a;
        if (!logit_args(a, op, v0, n, BF16, err)) return DRIFT_ECUDA;
        const StatsEpi epi{parts, target, op->bias ? op->bias + v0 : nullptr, n_t, n, v0, rows};
        int rc = tc::launch<tc::KIND_16, BF16, false, false>(a, epi, sm_count(), st);
        if (rc) return rc;
        const int n_parts = (int)((n + 127) / 128);
        const bool few = n_t < 256;
        rc = launch_pdl(few ? xent_join_kernel<1> : xent_join_kernel<32>,
                        dim3((unsigned)(few ? n_t : (n_t + 31) / 32)), few ? 128 : 1024, 0, st, 0,
                        parts, n_parts, n_t, run, v0 == 0, v0 + n == op->vocab, target, rows,
                        row_loss, lse, err);
        if (rc) return rc;
    }
    return mean ? launch_mean(row_loss, n_t, rows, mean, inv, st) : DRIFT_OK;
}

template <class T, bool BF16>
static int backward(const drift_xent *op, const float *lse, const float *g, int64_t g_stride, T *dx,
                    int64_t dx_stride, T *dw, int64_t dw_stride, float *db, char *ws, int *err,
                    cudaStream_t st) {
    const GradPlan p = grad_plan(op);
    const int64_t n_t = op->tokens, dep = op->depth;
    if (n_t == 0) {
        if (dw) cudaMemset2DAsync(dw, dw_stride * 2, 0, dep * 2, op->vocab, st);
        if (db) cudaMemsetAsync(db, 0, op->vocab * 4, st);
        return done();
    }
    const XentRows rows = rows_of(op);
    T *d = reinterpret_cast<T *>(ws + p.d);
    float *sums = reinterpret_cast<float *>(ws + p.sums);
    float *acc = reinterpret_cast<float *>(ws + p.acc);
    // One weight for all rows multiplies the results, and d is the plain p - [v = t]:
    // its large entries lie just below 1, where the type's steps are finest for their
    // size. Weights by row go into d.
    const bool one = g_stride == 0;
    float *scale = BF16 || one ? nullptr : reinterpret_cast<float *>(ws + p.scale);
    if (scale) {
        const int rc = launch_pdl(xent_scale_kernel, dim3(1), 1024, 0, st, 0, g, g_stride, rows,
                                  n_t, scale);
        if (rc) return rc;
    }
    const float fixed = !BF16 && one ? 32768.0f : 1.0f;
    const float *undo = one ? g : scale ? scale + 1 : nullptr, *sum_undo = one ? g : nullptr;
    const float beta = 1.0f / fixed;
    const float *row_g = one ? nullptr : g;
    T *x = reinterpret_cast<T *>(ws + p.x);
    if (dw) {
        const int rc = launch_pdl(xent_copy_kernel, dim3((unsigned)n_t), 128, 0, st, 0,
                                  copy_rows(op, x, p.x_ld), rows);
        if (rc) return rc;
    }
    for (int64_t v0 = 0; v0 < op->vocab; v0 += p.piece) {
        const int64_t n = std::min(p.piece, op->vocab - v0);
        tc::Args a;
        if (!logit_args(a, op, v0, n, BF16, err)) return DRIFT_ECUDA;
        const float *bias = op->bias ? op->bias + v0 : nullptr;
        a.early = !db;
        int rc;
        if (db) {
            const GradEpi<T, true> epi{d,   p.ld,  bias,     n_t,   n,     v0,  rows,
                                       lse, row_g, g_stride, scale, fixed, sums};
            rc = tc::launch<tc::KIND_16, BF16, false, false>(a, epi, sm_count(), st);
            if (!rc)
                rc = launch_pdl(xent_colsum_kernel, dim3((unsigned)((n + 31) / 32)), 256, 0, st, 0,
                                sums, (n_t + 31) / 32, n, n, sum_undo, db + v0);
        } else {
            const GradEpi<T, false> epi{d,   p.ld,  bias,     n_t,   n,     v0,     rows,
                                        lse, row_g, g_stride, scale, fixed, nullptr};
            rc = tc::launch<tc::KIND_16, BF16, false, false>(a, epi, sm_count(), st);
        }
        if (rc) return rc;
        const char *w = static_cast<const char *>(op->w) + v0 * op->w_stride * 2;
        if (dx) {
            // dx (T x D) contracts the piece: d K-major, W's rows are k.
            if (!tc::encode_16(&a.a, BF16, d, n_t, n, p.ld, true) ||
                !tc::encode_16(&a.b, BF16, w, dep, n, op->w_stride, false))
                return DRIFT_ECUDA;
            a.m_tiles = tiles(n_t), a.n_tiles = tiles(dep), a.k_stages = stages(n);
            a.run = kGradRun;
            a.splits = std::min(p.splits, a.k_stages);
            a.early = p.direct;
            if (p.direct) {
                const StoreEpi<T> epi{dx, dx_stride, n_t, dep, nullptr, undo, beta,
                                      rows_aligned(dx, dx_stride)};
                rc = tc::launch<tc::KIND_16, BF16, false, true>(a, epi, sm_count(), st);
            } else {
                const PartEpi epi{acc, p.part, p.acc_ld, n_t, dep, v0 > 0};
                rc = tc::launch<tc::KIND_16, BF16, false, true>(a, epi, sm_count(), st);
            }
            if (rc) return rc;
        }
        if (dw) {
            // dW (piece x D) contracts the tokens: rows of d and of x are k.
            if (!tc::encode_16(&a.a, BF16, d, n, n_t, p.ld, false) ||
                !tc::encode_16(&a.b, BF16, x, dep, n_t, p.x_ld, false))
                return DRIFT_ECUDA;
            a.m_tiles = tiles(n), a.n_tiles = tiles(dep), a.k_stages = stages(n_t);
            a.splits = 1, a.run = kGradRun, a.early = p.direct;
            T *to = dw + v0 * dw_stride;
            const StoreEpi<T> epi{to,      dw_stride, n,    dep,
                                  nullptr, undo,      beta, rows_aligned(to, dw_stride)};
            rc = tc::launch<tc::KIND_16, BF16, true, true>(a, epi, sm_count(), st);
            if (rc) return rc;
        }
    }
    if (dx && !p.direct)
        return launch_pdl(xent_dx_kernel<T>, dim3(sm_count() * 8), 256, 0, st, 0, acc, p.splits,
                          p.part, p.acc_ld, dx, n_t, dep, dx_stride, undo, beta);
    return DRIFT_OK;
}

template <class T, bool BF16>
static int mean_kept(const drift_xent *op, const KeptPlan &p, float *mean, T *dx, int64_t dx_stride,
                     T *dw, int64_t dw_stride, float *db, char *ws, int *err, cudaStream_t st) {
    const int64_t n_t = op->tokens, dep = op->depth, n = op->vocab;
    const XentRows rows = rows_of(op);
    float *logits = reinterpret_cast<float *>(ws + p.logits);
    float *row_loss = reinterpret_cast<float *>(ws + p.loss);
    float *acc = reinterpret_cast<float *>(ws + p.acc);
    T *d = reinterpret_cast<T *>(ws + p.d);
    float *inv = reinterpret_cast<float *>(ws + p.inv);
    T *x = reinterpret_cast<T *>(ws + p.x);
    const float scale = BF16 ? 1.0f : 32768.0f, beta = 1.0f / scale;
    tc::Args a;
    if (!logit_args(a, op, 0, n, BF16, err)) return DRIFT_ECUDA;
    a.splits = std::min(p.splits, a.k_stages), a.early = false;
    int rc = tc::launch<tc::KIND_16, BF16, false, false>(
        a, PartEpi{logits, p.part, p.ld, n_t, n, false}, sm_count(), st);
    if (rc) return rc;
    rc = launch_pdl(xent_row_kernel<T>, dim3((unsigned)n_t), 256, 0, st, 0, logits, a.splits, p.part,
                    p.ld, n, op->bias, rows, d, scale, db != nullptr, row_loss,
                    dw ? copy_rows(op, x, p.x_ld) : CopyRows{}, err);
    // Few rows: one kernel for the mean and db, whose CTAs all read the targets.
    if (!rc && db && n_t <= 4096) {
        rc = launch_pdl(xent_mean_db_kernel, dim3((unsigned)((n + 31) / 32)), 256, 0, st, 0,
                        row_loss, n_t, rows, mean, inv, logits, n, p.ld, db);
    } else {
        if (!rc) rc = launch_mean(row_loss, n_t, rows, mean, inv, st);
        if (!rc && db)
            rc = launch_pdl(xent_colsum_kernel, dim3((unsigned)((n + 31) / 32)), 256, 0, st, 0,
                            logits, n_t, n, p.ld, inv, db);
    }
    if (!rc && dx) {
        if (!tc::encode_16(&a.a, BF16, d, n_t, n, p.ld, true) ||
            !tc::encode_16(&a.b, BF16, op->w, dep, n, op->w_stride, false))
            return DRIFT_ECUDA;
        a.m_tiles = tiles(n_t), a.n_tiles = tiles(dep), a.k_stages = stages(n);
        a.splits = std::min(p.dx_splits, a.k_stages), a.run = kGradRun;
        a.early = a.splits == 1;
        if (a.splits == 1) {
            const StoreEpi<T> epi{dx,      dx_stride, n_t,  dep,
                                  nullptr, inv,       beta, rows_aligned(dx, dx_stride)};
            rc = tc::launch<tc::KIND_16, BF16, false, true>(a, epi, sm_count(), st);
        } else {
            const PartEpi epi{acc, p.acc_part, p.acc_ld, n_t, dep, false};
            rc = tc::launch<tc::KIND_16, BF16, false, true>(a, epi, sm_count(), st);
            if (!rc)
                rc = launch_pdl(xent_dx_kernel<T>, dim3(sm_count() * 8), 256, 0, st, 0, acc, a.splits,
                                p.acc_part, p.acc_ld, dx, n_t, dep, dx_stride, inv, beta);
        }
    }
    if (!rc && dw) {
        if (!tc::encode_16(&a.a, BF16, d, n, n_t, p.ld, false) ||
            !tc::encode_16(&a.b, BF16, x, dep, n_t, p.x_ld, false))
            return DRIFT_ECUDA;
        a.m_tiles = tiles(n), a.n_tiles = tiles(dep), a.k_stages = stages(n_t);
        a.splits = 1, a.run = kGradRun;
        const StoreEpi<T> epi{dw,      dw_stride, n,    dep,
                              nullptr, inv,       beta, rows_aligned(dw, dw_stride)};
        rc = tc::launch<tc::KIND_16, BF16, true, true>(a, epi, sm_count(), st);
    }
    return rc;
}

int launch_xent_mean(const drift_xent *op, float *mean, void *dx, int64_t dx_stride, void *dw,
                     int64_t dw_stride, float *db, void *ws, int *err, cudaStream_t st) {
    const KeptPlan k = kept_plan(op);
    if (k.use)
        return op->type == DRIFT_T_BF16
                   ? mean_kept<__nv_bfloat16, true>(op, k, mean, (__nv_bfloat16 *)dx, dx_stride,
                                                    (__nv_bfloat16 *)dw, dw_stride, db, (char *)ws,
                                                    err, st)
                   : mean_kept<__half, false>(op, k, mean, (__half *)dx, dx_stride, (__half *)dw,
                                              dw_stride, db, (char *)ws, err, st);
    char *more = (char *)ws + std::max(forward_plan(op).bytes, grad_plan(op).bytes);
    float *inv = reinterpret_cast<float *>(more), *lse = reinterpret_cast<float *>(more + 256);
    const int rc = op->type == DRIFT_T_BF16
                       ? forward<true>(op, nullptr, lse, mean, inv, (char *)ws, err, st)
                       : forward<false>(op, nullptr, lse, mean, inv, (char *)ws, err, st);
    return rc ? rc
              : launch_xent_grad(op, lse, inv, 0, dx, dx_stride, dw, dw_stride, db, ws, err, st);
}

int launch_xent(const drift_xent *op, float *loss, float *lse, float *mean, void *ws, int *err,
                cudaStream_t st) {
    return op->type == DRIFT_T_BF16 ? forward<true>(op, loss, lse, mean, mean + 1, (char *)ws, err, st)
                                    : forward<false>(op, loss, lse, mean, mean + 1, (char *)ws, err, st);
}

int launch_xent_grad(const drift_xent *op, const float *lse, const float *g, int64_t g_stride,
                     void *dx, int64_t dx_stride, void *dw, int64_t dw_stride, float *db, void *ws,
                     int *err, cudaStream_t st) {
    if (op->type == DRIFT_T_BF16)
        return backward<__nv_bfloat16, true>(op, lse, g, g_stride, (__nv_bfloat16 *)dx, dx_stride,
                                             (__nv_bfloat16 *)dw, dw_stride, db, (char *)ws, err,
                                             st);
    return backward<__half, false>(op, lse, g, g_stride, (__half *)dx, dx_stride, (__half *)dw,
                                   dw_stride, db, (char *)ws, err, st);
}

}  // namespace drift
