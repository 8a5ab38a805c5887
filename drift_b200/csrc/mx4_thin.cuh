// mx4_thin.cuh — the packed 4-bit product for few rows of A (tokens): the rows
// of B (weights) take the tensor cores' 128 lanes and a tile of NT tokens its
// columns, so that a single token wastes no reads, and a cluster of CTAs shares
// a tile's contraction, so that few tiles still reach every SM.
//
// Bound: the bytes of B, and for small products the latency of one launch; an SM
// keeps 160 KB and more of B in flight. Measured on one B200, back to back: one token
// through 8192 x 8192 7.5 us (35.7 MB, 4.8 TB/s), 64 through 2048 x 2048 4.7 us, 1 x
// 1 x 64 2.6 us. One CTA an SM with eight stages took 10.4 us for the first.
//
// The cluster's partial tiles meet in shared memory: CTA r adds up tokens
// [NT r / S, NT (r + 1) / S) of all S, in order, so results do not depend on timing.
#pragma once

#include "epilogue.cuh"
#include "tc.cuh"

namespace drift {
namespace thin {

constexpr int kThreads = 224;  // warps 0-3 epilogue, 4 TMA, 5 MMA, 6 scales
constexpr int kTmemCols = 256;
constexpr int kScaleCol = 128;

template <int NT> struct Shape {
    static constexpr int stage = 16384 + NT * 128 + 2048;
    // Up to 32 tokens two CTAs share an SM: one's scale copies and start fill the
    // other's waits.
    static constexpr int per_sm = NT <= 32 ? 2 : 1;
    static constexpr int stages = NT == 16 ? 5 : NT == 32 ? 4 : NT == 64 ? 7 : 6;
    static constexpr int smem = stage * stages + 1024;
    static_assert(NT * 512 <= stage * stages, "the partial tile reuses the stages");
    static_assert(NT <= kScaleCol && kScaleCol + stages * 16 <= kTmemCols, "TMEM columns");
};

struct Args {
    CUtensorMap w, x, sfw, sfx;  // weights (B) and tokens (A), and their scales
    int64_t rows, tokens;        // of weights, of tokens
    int w_tiles, k_stages;       // fewer than 128 columns: all tokens in one tile
    const float *bias;           // per weight row
    void *c;
    int64_t stride;
    bool vec;                    // rows of c start 16-byte aligned
    int *err;
};

__device__ __forceinline__ void tmem_load16(unsigned addr, float *v) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void copy_scales(unsigned to, uint64_t from) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(from)
                 : "memory");
}
__device__ __forceinline__ float4 load_cluster(unsigned addr) {
    float4 f;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                 : "r"(addr)
                 : "memory");
    return f;
}
// Four values, the address aligned to them.
template <class T> __device__ __forceinline__ void store4(T *p, const float (&y)[4]) {
    if constexpr (sizeof(T) == 8) {
        reinterpret_cast<double2 *>(p)[0] = make_double2(y[0], y[1]);
        reinterpret_cast<double2 *>(p)[1] = make_double2(y[2], y[3]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
    }
}

template <int NT, class T>
__global__ void __launch_bounds__(kThreads, Shape<NT>::per_sm) thin_kernel(const __grid_constant__ Args args) {
    using S = Shape<NT>;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::stages], empty[S::stages], sf_full[S::stages], acc_full;
    __shared__ unsigned tmem_base;
    const unsigned base = (smem_addr(raw) + 1023) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned ranks;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const unsigned rank = tc::cta_rank();
    const int tile = blockIdx.x / ranks;
    const int tw = tile % args.w_tiles, tt = tile / args.w_tiles;
    const int k0 = (int)((int64_t)args.k_stages * rank / ranks);
    const int k1 = (int)((int64_t)args.k_stages * (rank + 1) / ranks);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::stages; s++)
            mbar_init(&full[s], 1), mbar_init(&empty[s], 1), mbar_init(&sf_full[s], 1);
        mbar_init(&acc_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_addr(&tmem_base)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    const unsigned tmem = tmem_base;
    bool ok = true;
    pdl_wait();

    if (warp == 4) {
        if (lane == 0) {
            int s = 0;
            unsigned ph = 1;
            for (int k = k0; k < k1; k++) {
                ok = tc::wait(&empty[s], ph);
                if (!ok) break;
                mbar_expect_tx(&full[s], S::stage);
                const unsigned at = base + s * S::stage;
                const auto load = [&](unsigned to, const CUtensorMap *map, int x, int y) {
                    asm volatile(
                        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
                        " [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
                        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y),
                        "r"(smem_addr(&full[s]))
                        : "memory");
                };
                load(at, &args.w, k * 128, tw * 128);
                load(at + 16384, &args.x, k * 128, tt * NT);
                load(at + 16384 + NT * 128, &args.sfw, k * 256, tw);
                load(at + 16384 + NT * 128 + 1024, &args.sfx, k * 256, tt);
                if (++s == S::stages) s = 0, ph ^= 1;
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0) {
            // e2m1 by e2m1, E8M0 scales, 128 lanes, NT columns.
            const unsigned idesc = (unsigned)(NT >> 3) << 17 | 8u << 24 | 1u << 7 | 1u << 10 |
                                   1u << 23;
            const uint64_t da = tc::smem_desc(base, 16, 1024, 2);
            const uint64_t db = tc::smem_desc(base + 16384, 16, 1024, 2);
            int s = 0;
            unsigned ph = 0;
            for (int k = k0; k < k1; k++) {
                ok = tc::wait(&sf_full[s], ph);  // completes after the operands' barrier
                if (!ok) break;
                tc::fence_after();
                const unsigned fa = tmem + kScaleCol + s * 16, fb = fa + 8;
                const unsigned off = s * (S::stage >> 4);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const unsigned id = (j & 1) * 2;
                    asm volatile(
                        "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
                        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X"
                        " [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(tmem),
                        "l"(da + off + j * 2), "l"(db + off + j * 2),
                        "r"(idesc | id << 4 | id << 29), "r"(fa + (j >> 1) * 4),
                        "r"(fb + (j >> 1) * 4), "r"((unsigned)(j > 0 || k > k0))
                        : "memory");
                }
                commit(&empty[s]);
                if (++s == S::stages) s = 0, ph ^= 1;
            }
            if (ok) commit(&acc_full);
        }
        __syncwarp();
    } else if (warp == 6) {
        // A thread of their own issues the scale copies: in the MMAs' thread they would
        // run between them, not beside them.
        if (lane == 0) {
            int s = 0;
            unsigned ph = 0;
            for (int k = k0; k < k1; k++) {
                ok = tc::wait(&full[s], ph);
                if (!ok) break;
                tc::fence_after();
                const unsigned at = tmem + kScaleCol + s * 16;
                const uint64_t from =
                    tc::smem_desc(base + s * S::stage + 16384 + NT * 128, 0, 128, 0);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    copy_scales(at + h * 4, from + h * 32);
                    copy_scales(at + 8 + h * 4, from + 64 + h * 32);
                }
                commit(&sf_full[s]);
                if (++s == S::stages) s = 0, ph ^= 1;
            }
        }
        __syncwarp();
    } else {
        ok = __all_sync(0xffffffffu,
                        tc::wait(&acc_full, 0, (long long)(k1 - k0) * tc::kRoundsPerStage));
        tc::fence_after();
        const int64_t r = (int64_t)tw * 128 + warp * 32 + lane;
        const float b = args.bias && r < args.rows ? args.bias[r] : 0.0f;
        T *c = static_cast<T *>(args.c) + r;
#pragma unroll
        for (int j0 = 0; j0 < NT; j0 += 16) {
            float v[16];
            tmem_load16(tmem + j0 + ((unsigned)(warp * 32) << 16), v);
            tc::tmem_wait_load();
            if (ranks == 1) {
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int64_t t = (int64_t)tt * NT + j0 + j;
                    if (ok && r < args.rows && t < args.tokens) c[t * args.stride] = T(v[j] + b);
                }
            } else {
                // Every MMA is done, so every stage has been read.
#pragma unroll
                for (int j = 0; j < 16; j++)
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(
                                     base + ((j0 + j) * 128 + warp * 32 + lane) * 4),
                                 "f"(v[j])
                                 : "memory");
            }
        }
        tc::fence_before();
    }

    pdl_trigger();
    if (!ok) {
        atomicOr(args.err, DEV_ERR_TIMEOUT);
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    }
    __syncthreads();
    if (ranks > 1) {
        tc::cluster_sync();
        // A warp a token, four rows a lane, all ranks' loads of two tokens in flight.
        const int64_t r = (int64_t)tw * 128 + lane * 4;
        float b[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            b[i] = args.bias && r + i < args.rows ? args.bias[r + i] : 0.0f;
        const int t1 = min((int)(NT * (rank + 1) / ranks),
                           (int)min(args.tokens - (int64_t)tt * NT, (int64_t)NT));
        unsigned from[8];
#pragma unroll
        for (unsigned q = 0; q < 8; q++) from[q] = tc::map_cta(base + lane * 16, q < ranks ? q : 0);
        for (int t = (int)(NT * rank / ranks) + warp; t < t1; t += 2 * kThreads / 32) {
            float4 part[2][8];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (unsigned q = 0; q < 8; q++)
                    if (q < ranks && t + u * (kThreads / 32) < t1)
                        part[u][q] = load_cluster(from[q] + (t + u * (kThreads / 32)) * 512);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int tu = t + u * (kThreads / 32);
                if (tu >= t1) break;
                float4 sum = part[u][0];
#pragma unroll
                for (unsigned q = 1; q < 8; q++)
                    if (q < ranks) {
                        sum.x += part[u][q].x, sum.y += part[u][q].y;
                        sum.z += part[u][q].z, sum.w += part[u][q].w;
                    }
                const float y[4] = {sum.x + b[0], sum.y + b[1], sum.z + b[2], sum.w + b[3]};
                T *c = static_cast<T *>(args.c) + ((int64_t)tt * NT + tu) * args.stride + r;
                if (!ok) break;
                if (args.vec && r + 4 <= args.rows) {
                    store4(c, y);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (r + i < args.rows) c[i] = T(y[i]);
                }
            }
        }
        __syncwarp();
        tc::cluster_sync();
    }
    tc::fence_after();
    if (warp == 5)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(kTmemCols));
}

template <int NT, class T>
inline int launch(Args &args, int t_tiles, int split, cudaStream_t st) {
    const auto kernel = thin_kernel<NT, T>;
    static unsigned long long done = 0;
    if (!allow_smem(kernel, Shape<NT>::smem, done)) return DRIFT_ECUDA;
    return launch_pdl(kernel, dim3((unsigned)(args.w_tiles * t_tiles * split)), kThreads,
                      Shape<NT>::smem, st, split, args);
}

}  // namespace thin
}  // namespace drift
