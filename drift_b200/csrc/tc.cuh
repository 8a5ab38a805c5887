// tc.cuh — fifth-generation tensor-core products shared by the packed 4-bit
// GEMM and the linear cross entropy: a persistent kernel of CTA pairs whose
// epilogue is a functor.
//
//   D(i, o) = sum_k A(i, k) B(o, k), fp32, for kinds
//   KIND_16   A and B bf16 or fp16; each stored with k contiguous (K-major) or
//             with i (o) contiguous (MN-major);
//   KIND_MX4  packed e2m1 codes with power-of-two scales per 32 (mx4.cuh).
//
// A pair of CTAs owns a 256 x 256 tile: each loads 128 rows of A and 128 of B
// (the pair's MMA reads B from both), 128 bytes of k a stage, so a stage costs
// an SM 32 KiB of L2 reads per 512 tensor cycles in either kind: 64 bytes a
// cycle. A 128 x 256 tile of one CTA would need 96 and stall on them.
//
// Warps: 0-7 epilogue (two per quadrant of TMEM lanes, 128 columns each), 8
// fetches with TMA, 9 allocates TMEM and, in the pair's first CTA, issues the
// MMAs, 10 issues KIND_MX4's copies of scales to TMEM, in a thread of its own so
// that they run beside the MMAs, and 11 completes the group. A stage's barrier
// `full` sits in the first CTA and counts both CTAs' bytes; a commit of the stage's
// MMAs frees it in both CTAs. The accumulator passes to the epilogue by `acc_full`
// (a commit to both) and back by `acc_empty` (first CTA, one arrival an epilogue
// warp of either). The epilogue moves its 128 columns to registers first and then
// hands TMEM back, so the next tile's MMAs overlap its arithmetic and stores.
// KIND_16 has two accumulators (2 x 256 columns); KIND_MX4 has one, and 24 columns
// of scales a stage.
//
// Measured on one B200: KIND_16 1.49 PFLOP/s (92 % of a library product's rate) over
// 4096 x 131072 x 4096 in a burst, 1.2 under the power cap. KIND_MX4 5.07 PFLOP/s at
// 8192^3, 4.5 at 8192 x 8192 x 4096 (issued from the MMAs' thread, the scale copies
// queued between them, 60 cycles each: 3.8 and 3.4; copied with tcgen05.st by warps
// of their own, 2.7 and 2.5). The tensor pipe is busy 63 to 68 % of KIND_16's time at
// 2048 x 32768 x 4096 under the counters' cold caches, DRAM 9 to 16 %. By count shared
// memory is near its limit: a stage is written once and read by both CTAs' MMAs,
// 64 KiB in their 512 cycles, at 128 bytes a cycle all there is. No counter has shown
// that it is what holds KIND_MX4, whose pipe is busy 48 % of the time.
//
// Every wait is bounded; one that gives up flags DEV_ERR_TIMEOUT and the
// kernel drains and returns.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "pdl.cuh"
#include "tma.cuh"

namespace drift {
namespace tc {

constexpr int kRows = 128;            // rows of A, and of B, that one CTA loads
constexpr int kTile = 256;            // rows and columns of a pair's tile
constexpr int kStageBytes = 128;      // bytes of k in a stage
constexpr int kOperand = kRows * kStageBytes;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 4) * 32;  // three warpgroups
// Registers: 384 threads launch with 168 each; the control warpgroup gives 112 a
// thread back, from which each epilogue thread takes 56: (2 * 224 + 56) * 128 =
// 168 * 384, exactly the launch's total.
constexpr int kControlRegs = 56, kEpiRegs = 224;
static_assert(2 * kEpiRegs + kControlRegs == 3 * 168, "the split must not exceed the launch's");
constexpr int kWarpTma = kEpiWarps, kWarpMma = kEpiWarps + 1, kWarpScales = kEpiWarps + 2;
// A round of a wait is some 30 ns at the least, a stage of a contraction about 700 ns:
// 30 ms for a wait on one stage, and 64 rounds more for every stage that a wait spans.
constexpr int kWaitRounds = 1 << 20, kRoundsPerStage = 64;

enum Kind { KIND_16 = 0, KIND_MX4 = 1 };

template <int KIND> struct Shape;
template <> struct Shape<KIND_16> {
    static constexpr int stage_k = 64;   // elements of k in a stage
    static constexpr int scales = 0;
    static constexpr int stages = 6;
    static constexpr int accs = 2;
};
template <> struct Shape<KIND_MX4> {
    static constexpr int stage_k = 256;
    static constexpr int scales = 1024 + 2048;  // A's 128 rows, B's 256 rows
    static constexpr int stages = 5;
    static constexpr int accs = 1;
    static constexpr int sfa_col = 256, sfb_col = 256 + stages * 8;
};

template <int KIND> constexpr int stage_bytes() { return 2 * kOperand + Shape<KIND>::scales; }
constexpr int kStaging = 32 * 128;  // an epilogue warp's 32 rows of 128 bytes
template <int KIND> constexpr int smem_bytes() {
    return Shape<KIND>::stages * stage_bytes<KIND>() + kEpiWarps * kStaging + 1024;
}

// ------------------------------------------------------------------ PTX

__device__ __forceinline__ unsigned cta_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Shared-memory address of the same object in CTA `rank` of the cluster.
__device__ __forceinline__ unsigned map_cta(unsigned addr, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive_cluster(unsigned addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
                 : "memory");
}
// `more`: rounds beyond the usual limit, for a wait that spans a whole contraction.
__device__ __forceinline__ bool wait(uint64_t *bar, unsigned parity, long long more = 0) {
    const unsigned a = smem_addr(bar);
    for (long long i = 0; i < kWaitRounds + more; i++) {
        unsigned done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            " selp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
// A TMA box into this CTA's shared memory, counted on a barrier of either CTA
// of the pair. x times the element size is a multiple of 16 bytes.
__device__ __forceinline__ void load_pair(unsigned dst, const CUtensorMap *map, int x, int y,
                                          unsigned bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Arrives on the same barrier of both CTAs once this thread's MMAs so far are done.
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// Arrives on a barrier of this CTA once this thread's copies so far are done.
__device__ __forceinline__ void commit_one(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void copy_scales(unsigned to, uint64_t from) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(from)
                 : "memory");
}
// 32 columns of this warp's 32 TMEM lanes, one lane a thread.
__device__ __forceinline__ void tmem_load32(unsigned addr, float *v) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory matrix descriptor: start, leading and stride byte offsets,
// version 1, and the swizzle (2: 128 bytes, 0: none).
__device__ __forceinline__ uint64_t smem_desc(unsigned addr, unsigned lbo, unsigned sbo,
                                              unsigned swizzle) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lbo >> 4) & 0x3fff) << 16 |
           (uint64_t)((sbo >> 4) & 0x3fff) << 32 | 1ULL << 46 | (uint64_t)swizzle << 61;
}

// ------------------------------------------------------------------ the kernel

struct Args {
    CUtensorMap a, b, sfa, sfb;  // sfa, sfb: KIND_MX4
    int m_tiles, n_tiles;        // pair tiles
    int k_stages;                // stages of the whole contraction
    int splits;                  // the contraction is cut into this many parts
    int run = 1 << 30;           // KIND_16: stages summed in TMEM before registers take over
    // Whether the next kernel is set up while the last tiles run. Good before another
    // product or a join of a few small CTAs (2048^3 products in a row: 11.6 -> 10.95
    // us), bad before a kernel of many CTAs, which wait where the tiles work (the
    // gradients of 64 x 2048 x 96: 41.1 -> 45.6 us).
    bool early = true;
    int *err;
};

// Order of the work: within a part of the contraction, bands of up to 16 row
// tiles; in a band the rows vary fastest, so the tiles in flight at one time
// share their columns of B, and A's band stays in L2.
struct Work {
    int m, n, split, k0, k1;
};
__device__ __forceinline__ Work work_at(const Args &a, int t) {
    const int per_split = a.m_tiles * a.n_tiles;
    Work w;
    w.split = t / per_split;
    t -= w.split * per_split;
    const int band = t / (16 * a.n_tiles);
    const int height = min(16, a.m_tiles - band * 16);
    t -= band * 16 * a.n_tiles;
    w.n = t / height;
    w.m = band * 16 + (t - w.n * height);
    w.k0 = (int)((long long)a.k_stages * w.split / a.splits);
    w.k1 = (int)((long long)a.k_stages * (w.split + 1) / a.splits);
    return w;
}

// Instruction descriptor: fp32 accumulators, M 256 and N 256 over the pair.
template <int KIND>
__device__ __forceinline__ unsigned instr_desc(bool bf16, bool a_mn, bool b_mn) {
    const unsigned mn = (unsigned)(kTile >> 3) << 17 | (unsigned)(kTile >> 4) << 24;
    if (KIND == KIND_MX4) return mn | 1u << 7 | 1u << 10 | 1u << 23;  // e2m1, e2m1, E8M0
    return mn | 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (unsigned)a_mn << 15 |
           (unsigned)b_mn << 16;
}

template <int KIND, bool BF16, bool A_MN, bool B_MN, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ Args args, const Epi epi) {
    using S = Shape<KIND>;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::stages], empty[S::stages], acc_full[S::accs], acc_empty[S::accs];
    __shared__ uint64_t sf_full[S::stages];  // KIND_MX4: a stage's scales are in TMEM
    __shared__ unsigned tmem_base;
    const unsigned base = (smem_addr(raw) + 1023) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned rank = cta_rank();
    const int total = args.m_tiles * args.n_tiles * args.splits;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::stages; s++)
            mbar_init(&full[s], 1), mbar_init(&empty[s], 1), mbar_init(&sf_full[s], 1);
        for (int s = 0; s < S::accs; s++)
            mbar_init(&acc_full[s], 1), mbar_init(&acc_empty[s], 2 * kEpiWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_addr(&tmem_base)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        fence_before();
    }
    __syncthreads();
    cluster_sync();
    fence_after();
    const unsigned tmem = tmem_base;
    bool ok = true;
    pdl_wait();

    if (warp >= kEpiWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == kWarpTma && lane == 0) {
            int s = 0;
            unsigned ph = 1;  // parity of the empty barrier to wait for
            int loaded = 0;
            for (int t = first; t < total && ok; t += step) {
                const Work w = work_at(args, t);
                const int ra = w.m * kTile + (int)rank * kRows, rb = w.n * kTile + (int)rank * kRows;
                for (int k = w.k0; k < w.k1; k++) {
                    ok = wait(&empty[s], ph);
                    if (!ok) break;
                    if (rank == 0) mbar_expect_tx(&full[s], 2 * stage_bytes<KIND>());
                    const unsigned bar = map_cta(smem_addr(&full[s]), 0);
                    const unsigned da = base + s * stage_bytes<KIND>(), db = da + kOperand;
                    if (KIND == KIND_MX4) {
                        load_pair(da, &args.a, k * kStageBytes, ra, bar);
                        load_pair(db, &args.b, k * kStageBytes, rb, bar);
                        load_pair(db + kOperand, &args.sfa, k * 256, ra / 128, bar);
                        load_pair(db + kOperand + 1024, &args.sfb, k * 256, w.n * 2, bar);
                    } else {
                        const int kk = k * S::stage_k;
                        if (A_MN) {
                            load_pair(da, &args.a, ra, kk, bar);
                            load_pair(da + kOperand / 2, &args.a, ra + 64, kk, bar);
                        } else {
                            load_pair(da, &args.a, kk, ra, bar);
                        }
                        if (B_MN) {
                            load_pair(db, &args.b, rb, kk, bar);
                            load_pair(db + kOperand / 2, &args.b, rb + 64, kk, bar);
                        } else {
                            load_pair(db, &args.b, kk, rb, bar);
                        }
                    }
                    loaded = min(loaded + 1, S::stages);
                    if (++s == S::stages) s = 0, ph ^= 1;
                }
            }
            // The first CTA's commits also arrive on the second's barriers: stay
            // until the last `loaded` stages' have, in the order of their loads.
            if (loaded < S::stages) s = 0, ph = 0;
            for (int i = 0; i < loaded && ok; i++) {
                ok = wait(&empty[s], ph);
                if (++s == S::stages) s = 0, ph ^= 1;
            }
        } else if (KIND == KIND_MX4 && warp == kWarpScales && rank == 0 && lane == 0) {
            // Scales from shared memory to TMEM, in both CTAs, as soon as they are there.
            if constexpr (KIND == KIND_MX4) {
                int s = 0;
                unsigned ph = 0;
                for (int t = first; t < total && ok; t += step) {
                    const Work w = work_at(args, t);
                    for (int k = w.k0; k < w.k1; k++) {
                        ok = wait(&full[s], ph);
                        if (!ok) break;
                        fence_after();
                        const unsigned fa = tmem + S::sfa_col + s * 8;
                        const unsigned fb = tmem + S::sfb_col + s * 16;
                        // Tiles of scales: 32 lanes of 16 bytes, to all four lane quadrants.
                        const uint64_t sc =
                            smem_desc(base + s * stage_bytes<KIND>() + 2 * kOperand, 0, 128, 0);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            copy_scales(fa + h * 4, sc + h * 32);
                            copy_scales(fb + h * 8, sc + 64 + h * 32);
                            copy_scales(fb + h * 8 + 4, sc + 128 + h * 32);
                        }
                        commit_one(&sf_full[s]);
                        if (++s == S::stages) s = 0, ph ^= 1;
                    }
                }
            }
        } else if (warp == kWarpMma && rank == 0 && lane == 0) {
            // This thread's instructions between two stages are the tensor cores'
            // pauses, so its indexes run along and descriptors are a base plus a
            // stage's offset (addresses fit their field's 14 bits of 16 bytes).
            const unsigned idesc = instr_desc<KIND>(BF16, A_MN, B_MN);
            // MN-major: 64 of i (o) a swizzled row, groups of eight k 1024 bytes apart,
            // the next 64 of i half an operand further.
            const uint64_t da0 = A_MN ? smem_desc(base, kOperand / 2, 1024, 2)
                                      : smem_desc(base, 16, 1024, 2);
            const uint64_t db0 = B_MN ? smem_desc(base + kOperand, kOperand / 2, 1024, 2)
                                      : smem_desc(base + kOperand, 16, 1024, 2);
            constexpr unsigned a_step = A_MN ? 128 : 2, b_step = B_MN ? 128 : 2;
            int s = 0, acc = 0;
            unsigned ph = 0, acc_ph = 1;
            for (int t = first; t < total && ok; t += step) {
                const Work w = work_at(args, t);
                int left = KIND == KIND_16 ? args.run : 1 << 30;  // stages until this sum ends
                unsigned more = 0;
                for (int k = w.k0; k < w.k1; k++) {
                    // The scales' barrier completes after the operands'.
                    ok = wait(KIND == KIND_MX4 ? &sf_full[s] : &full[s], ph);
                    if (!ok) break;
                    fence_after();
                    const unsigned off = s * (stage_bytes<KIND>() >> 4);
                    if (more == 0) {
                        // A sum begins: its accumulator must have been read.
                        ok = wait(&acc_empty[acc], acc_ph);
                        if (!ok) break;
                        fence_after();
                    }
                    const unsigned d = tmem + acc * kTile;
                    if constexpr (KIND == KIND_MX4) {
                        const unsigned fa = tmem + S::sfa_col + s * 8;
                        const unsigned fb = tmem + S::sfb_col + s * 16;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            // 64 elements: two scales of a 32-bit column's four.
                            const unsigned id = (j & 1) * 2;
                            asm volatile(
                                "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
                                " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X"
                                " [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
                                "l"(da0 + off + j * 2), "l"(db0 + off + j * 2),
                                "r"(idesc | id << 4 | id << 29), "r"(fa + (j >> 1) * 4),
                                "r"(fb + (j >> 1) * 8), "r"(j > 0 ? 1u : more)
                                : "memory");
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            asm volatile(
                                "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                                " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                                "l"(da0 + off + j * a_step), "l"(db0 + off + j * b_step),
                                "r"(idesc), "r"(j > 0 ? 1u : more)
                                : "memory");
                    }
                    commit_pair(&empty[s]);
                    more = 1;
                    if (++s == S::stages) s = 0, ph ^= 1;
                    if (--left == 0 || k == w.k1 - 1) {
                        commit_pair(&acc_full[acc]);
                        if (++acc == S::accs) acc = 0, acc_ph ^= 1;
                        left = KIND == KIND_16 ? args.run : 1 << 30;
                        more = 0;
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        const int quad = warp & 3, half = warp >> 2;
        const unsigned staging = base + S::stages * stage_bytes<KIND>() + warp * kStaging;
        int n_acc = 0;
        for (int t = first; t < total && ok; t += step) {
            const Work w = work_at(args, t);
            const int64_t row0 = (int64_t)w.m * kTile + (int)rank * kRows + quad * 32;
            const int64_t col = (int64_t)w.n * kTile + half * 128;
            const bool live = row0 < epi.rows && col < epi.cols;  // else nothing to do
            // What the epilogue loads ahead of its accumulator.
            const auto before = epi.before(row0 + lane, col, lane);
            float v[128];
            const int run = KIND == KIND_16 ? min(args.run, w.k1 - w.k0) : w.k1 - w.k0;
            for (int k = w.k0; k < w.k1; k += run, n_acc++) {
                const int acc = n_acc % S::accs;
                ok = __all_sync(0xffffffffu, wait(&acc_full[acc], n_acc / S::accs & 1,
                                                  (long long)run * kRoundsPerStage));
                if (!ok) break;
                fence_after();
                const unsigned at = tmem + acc * kTile + half * 128 + ((unsigned)(quad * 32) << 16);
                if (!live) {
                } else if (S::accs == 1 || k == w.k0) {
#pragma unroll
                    for (int c = 0; c < 4; c++) tmem_load32(at + c * 32, v + c * 32);
                    tmem_wait_load();
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        float x[32];
                        tmem_load32(at + c * 32, x);
                        tmem_wait_load();
#pragma unroll
                        for (int j = 0; j < 32; j++) v[c * 32 + j] += x[j];
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) arrive_cluster(map_cta(smem_addr(&acc_empty[acc]), 0));
            }
            if (!ok) break;
            if (live) epi.run(v, before, row0, col, w, lane, staging);
        }
    }

    // Not before: a small kernel set up early would crowd on the first SMs to fall
    // free (a join of 32 CTAs then takes twice its time).
    if (args.early) pdl_trigger();
    if (!ok) {
        atomicOr(args.err, DEV_ERR_TIMEOUT);
        // Give copies and MMAs in flight time to land before TMEM and shared
        // memory go.
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    }
    __syncthreads();
    fence_before();
    cluster_sync();
    fence_after();
    if (warp == kWarpMma)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// ------------------------------------------------------------------ host

inline bool encode_2d(CUtensorMap *map, CUtensorMapDataType type, const void *base, uint64_t inner,
                      uint64_t outer, uint64_t stride_bytes, uint32_t box_inner,
                      uint32_t box_outer, CUtensorMapSwizzle swizzle) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {inner, outer}, strides[1] = {stride_bytes};
    const cuuint32_t box[2] = {box_inner, box_outer}, unit[2] = {1, 1};
    return fn(map, type, 2, const_cast<void *>(base), dims, strides, box, unit,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A matrix of `rows` rows (of i or o) and `k` contracted elements, 16-bit:
// k_major: row r at base + r * stride; else k index q at base + q * stride.
inline bool encode_16(CUtensorMap *map, bool bf16, const void *base, int64_t rows, int64_t k,
                      int64_t stride, bool k_major) {
    const auto type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return k_major ? encode_2d(map, type, base, k, rows, stride * 2, 64, kRows,
                               CU_TENSOR_MAP_SWIZZLE_128B)
                   : encode_2d(map, type, base, rows, k, stride * 2, 64, 64,
                               CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int KIND, bool BF16, bool A_MN, bool B_MN, class Epi>
inline int launch(const Args &args, const Epi &epi, int sms, cudaStream_t st) {
    const auto kernel = pair_kernel<KIND, BF16, A_MN, B_MN, Epi>;
    static unsigned long long done = 0;
    if (!allow_smem(kernel, smem_bytes<KIND>(), done)) return DRIFT_ECUDA;
    const int64_t total = (int64_t)args.m_tiles * args.n_tiles * args.splits;
    if (total > 0x7fffffff - sms) return DRIFT_EINVAL;  // the kernel steps past it once
    const int pairs = (int)(total < sms / 2 ? total : sms / 2);
    return launch_pdl(kernel, dim3(pairs * 2), kThreads, smem_bytes<KIND>(), st, 0, args, epi);
}

}  // namespace tc
}  // namespace drift
