// vdxs_i8_product.cu - the 8-bit unembedding product on the integer tensor cores:
//   logits[b][n] = scale[b] * w_scale[n] * sum_k q[b][k] * w[n][k].
//
// The vocabulary is the accumulator's row axis (128 rows a tile) and the batch its column
// axis (16..256 columns): a decode batch of any size then reads the weights once, as the
// A operand, and a tile's column leaves tensor memory with the 32 lanes of a warp on 32
// neighbouring vocabulary entries, so the logits go out as whole 128-byte lines without a
// stop in shared memory.
//
// Batches above 128 with sums of 2048 and more use pairs of CTAs: one product then spans both SMs of a pair (256 vocabulary
// entries, 128 to a CTA) and each CTA holds half of the batch columns' rows, which halves what
// the batch operand costs each SM in shared-memory fills.
// A small vocabulary has fewer tiles than the GPU has SMs, and one SM takes 0.3 us for each
// 128 bytes of a tile's rows: there a cluster of 2, 4 or 8 CTAs splits a tile's sums, and
// each adds up a share of the columns from all of them, in its shared memory.
//
// One persistent CTA per SM, ten warps: warp 0 copies 128-byte wide tiles of both operands
// into a ring of stages (TMA, 128-byte swizzle), warp 1 issues the products, warps 2 to 9
// scale and store one accumulator while the next tile is summed in the other one. Sums are
// exact 32-bit integers; the two scales are applied in fp32.
//
// What bounds it, on a B200 with 6456 GB/s and 1667 TFLOP/s in bf16 measured: to about 256
// rows the weights' bytes (batch 1 of 262144 x 1152 in 54-56 us, 0.84-0.87 of the copy rate; batch 64
// of 262144 x 2560 with fp32 logits in 118-121 us, 0.95-0.97). At batch 512 of the latter
// the products alone take 208 us, loads and stores alone 226, and together they run into the
// power limit: 280-296 us for the first tens of calls (2.4 POP/s), 325-331 once the SM clock has
// fallen (to about 1.16 GHz).
#include "vdxs_internal.h"
#include "../../include/vdx_sampler.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

namespace vdxs {
namespace {

constexpr int kEpiWarps = 8;         // two for each quarter of the accumulator's rows
constexpr int kThreadsP = 64 + 32 * kEpiWarps;
constexpr int kTileM = kI8TileM, kChunkK = kI8ChunkK, kMaxN = kI8MaxN;
constexpr int kMaxStages = 12;
constexpr int kStageBytesA = kTileM * kChunkK;
constexpr int kSmemBudget = 220 * 1024;
constexpr int32_t kErrTimeout = 3;   // the context's device error word: a bounded wait gave up

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Waits for a phase, at most about two seconds; `good` turns false when that gives up, and later
// waits try twice. The loop is closed to the compiler and no branch of the caller hangs on its
// outcome, so that a warp that waits together is known to stay together, which keeps the
// operands of what it issues in uniform registers.
#define VDXS_WAIT(TRY)                                                                        \
    asm volatile(                                                                             \
        "{\n .reg .pred p, q;\n .reg .u64 t, end;\n " TRY " p, [%1], %2;\n @p bra over;\n"     \
        " mov.u64 t, %%globaltimer;\n add.u64 end, t, %3;\n"                                  \
        "again:\n " TRY " p, [%1], %2;\n @p bra over;\n"                                      \
        " mov.u64 t, %%globaltimer;\n setp.lt.u64 q, t, end;\n @q bra again;\n"               \
        "over:\n selp.u32 %0, 1, 0, p;\n}"                                                    \
        : "=r"(done)                                                                          \
        : "r"(smem_addr(bar)), "r"(parity), "l"(limit)                                        \
        : "memory")
template <bool CLUSTER = false>
__device__ __forceinline__ void bar_wait(uint64_t* bar, uint32_t parity, bool& good) {
    uint32_t done;
    const uint64_t limit = good ? 2000000000ull : 0ull;
    if constexpr (CLUSTER) VDXS_WAIT("mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64");
    else VDXS_WAIT("mbarrier.try_wait.parity.shared::cta.b64");
    good = good && done != 0u;
}
#undef VDXS_WAIT
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
    return e;
}

// Instructions that one thread issues run with the whole warp converged and a predicate that
// holds in one lane (`one`): their operands then stay in uniform registers. Issued from a
// branch of a single lane, each product took 125 cycles of the issuing thread.
// `bar`: a barrier of this CTA, or with PAIR the address of one of the pair's first CTA.
template <bool PAIR>
__device__ __forceinline__ void copy_tile(uint32_t one, const CUtensorMap* map, uint32_t dst, int x, int y,
                                          uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.u32 q, %5, 0;\n"
            " @q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
            "[%1, {%2, %3}], [%4];\n}" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar), "r"(one)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.u32 q, %5, 0;\n"
            " @q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];\n}" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar), "r"(one)
            : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t one, uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.u32 q, %2, 0;\n @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(
            bar),
        "r"(bytes), "r"(one)
        : "memory");
}

// Shared-memory operand at an address: rows of 128 bytes, 128-byte swizzle, 8 rows (1024 bytes)
// to a group.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
            : "memory");
}
// With PAIR the barrier at the same place in both CTAs is arrived at.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t one, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n .reg .b16 both;\n mov.b16 both, 3;\n setp.ne.u32 q, %1, 0;\n"
            " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], "
            "both;\n}" ::"r"(bar),
            "r"(one)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
            " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
            "r"(one)
            : "memory");
}
// The address of this CTA's `addr` in a CTA of the cluster.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void load16(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
// The registers of a load pass through the wait, so that no use of them moves before it.
__device__ __forceinline__ void wait16(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::
                     "memory");
}

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

struct ProductParams {
    int in_dim, out_dim, batch, n, n_tiles, stages, columns, split;
    int64_t tiles;  // vocabulary tiles (of two CTAs, in pairs) * n_tiles
    const float *w_scale, *scale;
    void* logits;
    int64_t stride;
    int32_t* err;
};

// 16 columns of a thread's row to the logits; `columns` of them are in the batch.
template <typename O>
__device__ __forceinline__ void store16(O* o, int64_t stride, const uint32_t* v, const float* scales, float ws,
                                        int columns, bool have) {
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(scales + j);
        x[j] = f.x, x[j + 1] = f.y, x[j + 2] = f.z, x[j + 3] = f.w;
    }
    if (have && columns >= 16) {
#pragma unroll
        for (int j = 0; j < 16; ++j, o += stride) put(o, __fmul_rn(__fmul_rn((float)(int)v[j], ws), x[j]));
    } else if (have) {
#pragma unroll
        for (int j = 0; j < 16; ++j, o += stride)
            if (j < columns) put(o, __fmul_rn(__fmul_rn((float)(int)v[j], ws), x[j]));
    }
}

constexpr int kSingle = I8ProductForm::kSingle, kPair = I8ProductForm::kPair, kSplit = I8ProductForm::kSplit;

template <typename O, int MODE>
__global__ void __launch_bounds__(kThreadsP, 1)
    unembed_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q,
                      const ProductParams p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base;
    __shared__ __align__(16) float scales[2][kMaxN];
    unsigned char* stages = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    // (A shuffled value is one for the whole warp to the compiler too.)
    const int warp = __shfl_sync(0xFFFFFFFFu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    constexpr bool PAIR = MODE == kPair, SPLIT = MODE == kSplit;
    constexpr int kCtas = PAIR ? 2 : 1;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;  // in the pair
    const int part = SPLIT ? (int)(blockIdx.x % p.split) : 0;
    const int64_t first = SPLIT ? blockIdx.x / p.split : blockIdx.x / kCtas;      // of this CTA's tiles
    const int64_t step = SPLIT ? gridDim.x / p.split : gridDim.x / kCtas;         // (with SPLIT it has one)
    const int q_rows = p.n / kCtas;                     // batch rows that this CTA holds
    const int stage_bytes = kStageBytesA + q_rows * kChunkK;
    const int chunks = (p.in_dim + kChunkK - 1) / kChunkK;
    const int chunk0 = SPLIT ? (int)((int64_t)chunks * part / p.split) : 0;
    const int chunk1 = SPLIT ? (int)((int64_t)chunks * (part + 1) / p.split) : chunks;
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) bar_init(&full[i], 1), bar_init(&empty[i], 1);
        for (int i = 0; i < 2; ++i) bar_init(&acc_full[i], 1), bar_init(&acc_empty[i], kEpiWarps * kCtas);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                         "r"(p.columns)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                         "r"(p.columns)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base;

    bool good = true;
    if (warp == 0) {
        const uint32_t one = elect_one();
        const uint32_t base = smem_addr(stages), mine0 = smem_addr(full), full0 = PAIR ? in_cta(mine0, 0) : mine0;
        int s = 0, issued = 0;
        uint32_t phase = 0;
        for (int64_t t = first; t < p.tiles; t += step) {
            const int m = (int)(t / p.n_tiles), n = (int)(t - (int64_t)m * p.n_tiles);
            for (int c = chunk0; c < chunk1; ++c) {
                bar_wait(&empty[s], phase ^ 1, good);
                if (!good) break;
                // A pair's stages are counted together by its first CTA.
                const uint32_t a = base + s * stage_bytes, bar = full0 + 8 * s;
                if (rank == 0) bar_expect(one, mine0 + 8 * s, kCtas * stage_bytes);
                copy_tile<PAIR>(one, &map_w, a, c * kChunkK, (m * kCtas + rank) * kTileM, bar);
                copy_tile<PAIR>(one, &map_q, a + kStageBytesA, c * kChunkK, n * p.n + rank * q_rows, bar);
                issued = min(issued + 1, p.stages);
                if (++s == p.stages) s = 0, phase ^= 1;
            }
            if (!good) break;
        }
        // The copies in flight land before the CTA (the pair) may end: the products' warp, which waits
        // for them too, may have given up.
        if (rank == 0) {
            bool landed = true;
            for (; issued > 0; --issued) {
                if (--s < 0) s = p.stages - 1, phase ^= 1;
                bar_wait(&full[s], phase, landed);
            }
            good = good && landed;
        }
    } else if (warp == 1 && rank == 0) {
        // D: 32-bit integers; A, B: signed 8 bits, K-major.
        const uint32_t idesc =
            2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(p.n >> 3) << 17 | (uint32_t)(kCtas * kTileM >> 4) << 24;
        uint32_t one = elect_one();
        const uint32_t empty0 = smem_addr(empty), base = smem_addr(stages);
        // What lies behind in_dim is zero in shared memory; whole steps of it are left out.
        const int last = (p.in_dim - (chunks - 1) * kChunkK + 31) / 32;
        int s = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        for (int64_t t = first; t < p.tiles; t += step) {
            bar_wait<PAIR>(&acc_empty[acc], acc_phase ^ 1, good);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + acc * (p.columns >> 1);
            for (int c = chunk0; c < chunk1; ++c) {
                bar_wait(&full[s], phase, good);
                if (!good) one = 0;  // nothing more is issued
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t a = operand(base + s * stage_bytes);
                const uint64_t b = operand(base + s * stage_bytes + kStageBytesA);
                if (c + 1 < chunks || last == 4) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_i8<PAIR>(one, d, a + 2 * k, b + 2 * k, idesc, (uint32_t)((c - chunk0) | k));
                } else {
                    for (int k = 0; k < last; ++k) mma_i8<PAIR>(one, d, a + 2 * k, b + 2 * k, idesc, (uint32_t)((c - chunk0) | k));
                }
                mma_commit<PAIR>(one, empty0 + 8 * s);
                if (++s == p.stages) s = 0, phase ^= 1;
            }
            mma_commit<PAIR>(one, smem_addr(&acc_full[acc]));
            if (++acc == 2) acc = 0, acc_phase ^= 1;
        }
        // And the last products are in before tensor memory is freed, whether or not the epilogue gave up.
        if (first < p.tiles) bar_wait(&acc_full[acc ^ 1], acc == 0 ? acc_phase ^ 1 : acc_phase, good);
    } else if (warp >= 2) {
        const int quad = warp & 3;             // the tensor memory lanes that this warp may read
        const int half = (warp - 2) >> 2;      // even or odd groups of 16 columns
        const int thread = threadIdx.x - 64;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int64_t t = first; t < p.tiles; t += step) {
            const int m = (int)(t / p.n_tiles), n = (int)(t - (int64_t)m * p.n_tiles);
            const int64_t row = ((int64_t)m * kCtas + rank) * kTileM + quad * 32 + lane;
            const bool have = row < p.out_dim;
            const float ws = have ? __ldg(p.w_scale + row) : 0.0f;
            const int b0 = n * p.n, columns = min(p.n, p.batch - b0);
            // (This buffer was read two tiles ago, before the barrier of the last tile.)
            if (thread < columns) scales[acc][thread] = __ldg(p.scale + b0 + thread);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
            // Should the wait give up, the warps still meet at the barriers to come.
            bar_wait(&acc_full[acc], acc_phase, good);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = tmem + acc * (p.columns >> 1) + ((uint32_t)quad * 32 << 16);
            O* out = static_cast<O*>(p.logits) + (b0 + 16 * half) * p.stride + row;
            for (int c = 16 * half; !SPLIT && c < columns; c += 32, out += 32 * p.stride) {
                uint32_t v[16];
                load16(src + c, v);
                wait16(v);
                store16(out, p.stride, v, &scales[acc][c], ws, columns - c, have);
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) {
                if constexpr (PAIR)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                     in_cta(smem_addr(&acc_empty[acc]), 0))
                                 : "memory");
                else
                    bar_arrive(&acc_empty[acc]);
            }
            if (++acc == 2) acc = 0, acc_phase ^= 1;
        }
    }
    if constexpr (SPLIT) {
        // All parts of the tile are summed and every CTA's ring is idle: group g of 16 columns goes to
        // CTA g mod split, [part][its group][column][row] in the ring's room.
        __syncwarp();
        cluster_sync();
        const int quad = warp & 3, half = (warp - 2) >> 2, groups = p.n / 16;
        const int own = (groups + p.split - 1) / p.split;
        const uint32_t room = smem_addr(stages);
        if (warp >= 2) {
            for (int g = half; g < groups; g += 2) {
                uint32_t v[16];
                load16(tmem + ((uint32_t)quad * 32 << 16) + 16 * g, v);
                wait16(v);
                const uint32_t to = in_cta(room, g % p.split) +
                                    ((part * own + g / p.split) * 16 * kTileM + quad * 32 + lane) * 4;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + j * kTileM * 4), "r"(v[j]) : "memory");
            }
        }
        __syncwarp();
        cluster_sync();
        if (warp >= 2 && first < p.tiles) {
            const int m = (int)(first / p.n_tiles), n = (int)(first - (int64_t)m * p.n_tiles);
            const int64_t row = (int64_t)m * kTileM + quad * 32 + lane;
            const int b0 = n * p.n;
            const bool have = row < p.out_dim;
            const float ws = have ? __ldg(p.w_scale + row) : 0.0f;
            for (int i = half; i < own && i * p.split + part < groups; i += 2) {
                const int c = 16 * (i * p.split + part);
                const uint32_t* in = reinterpret_cast<const uint32_t*>(stages) + i * 16 * kTileM + quad * 32 + lane;
                uint32_t v[16] = {};
                for (int r = 0; r < p.split; ++r, in += own * 16 * kTileM)
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] += in[j * kTileM];
                store16(static_cast<O*>(p.logits) + (int64_t)(b0 + c) * p.stride + row, p.stride, v, &scales[0][c], ws,
                        p.batch - b0 - c, have);
            }
        }
    }
    if (!good) *p.err = kErrTimeout;
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 2) {
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.columns));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.columns));
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// Bytes [rows][pitch] of which `width` are used; boxes of 128 bytes by `box_rows` rows.
cudaError_t make_map(CUtensorMap* map, const void* base, int width, int rows, int64_t pitch, int box_rows) {
    const EncodeTiled encode = encoder();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {kChunkK, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace

template <typename O, int MODE>
static cudaError_t launch_product(const CUtensorMap& map_w, const CUtensorMap& map_q, const ProductParams& p, int smem,
                                  int sm_count, cudaStream_t stream) {
    static SmemLimit limit;
    cudaError_t e = limit.raise(unembed_i8_kernel<O, MODE>, kSmemBudget);
    if (e != cudaSuccess) return e;
    const int ctas = MODE == kPair ? 2 : MODE == kSplit ? p.split : 1;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = (unsigned)ctas, cluster.val.clusterDim.y = 1, cluster.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((MODE == kSplit ? p.tiles : std::min<int64_t>(p.tiles, sm_count / ctas)) * ctas));
    cfg.blockDim = dim3(kThreadsP);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cfg.attrs = &cluster;
    cfg.numAttrs = MODE == kSingle ? 0 : 1;
    return cudaLaunchKernelEx(&cfg, unembed_i8_kernel<O, MODE>, map_w, map_q, p);
}

template <typename O>
static cudaError_t launch_mode(int mode, const CUtensorMap& map_w, const CUtensorMap& map_q, const ProductParams& p,
                               int smem, int sm_count, cudaStream_t stream) {
    if (mode == kPair) return launch_product<O, kPair>(map_w, map_q, p, smem, sm_count, stream);
    if (mode == kSplit) return launch_product<O, kSplit>(map_w, map_q, p, smem, sm_count, stream);
    return launch_product<O, kSingle>(map_w, map_q, p, smem, sm_count, stream);
}

cudaError_t unembed_i8(const I8Matrix& w, const int8_t* q, int64_t q_stride, const float* scale, int batch,
                       void* logits, int dtype, int64_t logits_stride, int32_t* err, int sm_count, cudaStream_t stream,
                       int* launches) {
    ProductParams p{};
    p.in_dim = w.in_dim;
    p.out_dim = w.out_dim;
    p.batch = batch;
    const I8ProductForm form = i8_product_form(batch, w.in_dim, w.out_dim, sm_count);
    const bool pair = form.mode == kPair;
    const int ctas = pair ? 2 : 1;
    p.n_tiles = form.n_tiles;
    p.n = form.n;
    p.split = form.split;
    p.columns = 32;
    while (p.columns < 2 * p.n) p.columns *= 2;
    const int stage_bytes = kStageBytesA + p.n / ctas * kChunkK;
    p.stages = std::min(kMaxStages, (kSmemBudget - 1024) / stage_bytes);
    p.tiles = (int64_t)((w.out_dim + ctas * kTileM - 1) / (ctas * kTileM)) * p.n_tiles;
    p.w_scale = w.scale;
    p.scale = scale;
    p.logits = logits;
    p.stride = logits_stride;
    p.err = err;
    CUtensorMap map_w, map_q;
    static_assert(sizeof(map_w) == sizeof(w.map), "tensor map size");
    memcpy(&map_w, w.map, sizeof(map_w));
    cudaError_t e = make_map(&map_q, q, w.in_dim, batch, q_stride, p.n / ctas);
    if (e != cudaSuccess) return e;
    const int smem = p.stages * stage_bytes + 1024;
    e = dtype == VDXS_DTYPE_BF16 ? launch_mode<__nv_bfloat16>(form.mode, map_w, map_q, p, smem, sm_count, stream)
                                 : launch_mode<float>(form.mode, map_w, map_q, p, smem, sm_count, stream);
    if (e != cudaSuccess) return e;
    ++*launches;
    return cudaSuccess;
}

cudaError_t map_weights_i8(I8Matrix& w) {
    CUtensorMap map;
    const cudaError_t e = make_map(&map, w.q, w.in_dim, w.out_dim, w.pitch, kTileM);
    if (e == cudaSuccess) memcpy(w.map, &map, sizeof(map));
    return e;
}

}  // namespace vdxs
