// vdxs_beam.cu - beam search: the selection over beams and vocabulary, and the reordering of
// the search's rows by the selected parents (rings and the caller's caches).
//
// One pass over the logits. A row is cut into chunks, a CTA takes one: each thread keeps a
// running maximum and a sum of exponentials relative to it, and the CTA keeps a list of the
// elements that can still be among its K = beams largest. The K-th largest of the threads'
// maxima over the chunk's first tile is a lower bound of the chunk's K-th largest element,
// so from then on only elements above it enter the list. The last CTA of a row merges the
// row's lists and sums, the last row of a prompt merges the beams' offers; both are found
// by counters that reset themselves.
#include "vdxs_internal.h"
#include "../../include/vdx_sampler.h"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace vdxs {
namespace {

constexpr unsigned FULLMASK = 0xFFFFFFFFu;
constexpr int kBThreads = 256;
constexpr int kPer = 16;                    // elements of a tile per thread
constexpr int kTile = kBThreads * kPer;     // 4096
constexpr int kListLimit = 512;             // entries before a list is cut back to K
constexpr int kListCap = kTile + kListLimit;  // a tile may add every element it has
constexpr float kLog2e = 1.4426950408889634f;
typedef unsigned long long u64;

// Order-preserving key: larger value first, then the lower token. Never 0.
__device__ __forceinline__ u64 make_key(float v, int token) {
    uint32_t u = __float_as_uint(v + 0.0f);  // -0 is +0
    u ^= (u >> 31) ? 0xFFFFFFFFu : 0x80000000u;
    return ((u64)u << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float key_value(u64 k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u >> 31) ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int key_token(u64 k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct SelectShared {
    u64 list[kListCap];
    u64 best[VDXS_BEAM_MAX_BEAMS];
    u64 maxima[kBThreads];
    u64 bound;
    int count;
    int flag;
    float wm[kBThreads / 32];
    double ws[kBThreads / 32];
};

// The K-th largest of one value per thread (ties by thread), in sh.bound.
__device__ __forceinline__ void block_bound(SelectShared& sh, u64 mine, int K) {
    const int tid = threadIdx.x;
    sh.maxima[tid] = mine;
    __syncthreads();
    int above = 0;
    for (int j = 0; j < kBThreads; ++j) {
        const u64 o = sh.maxima[j];
        above += o > mine || (o == mine && j < tid);
    }
    if (above == K - 1) sh.bound = mine;
    __syncthreads();
}

// Cuts list[0..count) to its K largest, in order, in best[]; the rest of best is 0.
// While the list is long, each thread takes the maximum of its share: the K-th largest of
// those is a lower bound of the K-th largest entry, and at most a quarter plus K remain.
__device__ void block_select(SelectShared& sh, int K) {
    const int tid = threadIdx.x;
    __syncthreads();
    int n = sh.count;
    while (n > kListLimit) {
        u64 mx = 0;
        for (int i = tid; i < n; i += kBThreads) mx = max(mx, sh.list[i]);
        block_bound(sh, mx, K);
        const u64 bound = sh.bound;
        u64 mine[kListCap / kBThreads];
        int m = 0;
#pragma unroll
        for (int j = 0; j < kListCap / kBThreads; ++j) {
            const int i = tid + j * kBThreads;
            mine[j] = i < n && sh.list[i] >= bound ? sh.list[i] : 0;
            m += mine[j] != 0;
        }
        if (tid == 0) sh.count = 0;
        __syncthreads();
        int at = m ? atomicAdd(&sh.count, m) : 0;
#pragma unroll
        for (int j = 0; j < kListCap / kBThreads; ++j)
            if (mine[j]) sh.list[at++] = mine[j];
        __syncthreads();
        n = sh.count;
    }
    if (tid < K) sh.best[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kBThreads) {
        const u64 mine = sh.list[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += sh.list[j] > mine;
        if (above < K) sh.best[above] = mine;
    }
    __syncthreads();
}

template <typename T>
struct Vec;  // 16 bytes of logits
template <>
struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const float* p, float* v) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(p));
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    }
    static __device__ __forceinline__ float one(const float* p) { return __ldg(p); }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* v) {
        const uint4 f = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};

// x > 0: x / p, else x * p, once for every time the ring holds the token (Sampler.pas:285-303).
__device__ float penalised(float x, int token, const int32_t* ring, int n, float p) {
    for (int i = 0; i < n; ++i)
        if (ring[i] == token) x = x > 0.0f ? __fdiv_rn(x, p) : __fmul_rn(x, p);
    return x;
}

// The prompt's offers: each row's best[] is in order, so K times the best head is taken.
// Lane l holds the heads of beams l and l + 32. One warp.
__device__ void select_prompt(const BeamArgs& p, int prompt) {
    __shared__ double s_score[VDXS_BEAM_MAX_BEAMS], s_size[VDXS_BEAM_MAX_BEAMS];
    __shared__ int s_len[VDXS_BEAM_MAX_BEAMS], s_done[VDXS_BEAM_MAX_BEAMS], s_old[VDXS_BEAM_MAX_BEAMS];
    __shared__ double o_score[VDXS_BEAM_MAX_BEAMS];
    __shared__ int o_token[VDXS_BEAM_MAX_BEAMS], o_parent[VDXS_BEAM_MAX_BEAMS];
    const int lane = threadIdx.x & 31, K = p.beams;
    const int64_t row0 = (int64_t)prompt * K;
    for (int b = lane; b < K; b += 32) {
        const int64_t r = row0 + b;
        const int done = p.finished_in[r] != 0, len = p.lengths_in[r];
        s_score[b] = p.scores_in[r];
        s_done[b] = done;
        s_old[b] = len;
        s_len[b] = done ? len : len + 1;
        s_size[b] = pow((double)max(s_len[b], 1), p.alpha);
    }
    __syncwarp();
    int at[2] = {0, 0};
    double score[2], rank[2];
    int token[2];
    auto head = [&](int j) {
        const int b = lane + 32 * j;
        rank[j] = -INFINITY;
        if (b >= K || at[j] >= K) return;
        const double before = s_score[b];
        if (s_done[b]) {
            if (at[j] > 0) return;
            score[j] = before;
            token[j] = p.pad;
        } else {
            const u64 k = __ldcg(p.ws.best + (row0 + b) * K + at[j]);
            if (k == 0) return;
            score[j] = before + ((double)key_value(k) - __ldcg(p.ws.lse + row0 + b));
            token[j] = key_token(k);
        }
        if (score[j] > -INFINITY) rank[j] = score[j] / s_size[b];
    };
    head(0);
    head(1);
    for (int k = 0; k < K; ++k) {
        double best = rank[0];
        int from = lane;
        if (rank[1] > best) best = rank[1], from = lane + 32;
        for (int s = 16; s > 0; s >>= 1) {
            const double o = __shfl_xor_sync(FULLMASK, best, s);
            const int f = __shfl_xor_sync(FULLMASK, from, s);
            if (o > best || (o == best && f < from)) best = o, from = f;
        }
        if (!(best > -INFINITY)) {
            if (lane == 0) o_parent[k] = -1;
            continue;
        }
        if ((from & 31) == lane) {
            const int j = from >> 5;
            o_parent[k] = from;
            o_token[k] = j ? token[1] : token[0];
            o_score[k] = j ? score[1] : score[0];
            if (j) ++at[1], head(1);
            else ++at[0], head(0);
        }
    }
    __syncwarp();
    for (int k = lane; k < K; k += 32) {
        const int64_t r = row0 + k;
        const int b = o_parent[k];
        const bool none = b < 0, fresh = !none && !s_done[b];
        const int tok = none ? p.pad : o_token[k];
        bool stop = false;
        if (fresh)
            for (int i = 0; i < p.n_stop; ++i) stop |= p.stop_ids[i] == tok;
        p.tokens[r] = tok;
        p.parents[r] = none ? k : b;
        p.scores[r] = none ? -INFINITY : (float)o_score[k];
        p.lengths[r] = none ? s_old[k] : s_len[b];
        p.finished[r] = none ? 0 : fresh ? stop : 1;
        p.ws.push[r] = fresh;
    }
}

template <typename T>
__global__ void __launch_bounds__(kBThreads) beam_select_kernel(BeamArgs p) {
    extern __shared__ __align__(16) unsigned char smem[];
    SelectShared& sh = *reinterpret_cast<SelectShared*>(smem);
    uint32_t* marks = reinterpret_cast<uint32_t*>(smem + sizeof(SelectShared));
    constexpr int VN = Vec<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.beams;
    const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks;
    const bool live = p.finished_in[row] == 0 && p.scores_in[row] > -INFINITY;
    if (live) {
        // Positions count from the 16-byte boundary at or below the row's first element.
        const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
        const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
        const T* base = x - off;
        const int64_t lo = off, hi = (int64_t)p.vocab + off;
        const int64_t c0 = (int64_t)c * p.chunk, c1 = min(c0 + p.chunk, hi);
        const bool pen = p.window > 0 && p.penalty != 1.0f;
        const int32_t* ring = pen ? p.hist_in + (int64_t)row * p.window : nullptr;
        const int held = pen ? min(max(p.count_in[row], 0), p.window) : 0;
        if (pen) {
            for (int i = tid; i < p.chunk / 32; i += kBThreads) marks[i] = 0;
            __syncthreads();
            for (int i = tid; i < held; i += kBThreads) {
                const int64_t v = (int64_t)ring[i] + off;
                if (ring[i] >= 0 && ring[i] < p.vocab && v >= c0 && v < c1)
                    atomicOr(&marks[(v - c0) >> 5], 1u << ((v - c0) & 31));
            }
        }
        if (tid == 0) sh.count = 0;
        __syncthreads();
        float m = -FLT_MAX, s = 0.0f, tau = -INFINITY;
        bool first = true;
        for (int64_t t0 = c0; t0 < c1; t0 += kTile) {
            float v[kPer];
#pragma unroll
            for (int u = 0; u < kPer / VN; ++u) {
                const int64_t e = t0 + (int64_t)(u * kBThreads + tid) * VN;
                if (e >= lo && e + VN <= c1) {
                    Vec<T>::load(base + e, v + u * VN);
                } else {
#pragma unroll
                    for (int i = 0; i < VN; ++i)
                        v[u * VN + i] = e + i >= lo && e + i < c1 ? Vec<T>::one(base + e + i) : -INFINITY;
                }
                if (pen && e < c1) {
                    const uint32_t w = (marks[(e - c0) >> 5] >> ((e - c0) & 31)) & ((1u << VN) - 1);
                    if (w) {
#pragma unroll
                        for (int i = 0; i < VN; ++i)
                            if (w >> i & 1)
                                v[u * VN + i] = penalised(v[u * VN + i], (int)(e + i - off), ring, held, p.penalty);
                    }
                }
            }
            float top = v[0];
#pragma unroll
            for (int i = 1; i < kPer; ++i) top = fmaxf(top, v[i]);
            if (top > m) {
                s *= ex2((m - top) * kLog2e);
                m = top;
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) s += ex2((v[i] - m) * kLog2e);
            if (first) {
                block_bound(sh, make_key(top, tid), K);
                tau = key_value(sh.bound);
            }
            if (first ? top >= tau : top > tau) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    if ((first ? v[i] >= tau : v[i] > tau) && v[i] > -INFINITY) {
                        const int64_t e = t0 + (int64_t)((i / VN) * kBThreads + tid) * VN + i % VN;
                        sh.list[atomicAdd(&sh.count, 1)] = make_key(v[i], (int)(e - off));
                    }
                }
            }
            first = false;
            __syncthreads();
            if (sh.count > kListLimit && t0 + kTile < c1) {
                block_select(sh, K);
                if (tid < K) sh.list[tid] = sh.best[tid];
                if (tid == 0) sh.count = K;
                tau = key_value(sh.best[K - 1]);
            }
            __syncthreads();
        }
        block_select(sh, K);
        const int64_t slot = (int64_t)row * p.chunks + c;
        if (tid < K) p.ws.cand[slot * K + tid] = sh.best[tid];
        float wm = m;
        for (int d = 16; d > 0; d >>= 1) wm = fmaxf(wm, __shfl_xor_sync(FULLMASK, wm, d));
        double ws = (double)s * ex2((m - wm) * kLog2e);
        for (int d = 16; d > 0; d >>= 1) ws += __shfl_xor_sync(FULLMASK, ws, d);
        if (lane == 0) sh.wm[warp] = wm, sh.ws[warp] = ws;
        __syncthreads();
        if (tid == 0) {
            float M = sh.wm[0];
            for (int w = 1; w < kBThreads / 32; ++w) M = fmaxf(M, sh.wm[w]);
            double S = 0.0;
            for (int w = 0; w < kBThreads / 32; ++w) S += sh.ws[w] * ex2((sh.wm[w] - M) * kLog2e);
            p.ws.part[2 * slot] = M;
            p.ws.part[2 * slot + 1] = S;
        }
    }
    // The row's last CTA merges its chunks.
    __threadfence();
    __syncthreads();
    if (tid == 0) sh.flag = atomicAdd(&p.ws.row_done[row], 1u) == (uint32_t)p.chunks - 1;
    __syncthreads();
    if (!sh.flag) return;
    __threadfence();
    if (live) {
        const int n = p.chunks * K;
        if (tid == 0) sh.count = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kBThreads) {
            const u64 k = __ldcg(p.ws.cand + (int64_t)row * n + i);
            if (k) sh.list[atomicAdd(&sh.count, 1)] = k;
        }
        block_select(sh, K);
        if (warp == 0) {
            double M = -INFINITY, S = 0.0;
            const double* part = p.ws.part + (int64_t)row * p.chunks * 2;
            for (int i = lane; i < p.chunks; i += 32) M = fmax(M, __ldcg(part + 2 * i));
            for (int d = 16; d > 0; d >>= 1) M = fmax(M, __shfl_xor_sync(FULLMASK, M, d));
            for (int i = lane; i < p.chunks; i += 32) S += __ldcg(part + 2 * i + 1) * exp(__ldcg(part + 2 * i) - M);
            for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(FULLMASK, S, d);
            if (lane == 0) p.ws.lse[row] = M + log(S);
            // A NaN sum (a NaN or +infinity in the row) offers nothing.
            for (int k = lane; k < K; k += 32) p.ws.best[(int64_t)row * K + k] = S > 0.0 ? sh.best[k] : 0;
        }
    }
    __threadfence();
    __syncthreads();
    const int prompt = row / K;
    if (tid == 0) {
        p.ws.row_done[row] = 0;
        sh.flag = atomicAdd(&p.ws.prompt_done[prompt], 1u) == (uint32_t)K - 1;
    }
    __syncthreads();
    if (!sh.flag || warp != 0) return;
    __threadfence();
    select_prompt(p, prompt);
    if (lane == 0) p.ws.prompt_done[prompt] = 0;
}

constexpr int kRThreads = 128;
constexpr int kMaxCaches = 32;  // per launch
struct ReorderParams {
    int batch, beams, window, ring_blocks, n;
    const int32_t *parents, *tokens, *push;
    const int32_t *hist_in, *pos_in, *count_in;
    int32_t *hist, *pos, *count;
    struct {
        BeamCacheArgs a;
        int64_t seg_words, words;  // words of `shift` bytes
        int shift;                 // log2 of the word's bytes
        int64_t blocks;            // per prompt
        int64_t end;               // first block behind this cache
    } c[kMaxCaches];
};

// A thread owns one word of every row of a prompt: it reads the parents' words, then
// writes, so a cache may be moved in place without a second buffer or a barrier.
template <typename W>
__device__ void move_words(const ReorderParams& p, int i, int prompt, int64_t first, const int* parent, W* stage) {
    const auto& c = p.c[i];
    const bool same = c.a.src == c.a.dst;
    const int64_t w = first + threadIdx.x;
    if (w >= c.words) return;
    const int64_t seg = w / c.seg_words, in = (w - seg * c.seg_words) * (int64_t)sizeof(W);
    const unsigned char* src = c.a.src + (int64_t)prompt * p.beams * c.a.src_row + seg * c.a.src_segment + in;
    unsigned char* dst = c.a.dst + (int64_t)prompt * p.beams * c.a.dst_row + seg * c.a.dst_segment + in;
    for (int k = 0; k < p.beams; ++k)
        if (!same || parent[k] != k)
            stage[k * kRThreads + threadIdx.x] = *reinterpret_cast<const W*>(src + parent[k] * c.a.src_row);
    for (int k = 0; k < p.beams; ++k)
        if (!same || parent[k] != k) *reinterpret_cast<W*>(dst + k * c.a.dst_row) = stage[k * kRThreads + threadIdx.x];
}

__global__ void __launch_bounds__(kRThreads) beam_reorder_kernel(const __grid_constant__ ReorderParams p) {
    extern __shared__ __align__(16) unsigned char stage[];  // [beams][kRThreads] words
    __shared__ int parent[VDXS_BEAM_MAX_BEAMS], pos[VDXS_BEAM_MAX_BEAMS], count[VDXS_BEAM_MAX_BEAMS];
    const int K = p.beams;
    int64_t block = blockIdx.x;
    const bool ring = block < p.ring_blocks;
    int i = 0;
    int prompt;
    int64_t first = 0;
    if (ring) {
        prompt = (int)block;
    } else {
        block -= p.ring_blocks;
        while (block >= p.c[i].end) ++i;
        if (i > 0) block -= p.c[i - 1].end;
        prompt = (int)(block / p.c[i].blocks);
        first = (block - prompt * p.c[i].blocks) * kRThreads;
    }
    const int64_t row0 = (int64_t)prompt * K;
    for (int k = threadIdx.x; k < K; k += kRThreads) {
        const int b = p.parents[row0 + k];
        parent[k] = b >= 0 && b < K ? b : k;
    }
    __syncthreads();
    if (!ring) {
        switch (p.c[i].shift) {
            case 4: move_words(p, i, prompt, first, parent, reinterpret_cast<uint4*>(stage)); break;
            case 3: move_words(p, i, prompt, first, parent, reinterpret_cast<uint2*>(stage)); break;
            case 2: move_words(p, i, prompt, first, parent, reinterpret_cast<uint32_t*>(stage)); break;
            case 1: move_words(p, i, prompt, first, parent, reinterpret_cast<uint16_t*>(stage)); break;
            default: move_words(p, i, prompt, first, parent, reinterpret_cast<uint8_t*>(stage));
        }
        return;
    }
    // The rings, and AddToHistory (Sampler.pas:530-539) of the new tokens. The position and
    // the count of every parent are read before any is written.
    const int W = p.window;
    for (int k = threadIdx.x; k < K; k += kRThreads) {
        int at = p.pos_in[row0 + parent[k]] % W;
        pos[k] = at < 0 ? at + W : at;
        count[k] = p.count_in[row0 + parent[k]];
    }
    __syncthreads();
    int32_t* mine = reinterpret_cast<int32_t*>(stage) + threadIdx.x;
    for (int j = threadIdx.x; j < W; j += kRThreads) {
        for (int k = 0; k < K; ++k) mine[k * kRThreads] = p.hist_in[(row0 + parent[k]) * W + j];
        for (int k = 0; k < K; ++k)
            p.hist[(row0 + k) * W + j] = p.push[row0 + k] && pos[k] == j ? p.tokens[row0 + k] : mine[k * kRThreads];
    }
    for (int k = threadIdx.x; k < K; k += kRThreads) {
        const bool push = p.push[row0 + k] != 0;
        p.pos[row0 + k] = push ? (pos[k] + 1) % W : pos[k];
        p.count[row0 + k] = push && count[k] < W ? max(count[k], 0) + 1 : count[k];
    }
}

}  // namespace

void beam_plan(int rows, int vocab, int sm_count, int* chunks, int* chunk) {
    // A position is counted from a 16-byte boundary, so up to 7 lie before the row.
    const int64_t span = (int64_t)vocab + 7;
    const int64_t tiles = (span + kTile - 1) / kTile;
    // Two CTAs for each SM's four places at least, and at most kBeamMaxChunks lists to merge.
    int64_t want = std::min<int64_t>(kBeamMaxChunks, std::max<int64_t>(1, ((int64_t)sm_count * 8 + rows - 1) / rows));
    want = std::min(want, tiles);
    const int64_t per = (tiles + want - 1) / want;
    *chunk = (int)(per * kTile);
    *chunks = (int)((tiles + per - 1) / per);
}

cudaError_t beam_select(const BeamArgs& a, cudaStream_t stream) {
    const bool pen = a.window > 0 && a.penalty != 1.0f;
    const size_t smem = sizeof(SelectShared) + (pen ? (size_t)a.chunk / 8 : 0);
    const int grid = a.batch * a.beams * a.chunks;
    void (*kern)(BeamArgs) =
        a.dtype == VDXS_DTYPE_BF16 ? beam_select_kernel<__nv_bfloat16> : beam_select_kernel<float>;
    static SmemLimit limit[2];
    cudaError_t e = limit[a.dtype == VDXS_DTYPE_BF16].raise(kern, smem);
    if (e != cudaSuccess) return e;
    kern<<<grid, kBThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t beam_reorder(const BeamArgs& a, bool rings, const BeamCacheArgs* caches, int n_caches, cudaStream_t stream,
                         int* launches) {
    const size_t smem = (size_t)a.beams * kRThreads * 16;
    static SmemLimit limit;
    cudaError_t e = limit.raise(beam_reorder_kernel, smem);
    if (e != cudaSuccess) return e;
    int at = 0;
    while (rings || at < n_caches) {
        ReorderParams p{};
        p.batch = a.batch;
        p.beams = a.beams;
        p.window = a.window;
        p.parents = a.parents;
        if (rings) {
            p.ring_blocks = a.batch;
            p.tokens = a.tokens;
            p.push = a.ws.push;
            p.hist_in = a.hist_in, p.pos_in = a.pos_in, p.count_in = a.count_in;
            p.hist = a.hist, p.pos = a.pos, p.count = a.count;
            rings = false;
        }
        int64_t end = 0;
        for (; at < n_caches && p.n < kMaxCaches; ++at) {
            const BeamCacheArgs& c = caches[at];
            if (c.segment_bytes <= 0 || c.segments <= 0) continue;
            auto& d = p.c[p.n];
            d.a = c;
            // The widest word that every address and length is a multiple of.
            const uint64_t all = (uint64_t)(uintptr_t)c.src | (uint64_t)(uintptr_t)c.dst | (uint64_t)c.src_row |
                                 (uint64_t)c.dst_row | (uint64_t)c.src_segment | (uint64_t)c.dst_segment |
                                 (uint64_t)c.segment_bytes | 16u;
            while (!(all >> d.shift & 1)) ++d.shift;
            d.seg_words = c.segment_bytes >> d.shift;
            d.words = d.seg_words * c.segments;
            d.blocks = (d.words + kRThreads - 1) / kRThreads;
            end += d.blocks * a.batch;
            d.end = end;
            ++p.n;
        }
        const int64_t grid = p.ring_blocks + end;
        if (grid == 0) continue;
        if (grid > INT32_MAX) return cudaErrorInvalidValue;
        beam_reorder_kernel<<<(unsigned)grid, kRThreads, smem, stream>>>(p);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        ++*launches;
    }
    return cudaSuccess;
}

}  // namespace vdxs
