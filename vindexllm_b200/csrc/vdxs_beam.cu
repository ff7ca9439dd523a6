// vdxs_beam.cu - beam search: the selection over beams and vocabulary, and the reordering of
// the search's rows by the selected parents (rings and the caller's caches).
//
// One pass over the logits. A row is cut into chunks, a CTA takes one: each thread keeps a
// running maximum with a sum of exponentials relative to it, and notes the maximum of its 16
// elements of every tile. The K-th largest of disjoint groups' maxima is a lower bound of the
// chunk's K-th largest element (K = beams), and only the groups whose maximum reaches the
// bound, hardly more than K of them, are read again for their elements. The last CTA of a prompt
// merges the lists and sums of its rows, and moves its rings where nothing else moves; where the
// lists are too many for one CTA, the last CTA of each row merges that row's first. Both are
// found by counters that reset themselves.
//
// Rounding: exponentials and a thread's sum (at most 512 of them) are fp32, the sums of threads
// and chunks and every score are 64-bit. The logarithm of a row's sum is off by less than 2e-5: a
// thread adds 8 pairs in each of 32 tiles at most (41 roundings on a value's way, 2.4e-6) and
// rescales its sum as often at most (2^-22 for the exponential, 2^-24 for the product, and the
// argument's rounding: 1.1e-5), and three exponentials more make 9e-7. Measured over 512 rows each of 1000
// to 262144 tokens of both types: 3e-7 at most, 6e-8 in the mean square. Offers of different beams
// that are nearer may change places. Scores are stored in fp32.
//
// What bounds it: with many rows the logits' bytes and the selection behind each chunk's stream
// (512 rows of 262144 fp32 of which 15 % are finished and not read: 444 MB in 92-95 us, 4.8 TB/s;
// the stream alone takes 75, 5.9 TB/s or 0.92 of the copy rate; deeper rings in shared memory
// and a fetch of the next chunk into L2 changed neither). With few rows the chain of dependent
// steps behind the stream (64 rows of bf16 with rings in 26.5 us, of which the logits take 6; 4
// rows of 32000 in 8.6 us): bound, elements, selection, and a merge or two, each a count, loads
// and a selection. Notes of group maxima instead of a list that the stream itself fills took the
// 512 rows from 177 to 97 us: the list's code cost the loop its registers.
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
constexpr int kBWarps = kBThreads / 32;
constexpr int kPer = 16;                      // elements of a tile per thread
constexpr int kTile = kBThreads * kPer;       // 4096
constexpr int kVecs = 4;                      // 16-byte loads per thread that are in flight together
constexpr int kListLimit = 512;               // entries before a list is cut back to K
constexpr int kListShort = 96;                // entries that are ranked without a bound
constexpr int kListCap = kTile + kListLimit;  // a tile may add every element it has
constexpr int kMaxTiles = 32;                 // tiles of a chunk
constexpr int kGroups = kBThreads;            // groups that may be read again
constexpr int kOneMerge = 512;                // entries of a prompt's lists that are merged at once
constexpr int kStopsKept = 64;                // stop ids in shared memory
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
// The order of fp32 values without NaN as that of whole numbers (the upper half of their keys), and
// back.
__device__ __forceinline__ uint32_t order_of(float v) { return (uint32_t)(make_key(v, 0) >> 32); }
__device__ __forceinline__ float order_value(uint32_t order) { return key_value((u64)order << 32); }
// The order of doubles without NaN as that of whole numbers.
__device__ __forceinline__ u64 order_of(double v) {
    const u64 u = (u64)__double_as_longlong(v + 0.0);
    return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Counts one more of a group of CTAs, and orders what the CTA wrote before (its barrier) and what
// it reads behind the count.
__device__ __forceinline__ uint32_t count_in(uint32_t* counter) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}

struct SelectShared {
    u64 list[kListCap];
    u64 best[VDXS_BEAM_MAX_BEAMS];
    u64 maxima[kBThreads];
    u64 bound;
    int count, extra, reach;
    uint32_t marked;  // tiles with marks
    // The penalised tokens' maximum (in key order; 0: none), their sum of exponentials relative to it
    // in units of 2^-40, and whether one of them is NaN or +infinity.
    uint32_t held_max;
    int held_bad;
    u64 held_sum;
    int flag;
    uint32_t top_bound;
    float2 sums[kBThreads];  // each thread's maximum, and its sum of exponentials relative to that
    // The prompt's rows before the step.
    float score[VDXS_BEAM_MAX_BEAMS];
    int done[VDXS_BEAM_MAX_BEAMS], old[VDXS_BEAM_MAX_BEAMS];
    int stop[kStopsKept];
    // What becomes of them: where the rings are moved here.
    int parent[VDXS_BEAM_MAX_BEAMS], token[VDXS_BEAM_MAX_BEAMS], slot[VDXS_BEAM_MAX_BEAMS];
    int pos[VDXS_BEAM_MAX_BEAMS], held[VDXS_BEAM_MAX_BEAMS];
    double lse[VDXS_BEAM_MAX_BEAMS], size[VDXS_BEAM_MAX_BEAMS];  // size: length^alpha
    unsigned short group[kGroups];
};
// The selection's shared memory, named anew in every function: through a reference its accesses
// would be generic ones.
extern __shared__ __align__(16) unsigned char select_smem[];
__device__ __forceinline__ SelectShared& select_shared() { return *reinterpret_cast<SelectShared*>(select_smem); }
static_assert(kMaxTiles * kBThreads * sizeof(float) <= sizeof(u64) * kListCap, "the groups' maxima lie in the list");
static_assert(kGroups * kPer <= kListCap, "a list holds the groups' elements");

// How many of the n (a multiple of 4) values at p are above mine, or equal to it at a lower
// place.
__device__ __forceinline__ int count_above(const uint32_t* p, int n, uint32_t mine, int place) {
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(p + j);
        above += (o.x > mine || (o.x == mine && j < place)) + (o.y > mine || (o.y == mine && j + 1 < place)) +
                 (o.z > mine || (o.z == mine && j + 2 < place)) + (o.w > mine || (o.w == mine && j + 3 < place));
    }
    return above;
}

// The K-th largest of 64 (K <= 16) or 128 disjoint groups' maxima, of one value per thread: a
// lower bound of the K-th largest of what the values are the maxima of. In sh.top_bound. The
// values are upper halves of keys, compared as whole numbers: those of doubles (select_prompt) are
// no fp32 values, and some of them would be NaN.
__device__ __forceinline__ void block_bound(uint32_t v, int K) {
    SelectShared& sh = select_shared();
    uint32_t* groups = reinterpret_cast<uint32_t*>(sh.maxima);
    const int tid = threadIdx.x, share = K <= 16 ? 4 : 2, n = kBThreads / share;
    v = max(v, __shfl_xor_sync(FULLMASK, v, 1));
    if (share == 4) v = max(v, __shfl_xor_sync(FULLMASK, v, 2));
    if (tid % share == 0) groups[tid / share] = v;
    __syncthreads();
    if (tid < n && count_above(groups, n, groups[tid], tid) == K - 1) sh.top_bound = groups[tid];
    __syncthreads();
}

// Keeps list[0..n) entries that are at least `bound`, n at most M for each thread; their number
// in sh.count.
template <int M>
__device__ __forceinline__ void block_keep(int n, u64 bound) {
    SelectShared& sh = select_shared();
    const int tid = threadIdx.x;
    u64 mine[M];
    int m = 0;
#pragma unroll
    for (int j = 0; j < M; ++j) {
        const int i = tid + j * kBThreads;
        mine[j] = i < n && sh.list[i] >= bound ? sh.list[i] : 0;
        m += mine[j] != 0;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    int at = m ? atomicAdd(&sh.count, m) : 0;
#pragma unroll
    for (int j = 0; j < M; ++j)
        if (mine[j]) sh.list[at++] = mine[j];
    __syncthreads();
}

// Cuts list[0..count) to its K largest, in order, in best[]; the rest of best is 0.
// Of a longer list first those that reach a bound stay. Equal values get past that: while the
// list is still long, each thread takes the largest key of its share, the K-th largest of
// those (keys are all different) is a bound again, and at most a quarter plus K remain. Then
// every entry counts the ones above it.
__device__ __noinline__ void block_select(int K) {
    SelectShared& sh = select_shared();
    const int tid = threadIdx.x;
    __syncthreads();
    int n = sh.count;
    if (tid < K) sh.best[tid] = 0;
    if (n > kListShort) {
        u64 mx = 0;
        for (int i = tid; i < n; i += kBThreads) mx = max(mx, sh.list[i]);
        block_bound((uint32_t)(mx >> 32), K);
        const u64 bound = (u64)sh.top_bound << 32;
        if (n <= 2 * kBThreads) block_keep<2>(n, bound);
        else block_keep<kListCap / kBThreads>(n, bound);
        n = sh.count;
    }
    while (n > kListLimit) {
        u64 mx = 0;
        for (int i = tid; i < n; i += kBThreads) mx = max(mx, sh.list[i]);
        sh.maxima[tid] = mx;
        __syncthreads();
        int above = 0;
        for (int j = 0; j < kBThreads; ++j) {
            const u64 o = sh.maxima[j];
            above += o > mx || (o == mx && j < tid);
        }
        if (above == K - 1) sh.bound = mx;
        __syncthreads();
        block_keep<kListCap / kBThreads>(n, sh.bound);
        n = sh.count;
    }
    if (tid == 0) sh.list[n] = 0;  // an even number of entries
    __syncthreads();
    // A short list's entries have 8, 4 or 2 neighbouring threads each, which share the counting.
    const int lanes = n <= 32 ? 8 : n <= 64 ? 4 : n <= 128 ? 2 : 1;
    for (int i0 = 0; i0 < n; i0 += kBThreads / lanes) {
        const int i = i0 + tid / lanes;
        const u64 mine = i < n ? sh.list[i] : ~0ull;
        int above = 0;
#pragma unroll 4
        for (int j = 2 * (tid % lanes); j < n; j += 2 * lanes) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(sh.list + j);
            above += (o.x > mine) + (o.y > mine);
        }
        for (int d = 1; d < lanes; d *= 2) above += __shfl_xor_sync(FULLMASK, above, d);
        if (i < n && above < K) sh.best[above] = mine;
    }
    __syncthreads();
}

template <typename T>
struct Vec;  // 16 bytes of logits
template <>
struct Vec<float> {
    static constexpr int N = 4;
    static constexpr uint32_t kLowest = 0xFF800000u;  // -infinity
    static __device__ __forceinline__ float one(const float* p) { return __ldg(p); }
    // Elements e..e+3 (e a multiple of 4); what lies outside [lo, hi) is -infinity.
    static __device__ __forceinline__ void four(const float* p, int e, int lo, int hi, float* v) {
        const uint4 w = e >= lo && e + 4 <= hi ? __ldg(reinterpret_cast<const uint4*>(p + e)) : edge(p, e, lo, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = at(&w, i);
    }
    static __device__ __forceinline__ float at(const uint4* v, int i) {
        const uint4 w = v[i / 4];
        return __uint_as_float(i % 4 == 0 ? w.x : i % 4 == 1 ? w.y : i % 4 == 2 ? w.z : w.w);
    }
    // A vector of which only the elements [lo, hi) may be read.
    static __device__ __noinline__ uint4 edge(const float* p, int e, int lo, int hi) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = e + i >= lo && e + i < hi ? __float_as_uint(__ldg(p + e + i)) : kLowest;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void four(const __nv_bfloat16* p, int e, int lo, int hi, float* v) {
        uint4 w;
        if (e >= lo && e + 4 <= hi) {
            const uint2 two = __ldg(reinterpret_cast<const uint2*>(p + e));
            w = make_uint4(two.x, two.y, 0u, 0u);
        } else {
            w = edge(p, e, lo, hi);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = at(&w, i);
    }
    static __device__ __forceinline__ float at(const uint4* v, int i) {
        const uint4 q = v[i / 8];
        const int j = (i % 8) / 2;
        const uint32_t w = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
        return __uint_as_float(i % 2 ? w & 0xFFFF0000u : w << 16);
    }
    static __device__ __noinline__ uint4 edge(const __nv_bfloat16* p, int e, int lo, int hi) {
        const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int a = e + 2 * i;
            const uint32_t x = a >= lo && a < hi ? __ldg(s + a) : 0xFF80u;
            const uint32_t y = a + 1 >= lo && a + 1 < hi ? __ldg(s + a + 1) : 0xFF80u;
            w[i] = x | y << 16;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// Two fp32 values in one register pair, for the packed operations of sm_100.
__device__ __forceinline__ u64 pack2(float lo, float hi) {
    u64 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void unpack2(u64 v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
    u64 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// One vector of a chunk; what lies outside [lo, hi) is -infinity.
template <typename T>
__device__ __forceinline__ uint4 load_vector(const T* base, int e, int lo, int hi) {
    return e >= lo && e + Vec<T>::N <= hi ? __ldg(reinterpret_cast<const uint4*>(base + e))
                                          : Vec<T>::edge(base, e, lo, hi);
}

// The elements of a vector that can be among the K largest enter the list.
template <typename T>
__device__ __forceinline__ void enter(const T* base, const uint32_t* marks, int e, int lo, int hi,
                                      float tau, bool equal, int shift) {
    SelectShared& sh = select_shared();
    const uint4 raw = load_vector(base, e, lo, hi);
    const uint32_t out = marks && e < hi ? marks[e >> 5] >> (e & 31) : 0u;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) {
        const float v = Vec<T>::at(&raw, i);
        if ((equal ? v >= tau : v > tau) && v > -INFINITY && !(out >> i & 1))
            sh.list[atomicAdd(&sh.count, 1)] = make_key(v, e + i + shift);
    }
}

// Where many groups reach the bound (equal logits): the chunk tile by tile, the list cut to
// its K largest whenever it is long. From the first cut on the K entries have lower
// tokens than what follows, so an element equal to the K-th stays out.
template <typename T>
__device__ __noinline__ void select_slow(const T* base, bool marked, int lo, int hi, float tau, int shift, int K) {
    SelectShared& sh = select_shared();
    const uint32_t* marks = marked ? reinterpret_cast<uint32_t*>(select_smem + sizeof(SelectShared)) : nullptr;
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    bool equal = true;
    __syncthreads();
    for (int t0 = 0; t0 < hi; t0 += kTile) {
        for (int u = 0; u < kPer / Vec<T>::N; ++u)
            enter<T>(base, marks, t0 + (u * kBThreads + tid) * Vec<T>::N, lo, hi, tau, equal, shift);
        __syncthreads();
        if (sh.count > kListLimit) {
            block_select(K);
            if (tid < K) sh.list[tid] = sh.best[tid];
            if (tid == 0) sh.count = K;
            tau = key_value(sh.best[K - 1]);
            equal = false;
        }
        __syncthreads();
    }
}

// A row's sum of exponentials and its logarithm from its chunks (at most 64), by one warp.
__device__ __forceinline__ void row_sum(const BeamArgs& p, int64_t row, double* sum, double* lse) {
    const int lane = threadIdx.x & 31;
    const double2* part = reinterpret_cast<const double2*>(p.ws.part) + row * p.chunks;
    const double2 zero = make_double2(-INFINITY, 0.0);
    const double2 a = lane < p.chunks ? __ldcg(part + lane) : zero;
    const double2 b = lane + 32 < p.chunks ? __ldcg(part + lane + 32) : zero;
    float M = (float)fmax(a.x, b.x);  // maxima of fp32 values
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(FULLMASK, M, d));
    double S = a.y * ex2(((float)a.x - M) * kLog2e) + b.y * ex2(((float)b.x - M) * kLog2e);
    for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(FULLMASK, S, d);
    *sum = S;
    *lse = M + log(S);
}

// The prompt's offers: the K best of each beam's K (or, unmerged, of its chunks' lists). The order
// is that of the ranks in 64 bits with the offer's number (beam, then place) in the last 13 of
// them, so that equal ranks go to the lower beam and in a beam to the lower chunk and place;
// ranks within 2^-39 of one another count as equal.
__device__ __forceinline__ void select_prompt(const BeamArgs& p, int prompt) {
    SelectShared& sh = select_shared();
    const int tid = threadIdx.x, K = p.beams;
    const int64_t row0 = (int64_t)prompt * K;
    const int per = p.merge_rows ? K : p.chunks * K, n = K * per;  // offers of a beam, of the prompt
    const u64* lists = (p.merge_rows ? p.ws.best : p.ws.cand) + row0 * per;
    u64* keys = sh.list + n + 1;  // the offers' keys, where there is room (the select uses one place more)
    const bool kept = 2 * n + 1 <= kListCap;
    if (tid < min(p.n_stop, kStopsKept)) sh.stop[tid] = p.stop_ids[tid];
    if (p.merge_rows) {
        if (tid < K) sh.lse[tid] = sh.done[tid] ? 0.0 : __ldcg(p.ws.lse + row0 + tid);
    } else {
        for (int b = tid >> 5; b < K; b += kBWarps) {
            if (sh.done[b] || !(sh.score[b] > -INFINITY)) continue;
            double sum, lse;
            row_sum(p, row0 + b, &sum, &lse);
            // A NaN sum (a NaN or +infinity in the row), or none, offers nothing: its offers are NaN.
            if ((tid & 31) == 0) sh.lse[b] = sum > 0.0 ? lse : nan("");
        }
    }
    if (tid == 0) sh.count = n;
    auto offer = [&](int b, u64 key) { return (double)sh.score[b] + ((double)key_value(key) - sh.lse[b]); };
    for (int e0 = 0; e0 < n; e0 += kBThreads) {
        const int e = e0 + tid, b = e / per, i = e - b * per;
        const bool mine = e < n;
        const u64 k = mine && !sh.done[b] ? __ldcg(lists + e) : 0;
        if (e0 == 0) __syncthreads();
        if (!mine) break;
        if (kept) keys[e] = k;
        double score = -INFINITY;
        if (sh.done[b] ? i == 0 : !(sh.score[b] > -INFINITY)) score = sh.score[b];
        else if (k) score = offer(b, k);
        if (p.alpha != 0.0) score /= sh.size[b];
        sh.list[e] = score > -INFINITY ? (order_of(score) & ~8191ull) | (u64)(8191 - e) : 0;
    }
    block_select(K);
    if (tid < K) {
        const int64_t r = row0 + tid;
        const u64 pick = sh.best[tid];
        const bool nothing = pick == 0;
        const int e = 8191 - (int)(pick & 8191), b = nothing ? tid : e / per;
        const bool fresh = !nothing && !sh.done[b];
        u64 key = 0;
        if (fresh) key = kept ? keys[e] : __ldcg(lists + e);
        const int token = fresh ? key_token(key) : p.pad;
        bool stop = false;
        if (fresh) {
            for (int i = 0; i < min(p.n_stop, kStopsKept); ++i) stop |= sh.stop[i] == token;
            for (int i = kStopsKept; i < p.n_stop; ++i) stop |= p.stop_ids[i] == token;
        }
        if (p.move_rings) {
            sh.parent[tid] = b;
            sh.token[tid] = token;
            const int at = p.pos_in[row0 + b] % p.window;
            sh.pos[tid] = at < 0 ? at + p.window : at;
            sh.held[tid] = p.count_in[row0 + b];
            sh.slot[tid] = fresh ? sh.pos[tid] : -1;
        }
        p.tokens[r] = token;
        p.parents[r] = b;
        p.scores[r] = nothing ? -INFINITY : fresh ? (float)offer(b, key) : sh.score[b];
        p.lengths[r] = sh.old[b] + fresh;
        p.finished[r] = nothing ? 0 : fresh ? stop : 1;
        p.ws.push[r] = fresh;
    }
    if (!p.move_rings) return;
    // The rings, and AddToHistory (Sampler.pas:530-539) of the new tokens: as many columns of all
    // beams at a time as the list's room holds, read before any is written.
    const int W = p.window, most = (int)(sizeof(sh.list) / 4) / K;
    int32_t* stage = reinterpret_cast<int32_t*>(sh.list);
    for (int j0 = 0; j0 < W; j0 += most) {
        const int c = min(most, W - j0);
        __syncthreads();
        for (int i = tid; i < K * c; i += kBThreads)
            stage[i] = p.hist_in[(row0 + sh.parent[i / c]) * W + j0 + i % c];
        __syncthreads();
        for (int i = tid; i < K * c; i += kBThreads) {
            const int k = i / c, j = j0 + i % c;
            p.hist[(row0 + k) * W + j] = sh.slot[k] == j ? sh.token[k] : stage[i];
        }
    }
    if (tid < K) {
        const bool push = sh.slot[tid] >= 0;
        const int held = sh.held[tid];
        p.pos[row0 + tid] = push ? (sh.pos[tid] + 1) % W : sh.pos[tid];
        p.count[row0 + tid] = push && held < W ? max(held, 0) + 1 : held;
    }
}

// Registers for three CTAs on an SM, for four with bf16, whose tiles have half the bytes (64 x 8 of
// 262144 bf16 59 us against 64 with three; fp32 with four 96 against 94).
template <typename T, bool PEN>
__global__ void __launch_bounds__(kBThreads, sizeof(T) == 2 ? 4 : 3) beam_select_kernel(const __grid_constant__ BeamArgs p) {
    SelectShared& sh = select_shared();
    uint32_t* marks = reinterpret_cast<uint32_t*>(select_smem + sizeof(SelectShared));  // PEN: a bit for each position
    struct Held {
        int held;
        float value;
    };
    Held* extra = reinterpret_cast<Held*>(select_smem + sizeof(SelectShared) + p.chunk / 8);  // PEN: the ring's tokens
    constexpr int VN = Vec<T>::N;
    constexpr int kUnit = kBThreads * kVecs * VN;  // elements that are loaded together: one tile, two of bf16
    asm volatile("griddepcontrol.launch_dependents;");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.beams;
    const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks;
    const int prompt = row / K;
    const bool live = p.finished_in[row] == 0 && p.scores_in[row] > -INFINITY;
    if (tid < K) {
        // The prompt's rows, for its last CTA: nothing is written before that one.
        const int64_t r = (int64_t)prompt * K + tid;
        sh.score[tid] = p.scores_in[r];
        sh.done[tid] = p.finished_in[r] != 0;
        sh.old[tid] = p.lengths_in[r];
    }
    if (live) {
        // Positions count from the 16-byte boundary at or below the row's first element, and
        // within the chunk: [lo, hi) hold logits, position e is token e + shift.
        const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
        const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
        const int64_t c0 = (int64_t)c * p.chunk;
        const T* base = x - off + c0;
        const int lo = c == 0 ? off : 0, hi = (int)min((int64_t)p.chunk, p.vocab + off - c0);
        const int shift = (int)(c0 - off);
        auto load = [&](int u0, uint4* v) {
            const T* at = base + u0 + tid * VN;
            if (u0 >= lo && u0 + kUnit <= hi) {
#pragma unroll
                for (int u = 0; u < kVecs; ++u) v[u] = __ldg(reinterpret_cast<const uint4*>(at + u * kBThreads * VN));
            } else {
#pragma unroll
                for (int u = 0; u < kVecs; ++u) v[u] = load_vector<T>(base, u0 + (u * kBThreads + tid) * VN, lo, hi);
            }
        };
        uint4 next[kVecs];
        load(0, next);
        float m = -FLT_MAX, s = 0.0f;
        // The chunk's tokens that the ring holds leave the stream (their marks) and are added behind
        // it, with x / p for x > 0, else x * p, once for each time that the ring holds them
        // (Sampler.pas:285-303). The entry whose thread sets the mark stands for the token
        // (held >= 0), the others are ~token.
        const int32_t* ring = PEN ? p.hist_in + (int64_t)row * p.window : nullptr;
        int my_place = -1;
        float my_value = 0.0f;
        if (PEN) {
            const int count = p.count_in[row];
            if (tid == 0) sh.extra = 0, sh.marked = 0, sh.held_max = 0, sh.held_bad = 0, sh.held_sum = 0;
            for (int i = tid; i < p.chunk / 32; i += kBThreads) marks[i] = 0;
            int token = tid < p.window ? ring[tid] : -1;
            __syncthreads();
            for (int i = tid; i < p.window && i < count; i += kBThreads) {
                if (i != tid) token = ring[i];
                const int64_t e = (int64_t)token - shift;
                if (token >= 0 && token < p.vocab && e >= lo && e < hi) {
                    const uint32_t bit = 1u << (e & 31);
                    const bool first = !(atomicOr(&marks[e >> 5], bit) & bit);
                    atomicOr(&sh.marked, 1u << (e / kTile));
                    const int at = atomicAdd(&sh.extra, 1);
                    extra[at].held = first ? token : ~token;
                    if (i == tid) my_place = at, my_value = Vec<T>::one(base + e);
                    else extra[at].value = Vec<T>::one(base + e);
                }
            }
            __syncthreads();
        }
        const uint32_t marked = PEN ? sh.marked : 0u;
        float* tops = reinterpret_cast<float*>(sh.list);  // [tiles][threads]
        float most = -INFINITY;
        int tiles = 0;
        for (int u0 = 0; u0 < hi; u0 += kUnit) {
            uint4 raw[kVecs];
#pragma unroll
            for (int u = 0; u < kVecs; ++u) raw[u] = next[u];
            if (u0 + kUnit < hi) load(u0 + kUnit, next);
#pragma unroll
            for (int part = 0; part < kVecs * VN / kPer; ++part) {
                float v[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) v[i] = Vec<T>::at(raw, part * kPer + i);
                if (PEN && (marked >> tiles & 1)) {
#pragma unroll
                    for (int u = 0; u < kPer / VN; ++u) {
                        const int e = u0 + part * kTile + (u * kBThreads + tid) * VN;
                        const uint32_t w = e < hi ? (marks[e >> 5] >> (e & 31)) & ((1u << VN) - 1) : 0u;
                        if (w) {
#pragma unroll
                            for (int i = 0; i < VN; ++i)
                                if (w >> i & 1) v[u * VN + i] = -INFINITY;
                        }
                    }
                }
                float top = v[0];
#pragma unroll
                for (int i = 1; i < kPer; ++i) top = fmaxf(top, v[i]);
                tops[tiles++ * kBThreads + tid] = top;
                most = fmaxf(most, top);
                if (top > m) {
                    s *= ex2((m - top) * kLog2e);
                    m = top;
                }
                u64 sum = 0;
                const u64 minus = pack2(-m, -m), scale = pack2(kLog2e, kLog2e);
#pragma unroll
                for (int i = 0; i < kPer; i += 2) {
                    float y0, y1;
                    unpack2(mul2(add2(pack2(v[i], v[i + 1]), minus), scale), y0, y1);
                    sum = add2(sum, pack2(ex2(y0), ex2(y1)));
                }
                float sum0, sum1;
                unpack2(sum, sum0, sum1);
                s += sum0 + sum1;
            }
        }
        const int extras = PEN ? sh.extra : 0;
        if (PEN) {
            // Which thread has which token hangs on the order of atomics, so they are summed in whole
            // numbers.
            if (my_place >= 0) extra[my_place].value = my_value;  // fetched while the stream ran
            __syncthreads();
            for (int i = tid; i < extras; i += kBThreads) {
                const int token = extra[i].held;
                if (token < 0) continue;
                float v = extra[i].value;
                int times = 0;
                for (int j = 0; j < extras; ++j) {
                    const int other = extra[j].held;
                    times += other == token || ~other == token;
                }
                for (; times > 0; --times) v = v > 0.0f ? __fdiv_rn(v, p.penalty) : __fmul_rn(v, p.penalty);
                extra[i].value = v;
                if (!(v < INFINITY)) sh.held_bad = 1;
                else if (v > -INFINITY) atomicMax(&sh.held_max, (uint32_t)(make_key(v, 0) >> 32));
            }
            __syncthreads();
            const float top = key_value((u64)sh.held_max << 32);
            for (int i = tid; i < extras; i += kBThreads) {
                const float v = extra[i].value;
                if (extra[i].held >= 0 && v > -INFINITY && v < INFINITY)
                    atomicAdd(&sh.held_sum, (u64)(ex2((v - top) * kLog2e) * 1099511627776.0f));
            }
        }
        sh.sums[tid] = make_float2(m, s);
        if (tid == 0) sh.count = 0, sh.reach = 0;
        block_bound(order_of(most), K);
        const float tau = order_value(sh.top_bound);
        // Eight tiles' maxima are compared before any is counted, so that their loads do not wait for an
        // atomic's answer, which a group at a time would: 93.9 -> 92.0 us at 64 x 8 of 262144 fp32.
        if (__any_sync(FULLMASK, most >= tau)) {
            for (int t0 = 0; t0 < tiles; t0 += 8) {
                uint32_t mine = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float top = t0 + j < tiles ? tops[(t0 + j) * kBThreads + tid] : -INFINITY;
                    mine |= (uint32_t)(top >= tau && top > -INFINITY) << j;
                }
                int at = mine ? atomicAdd(&sh.reach, __popc(mine)) : 0;
                for (; mine; mine &= mine - 1, ++at)
                    if (at < kGroups) sh.group[at] = (unsigned short)((t0 + __ffs(mine) - 1) * kBThreads + tid);
            }
        }
        __syncthreads();
        const int64_t slot = (int64_t)row * p.chunks + c;
        if (warp == kBWarps - 1) {
            float2 part[kBWarps];
            float M = -FLT_MAX;
#pragma unroll
            for (int j = 0; j < kBWarps; ++j) part[j] = sh.sums[lane + 32 * j], M = fmaxf(M, part[j].x);
            for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(FULLMASK, M, d));
            double S = 0.0;
#pragma unroll
            for (int j = 0; j < kBWarps; ++j) S += (double)part[j].y * ex2((part[j].x - M) * kLog2e);
            for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(FULLMASK, S, d);
            if (PEN && sh.held_sum > 0) {
                const float top = key_value((u64)sh.held_max << 32), both = fmaxf(M, top);
                S = S * ex2((M - both) * kLog2e) + (double)sh.held_sum * 9.094947017729282e-13 * ex2((top - both) * kLog2e);
                M = both;
            }
            if (PEN && sh.held_bad) S = nan("");
            if (lane == 0) reinterpret_cast<double2*>(p.ws.part)[slot] = make_double2(M, S);
        }
        const int reach = sh.reach;
        if (reach <= kGroups) {
            // Four elements for each thread.
            for (int q = tid; q < reach * (kPer / 4); q += kBThreads) {
                const int at = sh.group[q / (kPer / 4)], i = q % (kPer / 4) * 4;
                const int e0 = at / kBThreads * kTile + (i / VN * kBThreads + at % kBThreads) * VN + i % VN;
                float v[4];
                Vec<T>::four(base, e0, lo, hi, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = e0 + j;
                    if (v[j] >= tau && v[j] > -INFINITY && !(PEN && (marks[e >> 5] >> (e & 31) & 1)))
                        sh.list[atomicAdd(&sh.count, 1)] = make_key(v[j], e + shift);
                }
            }
        } else {
            select_slow<T>(base, PEN, lo, hi, tau, shift, K);
        }
        if (PEN) {
            // The ring's tokens join the rest: at most a list's limit at a time, the rest cut before.
            for (int i0 = 0; i0 < extras; i0 += kListLimit) {
                if (i0 > 0 || reach > kGroups) {
                    block_select(K);
                    if (tid < K) sh.list[tid] = sh.best[tid];
                    if (tid == 0) sh.count = K;
                    __syncthreads();
                }
                for (int i = i0 + tid; i < min(extras, i0 + kListLimit); i += kBThreads)
                    if (extra[i].held >= 0 && extra[i].value >= tau && extra[i].value > -INFINITY)
                        sh.list[atomicAdd(&sh.count, 1)] = make_key(extra[i].value, extra[i].held);
            }
        }
        block_select(K);
        if (tid < K) p.ws.cand[slot * K + tid] = sh.best[tid];
    }
    __syncthreads();
    const int group = p.merge_rows ? K : K * p.chunks;  // that are counted for a prompt
    if (p.merge_rows) {
        // The row's last CTA merges its chunks.
        if (tid == 0) sh.flag = count_in(&p.ws.row_done[row]) == (uint32_t)p.chunks - 1;
        __syncthreads();
        if (!sh.flag) return;
        if (live) {
            const int n = p.chunks * K;
            if (tid == 0) sh.count = n;
            if (warp == kBWarps - 1) {
                double sum, lse;
                row_sum(p, row, &sum, &lse);
                if (lane == 0) p.ws.lse[row] = sum > 0.0 ? lse : nan("");
            }
            // Empty places have key 0 and stay below every entry.
            for (int i = tid; i < n; i += kBThreads) sh.list[i] = __ldcg(p.ws.cand + (int64_t)row * n + i);
            block_select(K);
            if (tid < K) p.ws.best[(int64_t)row * K + tid] = sh.best[tid];
        }
        __syncthreads();
        if (tid == 0) p.ws.row_done[row] = 0;
    }
    if (tid == 0) sh.flag = count_in(&p.ws.prompt_done[prompt]) == (uint32_t)group - 1;
    __syncthreads();
    if (!sh.flag) return;
    if (tid == 0) p.ws.prompt_done[prompt] = 0;
    if (p.alpha != 0.0 && tid >= kBThreads - K) {
        const int b = tid - (kBThreads - K);
        sh.size[b] = pow((double)max(sh.done[b] ? sh.old[b] : sh.old[b] + 1, 1), p.alpha);
    }
    select_prompt(p, prompt);
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

// Bound by the bytes: with two caches of 64 rows x 4 heads x 2500 x 256 bf16 and their rings to move, a
// step of 64 rows of 32000 fp32 takes 176-184 us, 149-160 of them here (0.66 GB written; parents
// that beams share are read once from memory and then from L2).
//
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
    __shared__ int token[VDXS_BEAM_MAX_BEAMS], slot[VDXS_BEAM_MAX_BEAMS];
    // A step's reordering is launched while its selection still runs, and waits here for its end.
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
        token[k] = p.tokens[row0 + k];
        slot[k] = p.push[row0 + k] ? pos[k] : -1;
    }
    __syncthreads();
    int32_t* mine = reinterpret_cast<int32_t*>(stage) + threadIdx.x;
    for (int j = threadIdx.x; j < W; j += kRThreads) {
#pragma unroll 8
        for (int k = 0; k < K; ++k) mine[k * kRThreads] = p.hist_in[(row0 + parent[k]) * W + j];
        for (int k = 0; k < K; ++k) p.hist[(row0 + k) * W + j] = slot[k] == j ? token[k] : mine[k * kRThreads];
    }
    for (int k = threadIdx.x; k < K; k += kRThreads) {
        const bool push = slot[k] >= 0;
        p.pos[row0 + k] = push ? (pos[k] + 1) % W : pos[k];
        p.count[row0 + k] = push && count[k] < W ? max(count[k], 0) + 1 : count[k];
    }
}

}  // namespace

void beam_plan(int rows, int vocab, int sm_count, int* chunks, int* chunk) {
    // A position is counted from a 16-byte boundary, so up to 7 lie before the row.
    const int64_t span = (int64_t)vocab + 7;
    const int64_t tiles = (span + kTile - 1) / kTile;
    // Three CTAs for each SM (for bf16 too, although four fit), at most kBeamMaxChunks lists to
    // merge, and at most kMaxTiles tiles to a chunk.
    int64_t want = std::min<int64_t>(kBeamMaxChunks, std::max<int64_t>(1, (int64_t)sm_count * 3 / rows));
    want = std::min(std::max(want, (tiles + kMaxTiles - 1) / kMaxTiles), tiles);
    const int64_t per = (tiles + want - 1) / want;
    *chunk = (int)(per * kTile);
    *chunks = (int)((tiles + per - 1) / per);
}

cudaError_t beam_select(const BeamArgs& a, cudaStream_t stream) {
    BeamArgs p = a;
    // One merge for a prompt while its lists are short; else the rows' first, which run beside one
    // another (2 x 10 of 262144 fp32, 2200 entries: 14.7 us with two merges, 17.4 with one; 16 x 4
    // of 262144 bf16, 96 entries: 18.4 and 17.1).
    p.merge_rows = (int64_t)a.beams * a.chunks * a.beams > kOneMerge;
    const bool pen = a.window > 0 && a.penalty != 1.0f;
    const size_t smem = sizeof(SelectShared) + (pen ? (size_t)a.chunk / 8 + (size_t)a.window * 8 : 0);
    const int grid = a.batch * a.beams * a.chunks;
    const bool half = a.dtype == VDXS_DTYPE_BF16;
    void (*kern)(BeamArgs) = half ? (pen ? beam_select_kernel<__nv_bfloat16, true> : beam_select_kernel<__nv_bfloat16, false>)
                                  : (pen ? beam_select_kernel<float, true> : beam_select_kernel<float, false>);
    static SmemLimit limit[4];
    cudaError_t e = limit[2 * half + pen].raise(kern, smem);
    if (e != cudaSuccess) return e;
    kern<<<grid, kBThreads, smem, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t beam_reorder(const BeamArgs& a, bool behind_select, const BeamCacheArgs* caches, int n_caches,
                         cudaStream_t stream, int* launches) {
    bool rings = behind_select && a.window > 0 && !a.move_rings;
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
        cudaLaunchAttribute early{};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3(kRThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cfg.attrs = &early;
        cfg.numAttrs = behind_select ? 1 : 0;
        behind_select = false;
        if ((e = cudaLaunchKernelEx(&cfg, beam_reorder_kernel, p)) != cudaSuccess) return e;
        ++*launches;
    }
    return cudaSuccess;
}

}  // namespace vdxs
