// vdxs_i8.cu - the operands of the 8-bit unembedding: the final norm with an 8-bit output
// (residual's addition, root-mean-square norm, a scale per token), and the weights with a
// scale per vocabulary entry. The norm stands where TVdxModel.UnembedToLogits
// (src/VindexLLM.Model.pas:1258-1271) runs it; the product is in vdxs_i8_product.cu.
#include "vdxs_internal.h"
#include "../../include/vdx_sampler.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

namespace vdxs {
namespace {

constexpr unsigned FULLMASK = 0xFFFFFFFFu;
constexpr int kNormThreads = 256;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Sum of `a` and maximum of `b` over the block, in every thread.
template <typename B>
__device__ __forceinline__ void block_sum_max(double& a, B& b) {
    __shared__ double sa[32];
    __shared__ B sb[32];
    for (int s = 16; s > 0; s >>= 1) {
        a += __shfl_xor_sync(FULLMASK, a, s);
        b = max(b, __shfl_xor_sync(FULLMASK, b, s));
    }
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0) sa[warp] = a, sb[warp] = b;
    __syncthreads();
    a = sa[0];
    b = sb[0];
    for (int w = 1; w < warps; ++w) a += sa[w], b = max(b, sb[w]);
}

// q = 127 t / top to the nearest even integer. Values of up to 35 bits (every product but that of two
// fp32 values): 127 t is exact, and a quotient that is not on a border is 2^-36 or more from
// it, far more than its rounding.
__device__ __forceinline__ int quantum(double t, double top) { return (int)rint(t * 127.0 / top); }
// Products of two fp32 values have 48 bits, so 127 t may be rounded, and the quotient fall on the wrong
// side. Where it comes out next to a border b = k + 1/2, the sign of 127 t - b top decides, both
// products in two parts: the high parts' difference is exact, and so is that of the low ones,
// which have four bits at most.
__device__ __noinline__ int border_quantum(double t, double top, double b) {
    const double p = t * 127.0, u = b * top, d = (p - u) + (fma(t, 127.0, -p) - fma(b, top, -u));
    return (int)(d > 0.0 ? b + 0.5 : d < 0.0 ? b - 0.5 : rint(b));
}
__device__ __forceinline__ int wide_quantum(double t, double top) {
    const double v = t * 127.0 / top, r = rint(v), off = v - r;
    return fabs(off) < 0.499999999 ? (int)r : border_quantum(t, top, r + copysign(0.5, off));
}
// Four of them as bytes. One call: written out where it is needed, it took registers from the rows that
// need none of it (8192 x 3840 fp32 68 us against 71).
__device__ __noinline__ uint32_t wide_quanta(float4 a, float4 b, double top) {
    const double t[4] = {(double)a.x * b.x, (double)a.y * b.y, (double)a.z * b.z, (double)a.w * b.w};
    uint32_t word = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) word |= (uint32_t)(wide_quantum(t[i], top) & 0xFF) << (8 * i);
    return word;
}
template <typename T, typename W>
__device__ __forceinline__ int quantum_of(double t, double top) {
    if constexpr (sizeof(T) == 4 && sizeof(W) == 4) return wide_quantum(t, top);
    else return quantum(t, top);
}

// The same from fp32 where that decides: t32, f = 127 / top and their product are rounded once
// each (2^-24 relative), so v is off by at most 127 * 3 * 2^-24 = 2.3e-5; a v that is 3e-5 from
// a border rounds as the exact quotient does. Else (one value in 17000) false.
__device__ __forceinline__ bool quick_quantum(float t32, float f, int* q) {
    // Adding 1.5 * 2^23 rounds to the nearest even integer and leaves it in the low bits.
    const float v = t32 * f, r = __fadd_rn(v, 12582912.0f);
    *q = __float_as_int(r) - 0x4B400000;
    return fabsf(v - __fadd_rn(r, -12582912.0f)) <= 0.49997f;
}

// A row in 64 bits throughout. `done`: h is in p.hidden (or is x itself) already.
template <typename T, typename W>
__device__ __noinline__ void norm_row(const NormI8Args& p, int64_t row, bool done) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
    T* hidden = p.hidden ? static_cast<T*>(p.hidden) + row * p.hidden_stride : nullptr;
    const W* w = static_cast<const W*>(p.weight);
    auto sum_of = [&](int i) { return r ? from_f32<T>(to_f32(x[i]) + to_f32(r[i])) : x[i]; };
    double sum = 0.0, top = 0.0;
    bool bad = false;
    for (int i = threadIdx.x; i < p.dim; i += blockDim.x) {
        const T v = done && hidden ? hidden[i] : sum_of(i);
        if (!done && hidden) hidden[i] = v;
        const double d = to_f32(v), t = d * (double)to_f32(w[i]);
        bad |= !(fabs(t) <= DBL_MAX) || !(fabs(d) <= DBL_MAX);
        sum += d * d;
        top = fmax(top, fabs(t));
    }
    block_sum_max(sum, top);
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0)
        p.scale[row] = bad         ? nanf("")
                       : top > 0.0 ? (float)(top / 127.0 * (1.0 / sqrt(sum / p.dim + (double)p.eps)))
                                   : 0.0f;  // (zeros without eps too)
    int8_t* q = p.q + row * p.q_stride;
    const float f = (float)(127.0 / top);
    for (int i = threadIdx.x; i < p.dim; i += blockDim.x) {
        // A thread reads what it wrote itself; without p.hidden the inputs are as they were.
        const double t = (double)to_f32(hidden ? hidden[i] : sum_of(i)) * (double)to_f32(w[i]);
        int v = 0;
        if (!bad && top > 0.0 && !(f < 1e30f && quick_quantum((float)t, f, &v))) v = quantum_of<T, W>(t, top);
        q[i] = (int8_t)v;
    }
}

// Rows of any alignment, one per CTA, with scalar loads and 64-bit products: 8192 rows of 3841 bf16 with
// a residual take 190 us.
template <typename T, typename W>
__global__ void __launch_bounds__(kNormThreads) rms_norm_i8_kernel(const __grid_constant__ NormI8Args p) {
    norm_row<T, W>(p, blockIdx.x, false);
}

template <typename T>
struct Pack;  // 16 bytes of a row
template <>
struct Pack<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4& v, float* f) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 put(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <typename T2>
__device__ __forceinline__ uint32_t bits_of(T2 v) {
    return *reinterpret_cast<uint32_t*>(&v);
}
template <>
struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& v, float* f) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
    static __device__ __forceinline__ uint4 put(const float* f) {
        return make_uint4(bits_of(__floats2bfloat162_rn(f[0], f[1])), bits_of(__floats2bfloat162_rn(f[2], f[3])),
                          bits_of(__floats2bfloat162_rn(f[4], f[5])), bits_of(__floats2bfloat162_rn(f[6], f[7])));
    }
};
template <>
struct Pack<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& v, float* f) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = g.x, f[2 * i + 1] = g.y;
        }
    }
    static __device__ __forceinline__ uint4 put(const float* f) {
        return make_uint4(bits_of(__floats2half2_rn(f[0], f[1])), bits_of(__floats2half2_rn(f[2], f[3])),
                          bits_of(__floats2half2_rn(f[4], f[5])), bits_of(__floats2half2_rn(f[6], f[7])));
    }
};
// N weights from an address that is a multiple of 16 bytes (8 for four 16-bit ones).
template <typename W, int N>
__device__ __forceinline__ void get_weights(const W* p, float* f) {
    if constexpr (sizeof(W) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) Pack<float>::get(__ldg(reinterpret_cast<const uint4*>(p + i)), f + i);
    } else if constexpr (N == 8) {
        Pack<W>::get(__ldg(reinterpret_cast<const uint4*>(p)), f);
    } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        float g[8];
        Pack<W>::get(make_uint4(v.x, v.y, 0u, 0u), g);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = g[i];
    }
}

// Rows whose 16-byte vectors are whole and aligned, one per CTA, kept in registers (NV vectors
// per thread), so that every byte crosses memory once. The squares are added in 64 bits. The
// maximum is found in fp32, its exact value among the few products that are within rounding
// of it, and q from fp32 except next to a border. A row whose fp32 maximum says nothing
// (NaN, overflow, subnormal) is done again in 64 bits.
//
// 8192 rows of 3840 with a residual take 51.5 us in bf16 (4.3 TB/s, 0.66 of the copy rate), 46 in fp16
// and 68 in fp32 (0.93). Issue slots and the latency of a row's three steps (load, sum, round) share
// it: 64 registers a thread hold 32 elements, which keeps seven rows on their way on an SM,
// but spill (92 bytes stored, 168 loaded a thread with bf16 rows and fp32 weights, 56 and 156 with
// fp16 rows, 28 and 40 with fp32), and nothing of a row is loaded while another is computed in
// its place. With the products kept in registers instead of the weights read again it took 73 us,
// with 64-bit arithmetic for every element 115.
template <typename T, typename W, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, 1024 / MAXT) rms_norm_i8_rows_kernel(const __grid_constant__ NormI8Args p) {
    constexpr int N = Pack<T>::N;
    __shared__ unsigned long long s_top;
    const int64_t row = blockIdx.x;
    const int nv = p.dim / N;
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + row * p.x_stride);
    const W* w = static_cast<const W*>(p.weight);
    uint4 h[NV];
    float largest[NV];  // of each vector's products
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int v = threadIdx.x + j * blockDim.x;
        h[j] = v < nv ? x[v] : make_uint4(0u, 0u, 0u, 0u);
    }
    if (p.residual) {
        const uint4* r = reinterpret_cast<const uint4*>(static_cast<const T*>(p.residual) + row * p.residual_stride);
        uint4 add[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int v = threadIdx.x + j * blockDim.x;
            add[j] = v < nv ? r[v] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float a[N], b[N];
            Pack<T>::get(h[j], a);
            Pack<T>::get(add[j], b);
#pragma unroll
            for (int i = 0; i < N; ++i) a[i] += b[i];
            h[j] = Pack<T>::put(a);
        }
    }
    if (p.hidden) {
        uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.hidden) + row * p.hidden_stride);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int v = threadIdx.x + j * blockDim.x;
            if (v < nv) out[v] = h[j];
        }
    }
    double sum = 0.0;
    float most = 0.0f, check = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int v = threadIdx.x + j * blockDim.x;
        float a[N], b[N];
        Pack<T>::get(h[j], a);
#pragma unroll
        for (int i = 0; i < N; ++i) b[i] = 0.0f;
        if (v < nv) get_weights<W, N>(w + v * N, b);
        largest[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = a[i] * b[i];
            largest[j] = fmaxf(largest[j], fabsf(t));
            check += t * 0.0f;  // NaN where a product is NaN or infinite
            sum += (double)a[i] * (double)a[i];
        }
        most = fmaxf(most, largest[j]);
    }
    if (!(check == 0.0f)) most = INFINITY;
    if (threadIdx.x == 0) s_top = 0ull;
    block_sum_max(sum, most);
    if (!(most >= 1e-30f && most < 1e38f && sum < DBL_MAX)) {
        // (The block is of one mind here.) h is in p.hidden, or the inputs are as they were.
        __syncthreads();
        norm_row<T, W>(p, row, p.hidden != nullptr);
        return;
    }
    if (blockDim.x == 32) __syncwarp();
    // The exact maximum: a product is off by 2^-24 relative in fp32.
    const float near = most * 0.9999996f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (largest[j] >= near) {
            float a[N], b[N];
            Pack<T>::get(h[j], a);
            get_weights<W, N>(w + (threadIdx.x + j * blockDim.x) * N, b);
            double d = 0.0;
#pragma unroll
            for (int i = 0; i < N; ++i) d = fmax(d, fabs((double)a[i] * (double)b[i]));
            atomicMax(&s_top, (unsigned long long)__double_as_longlong(d));
        }
    }
    __syncthreads();
    const double top = __longlong_as_double((long long)s_top);
    if (threadIdx.x == 0) p.scale[row] = (float)(top / 127.0 * (1.0 / sqrt(sum / p.dim + (double)p.eps)));
    const float f = (float)(127.0 / top);
    int8_t* q = p.q + row * p.q_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int v = threadIdx.x + j * blockDim.x;
        if (v >= nv) break;
        uint32_t word[N / 4];
        bool sure = true;
        float a[N], b[N];
        Pack<T>::get(h[j], a);
        get_weights<W, N>(w + v * N, b);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int k;
            sure &= quick_quantum(a[i] * b[i], f, &k);
            if (i % 4 == 0) word[i / 4] = 0u;
            word[i / 4] |= (uint32_t)(k & 0xFF) << (8 * (i % 4));
        }
        if (!sure) {
            if constexpr (sizeof(T) == 4 && sizeof(W) == 4) {
                word[0] = wide_quanta(make_float4(a[0], a[1], a[2], a[3]), make_float4(b[0], b[1], b[2], b[3]), top);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t k = (uint32_t)(quantum((double)a[i] * (double)b[i], top) & 0xFF);
                    word[i / 4] = (word[i / 4] & ~(0xFFu << (8 * (i % 4)))) | k << (8 * (i % 4));
                }
            }
        }
        if constexpr (N == 8) reinterpret_cast<uint2*>(q)[v] = make_uint2(word[0], word[1]);
        else reinterpret_cast<uint32_t*>(q)[v] = word[0];
    }
}

struct F32Rows {
    const float* p;
    int64_t stride;
    __device__ float at(int64_t row, int i) const { return p[row * stride + i]; }
};
struct Bf16Rows {
    const __nv_bfloat16* p;
    int64_t stride;
    __device__ float at(int64_t row, int i) const { return __bfloat162float(p[row * stride + i]); }
};
struct F16Rows {
    const __half* p;
    int64_t stride;
    __device__ float at(int64_t row, int i) const { return __half2float(p[row * stride + i]); }
};
// 18-byte blocks of 32 elements: an fp16 scale, then element j in the low nibble of byte j and
// element j + 16 in its high nibble.
struct Q40Rows {
    const uint8_t* p;
    int64_t blocks;
    __device__ float at(int64_t row, int i) const {
        const uint8_t* b = p + (row * blocks + (i >> 5)) * 18;
        const float d = __half2float(__ushort_as_half((unsigned short)(b[0] | (b[1] << 8))));
        const int j = i & 31, v = b[2 + (j & 15)];
        return d * (float)((j < 16 ? v & 15 : v >> 4) - 8);
    }
};

// Quantises weight rows once, when the weights are prepared; one row per CTA.
template <typename S>
__global__ void __launch_bounds__(kNormThreads) quantise_rows_kernel(S src, I8Matrix w) {
    const int64_t row = blockIdx.x;
    double sum = 0.0, top = 0.0;
    bool bad = false;
    for (int i = threadIdx.x; i < w.in_dim; i += kNormThreads) {
        const float v = src.at(row, i);
        bad |= !(fabsf(v) <= FLT_MAX);
        top = fmax(top, (double)fabsf(v));
    }
    block_sum_max(sum, top);
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) w.scale[row] = bad ? nanf("") : (float)(top / 127.0);
    for (int i = threadIdx.x; i < w.pitch; i += kNormThreads)
        w.q[row * w.pitch + i] =
            bad || top == 0.0 || i >= w.in_dim ? 0 : (int8_t)quantum((double)src.at(row, i), top);
}

template <typename T, typename W>
cudaError_t launch_norm(const NormI8Args& a, int sm_count, cudaStream_t stream) {
    constexpr int N = Pack<T>::N;
    auto whole = [](const void* p, int64_t stride, size_t size, size_t to) {
        return (uintptr_t)p % to == 0 && (uint64_t)stride * size % to == 0;
    };
    // Whole aligned vectors of every row; a lone row needs its base alone.
    const int64_t one = a.rows > 1;
    const bool rows = a.dim % N == 0 && whole(a.x, one * a.x_stride, sizeof(T), 16) &&
                      whole(a.residual, one * a.residual_stride, sizeof(T), 16) &&
                      whole(a.hidden, one * a.hidden_stride, sizeof(T), 16) && whole(a.q, one * a.q_stride, 1, N) &&
                      (uintptr_t)a.weight % 16 == 0;
    if (!rows) {
        rms_norm_i8_kernel<T, W><<<a.rows, kNormThreads, 0, stream>>>(a);
        return cudaGetLastError();
    }
    // More rows than SMs: 32 elements a thread, so that a row takes few threads and many rows are
    // on their way. Few rows, or short ones: one vector a thread, for the latency (1 row of 2560
    // fp32 in 3.1 us, with the launch).
    constexpr int kMost = 32 / N;
    const int nv = a.dim / N;
    const int per = nv > 1024 || (a.rows > sm_count && nv > 64) ? kMost : 1;
    const int threads = ((nv + per - 1) / per + 31) / 32 * 32;
    if (per == 1) rms_norm_i8_rows_kernel<T, W, 1, 1024><<<a.rows, threads, 0, stream>>>(a);
    else if (threads <= 256) rms_norm_i8_rows_kernel<T, W, kMost, 256><<<a.rows, threads, 0, stream>>>(a);
    else rms_norm_i8_rows_kernel<T, W, kMost, 1024><<<a.rows, threads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_norm_w(const NormI8Args& a, int sm_count, cudaStream_t stream) {
    if (a.weight_dtype == VDXS_DTYPE_BF16) return launch_norm<T, __nv_bfloat16>(a, sm_count, stream);
    if (a.weight_dtype == VDXS_DTYPE_F16) return launch_norm<T, __half>(a, sm_count, stream);
    return launch_norm<T, float>(a, sm_count, stream);
}

}  // namespace

cudaError_t rms_norm_i8(const NormI8Args& a, int sm_count, cudaStream_t stream) {
    if (a.dtype == VDXS_DTYPE_BF16) return launch_norm_w<__nv_bfloat16>(a, sm_count, stream);
    if (a.dtype == VDXS_DTYPE_F16) return launch_norm_w<__half>(a, sm_count, stream);
    return launch_norm_w<float>(a, sm_count, stream);
}

cudaError_t quantise_rows_i8(const void* src, int format, int64_t row_stride, const I8Matrix& w, cudaStream_t stream) {
    const int grid = w.out_dim;
    switch (format) {
        case VDXS_WEIGHTS_F32:
            quantise_rows_kernel<<<grid, kNormThreads, 0, stream>>>(F32Rows{(const float*)src, row_stride}, w);
            break;
        case VDXS_WEIGHTS_BF16:
            quantise_rows_kernel<<<grid, kNormThreads, 0, stream>>>(Bf16Rows{(const __nv_bfloat16*)src, row_stride}, w);
            break;
        case VDXS_WEIGHTS_F16:
            quantise_rows_kernel<<<grid, kNormThreads, 0, stream>>>(F16Rows{(const __half*)src, row_stride}, w);
            break;
        default:
            quantise_rows_kernel<<<grid, kNormThreads, 0, stream>>>(Q40Rows{(const uint8_t*)src, w.in_dim / 32}, w);
    }
    return cudaGetLastError();
}

}  // namespace vdxs
