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
__device__ __forceinline__ void block_sum_max(double& a, double& b) {
    __shared__ double sa[kNormThreads / 32], sb[kNormThreads / 32];
    for (int s = 16; s > 0; s >>= 1) {
        a += __shfl_xor_sync(FULLMASK, a, s);
        b = fmax(b, __shfl_xor_sync(FULLMASK, b, s));
    }
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) sa[warp] = a, sb[warp] = b;
    __syncthreads();
    a = sa[0];
    b = sb[0];
    for (int w = 1; w < kNormThreads / 32; ++w) a += sa[w], b = fmax(b, sb[w]);
}

// q = t / (top / 127) to the nearest even integer, in 64 bits: t * 127 is rounded once and
// the quotient once, so a value on a border falls as the exact quotient does.
__device__ __forceinline__ int quantum(double t, double top) { return (int)rint(t * 127.0 / top); }

// One row per CTA. The row's h stays in shared memory between the sums and the rounding,
// so an output in place of an input is safe.
template <typename T, typename W>
__global__ void __launch_bounds__(kNormThreads) rms_norm_i8_kernel(NormI8Args p) {
    extern __shared__ __align__(16) unsigned char smem[];
    T* keep = reinterpret_cast<T*>(smem);
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
    T* h = p.hidden ? static_cast<T*>(p.hidden) + row * p.hidden_stride : nullptr;
    const W* w = static_cast<const W*>(p.weight);
    double sum = 0.0, top = 0.0;
    bool bad = false;
    for (int i = threadIdx.x; i < p.dim; i += kNormThreads) {
        T v = x[i];
        if (r) v = from_f32<T>(to_f32(v) + to_f32(r[i]));
        if (h) h[i] = v;
        keep[i] = v;
        const double d = to_f32(v), t = d * (double)to_f32(w[i]);
        bad |= !(fabs(t) <= DBL_MAX) || !(fabs(d) <= DBL_MAX);
        sum += d * d;
        top = fmax(top, fabs(t));
    }
    block_sum_max(sum, top);
    bad = __syncthreads_or(bad);
    const double inv = 1.0 / sqrt(sum / p.dim + (double)p.eps);
    if (threadIdx.x == 0) p.scale[row] = bad ? nanf("") : (float)(top / 127.0 * inv);
    int8_t* q = p.q + row * p.q_stride;
    for (int i = threadIdx.x; i < p.dim; i += kNormThreads)
        q[i] = bad || top == 0.0 ? 0 : (int8_t)quantum((double)to_f32(keep[i]) * (double)to_f32(w[i]), top);
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
cudaError_t launch_norm(const NormI8Args& a, cudaStream_t stream) {
    const size_t smem = (size_t)a.dim * sizeof(T);
    static SmemLimit limit;
    cudaError_t e = limit.raise(rms_norm_i8_kernel<T, W>, smem);
    if (e != cudaSuccess) return e;
    rms_norm_i8_kernel<T, W><<<a.rows, kNormThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_norm_w(const NormI8Args& a, cudaStream_t stream) {
    if (a.weight_dtype == VDXS_DTYPE_BF16) return launch_norm<T, __nv_bfloat16>(a, stream);
    if (a.weight_dtype == VDXS_DTYPE_F16) return launch_norm<T, __half>(a, stream);
    return launch_norm<T, float>(a, stream);
}

}  // namespace

cudaError_t rms_norm_i8(const NormI8Args& a, cudaStream_t stream) {
    if (a.dtype == VDXS_DTYPE_BF16) return launch_norm_w<__nv_bfloat16>(a, stream);
    if (a.dtype == VDXS_DTYPE_F16) return launch_norm_w<__half>(a, stream);
    return launch_norm_w<float>(a, stream);
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
