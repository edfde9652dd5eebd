// The norms around a block with its gate and residual scale:
//   h = rs * x + bs * gate * post(y),  z = pre(h).
//
// One CTA per row keeps the row's FP32 values in shared memory.
#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) v += part[i];
    return v;
}

// Mean and 1 / sqrt(mean square + eps) of the row in `v`.
__device__ __forceinline__ void row_stats(const float* v, int cols, int kind, float eps, float* mean, float* rstd) {
    *mean = 0.0f;
    *rstd = 1.0f;
    if (kind == 0) return;
    const float inv = 1.0f / static_cast<float>(cols);
    if (kind == 2) {
        float s = 0.0f;
        for (int c = threadIdx.x; c < cols; c += kThreads) s += v[c];
        *mean = block_sum(s) * inv;
    }
    float q = 0.0f;
    for (int c = threadIdx.x; c < cols; c += kThreads) { const float t = v[c] - *mean; q = fmaf(t, t, q); }
    *rstd = rsqrtf(block_sum(q) * inv + eps);
}

template <typename TW>
__device__ __forceinline__ float apply(float v, int c, float mean, float rstd, const TW* w, const TW* b, float off) {
    v = (v - mean) * rstd;
    if (w) v *= to_f32(w[c]) + off;
    if (b) v += to_f32(b[c]);
    return v;
}

template <typename T, typename TW>
__global__ void __launch_bounds__(kThreads) block_norm_row_kernel(BlockNormArgs a) {
    extern __shared__ float row[];
    const int64_t r = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    float mean, rstd;
    if (a.y) {
        const T* y = static_cast<const T*>(a.y) + r * a.ldy;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) row[c] = to_f32(y[c]);
        row_stats(row, a.cols, a.post, a.eps, &mean, &rstd);
    }
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + r / a.gate_rows * a.ldg : nullptr;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
        float v = a.rs * to_f32(x[c]);
        if (a.y) {
            float t = row[c];
            if (a.post != 0)
                t = apply(t, c, mean, rstd, static_cast<const TW*>(a.post_w), static_cast<const TW*>(a.post_b), a.offset);
            if (gate) t *= to_f32(gate[c]);
            v = fmaf(a.bs, t, v);
        }
        row[c] = v;
        if (a.h) from_f32(static_cast<T*>(a.h) + r * a.ldh + c, v);
    }
    if (!a.z) return;
    row_stats(row, a.cols, a.pre, a.eps, &mean, &rstd);
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
        float v = row[c];
        if (a.pre != 0)
            v = apply(v, c, mean, rstd, static_cast<const TW*>(a.pre_w), static_cast<const TW*>(a.pre_b), a.offset);
        from_f32(static_cast<T*>(a.z) + r * a.ldz + c, v);
    }
}

template <typename T, typename TW>
cudaError_t launch_row(const BlockNormArgs& a, cudaStream_t s) {
    const void* fn = reinterpret_cast<const void*>(&block_norm_row_kernel<T, TW>);
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kBlockNormMaxCols * 4);
    if (e != cudaSuccess) return e;
    block_norm_row_kernel<T, TW><<<a.rows, kThreads, static_cast<size_t>(a.cols) * 4, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormArgs& a, cudaStream_t s) {
    if (a.io == DType::F32)
        return a.wt == DType::F32 ? launch_row<float, float>(a, s) : launch_row<float, __nv_bfloat16>(a, s);
    return a.wt == DType::F32 ? launch_row<__nv_bfloat16, float>(a, s)
                              : launch_row<__nv_bfloat16, __nv_bfloat16>(a, s);
}

}  // namespace dnnopt_b200
