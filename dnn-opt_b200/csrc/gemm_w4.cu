// Products of few rows with 4-bit weights and group scales:
//   C[m,n] = bias[n] + sum_k A[m,k] * scale[n,k/g] * (code[n,k] - zero[n,k/g]).
//
// gemm_w4_rows_kernel, for every layout: a warp owns one row n of W and up to
// eight rows of A, its lanes walk the row's bytes 32 at a time and each keeps
// eight FP32 sums, reduced over the lanes at the end.
#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

constexpr int kRowsMT = 8;       // rows of A per pass
constexpr int kRowsWarps = 8;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename TA, typename TS>
__global__ void __launch_bounds__(kRowsWarps * 32) gemm_w4_rows_kernel(W4Args g) {
    const int lane = threadIdx.x & 31;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * kRowsWarps + (threadIdx.x >> 5);
    if (n >= g.N) return;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kRowsMT;
    const int mt = g.M - m0 < kRowsMT ? static_cast<int>(g.M - m0) : kRowsMT;
    const TA* A = static_cast<const TA*>(g.A) + m0 * g.lda;
    const uint8_t* w = g.W + n * g.ldw;
    const TS* scale = static_cast<const TS*>(g.scale) + n * g.lds;
    const TS* zero = g.zero ? static_cast<const TS*>(g.zero) + n * g.lds : nullptr;
    float acc[kRowsMT] = {};
    const int bytes = (g.K + 1) / 2;
    for (int b = lane; b < bytes; b += 32) {
        const int k = 2 * b, gi = k / g.group;
        const float sc = to_f32(scale[gi]), z = zero ? to_f32(zero[gi]) : 8.0f;
        const uint32_t c = w[b];
        const bool two = k + 1 < g.K;
        const float lo = sc * (static_cast<float>(c & 15u) - z);
        const float hi = two ? sc * (static_cast<float>(c >> 4) - z) : 0.0f;
#pragma unroll
        for (int m = 0; m < kRowsMT; ++m) {
            if (m >= mt) break;
            const TA* a = A + m * g.lda + k;
            acc[m] = fmaf(to_f32(a[0]), lo, acc[m]);
            if (two) acc[m] = fmaf(to_f32(a[1]), hi, acc[m]);
        }
    }
#pragma unroll
    for (int m = 0; m < kRowsMT; ++m) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xFFFFFFFFu, acc[m], o);
        if (lane == 0 && m < mt)
            from_f32(static_cast<TA*>(g.C) + (m0 + m) * g.ldc + n, acc[m] + (g.bias ? g.bias[n] : 0.0f));
    }
}

template <typename TA, typename TS>
cudaError_t launch_rows(const W4Args& g, cudaStream_t s) {
    dim3 grid((g.N + kRowsWarps - 1) / kRowsWarps, (g.M + kRowsMT - 1) / kRowsMT);
    gemm_w4_rows_kernel<TA, TS><<<grid, kRowsWarps * 32, 0, s>>>(g);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gemm_w4(const W4Args& g, cudaStream_t s) {
    if (g.io == DType::F32)
        return g.st == DType::F32 ? launch_rows<float, float>(g, s) : launch_rows<float, __nv_bfloat16>(g, s);
    return g.st == DType::F32 ? launch_rows<__nv_bfloat16, float>(g, s)
                              : launch_rows<__nv_bfloat16, __nv_bfloat16>(g, s);
}

}  // namespace dnnopt_b200
