// Attention of one new token per sequence over a paged key-value cache.
//
// One CTA per (query head, sequence).  Each of its warps walks every fourth
// token with an online softmax: a running maximum m and sum l, and the
// weighted sum of values rescaled by exp(m_old - m_new) when the maximum moves.
// The warps' (m, l, sum) are joined in shared memory in warp order.
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxDim = 256;

template <DType T> struct Store;
template <> struct Store<DType::F32> {
    using S = float;
    static __device__ __forceinline__ float get(S v) { return v; }
    static __device__ __forceinline__ S put(float v) { return v; }
};
template <> struct Store<DType::BF16> {
    using S = __nv_bfloat16;
    static __device__ __forceinline__ float get(S v) { return __bfloat162float(v); }
    static __device__ __forceinline__ S put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Store<DType::E4M3> {
    using S = __nv_fp8_storage_t;
    static __device__ __forceinline__ float get(S v) { return e4m3x2_to_f32x2(v).x; }
    static __device__ __forceinline__ S put(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
};

template <DType IO, DType CT>
__global__ void __launch_bounds__(kWarps * 32) paged_attention_row_kernel(PagedAttnArgs a) {
    using I = Store<IO>;
    using C = Store<CT>;
    __shared__ float s_acc[kWarps][kMaxDim], s_m[kWarps], s_l[kWarps];
    const int head = blockIdx.x, b = blockIdx.y, group = a.heads / a.kv_heads, kvh = head / group;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int len = a.lens[b];
    const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page_size;
    if (len < 0 || len > cap) {
        if (threadIdx.x == 0) record_kernel_error(a.err, kKerrBadIndex);
        len = 0;
    }
    const int first = a.window > 0 && len > a.window ? len - a.window : 0;
    float q[8], acc[8];
    const typename I::S* qp = static_cast<const typename I::S*>(a.q) + b * a.q_batch + head * a.q_head;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < a.dim ? I::get(qp[d]) : 0.0f;
        acc[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = first + warp; j < len; j += kWarps) {
        const int page = a.table[b * a.table_stride + j / a.page_size];
        if (page < 0 || page >= a.num_pages) {
            if (lane == 0) record_kernel_error(a.err, kKerrBadIndex);
            continue;
        }
        const int64_t off = page * a.page_stride + j % a.page_size * a.token_stride + kvh * a.head_stride;
        typename C::S* kp = static_cast<typename C::S*>(a.k) + off;
        typename C::S* vp = static_cast<typename C::S*>(a.v) + off;
        const bool fresh = a.k_new && j == len - 1;
        const int64_t at = b * a.new_batch + kvh * a.new_head;
        float k[8], v[8], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d >= a.dim) { k[i] = v[i] = 0.0f; continue; }
            if (fresh) {
                const typename C::S ks = C::put(I::get(static_cast<const typename I::S*>(a.k_new)[at + d]) / a.k_scale);
                const typename C::S vs = C::put(I::get(static_cast<const typename I::S*>(a.v_new)[at + d]) / a.v_scale);
                k[i] = C::get(ks);
                v[i] = C::get(vs);
                if (head % group == 0) { kp[d] = ks; vp[d] = vs; }
            } else {
                k[i] = C::get(kp[d]);
                v[i] = C::get(vp[d]);
            }
            dot = fmaf(q[i], k[i], dot);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
        float s = dot * a.scale * a.k_scale;
        if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
        const float m2 = fmaxf(m, s), keep = m == -INFINITY ? 0.0f : expf(m - m2);
        const float p = m2 == -INFINITY ? 0.0f : expf(s - m2);
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fmaf(p, v[i], acc[i] * keep);
        m = m2;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s_acc[warp][lane + 32 * i] = acc[i];
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
    float f[kWarps];
    for (int w = 0; w < kWarps; ++w) {
        f[w] = s_m[w] == -INFINITY ? 0.0f : expf(s_m[w] - M);
        L += f[w] * s_l[w];
    }
    typename I::S* op = static_cast<typename I::S*>(a.out) + b * a.out_batch + head * a.out_head;
    for (int d = threadIdx.x; d < a.dim; d += kWarps * 32) {
        float o = 0.0f;
        for (int w = 0; w < kWarps; ++w) o += f[w] * s_acc[w][d];
        op[d] = I::put(L == 0.0f ? 0.0f : o * a.v_scale / L);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[static_cast<int64_t>(b) * a.heads + head] = L == 0.0f ? -INFINITY : M + logf(L);
}

}  // namespace

cudaError_t launch_paged_attention(const PagedAttnArgs& a, cudaStream_t s) {
    dim3 grid(a.heads, a.batch);
    if (a.ct == DType::F32) paged_attention_row_kernel<DType::F32, DType::F32><<<grid, kWarps * 32, 0, s>>>(a);
    else if (a.ct == DType::BF16) paged_attention_row_kernel<DType::BF16, DType::BF16><<<grid, kWarps * 32, 0, s>>>(a);
    else paged_attention_row_kernel<DType::BF16, DType::E4M3><<<grid, kWarps * 32, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace dnnopt_b200
