// The norms around a block with its gate and residual scale:
//   h = rs * x + bs * gate * post(y),  z = pre(h).
//
// What bounds it: x, y (and gate) are read and h, z written once, a dozen
// operations an element: HBM for many rows, the chain of load, sums over the
// row and store for few.  So a row stays in registers from its first load to
// its last store, and both norms, the gate and the residual take one kernel:
//   * rows of up to 512 columns belong to a warp each (no barrier), longer ones
//     to a CTA;
//   * few rows: eight elements to a thread, so that many threads share a row;
//   * many rows: 8 or 16 elements, and each CTA takes row after row, the next
//     one's loads under way while it works on this one;
//   * rows past 16384 columns stay in shared memory.
// Elements are read 16 bytes at a time where all rows and vectors allow, else
// in pairs (16384x1100 bf16: 49 us, one by one 71) or one by one, neighbouring
// threads neighbouring elements.  Means and mean
// squares are sums over the values themselves (a layer norm's squares are
// taken after its mean), in a fixed order.
//
// Measured, of 6.53 TB/s: 8192x8192 bf16 90 us (92%), 65536x1024 bf16 85 us
// (97%), 65536x512 bf16 44 us (94%), 4096x8192 FP32 with gate rows 110 us (93%),
// 16384x4093 FP32 with layer norms and a gate row each 259 us (79%: scalar loads,
// four sums over the row), 8192x2999 bf16 83 us (37%: two bytes an access),
// 1x4096 2.6 us.  Rows past 16384 columns, an element an access and a CTA an SM:
// 4096x28672 bf16 440 us (33%), FP32 627 (46%), 2048x49152 657 (19%) and 892 (28%).
#include <mutex>
#include <unordered_map>

#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Eight consecutive elements, 16-byte aligned.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Two, at a multiple of their size.
__device__ __forceinline__ void store2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void store2(__nv_bfloat16* p, float a, float b) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}

constexpr int kRowsPerCta = 8;      // of a warp each

// How rows lie, as far as it holds for all of them and the vectors: elements anywhere, pairs of elements
// at multiples of their size, or eight elements at multiples of 16 bytes.
enum { kAny = 0, kPairs = 1, kEights = 2 };

// Eight elements as they were read: 16-bit ones in pairs or one to a word (kAny).
template <typename T, int V>
struct Raw {
    float w[8];
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = w[j];
    }
};
template <int V>
struct Raw<__nv_bfloat16, V> {
    uint32_t w[V == kAny ? 8 : 4];
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = __uint_as_float(V == kAny ? w[V == kAny ? j : 0] << 16 : (j & 1) ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
    }
};

// EPT elements of a row to each of TH threads (0: as many as the CTA has), eight
// to a block: eight columns in a row (kEights), or pairs or single columns that
// neighbouring threads have next to each other.  With TH known, columns are
// offsets from one address.
template <int V, int EPT, int TH>
struct Row {
    int me, cols;

    __device__ __forceinline__ int threads() const { return TH ? TH : blockDim.x; }
    __device__ __forceinline__ int col(int i, int j) const {
        return V == kEights ? 8 * (me + i * threads()) + j
               : V == kPairs ? 2 * (me + (4 * i + (j >> 1)) * threads()) + (j & 1) : me + (8 * i + j) * threads();
    }
    // Whether all of block i is there: for kEights this thread's, else every thread's but for its last
    // element or pair.
    __device__ __forceinline__ bool full(int i) const {
        return V == kEights ? col(i, 0) + 8 <= cols : V == kPairs ? (8 * i + 6) * threads() <= cols : (8 * i + 7) * threads() <= cols;
    }
    // Whether element j of such a block is there.
    __device__ __forceinline__ bool in(int i, int j) const {
        return V == kEights || j < (V == kPairs ? 6 : 7) || col(i, j) < cols;
    }
    // Block i of a row; columns that are not there give 0.  ALL: but for in().
    template <bool ALL>
    __device__ __forceinline__ bool there(int i, int j) const { return ALL ? in(i, j) : col(i, j) < cols; }
    template <bool ALL>
    __device__ __forceinline__ void read_some(const float* p, int i, Raw<float, V>& r) const {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            if (V == kPairs && there<ALL>(i, j + 1)) {
                const float2 x = *reinterpret_cast<const float2*>(p + col(i, j));
                r.w[j] = x.x;
                r.w[j + 1] = x.y;
            } else {
                r.w[j] = there<ALL>(i, j) ? p[col(i, j)] : 0.0f;
                r.w[j + 1] = V != kPairs && there<ALL>(i, j + 1) ? p[col(i, j + 1)] : 0.0f;
            }
        }
    }
    template <bool ALL>
    __device__ __forceinline__ void read_some(const __nv_bfloat16* p, int i, Raw<__nv_bfloat16, V>& r) const {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
        if constexpr (V == kAny) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r.w[j] = there<ALL>(i, j) ? q[col(i, j)] : 0u;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (V == kPairs && there<ALL>(i, 2 * j + 1)) {
                    r.w[j] = *reinterpret_cast<const uint32_t*>(q + col(i, 2 * j));
                } else {
                    r.w[j] = there<ALL>(i, 2 * j) ? q[col(i, 2 * j)] : 0u;
                    if (V != kPairs && there<ALL>(i, 2 * j + 1)) r.w[j] |= static_cast<uint32_t>(q[col(i, 2 * j + 1)]) << 16;
                }
            }
        }
    }
    __device__ __forceinline__ void read_eight(const float* p, Raw<float, V>& r) const { load8(p, r.w); }
    __device__ __forceinline__ void read_eight(const __nv_bfloat16* p, Raw<__nv_bfloat16, V>& r) const {
        if constexpr (V != kAny) {
            const uint4 x = *reinterpret_cast<const uint4*>(p);
            r.w[0] = x.x; r.w[1] = x.y; r.w[2] = x.z; r.w[3] = x.w;
        }
    }
    template <typename P>
    __device__ __forceinline__ void read(const P* p, int i, Raw<P, V>& r) const {
        if (!full(i)) read_some<false>(p, i, r);
        else if (V == kEights) read_eight(p + col(i, 0), r);
        else read_some<true>(p, i, r);
    }
    template <typename P>
    __device__ __forceinline__ void load(const P* p, int i, float (&v)[8]) const {
        Raw<P, V> r;
        read(p, i, r);
        r.get(v);
    }
    template <bool ALL, typename P>
    __device__ __forceinline__ void store_some(P* p, int i, const float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            if (V == kPairs && there<ALL>(i, j + 1)) {
                store2(p + col(i, j), v[j], v[j + 1]);
            } else {
                if (there<ALL>(i, j)) from_f32(p + col(i, j), v[j]);
                if (V != kPairs && there<ALL>(i, j + 1)) from_f32(p + col(i, j + 1), v[j + 1]);
            }
        }
    }
    template <typename P>
    __device__ __forceinline__ void store(P* p, int i, const float (&v)[8]) const {
        if (!full(i)) store_some<false>(p, i, v);
        else if (V == kEights) store8(p + col(i, 0), v);
        else store_some<true>(p, i, v);
    }
};

// Sum over the row's threads, the same for all of them.  Two buffers in turn:
// a barrier lies between a buffer's reading and its next writing.
template <bool WARP, int TH>
__device__ __forceinline__ float row_sum(float v, float (&part)[2][32], int& buffer) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (!WARP) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) part[buffer][threadIdx.x >> 5] = v;
        __syncthreads();
        if constexpr (TH > 0 && TH % 128 == 0) {    // every thread adds them all: less to wait for than five shuffles
            v = 0.0f;
#pragma unroll
            for (int i = 0; i < TH / 128; ++i) {
                const float4 x = reinterpret_cast<const float4*>(part[buffer])[i];
                v += (x.x + x.y) + (x.z + x.w);
            }
        } else {
            v = lane < static_cast<int>(blockDim.x >> 5) ? part[buffer][lane] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        }
        buffer ^= 1;
    }
    return v;
}

template <typename TW, bool WARP, int V, int EPT, int TH>
__device__ __forceinline__ void norm_row(const Row<V, EPT, TH>& row, float (&v)[EPT / 8][8], int kind, const TW* w, const TW* b,
                                         float eps, float offset, float inv, float (&part)[2][32], int& buffer) {
    constexpr int NB = EPT / 8;
    if (kind == 0) return;
    if (kind == 2) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[i][j];
        const float mean = row_sum<WARP, TH>(s, part, buffer) * inv;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (row.full(i)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = row.in(i, j) ? v[i][j] - mean : 0.0f;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = row.col(i, j) < row.cols ? v[i][j] - mean : 0.0f;
            }
        }
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) q = fmaf(v[i][j], v[i][j], q);
    const float rstd = rsqrtf(row_sum<WARP, TH>(q, part, buffer) * inv + eps);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= rstd;
        if (w) {
            row.load(w, i, t);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= t[j] + offset;
        }
        if (b) {
            row.load(b, i, t);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] += t[j];
        }
    }
}

// Whether 1024 threads an SM (64 registers each) beat fewer with more: not for 16 FP32 elements, which
// would spill (4096x8192 with gate rows: 109 us as it is, 140 so; 8192x8192 bf16 119 and 91).
template <typename T>
constexpr bool tight(int ept) { return ept == 8 || sizeof(T) == 2; }

// STREAM: row after row, gridDim rows apart.
template <typename T, typename TW, int V, int EPT, bool WARP, bool STREAM, int TH>
__global__ void __launch_bounds__(WARP ? 32 * kRowsPerCta : (STREAM ? TH : 1024), STREAM && tight<T>(EPT) ? 1024 / (TH ? TH : 1024) : 1) block_norm_kernel(const BlockNormArgs a) {
    constexpr int NB = EPT / 8;
    __shared__ __align__(16) float part[2][32];
    int buffer = 0;
    pdl_wait();
    pdl_launch_dependents();
    int64_t r = WARP ? static_cast<int64_t>(blockIdx.x) * kRowsPerCta + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? kRowsPerCta : 1);
    if (r >= a.rows) return;
    Row<V, EPT, TH> row;
    row.me = WARP ? threadIdx.x & 31 : threadIdx.x;
    row.cols = a.cols;
    const float inv = 1.0f / static_cast<float>(a.cols);

    Raw<T, V> x[NB], y[NB], g[NB];
    auto read = [&](int64_t at) {
#pragma unroll
        for (int i = 0; i < NB; ++i) row.read(static_cast<const T*>(a.x) + at * a.ldx, i, x[i]);
        if (!a.y) return;
#pragma unroll
        for (int i = 0; i < NB; ++i) row.read(static_cast<const T*>(a.y) + at * a.ldy, i, y[i]);
        if (!a.gate) return;
#pragma unroll
        for (int i = 0; i < NB; ++i) row.read(static_cast<const T*>(a.gate) + at / a.gate_rows * a.ldg, i, g[i]);
    };
    read(r);
    for (;;) {
        float v[NB][8];
        if (a.y) {
            float t[NB][8], u[8];
#pragma unroll
            for (int i = 0; i < NB; ++i) y[i].get(t[i]);
            norm_row<TW, WARP, V, EPT, TH>(row, t, a.post, static_cast<const TW*>(a.post_w), static_cast<const TW*>(a.post_b),
                                         a.eps, a.offset, inv, part, buffer);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                if (a.gate) {
                    g[i].get(u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[i][j] *= u[j];
                }
                x[i].get(v[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = fmaf(a.bs, t[i][j], a.rs * v[i][j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                x[i].get(v[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] *= a.rs;
            }
        }
        const int64_t now = r;
        r += step;
        if (STREAM && r < a.rows) read(r);      // in-place rows are this row's own
        if (a.h) {
#pragma unroll
            for (int i = 0; i < NB; ++i) row.store(static_cast<T*>(a.h) + now * a.ldh, i, v[i]);
        }
        if (a.z) {
            norm_row<TW, WARP, V, EPT, TH>(row, v, a.pre, static_cast<const TW*>(a.pre_w), static_cast<const TW*>(a.pre_b), a.eps,
                                         a.offset, inv, part, buffer);
#pragma unroll
            for (int i = 0; i < NB; ++i) row.store(static_cast<T*>(a.z) + now * a.ldz, i, v[i]);
        }
        if (!STREAM || r >= a.rows) return;
    }
}

// ---- rows that fill no CTA's registers: FP32 values in shared memory ----------
constexpr int kLongThreads = 1024;

__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[kLongThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
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
        for (int c = threadIdx.x; c < cols; c += kLongThreads) s += v[c];
        *mean = block_sum(s) * inv;
    }
    float q = 0.0f;
    for (int c = threadIdx.x; c < cols; c += kLongThreads) { const float t = v[c] - *mean; q = fmaf(t, t, q); }
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
__global__ void __launch_bounds__(kLongThreads) block_norm_long_kernel(const BlockNormArgs a) {
    extern __shared__ float row[];
    pdl_wait();
    pdl_launch_dependents();
    const int64_t r = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    float mean, rstd;
    if (a.y) {
        const T* y = static_cast<const T*>(a.y) + r * a.ldy;
        for (int c = threadIdx.x; c < a.cols; c += kLongThreads) row[c] = to_f32(y[c]);
        row_stats(row, a.cols, a.post, a.eps, &mean, &rstd);
    }
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + r / a.gate_rows * a.ldg : nullptr;
    for (int c = threadIdx.x; c < a.cols; c += kLongThreads) {
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
    for (int c = threadIdx.x; c < a.cols; c += kLongThreads) {
        float v = row[c];
        if (a.pre != 0)
            v = apply(v, c, mean, rstd, static_cast<const TW*>(a.pre_w), static_cast<const TW*>(a.pre_b), a.offset);
        from_f32(static_cast<T*>(a.z) + r * a.ldz + c, v);
    }
}

template <typename K>
cudaError_t launch_pdl(K fn, int64_t grid, int threads, size_t smem, const BlockNormArgs& a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, a);
}

// Resident CTAs per SM, asked once per kernel, size of CTA and device.
cudaError_t resident(const void* fn, int threads, int* ctas) {
    static std::mutex mu;
    static std::unordered_map<const void*, int> known[64][17];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    int& n = known[dev][threads / 32][fn];
    if (n == 0) {
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, threads, 0);
        if (e != cudaSuccess) return e;
        if (n < 1) return cudaErrorLaunchOutOfResources;
    }
    *ctas = n;
    return cudaSuccess;
}

template <typename T, typename TW, int V, int EPT, int TH>
cudaError_t launch_stream(const BlockNormArgs& a, int num_sms, cudaStream_t s) {
    int ctas = 0;
    cudaError_t e = resident(reinterpret_cast<const void*>(&block_norm_kernel<T, TW, V, EPT, false, true, TH>), TH, &ctas);
    if (e != cudaSuccess) return e;
    const int64_t most = static_cast<int64_t>(ctas) * num_sms;
    return launch_pdl(block_norm_kernel<T, TW, V, EPT, false, true, TH>, a.rows < most ? a.rows : most, TH, 0, a, s);
}

template <typename T, typename TW, int V>
cudaError_t launch_short(const BlockNormArgs& a, int num_sms, cudaStream_t s) {
    // 65536x512 bf16: 44 us, a CTA to each row 97; rows of 1024 take 105 us this way and 85 the other.
    // (Row after row, as below, took 55 for 65536x512: here the other warps' rows hide a row's chain.)
    if (a.cols <= 512) {
        const int64_t grid = (static_cast<int64_t>(a.rows) + kRowsPerCta - 1) / kRowsPerCta;
        return a.cols <= 256 ? launch_pdl(block_norm_kernel<T, TW, V, 8, true, false, 32>, grid, 32 * kRowsPerCta, 0, a, s)
                             : launch_pdl(block_norm_kernel<T, TW, V, 16, true, false, 32>, grid, 32 * kRowsPerCta, 0, a, s);
    }
    auto threads = [&](int ept) { return ((a.cols + ept - 1) / ept + 31) / 32 * 32; };
    if (a.cols <= 8192) {
        // Row after row pays from two (longer rows) or four rows an SM on: 8192x8192 bf16 90 us, a CTA to
        // each row 114; 2400x4096 17.1 and 18.5, but 600x1024 3.1 and 2.7.
        if (a.rows > (a.cols > 4096 ? 2 : 4) * num_sms) {
            // Element by element, half as many to a thread hide more of each other's latency
            // (16384x4093 FP32: 262 against 288 us); 16 bytes at a time it is the other way round
            // (4096x4096 bf16: 32 against 27 us) but for short rows (16384x600 FP32: 30 against 36).
            // As few threads as hold a row: 8192x5120 bf16 71 us, with 512 threads 96.
            constexpr int EPT = V == kEights ? 16 : 8;
            const int need = (a.cols + EPT - 1) / EPT;
            if (a.cols > 4096)
                return a.cols <= 6144 ? launch_stream<T, TW, V, 16, 384>(a, num_sms, s) : launch_stream<T, TW, V, 16, 512>(a, num_sms, s);
            if (a.cols <= 768) return launch_stream<T, TW, V, 8, 96>(a, num_sms, s);
            if (need <= 64) return launch_stream<T, TW, V, EPT, 64>(a, num_sms, s);
            if (need <= 96) return launch_stream<T, TW, V, EPT, 96>(a, num_sms, s);
            if (need <= 128) return launch_stream<T, TW, V, EPT, 128>(a, num_sms, s);
            if (need <= 192) return launch_stream<T, TW, V, EPT, 192>(a, num_sms, s);
            if (EPT == 16 || need <= 256) return launch_stream<T, TW, V, EPT, 256>(a, num_sms, s);
            if (need <= 384) return launch_stream<T, TW, V, EPT, EPT == 16 ? 256 : 384>(a, num_sms, s);
            return launch_stream<T, TW, V, EPT, EPT == 16 ? 256 : 512>(a, num_sms, s);
        }
        return launch_pdl(block_norm_kernel<T, TW, V, 8, false, false, 0>, a.rows, threads(8), 0, a, s);
    }
    return launch_pdl(block_norm_kernel<T, TW, V, 16, false, false, 0>, a.rows, threads(16), 0, a, s);
}

template <typename T, typename TW>
cudaError_t launch(const BlockNormArgs& a, int num_sms, cudaStream_t s) {
    if (a.cols > 16384) {
        const void* fn = reinterpret_cast<const void*>(&block_norm_long_kernel<T, TW>);
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kBlockNormMaxCols * 4);
        if (e != cudaSuccess) return e;
        return launch_pdl(block_norm_long_kernel<T, TW>, a.rows, kLongThreads, static_cast<size_t>(a.cols) * 4, a, s);
    }
    // The elements that all addresses and pitches are a multiple of.
    const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.gate) |
                           reinterpret_cast<uintptr_t>(a.h) | reinterpret_cast<uintptr_t>(a.z);
    const uintptr_t vectors = reinterpret_cast<uintptr_t>(a.post_w) | reinterpret_cast<uintptr_t>(a.post_b) |
                              reinterpret_cast<uintptr_t>(a.pre_w) | reinterpret_cast<uintptr_t>(a.pre_b);
    const int64_t pitch = a.ldx | (a.y ? a.ldy : 0) | (a.gate ? a.ldg : 0) | (a.h ? a.ldh : 0) | (a.z ? a.ldz : 0);
    const uintptr_t bytes = ptrs | static_cast<uintptr_t>(pitch * static_cast<int64_t>(sizeof(T)));
    if (bytes % 16 == 0 && vectors % 16 == 0) return launch_short<T, TW, kEights>(a, num_sms, s);
    if (bytes % (2 * sizeof(T)) == 0 && vectors % (2 * sizeof(TW)) == 0) return launch_short<T, TW, kPairs>(a, num_sms, s);
    return launch_short<T, TW, kAny>(a, num_sms, s);
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormArgs& a, int num_sms, cudaStream_t s) {
    if (a.io == DType::F32)
        return a.wt == DType::F32 ? launch<float, float>(a, num_sms, s) : launch<float, __nv_bfloat16>(a, num_sms, s);
    return a.wt == DType::F32 ? launch<__nv_bfloat16, float>(a, num_sms, s)
                              : launch<__nv_bfloat16, __nv_bfloat16>(a, num_sms, s);
}

}  // namespace dnnopt_b200
