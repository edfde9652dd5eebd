// Products of few rows with 4-bit weights and group scales:
//   C[m,n] = bias[n] + sum_k A[m,k] * scale[n,k/g] * (code[n,k] - zero[n,k/g]).
//
// What bounds it: a weight is half a byte and used M times, so HBM up to
// M of about 64; below that, turning codes into operands is the work, on the
// pipe that shifts and masks 16 lanes a cycle.  The products are therefore
// integer ones of bytes: the eight codes of a word become two operand words in
// three operations (a code to bf16 takes one for each and held this kernel at
// 2.1 TB/s).  Rows of W are the rows, digits of the activations the columns.
// Two kernels: mma.sync m16n8k32 out of registers, and for long products with
// three rows of A or more tcgen05 out of tensor memory (further down).
//
// Mathematics.  Within 128 consecutive k, a row of A is a power of two times
// whole numbers |i| < 2^22 (bf16) or 2^30 (FP32), the power chosen by the
// largest of the 128, and i = sum_d 256^d i_d with signed bytes i_d.  The sums
// sum_k (code - 8) i_d are exact in 32-bit integers: they start from -8 sum i_d
// and the bits of 1.5 * 2^23, so that they come out as FP32 numbers.  Then, in
// FP32, once for every group or 128 weights:
//   scale sum (code - zero) a = 2^e (scale (sum_d 256^d sum (code - 8) i_d - (zero - 8) sum i)),
// multiplied in this order: nothing on the way is below FP32's normal numbers
// where the result is not.
// What is rounded are activations below 2^-14 (bf16; 2^-6, FP32) of the largest
// of their 128, by up to 2^-22 (2^-30) of it.  That is below what an FP32 sum of
// the 128 rounds, unless scales differ within them by as much as the activations.
// Activations that are infinite or NaN stay out of the products and are added
// for their own row at the end.
//
// Work.  128 weights of 32 rows (2 KB) are a step, a TMA box into the ring of the
// warp that works on it (16-byte cp.async of the same rows cost 23 shared-memory
// cycles an instruction and held the kernel at 1.6 TB/s).  All steps, tile after
// tile of 32 rows, are cut into equal shares, one for each team of four warps, four
// teams to an SM; a team's warps take the steps of a tile in turn and add up
// in shared memory.  A tile cut by a share's end, or by the ends of a K-range, is
// finished by the last of its shares to arrive, adding the parts in order.  The
// digits of the K-range sit in shared memory in the order in which the operand
// reads them.  Rows of W that do not start at multiples of 16 bytes are first
// copied to a workspace where they do: 8x28672x8189 with dense rows 78 us, with
// rows at 16 bytes 38; one row 69 and 30.
//
// Measured, of 6.53 TB/s (bf16, groups of 128): 1x28672x8192 30.0 us (62%); groups
// of 32, 8 rows 63 us; 4x11008x4096 in groups of 64 with zero points 22.5 us;
// 1x4096x4096 9.0 us, of which the chain of start, digits, first weights, sums
// and joining takes seven.  16 warps an SM issue two instructions a cycle of
// four: decoding, products and scaling wait on one another's results, and
// registers allow no more warps.
#include <cuda.h>

#include <mutex>
#include <type_traits>
#include <unordered_set>

#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

constexpr int kTeams = 4;           // per CTA
constexpr int kTeamThreads = 128;
constexpr int kWarps = 4;           // per team
constexpr int kMaxSlots = 4;        // steps under way per warp, where the activations leave room
constexpr int kMinSlots = 2;
constexpr int kStepK = 128;
constexpr int kRows = 32;           // of W in a tile: two blocks of 16
constexpr int kStepBytes = kRows * kStepK / 2;
constexpr int kMaxSmem = 227 * 1024;
constexpr int kTcRows = 128;        // of W in a tile of the tensor-memory kernel
constexpr int kTcStepBytes = kTcRows * kStepK / 2;
constexpr int kTcColumns = 128;     // of tensor memory for each of its teams
constexpr int kTcThreads = kTeams * kTeamThreads + kTeams * 32;

struct Params {
    W4Args g;
    int tiles;                      // of 32 rows of W
    int steps;                      // ceil(K / 128)
    int split_steps;                // steps of one K-range (gridDim.y of them)
    int slots;                      // of a warp's ring
    int rows, cols;                 // rows of A at a time, and columns: a digit of each
    int bars_at;                    // of the barriers, in shared memory
    uint32_t image_bytes;           // of a K-range's activations
    unsigned char* images;          // made by the kernel before; nullptr: each CTA makes its own
    uint8_t* copy;                  // of W, made by the kernel before; nullptr: W is read as it is
    int64_t copy_pitch;
    uint32_t digit_ctas;            // of that kernel's grid in x; the rest copy
    uint32_t gmul, gshift;          // chunk of 32 weights -> group
    float* ws;                      // partial tiles of a K-range: the part with a tile's first step by
                                    // tile, then the parts that begin a share by share
    uint32_t* tickets;              // one per tile and block of rows of A
    uint32_t* err;                  // receives kKerrMbarTimeout
};

__device__ __forceinline__ void mma_u8s8(uint32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
// A scale as it lies in memory: 32 bits, or 16 in the low half.
__device__ __forceinline__ uint32_t ldg_scale(const char* p, bool f32) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t@p ld.global.nc.u32 %0, [%1];\n\t@!p ld.global.nc.u16 %0, [%1];\n\t}"
                 : "=r"(v) : "l"(p), "r"(static_cast<int>(f32)));
    return v;
}
// Two FP32 operations in one instruction.
__device__ __forceinline__ unsigned long long as64(float2 v) {
    unsigned long long r;
    asm("mov.b64 %0, {%1,%2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 as_pair(unsigned long long r) {
    float2 v;
    asm("mov.b64 {%0,%1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(as64(a)), "l"(as64(b)), "l"(as64(c)));
    return as_pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as64(a)), "l"(as64(b)));
    return as_pair(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as64(a)), "l"(as64(b)));
    return as_pair(r);
}
__device__ __forceinline__ float2 bits2(const uint32_t* c) { return make_float2(__uint_as_float(c[0]), __uint_as_float(c[1])); }
constexpr float kMagic = 12582912.0f;           // 1.5 * 2^23: whole numbers below 2^22 added to it keep their bits
constexpr uint32_t kMagicBits = 0x4B400000u;

// Equal shares of all steps but for one step, at least one step for each warp
// of a team: the first `more` shares have one more than the others.  Where every
// tile finds a team of its own and has at most four steps for each of its warps,
// the shares are the tiles: adding up parts would take longer than two steps
// (1x4096x2048 5.2 us, in equal shares 6.7; 1x1024x1024 4.2 and 5.8).
struct Shares {
    uint32_t n, each, more;

    __device__ Shares(uint32_t tiles, uint32_t per_tile, uint32_t most, uint32_t warps) {
        const uint32_t steps = tiles * per_tile;
        n = tiles <= most && per_tile <= 4 * warps ? tiles : min(steps / warps, most);
        if (n < 1) n = 1;
        each = steps / n;
        more = steps - each * n;
    }
    __device__ __forceinline__ uint32_t start(uint32_t s) const { return s * each + min(s, more); }
    // The share that holds step t: the last one that starts at or before it.
    __device__ __forceinline__ uint32_t holder(uint32_t t) const {
        const uint32_t big = more * (each + 1);
        return t < big ? t / (each + 1) : more + (t - big) / each;
    }
};

// One warp's steps of a share: every fourth of each tile's.
struct Cursor {
    uint32_t tile, q, end, left;    // step q of [.., end) of the tile; steps of the share after it

    __device__ Cursor(uint32_t lo, uint32_t hi, uint32_t per_tile, int warp) {
        tile = lo / per_tile;
        const uint32_t q0 = lo - tile * per_tile;
        const uint32_t n = hi - lo < per_tile - q0 ? hi - lo : per_tile - q0;
        end = q0 + n;
        left = hi - lo - n;
        q = q0 + warp;
        settle(per_tile, warp);
    }
    __device__ __forceinline__ void settle(uint32_t per_tile, int warp) {
        while (q >= end && left > 0) {
            ++tile;
            end = left < per_tile ? left : per_tile;
            left -= end;
            q = warp;
        }
    }
};

// The activations of a K-range as the products read them.
struct Image {
    unsigned char* act;     // [step][2][col][t] 16 bytes: the digits of two words' activations
    uint32_t* base;         // [step][flush][col]: -8 times the sum of the digits, as the bits of an FP32 number
    float* unit;            // [step][tcol]: what 1 stands for; negative where an infinity or NaN was left out
    float* isum;            // [step][flush][tcol]: the sum of the whole numbers (packed: of the digits)

    __device__ Image(unsigned char* at, uint32_t steps, int cols, int tcols, int f) : act(at) {
        base = reinterpret_cast<uint32_t*>(act + static_cast<size_t>(steps) * cols * 128);
        unit = reinterpret_cast<float*>(base + steps * (4 / f) * cols);
        isum = unit + steps * tcols;
    }
};

// 128 activations of row m0 + m, eight (a word's worth) to each lane of half a
// warp: r is the lane's place, q the stretch within the K-range, `in` false for
// a half that has nothing to do.  The whole warp takes part.
template <DType IO, bool PACKED, int F, bool TC>
__device__ __forceinline__ void stage(const Params& p, const Image& img, int m0, int k_step0, uint32_t m, uint32_t q, uint32_t r,
                                      bool vec, bool in) {
    using T = typename std::conditional<IO == DType::F32, float, __nv_bfloat16>::type;
    constexpr bool PARTS = IO == DType::F32;
    constexpr int D = PARTS ? 4 : 3, BITS = PARTS ? 30 : 22;
    const W4Args& g = p.g;
    const int tcols = PACKED ? p.cols : p.rows;
    // Which word of which lane these eight weights are, after the exchanges of the product's loop.
    const uint32_t w = F == 4 ? (r & 3) : (F == 1 ? (r >> 2) : ((r >> 3) * 2 + (r & 1)));
    const uint32_t t = F == 4 ? (r >> 2) : (F == 1 ? (r & 3) : (((r >> 2) & 1) + (r & 2)));
    const int64_t k = static_cast<int64_t>(k_step0) * kStepK + q * 128 + r * 8;
    const T* a = static_cast<const T*>(g.A) + static_cast<int64_t>(m0 + m) * g.lda + k;
    float v[8] = {};
    if (in) {
        if (vec && k + 8 <= g.K) {
            if constexpr (PARTS) {
                const float4 x = __ldg(reinterpret_cast<const float4*>(a)), y = __ldg(reinterpret_cast<const float4*>(a) + 1);
                v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
            } else {
                const uint4 y = __ldg(reinterpret_cast<const uint4*>(a));
                const uint32_t x[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = __uint_as_float(x[i] << 16);
                    v[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < g.K ? static_cast<float>(a[i]) : 0.0f;
        }
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    bool bad = top > 3.402823466e38f;
#pragma unroll
    for (int i = 0; i < 8; ++i) bad = bad || v[i] != v[i];
    if (bad) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!(fabsf(v[i]) <= 3.402823466e38f)) v[i] = 0.0f;
            top = fmaxf(top, fabsf(v[i]));
        }
    }
    const bool odd = (__ballot_sync(0xFFFFFFFFu, bad) >> (threadIdx.x & 16)) & 0xFFFFu;
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
    // 2^e is above every |v|; the unit 2^(e - BITS) stays a normal number.
    int e = static_cast<int>(__float_as_uint(top) >> 23) - 126;
    e = max(e, BITS - 126);
    const float scale = __uint_as_float(static_cast<uint32_t>(127 + BITS - e) << 23);
    uint32_t x[8];
    if constexpr (PARTS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<uint32_t>(__float2int_rn(v[i] * scale)) + 0x80808080u;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)     // every digit plus 128
            x[i] = __float_as_uint(fmaf(v[i], scale, kMagic)) - kMagicBits + 0x00808080u;
    }
    // Even k are the low nibbles, the first operand register; odd k the second.
    uint2 o[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t p0 = __byte_perm(x[h], x[h + 2], 0x5140), p1 = __byte_perm(x[h + 4], x[h + 6], 0x5140);
        const uint32_t p2 = __byte_perm(x[h], x[h + 2], 0x7362), p3 = __byte_perm(x[h + 4], x[h + 6], 0x7362);
        const uint32_t d0 = __byte_perm(p0, p1, 0x5410) ^ 0x80808080u, d1 = __byte_perm(p0, p1, 0x7632) ^ 0x80808080u;
        const uint32_t d2 = __byte_perm(p2, p3, 0x5410) ^ 0x80808080u, d3 = __byte_perm(p2, p3, 0x7632) ^ 0x80808080u;
        (h ? o[0].y : o[0].x) = d0;
        (h ? o[1].y : o[1].x) = d1;
        (h ? o[2].y : o[2].x) = d2;
        (h ? o[3].y : o[3].x) = d3;
    }
    // Sums of the digits, two to a word: each stays within 16 bits.
    int pair[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int lo = __dp4a(static_cast<int>(o[2 * h].x), 0x01010101, __dp4a(static_cast<int>(o[2 * h].y), 0x01010101, 0));
        const int up = __dp4a(static_cast<int>(o[2 * h + 1].x), 0x01010101, __dp4a(static_cast<int>(o[2 * h + 1].y), 0x01010101, 0));
        pair[h] = lo + up * 65536;
        if (2 * h + 1 >= D) pair[h] = lo;
#pragma unroll
        for (int s = 1; s < 4 * F; s <<= 1) pair[h] += __shfl_xor_sync(0xFFFFFFFFu, pair[h], s);
    }
    if (in) {
        if constexpr (TC) {     // a digit's column is a row of 128 bytes, even k before odd k within each eight
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const uint32_t n = d * p.rows + m;
                *reinterpret_cast<uint2*>(img.act + q * (p.cols * 128) + n * 128 + (((r >> 1) ^ (n & 7)) << 4) + (r & 1) * 8) = o[d];
            }
        } else {
            unsigned char* dst = img.act + ((q * 2 + (w >> 1)) * p.cols + m) * 64 + t * 16 + (w & 1) * 8;
#pragma unroll
            for (int d = 0; d < D; ++d) *reinterpret_cast<uint2*>(dst + d * p.rows * 64) = o[d];
        }
        const float u1 = __uint_as_float((static_cast<uint32_t>(127 + e - BITS) << 23) | (odd ? 0x80000000u : 0u));
        if (r == 0) {
#pragma unroll
            for (int d = 0; d < (PACKED ? D : 1); ++d)      // packed: digit d has a column of its own, worth 256^d
                img.unit[q * tcols + d * p.rows + m] = u1 * static_cast<float>(1u << (8 * d));
        }
        if ((r & (4 * F - 1)) == 0) {
            const uint32_t at = q * (4 / F) + r / (4 * F);
            float sum = 0.0f;
#pragma unroll
            for (int d = D - 1; d >= 0; --d) {
                const int lo = static_cast<int16_t>(pair[d / 2] & 0xFFFF);
                const int digits = d % 2 ? (pair[d / 2] - lo) >> 16 : (d == 2 && D == 3 ? pair[1] : lo);
                img.base[at * p.cols + d * p.rows + m] = kMagicBits - static_cast<uint32_t>(8 * digits);
                if constexpr (PACKED) img.isum[at * tcols + d * p.rows + m] = static_cast<float>(digits);
                sum = fmaf(sum, 256.0f, static_cast<float>(digits));
            }
            if constexpr (!PACKED) img.isum[at * tcols + m] = sum;
        }
    }
}

// A row of W at a multiple of 16 bytes: a warp copies its words of four bytes, each cut from the two
// aligned words that hold it.
__device__ __forceinline__ void copy_row(const Params& p, int64_t n) {
    const W4Args& g = p.g;
    if (n >= g.N) return;
    const int bytes = (g.K >> 1) + (g.K & 1);
    const uintptr_t row = reinterpret_cast<uintptr_t>(g.W) + n * g.ldw, end = row + bytes;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(row & ~uintptr_t(3));
    const uint32_t shift = static_cast<uint32_t>(row & 3) * 8;
    for (int i = threadIdx.x & 31; i < (bytes + 3) / 4; i += 32) {
        const uint32_t lo = __ldg(from + i);
        const uint32_t hi = shift && reinterpret_cast<uintptr_t>(from + i + 1) < end ? __ldg(from + i + 1) : 0u;
        *reinterpret_cast<uint32_t*>(p.copy + n * p.copy_pitch + i * 4) = __funnelshift_r(lo, hi, shift);
    }
}

// What a product wants made before it.  Images of all K-ranges and blocks of rows, where making them in
// every CTA takes longer than reading them back: a half-warp per 128 activations.  And the rows of W at
// multiples of 16 bytes, if they are not there: a warp to a row.
template <DType IO, bool PACKED, int F, bool TC>
__global__ void __launch_bounds__(128) gemm_w4_digits_kernel(const Params p) {
    pdl_wait();
    pdl_launch_dependents();    // what runs next finds everything older than this kernel done
    if (blockIdx.x >= p.digit_ctas) {
        if (blockIdx.y == 0 && blockIdx.z == 0) copy_row(p, static_cast<int64_t>(blockIdx.x - p.digit_ctas) * 4 + (threadIdx.x >> 5));
        return;
    }
    using T = typename std::conditional<IO == DType::F32, float, __nv_bfloat16>::type;
    constexpr int D = IO == DType::F32 ? 4 : 3;
    const int ROWS = TC ? p.rows : (PACKED ? 8 / D : 8);
    const W4Args& g = p.g;
    const int m0 = blockIdx.z * ROWS, mt = g.M - m0 < ROWS ? g.M - m0 : ROWS;
    const int k_step0 = blockIdx.y * p.split_steps;
    const uint32_t nq = p.steps - k_step0 < p.split_steps ? p.steps - k_step0 : p.split_steps;
    const Image img(p.images + (static_cast<size_t>(blockIdx.z) * gridDim.y + blockIdx.y) * p.image_bytes, p.split_steps, p.cols,
                    PACKED ? p.cols : p.rows, F);
    const bool vec = g.lda % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(g.A) % 16 == 0;
    const uint32_t u = blockIdx.x * 8 + (threadIdx.x >> 4), m = u / nq, q = u - m * nq;
    stage<IO, PACKED, F, TC>(p, img, m0, k_step0, m, q, threadIdx.x & 15, vec, u < mt * nq);
}

// Tiles that other shares worked on too: the last to arrive adds the parts, K-range after K-range and
// share after share, so that the sum does not depend on who that is.  R: rows of a tile; WARPS: of
// which each takes steps of its own; `last` has a word for each thread of the team.
template <typename T, int R, int ROWS, int WARPS, typename Slots, typename Sync>
__device__ __forceinline__ void join_tiles(const Params& p, const Shares& shares, uint32_t share, uint32_t nq, int m0, int mt,
                                           uint32_t tile, uint32_t* last, Slots range_slots, Sync sync) {
    const W4Args& g = p.g;
    const int tt = threadIdx.x % kTeamThreads;
    const uint32_t per = static_cast<uint32_t>(p.split_steps);
    const uint32_t lo = shares.start(share), hi = shares.start(share + 1), tile0 = lo / nq;
    for (uint32_t t0 = tile0; t0 <= tile; t0 += kTeamThreads) {
        const uint32_t t = t0 + tt;
        if (t <= tile) {
            uint32_t parts = 0;
            if (gridDim.y > 1 || t * nq < lo || (t + 1) * nq > hi) {
                for (uint32_t y = 0; y < gridDim.y; ++y) {
                    const uint32_t ny = p.steps - y * per < per ? p.steps - y * per : per;
                    const Shares sy(p.tiles, ny, gridDim.x * kTeams, WARPS);
                    parts += sy.holder(t * ny + ny - 1) - sy.holder(t * ny) + 1;
                }
                uint32_t* ticket = p.tickets + static_cast<size_t>(blockIdx.z) * p.tiles + t;
                if (atom_add_acq_rel_gpu_u32(ticket, 1u) == parts - 1) *ticket = 0u;
                else parts = 0;
            }
            last[tt] = parts;
        }
        sync();
        constexpr int EACH = R > 32 ? kTeamThreads : 32;        // threads to a tile
        constexpr int NV = (R / 4 * ROWS + EACH - 1) / EACH;    // four rows of W and one of A each
        for (uint32_t i = tt / EACH; i < kTeamThreads && t0 + i <= tile; i += kTeamThreads / EACH) {
            if (last[i] == 0) continue;
            const uint32_t at = t0 + i;
            float4 sum[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) sum[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t y = 0; y < gridDim.y; y += 2) {       // two K-ranges' parts, four asked for at once
                const float4* from[2] = {};
                uint32_t s0[2], n[2] = {};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (y + h >= gridDim.y) continue;
                    const uint32_t ny = p.steps - (y + h) * per < per ? p.steps - (y + h) * per : per;
                    const Shares sy(p.tiles, ny, gridDim.x * kTeams, WARPS);
                    s0[h] = sy.holder(at * ny);
                    n[h] = sy.holder(at * ny + ny - 1) - s0[h] + 1;
                    from[h] = reinterpret_cast<const float4*>(range_slots(y + h)) + tt % EACH;
                }
                for (uint32_t i0 = 0; i0 < n[0] + n[1]; i0 += 4) {
                    float4 x[4][NV];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t i = i0 + k;
                        const bool h = i >= n[0];
                        const uint32_t s = h ? i - n[0] : i;
                        const float4* part = (h ? from[1] : from[0]) + (s == 0 ? at : p.tiles + (h ? s0[1] : s0[0]) + s) * static_cast<size_t>(R / 4 * ROWS);
#pragma unroll
                        for (int j = 0; j < NV; ++j)
                            x[k][j] = i < n[0] + n[1] && tt % EACH + j * EACH < R / 4 * mt ? __ldcg(part + j * EACH) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int j = 0; j < NV; ++j) {
                            sum[j].x += x[k][j].x;
                            sum[j].y += x[k][j].y;
                            sum[j].z += x[k][j].z;
                            sum[j].w += x[k][j].w;
                        }
                }
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int v = tt % EACH + j * EACH;
                if (v >= R / 4 * mt) continue;
                const int r = 4 * v % R, m = 4 * v / R;
                const float x[4] = {sum[j].x, sum[j].y, sum[j].z, sum[j].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t row = static_cast<int64_t>(at) * R + r + e;
                    if (row < g.N)
                        static_cast<T*>(g.C)[static_cast<int64_t>(m0 + m) * g.ldc + row] =
                            static_cast<T>(x[e] + (g.bias ? g.bias[row] : 0.0f));
                }
            }
        }
        sync();
    }
}

// D digits of an activation: three of bf16, four of FP32.  PACKED: the digits of
// up to 8 / D rows of A share one block of eight columns; else each digit has a
// block for up to eight rows.  (16 rows at once took longer than eight twice, 105
// against 86 us for 16x28672x8192 by this kernel: their sums spill.)  F: chunks of 32 weights that share their scales
// for sure (4, 2 or 1); sums are scaled every F chunks.
template <DType IO, bool PACKED, int F>
__global__ void __launch_bounds__(kTeams * kTeamThreads, 1)
gemm_w4_kernel(const Params p, const __grid_constant__ CUtensorMap map) {
    using T = typename std::conditional<IO == DType::F32, float, __nv_bfloat16>::type;
    constexpr bool PARTS = IO == DType::F32;
    constexpr int D = PARTS ? 4 : 3;
    constexpr int NT = PACKED ? 1 : D;              // blocks of eight columns
    constexpr int ROWS = PACKED ? 8 / D : 8;        // rows of A per pass
    constexpr int RED = 256;                        // floats of a warp's sums of a tile
    extern __shared__ __align__(1024) unsigned char smem[];
    const W4Args& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31, team = tid / kTeamThreads, tt = tid % kTeamThreads, warp = tt >> 5;
    const int gr = lane >> 2, t4 = lane & 3;
    const int m0 = blockIdx.z * ROWS, mt = g.M - m0 < ROWS ? g.M - m0 : ROWS;
    const int tcols = PACKED ? p.cols : p.rows;             // columns of the two tables below
    const int k_step0 = blockIdx.y * p.split_steps;
    const uint32_t nq = p.steps - k_step0 < p.split_steps ? p.steps - k_step0 : p.split_steps;
    const uint32_t per = static_cast<uint32_t>(p.split_steps);

    unsigned char* ring = smem + (team * kWarps + warp) * p.slots * kStepBytes;
    unsigned char* act = smem + kTeams * kWarps * p.slots * kStepBytes;
    const Image img(act, per, p.cols, tcols, F);
    float* const unit = img.unit;
    uint32_t* const base = img.base;
    float* const isum = img.isum;
    float* red = reinterpret_cast<float*>(act + p.image_bytes) + team * kWarps * RED;        // [warp][block of 16][4][lane]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.bars_at);
    uint64_t* image_bar = bars + kTeams * kWarps * kMaxSlots;
    uint32_t* odd = reinterpret_cast<uint32_t*>(image_bar + 1);                 // rows of A with an infinity or NaN
    bars += (team * kWarps + warp) * kMaxSlots;
    const bool zeros = g.zero != nullptr;
    const bool f32s = g.st == DType::F32;

    if (!p.images || p.copy) pdl_wait();
    pdl_launch_dependents();
    const Shares shares(p.tiles, nq, gridDim.x * kTeams, kWarps);
    const uint32_t share = team * gridDim.x + blockIdx.x;
    const bool busy = share < shares.n;
    const uint32_t lo = busy ? shares.start(share) : 0, hi = busy ? shares.start(share + 1) : 0;

    // --- producer: one step's weights, lane (g, t) four rows of the tile and 32 weights of each
    if (lane == 0)
        for (int i = 0; i < p.slots; ++i) mbar_init(bars + i, 1);
    if (tid == 0) {
        *odd = 0u;
        mbar_init(image_bar, 1);
    }
    fence_mbar_init();
    __syncwarp();
    Cursor prod(lo, hi, nq, warp);
    auto request = [&](int slot) {      // the warp's next step, into a slot that it is done with
        if (prod.q < prod.end) {
            if (lane == 0) {
                mbar_arrive_expect_tx(bars + slot, kStepBytes);
                tma_load_2d(ring + slot * kStepBytes, &map, bars + slot, static_cast<int>((k_step0 + prod.q) * (kStepK / 2)),
                            static_cast<int>(prod.tile * kRows));
            }
            prod.q += kWarps;
            if (prod.q >= prod.end) prod.settle(nq, warp);
        }
    };
    for (int s = 0; s < p.slots; ++s) request(s);

    // A scale or zero point as it lies in memory (bf16: in the low half), and its value.
    const int up = f32s ? 0 : 16;
    auto fetch = [&](const void* base, int64_t e) -> uint32_t {
        return f32s ? __ldg(static_cast<const uint32_t*>(base) + e) : __ldg(static_cast<const uint16_t*>(base) + e);
    };
    auto value = [&](uint32_t raw) { return __uint_as_float(raw << up); };
    auto group_of = [&](uint32_t chunk) { return min(static_cast<int>(__umulhi(2 * chunk, p.gmul) >> p.gshift), g.groups - 1); };
    const int scale_bytes = f32s ? 4 : 2;
    const int64_t to_zero = reinterpret_cast<intptr_t>(g.zero) - reinterpret_cast<intptr_t>(g.scale);
    // Scales are read one step ahead of their products, across the ends of tiles.
    Cursor ahead(lo, hi, nq, warp);
    const char* srow[4];    // the lane's four rows' first scales
    uint32_t raw[4] = {}, rawz[4] = {};
    auto open = [&](uint32_t t) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int64_t row = static_cast<int64_t>(t) * kRows + gr + 8 * h;
            srow[h] = static_cast<const char*>(g.scale) + (row < g.N ? row : g.N - 1) * g.lds * scale_bytes;
        }
    };
    auto fetch_scales = [&]() {
        if (ahead.q >= ahead.end) return;
        const int64_t gi = static_cast<int64_t>(group_of((k_step0 + ahead.q) * 4 + t4)) * scale_bytes;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            raw[h] = ldg_scale(srow[h] + gi, f32s);
            if (zeros) rawz[h] = ldg_scale(srow[h] + gi + to_zero, f32s);
        }
        ahead.q += kWarps;
        if (ahead.q >= ahead.end && ahead.left > 0) {
            ahead.settle(nq, warp);
            open(ahead.tile);
        }
    };
    if (busy) {
        open(ahead.tile);
        fetch_scales();
    }

    // --- the K-range's activations as digits: from the kernel before, or made here
    __syncthreads();
    if (p.images) {
        if (tid == 0) {
            pdl_wait();
            asm volatile("fence.proxy.async;" ::: "memory");
            const size_t at = (static_cast<size_t>(blockIdx.z) * gridDim.y + blockIdx.y) * p.image_bytes;
            mbar_arrive_expect_tx(image_bar, p.image_bytes);
            bulk_load_1d(act, p.images + at, p.image_bytes, image_bar);
        }
        mbar_wait(image_bar, 0, nullptr, p.err);
    } else {
        const bool vec = g.lda % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(g.A) % 16 == 0;
        const uint32_t units = mt * nq, r = tid & 15;
        uint32_t u = tid >> 4, m = u / nq, q = u - m * nq;
        const uint32_t dm = (kTeams * kTeamThreads / 16) / nq, dq = (kTeams * kTeamThreads / 16) - dm * nq;
        for (uint32_t u0 = u & ~1u; u0 < units; u0 += kTeams * kTeamThreads / 16) {     // the same count for a whole warp
            stage<IO, PACKED, F, false>(p, img, m0, k_step0, m, q, r, vec, u < units);
            u += kTeams * kTeamThreads / 16;
            m += dm;
            q += dq;
            if (q >= nq) { q -= nq; ++m; }
        }
        __syncthreads();
    }
    for (uint32_t i = tid; i < mt * nq; i += kTeams * kTeamThreads) {
        const uint32_t q = i / mt, m = i - q * mt;
        if (unit[q * tcols + m] < 0.0f) atomicOr(odd, 1u << m);
    }
    __syncthreads();
    if (!busy) return;

    auto sync = [&]() { named_barrier_sync(1 + team, kTeamThreads); };
    // The slots of K-range y.
    auto range_slots = [&](uint32_t y) {
        return p.ws + (static_cast<size_t>(blockIdx.z) * gridDim.y + y) * (p.tiles + gridDim.x * kTeams) * (kRows * ROWS);
    };

    // The lane's operand columns (those that are not there repeat the last) and its columns in the tables.
    const unsigned char* act_at[NT];
    uint32_t base_at[NT][2], tab[2];
    const uint32_t ring_at = smem_u32(ring) + lane * 16, act_half = p.cols * 64;
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        const int col = PACKED ? min(gr, p.cols - 1) : b * p.rows + min(gr, mt - 1);
        act_at[b] = act + col * 64 + t4 * 16;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            base_at[b][e] = PACKED ? min(2 * t4 + e, p.cols - 1) : b * p.rows + min(2 * t4 + e, mt - 1);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) tab[e] = min(2 * t4 + e, tcols - 1);
    uint32_t tile = lo / nq, q0 = lo - tile * nq, done = lo;
    uint32_t phase = 0;
    int slot = 0;
    bool dead = false;
    while (done < hi) {
        const uint32_t n = hi - done < nq - q0 ? hi - done : nq - q0, q1 = q0 + n;
        float2 tot[2][2] = {};      // [block of 16 rows][its half]
        for (uint32_t q = q0 + warp; q < q1; q += kWarps) {
            float sc[4], zr[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                sc[h] = value(raw[h]);
                zr[h] = 8.0f - (zeros ? value(rawz[h]) : 8.0f);
            }
            fetch_scales();
            if (!mbar_try_wait(bars + slot, phase) && !dead) dead = !mbar_wait(bars + slot, phase, nullptr, p.err);
            uint32_t w[4][4];           // [row][word]
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint4 v = lds128(ring_at + slot * kStepBytes + h * 512);
                w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
            }
            __syncwarp();
            request(slot);      // every lane has read it
            if (++slot == p.slots) { slot = 0; phase ^= 1u; }

            // A product takes a word from each lane of a quad.  Lane t holds the four words of chunk t:
            // scales shared by fewer chunks want the words of one chunk (or two) on all four lanes.
            if constexpr (F <= 2) {
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {       // words 2, 3 of lanes 0, 1 for words 0, 1 of lanes 2, 3
                        const uint32_t give = (t4 & 2) ? w[h][i] : w[h][i + 2];
                        const uint32_t have = __shfl_xor_sync(0xFFFFFFFFu, give, 2);
                        if (t4 & 2) w[h][i] = have; else w[h][i + 2] = have;
                    }
            }
            if constexpr (F == 1) {
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {    // odd words of even lanes for even words of odd lanes
                        const uint32_t give = (t4 & 1) ? w[h][i] : w[h][i + 1];
                        const uint32_t have = __shfl_xor_sync(0xFFFFFFFFu, give, 1);
                        if (t4 & 1) w[h][i] = have; else w[h][i + 1] = have;
                    }
            }
            float un[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) un[e] = fabsf(unit[q * tcols + tab[e]]);
            uint4 x[NT];        // the operand columns of two words
            uint32_t c[2][NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i % F == 0) {
#pragma unroll
                    for (int b = 0; b < NT; ++b)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t from = base[(q * (4 / F) + i / F) * p.cols + base_at[b][e]];
#pragma unroll
                            for (int k = 0; k < 2; ++k) c[k][b][e] = c[k][b][e + 2] = from;
                        }
                }
                if (i % 2 == 0) {
#pragma unroll
                    for (int b = 0; b < NT; ++b) x[b] = *reinterpret_cast<const uint4*>(act_at[b] + (q * 2 + i / 2) * act_half);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t (&w0)[4] = w[2 * k], (&w1)[4] = w[2 * k + 1];
                    const uint32_t av[4] = {w0[i] & 0x0F0F0F0Fu, w1[i] & 0x0F0F0F0Fu, (w0[i] >> 4) & 0x0F0F0F0Fu,
                                            (w1[i] >> 4) & 0x0F0F0F0Fu};
#pragma unroll
                    for (int b = 0; b < NT; ++b) mma_u8s8(c[k][b], av, i % 2 ? x[b].z : x[b].x, i % 2 ? x[b].w : x[b].y);
                }
                if ((i + 1) % F != 0) continue;
                const int f = i / F;
                float is[2] = {};
                if (zeros) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) is[e] = isum[(q * (4 / F) + f) * tcols + tab[e]];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float s0 = sc[2 * k], s1 = sc[2 * k + 1], z0 = zr[2 * k], z1 = zr[2 * k + 1];
                    if constexpr (F < 4) {
                        const int from = (lane & 28) | (f * F);
                        s0 = __shfl_sync(0xFFFFFFFFu, s0, from);
                        s1 = __shfl_sync(0xFFFFFFFFu, s1, from);
                        if (zeros) {
                            z0 = __shfl_sync(0xFFFFFFFFu, z0, from);
                            z1 = __shfl_sync(0xFFFFFFFFu, z1, from);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {       // a row's two columns at once
                        const float sh = h ? s1 : s0, zh = h ? z1 : z0;
                        float2 y = add2(bits2(&c[k][NT - 1][2 * h]), make_float2(-kMagic, -kMagic));
#pragma unroll
                        for (int d = NT - 2; d >= 0; --d)
                            y = fma2(y, make_float2(256.0f, 256.0f), add2(bits2(&c[k][d][2 * h]), make_float2(-kMagic, -kMagic)));
                        if (zeros) y = fma2(make_float2(zh, zh), make_float2(is[0], is[1]), y);
                        // The unit comes last: it and the scale alone may multiply to less than FP32's normal numbers.
                        tot[k][h] = fma2(mul2(make_float2(sh, sh), y), make_float2(un[0], un[1]), tot[k][h]);
                    }
                }
            }
        }

        // --- the tile's end in this share: add up the warps
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[((warp * 2 + k) * 4 + e) * 32 + lane] = e % 2 ? tot[k][e / 2].y : tot[k][e / 2].x;
        sync();
        const bool whole = n == nq && gridDim.y == 1;
        float* part_sums = whole ? nullptr : range_slots(blockIdx.y) + static_cast<size_t>(lo <= tile * nq ? tile : p.tiles + share) * (kRows * ROWS);
        for (int idx = tt; idx < kRows * mt; idx += kTeamThreads) {
            const int r = idx % kRows, m = idx / kRows;
            const int64_t row = static_cast<int64_t>(tile) * kRows + r;
            if (row >= g.N) continue;
            float sum = 0.0f;
#pragma unroll
            for (int d = 0; d < (PACKED ? D : 1); ++d) {
                const int col = d * p.rows + m, e = (col & 1) + 2 * ((r >> 3) & 1), ln = (r & 7) * 4 + (col >> 1);
#pragma unroll
                for (int wv = 0; wv < kWarps; ++wv) sum += red[((wv * 2 + (r >> 4)) * 4 + e) * 32 + ln];
            }
            if ((*odd >> m) & 1u) {
                // The activations that stayed out.
                const T* a = static_cast<const T*>(g.A) + static_cast<int64_t>(m0 + m) * g.lda;
                const int64_t k1 = static_cast<int64_t>(k_step0 + q1) * kStepK < g.K ? static_cast<int64_t>(k_step0 + q1) * kStepK : g.K;
                for (int64_t k = static_cast<int64_t>(k_step0 + q0) * kStepK; k < k1; ++k) {
                    const float v = static_cast<float>(a[k]);
                    if (fabsf(v) <= 3.402823466e38f) continue;
                    const uint32_t code = (g.W[row * g.ldw + k / 2] >> (4 * (k & 1))) & 15u;
                    const int64_t e = row * g.lds + k / g.group;
                    sum += v * (value(fetch(g.scale, e)) * (static_cast<float>(code) - (zeros ? value(fetch(g.zero, e)) : 8.0f)));
                }
            }
            if (whole) {
                const float out = sum + (g.bias ? g.bias[row] : 0.0f);
                static_cast<T*>(g.C)[static_cast<int64_t>(m0 + m) * g.ldc + row] = static_cast<T>(out);
            } else {
                part_sums[idx] = sum;
            }
        }
        sync();     // the sums have been read, and written where they go
        done += n;
        if (done < hi) { ++tile; q0 = 0; }
    }

    join_tiles<T, kRows, ROWS, kWarps>(p, shares, share, nq, m0, mt, tile, reinterpret_cast<uint32_t*>(red), range_slots, sync);
}

// ---- the same products by tcgen05, the codes as bytes in tensor memory -------
// A step is 128 weights of 128 rows (8 KB), a team's thread has a row: it decodes
// the row's 64 bytes into 32 columns of its lane, where a warp of its own for
// each team multiplies them (four products of K = 32, 128 rows and 16 or 32
// columns) by the digits in shared memory, and it scales its row's sums of the
// step before out of tensor memory.  So no operand of W passes through shared
// memory again, no instruction is spent on operands of A, and a row's scale is
// read once, not by four lanes.  Codes and sums are double: 128 columns a team.
// Even k come before odd k within eight, in the digits as in the decoded codes.
// Measured: 8x28672x8192 38.1 us (49%; by registers 42.3), 4 rows 34.1 (40.5), FP32
// 40.8, 16 rows 69.  A warp issues 299 instructions a step, half of the issue slots
// go by: on tensor memory, barriers and fixed latencies.  Waiting for a quarter
// of the digits at a time instead of all took longer (39.2).
__device__ __forceinline__ void umma_i8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
                 "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
                 "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
                 "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

// ROWS: of A per pass, 4 or 8.
template <DType IO, int ROWS, bool ZEROS>
__global__ void __launch_bounds__(kTcThreads, 1)
gemm_w4_tc_kernel(const Params p, const __grid_constant__ CUtensorMap map) {
    using T = typename std::conditional<IO == DType::F32, float, __nv_bfloat16>::type;
    constexpr int D = IO == DType::F32 ? 4 : 3;
    constexpr int NC = (D * ROWS + 7) / 8 * 8;      // digits' columns in shared memory
    constexpr int NM = (NC + 15) / 16 * 16;         // of a product: of 128 rows it has multiples of 16, the last 8 are not read
    static_assert(NM <= 32, "two steps' products and codes in a team's tensor memory");
    constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NM >> 3) << 17) | ((128u >> 4) << 24);
    extern __shared__ __align__(1024) unsigned char smem[];
    const W4Args& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31;
    const bool issuer = tid >= kTeams * kTeamThreads;   // a warp for each team asks for weights and issues products
    const int team = issuer ? (tid - kTeams * kTeamThreads) >> 5 : tid / kTeamThreads, tt = tid % kTeamThreads, warp = tt >> 5;
    const int m0 = blockIdx.z * ROWS, mt = g.M - m0 < ROWS ? g.M - m0 : ROWS;
    const int k_step0 = blockIdx.y * p.split_steps;
    const uint32_t nq = p.steps - k_step0 < p.split_steps ? p.steps - k_step0 : p.split_steps;
    const uint32_t per = static_cast<uint32_t>(p.split_steps);

    unsigned char* ring = smem + team * p.slots * kTcStepBytes;
    unsigned char* act = smem + kTeams * p.slots * kTcStepBytes;
    const Image img(act, per, NC, ROWS, 4);
    uint32_t* last = reinterpret_cast<uint32_t*>(act + p.image_bytes) + team * kTeamThreads;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.bars_at);
    uint64_t* image_bar = bars + kTeams * (kMaxSlots + 4);
    uint32_t* odd = reinterpret_cast<uint32_t*>(image_bar + 1);                 // rows of A with an infinity or NaN
    uint32_t* tmem_at = odd + 1;
    bars += team * (kMaxSlots + 4);
    uint64_t* code_bars = bars + kMaxSlots;         // a step's codes are in tensor memory
    uint64_t* done_bars = code_bars + 2;            // and its products
    const bool f32s = g.st == DType::F32;

    if (!p.images || p.copy) pdl_wait();
    const Shares shares(p.tiles, nq, gridDim.x * kTeams, 1);
    const uint32_t share = team * gridDim.x + blockIdx.x;
    const bool busy = share < shares.n;
    const uint32_t lo = busy ? shares.start(share) : 0, hi = busy ? shares.start(share + 1) : 0;

    // --- weights, a step at a time
    uint32_t ptile = lo / nq, pq = lo - ptile * nq, pleft = hi - lo;
    auto request = [&](int slot) {
        if (pleft == 0) return;
        mbar_arrive_expect_tx(bars + slot, kTcStepBytes);
        tma_load_2d(ring + slot * kTcStepBytes, &map, bars + slot, static_cast<int>((k_step0 + pq) * (kStepK / 2)),
                    static_cast<int>(ptile * kTcRows));
        --pleft;
        if (++pq == nq) { pq = 0; ++ptile; }
    };
    if (issuer && lane == 0) {
        for (int i = 0; i < p.slots; ++i) mbar_init(bars + i, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(code_bars + i, kWarps);
            mbar_init(done_bars + i, 1);
        }
        if (team == 0) {
            *odd = 0u;
            mbar_init(image_bar, 1);
        }
        fence_mbar_init();
        for (int s = 0; s < p.slots; ++s) request(s);
    }
    __syncwarp();
    if (tid < 32) {
        tmem_alloc(tmem_at, kTeams * kTcColumns);
        tmem_relinquish();
    }

    // --- scales are read one step ahead, across the ends of tiles
    const int up = f32s ? 0 : 16;
    auto fetch = [&](const void* base, int64_t e) -> uint32_t {
        return f32s ? __ldg(static_cast<const uint32_t*>(base) + e) : __ldg(static_cast<const uint16_t*>(base) + e);
    };
    auto value = [&](uint32_t raw) { return __uint_as_float(raw << up); };
    const int scale_bytes = f32s ? 4 : 2;
    const int64_t to_zero = reinterpret_cast<intptr_t>(g.zero) - reinterpret_cast<intptr_t>(g.scale);
    uint32_t atile = lo / nq, aq = lo - atile * nq, aleft = hi - lo;
    const char* sat = nullptr;      // the scale of the row's group
    int within = 0;                 // weights of that group before
    uint32_t raw = 0u, rawz = 0u;
    auto open = [&]() {
        const int64_t row = static_cast<int64_t>(atile) * kTcRows + tt, k = static_cast<int64_t>(k_step0 + aq) * kStepK;
        const int group = static_cast<int>(g.groups > 1 ? k / g.group : 0);
        within = static_cast<int>(k - static_cast<int64_t>(group) * g.group);
        sat = static_cast<const char*>(g.scale) + ((row < g.N ? row : g.N - 1) * g.lds + group) * scale_bytes;
    };
    auto fetch_scales = [&]() {
        if (aleft == 0) return;
        --aleft;
        raw = ldg_scale(sat, f32s);
        if constexpr (ZEROS) rawz = ldg_scale(sat + to_zero, f32s);
        within += kStepK;
        if (within >= g.group) {
            within = 0;
            sat += scale_bytes;
        }
        if (++aq == nq) {
            aq = 0;
            ++atile;
            open();
        }
    };
    if (busy && !issuer) {
        open();
        fetch_scales();
    }

    // --- the K-range's activations as digits: from the kernel before, or made here
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;
    // Dependent kernels may start once every CTA holds its tensor memory: one that allocated first would
    // wait for this grid to end, and this grid for its columns.
    pdl_launch_dependents();
    if (p.images) {
        if (tid == 0) {
            pdl_wait();
            asm volatile("fence.proxy.async;" ::: "memory");
            const size_t at = (static_cast<size_t>(blockIdx.z) * gridDim.y + blockIdx.y) * p.image_bytes;
            mbar_arrive_expect_tx(image_bar, p.image_bytes);
            bulk_load_1d(act, p.images + at, p.image_bytes, image_bar);
        }
        mbar_wait(image_bar, 0, nullptr, p.err);
    } else {
        const bool vec = g.lda % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(g.A) % 16 == 0;
        const uint32_t units = mt * nq, r = tid & 15;
        uint32_t u0 = (tid >> 4) & ~1u;
        if (issuer) u0 = units;
        for (; u0 < units; u0 += kTeams * kTeamThreads / 16) {    // the same count for a whole warp
            const uint32_t u = u0 + ((tid >> 4) & 1), m = u / nq, q = u - m * nq;
            stage<IO, false, 4, true>(p, img, m0, k_step0, m, q, r, vec, u < units);
        }
        fence_proxy_async_smem();
        __syncthreads();
    }
    for (uint32_t i = tid; i < mt * nq; i += kTcThreads) {
        const uint32_t q = i / mt, m = i - q * mt;
        const float u = img.unit[q * ROWS + m];
        if (u < 0.0f) {
            atomicOr(odd, 1u << m);
            img.unit[q * ROWS + m] = -u;
        }
    }
    __syncthreads();

    auto sync = [&]() { named_barrier_sync(1 + team, kTeamThreads); };
    // The slots of K-range y.
    auto range_slots = [&](uint32_t y) {
        return p.ws + (static_cast<size_t>(blockIdx.z) * gridDim.y + y) * (p.tiles + gridDim.x * kTeams) * (kTcRows * ROWS);
    };
    const uint32_t own = tmem + team * kTcColumns, lanes = static_cast<uint32_t>(warp) << 21;  // 32 lanes a warp, in bits 16 up
    const uint32_t ring_at = smem_u32(ring) + tt * 64, swz = (tt >> 1) & 3, act_at = smem_u32(act);
    const uint32_t base_at = smem_u32(img.base), unit_at = smem_u32(img.unit);
    uint32_t step = 0, phase = 0;
    int slot = 0;
    bool dead = false;
    if (issuer) {
        if (lane == 0) {
            uint32_t q = lo - lo / nq * nq;
            for (uint32_t left = hi - lo; left > 0; --left, ++step) {
                const uint32_t i = step & 1;
                if (!mbar_try_wait(code_bars + i, (step >> 1) & 1) && !dead) dead = !mbar_wait(code_bars + i, (step >> 1) & 1, nullptr, p.err);
                tc_fence_after();
                const uint64_t b = umma_desc_k_sw128(act_at + q * (NC * 128));
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_i8_ts(own + 64 + i * 32, own + i * 32 + k * 8, b + k * 2, IDESC, k != 0);
                umma_commit(done_bars + i);
                request(slot);      // every thread has read it
                if (++slot == p.slots) slot = 0;
                if (++q == nq) q = 0;
            }
        }
        __syncwarp();
    }
    float2 tot[ROWS / 2];
    // Scales the products of the step before: i counts steps, q is its place in the K-range.
    auto scale_step = [&](uint32_t i, uint32_t q, float sc, float zr) {
        if (!mbar_try_wait(done_bars + (i & 1), (i >> 1) & 1) && !dead) dead = !mbar_wait(done_bars + (i & 1), (i >> 1) & 1, nullptr, p.err);
        __syncwarp();
        tc_fence_after();
        const uint32_t from = own + lanes + 64 + (i & 1) * 32;
        uint32_t c[NC];
#pragma unroll
        for (int b = 0; b < NC; b += 8) tmem_ld_x8(from + b, c + b);
        float un[ROWS];
#pragma unroll
        for (int m = 0; m < ROWS; m += 4) {
            const uint4 v = lds128(unit_at + (q * ROWS + m) * 4);
            un[m] = __uint_as_float(v.x); un[m + 1] = __uint_as_float(v.y);
            un[m + 2] = __uint_as_float(v.z); un[m + 3] = __uint_as_float(v.w);
        }
        tmem_ld_wait();
#pragma unroll
        for (int b = 0; b < NC; b += 4) {
            const uint4 v = lds128(base_at + (q * NC + b) * 4);
            c[b] += v.x; c[b + 1] += v.y; c[b + 2] += v.z; c[b + 3] += v.w;
        }
#pragma unroll
        for (int m = 0; m < ROWS; m += 2) {
            auto digit = [&](int d) { return add2(bits2(c + d * ROWS + m), make_float2(-kMagic, -kMagic)); };
            float2 y = digit(D - 1);
#pragma unroll
            for (int d = D - 2; d >= 0; --d) y = fma2(y, make_float2(256.0f, 256.0f), digit(d));
            if constexpr (ZEROS) y = fma2(make_float2(zr, zr), *reinterpret_cast<const float2*>(img.isum + q * ROWS + m), y);
            // The unit comes last: it and the scale alone may multiply to less than FP32's normal numbers.
            tot[m / 2] = fma2(mul2(make_float2(sc, sc), y), make_float2(un[m], un[m + 1]), tot[m / 2]);
        }
    };

    if (busy && !issuer) {
        uint32_t tile = lo / nq, q0 = lo - tile * nq, done = lo;
        while (done < hi) {
            const uint32_t n = hi - done < nq - q0 ? hi - done : nq - q0, q1 = q0 + n;
#pragma unroll
            for (int m = 0; m < ROWS / 2; ++m) tot[m] = make_float2(0.0f, 0.0f);
            float sc = 0.0f, zr = 0.0f;
            for (uint32_t q = q0; q < q1; ++q) {
                if (!mbar_try_wait(bars + slot, phase) && !dead) dead = !mbar_wait(bars + slot, phase, nullptr, p.err);
                uint32_t a[32];     // byte b of word 2j + h is code 8j + 2b + h
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint4 v = lds128(ring_at + slot * kTcStepBytes + ((c ^ swz) << 4));
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[8 * c + 2 * j] = w[j] & 0x0F0F0F0Fu;
                        a[8 * c + 2 * j + 1] = (w[j] >> 4) & 0x0F0F0F0Fu;
                    }
                }
                __syncwarp();
                tmem_st_x32(own + lanes + (step & 1) * 32, a);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(code_bars + (step & 1));
                if (++slot == p.slots) { slot = 0; phase ^= 1u; }
                if (q > q0) scale_step(step - 1, q - 1, sc, zr);
                sc = value(raw);
                if constexpr (ZEROS) zr = 8.0f - value(rawz);
                fetch_scales();
                ++step;
            }
            scale_step(step - 1, q1 - 1, sc, zr);

            // --- the tile's end in this share
            const bool whole = n == nq && gridDim.y == 1;
            float* part_sums = whole ? nullptr : range_slots(blockIdx.y) + static_cast<size_t>(lo <= tile * nq ? tile : p.tiles + share) * (kTcRows * ROWS);
            const int64_t row = static_cast<int64_t>(tile) * kTcRows + tt;
            if (row < g.N) {
#pragma unroll
                for (int m = 0; m < ROWS; ++m) {
                    if (m >= mt) continue;
                    float sum = m % 2 ? tot[m / 2].y : tot[m / 2].x;
                    if ((*odd >> m) & 1u) {
                        // The activations that stayed out.
                        const T* x = static_cast<const T*>(g.A) + static_cast<int64_t>(m0 + m) * g.lda;
                        const int64_t k1 = static_cast<int64_t>(k_step0 + q1) * kStepK < g.K ? static_cast<int64_t>(k_step0 + q1) * kStepK : g.K;
                        for (int64_t k = static_cast<int64_t>(k_step0 + q0) * kStepK; k < k1; ++k) {
                            const float v = static_cast<float>(x[k]);
                            if (fabsf(v) <= 3.402823466e38f) continue;
                            const uint32_t code = (g.W[row * g.ldw + k / 2] >> (4 * (k & 1))) & 15u;
                            const int64_t e = row * g.lds + k / g.group;
                            sum += v * (value(fetch(g.scale, e)) * (static_cast<float>(code) - (ZEROS ? value(fetch(g.zero, e)) : 8.0f)));
                        }
                    }
                    if (whole) {
                        const float out = sum + (g.bias ? g.bias[row] : 0.0f);
                        static_cast<T*>(g.C)[static_cast<int64_t>(m0 + m) * g.ldc + row] = static_cast<T>(out);
                    } else {
                        part_sums[m * kTcRows + tt] = sum;
                    }
                }
            }
            done += n;
            if (done < hi) { ++tile; q0 = 0; }
        }
        sync();     // the team's sums are written
        join_tiles<T, kTcRows, ROWS, 1>(p, shares, share, nq, m0, mt, tile, last, range_slots, sync);
    }
    tc_fence_before();
    __syncthreads();
    if (tid < 32) tmem_dealloc(tmem, kTeams * kTcColumns);
}

struct Kernel {
    const void* fn;
    const void* digits;
    int rows, n_digits, flush;
    bool packed, tc;
};

template <DType IO, int ROWS>
Kernel tc_kernel(bool zeros) {
    return {zeros ? reinterpret_cast<const void*>(&gemm_w4_tc_kernel<IO, ROWS, true>) : reinterpret_cast<const void*>(&gemm_w4_tc_kernel<IO, ROWS, false>),
            reinterpret_cast<const void*>(&gemm_w4_digits_kernel<IO, false, 4, true>), ROWS, IO == DType::F32 ? 4 : 3, 4, false, true};
}

template <DType IO, bool PACKED>
Kernel kernel_for_flush(int f) {
    constexpr int D = IO == DType::F32 ? 4 : 3;
    const void* fn = f == 4 ? reinterpret_cast<const void*>(&gemm_w4_kernel<IO, PACKED, 4>)
                     : f == 2 ? reinterpret_cast<const void*>(&gemm_w4_kernel<IO, PACKED, 2>)
                              : reinterpret_cast<const void*>(&gemm_w4_kernel<IO, PACKED, 1>);
    const void* digits = f == 4 ? reinterpret_cast<const void*>(&gemm_w4_digits_kernel<IO, PACKED, 4, false>)
                         : f == 2 ? reinterpret_cast<const void*>(&gemm_w4_digits_kernel<IO, PACKED, 2, false>)
                                  : reinterpret_cast<const void*>(&gemm_w4_digits_kernel<IO, PACKED, 1, false>);
    return {fn, digits, PACKED ? 8 / D : 8, D, f, PACKED, false};
}

Kernel select(const W4Args& g) {
    // How many chunks of 32 weights share their scales for sure, up to the four of a step.
    const int f = g.groups == 1 || g.group % 128 == 0 ? 4 : (g.group % 64 == 0 ? 2 : 1);
    // Codes in tensor memory: 8x28672x8192 38.1 us (products of registers 42.3), 4 rows 34.2 (40.5), 3 rows
    // 34.0 (41.4), 8x28672x4096 23.3 (26.4), 8x65536x512 10.4 (15.3), 8x11008x4096 17.1 (18.1), 3x8192x4096
    // 14.3 (15.1).  At the rule's edge it can lose: 8x8192x4096 16.4 (15.7), 8x8192x8192 22.4 (21.0),
    // 8x16384x2048 15.0 (12.4), whose tiles of 32 rows the registers' teams take whole.  Below it, its
    // tiles of 128 rows are too few of too many parts: 8x8192x2048 11.6 (9.1), 8x4096x11008 21.9 (19.0).
    if (f == 4 && g.M > 2 && g.N >= 8192 && static_cast<int64_t>(g.N) * g.K >= int64_t(1) << 25) {
        const bool zeros = g.zero != nullptr;
        if (g.io == DType::F32) return g.M <= 4 ? tc_kernel<DType::F32, 4>(zeros) : tc_kernel<DType::F32, 8>(zeros);
        return g.M <= 4 ? tc_kernel<DType::BF16, 4>(zeros) : tc_kernel<DType::BF16, 8>(zeros);
    }
    // Two rows' digits fit one block of columns: a third (a quarter) of the products.
    if (g.io == DType::F32) return g.M <= 2 ? kernel_for_flush<DType::F32, true>(f) : kernel_for_flush<DType::F32, false>(f);
    return g.M <= 2 ? kernel_for_flush<DType::BF16, true>(f) : kernel_for_flush<DType::BF16, false>(f);
}

bool aligned_rows(const W4Args& g) { return g.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(g.W) % 16 == 0; }

int64_t row_bytes_of(const W4Args& g) { return (static_cast<int64_t>(g.K) + 1) / 2; }

cudaError_t launch_pdl(const void* fn, dim3 grid, int threads, void** args, int smem, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return static_cast<EncodeTiled>(nullptr);
        return reinterpret_cast<EncodeTiled>(ptr);
    }();
    return fn;
}

// W as bytes [N][(K+1)/2], read in boxes of 64 bytes x 32 rows; bytes and rows past the ends read as zeros.
bool encode_weights(const W4Args& g, const uint8_t* w, int64_t pitch, bool tc, CUtensorMap* map) {
    EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes_of(g)), static_cast<cuuint64_t>(g.N)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
    const cuuint32_t box[2] = {kStepK / 2, static_cast<cuuint32_t>(tc ? kTcRows : kRows)}, one[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(w), dims, strides, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, tc ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool gemm_w4_plan(const W4Args& g, int num_sms, W4Plan* plan) {
    const Kernel k = select(g);
    const int tile_rows = k.tc ? kTcRows : kRows, step_bytes = k.tc ? kTcStepBytes : kStepBytes;
    plan->rows = !k.tc && g.M < k.rows ? g.M : k.rows;
    const int64_t steps = (static_cast<int64_t>(g.K) + kStepK - 1) / kStepK, tiles = (static_cast<int64_t>(g.N) + tile_rows - 1) / tile_rows;
    plan->cols = k.tc ? (k.n_digits * plan->rows + 7) / 8 * 8 : k.n_digits * plan->rows;
    // As much of K at a time as the digits leave room for beside the smallest rings; the rings take
    // what is left.
    const int rings = k.tc ? kTeams : kTeams * kWarps, bars = k.tc ? kTeams * (kMaxSlots + 4) * 8 : kTeams * kWarps * kMaxSlots * 8;
    const int fixed = kTeams * (k.tc ? kTeamThreads * 4 : kWarps * 1024) + bars + 64 + 16;
    const int per_step = plan->cols * (128 + 4 * (4 / k.flush)) + 4 * (k.packed ? plan->cols : plan->rows) * (1 + 4 / k.flush);
    const int64_t most = (kMaxSmem - fixed - rings * kMinSlots * step_bytes) / per_step;
    const int64_t splits = (steps + most - 1) / most;
    plan->split_steps = static_cast<int>((steps + splits - 1) / splits);
    plan->splits = static_cast<int>((steps + plan->split_steps - 1) / plan->split_steps);
    const int rest = (kMaxSmem - fixed - per_step * plan->split_steps) / (rings * step_bytes);
    plan->slots = rest < kMaxSlots ? rest : kMaxSlots;
    plan->smem = fixed + per_step * plan->split_steps + rings * plan->slots * step_bytes;
    plan->bars_at = (plan->smem - bars - 16) & ~7;
    plan->image_bytes = (per_step * plan->split_steps + 15) & ~15;
    // 512 threads take half a microsecond for every 32 stretches of 128 activations; a kernel before
    // this one takes about one and overlaps this one's start (products of registers: 1x28672x8192, 64
    // stretches, 30.0 us without and 31.0 with it; 5x4093x4099 FP32, 165, 21.6 and 19.5; 8x28672x8192,
    // 256, 47.3 and 44.1).
    const int64_t stretches = static_cast<int64_t>(g.M < k.rows ? g.M : k.rows) * plan->split_steps;
    plan->prepared = stretches > 64;
    plan->pitch = aligned_rows(g) ? 0 : (row_bytes_of(g) + 15) / 16 * 16;
    plan->copy_bytes = static_cast<size_t>(plan->pitch) * g.N;
    plan->blocks = (g.M + k.rows - 1) / k.rows;
    plan->extra_bytes = plan->copy_bytes;
    if (plan->prepared) plan->extra_bytes += static_cast<size_t>(plan->blocks) * plan->splits * plan->image_bytes;
    // Every SM a CTA, shared among the K-ranges (one more would wait for a second round); no more than
    // there are shares.
    int64_t ctas = num_sms / plan->splits;
    if (ctas < 1) ctas = 1;
    const int64_t shares = (tiles * plan->split_steps + (k.tc ? kTeams : kWarps) - 1) / (k.tc ? kTeams : kWarps);
    if (ctas > shares) ctas = shares;
    plan->ctas = static_cast<int>(ctas);
    // Steps are counted in 32 bits; blocks and splits are grid dimensions.
    if (tiles * plan->split_steps > INT32_MAX || plan->splits > 65535 || plan->blocks > 65535) return false;
    plan->ws_floats = static_cast<size_t>(plan->blocks) * plan->splits * (tiles + ctas * kTeams) * tile_rows * k.rows;
    plan->tickets = static_cast<size_t>(plan->blocks) * tiles;
    return true;
}

cudaError_t launch_gemm_w4(const W4Args& g, const W4Plan& plan, float* ws, uint32_t* tickets, void* extra,
                           uint32_t* err, cudaStream_t s) {
    const Kernel k = select(g);
    static std::mutex mu;
    static std::unordered_set<const void*> known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!known[dev].count(k.fn)) {
            e = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
            if (e != cudaSuccess) return e;
            known[dev].insert(k.fn);
        }
    }
    Params p;
    p.g = g;
    const int tile_rows = k.tc ? kTcRows : kRows;
    p.tiles = static_cast<int>((static_cast<int64_t>(g.N) + tile_rows - 1) / tile_rows);
    p.steps = static_cast<int>((static_cast<int64_t>(g.K) + kStepK - 1) / kStepK);
    p.split_steps = plan.split_steps;
    p.slots = plan.slots;
    p.cols = plan.cols;
    p.rows = plan.rows;
    p.bars_at = plan.bars_at;
    // chunk / (group / 32) = mulhi(2 chunk, mul) >> log for chunks below 2^31: mul = ceil(2^(31 + ceil(log2 d)) / d).
    const int64_t d = g.groups > 1 ? g.group / 32 : int64_t(1) << 30;
    int log = 0;
    while ((int64_t(1) << log) < d) ++log;
    p.gmul = static_cast<uint32_t>(((uint64_t(1) << (31 + log)) + d - 1) / d);
    p.gshift = log;
    p.ws = ws;
    p.tickets = tickets;
    p.err = err;
    p.copy = plan.pitch ? static_cast<uint8_t*>(extra) : nullptr;
    p.copy_pitch = plan.pitch;
    CUtensorMap map;
    if (!encode_weights(g, plan.pitch ? p.copy : g.W, plan.pitch ? plan.pitch : g.ldw, k.tc, &map)) return cudaErrorNotSupported;
    p.image_bytes = plan.image_bytes;
    p.images = plan.prepared ? static_cast<unsigned char*>(extra) + plan.copy_bytes : nullptr;
    p.digit_ctas = 0;
    if (plan.prepared || plan.pitch) {
        const unsigned stretches = static_cast<unsigned>(g.M < plan.rows ? g.M : plan.rows) * plan.split_steps;
        if (plan.prepared) p.digit_ctas = (stretches + 7) / 8;
        const unsigned copies = plan.pitch ? (static_cast<unsigned>(g.N) + 3) / 4 : 0;
        void* first[] = {&p};
        e = launch_pdl(k.digits, plan.prepared ? dim3(p.digit_ctas + copies, plan.splits, plan.blocks) : dim3(copies), 128, first, 0, s);
        if (e != cudaSuccess) return e;
    }
    // With only digits made before it, the kernel starts before they are done: all that it reads or
    // writes until it waits for them is older than the kernel that makes them, or its own.
    void* args[] = {&p, &map};
    return launch_pdl(k.fn, dim3(plan.ctas, plan.splits, plan.blocks), k.tc ? kTcThreads : kTeams * kTeamThreads, args, plan.smem, s);
}

}  // namespace dnnopt_b200
