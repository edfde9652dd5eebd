// Products of few rows with 4-bit weights and group scales:
//   C[m,n] = bias[n] + sum_k A[m,k] * scale[n,k/g] * (code[n,k] - zero[n,k/g]).
//
// What bounds it: a weight is half a byte and used M times, so HBM up to
// M of about 64; below that, turning codes into operands is the work.  The
// products are mma.sync m16n8k16 with 16 rows of W and eight columns of
// activations: a code becomes a bf16 number by placing its four bits in the
// mantissa of 16.0 (16 + code, one shift and one three-input logic operation
// for two codes), and the 16 and the zero point are taken off once a group:
//   sum (code - zero) a = sum (16 + code) a - (16 + zero) sum a.
// A tcgen05 tile would need the decoded weights in shared memory first, four
// times the bytes that arrive, for 8 of its at least 64 columns.
//
// Exactness.  16 + code and bf16 activations multiply exactly; sums are FP32
// and start from zero every 128 (64, 32) weights, because the matrix units
// truncate what they add to.  FP32 activations are cut into three bf16 parts
// (24 bits, no loss) that take a column each; there the codes have 8 taken off
// before the product, since (16 + zero) sum a would cost five bits.
// Activations that are infinite or NaN stay out of the products (they would
// meet the zero points' sums) and are added for their own row at the end.
//
// Work.  128 weights of 16 rows (1 KB) are a step.  All steps, tile after tile
// of 16 rows, are cut into equal shares, one for each team of eight warps, two
// teams to an SM; a team's warps take the steps of a tile in turn and add up
// in shared memory.  A tile cut by a share's end, or by the ends of a K-range, is
// finished by the last of its shares to arrive, adding the parts in order.  The
// activations of the K-range sit in shared memory in the order in which the
// operand reads them.
#include <mutex>
#include <type_traits>
#include <unordered_set>

#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

constexpr int kTeams = 2;           // per CTA
constexpr int kTeamThreads = 256;
constexpr int kWarps = 8;           // per team
constexpr int kSlots = 4;           // steps under way per warp
constexpr int kStepK = 128;
constexpr int kMaxSmem = 227 * 1024;

struct Params {
    W4Args g;
    int tiles;                      // of 16 rows of W
    int steps;                      // ceil(K / 128)
    int split_steps;                // steps of one K-range (gridDim.y of them)
    int slot_bytes;
    int cols;                       // columns of activations: rows of A, or three parts of each
    uint32_t gmul, gshift;          // chunk of 32 weights -> group
    float* ws;                      // partial tiles, see part_slot
    uint32_t* tickets;              // one per tile and block of rows of A
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Codes I and I + 4 of a word as two bf16 numbers: 16 + code, or (MINUS8) code - 8.
template <int I, bool MINUS8>
__device__ __forceinline__ uint32_t decode(uint32_t w) {
    const uint32_t s = I == 0 ? w << 3 : w >> (4 * I - 3);
    uint32_t r = (s & 0x00780078u) | 0x41804180u;
    if constexpr (MINUS8) {
        const __nv_bfloat162 off = __floats2bfloat162_rn(24.0f, 24.0f);
        __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&r), off);
        r = *reinterpret_cast<uint32_t*>(&v);
    }
    return r;
}

// Equal shares of `total` steps, at least eight (one for each warp of a team).
struct Shares {
    uint32_t total, n;

    __device__ Shares(uint32_t steps, uint32_t most) : total(steps), n(steps / kWarps) {
        if (n > most) n = most;
        if (n < 1) n = 1;
    }
    __device__ __forceinline__ uint32_t start(uint32_t s) const {
        return static_cast<uint32_t>(static_cast<uint64_t>(s) * total / n);
    }
    // The share that holds step t: the last one that starts at or before it.
    __device__ __forceinline__ uint32_t holder(uint32_t t) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(t + 1) * n - 1) / total);
    }
};

// One warp's steps of a share: every eighth of each tile's.
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

// Slot of a partial tile within its K-range: the part with the tile's first
// step goes by the tile, a later part begins its share and goes by the share.
__device__ __forceinline__ size_t part_slot(const Shares& s, uint32_t share, uint32_t tile, uint32_t per_tile, int tiles) {
    return s.start(share) <= tile * per_tile ? tile : tiles + share;
}

// F: chunks of 32 weights that share their scales for sure (4, 2 or 1); sums
// are scaled every F chunks.  NT: blocks of eight columns.
template <DType IO, int NT, int F>
__global__ void __launch_bounds__(kTeams * kTeamThreads, 1) gemm_w4_kernel(const Params p) {
    using T = typename std::conditional<IO == DType::F32, float, __nv_bfloat16>::type;
    constexpr bool PARTS = IO == DType::F32;
    constexpr int ROWS = PARTS ? NT * 8 / 3 : NT * 8;       // rows of A per pass
    extern __shared__ __align__(128) unsigned char smem[];
    const W4Args& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31, team = tid / kTeamThreads, tt = tid % kTeamThreads, warp = tt >> 5;
    const int gr = lane >> 2, t4 = lane & 3;
    const int m0 = blockIdx.z * ROWS, mt = g.M - m0 < ROWS ? g.M - m0 : ROWS;
    const int cols = PARTS ? 3 * mt : mt;
    const int k_step0 = blockIdx.y * p.split_steps;
    const uint32_t nq = p.steps - k_step0 < p.split_steps ? p.steps - k_step0 : p.split_steps;
    const uint32_t per = static_cast<uint32_t>(p.split_steps);

    unsigned char* ring = smem + (team * kWarps + warp) * kSlots * p.slot_bytes;
    unsigned char* act = smem + kTeams * kWarps * kSlots * p.slot_bytes;
    float* asum = reinterpret_cast<float*>(act + static_cast<size_t>(per) * p.cols * 256);   // [step][flush][col]
    float* red = asum + per * (4 / F) * p.cols + team * kWarps * NT * 128;                   // [warp][4 NT][lane]
    // Rows of A with an infinity or NaN.
    uint32_t* odd = reinterpret_cast<uint32_t*>(asum + per * (4 / F) * p.cols + kTeams * kWarps * NT * 128);
    const bool zeros = g.zero != nullptr;
    const bool f32s = g.st == DType::F32;
    const int row_bytes = (g.K + 1) / 2;

    const Shares shares(p.tiles * nq, gridDim.x * kTeams);
    const uint32_t share = team * gridDim.x + blockIdx.x;
    const bool busy = share < shares.n;
    const uint32_t lo = busy ? shares.start(share) : 0, hi = busy ? shares.start(share + 1) : 0;

    // --- producer: a step's weights (two rows of the tile to a lane, 32 weights each) and their scales
    const bool aligned = g.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(g.W) % 16 == 0;
    auto group_of = [&](uint32_t chunk) {
        const int gi = p.gmul ? static_cast<int>(__umulhi(chunk, p.gmul) >> p.gshift) : static_cast<int>(chunk);
        return gi < g.groups ? gi : g.groups - 1;
    };
    const int es = f32s ? 2 : 1;            // log2 of a scale's bytes
    const int64_t to_zero = reinterpret_cast<intptr_t>(g.zero) - reinterpret_cast<intptr_t>(g.scale);
    const uint8_t* wrow[2];                 // the lane's two rows of the tile being requested
    uintptr_t srow[2];
    auto open = [&](uint32_t t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int64_t n = static_cast<int64_t>(t) * 16 + gr + 8 * h;
            if (n >= g.N) n = g.N - 1;
            wrow[h] = g.W + n * g.ldw;
            srow[h] = reinterpret_cast<uintptr_t>(g.scale) + ((n * g.lds) << es);
        }
    };
    const uint32_t mine = smem_u32(ring) + lane * 16;
    auto issue = [&](uint32_t q, uint32_t slot_off) {
        const uint32_t dst = mine + slot_off, sdst = dst - lane * 12 + 1024;
        const uint32_t chunk = (k_step0 + q) * 4 + t4;
        const int at = static_cast<int>(chunk) * 16, here = max(0, min(16, row_bytes - at));
        const uint32_t gi = static_cast<uint32_t>(group_of(chunk)) << es;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (aligned) {
                cp_async16(dst + h * 512, here > 0 ? wrow[h] + at : wrow[h], here);
            } else {
                // Rows that start anywhere: whole 4-byte words that hold at least one byte of the row.
                const uintptr_t row = reinterpret_cast<uintptr_t>(wrow[h]), from = row + at, end = row + row_bytes;
                const uint32_t* a4 = reinterpret_cast<const uint32_t*>(from & ~uintptr_t(3));
                uint32_t x[5];
#pragma unroll
                for (int i = 0; i < 5; ++i) x[i] = here > 0 && reinterpret_cast<uintptr_t>(a4 + i) < end ? __ldg(a4 + i) : 0u;
                const uint32_t sh = static_cast<uint32_t>(from & 3) * 8;
                *reinterpret_cast<uint4*>(ring + slot_off + lane * 16 + h * 512) =
                    make_uint4(__funnelshift_r(x[0], x[1], sh), __funnelshift_r(x[1], x[2], sh),
                               __funnelshift_r(x[2], x[3], sh), __funnelshift_r(x[3], x[4], sh));
            }
            // The 4-byte word that holds the scale (bf16: its half is told apart when it is read).
            cp_async4(sdst + h * 128, reinterpret_cast<const void*>((srow[h] + gi) & ~uintptr_t(3)));
            if (zeros) cp_async4(sdst + 256 + h * 128, reinterpret_cast<const void*>((srow[h] + to_zero + gi) & ~uintptr_t(3)));
        }
    };
    Cursor prod(lo, hi, nq, warp);
    open(prod.tile);
    auto request = [&](uint32_t slot_off) {     // the warp's next step
        if (prod.q < prod.end) {
            issue(prod.q, slot_off);
            prod.q += kWarps;
            if (prod.q >= prod.end && prod.left > 0) {
                prod.settle(nq, warp);
                open(prod.tile);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kSlots; ++s) request(s * p.slot_bytes);

    // --- the K-range's activations, eight to a thread: as bf16 in the operand's order, and their
    // sums over each stretch of F chunks
    if (tid == 0) *odd = 0u;
    __syncthreads();
    {
        const uint32_t blocks = nq * 16;
        const bool vec = g.lda % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(g.A) % 16 == 0;
        for (uint32_t idx = tid; idx < blocks * mt; idx += kTeams * kTeamThreads) {
            const uint32_t m = idx / blocks, j = idx - m * blocks, q = j >> 4, r = j & 15;
            const int64_t k = static_cast<int64_t>(k_step0) * kStepK + j * 8;
            const T* a = static_cast<const T*>(g.A) + (m0 + m) * g.lda + k;
            float v[8];
            if (vec && k + 8 <= g.K) {
                if constexpr (PARTS) {
                    const float4 x = __ldg(reinterpret_cast<const float4*>(a)), y = __ldg(reinterpret_cast<const float4*>(a) + 1);
                    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
                } else {
                    const uint4 x = __ldg(reinterpret_cast<const uint4*>(a));
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[2 * i] = __uint_as_float(w[i] << 16);
                        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = k + i < g.K ? static_cast<float>(a[i]) : 0.0f;
            }
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(fabsf(v[i]) <= 3.402823466e38f)) { v[i] = 0.0f; bad = true; }
            if (bad) atomicOr(odd, 1u << m);
            // Which word of which lane these eight weights are, after the exchanges below.
            const uint32_t w = F == 4 ? (r & 3) : (F == 1 ? (r >> 2) : ((r >> 3) * 2 + (r & 1)));
            const uint32_t t = F == 4 ? (r >> 2) : (F == 1 ? (r & 3) : (((r >> 2) & 1) + (r & 2)));
            const uint32_t col = PARTS ? 3 * m : m;
            unsigned char* dst = act + (static_cast<size_t>(q * 4 + w) * p.cols + col) * 64 + t * 16;
#pragma unroll
            for (int part = 0; part < (PARTS ? 3 : 1); ++part) {
                uint32_t o[4];
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = v[i], y = v[i + 4];
                    o[i] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
                    if constexpr (PARTS) {
                        const float hx = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
                        const float hy = __uint_as_float(__float_as_uint(y) & 0xFFFF0000u);
                        sum += hx + hy;
                        v[i] = x - hx;
                        v[i + 4] = y - hy;
                    } else {
                        sum += x + y;
                    }
                }
                *reinterpret_cast<uint4*>(dst + part * 64) = make_uint4(o[0], o[1], o[2], o[3]);
                // There is a multiple of 16 of blocks, so the lanes of a stretch are all here or all gone.
                const uint32_t here = blocks * mt - (idx - lane) >= 32 ? 0xFFFFFFFFu : 0xFFFFu;
#pragma unroll
                for (int s = 1; s < 4 * F; s <<= 1) sum += __shfl_xor_sync(here, sum, s);
                if ((r & (4 * F - 1)) == 0) asum[(q * (4 / F) + r / (4 * F)) * p.cols + col + part] = sum;
            }
        }
    }
    __syncthreads();
    if (!busy) return;

    auto sync = [&]() { named_barrier_sync(1 + team, kTeamThreads); };
    auto to_float = [&](uint32_t word, uint32_t index) {    // index: the element's, counted from its 4-byte word
        return f32s ? __uint_as_float(word) : __uint_as_float((index & 1u) ? word & 0xFFFF0000u : word << 16);
    };
    const uint32_t sbase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(g.scale) >> 1);
    const uint32_t zflip = static_cast<uint32_t>(to_zero >> 1);
    const uint32_t ring_end = kSlots * p.slot_bytes;
    const unsigned char* act_lane = act + gr * 64 + t4 * 16;
    const uint32_t act_word = p.cols * 64;
    // The slots of K-range y.
    auto range_slots = [&](uint32_t y) {
        return p.ws + (static_cast<size_t>(blockIdx.z) * gridDim.y + y) * (p.tiles + gridDim.x * kTeams) * (16 * ROWS);
    };
    uint32_t tile = lo / nq, q0 = lo - tile * nq, done = lo;
    uint32_t slot = 0;      // byte offset in the ring
    while (done < hi) {
        const uint32_t n = hi - done < nq - q0 ? hi - done : nq - q0, q1 = q0 + n;
        float tot[NT][4] = {};
        uint32_t half[2];       // which half of its word a bf16 scale of group 0 is
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t row = tile * 16 + gr + 8 * h;
            half[h] = (row < static_cast<uint32_t>(g.N) ? row : g.N - 1) * static_cast<uint32_t>(g.lds) + sbase;
        }
        for (uint32_t q = q0 + warp; q < q1; q += kWarps) {
            cp_async_wait<kSlots - 1>();
            const unsigned char* src = ring + slot + lane * 16;
            const uint4 x0 = *reinterpret_cast<const uint4*>(src);
            const uint4 x1 = *reinterpret_cast<const uint4*>(src + 512);
            uint32_t w[2][4] = {{x0.x, x0.y, x0.z, x0.w}, {x1.x, x1.y, x1.z, x1.w}};
            const uint32_t gi = group_of((k_step0 + q) * 4 + t4);
            float sc[2], zr[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t* words = reinterpret_cast<const uint32_t*>(src - lane * 12 + 1024 + h * 128);
                sc[h] = to_float(words[0], half[h] + gi);
                zr[h] = zeros ? to_float(words[64], half[h] + gi + zflip) : 8.0f;
            }
            // The slot is free: its next step is requested before this one is worked on.
            request(slot);
            slot = slot + p.slot_bytes == ring_end ? 0 : slot + p.slot_bytes;

            // A product takes a word from each lane of a quad.  Lane t holds the four words of chunk t:
            // scales shared by fewer chunks want the words of one chunk (or two) on all four lanes.
            if constexpr (F <= 2) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {       // words 2, 3 of lanes 0, 1 for words 0, 1 of lanes 2, 3
                        const uint32_t give = (t4 & 2) ? w[h][i] : w[h][i + 2];
                        const uint32_t have = __shfl_xor_sync(0xFFFFFFFFu, give, 2);
                        if (t4 & 2) w[h][i] = have; else w[h][i + 2] = have;
                    }
            }
            if constexpr (F == 1) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {    // odd words of even lanes for even words of odd lanes
                        const uint32_t give = (t4 & 1) ? w[h][i] : w[h][i + 1];
                        const uint32_t have = __shfl_xor_sync(0xFFFFFFFFu, give, 1);
                        if (t4 & 1) w[h][i] = have; else w[h][i + 1] = have;
                    }
            }
#pragma unroll
            for (int f = 0; f < 4 / F; ++f) {
                float c[NT][4] = {};
#pragma unroll
                for (int i = 0; i < F; ++i) {
                    const int wi = f * F + i;
                    const uint32_t a0[4] = {decode<0, PARTS>(w[0][wi]), decode<0, PARTS>(w[1][wi]),
                                            decode<1, PARTS>(w[0][wi]), decode<1, PARTS>(w[1][wi])};
                    const uint32_t a1[4] = {decode<2, PARTS>(w[0][wi]), decode<2, PARTS>(w[1][wi]),
                                            decode<3, PARTS>(w[0][wi]), decode<3, PARTS>(w[1][wi])};
#pragma unroll
                    for (int b = 0; b < NT; ++b) {
                        uint4 x = make_uint4(0u, 0u, 0u, 0u);
                        if (8 * b + gr < cols) x = *reinterpret_cast<const uint4*>(act_lane + (q * 4 + wi) * act_word + b * 512);
                        mma_bf16(c[b], a0, x.x, x.y);
                        mma_bf16(c[b], a1, x.z, x.w);
                    }
                }
                float s0 = sc[0], s1 = sc[1], z0 = zr[0], z1 = zr[1];
                if constexpr (F < 4) {
                    const int from = (lane & 28) | (f * F);
                    s0 = __shfl_sync(0xFFFFFFFFu, s0, from);
                    s1 = __shfl_sync(0xFFFFFFFFu, s1, from);
                    if (zeros) {
                        z0 = __shfl_sync(0xFFFFFFFFu, z0, from);
                        z1 = __shfl_sync(0xFFFFFFFFu, z1, from);
                    }
                }
                const float off0 = PARTS ? z0 - 8.0f : z0 + 16.0f, off1 = PARTS ? z1 - 8.0f : z1 + 16.0f;
#pragma unroll
                for (int b = 0; b < NT; ++b) {
                    if (!PARTS || zeros) {
                        const int col = 8 * b + 2 * t4;
                        const float* as = asum + (q * (4 / F) + f) * p.cols + col;
                        const float u0 = col < cols ? as[0] : 0.0f, u1 = col + 1 < cols ? as[1] : 0.0f;
                        c[b][0] = fmaf(-off0, u0, c[b][0]);
                        c[b][1] = fmaf(-off0, u1, c[b][1]);
                        c[b][2] = fmaf(-off1, u0, c[b][2]);
                        c[b][3] = fmaf(-off1, u1, c[b][3]);
                    }
                    tot[b][0] = fmaf(s0, c[b][0], tot[b][0]);
                    tot[b][1] = fmaf(s0, c[b][1], tot[b][1]);
                    tot[b][2] = fmaf(s1, c[b][2], tot[b][2]);
                    tot[b][3] = fmaf(s1, c[b][3], tot[b][3]);
                }
            }
        }

        // --- the tile's end in this share: add up the warps
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[(warp * NT * 4 + b * 4 + e) * 32 + lane] = tot[b][e];
        sync();
        const bool whole = n == nq && gridDim.y == 1;
        float* part_sums = whole ? nullptr : range_slots(blockIdx.y) + part_slot(shares, share, tile, nq, p.tiles) * (16 * ROWS);
        for (int idx = tt; idx < 16 * mt; idx += kTeamThreads) {
            const int r = idx & 15, m = idx >> 4;
            const int64_t row = static_cast<int64_t>(tile) * 16 + r;
            if (row >= g.N) continue;
            float sum = 0.0f;
#pragma unroll
            for (int part = 0; part < (PARTS ? 3 : 1); ++part) {
                // The smallest parts first.
                const int col = PARTS ? 3 * m + 2 - part : m, b = col >> 3, e = (col & 1) + 2 * (r >> 3);
                const int ln = (r & 7) * 4 + ((col & 7) >> 1);
#pragma unroll
                for (int wv = 0; wv < kWarps; ++wv) sum += red[(wv * NT * 4 + b * 4 + e) * 32 + ln];
            }
            if ((*odd >> m) & 1u) {
                const T* a = static_cast<const T*>(g.A) + (m0 + m) * g.lda;
                const int64_t k1 = static_cast<int64_t>(k_step0 + q1) * kStepK < g.K ? static_cast<int64_t>(k_step0 + q1) * kStepK : g.K;
                for (int64_t k = static_cast<int64_t>(k_step0 + q0) * kStepK; k < k1; ++k) {
                    const float v = static_cast<float>(a[k]);
                    if (fabsf(v) <= 3.402823466e38f) continue;
                    const uint32_t code = (g.W[row * g.ldw + k / 2] >> (4 * (k & 1))) & 15u;
                    const int64_t e = row * g.lds + k / g.group;
                    auto value = [&](const void* s) {
                        return f32s ? static_cast<const float*>(s)[e] : __bfloat162float(static_cast<const __nv_bfloat16*>(s)[e]);
                    };
                    sum += v * (value(g.scale) * (static_cast<float>(code) - (zeros ? value(g.zero) : 8.0f)));
                }
            }
            if (whole) {
                const float out = sum + (g.bias ? g.bias[row] : 0.0f);
                static_cast<T*>(g.C)[(m0 + m) * g.ldc + row] = static_cast<T>(out);
            } else {
                part_sums[idx] = sum;
            }
        }
        sync();
        done += n;
        if (done < hi) { ++tile; q0 = 0; }
    }
    cp_async_wait<0>();

    // --- tiles that other shares worked on too: the last to arrive adds the parts, K-range after
    // K-range and share after share, so that the sum does not depend on who that is
    const uint32_t tile0 = lo / nq;
    uint32_t* last = reinterpret_cast<uint32_t*>(red);
    for (uint32_t t0 = tile0; t0 <= tile; t0 += kTeamThreads) {
        const uint32_t t = t0 + tt;
        if (t <= tile) {
            uint32_t parts = 0;
            if (gridDim.y > 1 || t * nq < lo || (t + 1) * nq > hi) {
                for (uint32_t y = 0; y < gridDim.y; ++y) {
                    const uint32_t ny = p.steps - y * per < per ? p.steps - y * per : per;
                    const Shares sy(p.tiles * ny, gridDim.x * kTeams);
                    parts += sy.holder(t * ny + ny - 1) - sy.holder(t * ny) + 1;
                }
                uint32_t* ticket = p.tickets + static_cast<size_t>(blockIdx.z) * p.tiles + t;
                if (atom_add_acq_rel_gpu_u32(ticket, 1u) == parts - 1) *ticket = 0u;
                else parts = 0;
            }
            last[tt] = parts;
        }
        sync();
        for (uint32_t i = 0; i < kTeamThreads && t0 + i <= tile; ++i) {
            if (last[i] == 0) continue;
            const uint32_t at = t0 + i;
            for (int idx = tt; idx < 16 * mt; idx += kTeamThreads) {
                const int r = idx & 15, m = idx >> 4;
                const int64_t row = static_cast<int64_t>(at) * 16 + r;
                if (row >= g.N) continue;
                float sum = 0.0f;
                for (uint32_t y = 0; y < gridDim.y; ++y) {
                    const uint32_t ny = p.steps - y * per < per ? p.steps - y * per : per;
                    const Shares sy(p.tiles * ny, gridDim.x * kTeams);
                    const uint32_t s0 = sy.holder(at * ny), s1 = sy.holder(at * ny + ny - 1);
                    const float* base = range_slots(y) + idx;
#pragma unroll 4
                    for (uint32_t s = s0; s <= s1; ++s)
                        sum += __ldcg(base + (s == s0 ? at : p.tiles + s) * static_cast<size_t>(16 * ROWS));
                }
                static_cast<T*>(g.C)[(m0 + m) * g.ldc + row] = static_cast<T>(sum + (g.bias ? g.bias[row] : 0.0f));
            }
        }
        sync();
    }
}

struct Kernel {
    const void* fn;
    int nt, rows, flush;
};

template <DType IO, int NT>
Kernel kernel_for_flush(int f) {
    const int rows = IO == DType::F32 ? NT * 8 / 3 : NT * 8;
    const void* fn = f == 4 ? reinterpret_cast<const void*>(&gemm_w4_kernel<IO, NT, 4>)
                     : f == 2 ? reinterpret_cast<const void*>(&gemm_w4_kernel<IO, NT, 2>)
                              : reinterpret_cast<const void*>(&gemm_w4_kernel<IO, NT, 1>);
    return {fn, NT, rows, f};
}

Kernel select(const W4Args& g) {
    // How many chunks of 32 weights share their scales for sure, up to the four of a step.
    const int f = g.groups == 1 || g.group % 128 == 0 ? 4 : (g.group % 64 == 0 ? 2 : 1);
    if (g.io == DType::F32)
        return g.M <= 2 ? kernel_for_flush<DType::F32, 1>(f)
               : g.M <= 5 ? kernel_for_flush<DType::F32, 2>(f) : kernel_for_flush<DType::F32, 3>(f);
    return g.M <= 8 ? kernel_for_flush<DType::BF16, 1>(f)
           : g.M <= 16 ? kernel_for_flush<DType::BF16, 2>(f) : kernel_for_flush<DType::BF16, 4>(f);
}

}  // namespace

bool gemm_w4_plan(const W4Args& g, int num_sms, W4Plan* plan) {
    const Kernel k = select(g);
    const int rows = g.M < k.rows ? g.M : k.rows;
    const int64_t steps = (static_cast<int64_t>(g.K) + kStepK - 1) / kStepK, tiles = (static_cast<int64_t>(g.N) + 15) / 16;
    plan->cols = g.io == DType::F32 ? 3 * rows : rows;
    plan->slot_bytes = 1024 + 256 + (g.zero ? 256 : 0);
    // As much of K at a time as the activations leave room for beside the rings.
    const int fixed = kTeams * kWarps * (kSlots * plan->slot_bytes + k.nt * 512) + 64;
    const int per_step = plan->cols * (256 + 4 * (4 / k.flush));
    const int64_t most = (kMaxSmem - fixed) / per_step;
    const int64_t splits = (steps + most - 1) / most;
    plan->split_steps = static_cast<int>((steps + splits - 1) / splits);
    plan->splits = static_cast<int>((steps + plan->split_steps - 1) / plan->split_steps);
    plan->smem = fixed + per_step * plan->split_steps;
    plan->blocks = (g.M + k.rows - 1) / k.rows;
    // Every SM a CTA, shared among the K-ranges; no more than there are shares of eight steps.
    int64_t ctas = (num_sms + plan->splits - 1) / plan->splits;
    const int64_t shares = (tiles * plan->split_steps + kWarps - 1) / kWarps;
    if (ctas > shares) ctas = shares;
    plan->ctas = static_cast<int>(ctas);
    // Steps are counted in 32 bits; blocks and splits are grid dimensions.
    if (tiles * plan->split_steps > INT32_MAX || plan->splits > 65535 || plan->blocks > 65535) return false;
    plan->ws_floats = static_cast<size_t>(plan->blocks) * plan->splits * (tiles + ctas * kTeams) * 16 * k.rows;
    plan->tickets = static_cast<size_t>(plan->blocks) * tiles;
    return true;
}

cudaError_t launch_gemm_w4(const W4Args& g, const W4Plan& plan, float* ws, uint32_t* tickets, cudaStream_t s) {
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
    p.tiles = (g.N + 15) / 16;
    p.steps = static_cast<int>((static_cast<int64_t>(g.K) + kStepK - 1) / kStepK);
    p.split_steps = plan.split_steps;
    p.slot_bytes = plan.slot_bytes;
    p.cols = plan.cols;
    // chunk / (group / 32) for chunks below 2^31: mul = ceil(2^(31 + ceil(log2 d)) / d).
    const int64_t d = g.groups > 1 ? g.group / 32 : int64_t(1) << 30;
    int log = 0;
    while ((int64_t(1) << log) < d) ++log;
    p.gmul = d == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << (31 + log)) + d - 1) / d);
    p.gshift = log > 0 ? log - 1 : 0;
    p.ws = ws;
    p.tickets = tickets;
    void* args[] = {&p};
    return cudaLaunchKernel(k.fn, dim3(plan.ctas, plan.splits, plan.blocks), dim3(kTeams * kTeamThreads), args,
                            static_cast<size_t>(plan.smem), s);
}

}  // namespace dnnopt_b200
