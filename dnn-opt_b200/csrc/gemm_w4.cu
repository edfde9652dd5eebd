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
// Work.  128 weights of 16 rows (1 KB) are a step, one TMA box into the ring of the
// warp that works on it (16-byte cp.async of the same rows cost 23 shared-memory
// cycles an instruction and held the kernel at 1.6 TB/s).  All steps, tile after tile
// of 16 rows, are cut into equal shares, one for each team of eight warps, two
// teams to an SM; a team's warps take the steps of a tile in turn and add up
// in shared memory.  A tile cut by a share's end, or by the ends of a K-range, is
// finished by the last of its shares to arrive, adding the parts in order.  The
// activations of the K-range sit in shared memory in the order in which the
// operand reads them.
#include <cuda.h>

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
constexpr int kMaxSlots = 8;        // steps under way per warp, where the activations leave room
constexpr int kMinSlots = 4;
constexpr int kStepK = 128;
constexpr int kStepBytes = 1024;
constexpr int kMaxSmem = 227 * 1024;

struct Params {
    W4Args g;
    int tiles;                      // of 16 rows of W
    int steps;                      // ceil(K / 128)
    int split_steps;                // steps of one K-range (gridDim.y of them)
    int slots;                      // of a warp's ring
    int aligned;                    // rows of W start at multiples of 16 bytes: the map below holds
    int cols;                       // columns of activations: rows of A, or three parts of each
    uint32_t gmul, gshift;          // chunk of 32 weights -> group
    float* ws;                      // partial tiles, see part_slot
    uint32_t* tickets;              // one per tile and block of rows of A
    uint32_t* err;                  // receives kKerrMbarTimeout
};

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
__global__ void __launch_bounds__(kTeams * kTeamThreads, 1)
gemm_w4_kernel(const Params p, const __grid_constant__ CUtensorMap map) {
    using T = typename std::conditional<IO == DType::F32, float, __nv_bfloat16>::type;
    constexpr bool PARTS = IO == DType::F32;
    constexpr int ROWS = PARTS ? NT * 8 / 3 : NT * 8;       // rows of A per pass
    constexpr int RED = NT * 128;                           // floats of a warp's sums of a tile
    extern __shared__ __align__(128) unsigned char smem[];
    const W4Args& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31, team = tid / kTeamThreads, tt = tid % kTeamThreads, warp = tt >> 5;
    const int gr = lane >> 2, t4 = lane & 3;
    const int m0 = blockIdx.z * ROWS, mt = g.M - m0 < ROWS ? g.M - m0 : ROWS;
    const int cols = PARTS ? 3 * mt : mt;
    const int k_step0 = blockIdx.y * p.split_steps;
    const uint32_t nq = p.steps - k_step0 < p.split_steps ? p.steps - k_step0 : p.split_steps;
    const uint32_t per = static_cast<uint32_t>(p.split_steps);

    unsigned char* ring = smem + (team * kWarps + warp) * p.slots * kStepBytes;
    unsigned char* act = smem + kTeams * kWarps * p.slots * kStepBytes;
    float* asum = reinterpret_cast<float*>(act + static_cast<size_t>(per) * p.cols * 256);   // [step][flush][col]
    float* red = asum + per * (4 / F) * p.cols + team * 2 * kWarps * RED;                    // [2][warp][4 NT][lane]
    uint64_t* bars = reinterpret_cast<uint64_t*>(
        (reinterpret_cast<uintptr_t>(asum + per * (4 / F) * p.cols + kTeams * 2 * kWarps * RED) + 7) & ~uintptr_t(7));
    uint32_t* odd = reinterpret_cast<uint32_t*>(bars + kTeams * kWarps * kMaxSlots);    // rows of A with an infinity or NaN
    bars += (team * kWarps + warp) * kMaxSlots;
    const bool zeros = g.zero != nullptr;
    const bool f32s = g.st == DType::F32;
    const int row_bytes = (g.K + 1) / 2;

    const Shares shares(p.tiles * nq, gridDim.x * kTeams);
    const uint32_t share = team * gridDim.x + blockIdx.x;
    const bool busy = share < shares.n;
    const uint32_t lo = busy ? shares.start(share) : 0, hi = busy ? shares.start(share + 1) : 0;

    // --- producer: one step's weights, lane (g, t) two rows of the tile and 32 weights of each
    if (lane == 0)
        for (int i = 0; i < p.slots; ++i) mbar_init(bars + i, 1);
    if (tid == 0) *odd = 0u;
    fence_mbar_init();
    __syncwarp();
    Cursor prod(lo, hi, nq, warp);
    auto request = [&](int slot) {      // the warp's next step, into a slot that it is done with
        if (prod.q < prod.end) {
            if (p.aligned) {
                if (lane == 0) {
                    mbar_arrive_expect_tx(bars + slot, kStepBytes);
                    tma_load_2d(ring + slot * kStepBytes, &map, bars + slot, static_cast<int>((k_step0 + prod.q) * 64),
                                static_cast<int>(prod.tile * 16));
                }
            } else {
                // Rows that start anywhere: whole 4-byte words that hold at least one byte of the row.
                const uint32_t at = ((k_step0 + prod.q) * 4 + t4) * 16;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    int64_t n = static_cast<int64_t>(prod.tile) * 16 + gr + 8 * h;
                    if (n >= g.N) n = g.N - 1;
                    const uintptr_t row = reinterpret_cast<uintptr_t>(g.W) + n * g.ldw, from = row + at, end = row + row_bytes;
                    const uint32_t* a4 = reinterpret_cast<const uint32_t*>(from & ~uintptr_t(3));
                    uint32_t x[5];
#pragma unroll
                    for (int i = 0; i < 5; ++i)
                        x[i] = from < end && reinterpret_cast<uintptr_t>(a4 + i) < end ? __ldg(a4 + i) : 0u;
                    const uint32_t sh = static_cast<uint32_t>(from & 3) * 8;
                    *reinterpret_cast<uint4*>(ring + slot * kStepBytes + lane * 16 + h * 512) =
                        make_uint4(__funnelshift_r(x[0], x[1], sh), __funnelshift_r(x[1], x[2], sh),
                                   __funnelshift_r(x[2], x[3], sh), __funnelshift_r(x[3], x[4], sh));
                }
            }
            prod.q += kWarps;
            if (prod.q >= prod.end) prod.settle(nq, warp);
        }
    };
    for (int s = 0; s < p.slots; ++s) request(s);

    // --- the K-range's activations: as bf16 in the operand's order, and their sums over each stretch
    // of F chunks.  Half a warp takes 128 activations of a row, eight to a lane.
    __syncthreads();
    {
        const bool vec = g.lda % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(g.A) % 16 == 0;
        const uint32_t units = mt * nq, r = tid & 15;
        // Which word of which lane these eight weights are, after the exchanges below.
        const uint32_t w = F == 4 ? (r & 3) : (F == 1 ? (r >> 2) : ((r >> 3) * 2 + (r & 1)));
        const uint32_t t = F == 4 ? (r >> 2) : (F == 1 ? (r & 3) : (((r >> 2) & 1) + (r & 2)));
        uint32_t u = tid >> 4, m = u / nq, q = u - m * nq;
        const uint32_t dm = (kTeams * kTeamThreads / 16) / nq, dq = (kTeams * kTeamThreads / 16) - dm * nq;
        for (uint32_t u0 = u & ~1u; u0 < units; u0 += kTeams * kTeamThreads / 16) {     // the same count for a whole warp
            const bool in = u < units;
            const int64_t k = static_cast<int64_t>(k_step0 + q) * kStepK + r * 8;
            const T* a = static_cast<const T*>(g.A) + static_cast<int64_t>(m0 + m) * g.lda + k;
            const uint32_t col = PARTS ? 3 * m : m;
            unsigned char* dst = act + ((q * 4 + w) * p.cols + col) * 64 + t * 16;
            float* sums = asum + (q * (4 / F) + r / (4 * F)) * p.cols + col;
            if constexpr (PARTS) {
                float v[8] = {};
                if (in) {
                    if (vec && k + 8 <= g.K) {
                        const float4 x = __ldg(reinterpret_cast<const float4*>(a)), y = __ldg(reinterpret_cast<const float4*>(a) + 1);
                        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                        v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = k + i < g.K ? a[i] : 0.0f;
                    }
                }
                bool bad = false;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(fabsf(v[i]) <= 3.402823466e38f)) { v[i] = 0.0f; bad = true; }
                if (bad) atomicOr(odd, 1u << m);
#pragma unroll
                for (int part = 0; part < 3; ++part) {
                    uint32_t o[4];
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[i] = __byte_perm(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), 0x7632);
                        const float hx = __uint_as_float(o[i] << 16), hy = __uint_as_float(o[i] & 0xFFFF0000u);
                        sum += hx + hy;
                        v[i] -= hx;
                        v[i + 4] -= hy;
                    }
                    if (in) *reinterpret_cast<uint4*>(dst + part * 64) = make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
                    for (int s = 1; s < 4 * F; s <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
                    if (in && (r & (4 * F - 1)) == 0) sums[part] = sum;
                }
            } else {
                uint32_t x[4] = {};
                if (in) {
                    if (vec && k + 8 <= g.K) {
                        const uint4 y = __ldg(reinterpret_cast<const uint4*>(a));
                        x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
                    } else {
                        const uint16_t* b = reinterpret_cast<const uint16_t*>(a);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (k + i < g.K) x[i >> 1] |= static_cast<uint32_t>(b[i]) << (16 * (i & 1));
                    }
                }
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += __uint_as_float(x[i] << 16) + __uint_as_float(x[i] & 0xFFFF0000u);
                if (!(fabsf(sum) <= 3.402823466e38f)) {
                    // An infinity or NaN among them, or finite values whose sum is none: all go the long way.
                    atomicOr(odd, 1u << m);
                    sum = 0.0f;
                    x[0] = x[1] = x[2] = x[3] = 0u;
                }
                if (in)
                    *reinterpret_cast<uint4*>(dst) = make_uint4(__byte_perm(x[0], x[2], 0x5410), __byte_perm(x[0], x[2], 0x7632),
                                                                __byte_perm(x[1], x[3], 0x5410), __byte_perm(x[1], x[3], 0x7632));
#pragma unroll
                for (int s = 1; s < 4 * F; s <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
                if (in && (r & (4 * F - 1)) == 0) sums[0] = sum;
            }
            u += kTeams * kTeamThreads / 16;
            m += dm;
            q += dq;
            if (q >= nq) { q -= nq; ++m; }
        }
    }
    __syncthreads();
    if (!busy) return;

    auto sync = [&]() { named_barrier_sync(1 + team, kTeamThreads); };
    // A scale or zero point as it lies in memory (bf16: in the low half), and its value.
    const int up = f32s ? 0 : 16;
    auto fetch = [&](const void* base, int64_t e) -> uint32_t {
        return f32s ? __ldg(static_cast<const uint32_t*>(base) + e) : __ldg(static_cast<const uint16_t*>(base) + e);
    };
    auto value = [&](uint32_t raw) { return __uint_as_float(raw << up); };
    auto group_of = [&](uint32_t chunk) {
        const int gi = p.gmul ? static_cast<int>(__umulhi(chunk, p.gmul) >> p.gshift) : static_cast<int>(chunk);
        return gi < g.groups ? gi : g.groups - 1;
    };
    // The slots of K-range y.
    auto range_slots = [&](uint32_t y) {
        return p.ws + (static_cast<size_t>(blockIdx.z) * gridDim.y + y) * (p.tiles + gridDim.x * kTeams) * (16 * ROWS);
    };

    const unsigned char* act_lane = act + gr * 64 + t4 * 16;
    const uint32_t act_word = p.cols * 64;
    uint32_t tile = lo / nq, q0 = lo - tile * nq, done = lo;
    uint32_t phase = 0, buffer = 0;
    int slot = 0;
    bool dead = false;
    while (done < hi) {
        const uint32_t n = hi - done < nq - q0 ? hi - done : nq - q0, q1 = q0 + n;
        int64_t srow[2];        // the lane's two rows' first scales
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t row = static_cast<int64_t>(tile) * 16 + gr + 8 * h;
            srow[h] = (row < g.N ? row : g.N - 1) * g.lds;
        }
        // A step's scales are read one step ahead; here the tile's come into L2.
        uint32_t raw[2] = {0, 0}, rawz[2] = {0, 0};
        auto scales_of = [&](uint32_t q) {
            const int gi = group_of((k_step0 + q) * 4 + t4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                raw[h] = fetch(g.scale, srow[h] + gi);
                if (zeros) rawz[h] = fetch(g.zero, srow[h] + gi);
            }
        };
        if (q0 + warp < q1) scales_of(q0 + warp);
        float tot[NT][4] = {};
        for (uint32_t q = q0 + warp; q < q1; q += kWarps) {
            float sc[2], zr[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sc[h] = value(raw[h]);
                zr[h] = zeros ? value(rawz[h]) : 8.0f;
            }
            if (q + kWarps < q1) scales_of(q + kWarps);
            if (p.aligned && !mbar_try_wait(bars + slot, phase) && !dead) dead = !mbar_wait(bars + slot, phase, nullptr, p.err);
            const unsigned char* src = ring + slot * kStepBytes + lane * 16;
            const uint4 x0 = *reinterpret_cast<const uint4*>(src);
            const uint4 x1 = *reinterpret_cast<const uint4*>(src + 512);
            uint32_t w[2][4] = {{x0.x, x0.y, x0.z, x0.w}, {x1.x, x1.y, x1.z, x1.w}};
            __syncwarp();
            request(slot);      // every lane has read it
            if (++slot == p.slots) { slot = 0; phase ^= 1u; }

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
            const unsigned char* act_q = act_lane + q * 4 * act_word;
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
                        if (8 * b + gr < cols) x = *reinterpret_cast<const uint4*>(act_q + wi * act_word + b * 512);
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

        // --- the tile's end in this share: add up the warps.  Two buffers in turn: whoever writes one
        // again has passed the barrier that follows its last reading.
        float* sums = red + buffer * kWarps * RED;
        buffer ^= 1u;
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[(warp * NT * 4 + b * 4 + e) * 32 + lane] = tot[b][e];
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
                for (int wv = 0; wv < kWarps; ++wv) sum += sums[(wv * NT * 4 + b * 4 + e) * 32 + ln];
            }
            if ((*odd >> m) & 1u) {
                // The activations that stayed out: each stretch of eight that is not finite as a whole.
                const T* a = static_cast<const T*>(g.A) + static_cast<int64_t>(m0 + m) * g.lda;
                const int64_t k1 = static_cast<int64_t>(k_step0 + q1) * kStepK < g.K ? static_cast<int64_t>(k_step0 + q1) * kStepK : g.K;
                for (int64_t k = static_cast<int64_t>(k_step0 + q0) * kStepK; k < k1; ++k) {
                    const float v = static_cast<float>(a[k]);
                    bool out = !(fabsf(v) <= 3.402823466e38f);
                    if (!PARTS) {
                        float eight[8], s8 = 0.0f;
                        for (int i = 0; i < 8; ++i) eight[i] = (k & ~7) + i < g.K ? static_cast<float>(a[(k & ~7) + i]) : 0.0f;
                        for (int i = 0; i < 8; i += 2) s8 += eight[i] + eight[i + 1];
                        out = !(fabsf(s8) <= 3.402823466e38f);
                    }
                    if (!out) continue;
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
        done += n;
        if (done < hi) { ++tile; q0 = 0; }
    }
    sync();

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
                static_cast<T*>(g.C)[static_cast<int64_t>(m0 + m) * g.ldc + row] = static_cast<T>(sum + (g.bias ? g.bias[row] : 0.0f));
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

// W as bytes [N][(K+1)/2], read in boxes of 64 bytes x 16 rows; bytes and rows past the ends read as zeros.
bool encode_weights(const W4Args& g, CUtensorMap* map) {
    EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>((static_cast<int64_t>(g.K) + 1) / 2), static_cast<cuuint64_t>(g.N)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(g.ldw)};
    const cuuint32_t box[2] = {64, 16}, one[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(g.W), dims, strides, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool gemm_w4_plan(const W4Args& g, int num_sms, W4Plan* plan) {
    const Kernel k = select(g);
    const int rows = g.M < k.rows ? g.M : k.rows;
    const int64_t steps = (static_cast<int64_t>(g.K) + kStepK - 1) / kStepK, tiles = (static_cast<int64_t>(g.N) + 15) / 16;
    plan->cols = g.io == DType::F32 ? 3 * rows : rows;
    // As much of K at a time as the activations leave room for beside the smallest rings; the rings
    // take what is left.
    const int warps = kTeams * kWarps;
    const int fixed = warps * (2 * k.nt * 512 + kMaxSlots * 8) + 64;
    const int per_step = plan->cols * (256 + 4 * (4 / k.flush));
    const int64_t most = (kMaxSmem - fixed - warps * kMinSlots * kStepBytes) / per_step;
    const int64_t splits = (steps + most - 1) / most;
    plan->split_steps = static_cast<int>((steps + splits - 1) / splits);
    plan->splits = static_cast<int>((steps + plan->split_steps - 1) / plan->split_steps);
    const int rest = (kMaxSmem - fixed - per_step * plan->split_steps) / (warps * kStepBytes);
    plan->slots = rest < kMaxSlots ? rest : kMaxSlots;
    plan->smem = fixed + per_step * plan->split_steps + warps * plan->slots * kStepBytes;
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

cudaError_t launch_gemm_w4(const W4Args& g, const W4Plan& plan, float* ws, uint32_t* tickets, uint32_t* err,
                           cudaStream_t s) {
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
    p.slots = plan.slots;
    p.cols = plan.cols;
    // chunk / (group / 32) for chunks below 2^31: mul = ceil(2^(31 + ceil(log2 d)) / d).
    const int64_t d = g.groups > 1 ? g.group / 32 : int64_t(1) << 30;
    int log = 0;
    while ((int64_t(1) << log) < d) ++log;
    p.gmul = d == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << (31 + log)) + d - 1) / d);
    p.gshift = log > 0 ? log - 1 : 0;
    p.ws = ws;
    p.tickets = tickets;
    p.err = err;
    CUtensorMap map = {};
    p.aligned = g.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(g.W) % 16 == 0 && encode_weights(g, &map);
    void* args[] = {&p, &map};
    return cudaLaunchKernel(k.fn, dim3(plan.ctas, plan.splits, plan.blocks), dim3(kTeams * kTeamThreads), args,
                            static_cast<size_t>(plan.smem), s);
}

}  // namespace dnnopt_b200
