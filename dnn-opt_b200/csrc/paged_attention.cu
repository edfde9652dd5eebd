// Attention of one new token per sequence over a paged key-value cache.
//
// Mathematics.  A head's output is sum_j exp(s_j - M) v_j / sum_j exp(s_j - M);
// numerator and denominator are sums over tokens, so any part of the tokens
// yields (m, l, O) = (max s, sum exp(s - m), sum exp(s - m) v) and two parts
// join as m = max, l = l1 e^(m1-m) + l2 e^(m2-m), O likewise.  Every warp keeps
// one running (m, l, O) over its tokens; warps join in shared memory, CTAs
// through the workspace.  Scores are kept in units of log 2.
//
// What bounds it: each cached element is read once and used by the 1-16 query
// heads of its group, far below the tensor rate, so HBM.  The products are
// mma.sync m16n8k16 with the tokens (scores) or the dimensions (output) as the
// 16 rows and eight heads as the columns, so that one head or eight cost the
// same and nothing is computed twice; a 128-row tcgen05 tile would have at
// most 16 of its rows or columns filled.
//
// Exactness.  bf16 products are exact and summed in FP32; weights exp(s - m)
// enter the second product as three bf16 parts, which hold all 24 bits.  E4M3
// keys and values are exact in f16: they are multiplied there, the query
// normalised by a power of two per head and the weights scaled by 2^7 so that
// neither leaves f16's range, and cut into two f16 parts (22 bits).  FP32 operands
// are cut into three bf16 parts each (24 bits, no loss); products below 2^-24
// of the largest are left out.  The matrix units truncate what they add to, so
// sums start from zero at every step, or now and then where that is dearer.
//
// The reference m of exp(s - m) moves only when a score exceeds it by 2^8:
// finding a tile's maximum takes six shuffles, asking whether any score
// exceeds a bound takes one vote.
//
// Work.  The tiles of all items (a sequence's heads that share a key) are cut
// into equal shares, one for each resident CTA, so that one long sequence or many
// ragged ones fill the GPU alike.  Each warp of a CTA has its own tokens of a tile
// and its own ring of cp.async stages: no barrier but at an item's end.  An item
// cut by shares is joined from the workspace by the last of them to arrive, in
// the parts' order, so that results do not depend on who that is.
//
// Measured, of 6.53 TB/s (bf16, 32 heads on 8 keys of 128 unless said): 1 x 131072
// tokens 89 us (92%), 64 ragged sequences up to 8192 159 us (96%), 16 heads to a
// key, 32 x 8192 112 us (73%), heads of 256, 1 x 65536 99 us (83%), 32 x 4096 183 us
// (90%); 32 x 8192 e4m3 104 us (79%: products, decoding and softmax of one-byte
// elements), FP32 16 heads of 64, 16 x 4096 106 us (78%); 8 x 1024 14.9 us, 1 x 17
// 5.5 us: start, first page number, first keys, join.
#include <cuda_fp8.h>

#include <mutex>
#include <type_traits>
#include <unordered_map>

#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;      // log2 by which a score may exceed the reference
constexpr float kUp = 7.0f;         // log2 of the scale of f16 weights: 2^(7 + 8) is below f16's 65504

struct Params {
    PagedAttnArgs a;
    float* ws;                      // partial results: two slots per share
    float* aside;                   // sums that warps have put aside
    uint32_t* tickets;              // one per item, then two per share
    int group, hpb, hblocks;        // heads per kv head; per item; items per kv head
    uint32_t page_mul, page_shift;  // pos / page_size = mulhi(pos, page_mul) >> page_shift (page_size > 1)
};

template <DType T> struct Io;
template <> struct Io<DType::F32> {
    using S = float;
    static __device__ __forceinline__ float get(S v) { return v; }
    static __device__ __forceinline__ S put(float v) { return v; }
};
template <> struct Io<DType::BF16> {
    using S = __nv_bfloat16;
    static __device__ __forceinline__ float get(S v) { return __bfloat162float(v); }
    static __device__ __forceinline__ S put(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    const int n = real ? 16 : 0;    // the rest is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c += x, two at a time.
__device__ __forceinline__ void add4(float (&c)[4], const float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2)
        asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0,%1};\n\tmov.b64 b, {%2,%3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0,%1}, a;\n\t}"
            : "+f"(c[i]), "+f"(c[i + 1]) : "f"(x[i]), "f"(x[i + 1]));
}

// Transposes an 8 x 8 matrix of 16-bit elements over the warp's lanes.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
__device__ __forceinline__ float hi16(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }
// The upper halves of two floats (truncation to bf16), x in the low half.
__device__ __forceinline__ uint32_t pack_hi16(float x, float y) {
    return prmt(__float_as_uint(x), __float_as_uint(y), 0x7632);
}
// x and y cut into three bf16 parts that add up to them.
__device__ __forceinline__ void cut3(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {
    h = pack_hi16(x, y);
    x -= hi16(x);
    y -= hi16(y);
    m = pack_hi16(x, y);
    l = pack_hi16(x - hi16(x), y - hi16(y));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack_rn(float x, float y) {
    uint32_t r;
    if constexpr (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
// x and y as a rounded f16 part and what it leaves.
__device__ __forceinline__ void cut2(float x, float y, uint32_t& h, uint32_t& l) {
    h = pack_rn<true>(x, y);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    l = pack_rn<true>(x - f.x, y - f.y);
}
// The power of two that brings `top` to [1, 2); 1 for zero, denormal and infinite values.
__device__ __forceinline__ float to_unit(float top) {
    uint32_t e = __float_as_uint(top) >> 23;
    if (e == 0 || e >= 254) e = 127;
    return __uint_as_float((254 - e) << 23);
}
// Four E4M3 bytes as f16, exactly.
__device__ __forceinline__ void e4m3x4_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(four));
}

// Tile geometry of one instantiation.  DP: head_dim rounded up to 64, 128 or
// 256; NT: blocks of eight heads per item.
template <DType CT, int DP, int NT>
struct Geo {
    static constexpr int EC = CT == DType::F32 ? 4 : (CT == DType::BF16 ? 2 : 1);
    static constexpr int HEADS = 8 * NT;                           // heads per item
    static constexpr int PITCH = DP * EC;                          // bytes of a cached row in shared memory
    // 16-token blocks per warp and tile: two where one would be only 2 KB of keys (32 x 8192 e4m3 tokens
    // of 128: 106 us, one block 127; of 64, 16 heads to a key: 57 and 69).
    static constexpr int MT = CT == DType::E4M3 && DP <= 128 ? 2 : 1;
    static constexpr int TOK = 16 * MT;
    static constexpr int KV = TOK * PITCH;                         // one warp's keys (or values) of a tile
    static constexpr int OUT = HEADS * DP * 4;                     // one warp's O at the end of an item
    static constexpr int WS = 2 * KV > OUT ? 2 * KV : OUT;         // one warp's part of a stage
    static constexpr int NW = WS >= 32768 ? 2 : 4;                 // warps
    static constexpr int TILE = NW * TOK;                          // tokens per tile
    // CTAs per SM: three where two stages fit three times and the registers (168 a thread) suffice
    // (64 ragged sequences up to 8192 160 us, two CTAs 167; 32 x 8192 e4m3 106 and 112; one sequence
    // of 131072 91 and 87).
    static constexpr int CTAS = WS * NW <= 32768 && DP <= 128 && NT == 1 ? 3
                                : (WS * NW <= 36 * 1024 ? 2 : 1);
    static constexpr int FIT = (CTAS == 3 ? 70 : (CTAS == 2 ? 108 : 216)) * 1024 / (WS * NW);
    static constexpr int STAGES = FIT > 4 ? 4 : FIT;
    static constexpr int QPARTS = CT == DType::F32 ? 3 : 1;
    static constexpr int QWORDS = 2 * QPARTS * NT;                 // 32-bit words of Q per lane and 16 dims
    static constexpr int QBYTES = DP / 16 * 32 * QWORDS * 4;
    static constexpr bool QREG = DP / 16 * QWORDS <= 32;           // queries stay in registers over an item
    static constexpr int SMALL = 2 * NW * 16 * 4 + 16 * 4 + STAGES * NW * 4 + 64;
    static constexpr int SMEM = STAGES * NW * WS + QBYTES + SMALL;
    static constexpr int PART = HEADS * (DP + 2);                  // floats of one partial result
    // Each step's products start from zero, or all sums of a CTA's warps are put aside now and then.
    static constexpr bool FRESH = CT == DType::F32 || (CT == DType::BF16 && DP <= 128);
    static constexpr int ASIDE = FRESH ? 0 : NW * HEADS * DP;
    static_assert(STAGES >= 2, "a pipeline needs two stages");
};

// Rotation of a row's 16-byte chunks.  bf16 rows are read by ldmatrix, eight
// rows of one chunk at a time; the others four chunks from two rows (keys) or
// two chunks from four even rows (values): all without bank conflicts.
template <DType CT, int PITCH>
__device__ __forceinline__ int rotation(int row) {
    int x;
    if constexpr (CT == DType::BF16) x = row & 7;
    else x = ((row & 6) ^ ((row & 1) << 2));
    if constexpr (PITCH == 64) x &= 3;
    return x;
}
// 16-byte chunk `c` of row `row` in a warp's tile.
template <DType CT, int PITCH>
__device__ __forceinline__ int chunk_at(int row, int c) { return row * PITCH + ((c ^ rotation<CT, PITCH>(row)) << 4); }

// First dimension of the pair that lane t of a quad holds in step s of the
// score product (the second pair follows at +8 / +2): the order of dimensions
// is free there as long as queries and keys agree.
template <DType CT>
__device__ __forceinline__ int q_dim(int s, int t) {
    if constexpr (CT == DType::BF16) return 16 * s + 2 * t;
    else if constexpr (CT == DType::E4M3) return 64 * (s >> 2) + 16 * t + 4 * (s & 3);
    else return 16 * s + 4 * t;
}
template <DType CT>
__device__ __forceinline__ int q_second() { return CT == DType::BF16 ? 8 : 2; }

// Dimensions of rows g and g + 8 of output block j.
template <DType CT>
__device__ __forceinline__ int o_dim(int j, int g) {
    if constexpr (CT == DType::BF16) return 16 * j + g;
    else if constexpr (CT == DType::E4M3) return 64 * (j >> 2) + 8 * g + 2 * (j & 3);
    else return 32 * (j >> 1) + 4 * g + 2 * (j & 1);
}
template <DType CT>
__device__ __forceinline__ int o_second() { return CT == DType::BF16 ? 8 : 1; }
// A warp's O in shared memory; the rotation keeps the four heads that it
// stores at once in different banks.
__device__ __forceinline__ int o_at(int head, int d, int pitch) { return head * pitch + (d ^ (((head >> 1) & 3) << 3)); }

// A tile's place: sequence, item of the sequence, tile of the item.
struct Cursor {
    int b, r, t;
    int tiles, first, len;          // of sequence b

    __device__ __forceinline__ void load(const Params& p, int tile_tokens) {
        len = __ldg(p.a.lens + b);
        if (len < 0 || len > static_cast<int64_t>(p.a.max_pages) * p.a.page_size) {
            record_kernel_error(p.a.err, kKerrBadIndex);    // a sequence may be one thread's alone
            len = 0;
        }
        first = p.a.window > 0 && len > p.a.window ? len - p.a.window : 0;
        tiles = (len - first + tile_tokens - 1) / tile_tokens;
    }
    __device__ __forceinline__ void next(const Params& p, int items, int tile_tokens) {
        if (++t < tiles) return;
        t = 0;
        if (++r < items) return;
        r = 0;
        do {
            if (++b >= p.a.batch) return;
            load(p, tile_tokens);
        } while (tiles == 0);
    }
};

// Every CTA takes one share of the tiles, equal but for one tile: the first
// `more` shares have one more than the others.
struct Shares {
    uint32_t ctas, each, more;

    __device__ Shares(uint32_t tiles, uint32_t grid) : ctas(tiles < grid ? tiles : grid) {
        each = tiles / ctas;
        more = tiles - each * ctas;
    }
    __device__ __forceinline__ uint32_t start(uint32_t c) const { return c * each + min(c, more); }
    // The share that holds tile t: the last one that starts at or before it.
    __device__ __forceinline__ uint32_t holder(uint32_t t) const {
        const uint32_t big = more * (each + 1);
        return t < big ? t / (each + 1) : more + (t - big) / each;
    }
};

template <DType IO, DType CT, int DP, int NT>
__global__ void __launch_bounds__(Geo<CT, DP, NT>::NW * 32, Geo<CT, DP, NT>::CTAS) paged_attention_kernel(const Params p) {
    using G = Geo<CT, DP, NT>;
    using I = Io<IO>;
    constexpr int NW = G::NW, S = G::STAGES, TILE = G::TILE, TOK = G::TOK, MT = G::MT, HEADS = G::HEADS;
    constexpr bool F16 = CT == DType::E4M3;
    constexpr int KSTEPS = DP / 16, QW = G::QWORDS;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* ring = smem;
    uint32_t* s_q = reinterpret_cast<uint32_t*>(smem + S * NW * G::WS);
    float* s_m = reinterpret_cast<float*>(smem + S * NW * G::WS + G::QBYTES);    // [NW][16]
    float* s_l = s_m + NW * 16;
    float* s_f = s_l + NW * 16;                                                  // [16] query scale per head
    uint32_t* s_mask = reinterpret_cast<uint32_t*>(s_f + 16);                    // [S][NW]
    int* s_find = reinterpret_cast<int*>(s_mask + S * NW);                       // [4], words passed between threads
    uint32_t* s_own = reinterpret_cast<uint32_t*>(s_find + 4);                   // [3]

    const PagedAttnArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int items = a.kv_heads * p.hblocks;
    const int dim = a.dim;
    pdl_wait();
    pdl_launch_dependents();

    // --- all tiles in (sequence, item, tile) order; a thread (a lane, for up to 32 sequences) knows
    // the tiles of its own sequences and of those before them
    const bool few = a.batch <= 32;
    const int per = few ? 1 : (a.batch + NW * 32 - 1) / (NW * 32);
    const int b0 = (few ? lane : tid) * per;
    uint32_t mine = 0;
    for (int i = 0; i < per && b0 + i < a.batch; ++i) {
        Cursor c;
        c.b = b0 + i;
        c.load(p, TILE);
        mine += c.tiles;
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += v;
    }
    uint32_t total = __shfl_sync(0xFFFFFFFFu, incl, 31);
    if (!few) {
        if (lane == 31) s_find[warp] = static_cast<int>(incl);
        __syncthreads();
        uint32_t before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += s_find[w];
            total += s_find[w];
        }
        incl += before;
        __syncthreads();
    }
    total *= items;

    // --- sequences without a token: zeros
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        uint32_t tiles = 0;
        if (few) {
            tiles = __shfl_sync(0xFFFFFFFFu, mine, b);
        } else {
            Cursor c;
            c.b = b;
            c.load(p, TILE);
            tiles = c.tiles;
        }
        if (tiles != 0) continue;
        constexpr int N = 16 / sizeof(typename I::S);
        typename I::S* out = static_cast<typename I::S*>(a.out) + b * a.out_batch;
        for (int i = tid; i < a.heads * (dim / N); i += NW * 32) {
            const int h = i / (dim / N), d = (i - h * (dim / N)) * N;
            *reinterpret_cast<uint4*>(out + h * a.out_head + d) = make_uint4(0u, 0u, 0u, 0u);
        }
        if (a.lse)
            for (int h = tid; h < a.heads; h += NW * 32) a.lse[static_cast<int64_t>(b) * a.heads + h] = -INFINITY;
    }
    if (total == 0) return;

    const Shares shares(total, gridDim.x);
    const uint32_t share = blockIdx.x, end = incl * items, start = (incl - mine) * items;
    uint32_t lo, hi, off0;
    Cursor cons;
    // Ending an item and beginning the next within a share costs about as much as two tiles.  So
    // with few items each gets CTAs of its own, if these then have at most two tiles more (8 x 1024
    // tokens 14.9 us, in equal shares some 2.4 more; 16 ragged windowed e4m3 sequences 31.9 and 35.7).
    bool own = false;
    if (few) {
        uint32_t most = (total + gridDim.x - 1) / gridDim.x, k = 0, sum = 0;
        for (int tries = 0; tries < 3 && !own; ++tries, ++most) {
            k = (mine + most - 1) / most;       // CTAs to each item of the lane's sequence
            sum = k * items;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
                if (lane >= o) sum += v;
            }
            own = __shfl_sync(0xFFFFFFFFu, sum, 31) <= gridDim.x;
        }
        if (own) {
            const uint32_t owners = __ballot_sync(0xFFFFFFFFu, share < sum);
            if (owners == 0) return;
            const int owner = __ffs(owners) - 1;
            cons.b = owner;
            k = __shfl_sync(0xFFFFFFFFu, k, owner);
            const uint32_t at = share - (__shfl_sync(0xFFFFFFFFu, sum, owner) - k * items);
            const uint32_t r = at / k, part = at - r * k;
            const uint32_t tiles = __shfl_sync(0xFFFFFFFFu, mine, owner), each = tiles / k, more = tiles - each * k;
            off0 = __shfl_sync(0xFFFFFFFFu, start, owner);
            lo = off0 + r * tiles + part * each + min(part, more);
            hi = lo + each + (part < more ? 1 : 0);
            if (tid == 0) {
                s_own[1] = share - part;
                s_own[2] = share - part + k - 1;
            }
        }
        if (tid == 0) s_own[0] = own;
    } else if (tid == 0) {
        s_own[0] = 0;
    }
    if (!own) {
        if (share >= shares.ctas) return;
        lo = shares.start(share);
        hi = shares.start(share + 1);
        if (few) {
            const int owner = __ffs(__ballot_sync(0xFFFFFFFFu, lane < a.batch && lo < end)) - 1;
            cons.b = owner;
            off0 = __shfl_sync(0xFFFFFFFFu, start, owner);
        } else {
            if (lo >= start && lo < end) {
                uint32_t at = start;
                Cursor c;
                c.b = b0;
                for (;; ++c.b) {
                    c.load(p, TILE);
                    if (lo < at + c.tiles * items) break;
                    at += c.tiles * items;
                }
                s_find[0] = c.b;
                s_find[1] = static_cast<int>(at);
            }
            __syncthreads();
            cons.b = s_find[0];
            off0 = s_find[1];
        }
    }
    __syncthreads();
    cons.load(p, TILE);
    cons.r = static_cast<int>((lo - off0) / cons.tiles);
    cons.t = static_cast<int>((lo - off0) % cons.tiles);
    uint32_t item0 = lo - cons.t;       // first tile of the current item
    Cursor prod = cons;

    // --- producer: one warp's tokens of one tile
    constexpr int LPR = G::PITCH / 16 < 8 ? G::PITCH / 16 : 8;      // lanes per row
    constexpr int RPP = 32 / LPR;                                   // rows per pass
    const int nch = dim * G::EC / 16, lrow = lane / LPR, lch = lane % LPR;
    struct Ask {            // where a tile's row `lane` is, asked two tiles ahead of its loads
        int ent, slot, b, r;
        bool want, fresh;
    };
    auto look = [&]() {
        Ask k;
        const int pos = prod.first + prod.t * TILE + warp * TOK + (lane & (TOK - 1));
        k.want = pos < prod.len;
        const int pg = a.page_size == 1 ? pos : static_cast<int>(__umulhi(pos, p.page_mul) >> p.page_shift);
        k.slot = pos - pg * a.page_size;
        k.ent = k.want ? __ldg(a.table + prod.b * a.table_stride + pg) : -1;
        k.fresh = a.k_new != nullptr && pos == prod.len - 1;
        k.b = prod.b;
        k.r = prod.r;
        return k;
    };
    auto issue = [&](int stage, const Ask& k) {
        const bool ok = k.want && k.ent >= 0 && k.ent < a.num_pages;
        if (k.want && !ok) record_kernel_error(a.err, kKerrBadIndex);
        uint32_t valid = __ballot_sync(0xFFFFFFFFu, ok);
        const uint32_t real = __ballot_sync(0xFFFFFFFFu, ok && !k.fresh);
        if constexpr (TOK < 32) valid &= 0xFFFFu;
        if (lane == 0) s_mask[stage * NW + warp] = valid;
        if (valid) {
            const int kvh = p.hblocks == 1 ? k.r : k.r / p.hblocks;
            const long long off = ok ? (k.ent * a.page_stride + k.slot * a.token_stride + kvh * a.head_stride) * G::EC : 0;
            const uint32_t base = smem_u32(ring + (stage * NW + warp) * G::WS) + lrow * G::PITCH;
#pragma unroll
            for (int i = 0; i < TOK / RPP; ++i) {
                const long long o = __shfl_sync(0xFFFFFFFFu, off, i * RPP + lrow) + lch * 16;
                const bool load = (real >> (i * RPP + lrow)) & 1u;
                if (CT != DType::E4M3 && ((valid & ~real) >> (i * RPP + lrow)) & 1u) continue;   // filled below
                const int x = rotation<CT, G::PITCH>((i * RPP) % 8 + lrow);
                const uint32_t dst = base + i * RPP * G::PITCH + ((lch ^ x) << 4);
                const char* ks = static_cast<const char*>(a.k) + o;
                const char* vs = static_cast<const char*>(a.v) + o;
#pragma unroll
                for (int u = 0; u < G::PITCH / 16 / LPR; ++u) {
                    // Rows that are not there and dimensions past head_dim become zeros: nothing of
                    // their addresses is read.
                    const bool in = load && u * LPR + lch < nch;
                    cp_async16(dst + u * LPR * 16, ks + u * LPR * 16, in);
                    cp_async16(dst + u * LPR * 16 + G::KV, vs + u * LPR * 16, in);
                }
            }
            if constexpr (CT != DType::E4M3) {
                if (valid & ~real) {
                    // The new token's row, from its own tensors.
                    const int row = __ffs(valid & ~real) - 1;
                    const int64_t from = k.b * a.new_batch + kvh * a.new_head;
                    const uint32_t dst = smem_u32(ring + (stage * NW + warp) * G::WS);
                    const char* kn = reinterpret_cast<const char*>(static_cast<const typename I::S*>(a.k_new) + from);
                    const char* vn = reinterpret_cast<const char*>(static_cast<const typename I::S*>(a.v_new) + from);
                    for (int c = lane; c < G::PITCH / 16; c += 32) {
                        const bool in = c < nch;
                        cp_async16(dst + chunk_at<CT, G::PITCH>(row, c), in ? kn + c * 16 : kn, in);
                        cp_async16(dst + G::KV + chunk_at<CT, G::PITCH>(row, c), in ? vn + c * 16 : vn, in);
                    }
                }
            }
        }
    };
    const int count = static_cast<int>(hi - lo);
    int issued = 0, asked = 0;
    Ask near_ask = {}, far_ask = {};
    auto ask = [&]() {
        near_ask = far_ask;
        if (asked < count) {
            far_ask = look();
            if (++asked < count) prod.next(p, items, TILE);
        }
    };
    auto request = [&](int stage) {     // the next tile's loads, into a stage that the warp is done with
        if (issued < count) {
            issue(stage, near_ask);
            ++issued;
            ask();
        }
        cp_async_commit();
    };
    ask();
    ask();
#pragma unroll
    for (int s = 0; s < S; ++s) request(s);

    // Lane (g, t) holds heads 2t and 2t + 1 of each block of eight, and of the queries head g.
    float acc[KSTEPS][NT][4], m[NT][2], l[NT][2], rowscale[NT][2];
    // The matrix units truncate what they add to, two or three times for every 16 tokens: together 2^-13 of
    // the sum of one CTA's 65536 tokens.  So each step's products start from zero and are added (FRESH), or,
    // where that takes longer, sums are put aside every 1024 tokens of a warp and start anew: one sequence
    // of 65536 tokens, heads of 256, 99 us (from zero 113, neither 96); 32 x 8192 e4m3 107 (109, 105); but
    // bf16, 16 heads of 128 to a key, 32 x 8192, 115 (112, 104).
    constexpr bool FRESH = G::FRESH;
    constexpr int RUN = 64 / MT;
    float* const aside = FRESH ? nullptr : p.aside + static_cast<size_t>(blockIdx.x * NW + warp) * (HEADS * DP) + lane * 4;
    float kept[NT][2];          // what the sums put aside are multiplied by: the reference has moved since
    bool held = false;          // there are some
    int run = 0;
    auto take_back = [&]() {
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float4 x = *reinterpret_cast<const float4*>(aside + (j * NT + n) * 128);
                acc[j][n][0] = fmaf(x.x, kept[n][0], acc[j][n][0]);
                acc[j][n][1] = fmaf(x.y, kept[n][1], acc[j][n][1]);
                acc[j][n][2] = fmaf(x.z, kept[n][0], acc[j][n][2]);
                acc[j][n][3] = fmaf(x.w, kept[n][1], acc[j][n][3]);
            }
    };
    auto put_aside = [&]() {
        if (held) take_back();
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float (&c)[4] = acc[j][n];
                *reinterpret_cast<float4*>(aside + (j * NT + n) * 128) = make_float4(c[0], c[1], c[2], c[3]);
                c[0] = c[1] = c[2] = c[3] = 0.0f;
            }
#pragma unroll
        for (int n = 0; n < NT; ++n) kept[n][0] = kept[n][1] = 1.0f;
        held = true;
        run = 0;
    };
    uint32_t qreg[G::QREG ? KSTEPS : 1][QW];
    const float cap2 = a.softcap * kLog2e;
    auto heads_of = [&](const Cursor& c, int64_t& head0) {
        const int kvh = p.hblocks == 1 ? c.r : c.r / p.hblocks, h0 = (c.r - kvh * p.hblocks) * p.hpb;
        head0 = static_cast<int64_t>(kvh) * p.group + h0;
        return p.group - h0 < HEADS ? p.group - h0 : HEADS;
    };
    // Two neighbouring query elements, as they lie in memory.
    using Pair = typename std::conditional<IO == DType::F32, float2, uint32_t>::type;
    Pair raw[G::QREG ? KSTEPS : 1][NT][2];
    auto fetch_queries = [&](const Cursor& c) {     // this warp's part of the loads
        if constexpr (G::QREG) {
            int64_t head0;
            const int nh = heads_of(c, head0);
            const typename I::S* q = static_cast<const typename I::S*>(a.q) + c.b * a.q_batch + head0 * a.q_head;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int d = q_dim<CT>(ks, t4) + e * q_second<CT>(), h = g + 8 * n;
                        raw[ks][n][e] = Pair{};
                        if (h < nh && d < dim) raw[ks][n][e] = __ldg(reinterpret_cast<const Pair*>(q + h * a.q_head + d));
                    }
        }
    };
    auto begin_item = [&](const Cursor& c) {
        float f8[NT];       // 8-bit caches: power of two that brings head g's largest |q| to [1, 2)
#pragma unroll
        for (int n = 0; n < NT; ++n) f8[n] = 1.0f;
        if constexpr (G::QREG) {
            if constexpr (CT == DType::E4M3) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float top = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(raw[ks][n][e] << 16)),
                                                   fabsf(__uint_as_float(raw[ks][n][e] & 0xFFFF0000u))));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    f8[n] = to_unit(top);
                }
            }
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if constexpr (CT == DType::BF16) qreg[ks][2 * n + e] = raw[ks][n][e];
                        else if constexpr (CT == DType::E4M3)
                            qreg[ks][2 * n + e] = pack_rn<true>(__uint_as_float(raw[ks][n][e] << 16) * f8[n],
                                                                __uint_as_float(raw[ks][n][e] & 0xFFFF0000u) * f8[n]);
                        else cut3(raw[ks][n][e].x, raw[ks][n][e].y, qreg[ks][6 * n + e], qreg[ks][6 * n + 2 + e], qreg[ks][6 * n + 4 + e]);
                    }
        } else {
            // Queries that do not fit the registers: one copy for the CTA, in the order of the operand.
            int64_t head0;
            const int nh = heads_of(c, head0);
            const typename I::S* q = static_cast<const typename I::S*>(a.q) + c.b * a.q_batch + head0 * a.q_head;
            if constexpr (CT == DType::E4M3) {
                for (int h = warp; h < HEADS; h += NW) {
                    float top = 0.0f;
                    if (h < nh)
                        for (int d = lane; d < dim; d += 32) top = fmaxf(top, fabsf(I::get(q[h * a.q_head + d])));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                    if (lane == 0) s_f[h] = to_unit(top);
                }
                __syncthreads();
#pragma unroll
                for (int n = 0; n < NT; ++n) f8[n] = s_f[g + 8 * n];
            }
            for (int ks = warp; ks < KSTEPS; ks += NW)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int d0 = q_dim<CT>(ks, t4), d1 = d0 + q_second<CT>(), h = g + 8 * n;
                    const typename I::S* qh = q + h * a.q_head;
                    uint32_t* dst = s_q + (ks * 32 + lane) * QW;
                    const float v0 = h < nh && d0 < dim ? I::get(qh[d0]) * f8[n] : 0.0f;
                    const float v1 = h < nh && d0 < dim ? I::get(qh[d0 + 1]) * f8[n] : 0.0f;
                    const float v2 = h < nh && d1 < dim ? I::get(qh[d1]) * f8[n] : 0.0f;
                    const float v3 = h < nh && d1 < dim ? I::get(qh[d1 + 1]) * f8[n] : 0.0f;
                    if constexpr (CT == DType::F32) {
                        cut3(v0, v1, dst[6 * n], dst[6 * n + 2], dst[6 * n + 4]);
                        cut3(v2, v3, dst[6 * n + 1], dst[6 * n + 3], dst[6 * n + 5]);
                    } else {
                        dst[2 * n] = pack_rn<F16>(v0, v1);
                        dst[2 * n + 1] = pack_rn<F16>(v2, v3);
                    }
                }
            __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[n][e] = -INFINITY;
                l[n][e] = 0.0f;
                kept[n][e] = 0.0f;
                float f = a.scale * a.k_scale;
                if constexpr (CT == DType::E4M3) f /= __shfl_sync(0xFFFFFFFFu, f8[n], 4 * (2 * t4 + e));    // exact
                rowscale[n][e] = a.softcap > 0.0f ? f / a.softcap : f * kLog2e;
            }
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j) acc[j][n][0] = acc[j][n][1] = acc[j][n][2] = acc[j][n][3] = 0.0f;
        }
    };

    // Where an item's parts are: its shares, and the slots of their partial results.
    struct Parts {
        uint32_t first, last, tail;     // an item that begins inside its first share is that share's last one
    };
    auto parts_of = [&](uint32_t item0, int tiles) {
        Parts r;
        if (s_own[0]) {
            r.first = s_own[1];
            r.last = s_own[2];
            r.tail = 0;
            return r;
        }
        r.first = shares.holder(item0);
        r.last = shares.holder(item0 + tiles - 1);
        r.tail = shares.start(r.first) < item0 ? 1 : 0;
        return r;
    };
    auto slot_of = [&](const Parts& r, uint32_t c) { return 2 * c + (c == r.first ? r.tail : 0); };
    // The parts that one CTA joins at a time, and the ticket that says who is the last of them: with
    // up to 32 parts all (1 x 2048 tokens, 32 parts: 11.5 us, in two steps a microsecond more), else groups of
    // neighbours, and then the groups (131072 tokens, 56 parts: 91 us, in one step 93).
    auto near_of = [](uint32_t n) { return n <= 32 ? n : (n <= 256 ? 16u : 32u); };
    auto first_ticket = [&](const Parts& r, const Cursor& c) {
        const uint32_t n = r.last - r.first + 1, near = near_of(n);
        return n <= near ? p.tickets + static_cast<int64_t>(c.b) * items + c.r
                         : p.tickets + static_cast<int64_t>(a.batch) * items + slot_of(r, r.first + (share - r.first) / near * near);
    };
    auto finish = [&](const Cursor& c, int row, int v, float4 sum, float M, float L) {
        int64_t head0;
        heads_of(c, head0);
        const float f = L == 0.0f ? 0.0f : __fdiv_rn(a.v_scale, L);
        typename I::S* dst = static_cast<typename I::S*>(a.out) + c.b * a.out_batch + (head0 + row) * a.out_head + 4 * v;
        typename I::S r[4] = {I::put(sum.x * f), I::put(sum.y * f), I::put(sum.z * f), I::put(sum.w * f)};
        if constexpr (sizeof(typename I::S) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(r);
        else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(r);
        if (v == 0 && a.lse)
            a.lse[static_cast<int64_t>(c.b) * a.heads + head0 + row] =
                L == 0.0f ? -INFINITY : (M + log2f(L) - (F16 ? kUp : 0.0f)) * kLn2;
    };
    constexpr int VPR = DP / 4, RPT = NW * 32 / VPR;        // threads per output row, rows at a time
    const int orow = tid / VPR, ov = tid % VPR;

    const Cursor head = cons;           // the first item: it may have begun in another share
    const uint32_t head_item0 = item0;
    uint32_t ticket0 = 0, ticket1 = 0;  // of the first and the last item, thread 0's
    bool partial0 = false, partial1 = false;
    int stage = 0;
    fetch_queries(cons);
    begin_item(cons);
    for (int i = 0; i < count; ++i) {
        cp_async_wait<S - 1>();
        __syncwarp();
        const uint32_t mask = s_mask[stage * NW + warp];
        unsigned char* kt = ring + (stage * NW + warp) * G::WS;
        if (mask) {
            if (a.k_new) {
                // --- the new token's row goes into the cache (8-bit caches: and into the tile, rounded)
                const int row = cons.len - 1 - (cons.first + cons.t * TILE + warp * TOK);
                if (row >= 0 && row < TOK && ((mask >> row) & 1u)) {
                    const int pos = cons.len - 1, pg = pos / a.page_size, kvh = cons.r / p.hblocks;
                    const long long off = __ldg(a.table + cons.b * a.table_stride + pg) * a.page_stride +
                                          (pos - pg * a.page_size) * a.token_stride + kvh * a.head_stride;
                    const bool keep = cons.r == kvh * p.hblocks;    // one item of the head stores it
                    for (int c = lane; c < 2 * nch; c += 32) {
                        const int which = c >= nch, ch = which ? c - nch : c;
                        uint4* tile = reinterpret_cast<uint4*>(kt + which * G::KV + chunk_at<CT, G::PITCH>(row, ch));
                        if constexpr (CT == DType::E4M3) {
                            const uint4* src = reinterpret_cast<const uint4*>(
                                static_cast<const typename I::S*>(which ? a.v_new : a.k_new) + cons.b * a.new_batch +
                                kvh * a.new_head + ch * 16);
                            const float div = which ? a.v_scale : a.k_scale;
                            const uint4 x = src[0], y = src[1];
                            const uint32_t in[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                            uint32_t o[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                o[e] = 0;
#pragma unroll
                                for (int f = 0; f < 2; ++f) {
                                    const float2 v = make_float2(__fdiv_rn(__uint_as_float(in[2 * e + f] << 16), div),
                                                                 __fdiv_rn(__uint_as_float(in[2 * e + f] & 0xFFFF0000u), div));
                                    o[e] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3)) << (16 * f);
                                }
                            }
                            *tile = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                        if (keep) *reinterpret_cast<uint4*>(static_cast<char*>(which ? a.v : a.k) + off * G::EC + ch * 16) = *tile;
                    }
                    __syncwarp();
                }
            }

            // --- scores: 16 tokens x 8 heads per block, four to a lane
            float s[MT][NT][4];
#pragma unroll
            for (int b = 0; b < MT; ++b)
#pragma unroll
                for (int n = 0; n < NT; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.0f;
            const uint32_t k32 = smem_u32(kt);
            auto query = [&](int ks, uint32_t (&q)[QW]) {
                if constexpr (G::QREG) {
#pragma unroll
                    for (int w = 0; w < QW; ++w) q[w] = qreg[ks][w];
                } else {
#pragma unroll
                    for (int w = 0; w < QW; w += 2) {
                        const uint2 v = *reinterpret_cast<const uint2*>(s_q + (ks * 32 + lane) * QW + w);
                        q[w] = v.x;
                        q[w + 1] = v.y;
                    }
                }
            };
            if constexpr (CT == DType::BF16) {
                const int row = lane & 15;      // ldmatrix: lanes 0-15 the step's first half, 16-31 its second
#pragma unroll
                for (int ks = 0; ks < KSTEPS; ++ks) {
                    uint32_t q[QW];
                    query(ks, q);
#pragma unroll
                    for (int b = 0; b < MT; ++b) {
                        uint32_t k[4];
                        ldsm_x4(k32 + b * 16 * G::PITCH + chunk_at<CT, G::PITCH>(row, 2 * ks + (lane >> 4)), k);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma<false>(s[b][n], k, q[2 * n], q[2 * n + 1]);
                    }
                }
            } else if constexpr (CT == DType::E4M3) {
#pragma unroll
                for (int c = 0; c < DP / 64; ++c)
#pragma unroll
                    for (int b = 0; b < MT; ++b) {
                        const uint4 x = *reinterpret_cast<const uint4*>(kt + chunk_at<CT, G::PITCH>(16 * b + g, 4 * c + t4));
                        const uint4 y = *reinterpret_cast<const uint4*>(kt + chunk_at<CT, G::PITCH>(16 * b + g + 8, 4 * c + t4));
                        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t q[QW], k[4];
                            query(4 * c + j, q);
                            e4m3x4_f16x4(xw[j], k[0], k[2]);
                            e4m3x4_f16x4(yw[j], k[1], k[3]);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma<true>(s[b][n], k, q[2 * n], q[2 * n + 1]);
                        }
                    }
            } else {
#pragma unroll
                for (int ks = 0; ks < KSTEPS; ++ks) {
                    uint32_t q[QW];
                    query(ks, q);
#pragma unroll
                    for (int b = 0; b < MT; ++b) {
                        const float4 x = *reinterpret_cast<const float4*>(kt + chunk_at<CT, G::PITCH>(16 * b + g, 4 * ks + t4));
                        const float4 y = *reinterpret_cast<const float4*>(kt + chunk_at<CT, G::PITCH>(16 * b + g + 8, 4 * ks + t4));
                        uint32_t kh[4], km[4], kl[4];
                        cut3(x.x, x.y, kh[0], km[0], kl[0]);
                        cut3(y.x, y.y, kh[1], km[1], kl[1]);
                        cut3(x.z, x.w, kh[2], km[2], kl[2]);
                        cut3(y.z, y.w, kh[3], km[3], kl[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint32_t* qn = q + 6 * n;
                            float c[4] = {};
                            mma<false>(c, kl, qn[0], qn[1]);
                            mma<false>(c, km, qn[2], qn[3]);
                            mma<false>(c, kh, qn[4], qn[5]);
                            mma<false>(c, km, qn[0], qn[1]);
                            mma<false>(c, kh, qn[2], qn[3]);
                            mma<false>(c, kh, qn[0], qn[1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[b][n][e] += c[e];
                        }
                    }
                }
            }

            // --- softmax
            bool over = false;
#pragma unroll
            for (int b = 0; b < MT; ++b) {
                const bool in0 = (mask >> (16 * b + g)) & 1u, in1 = (mask >> (16 * b + g + 8)) & 1u;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& x = s[b][n][e];
                        x *= rowscale[n][e & 1];
                        if (a.softcap > 0.0f) x = cap2 * tanhf(x);
                        x = (e < 2 ? in0 : in1) ? x : -INFINITY;
                        over = over || x > m[n][e & 1] + kSlack;
                    }
            }
            if (__any_sync(0xFFFFFFFFu, over)) {
                // The reference moves to the largest score so far.
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = m[n][e];
#pragma unroll
                        for (int b = 0; b < MT; ++b) top = fmaxf(top, fmaxf(s[b][n][e], s[b][n][e + 2]));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                        const float alpha = m[n][e] == -INFINITY ? 0.0f : ex2(m[n][e] - top);
                        m[n][e] = top;
                        l[n][e] *= alpha;
                        if constexpr (!FRESH) kept[n][e] *= alpha;
#pragma unroll
                        for (int j = 0; j < KSTEPS; ++j) {
                            acc[j][n][e] *= alpha;
                            acc[j][n][e + 2] *= alpha;
                        }
                    }
            }

            // --- weights, transposed into the second product's operand: tokens by pairs, a head to each g
            constexpr int PP = F16 ? 2 : 3;     // parts of a weight
            uint32_t w[MT][NT][PP][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float up[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) up[e] = m[n][e] == -INFINITY ? 0.0f : (F16 ? kUp - m[n][e] : -m[n][e]);
#pragma unroll
                for (int b = 0; b < MT; ++b) {
                    float (&x)[4] = s[b][n];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = ex2(x[e] + up[e & 1]);
                        l[n][e & 1] += x[e];
                    }
                    uint32_t c[PP][2];
                    if constexpr (F16) {
                        cut2(x[0], x[1], c[0][0], c[1][0]);
                        cut2(x[2], x[3], c[0][1], c[1][1]);
                    } else {
                        cut3(x[0], x[1], c[0][0], c[1][0], c[PP - 1][0]);
                        cut3(x[2], x[3], c[0][1], c[1][1], c[PP - 1][1]);
                    }
#pragma unroll
                    for (int q = 0; q < PP; ++q) {
                        w[b][n][q][0] = transpose8x8(c[q][0]);
                        w[b][n][q][1] = transpose8x8(c[q][1]);
                    }
                }
            }

            // --- values times weights: 16 dimensions x 8 heads per block
            const unsigned char* vt = kt + G::KV;
            if constexpr (CT == DType::BF16) {
                const int row = (lane & 7) + ((lane >> 4) << 3);    // lanes 8-15, 24-31 the block's second half
                constexpr int JB = FRESH && NT == 1 ? 4 : 1;        // blocks at a time (64 ragged sequences, heads of 64: 105 us, one 109)
#pragma unroll
                for (int j = 0; j < KSTEPS; j += JB)
#pragma unroll
                    for (int b = 0; b < MT; ++b) {
                        uint32_t v[JB][4];
                        float o[JB][NT][4] = {};
#pragma unroll
                        for (int u = 0; u < JB; ++u)
                            ldsm_x4_t(k32 + G::KV + b * 16 * G::PITCH + chunk_at<CT, G::PITCH>(row, 2 * (j + u) + ((lane >> 3) & 1)), v[u]);
#pragma unroll
                        for (int q = PP - 1; q >= 0; --q)
#pragma unroll
                            for (int u = 0; u < JB; ++u)
#pragma unroll
                                for (int n = 0; n < NT; ++n)
                                    mma<false>(FRESH ? o[u][n] : acc[j + u][n], v[u], w[b][n][q][0], w[b][n][q][1]);
                        if constexpr (FRESH) {
#pragma unroll
                            for (int u = 0; u < JB; ++u)
#pragma unroll
                                for (int n = 0; n < NT; ++n) add4(acc[j + u][n], o[u][n]);
                        }
                    }
            } else if constexpr (CT == DType::E4M3) {
#pragma unroll
                for (int c = 0; c < DP / 64; ++c)
#pragma unroll
                    for (int b = 0; b < MT; ++b) {
                        uint2 x[4];     // eight dimensions of the lane's four tokens
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            x[k] = *reinterpret_cast<const uint2*>(
                                vt + chunk_at<CT, G::PITCH>(16 * b + 2 * t4 + (k & 1) + 8 * (k >> 1), 4 * c + (g >> 1)) + (g & 1) * 8);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            uint32_t f[4][2];
#pragma unroll
                            for (int k = 0; k < 4; ++k) e4m3x4_f16x4(half ? x[k].y : x[k].x, f[k][0], f[k][1]);
#pragma unroll
                            for (int pr = 0; pr < 2; ++pr) {
                                const int j = 4 * c + 2 * half + pr;
                                const uint32_t v[4] = {prmt(f[0][pr], f[1][pr], 0x5410), prmt(f[0][pr], f[1][pr], 0x7632),
                                                       prmt(f[2][pr], f[3][pr], 0x5410), prmt(f[2][pr], f[3][pr], 0x7632)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    mma<true>(acc[j][n], v, w[b][n][1][0], w[b][n][1][1]);
                                    mma<true>(acc[j][n], v, w[b][n][0][0], w[b][n][0][1]);
                                }
                            }
                        }
                    }
            } else {
#pragma unroll
                for (int c = 0; c < DP / 32; ++c)
#pragma unroll
                    for (int b = 0; b < MT; ++b) {
                        float4 x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            x[k] = *reinterpret_cast<const float4*>(
                                vt + chunk_at<CT, G::PITCH>(16 * b + 2 * t4 + (k & 1) + 8 * (k >> 1), 8 * c + g));
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj) {
                            uint32_t vh[4], vm[4], vl[4];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                cut3((&x[0].x)[2 * jj + e], (&x[1].x)[2 * jj + e], vh[e], vm[e], vl[e]);
                                cut3((&x[2].x)[2 * jj + e], (&x[3].x)[2 * jj + e], vh[e + 2], vm[e + 2], vl[e + 2]);
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const auto& wn = w[b][n];
                                float o[4] = {};
                                mma<false>(o, vl, wn[0][0], wn[0][1]);
                                mma<false>(o, vm, wn[1][0], wn[1][1]);
                                mma<false>(o, vh, wn[PP - 1][0], wn[PP - 1][1]);
                                mma<false>(o, vm, wn[0][0], wn[0][1]);
                                mma<false>(o, vh, wn[1][0], wn[1][1]);
                                mma<false>(o, vh, wn[0][0], wn[0][1]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[2 * c + jj][n][e] += o[e];
                            }
                        }
                    }
            }
        }

        const bool ends = cons.t == cons.tiles - 1 || i + 1 == count;
        if constexpr (!FRESH) {
            if (++run == RUN && !ends) put_aside();
            if (ends) {
                if (held) take_back();
                held = false;
                run = 0;
            }
        }
        if (ends) {
            // --- the item's end in this share: join the warps; the stage just used holds their sums
            __syncwarp();
            float* o = reinterpret_cast<float*>(kt);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int h = 8 * n + 2 * t4 + e;
                    float sum = l[n][e];
                    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
                    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
                    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
                    if (g == 0) {
                        s_m[warp * 16 + h] = m[n][e];
                        s_l[warp * 16 + h] = sum;
                    }
#pragma unroll
                    for (int j = 0; j < KSTEPS; ++j) {
                        const int d = o_dim<CT>(j, g);
                        o[o_at(h, d, DP)] = acc[j][n][e];
                        o[o_at(h, d + o_second<CT>(), DP)] = acc[j][n][e + 2];
                    }
                }
            const Cursor done = cons;
            cons.next(p, items, TILE);
            if (i + 1 < count) fetch_queries(cons);     // under way while the warps join
            __syncthreads();
            int64_t head0;
            const int nh = heads_of(done, head0);
            const bool whole = item0 >= lo && item0 + done.tiles <= hi;
            Parts at = {};
            float* part = nullptr;
            if (!whole) {
                at = parts_of(item0, done.tiles);
                part = p.ws + static_cast<size_t>(slot_of(at, share)) * G::PART;
            }
            for (int row = orow; row < nh; row += RPT) {
                if (4 * ov >= dim) break;
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w * 16 + row]);
                const float ref = M == -INFINITY ? 0.0f : M;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float f = ex2(s_m[w * 16 + row] - ref);
                    const float4 x = *reinterpret_cast<const float4*>(
                        reinterpret_cast<const float*>(ring + (stage * NW + w) * G::WS) + o_at(row, 4 * ov, DP));
                    L = fmaf(f, s_l[w * 16 + row], L);
                    sum.x = fmaf(f, x.x, sum.x);
                    sum.y = fmaf(f, x.y, sum.y);
                    sum.z = fmaf(f, x.z, sum.z);
                    sum.w = fmaf(f, x.w, sum.w);
                }
                if (whole) {
                    finish(done, row, ov, sum, M, L);
                } else {
                    *reinterpret_cast<float4*>(part + row * DP + 4 * ov) = sum;
                    if (ov == 0) *reinterpret_cast<float2*>(part + HEADS * DP + 2 * row) = make_float2(M, L);
                }
            }
            __syncthreads();
            if (!whole) {
                // Whether this share is the last of its item is asked now and looked at when the share is done.
                uint32_t got = 0;
                if (tid == 0) got = atom_add_acq_rel_gpu_u32(first_ticket(at, done), 1u);
                if (item0 == head_item0) { partial0 = true; ticket0 = got; }
                else { partial1 = true; ticket1 = got; }
            }
            item0 += done.tiles;
            if (i + 1 < count) begin_item(cons);
            else cons = done;
        } else {
            cons.next(p, items, TILE);
        }
        // The stage is free: every stage's loads but this one's are under way while the next is awaited.
        __syncwarp();
        request(stage);
        stage = stage + 1 == S ? 0 : stage + 1;
    }
    cp_async_wait<0>();

    // --- join the shares of the first and the last item, if this one was the last to arrive: the
    // parts in their order, so that results do not depend on which share that is
    if (tid == 0) {
        s_find[0] = static_cast<int>(ticket0);
        s_find[1] = static_cast<int>(ticket1);
    }
    __syncthreads();
    for (int which = 0; which < 2; ++which) {
        if (!(which == 0 ? partial0 : partial1)) continue;
        const Cursor c = which == 0 ? head : cons;
        const Parts at = parts_of(which == 0 ? head_item0 : item0 - cons.tiles, c.tiles);
        const uint32_t all = at.last - at.first + 1, near = near_of(all), group = (share - at.first) / near;
        int64_t head0;
        const int nh = heads_of(c, head0);
        uint32_t c0 = at.first + group * near, step = 1, n = all - group * near < near ? all - group * near : near;
        uint32_t got = static_cast<uint32_t>(s_find[which]);
        uint32_t* ticket = first_ticket(at, c);
        for (bool top = all <= near;; top = true) {
            if (got != n - 1) break;
            if (tid == 0) *ticket = 0u;
            float* dst = p.ws + static_cast<size_t>(slot_of(at, c0)) * G::PART;
            for (int row = orow; row < nh; row += RPT) {
                if (4 * ov >= dim) break;
                float M = -INFINITY, L = 0.0f;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                constexpr uint32_t B = 16;      // parts whose loads are under way together
                for (uint32_t k0 = 0; k0 < n; k0 += B) {
                    float2 ml[B];
                    float4 x[B];
#pragma unroll
                    for (uint32_t k = 0; k < B; ++k) {
                        ml[k] = make_float2(-INFINITY, 0.0f);
                        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (k0 + k < n) {
                            const float* from = p.ws + static_cast<size_t>(slot_of(at, c0 + (k0 + k) * step)) * G::PART;
                            ml[k] = __ldcg(reinterpret_cast<const float2*>(from + HEADS * DP + 2 * row));
                            x[k] = __ldcg(reinterpret_cast<const float4*>(from + row * DP + 4 * ov));
                        }
                    }
                    float most = M;
#pragma unroll
                    for (uint32_t k = 0; k < B; ++k) most = fmaxf(most, ml[k].x);
                    const float ref = most == -INFINITY ? 0.0f : most, f0 = ex2(M - ref);
                    L *= f0;
                    sum.x *= f0; sum.y *= f0; sum.z *= f0; sum.w *= f0;
                    M = most;
#pragma unroll
                    for (uint32_t k = 0; k < B; ++k) {
                        const float f = ex2(ml[k].x - ref);
                        L = fmaf(f, ml[k].y, L);
                        sum.x = fmaf(f, x[k].x, sum.x);
                        sum.y = fmaf(f, x[k].y, sum.y);
                        sum.z = fmaf(f, x[k].z, sum.z);
                        sum.w = fmaf(f, x[k].w, sum.w);
                    }
                }
                if (top) {
                    finish(c, row, ov, sum, M, L);
                } else {
                    // Each thread replaces only elements that it alone reads, the maxima and sums after
                    // the barrier below.
                    *reinterpret_cast<float4*>(dst + row * DP + 4 * ov) = sum;
                    if (ov == 0) { s_m[row] = M; s_l[row] = L; }
                }
            }
            if (top) break;
            __syncthreads();
            if (tid < nh) *reinterpret_cast<float2*>(dst + HEADS * DP + 2 * tid) = make_float2(s_m[tid], s_l[tid]);
            __syncthreads();
            ticket = p.tickets + static_cast<int64_t>(c.b) * items + c.r;
            if (tid == 0) s_find[2] = static_cast<int>(atom_add_acq_rel_gpu_u32(ticket, 1u));
            __syncthreads();
            got = static_cast<uint32_t>(s_find[2]);
            c0 = at.first;
            step = near;
            n = (all + near - 1) / near;
        }
        __syncthreads();
    }
}

struct Kernel {
    const void* fn;
    int threads, smem, rows, part_floats, tile, aside_floats;
};

template <DType IO, DType CT, int DP, int NT>
Kernel kernel_of() {
    using G = Geo<CT, DP, NT>;
    return {reinterpret_cast<const void*>(&paged_attention_kernel<IO, CT, DP, NT>), G::NW * 32, G::SMEM, G::HEADS, G::PART, G::TILE, G::ASIDE};
}

template <DType IO, DType CT, int NT>
Kernel kernel_for_dim(int dim) {
    if (dim <= 64) return kernel_of<IO, CT, 64, NT>();
    if (dim <= 128) return kernel_of<IO, CT, 128, NT>();
    return kernel_of<IO, CT, 256, NT>();
}

Kernel select(const PagedAttnArgs& a) {
    // Up to eight heads of a group are one block of columns, more are blocks of 16 (two at a time).
    const bool two = a.heads / a.kv_heads > 8;
    if (a.ct == DType::F32)
        return two ? kernel_for_dim<DType::F32, DType::F32, 2>(a.dim) : kernel_for_dim<DType::F32, DType::F32, 1>(a.dim);
    if (a.ct == DType::BF16)
        return two ? kernel_for_dim<DType::BF16, DType::BF16, 2>(a.dim) : kernel_for_dim<DType::BF16, DType::BF16, 1>(a.dim);
    return two ? kernel_for_dim<DType::BF16, DType::E4M3, 2>(a.dim) : kernel_for_dim<DType::BF16, DType::E4M3, 1>(a.dim);
}

// Resident CTAs per SM, asked once per kernel and device.
cudaError_t occupancy(const Kernel& k, int* per_sm) {
    static std::mutex mu;
    static std::unordered_map<const void*, int> known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    auto it = known[dev].find(k.fn);
    if (it != known[dev].end()) { *per_sm = it->second; return cudaSuccess; }
    e = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
    if (e != cudaSuccess) return e;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, k.fn, k.threads, static_cast<size_t>(k.smem));
    if (e != cudaSuccess) return e;
    if (*per_sm < 1) return cudaErrorLaunchOutOfResources;
    known[dev][k.fn] = *per_sm;
    return cudaSuccess;
}

int64_t items_of(const PagedAttnArgs& a, const Kernel& k) {
    const int group = a.heads / a.kv_heads;
    return static_cast<int64_t>(a.batch) * a.kv_heads * ((group + k.rows - 1) / k.rows);
}

}  // namespace

cudaError_t paged_attention_plan(const PagedAttnArgs& a, int num_sms, PagedAttnPlan* plan) {
    const Kernel k = select(a);
    int per_sm = 0;
    cudaError_t e = occupancy(k, &per_sm);
    if (e != cudaSuccess) return e;
    // No more CTAs than tiles that the longest possible sequences would make.
    int64_t longest = static_cast<int64_t>(a.max_pages) * a.page_size;
    if (a.window > 0 && a.window < longest) longest = a.window;
    const int64_t items = items_of(a, k);
    int64_t tiles = (longest + k.tile - 1) / k.tile;
    if (tiles < 1) tiles = 1;
    int64_t ctas = static_cast<int64_t>(num_sms) * per_sm;
    if (tiles * items < ctas) ctas = tiles * items;
    plan->ctas = static_cast<int>(ctas);
    // Tiles are counted in 32 bits.
    if (tiles * items > INT32_MAX) return cudaErrorNotSupported;
    plan->ws_floats = static_cast<size_t>(ctas) * (2 * k.part_floats + k.aside_floats);
    plan->tickets = static_cast<size_t>(items + 2 * ctas);
    return cudaSuccess;
}

cudaError_t launch_paged_attention(const PagedAttnArgs& a, const PagedAttnPlan& plan, float* ws, uint32_t* tickets,
                                   cudaStream_t s) {
    const Kernel k = select(a);
    Params p;
    p.a = a;
    p.ws = ws;
    p.aside = ws + static_cast<size_t>(2 * plan.ctas) * k.part_floats;
    p.tickets = tickets;
    p.group = a.heads / a.kv_heads;
    p.hpb = k.rows;
    p.hblocks = (p.group + k.rows - 1) / k.rows;
    // Exact for every position below 2^31: mul = ceil(2^(31 + ceil(log2 size)) / size).
    int log = 0;
    while (log < 31 && (int64_t(1) << log) < a.page_size) ++log;
    p.page_mul = static_cast<uint32_t>(((uint64_t(1) << (31 + log)) + a.page_size - 1) / a.page_size);
    p.page_shift = log > 0 ? log - 1 : 0;
    void* args[] = {&p};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.ctas);
    cfg.blockDim = dim3(k.threads);
    cfg.dynamicSmemBytes = static_cast<size_t>(k.smem);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, k.fn, args);
}

}  // namespace dnnopt_b200
