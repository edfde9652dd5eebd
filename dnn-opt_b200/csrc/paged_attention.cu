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
// heads of its group, far below the tensor rate, so HBM.  The group's query
// heads are the 16 rows of an m16n8k16 product (mma.sync): a 64-token tile
// costs a warp some 200 instructions per 8 KB, about a seventh of what an SM
// issues while HBM delivers it, so the 128-row tcgen05 tile (at most 16 rows
// of which would hold a head) has nothing to win.
//
// Exactness.  bf16 products are exact and summed in FP32; weights exp(s - m)
// enter the second product as two bf16 parts (16 bits), so that the output
// carries one rounding, its own.  E4M3 keys and values are exact in f16: they
// are multiplied there, the query normalised by a power of two per head and
// the weights scaled by 2^15 so that neither leaves f16's range.  FP32 operands
// are cut into three bf16 parts each (24 bits, no loss); products below 2^-24
// of the largest are left out.
#include <cuda_fp8.h>

#include <mutex>
#include <unordered_map>

#include "common.cuh"
#include "kernels.h"

namespace dnnopt_b200 {
namespace {

constexpr int kTok = 16;            // tokens per warp and tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kJoin = 16;           // parts joined by one CTA at a time

struct Params {
    PagedAttnArgs a;
    float* ws;                      // partial results: two slots per CTA
    uint32_t* tickets;              // one per item, then two per CTA
    int group, hpb, hblocks;        // heads per kv head; per item; items per kv head
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
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// x and y as a rounded part and what it leaves.
template <bool F16>
__device__ __forceinline__ void cut2(float x, float y, uint32_t& h, uint32_t& l) {
    h = pack_rn<F16>(x, y);
    float hx, hy;
    if constexpr (F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        hx = f.x; hy = f.y;
    } else {
        hx = __uint_as_float(h << 16);
        hy = __uint_as_float(h & 0xFFFF0000u);
    }
    l = pack_rn<F16>(x - hx, y - hy);
}
// Four E4M3 bytes as f16, exactly.
__device__ __forceinline__ void e4m3x4_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(four));
}

// Tile geometry of one instantiation.  DP: head_dim rounded up to 64, 128 or 256.
template <DType CT, int DP, bool WIDE>
struct Geo {
    static constexpr int EC = CT == DType::F32 ? 4 : (CT == DType::BF16 ? 2 : 1);
    static constexpr int ROWS = WIDE ? 16 : 8;                     // heads per item
    static constexpr int PITCH = DP * EC;                          // bytes of a cached row in shared memory
    static constexpr int KV = kTok * PITCH;                        // one warp's keys (or values) of a tile
    static constexpr int OUT = ROWS * DP * 4;                      // one warp's O at the end of an item
    static constexpr int WS = 2 * KV > OUT ? 2 * KV : OUT;         // one warp's part of a stage
    static constexpr int NW = WS >= 32768 ? 2 : 4;                 // warps
    static constexpr int TILE = NW * kTok;                         // tokens per tile
    // Two CTAs per SM where three stages fit twice, so that one streams while the other joins.
    static constexpr int TWO = 108 * 1024 / (WS * NW), ONE = 216 * 1024 / (WS * NW);
    static constexpr int STAGES = TWO >= 3 ? (TWO > 6 ? 6 : TWO) : (ONE > 3 ? 3 : ONE);
    static constexpr int QREGS = CT == DType::F32 ? 6 : (WIDE ? 4 : 2);   // 32-bit words of Q per lane and 16 dims
    static constexpr int QBYTES = DP / 16 * 32 * QREGS * 4;
    static constexpr int SMALL = 2 * NW * 16 * 4 + 16 * 4 + STAGES * NW * 4 + 64;
    static constexpr int SMEM = STAGES * NW * WS + QBYTES + SMALL;
    static constexpr int PART = ROWS * (DP + 2);                   // floats of one partial result
    static_assert(STAGES >= 2, "a pipeline needs two stages");
};

// 16-byte chunk `c` of row `row` in a warp's tile.  bf16 rows are read by
// ldmatrix, eight rows of one chunk at a time; the others eight chunks at a
// time from two rows (keys) or four even rows (values): both without bank
// conflicts.
template <DType CT, int PITCH>
__device__ __forceinline__ int chunk_at(int row, int c) {
    int x;
    if constexpr (CT == DType::BF16) x = row & 7;
    else x = ((row & 6) ^ ((row & 1) << 2));
    if constexpr (PITCH == 64) x &= 3;
    return row * PITCH + ((c ^ x) << 4);
}

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

// Where dimension d of an output row lies among the accumulator columns.
template <DType CT>
__device__ __forceinline__ int o_col(int d) {
    if constexpr (CT == DType::BF16) return d;
    else if constexpr (CT == DType::E4M3) return (d & ~63) | ((d & 7) << 3) | ((d >> 3) & 7);
    else return (d & ~31) | ((d & 3) << 3) | ((d >> 2) & 7);
}
// Columns of a row are rotated in groups of eight so that the eight rows that
// a warp stores at once fall into different banks.
__device__ __forceinline__ int o_at(int row, int col, int pitch) { return row * pitch + (col ^ ((row & 7) << 3)); }

// A tile's place: sequence, item of the sequence, tile of the item.
struct Cursor {
    int b, r, t;
    int tiles, first, len;          // of sequence b

    __device__ __forceinline__ void load(const Params& p, int tile_tokens) {
        len = __ldg(p.a.lens + b);
        if (len < 0 || len > static_cast<int64_t>(p.a.max_pages) * p.a.page_size) {
            if (threadIdx.x == 0) record_kernel_error(p.a.err, kKerrBadIndex);
            len = 0;
        }
        first = p.a.window > 0 && len > p.a.window ? len - p.a.window : 0;
        const int n = (len - first + tile_tokens - 1) / tile_tokens;
        tiles = n > 0 ? n : 1;      // an empty sequence still has outputs to write
    }
    __device__ __forceinline__ void next(const Params& p, int items, int tile_tokens) {
        if (++t < tiles) return;
        t = 0;
        if (++r < items) return;
        r = 0;
        if (++b < p.a.batch) load(p, tile_tokens);
    }
};

template <DType IO, DType CT, int DP, bool WIDE>
__global__ void __launch_bounds__(Geo<CT, DP, WIDE>::NW * 32) paged_attention_kernel(const Params p) {
    using G = Geo<CT, DP, WIDE>;
    using I = Io<IO>;
    constexpr int NW = G::NW, S = G::STAGES, TILE = G::TILE, ROWS = G::ROWS;
    constexpr bool F16 = CT == DType::E4M3;
    constexpr int KSTEPS = DP / 16, OT = DP / 8;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* ring = smem;
    uint32_t* s_q = reinterpret_cast<uint32_t*>(smem + S * NW * G::WS);
    float* s_m = reinterpret_cast<float*>(smem + S * NW * G::WS + G::QBYTES);    // [NW][16]
    float* s_l = s_m + NW * 16;
    float* s_f = s_l + NW * 16;                                                  // [16] query scale per head
    uint32_t* s_mask = reinterpret_cast<uint32_t*>(s_f + 16);                    // [S][NW]
    int* s_find = reinterpret_cast<int*>(s_mask + S * NW);                       // b, ticket
    long long* s_off = reinterpret_cast<long long*>((reinterpret_cast<uintptr_t>(s_find + 2) + 7) & ~uintptr_t(7));  // sum, offset of b

    const PagedAttnArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int items = a.kv_heads * p.hblocks;
    const int dim = a.dim;

    // --- the CTA's share: tiles [lo, hi) of all tiles in (sequence, item, tile) order
    const int per = (a.batch + NW * 32 - 1) / (NW * 32);
    long long mine = 0;
    for (int i = 0; i < per; ++i) {
        Cursor c;
        c.b = tid * per + i;
        if (c.b >= a.batch) break;
        c.load(p, TILE);
        mine += c.tiles;
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += v;
    }
    long long* s_sum = reinterpret_cast<long long*>(ring);
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    total *= items;
    const long long P = total < gridDim.x ? total : gridDim.x;
    const long long cta = blockIdx.x;
    if (cta >= P) return;
    const long long lo = cta * total / P, hi = (cta + 1) * total / P;
    {
        const long long start = (before + incl - mine) * items, end = (before + incl) * items;
        if (lo >= start && lo < end) {
            long long at = start;
            Cursor c;
            c.b = tid * per;
            for (;; ++c.b) {
                c.load(p, TILE);
                const long long n = static_cast<long long>(c.tiles) * items;
                if (lo < at + n) break;
                at += n;
            }
            s_find[0] = c.b;
            s_off[0] = at;
        }
    }
    __syncthreads();
    Cursor cons;
    cons.b = s_find[0];
    cons.load(p, TILE);
    {
        const long long in = lo - s_off[0];
        cons.r = static_cast<int>(in / cons.tiles);
        cons.t = static_cast<int>(in % cons.tiles);
    }
    long long item0 = lo - cons.t;      // first tile of the current item
    Cursor prod = cons;
    __syncthreads();

    // --- producer: one warp's tokens of one tile, the page numbers one tile ahead
    int ent = -1, slot = 0;
    bool want = false, fresh = false;
    auto look = [&]() {
        const int pos = prod.first + prod.t * TILE + warp * kTok + (lane & 15);
        want = pos < prod.len;
        const int pg = pos / a.page_size;
        slot = pos - pg * a.page_size;
        ent = want ? __ldg(a.table + prod.b * a.table_stride + pg) : -1;
        fresh = a.k_new != nullptr && pos == prod.len - 1;
    };
    auto issue = [&](int stage) {
        const bool ok = want && ent >= 0 && ent < a.num_pages;
        if (want && !ok) record_kernel_error(a.err, kKerrBadIndex);
        const uint32_t valid = __ballot_sync(0xFFFFFFFFu, ok) & 0xFFFFu;
        const uint32_t real = __ballot_sync(0xFFFFFFFFu, ok && !fresh) & 0xFFFFu;
        if (lane == 0) s_mask[stage * NW + warp] = valid;
        if (valid) {
            const int kvh = prod.r / p.hblocks;
            const long long off = ok ? (ent * a.page_stride + slot * a.token_stride + kvh * a.head_stride) * G::EC : 0;
            constexpr int LPR = G::PITCH / 16 > 32 ? 32 : G::PITCH / 16;    // lanes per row
            const uint32_t kbase = smem_u32(ring + (stage * NW + warp) * G::WS);
            const int nch = dim * G::EC / 16;
#pragma unroll
            for (int i = 0; i < kTok * LPR / 32; ++i) {
                const int row = i * (32 / LPR) + lane / LPR;
                const long long o = __shfl_sync(0xFFFFFFFFu, off, row);
                const bool load = (real >> row) & 1u;
#pragma unroll
                for (int c = lane % LPR; c < G::PITCH / 16; c += LPR) {
                    if (c < nch) {
                        const uint32_t dst = kbase + chunk_at<CT, G::PITCH>(row, c);
                        cp_async16(dst, static_cast<const char*>(a.k) + o + c * 16, load);
                        cp_async16(dst + G::KV, static_cast<const char*>(a.v) + o + c * 16, load);
                    }
                }
            }
        }
    };
    const long long count = hi - lo;
    long long issued = 0;
    look();
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        if (issued < count) {
            issue(s);
            if (++issued < count) { prod.next(p, items, TILE); look(); }
        }
        cp_async_commit();
    }

    float acc[OT][4], m[2], l[2], rowscale[2];
    int stage = 0;
    bool begin = true;
    for (long long i = 0; i < count; ++i) {
        if (begin) {
            // --- a new item: its queries in the order of the score product's operand
            begin = false;
            const int kvh = cons.r / p.hblocks, h0 = (cons.r - kvh * p.hblocks) * p.hpb;
            const int nh = p.group - h0 < ROWS ? p.group - h0 : ROWS;
            const typename I::S* q = static_cast<const typename I::S*>(a.q) + cons.b * a.q_batch +
                                     (static_cast<int64_t>(kvh) * p.group + h0) * a.q_head;
            if constexpr (CT == DType::E4M3) {
                // Power of two that brings the head's largest |q| to [1, 2).
                for (int h = warp; h < ROWS; h += NW) {
                    float top = 0.0f;
                    if (h < nh)
                        for (int d = lane; d < dim; d += 32) top = fmaxf(top, fabsf(I::get(q[h * a.q_head + d])));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                    uint32_t e = __float_as_uint(top) >> 23;
                    if (e == 0 || e >= 254) e = 127;
                    if (lane == 0) s_f[h] = __uint_as_float((254 - e) << 23);
                }
                __syncthreads();
            }
            for (int idx = tid; idx < KSTEPS * 32; idx += NW * 32) {
                const int ks = idx >> 5, ln = idx & 31, gg = ln >> 2, tt = ln & 3;
                const int d0 = q_dim<CT>(ks, tt), d1 = d0 + q_second<CT>();
                float v[ROWS / 8][4];
#pragma unroll
                for (int w = 0; w < ROWS / 8; ++w) {
                    const int h = gg + 8 * w;
                    const typename I::S* qh = q + h * a.q_head;
                    const float f = CT == DType::E4M3 ? s_f[h] : 1.0f;
                    v[w][0] = h < nh && d0 < dim ? I::get(qh[d0]) * f : 0.0f;
                    v[w][1] = h < nh && d0 < dim ? I::get(qh[d0 + 1]) * f : 0.0f;
                    v[w][2] = h < nh && d1 < dim ? I::get(qh[d1]) * f : 0.0f;
                    v[w][3] = h < nh && d1 < dim ? I::get(qh[d1 + 1]) * f : 0.0f;
                }
                uint32_t* dst = s_q + idx * G::QREGS;
                if constexpr (CT == DType::F32) {
                    // rows 0-7 the first part, rows 8-15 the second; then the third
                    cut3(v[0][0], v[0][1], dst[0], dst[1], dst[4]);
                    cut3(v[0][2], v[0][3], dst[2], dst[3], dst[5]);
                } else if constexpr (WIDE) {
                    dst[0] = pack_rn<F16>(v[0][0], v[0][1]);
                    dst[1] = pack_rn<F16>(v[1][0], v[1][1]);
                    dst[2] = pack_rn<F16>(v[0][2], v[0][3]);
                    dst[3] = pack_rn<F16>(v[1][2], v[1][3]);
                } else {
                    dst[0] = pack_rn<F16>(v[0][0], v[0][1]);
                    dst[1] = pack_rn<F16>(v[0][2], v[0][3]);
                }
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < ROWS / 8; ++w) {
                m[w] = -INFINITY;
                l[w] = 0.0f;
                rowscale[w] = a.scale * a.k_scale;
                if constexpr (CT == DType::E4M3) rowscale[w] /= s_f[g + 8 * w];     // exact: a power of two
            }
#pragma unroll
            for (int j = 0; j < OT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
        }

        cp_async_wait<S - 2>();
        __syncwarp();
        // The next tile goes where the previous one was.
        if (issued < count) {
            issue(stage == 0 ? S - 1 : stage - 1);
            if (++issued < count) { prod.next(p, items, TILE); look(); }
        }
        cp_async_commit();

        const uint32_t mask = s_mask[stage * NW + warp];
        unsigned char* kt = ring + (stage * NW + warp) * G::WS;
        if (mask) {
            if (a.k_new) {
                // --- the new token's row: into the tile and into the cache
                const int row = cons.len - 1 - (cons.first + cons.t * TILE + warp * kTok);
                if (row >= 0 && row < kTok && ((mask >> row) & 1u)) {
                    const int pos = cons.len - 1, pg = pos / a.page_size, kvh = cons.r / p.hblocks;
                    const long long off = __ldg(a.table + cons.b * a.table_stride + pg) * a.page_stride +
                                          (pos - pg * a.page_size) * a.token_stride + kvh * a.head_stride;
                    const bool keep = cons.r == kvh * p.hblocks;    // one item of the head stores it
                    const int64_t from = cons.b * a.new_batch + kvh * a.new_head;
#pragma unroll
                    for (int which = 0; which < 2; ++which) {
                        const typename I::S* src = static_cast<const typename I::S*>(which ? a.v_new : a.k_new) + from;
                        char* dst = static_cast<char*>(which ? a.v : a.k) + off * G::EC;
                        unsigned char* tile = kt + which * G::KV;
                        constexpr int N = 16 / G::EC;       // elements of a chunk
                        for (int c = lane; c * N < dim; c += 32) {
                            uint4 w;
                            if constexpr (CT == DType::E4M3) {
                                const float div = which ? a.v_scale : a.k_scale;
                                uint32_t* o = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    o[e] = 0;
#pragma unroll
                                    for (int f = 0; f < 4; ++f)
                                        o[e] |= static_cast<uint32_t>(__nv_cvt_float_to_fp8(
                                                    __fdiv_rn(I::get(src[c * 16 + e * 4 + f]), div), __NV_SATFINITE, __NV_E4M3))
                                                << (8 * f);
                                }
                            } else {
                                w = *reinterpret_cast<const uint4*>(src + c * N);
                            }
                            *reinterpret_cast<uint4*>(tile + chunk_at<CT, G::PITCH>(row, c)) = w;
                            if (keep) *reinterpret_cast<uint4*>(dst + c * 16) = w;
                        }
                    }
                    __syncwarp();
                }
            }

            // --- scores of 16 tokens: two products of 8
            float s[2][4] = {};
            const uint32_t k32 = smem_u32(kt);
            if constexpr (CT == DType::BF16) {
                // ldmatrix: lanes 0-7 tokens 0-7 first half of the step, 8-15 second half, 16-31 tokens 8-15
                const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                for (int ks = 0; ks < KSTEPS; ++ks) {
                    if (ks * 16 < dim) {
                        uint32_t b[4], q[4];
                        ldsm_x4(k32 + chunk_at<CT, G::PITCH>(row, 2 * ks + ((lane >> 3) & 1)), b);
                        if constexpr (WIDE) {
                            const uint4 v = reinterpret_cast<const uint4*>(s_q)[ks * 32 + lane];
                            q[0] = v.x; q[1] = v.y; q[2] = v.z; q[3] = v.w;
                        } else {
                            const uint2 v = reinterpret_cast<const uint2*>(s_q)[ks * 32 + lane];
                            q[0] = v.x; q[1] = 0u; q[2] = v.y; q[3] = 0u;
                        }
                        mma<false>(s[0], q, b[0], b[1]);
                        mma<false>(s[1], q, b[2], b[3]);
                    }
                }
            } else if constexpr (CT == DType::E4M3) {
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) {
                    if (c * 64 < dim) {
                        uint32_t w[2][4];
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            // Past head_dim the tile holds whatever was there before: no NaN may meet the query's zero.
                            uint4 v = make_uint4(0u, 0u, 0u, 0u);
                            if (64 * c + 16 * t4 < dim)
                                v = *reinterpret_cast<const uint4*>(kt + chunk_at<CT, G::PITCH>(g + 8 * n, 4 * c + t4));
                            w[n][0] = v.x; w[n][1] = v.y; w[n][2] = v.z; w[n][3] = v.w;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t q[4];
                            if constexpr (WIDE) {
                                const uint4 v = reinterpret_cast<const uint4*>(s_q)[(4 * c + j) * 32 + lane];
                                q[0] = v.x; q[1] = v.y; q[2] = v.z; q[3] = v.w;
                            } else {
                                const uint2 v = reinterpret_cast<const uint2*>(s_q)[(4 * c + j) * 32 + lane];
                                q[0] = v.x; q[1] = 0u; q[2] = v.y; q[3] = 0u;
                            }
#pragma unroll
                            for (int n = 0; n < 2; ++n) {
                                uint32_t b0, b1;
                                e4m3x4_f16x4(w[n][j], b0, b1);
                                mma<true>(s[n], q, b0, b1);
                            }
                        }
                    }
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < KSTEPS; ++ks) {
                    if (ks * 16 < dim) {
                        const uint2* qs = reinterpret_cast<const uint2*>(s_q + (ks * 32 + lane) * 6);
                        const uint2 q01 = qs[0], q23 = qs[1], q45 = qs[2];
                        const uint32_t qa[4] = {q01.x, q01.y, q23.x, q23.y}, qb[4] = {q45.x, 0u, q45.y, 0u};
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const float4 v = *reinterpret_cast<const float4*>(kt + chunk_at<CT, G::PITCH>(g + 8 * n, 4 * ks + t4));
                            uint32_t h0, m0, l0, h1, m1, l1;
                            cut3(v.x, v.y, h0, m0, l0);
                            cut3(v.z, v.w, h1, m1, l1);
                            mma<false>(s[n], qa, l0, l1);
                            mma<false>(s[n], qb, h0, h1);
                            mma<false>(s[n], qa, m0, m1);
                            mma<false>(s[n], qa, h0, h1);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {       // rows 8-15 hold the second part's share
                    s[n][0] += s[n][2];
                    s[n][1] += s[n][3];
                }
            }

            // --- softmax over the tile's tokens: each lane has two of every eight
            float alpha[2];
#pragma unroll
            for (int w = 0; w < ROWS / 8; ++w) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = s[n][2 * w + e];
                        x *= rowscale[w];
                        if (a.softcap > 0.0f) x = a.softcap * tanhf(__fdividef(x, a.softcap));
                        x = (mask >> (8 * n + 2 * t4 + e)) & 1u ? x * kLog2e : -INFINITY;
                        top = fmaxf(top, x);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                top = fmaxf(top, m[w]);
                const float ref = top == -INFINITY ? 0.0f : top;
                alpha[w] = exp2f(m[w] - ref);
                m[w] = top;
                l[w] *= alpha[w];
                const float up = F16 ? 15.0f - ref : -ref;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = s[n][2 * w + e];
                        x = exp2f(x + up);
                        l[w] += x;
                    }
            }
            const bool moved = WIDE ? (alpha[0] != 1.0f || alpha[ROWS / 8 - 1] != 1.0f) : alpha[0] != 1.0f;
            if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
                for (int j = 0; j < OT; ++j) {
                    acc[j][0] *= alpha[0];
                    acc[j][1] *= alpha[0];
                    acc[j][2] *= alpha[WIDE ? ROWS / 8 - 1 : 0];
                    acc[j][3] *= alpha[WIDE ? ROWS / 8 - 1 : 0];
                }
            }

            // --- weights as operand parts; narrow items carry the second part in rows 8-15
            uint32_t pa[4], pb[4];
            if constexpr (CT == DType::F32) {
                pb[1] = pb[3] = 0u;
                cut3(s[0][0], s[0][1], pa[0], pa[1], pb[0]);
                cut3(s[1][0], s[1][1], pa[2], pa[3], pb[2]);
            } else if constexpr (WIDE) {
                cut2<F16>(s[0][0], s[0][1], pa[0], pb[0]);
                cut2<F16>(s[0][2], s[0][3], pa[1], pb[1]);
                cut2<F16>(s[1][0], s[1][1], pa[2], pb[2]);
                cut2<F16>(s[1][2], s[1][3], pa[3], pb[3]);
            } else {
                cut2<F16>(s[0][0], s[0][1], pa[0], pa[1]);
                cut2<F16>(s[1][0], s[1][1], pa[2], pa[3]);
            }

            // --- weights times values
            const unsigned char* vt = kt + G::KV;
            if constexpr (CT == DType::BF16) {
                const int row = lane & 15;
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) {
                    if (j * 16 < dim) {
                        uint32_t b[4];
                        ldsm_x4_t(k32 + G::KV + chunk_at<CT, G::PITCH>(row, 2 * j + (lane >> 4)), b);
                        mma<false>(acc[2 * j], pa, b[0], b[1]);
                        mma<false>(acc[2 * j + 1], pa, b[2], b[3]);
                        if constexpr (WIDE) {
                            mma<false>(acc[2 * j], pb, b[0], b[1]);
                            mma<false>(acc[2 * j + 1], pb, b[2], b[3]);
                        }
                    }
                }
            } else if constexpr (CT == DType::E4M3) {
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) {
                    if (c * 64 < dim) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {      // four dims of the lane's eight
                            uint32_t f[4][2];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const int row = 2 * t4 + (k & 1) + 8 * (k >> 1);
                                const uint32_t w = *reinterpret_cast<const uint32_t*>(
                                    vt + chunk_at<CT, G::PITCH>(row, 4 * c + (g >> 1)) + (g & 1) * 8 + half * 4);
                                e4m3x4_f16x4(w, f[k][0], f[k][1]);
                            }
#pragma unroll
                            for (int pr = 0; pr < 2; ++pr) {
                                const int j = 8 * c + half * 4 + pr * 2;
                                const uint32_t x0 = prmt(f[0][pr], f[1][pr], 0x5410), x1 = prmt(f[2][pr], f[3][pr], 0x5410);
                                const uint32_t y0 = prmt(f[0][pr], f[1][pr], 0x7632), y1 = prmt(f[2][pr], f[3][pr], 0x7632);
                                mma<true>(acc[j], pa, x0, x1);
                                mma<true>(acc[j + 1], pa, y0, y1);
                                if constexpr (WIDE) {
                                    mma<true>(acc[j], pb, x0, x1);
                                    mma<true>(acc[j + 1], pb, y0, y1);
                                }
                            }
                        }
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    if (c * 32 < dim) {
                        float4 v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            v[k] = *reinterpret_cast<const float4*>(vt + chunk_at<CT, G::PITCH>(2 * t4 + (k & 1) + 8 * (k >> 1), 8 * c + g));
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float x[4] = {(&v[0].x)[j], (&v[1].x)[j], (&v[2].x)[j], (&v[3].x)[j]};
                            uint32_t h0, m0, l0, h1, m1, l1;
                            cut3(x[0], x[1], h0, m0, l0);
                            cut3(x[2], x[3], h1, m1, l1);
                            mma<false>(acc[4 * c + j], pa, l0, l1);
                            mma<false>(acc[4 * c + j], pb, h0, h1);
                            mma<false>(acc[4 * c + j], pa, m0, m1);
                            mma<false>(acc[4 * c + j], pa, h0, h1);
                        }
                    }
                }
            }
        }

        const bool last = cons.t == cons.tiles - 1 || i + 1 == count;
        if (last) {
            // --- the item's end in this CTA: join the warps; the stage just used holds their sums
            begin = true;
            __syncwarp();
            float* o = reinterpret_cast<float*>(kt);
#pragma unroll
            for (int w = 0; w < ROWS / 8; ++w) {
                l[w] += __shfl_xor_sync(0xFFFFFFFFu, l[w], 1);
                l[w] += __shfl_xor_sync(0xFFFFFFFFu, l[w], 2);
                if (t4 == 0) {
                    s_m[warp * 16 + g + 8 * w] = m[w];
                    s_l[warp * 16 + g + 8 * w] = l[w];
                }
            }
#pragma unroll
            for (int j = 0; j < OT; ++j) {
                if constexpr (WIDE) {
                    *reinterpret_cast<float2*>(o + o_at(g, 8 * j + 2 * t4, DP)) = make_float2(acc[j][0], acc[j][1]);
                    *reinterpret_cast<float2*>(o + o_at(g + 8, 8 * j + 2 * t4, DP)) = make_float2(acc[j][2], acc[j][3]);
                } else {
                    *reinterpret_cast<float2*>(o + o_at(g, 8 * j + 2 * t4, DP)) =
                        make_float2(acc[j][0] + acc[j][2], acc[j][1] + acc[j][3]);
                }
            }
            __syncthreads();
            const int kvh = cons.r / p.hblocks, h0 = (cons.r - kvh * p.hblocks) * p.hpb;
            const int nh = p.group - h0 < ROWS ? p.group - h0 : ROWS;
            const int64_t head0 = static_cast<int64_t>(kvh) * p.group + h0;
            typename I::S* out = static_cast<typename I::S*>(a.out) + cons.b * a.out_batch + head0 * a.out_head;
            float* lse = a.lse ? a.lse + static_cast<int64_t>(cons.b) * a.heads + head0 : nullptr;
            const bool whole = item0 >= lo && item0 + cons.tiles <= hi;
            auto slot_of = [&](long long c, long long first_c) {
                // An item that begins inside its first CTA's share is that CTA's last one.
                const bool tail = c == first_c && c * total / P < item0;
                return p.ws + (2 * c + (tail ? 1 : 0)) * G::PART;
            };
            const int vecs = dim / 4;
            auto finish = [&](int row, int v, float4 sum, float M, float L) {
                const float f = L == 0.0f ? 0.0f : __fdiv_rn(a.v_scale, L);
                typename I::S* dst = out + row * a.out_head + 4 * v;
                typename I::S r[4] = {I::put(sum.x * f), I::put(sum.y * f), I::put(sum.z * f), I::put(sum.w * f)};
                if constexpr (sizeof(typename I::S) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(r);
                else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(r);
                if (v == 0 && lse) lse[row] = L == 0.0f ? -INFINITY : (M + log2f(L) - (F16 ? 15.0f : 0.0f)) * kLn2;
            };
            const long long c_first = ((item0 + 1) * P - 1) / total, c_last = ((item0 + cons.tiles) * P - 1) / total;
            float* part = whole ? nullptr : slot_of(cta, c_first);
            for (int idx = tid; idx < nh * vecs; idx += NW * 32) {
                const int row = idx / vecs, v = idx - row * vecs;
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w * 16 + row]);
                const float ref = M == -INFINITY ? 0.0f : M;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float f = exp2f(s_m[w * 16 + row] - ref);
                    const float* ow = reinterpret_cast<const float*>(ring + (stage * NW + w) * G::WS);
                    L = fmaf(f, s_l[w * 16 + row], L);
                    sum.x = fmaf(f, ow[o_at(row, o_col<CT>(4 * v), DP)], sum.x);
                    sum.y = fmaf(f, ow[o_at(row, o_col<CT>(4 * v + 1), DP)], sum.y);
                    sum.z = fmaf(f, ow[o_at(row, o_col<CT>(4 * v + 2), DP)], sum.z);
                    sum.w = fmaf(f, ow[o_at(row, o_col<CT>(4 * v + 3), DP)], sum.w);
                }
                if (whole) {
                    finish(row, v, sum, M, L);
                } else {
                    *reinterpret_cast<float4*>(part + row * DP + 4 * v) = sum;
                    if (v == 0) {
                        part[ROWS * DP + row] = M;
                        part[ROWS * DP + ROWS + row] = L;
                    }
                }
            }
            if (!whole) {
                // --- join the CTAs of the item: the last of every kJoin neighbours to arrive joins
                // theirs, in order, and the last of those joins the joined ones.
                const long long parts = c_last - c_first + 1;
                const long long mine_g = (cta - c_first) / kJoin, groups = (parts + kJoin - 1) / kJoin;
                long long c0 = c_first + mine_g * kJoin, step = 1;
                long long n = c_last - c0 + 1 < kJoin ? c_last - c0 + 1 : kJoin;
                uint32_t* ticket = p.tickets + static_cast<int64_t>(a.batch) * items + (slot_of(c0, c_first) - p.ws) / G::PART;
                for (int level = groups > 1 ? 0 : 1;; ++level) {
                    if (level == 1) {
                        ticket = p.tickets + static_cast<int64_t>(cons.b) * items + cons.r;
                        if (groups > 1) { c0 = c_first; step = kJoin; n = groups; }
                    }
                    __syncthreads();
                    if (tid == 0) s_find[1] = static_cast<int>(atom_add_acq_rel_gpu_u32(ticket, 1u));
                    __syncthreads();
                    if (s_find[1] != static_cast<int>(n) - 1) break;
                    __threadfence();
                    if (tid == 0) *ticket = 0u;
                    float* dst0 = slot_of(c0, c_first);
                    for (int idx = tid; idx < nh * vecs; idx += NW * 32) {
                        const int row = idx / vecs, v = idx - row * vecs;
                        float M = -INFINITY, L = 0.0f;
                        for (long long k = 0; k < n; ++k)
                            M = fmaxf(M, __ldcg(slot_of(c0 + k * step, c_first) + ROWS * DP + row));
                        const float ref = M == -INFINITY ? 0.0f : M;
                        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                        for (long long k = 0; k < n; ++k) {
                            const float* from = slot_of(c0 + k * step, c_first);
                            const float f = exp2f(__ldcg(from + ROWS * DP + row) - ref);
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(from + row * DP + 4 * v));
                            L = fmaf(f, __ldcg(from + ROWS * DP + ROWS + row), L);
                            sum.x = fmaf(f, x.x, sum.x);
                            sum.y = fmaf(f, x.y, sum.y);
                            sum.z = fmaf(f, x.z, sum.z);
                            sum.w = fmaf(f, x.w, sum.w);
                        }
                        if (level == 1) {
                            finish(row, v, sum, M, L);
                        } else {
                            // Each thread replaces only elements that it alone reads, the maxima and
                            // sums after the barrier below.
                            *reinterpret_cast<float4*>(dst0 + row * DP + 4 * v) = sum;
                            if (v == 0) { s_m[row] = M; s_l[row] = L; }
                        }
                    }
                    if (level == 1) break;
                    __syncthreads();
                    if (tid < nh) {
                        dst0[ROWS * DP + tid] = s_m[tid];
                        dst0[ROWS * DP + ROWS + tid] = s_l[tid];
                    }
                }
            }
            __syncthreads();
            item0 += cons.tiles;
        }
        cons.next(p, items, TILE);
        stage = stage + 1 == S ? 0 : stage + 1;
    }
    cp_async_wait<0>();
}

struct Kernel {
    const void* fn;
    int threads, smem, rows, part_floats, tile;
};

template <DType IO, DType CT, int DP, bool WIDE>
Kernel kernel_of() {
    using G = Geo<CT, DP, WIDE>;
    return {reinterpret_cast<const void*>(&paged_attention_kernel<IO, CT, DP, WIDE>), G::NW * 32, G::SMEM, G::ROWS, G::PART, G::TILE};
}

template <DType IO, DType CT, bool WIDE>
Kernel kernel_for_dim(int dim) {
    if (dim <= 64) return kernel_of<IO, CT, 64, WIDE>();
    if (dim <= 128) return kernel_of<IO, CT, 128, WIDE>();
    return kernel_of<IO, CT, 256, WIDE>();
}

Kernel select(const PagedAttnArgs& a) {
    const bool wide = a.heads / a.kv_heads > 8;
    if (a.ct == DType::F32) return kernel_for_dim<DType::F32, DType::F32, false>(a.dim);
    if (a.ct == DType::BF16)
        return wide ? kernel_for_dim<DType::BF16, DType::BF16, true>(a.dim) : kernel_for_dim<DType::BF16, DType::BF16, false>(a.dim);
    return wide ? kernel_for_dim<DType::BF16, DType::E4M3, true>(a.dim) : kernel_for_dim<DType::BF16, DType::E4M3, false>(a.dim);
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
    plan->ws_floats = static_cast<size_t>(2 * ctas) * k.part_floats;
    plan->tickets = static_cast<size_t>(items + 2 * ctas);
    return cudaSuccess;
}

cudaError_t launch_paged_attention(const PagedAttnArgs& a, const PagedAttnPlan& plan, float* ws, uint32_t* tickets,
                                   cudaStream_t s) {
    const Kernel k = select(a);
    Params p;
    p.a = a;
    p.ws = ws;
    p.tickets = tickets;
    p.group = a.heads / a.kv_heads;
    p.hpb = k.rows;
    p.hblocks = (p.group + k.rows - 1) / k.rows;
    void* args[] = {&p};
    return cudaLaunchKernel(k.fn, dim3(plan.ctas), dim3(k.threads), args, static_cast<size_t>(k.smem), s);
}

}  // namespace dnnopt_b200
