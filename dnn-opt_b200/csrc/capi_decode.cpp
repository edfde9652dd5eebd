// C ABI of the decoder-step operators: products with 4-bit weights, attention
// over a paged key-value cache, and the norms around a block.  Argument checks,
// workspace and launch; see include/dnnopt_b200.h for each entry's contract.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "kernels.h"
#include "runtime.h"

using namespace dnnopt_b200;

namespace {

bool float_type(int t) { return t == DNNOPT_TYPE_F32 || t == DNNOPT_TYPE_BF16; }

int type_bytes(int t) { return t == DNNOPT_TYPE_F32 ? 4 : (t == DNNOPT_TYPE_BF16 ? 2 : 1); }

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Element alignment: a pointer into the middle of an element is a caller's error.
bool element_aligned(const void* p, int type) { return aligned(p, static_cast<size_t>(type_bytes(type))); }

int inject_launch() {
    int inj = check_injected_fault(2);
    return inj == DNNOPT_STATUS_SUCCESS ? inj : set_status(inj);
}

}  // namespace

extern "C" {

int dnnopt_cuda_gemm_w4(const dnnopt_w4_desc* d, const void* A, const uint8_t* W, const void* scale,
                        const void* zero, const float* bias, void* C, void* stream) {
    if (!d || d->M < 0 || d->N < 0 || d->K < 0) return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (!float_type(d->io_type) || !float_type(d->scale_type) || d->group < 0 || d->group % 32 != 0)
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (d->M == 0 || d->N == 0 || d->K == 0) return set_status(DNNOPT_STATUS_SUCCESS);
    const int groups = d->group ? static_cast<int>((static_cast<int64_t>(d->K) + d->group - 1) / d->group) : 1;
    if (d->lda < d->K || d->ldc < d->N || d->lds < groups ||
        d->ldw < static_cast<int>((static_cast<int64_t>(d->K) + 1) / 2))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (!A || !W || !scale || !C || !element_aligned(A, d->io_type) || !element_aligned(C, d->io_type) ||
        !element_aligned(scale, d->scale_type) || !element_aligned(zero, d->scale_type) ||
        !element_aligned(bias, DNNOPT_TYPE_F32))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    // The kernels round K up to whole groups in 32-bit arithmetic.
    if (d->K > INT32_MAX - 65536) return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    int st;
    DeviceContext* ctx = current_context(&st);
    if (!ctx) return st;
    W4Args g;
    g.M = d->M; g.N = d->N; g.K = d->K;
    g.groups = groups;
    g.group = groups > 1 ? d->group : (d->K + 31) / 32 * 32;
    g.io = static_cast<DType>(d->io_type);
    g.st = static_cast<DType>(d->scale_type);
    g.A = A; g.lda = d->lda;
    g.W = W; g.ldw = d->ldw;
    g.scale = scale; g.zero = zero; g.lds = d->lds;
    g.bias = bias;
    g.C = C; g.ldc = d->ldc;
    // kW4RowsAtOnce rows of A at a time, and what is left: the workspace grows with the rows of a launch.
    W4Plan plan, rest = {};
    W4Args part = g;
    part.M = g.M < kW4RowsAtOnce ? g.M : kW4RowsAtOnce;
    if (!gemm_w4_plan(part, ctx->num_sms, &plan)) return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    const int left = g.M > kW4RowsAtOnce ? g.M % kW4RowsAtOnce : 0;
    part.M = left;
    if (left > 0 && !gemm_w4_plan(part, ctx->num_sms, &rest)) return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Workspace* w = nullptr;
    st = ensure_workspace(ctx, s, std::max(plan.ws_floats, rest.ws_floats), std::max(plan.tickets, rest.tickets),
                          std::max(plan.extra_bytes, rest.extra_bytes), &w);
    if (st != DNNOPT_STATUS_SUCCESS) return st;
    if ((st = inject_launch()) != DNNOPT_STATUS_SUCCESS) return st;
    const int64_t a_row = static_cast<int64_t>(d->lda) * type_bytes(d->io_type), c_row = static_cast<int64_t>(d->ldc) * type_bytes(d->io_type);
    for (int64_t m = 0; m < g.M; m += kW4RowsAtOnce) {
        const bool last = g.M - m < kW4RowsAtOnce && left > 0;
        const W4Plan& now = last ? rest : plan;
        part.M = last ? left : (g.M < kW4RowsAtOnce ? g.M : kW4RowsAtOnce);
        part.A = static_cast<const char*>(A) + m * a_row;
        part.C = static_cast<char*>(C) + m * c_row;
        const cudaError_t e = launch_gemm_w4(part, now, w->ws, w->counters, w->quant, w->err, s);
        if (e != cudaSuccess) return cuda_status(e);
        note_launch(now.pitch || now.prepared ? 2 : 1);
    }
    return set_status(DNNOPT_STATUS_SUCCESS);
}

int dnnopt_cuda_paged_attention(const dnnopt_paged_attn_desc* d, const void* q, void* k_cache,
                                void* v_cache, const int32_t* page_table, const int32_t* seq_lens,
                                const void* k_new, const void* v_new, void* out, float* lse,
                                void* stream) {
    if (!d || d->batch < 0 || d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads != 0 ||
        d->head_dim < 1 || d->page_size < 1 || d->num_pages < 0 || d->max_pages < 0 || d->window < 0 ||
        !float_type(d->io_type) || d->cache_type < DNNOPT_TYPE_F32 || d->cache_type > DNNOPT_TYPE_E4M3 ||
        d->table_stride < 0 || !std::isfinite(d->scale) || !(d->softcap >= 0.0f) ||
        !std::isfinite(d->softcap) || !(d->k_scale > 0.0f) || !(d->v_scale > 0.0f) ||
        !std::isfinite(d->k_scale) || !std::isfinite(d->v_scale))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if ((k_new == nullptr) != (v_new == nullptr)) return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (d->batch > 1 && d->table_stride < d->max_pages) return set_status(DNNOPT_STATUS_INVALID_VALUE);
    // Positions, rounded up to whole tiles, are 32-bit.
    if (static_cast<int64_t>(d->max_pages) * d->page_size > INT32_MAX - 65536)
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (d->batch == 0) return set_status(DNNOPT_STATUS_SUCCESS);
    if (!q || !out || !seq_lens || !element_aligned(lse, DNNOPT_TYPE_F32) ||
        !element_aligned(seq_lens, DNNOPT_TYPE_F32) || !element_aligned(page_table, DNNOPT_TYPE_F32))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    // A cache without pages holds no tokens: every sequence has to be empty.
    if (d->num_pages > 0 && d->max_pages > 0 && (!k_cache || !v_cache || !page_table))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    const bool f32 = d->io_type == DNNOPT_TYPE_F32;
    if (f32 != (d->cache_type == DNNOPT_TYPE_F32)) return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    if (d->cache_type != DNNOPT_TYPE_E4M3 && (d->k_scale != 1.0f || d->v_scale != 1.0f))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (d->head_dim % 16 != 0 || d->head_dim > 256) return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    const int64_t eio = type_bytes(d->io_type), ec = type_bytes(d->cache_type);
    auto whole16 = [](int64_t stride, int64_t size) { return stride * size % 16 == 0; };
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
        !whole16(d->q_batch_stride, eio) || !whole16(d->q_head_stride, eio) ||
        !whole16(d->out_batch_stride, eio) || !whole16(d->out_head_stride, eio) ||
        !whole16(d->page_stride, ec) || !whole16(d->token_stride, ec) || !whole16(d->head_stride, ec))
        return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    if (k_new && (!aligned(k_new, 16) || !aligned(v_new, 16) || !whole16(d->new_batch_stride, eio) ||
                  !whole16(d->new_head_stride, eio)))
        return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    int st;
    DeviceContext* ctx = current_context(&st);
    if (!ctx) return st;
    PagedAttnArgs a;
    a.batch = d->batch; a.heads = d->heads; a.kv_heads = d->kv_heads; a.dim = d->head_dim;
    a.page_size = d->page_size; a.num_pages = d->num_pages;
    // Without pages every length above 0 is out of range: a table, which may then be NULL, is not read.
    a.max_pages = d->num_pages > 0 ? d->max_pages : 0;
    a.window = d->window;
    a.io = static_cast<DType>(d->io_type); a.ct = static_cast<DType>(d->cache_type);
    a.scale = d->scale; a.softcap = d->softcap; a.k_scale = d->k_scale; a.v_scale = d->v_scale;
    a.q = q; a.q_batch = d->q_batch_stride; a.q_head = d->q_head_stride;
    a.k = k_cache; a.v = v_cache;
    a.page_stride = d->page_stride; a.token_stride = d->token_stride; a.head_stride = d->head_stride;
    a.table = page_table; a.table_stride = d->table_stride; a.lens = seq_lens;
    a.k_new = k_new; a.v_new = v_new; a.new_batch = d->new_batch_stride; a.new_head = d->new_head_stride;
    a.out = out; a.out_batch = d->out_batch_stride; a.out_head = d->out_head_stride;
    a.lse = lse; a.err = nullptr;
    PagedAttnPlan plan;
    cudaError_t e = paged_attention_plan(a, ctx->num_sms, &plan);
    if (e == cudaErrorNotSupported) return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    if (e != cudaSuccess) return cuda_status(e);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Workspace* w = nullptr;
    st = ensure_workspace(ctx, s, plan.ws_floats, plan.tickets, 0, &w);
    if (st != DNNOPT_STATUS_SUCCESS) return st;
    if ((st = inject_launch()) != DNNOPT_STATUS_SUCCESS) return st;
    a.err = w->bad_index;
    e = launch_paged_attention(a, plan, w->ws, w->counters, s);
    note_launch();
    return cuda_status(e);
}

int dnnopt_cuda_block_norm(const dnnopt_block_norm_desc* d, const void* x, const void* y,
                           const void* gate, const void* post_w, const void* post_b,
                           const void* pre_w, const void* pre_b, void* h, void* z, void* stream) {
    if (!d || d->rows < 0 || d->cols < 0 || d->post < DNNOPT_NORM_NONE || d->post > DNNOPT_NORM_LAYER ||
        d->pre < DNNOPT_NORM_NONE || d->pre > DNNOPT_NORM_LAYER || !float_type(d->io_type) ||
        !float_type(d->weight_type) || !(d->eps >= 0.0f) || d->gate_rows < 1)
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (d->rows == 0 || d->cols == 0) return set_status(DNNOPT_STATUS_SUCCESS);
    if (!x || (!h && !z)) return set_status(DNNOPT_STATUS_INVALID_VALUE);
    if (d->cols > kBlockNormMaxCols) return set_status(DNNOPT_STATUS_NOT_SUPPORTED);
    auto pitch_ok = [&](const void* p, int64_t ld) {
        return !p || (element_aligned(p, d->io_type) && (ld >= d->cols || (d->rows == 1 && ld >= 0)));
    };
    if (!pitch_ok(x, d->ldx) || !pitch_ok(y, d->ldy) || !pitch_ok(h, d->ldh) || !pitch_ok(z, d->ldz))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    const int64_t gates = (static_cast<int64_t>(d->rows) + d->gate_rows - 1) / d->gate_rows;
    if (gate && (!element_aligned(gate, d->io_type) || (d->ldg != 0 && d->ldg < d->cols && gates > 1)))
        return set_status(DNNOPT_STATUS_INVALID_VALUE);
    for (const void* v : {post_w, post_b, pre_w, pre_b})
        if (v && !element_aligned(v, d->weight_type)) return set_status(DNNOPT_STATUS_INVALID_VALUE);
    // Whole-row aliases are read before they are written; any other pitch would not be.
    for (const void* in : {x, y}) {
        const int64_t ld = in == x ? d->ldx : d->ldy;
        if (in && d->rows > 1 && ((in == h && ld != d->ldh) || (in == z && ld != d->ldz)))
            return set_status(DNNOPT_STATUS_INVALID_VALUE);
    }
    if (h && h == z) return set_status(DNNOPT_STATUS_INVALID_VALUE);
    int st;
    DeviceContext* ctx = current_context(&st);
    if (!ctx) return st;
    if ((st = inject_launch()) != DNNOPT_STATUS_SUCCESS) return st;
    BlockNormArgs a;
    a.rows = d->rows; a.cols = d->cols; a.post = y ? d->post : DNNOPT_NORM_NONE; a.pre = d->pre;
    a.io = static_cast<DType>(d->io_type); a.wt = static_cast<DType>(d->weight_type);
    a.eps = d->eps; a.offset = d->weight_offset; a.rs = d->residual_scale; a.bs = d->block_scale;
    a.x = x; a.y = y; a.gate = y ? gate : nullptr;
    a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
    a.h = h; a.z = z;
    a.ldx = d->ldx; a.ldy = d->ldy; a.ldh = d->ldh; a.ldz = d->ldz; a.ldg = d->ldg;
    a.gate_rows = d->gate_rows;
    cudaError_t e = launch_block_norm(a, ctx->num_sms, static_cast<cudaStream_t>(stream));
    note_launch();
    return cuda_status(e);
}

}  // extern "C"
