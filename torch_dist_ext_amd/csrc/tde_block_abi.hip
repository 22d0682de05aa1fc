// C entry points of the attention block's operators: checks, and the arguments of the kernels in bytes.
#include <climits>
#include <cmath>

#include "tde_abi.h"
#include "tde_head_rows.h"
#include "tde_int8_linear.h"
#include "tde_paged_attention.h"

using namespace tde::block;

namespace {

constexpr int64_t kMaxRows = (int64_t)1 << 31; // rows of a call: kernels count them in 32 bits
constexpr int64_t kMaxStride = (int64_t)1 << 40;

int elem_bytes(int dtype) { return dtype == TDE_F32 ? 4 : 2; }
bool stride_ok(int64_t s) { return s >= 0 && s < kMaxStride; }
bool heads_ok(const tde_heads &h) { return stride_ok(h.row_stride) && stride_ok(h.head_stride); }
bool cache_ok(const tde_cache &c) { return stride_ok(c.page_stride) && stride_ok(c.slot_stride) && stride_ok(c.head_stride); }

int check_batch(const tde_paged_batch &b) {
    if (b.seqs < 0 || b.table_pages < 0 || b.cache_pages < 0 || b.page_size < 1) return TDE_ESHAPE;
    if (b.seqs > (1 << 24) || !stride_ok(b.table_stride)) return TDE_ESHAPE;
    if (!b.q_starts || (b.seqs > 0 && !b.kv_lens) || (b.seqs > 0 && b.table_pages > 0 && !b.page_table)) return TDE_EINVAL;
    return TDE_OK;
}

PagedBatch device_batch(const tde_paged_batch &b) {
    PagedBatch d;
    d.table = b.page_table;
    d.starts = b.q_starts;
    d.lens = b.kv_lens;
    d.table_stride = b.table_stride;
    d.seqs = b.seqs;
    d.table_pages = b.table_pages;
    d.cache_pages = b.cache_pages;
    d.page = Divisor32((uint32_t)b.page_size);
    return d;
}

int head_rows(const tde_head_rows *r, bool paged, void *hip_stream) {
    if (r == nullptr || r->reserved != 0) return TDE_EINVAL;
    if (r->dtype != TDE_BF16 && r->dtype != TDE_F16 && r->dtype != TDE_F32) return TDE_EDTYPE;
    if (r->dim < 1 || r->tokens < 0 || r->tokens >= kMaxRows || r->q_heads < 0 || r->kv_heads < 0) return TDE_ESHAPE;
    if (r->q_heads > (1 << 16) || r->kv_heads > (1 << 16)) return TDE_ESHAPE;
    if (r->dim > TDE_MAX_HEAD_DIM) return TDE_EHIDDEN;
    if (r->rot_dim < 0 || r->rot_dim > r->dim || r->rot_dim % 2 != 0 || r->cos_sin_rows < 0 || !stride_ok(r->cos_sin_stride)) return TDE_ESHAPE;
    if (r->interleaved != 0 && r->interleaved != 1) return TDE_EINVAL;
    if (r->positions != nullptr && r->positions_bytes != 4 && r->positions_bytes != 8) return TDE_EINVAL;
    if (!(r->eps >= 0.0f) || !std::isfinite(r->eps)) return TDE_EINVAL;
    const tde_heads *views[] = {&r->q, &r->k, &r->v, &r->q_out, &r->k_out};
    for (const tde_heads *v : views)
        if (!heads_ok(*v)) return TDE_ESHAPE;
    if (paged) {
        if (!cache_ok(r->k_cache) || !cache_ok(r->v_cache)) return TDE_ESHAPE;
        const int st = check_batch(r->batch);
        if (st != TDE_OK) return st;
    }
    if (r->tokens == 0 || r->q_heads + r->kv_heads == 0) return TDE_OK;
    if (r->rot_dim > 0 && (r->cos_sin == nullptr || (!paged && r->positions == nullptr))) return TDE_EINVAL;
    if (r->q_heads > 0 && (!r->q.data || !r->q_out.data)) return TDE_EINVAL;
    if (r->kv_heads > 0) {
        if (!r->k.data || (!paged && !r->k_out.data)) return TDE_EINVAL;
        if (paged && (!r->v.data || (r->batch.cache_pages > 0 && (!r->k_cache.data || !r->v_cache.data)))) return TDE_EINVAL;
    }

    const int64_t e = elem_bytes(r->dtype);
    HeadRowsArgs a{};
    const tde_heads *in[] = {&r->q, &r->k, &r->v};
    for (int i = 0; i < 3; ++i) {
        a.in[i] = static_cast<const char *>(in[i]->data);
        a.in_token[i] = in[i]->row_stride * e;
        a.in_head[i] = in[i]->head_stride * e;
    }
    a.out[0] = static_cast<char *>(r->q_out.data);
    a.out_token[0] = r->q_out.row_stride * e;
    a.out_head[0] = r->q_out.head_stride * e;
    a.heads[0] = r->q_heads;
    a.heads[1] = r->kv_heads;
    a.heads[2] = paged ? r->kv_heads : 0;
    if (paged) {
        const tde_cache *caches[] = {&r->k_cache, &r->v_cache};
        for (int i = 0; i < 2; ++i) {
            a.out[1 + i] = static_cast<char *>(caches[i]->data);
            a.out_page[1 + i] = caches[i]->page_stride * e;
            a.out_token[1 + i] = caches[i]->slot_stride * e;
            a.out_head[1 + i] = caches[i]->head_stride * e;
        }
        a.batch = device_batch(r->batch);
    } else {
        a.out[1] = static_cast<char *>(r->k_out.data);
        a.out_token[1] = r->k_out.row_stride * e;
        a.out_head[1] = r->k_out.head_stride * e;
    }
    a.gamma[0] = static_cast<const char *>(r->q_gamma);
    a.gamma[1] = static_cast<const char *>(r->k_gamma);
    a.cos_sin = r->cos_sin;
    a.table_rows = r->cos_sin_rows;
    a.table_stride = r->cos_sin_stride;
    a.positions = r->positions;
    a.positions_wide = r->positions_bytes == 8;
    a.tokens = r->tokens;
    a.dim = r->dim;
    a.half = r->rot_dim / 2;
    a.eps = r->eps;
    a.interleaved = r->interleaved != 0;
    a.paged = paged;
    return launch_head_rows(a, r->dtype, static_cast<hipStream_t>(hip_stream));
}

int check_attention(const tde_attention *t, AttentionPlan *plan) {
    if (t == nullptr || t->reserved != 0) return TDE_EINVAL;
    if (t->dtype != TDE_BF16 && t->dtype != TDE_F16) return TDE_EDTYPE;
    if (t->tokens < 0 || t->tokens >= kMaxRows || t->dim < 1 || t->dim % 8 != 0) return TDE_ESHAPE;
    if (t->q_heads < 1 || t->kv_heads < 1 || t->q_heads % t->kv_heads != 0 || t->q_heads > (1 << 16)) return TDE_ESHAPE;
    if (t->dim > 256) return TDE_EHIDDEN;
    if (!(t->scale > 0.0f && t->scale <= TDE_MAX_SCALE) || (t->zero_tail != 0 && t->zero_tail != 1)) return TDE_EINVAL;
    if (!heads_ok(t->q) || !heads_ok(t->out) || !cache_ok(t->k_cache) || !cache_ok(t->v_cache)) return TDE_ESHAPE;
    for (const tde_cache *c : {&t->k_cache, &t->v_cache}) // in bytes they are 32-bit factors of the keys' offsets
        if (c->page_stride >= (int64_t)1 << 31 || c->slot_stride >= (int64_t)1 << 31) return TDE_ESHAPE;
    const int st = check_batch(t->batch);
    if (st != TDE_OK) return st;
    return plan_attention(t->dim, t->tokens, t->q_heads, t->kv_heads, t->batch.seqs, (int64_t)t->batch.table_pages * t->batch.page_size, plan);
}

bool lines_of_16(const tde_cache &c) {
    return (reinterpret_cast<uintptr_t>(c.data) & 15u) == 0 && c.page_stride % 8 == 0 && c.slot_stride % 8 == 0 && c.head_stride % 8 == 0;
}

} // namespace

extern "C" {

int tde_int8_linear(const tde_int8_product *p, void *hip_stream) {
    if (p == nullptr || p->reserved != 0) return TDE_EINVAL;
    if (p->out_dtype != TDE_BF16 && p->out_dtype != TDE_F16 && p->out_dtype != TDE_F32) return TDE_EDTYPE;
    if (p->tokens < 0 || p->n < 0 || p->k < 1 || p->tokens >= kMaxRows || p->n >= kMaxRows) return TDE_ESHAPE;
    if (p->k > TDE_INT8_MAX_K) return TDE_EHIDDEN;
    if (p->tokens == 0 || p->n == 0) return TDE_OK;
    if (!p->codes || !p->weight || !p->scales || !p->weight_scales || !p->out) return TDE_EINVAL;
    const LinearArgs a{p->codes, p->weight, p->scales, p->weight_scales, p->bias, static_cast<char *>(p->out), p->tokens, p->k, p->n};
    return launch_int8_linear(a, p->out_dtype, static_cast<hipStream_t>(hip_stream));
}

int tde_qk_norm_rope(const tde_head_rows *rows, void *hip_stream) { return head_rows(rows, false, hip_stream); }

int tde_append_kv(const tde_head_rows *rows, void *hip_stream) { return head_rows(rows, true, hip_stream); }

int tde_paged_attention_workspace(const tde_attention *t, int64_t *bytes) {
    if (bytes == nullptr) return TDE_EINVAL;
    AttentionPlan plan;
    const int st = check_attention(t, &plan);
    if (st != TDE_OK) return st;
    *bytes = t->tokens == 0 ? 0 : plan.workspace_bytes;
    return TDE_OK;
}

int tde_paged_attention(const tde_attention *t, void *hip_stream) {
    AttentionPlan plan;
    const int st = check_attention(t, &plan);
    if (st != TDE_OK) return st;
    if (t->tokens == 0) return TDE_OK;
    if (!t->q.data || !t->out.data) return TDE_EINVAL;
    if (t->batch.cache_pages > 0 && (!t->k_cache.data || !t->v_cache.data)) return TDE_EINVAL;
    if (!lines_of_16(t->k_cache) || !lines_of_16(t->v_cache)) return TDE_EALIGN;
    if (plan.workspace_bytes > 0) {
        if (t->workspace == nullptr || t->workspace_bytes < plan.workspace_bytes) return TDE_EINVAL;
        if ((reinterpret_cast<uintptr_t>(t->workspace) & 15u) != 0) return TDE_EALIGN;
    }
    AttentionArgs a{};
    a.q = static_cast<const char *>(t->q.data);
    a.k = static_cast<const char *>(t->k_cache.data);
    a.v = static_cast<const char *>(t->v_cache.data);
    a.out = static_cast<char *>(t->out.data);
    a.q_token = t->q.row_stride * 2;
    a.q_head = t->q.head_stride * 2;
    a.out_token = t->out.row_stride * 2;
    a.out_head = t->out.head_stride * 2;
    a.k_page = (uint32_t)(t->k_cache.page_stride * 2);
    a.k_slot = (uint32_t)(t->k_cache.slot_stride * 2);
    a.k_head = t->k_cache.head_stride * 2;
    a.v_page = (uint32_t)(t->v_cache.page_stride * 2);
    a.v_slot = (uint32_t)(t->v_cache.slot_stride * 2);
    a.v_head = t->v_cache.head_stride * 2;
    a.batch = device_batch(t->batch);
    a.group = Divisor32((uint32_t)(t->q_heads / t->kv_heads));
    a.kv_heads = Divisor32((uint32_t)t->kv_heads);
    a.tokens = t->tokens;
    a.dim = t->dim;
    a.scale_log2 = t->scale * 1.4426950408889634f;
    a.partial = static_cast<float *>(t->workspace);
    a.zero_tail = t->zero_tail != 0;
    return launch_attention(a, plan, t->dtype, static_cast<hipStream_t>(hip_stream));
}

} // extern "C"
