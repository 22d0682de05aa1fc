// Operators of the attention block behind the norm: registration in the `torch_dist_ext` namespace, argument checks, outputs.
#include <torch/library.h>

#include <cmath>
#include <tuple>

#include "tde_overlap.h"
#include "tde_torch.h"

namespace {

const Tensor *given_or_null(const c10::optional<Tensor> &t) { return t.has_value() && t->defined() ? &*t : nullptr; }

void check_on(const Tensor &t, const Tensor &like, const char *op, const char *name) {
    TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a GPU tensor");
    TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on a different device");
}

int32_t out_code(at::ScalarType t, const char *op) {
    TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, op, ": out_dtype must be bf16, fp16 or fp32, not ", t);
    return t == at::kBFloat16 ? TDE_BF16 : (t == at::kHalf ? TDE_F16 : TDE_F32);
}

// ---- int8_linear ----------------------------------------------------------------------------------------------------

Tensor int8_linear(const Tensor &codes, const Tensor &scales, const Tensor &weight, const Tensor &weight_scales,
                   const c10::optional<Tensor> &bias, c10::optional<at::ScalarType> out_dtype) {
    constexpr const char *op = "int8_linear";
    TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kChar && codes.dim() >= 1 && codes.is_contiguous(), op,
                ": codes must be a contiguous int8 GPU tensor [..., k]");
    check_on(weight, codes, op, "weight");
    TORCH_CHECK(weight.scalar_type() == at::kChar && weight.dim() == 2 && weight.is_contiguous() && weight.size(1) == codes.size(-1), op,
                ": weight must be contiguous int8 [n, k] with k = ", codes.size(-1));
    check_on(scales, codes, op, "scales");
    check_on(weight_scales, codes, op, "weight_scales");
    const int64_t k = codes.size(-1), n = weight.size(0);
    TORCH_CHECK(k >= 1 && k <= TDE_INT8_MAX_K, op, ": 1 <= k <= ", TDE_INT8_MAX_K, " expected (sums are 32-bit integers), not ", k);
    const int64_t tokens = codes.numel() / k;
    TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.is_contiguous() && scales.numel() == tokens, op,
                ": scales must be contiguous fp32 with one value for each of the ", tokens, " rows of codes");
    TORCH_CHECK(weight_scales.scalar_type() == at::kFloat && weight_scales.is_contiguous() && weight_scales.numel() == n, op,
                ": weight_scales must be contiguous fp32 [n], n = ", n);
    const Tensor *b = given_or_null(bias);
    if (b != nullptr) {
        check_on(*b, codes, op, "bias");
        TORCH_CHECK(b->scalar_type() == at::kFloat && b->is_contiguous() && b->numel() == n, op, ": bias must be contiguous fp32 [n], n = ", n);
    }
    const at::ScalarType type = out_dtype.value_or(at::kBFloat16);
    tde_int8_product p{};
    p.out_dtype = out_code(type, op);
    const CallDevice device(codes);
    c10::SmallVector<int64_t, 5> shape(codes.sizes().begin(), codes.sizes().end());
    shape.back() = n;
    Tensor out = device.new_output(shape, type);
    p.tokens = tokens;
    p.k = k;
    p.n = n;
    p.codes = codes.data_ptr<int8_t>();
    p.weight = weight.data_ptr<int8_t>();
    p.scales = scales.data_ptr<float>();
    p.weight_scales = weight_scales.data_ptr<float>();
    p.bias = b != nullptr ? b->data_ptr<float>() : nullptr;
    p.out = out.data_ptr();
    check_status(tde_int8_linear(&p, device.stream()), op);
    return out;
}

Tensor int8_linear_meta(const Tensor &codes, const Tensor &, const Tensor &weight, const Tensor &, const c10::optional<Tensor> &,
                        c10::optional<at::ScalarType> out_dtype) {
    TORCH_CHECK(codes.dim() >= 1 && weight.dim() == 2, "int8_linear: codes [..., k] and weight [n, k] expected");
    c10::SymDimVector shape(codes.sym_sizes().begin(), codes.sym_sizes().end());
    shape.back() = weight.sym_size(0);
    return at::empty_symint(shape, codes.options().dtype(out_dtype.value_or(at::kBFloat16)));
}

// ---- heads and caches -----------------------------------------------------------------------------------------------

// What separates the elements of a dimension: nothing where there is one at most, whatever stride the tensor names.
int64_t stride_of(const Tensor &t, int64_t d) { return t.size(d) <= 1 ? 0 : t.stride(d); }

// [rows, heads, dim] with neighbouring channels; any row and head strides.
tde_heads heads_of(const Tensor &t, const Tensor &like, const char *op, const char *name) {
    check_on(t, like, op, name);
    TORCH_CHECK(t.dim() == 3, op, ": ", name, " must be [tokens, heads, dim]");
    TORCH_CHECK(t.size(1) <= 1 << 16, op, ": at most ", 1 << 16, " heads expected in ", name, ", not ", t.size(1));
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), op, ": ", name, " dtype differs");
    TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, op, ": channels of ", name, " must be contiguous");
    return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1)};
}

// Keys and values: [pages, page_size, heads, dim], any strides but the channels'.
tde_cache cache_of(const Tensor &t, const Tensor &like, int64_t heads, int64_t dim, const char *op, const char *name) {
    check_on(t, like, op, name);
    TORCH_CHECK(t.dim() == 4 && t.size(2) == heads && t.size(3) == dim, op, ": ", name, " must be [pages, page_size, kv_heads, dim] with ",
                heads, " heads of ", dim);
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), op, ": ", name, " dtype differs");
    TORCH_CHECK(t.size(3) <= 1 || t.stride(3) == 1, op, ": channels of ", name, " must be contiguous");
    return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)};
}

// A tensor and the addresses that it lies between, which is all that most calls need to know of it.
struct Spanned {
    const Tensor &t;
    const char *begin, *end;
    Spanned(const Tensor &tensor, const void *data) : t(tensor), begin(static_cast<const char *>(data)), end(begin) {
        int64_t last = 0;
        for (size_t i = 0; i < t.sizes().size(); ++i) {
            if (t.sizes()[i] == 0) return;
            last += (t.sizes()[i] - 1) * t.strides()[i];
        }
        end += (last + 1) * (int64_t)t.element_size();
    }
    tde::Region region() const { return {begin, (int)t.dim(), t.sizes().data(), t.strides().data(), (int64_t)t.element_size()}; }
};

// What a call writes takes every byte once, and shares none with what it reads or writes besides: rows run in no order.
void check_written(const Spanned &x, const char *op, const char *name) {
    TORCH_CHECK(x.t.is_contiguous() || !tde::overlaps_itself(x.region()), op, ": elements of ", name, " overlap");
}
void check_apart(const Spanned &written, const Spanned &other, const char *op, const char *name, const char *other_name) {
    TORCH_CHECK(written.end <= other.begin || other.end <= written.begin || !tde::overlap(written.region(), other.region()), op, ": ", name, " overlaps ",
                other_name);
}

// Counts a change of the tensor, so that a backward pass that saved it before refuses to run on other values.
void changed(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const int32_t *ints_of(const Tensor &t, const Tensor &like, int64_t size, const char *op, const char *name) {
    check_on(t, like, op, name);
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.size(0) == size, op, ": ", name,
                " must be contiguous int32 [", size, "]");
    return t.data_ptr<int32_t>();
}

tde_paged_batch batch_of(const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, const Tensor &k_cache, const Tensor &v_cache,
                         const Tensor &like, const char *op) {
    check_on(page_table, like, op, "page_table");
    TORCH_CHECK(page_table.scalar_type() == at::kInt && page_table.dim() == 2 && (page_table.size(1) <= 1 || page_table.stride(1) == 1), op,
                ": page_table must be int32 [sequences, pages] with contiguous rows");
    TORCH_CHECK(v_cache.size(0) == k_cache.size(0) && v_cache.size(1) == k_cache.size(1), op, ": the caches differ in pages or page size");
    TORCH_CHECK(k_cache.size(1) >= 1, op, ": pages must hold at least one token");
    const int64_t seqs = page_table.size(0), limit = 0x7fffffff;
    TORCH_CHECK(seqs <= limit && page_table.size(1) <= limit && k_cache.size(0) <= limit && k_cache.size(1) <= limit, op, ": too many pages");
    tde_paged_batch b{};
    b.page_table = page_table.data_ptr<int32_t>();
    b.table_stride = stride_of(page_table, 0);
    b.seqs = (int32_t)seqs;
    b.table_pages = (int32_t)page_table.size(1);
    b.cache_pages = (int32_t)k_cache.size(0);
    b.page_size = (int32_t)k_cache.size(1);
    b.q_starts = ints_of(q_starts, like, seqs + 1, op, "q_starts");
    b.kv_lens = ints_of(kv_lens, like, seqs, op, "kv_lens");
    return b;
}

const void *gamma_of(const Tensor *t, const Tensor &like, int64_t dim, const char *op, const char *name) {
    if (t == nullptr) return nullptr;
    check_on(*t, like, op, name);
    TORCH_CHECK(t->scalar_type() == like.scalar_type() && t->is_contiguous() && t->numel() == dim, op, ": ", name,
                " must be contiguous, of the heads' dtype, with ", dim, " elements");
    return t->data_ptr();
}

void rotation_of(tde_head_rows &r, const Tensor *cos_sin, const Tensor *positions, const Tensor &like, int64_t tokens, bool interleaved,
                 const char *op) {
    r.interleaved = interleaved;
    if (positions != nullptr) {
        check_on(*positions, like, op, "positions");
        TORCH_CHECK((positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt) && positions->dim() == 1 &&
                        positions->is_contiguous() && positions->size(0) == tokens,
                    op, ": positions must be contiguous int64 or int32 [", tokens, "]");
        r.positions = positions->data_ptr();
        r.positions_bytes = (int32_t)positions->element_size();
    }
    if (cos_sin == nullptr) return;
    check_on(*cos_sin, like, op, "cos_sin");
    TORCH_CHECK(cos_sin->scalar_type() == at::kFloat && cos_sin->dim() == 2 && (cos_sin->size(1) <= 1 || cos_sin->stride(1) == 1), op,
                ": cos_sin must be fp32 [positions, rot_dim] with contiguous rows");
    TORCH_CHECK(cos_sin->size(1) % 2 == 0 && cos_sin->size(1) <= like.size(2), op, ": rot_dim (columns of cos_sin) must be even and at most ",
                like.size(2), ", not ", cos_sin->size(1));
    r.cos_sin = cos_sin->data_ptr<float>();
    r.cos_sin_rows = cos_sin->size(0);
    r.cos_sin_stride = cos_sin->stride(0);
    r.rot_dim = (int32_t)cos_sin->size(1);
}

void common_of(tde_head_rows &r, const Tensor &k, double eps, const char *op) {
    TORCH_CHECK(k.is_cuda() && k.dim() == 3, op, ": k must be a GPU tensor [tokens, kv_heads, dim]");
    TORCH_CHECK(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf || k.scalar_type() == at::kFloat, op,
                ": unsupported dtype ", k.scalar_type(), " (bf16, fp16, fp32)");
    TORCH_CHECK(k.size(2) >= 1 && k.size(2) <= TDE_MAX_HEAD_DIM, op, ": heads of 1 to ", TDE_MAX_HEAD_DIM, " channels expected, not ", k.size(2));
    TORCH_CHECK(std::isfinite((float)eps) && eps >= 0.0, op, ": eps must be finite and not negative");
    r.dtype = dtype_code(k);
    r.dim = (int32_t)k.size(2);
    r.tokens = k.size(0);
    r.kv_heads = (int32_t)k.size(1);
    r.eps = (float)eps;
}

// ---- qk_norm_rope ---------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor &q, const Tensor &k, const Tensor &q_gamma, const Tensor &k_gamma, double eps,
                                        const Tensor &positions, const Tensor &cos_sin, bool interleaved) {
    constexpr const char *op = "qk_norm_rope";
    tde_head_rows r{};
    common_of(r, k, eps, op);
    r.q = heads_of(q, k, op, "q");
    r.k = heads_of(k, k, op, "k");
    TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2), op, ": q and k differ in tokens or dim");
    r.q_heads = (int32_t)q.size(1);
    r.q_gamma = gamma_of(&q_gamma, k, r.dim, op, "q_gamma");
    r.k_gamma = gamma_of(&k_gamma, k, r.dim, op, "k_gamma");
    rotation_of(r, &cos_sin, &positions, k, r.tokens, interleaved, op);
    const CallDevice device(k);
    Tensor q_out = device.new_like(q), k_out = device.new_like(k);
    r.q_out = heads_of(q_out, k, op, "q_out");
    r.k_out = heads_of(k_out, k, op, "k_out");
    check_status(tde_qk_norm_rope(&r, device.stream()), op);
    return {q_out, k_out};
}

std::tuple<Tensor, Tensor> qk_norm_rope_meta(const Tensor &q, const Tensor &k, const Tensor &, const Tensor &, double, const Tensor &,
                                             const Tensor &, bool) {
    return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options())};
}

// ---- append_kv ------------------------------------------------------------------------------------------------------

Tensor run_append(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table,
                  const Tensor &q_starts, const Tensor &kv_lens, const Tensor *q, const Tensor *cos_sin, const Tensor *positions,
                  const Tensor *q_gamma, const Tensor *k_gamma, double eps, bool interleaved) {
    constexpr const char *op = "append_kv";
    tde_head_rows r{};
    common_of(r, k, eps, op);
    r.k = heads_of(k, k, op, "k");
    r.v = heads_of(v, k, op, "v");
    TORCH_CHECK(v.sizes() == k.sizes(), op, ": k and v differ in shape");
    r.k_cache = cache_of(k_cache, k, r.kv_heads, r.dim, op, "k_cache");
    r.v_cache = cache_of(v_cache, k, r.kv_heads, r.dim, op, "v_cache");
    const Spanned keys(k_cache, r.k_cache.data), values(v_cache, r.v_cache.data);
    check_written(keys, op, "k_cache");
    check_written(values, op, "v_cache");
    check_apart(keys, values, op, "k_cache", "v_cache");
    const auto check_input = [&](const Spanned &rows, const char *name) {
        check_apart(keys, rows, op, "k_cache", name);
        check_apart(values, rows, op, "v_cache", name);
    };
    check_input({k, r.k.data}, "k");
    check_input({v, r.v.data}, "v");
    r.batch = batch_of(page_table, q_starts, kv_lens, k_cache, v_cache, k, op);
    r.k_gamma = gamma_of(k_gamma, k, r.dim, op, "k_gamma");
    rotation_of(r, cos_sin, positions, k, r.tokens, interleaved, op);
    const CallDevice device(k);
    Tensor q_out;
    if (q != nullptr) {
        r.q = heads_of(*q, k, op, "q");
        TORCH_CHECK(q->size(0) == k.size(0) && q->size(2) == k.size(2), op, ": q and k differ in tokens or dim");
        check_input({*q, r.q.data}, "q");
        r.q_heads = (int32_t)q->size(1);
        r.q_gamma = gamma_of(q_gamma, k, r.dim, op, "q_gamma");
        q_out = device.new_like(*q);
        r.q_out = heads_of(q_out, k, op, "q_out");
    }
    check_status(tde_append_kv(&r, device.stream()), op);
    changed(k_cache);
    changed(v_cache);
    return q_out;
}

// Two overloads, with queries and without: an optional output beside changed inputs is nothing that compiled graphs can hold.
void append_kv(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table, const Tensor &q_starts,
               const Tensor &kv_lens, const c10::optional<Tensor> &cos_sin, const c10::optional<Tensor> &positions,
               const c10::optional<Tensor> &k_gamma, double eps, bool interleaved) {
    run_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, nullptr, given_or_null(cos_sin), given_or_null(positions), nullptr,
               given_or_null(k_gamma), eps, interleaved);
}

Tensor append_kv_queries(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table,
                         const Tensor &q_starts, const Tensor &kv_lens, const Tensor &q, const c10::optional<Tensor> &cos_sin,
                         const c10::optional<Tensor> &positions, const c10::optional<Tensor> &q_gamma, const c10::optional<Tensor> &k_gamma,
                         double eps, bool interleaved) {
    return run_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, &q, given_or_null(cos_sin), given_or_null(positions),
                      given_or_null(q_gamma), given_or_null(k_gamma), eps, interleaved);
}

void append_kv_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                    const c10::optional<Tensor> &, const c10::optional<Tensor> &, const c10::optional<Tensor> &, double, bool) {}

Tensor append_kv_queries_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                              const Tensor &q, const c10::optional<Tensor> &, const c10::optional<Tensor> &, const c10::optional<Tensor> &,
                              const c10::optional<Tensor> &, double, bool) {
    return at::empty_symint(q.sym_sizes(), q.options());
}

// ---- paged_attention ------------------------------------------------------------------------------------------------

void run_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table, const Tensor &q_starts,
                   const Tensor &kv_lens, c10::optional<double> scale, const Tensor &out, bool zero_tail, const CallDevice &device) {
    constexpr const char *op = "paged_attention";
    tde_attention t{};
    t.dtype = dtype_code(q);
    t.q = heads_of(q, q, op, "q");
    t.out = heads_of(out, q, op, "out");
    TORCH_CHECK(out.sizes() == q.sizes(), op, ": out must be shaped like q");
    TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4, op, ": caches must be [pages, page_size, kv_heads, dim]");
    const int64_t heads = k_cache.size(2), dim = q.size(2);
    TORCH_CHECK(heads >= 1 && q.size(1) >= 1 && q.size(1) % heads == 0, op, ": ", q.size(1), " query heads are no multiple of ", heads, " key heads");
    TORCH_CHECK(dim >= 8 && dim <= 256 && dim % 8 == 0, op, ": heads of 8 to 256 channels in steps of 8 expected, not ", dim);
    t.k_cache = cache_of(k_cache, q, heads, dim, op, "k_cache");
    t.v_cache = cache_of(v_cache, q, heads, dim, op, "v_cache");
    if (!zero_tail) { // the caller's output
        const Spanned written(out, t.out.data);
        check_written(written, op, "out");
        check_apart(written, {q, t.q.data}, op, "out", "q");
        check_apart(written, {k_cache, t.k_cache.data}, op, "out", "k_cache");
        check_apart(written, {v_cache, t.v_cache.data}, op, "out", "v_cache");
    }
    t.batch = batch_of(page_table, q_starts, kv_lens, k_cache, v_cache, q, op);
    t.dim = (int32_t)dim;
    t.q_heads = (int32_t)q.size(1);
    t.kv_heads = (int32_t)heads;
    t.tokens = q.size(0);
    const double s = scale.value_or(1.0 / std::sqrt((double)dim));
    TORCH_CHECK((float)s > 0.0f && (float)s <= TDE_MAX_SCALE, op, ": scale must be positive and at most ", TDE_MAX_SCALE);
    t.scale = (float)s;
    t.zero_tail = zero_tail;
    check_status(tde_paged_attention_workspace(&t, &t.workspace_bytes), op);
    // allocated for this call: two captured graphs, or calls on two streams, share none
    Tensor workspace;
    if (t.workspace_bytes > 0) {
        workspace = device.new_output({t.workspace_bytes}, at::kByte);
        t.workspace = workspace.data_ptr();
    }
    check_status(tde_paged_attention(&t, device.stream()), op);
    if (!zero_tail) changed(out);
}

void check_queries(const Tensor &q) {
    TORCH_CHECK(q.is_cuda() && q.dim() == 3, "paged_attention: q must be a GPU tensor [tokens, heads, dim]");
    TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "paged_attention: unsupported dtype ", q.scalar_type(),
                " (bf16, fp16)");
}

Tensor paged_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table, const Tensor &q_starts,
                       const Tensor &kv_lens, c10::optional<double> scale) {
    check_queries(q);
    const CallDevice device(q);
    Tensor out = device.new_like(q);
    run_attention(q, k_cache, v_cache, page_table, q_starts, kv_lens, scale, out, true, device);
    return out;
}

void paged_attention_out(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table, const Tensor &q_starts,
                         const Tensor &kv_lens, const Tensor &out, c10::optional<double> scale) {
    check_queries(q);
    run_attention(q, k_cache, v_cache, page_table, q_starts, kv_lens, scale, out, false, CallDevice(q));
}

Tensor paged_attention_meta(const Tensor &q, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, c10::optional<double>) {
    return at::empty_symint(q.sym_sizes(), q.options());
}

void paged_attention_out_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                              c10::optional<double>) {}

} // namespace

TORCH_LIBRARY_FRAGMENT(torch_dist_ext, m) {
    m.def("int8_linear(Tensor codes, Tensor scales, Tensor weight, Tensor weight_scales, Tensor? bias=None, ScalarType? out_dtype=None) -> Tensor");
    m.def("qk_norm_rope(Tensor q, Tensor k, Tensor q_gamma, Tensor k_gamma, float eps, Tensor positions, Tensor cos_sin, "
          "bool interleaved=False) -> (Tensor, Tensor)");
    m.def("append_kv(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor q_starts, Tensor kv_lens, "
          "Tensor? cos_sin=None, Tensor? positions=None, Tensor? k_gamma=None, float eps=1e-06, bool interleaved=False) -> ()");
    m.def("append_kv.queries(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor q_starts, "
          "Tensor kv_lens, Tensor q, Tensor? cos_sin=None, Tensor? positions=None, Tensor? q_gamma=None, Tensor? k_gamma=None, "
          "float eps=1e-06, bool interleaved=False) -> Tensor");
    m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor q_starts, Tensor kv_lens, "
          "float? scale=None) -> Tensor");
    m.def("paged_attention_out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor q_starts, Tensor kv_lens, "
          "Tensor(a!) out, float? scale=None) -> ()");
}

TORCH_LIBRARY_IMPL(torch_dist_ext, CUDA, m) {
    m.impl("int8_linear", &int8_linear);
    m.impl("qk_norm_rope", &qk_norm_rope);
    m.impl("append_kv", &append_kv);
    m.impl("append_kv.queries", &append_kv_queries);
    m.impl("paged_attention", &paged_attention);
    m.impl("paged_attention_out", &paged_attention_out);
}

// Plain outputs, also where an input (a gamma as a parameter) requires a gradient: these operators serve, they have none.
TORCH_LIBRARY_IMPL(torch_dist_ext, Autograd, m) {
    m.impl("int8_linear", torch::CppFunction::makeFallthrough());
    m.impl("qk_norm_rope", torch::CppFunction::makeFallthrough());
    m.impl("append_kv", torch::CppFunction::makeFallthrough());
    m.impl("append_kv.queries", torch::CppFunction::makeFallthrough());
    m.impl("paged_attention", torch::CppFunction::makeFallthrough());
    m.impl("paged_attention_out", torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(torch_dist_ext, Meta, m) {
    m.impl("int8_linear", &int8_linear_meta);
    m.impl("qk_norm_rope", &qk_norm_rope_meta);
    m.impl("append_kv", &append_kv_meta);
    m.impl("append_kv.queries", &append_kv_queries_meta);
    m.impl("paged_attention", &paged_attention_meta);
    m.impl("paged_attention_out", &paged_attention_out_meta);
}
