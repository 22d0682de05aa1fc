// Operators of the attention block over a paged cache in 4 bits: registration in the `torch_dist_ext` namespace, argument checks, outputs.
#include <torch/library.h>

#include <cmath>
#include <tuple>

#include "tde_block_torch.h"

namespace {

void check_dim(int64_t dim, const char *op) {
    TORCH_CHECK(dim >= TDE_FP4_BLOCK && dim <= TDE_FP4_MAX_DIM && dim % TDE_FP4_BLOCK == 0, op, ": heads of ", TDE_FP4_BLOCK, " to ", TDE_FP4_MAX_DIM,
                " channels in steps of ", TDE_FP4_BLOCK, " expected, not ", dim);
}

// Codes or scales of keys or values: bytes [pages, page_size, heads, width], any strides but the last dimension's.
tde_cache bytes_of(const Tensor &t, const Tensor &like, int64_t heads, int64_t width, const char *op, const char *name) {
    check_on(t, like, op, name);
    TORCH_CHECK(t.scalar_type() == at::kByte, op, ": ", name, " must be uint8, not ", t.scalar_type());
    TORCH_CHECK(t.dim() == 4 && t.size(2) == heads && t.size(3) == width, op, ": ", name, " must be [pages, page_size, kv_heads, ", width, "] with ", heads, " heads");
    TORCH_CHECK(t.size(3) <= 1 || t.stride(3) == 1, op, ": bytes of a head in ", name, " must be contiguous");
    return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)};
}

void check_scales(const Tensor &scales, const Tensor &codes, const char *op, const char *name) {
    TORCH_CHECK(scales.size(0) == codes.size(0) && scales.size(1) == codes.size(1), op, ": ", name, " differs from its cache in pages or page size");
}

// ---- append_kv_fp4 --------------------------------------------------------------------------------------------------

Tensor run_append(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &k_scales, const Tensor &v_cache, const Tensor &v_scales,
                  const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, const Tensor *q, const Tensor *cos_sin,
                  const Tensor *positions, const Tensor *q_gamma, const Tensor *k_gamma, double eps, bool interleaved) {
    constexpr const char *op = "append_kv_fp4";
    tde_append_fp4 t{};
    tde_head_rows &r = t.rows;
    common_of(r, k, eps, op);
    check_dim(r.dim, op);
    r.k = heads_of(k, k, op, "k");
    r.v = heads_of(v, k, op, "v");
    TORCH_CHECK(v.sizes() == k.sizes(), op, ": k and v differ in shape");
    r.k_cache = bytes_of(k_cache, k, r.kv_heads, r.dim / 2, op, "k_cache");
    r.v_cache = bytes_of(v_cache, k, r.kv_heads, r.dim / 2, op, "v_cache");
    t.k_scales = bytes_of(k_scales, k, r.kv_heads, r.dim / TDE_FP4_BLOCK, op, "k_scales");
    t.v_scales = bytes_of(v_scales, k, r.kv_heads, r.dim / TDE_FP4_BLOCK, op, "v_scales");
    check_scales(k_scales, k_cache, op, "k_scales");
    check_scales(v_scales, v_cache, op, "v_scales");
    const Spanned written[] = {{k_cache, r.k_cache.data}, {k_scales, t.k_scales.data}, {v_cache, r.v_cache.data}, {v_scales, t.v_scales.data}};
    constexpr const char *names[] = {"k_cache", "k_scales", "v_cache", "v_scales"};
    for (int i = 0; i < 4; ++i) {
        check_written(written[i], op, names[i]);
        for (int j = i + 1; j < 4; ++j) check_apart(written[i], written[j], op, names[i], names[j]);
    }
    const auto check_input = [&](const Spanned &rows, const char *name) {
        for (int i = 0; i < 4; ++i) check_apart(written[i], rows, op, names[i], name);
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
    check_status(tde_append_kv_fp4(&t, device.stream()), op);
    for (const Spanned &w : written) changed(w.t);
    return q_out;
}

// Two overloads, with queries and without, as append_kv's.
void append_kv_fp4(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &k_scales, const Tensor &v_cache, const Tensor &v_scales,
                   const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, const c10::optional<Tensor> &cos_sin,
                   const c10::optional<Tensor> &positions, const c10::optional<Tensor> &k_gamma, double eps, bool interleaved) {
    run_append(k, v, k_cache, k_scales, v_cache, v_scales, page_table, q_starts, kv_lens, nullptr, given_or_null(cos_sin), given_or_null(positions), nullptr,
               given_or_null(k_gamma), eps, interleaved);
}

Tensor append_kv_fp4_queries(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &k_scales, const Tensor &v_cache,
                             const Tensor &v_scales, const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, const Tensor &q,
                             const c10::optional<Tensor> &cos_sin, const c10::optional<Tensor> &positions, const c10::optional<Tensor> &q_gamma,
                             const c10::optional<Tensor> &k_gamma, double eps, bool interleaved) {
    return run_append(k, v, k_cache, k_scales, v_cache, v_scales, page_table, q_starts, kv_lens, &q, given_or_null(cos_sin), given_or_null(positions),
                      given_or_null(q_gamma), given_or_null(k_gamma), eps, interleaved);
}

void append_kv_fp4_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                        const Tensor &, const c10::optional<Tensor> &, const c10::optional<Tensor> &, const c10::optional<Tensor> &, double, bool) {}

Tensor append_kv_fp4_queries_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                  const Tensor &, const Tensor &, const Tensor &q, const c10::optional<Tensor> &, const c10::optional<Tensor> &,
                                  const c10::optional<Tensor> &, const c10::optional<Tensor> &, double, bool) {
    return at::empty_symint(q.sym_sizes(), q.options());
}

// ---- paged_attention_fp4 --------------------------------------------------------------------------------------------

void run_attention(const Tensor &q, const Tensor &k_cache, const Tensor &k_scales, const Tensor &v_cache, const Tensor &v_scales,
                   const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, c10::optional<double> scale, const Tensor &out,
                   bool zero_tail, const CallDevice &device) {
    constexpr const char *op = "paged_attention_fp4";
    tde_attention_fp4 f{};
    tde_attention &t = f.attention;
    t.dtype = dtype_code(q);
    t.q = heads_of(q, q, op, "q");
    t.out = heads_of(out, q, op, "out");
    TORCH_CHECK(out.sizes() == q.sizes(), op, ": out must be shaped like q");
    TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4, op, ": caches must be [pages, page_size, kv_heads, dim / 2]");
    const int64_t heads = k_cache.size(2), dim = q.size(2);
    TORCH_CHECK(heads >= 1 && q.size(1) >= 1 && q.size(1) % heads == 0, op, ": ", q.size(1), " query heads are no multiple of ", heads, " key heads");
    check_dim(dim, op);
    t.k_cache = bytes_of(k_cache, q, heads, dim / 2, op, "k_cache");
    t.v_cache = bytes_of(v_cache, q, heads, dim / 2, op, "v_cache");
    f.k_scales = bytes_of(k_scales, q, heads, dim / TDE_FP4_BLOCK, op, "k_scales");
    f.v_scales = bytes_of(v_scales, q, heads, dim / TDE_FP4_BLOCK, op, "v_scales");
    check_scales(k_scales, k_cache, op, "k_scales");
    check_scales(v_scales, v_cache, op, "v_scales");
    if (!zero_tail) { // the caller's output
        const Spanned written(out, t.out.data);
        check_written(written, op, "out");
        check_apart(written, {q, t.q.data}, op, "out", "q");
        check_apart(written, {k_cache, t.k_cache.data}, op, "out", "k_cache");
        check_apart(written, {v_cache, t.v_cache.data}, op, "out", "v_cache");
        check_apart(written, {k_scales, f.k_scales.data}, op, "out", "k_scales");
        check_apart(written, {v_scales, f.v_scales.data}, op, "out", "v_scales");
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
    check_status(tde_paged_attention_fp4_workspace(&f, &t.workspace_bytes), op);
    // allocated for this call: two captured graphs, or calls on two streams, share none
    Tensor workspace;
    if (t.workspace_bytes > 0) {
        workspace = device.new_output({t.workspace_bytes}, at::kByte);
        t.workspace = workspace.data_ptr();
    }
    check_status(tde_paged_attention_fp4(&f, device.stream()), op);
    if (!zero_tail) changed(out);
}

void check_queries(const Tensor &q) {
    TORCH_CHECK(q.is_cuda() && q.dim() == 3, "paged_attention_fp4: q must be a GPU tensor [tokens, heads, dim]");
    TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "paged_attention_fp4: unsupported dtype ", q.scalar_type(),
                " (bf16, fp16)");
}

Tensor paged_attention_fp4(const Tensor &q, const Tensor &k_cache, const Tensor &k_scales, const Tensor &v_cache, const Tensor &v_scales,
                           const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, c10::optional<double> scale) {
    check_queries(q);
    const CallDevice device(q);
    Tensor out = device.new_like(q);
    run_attention(q, k_cache, k_scales, v_cache, v_scales, page_table, q_starts, kv_lens, scale, out, true, device);
    return out;
}

void paged_attention_fp4_out(const Tensor &q, const Tensor &k_cache, const Tensor &k_scales, const Tensor &v_cache, const Tensor &v_scales,
                             const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, const Tensor &out, c10::optional<double> scale) {
    check_queries(q);
    run_attention(q, k_cache, k_scales, v_cache, v_scales, page_table, q_starts, kv_lens, scale, out, false, CallDevice(q));
}

Tensor paged_attention_fp4_meta(const Tensor &q, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                const Tensor &, c10::optional<double>) {
    return at::empty_symint(q.sym_sizes(), q.options());
}

void paged_attention_fp4_out_meta(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                  const Tensor &, const Tensor &, c10::optional<double>) {}

// ---- unpack_fp4 -----------------------------------------------------------------------------------------------------

Tensor unpack_fp4(const Tensor &codes, const Tensor &scales, c10::optional<at::ScalarType> out_dtype) {
    constexpr const char *op = "unpack_fp4";
    TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kByte && codes.dim() >= 1, op, ": codes must be a uint8 GPU tensor [..., dim / 2]");
    check_on(scales, codes, op, "scales");
    const int64_t last = codes.dim() - 1, dim = codes.size(last) * 2;
    check_dim(dim, op);
    TORCH_CHECK(scales.scalar_type() == at::kByte && scales.dim() == codes.dim() && scales.size(last) == dim / TDE_FP4_BLOCK &&
                    scales.sizes().slice(0, last) == codes.sizes().slice(0, last),
                op, ": scales must be uint8, one for each ", TDE_FP4_BLOCK, " channels of codes");
    TORCH_CHECK(codes.stride(last) == 1 && (scales.size(last) <= 1 || scales.stride(last) == 1), op, ": bytes of a row must be contiguous");
    const at::ScalarType type = out_dtype.value_or(at::kBFloat16);
    tde_unpack_fp4_rows r{};
    r.out_dtype = out_code(type, op);
    r.dim = (int32_t)dim;
    // dimensions from the last one on; one that continues the one before it joins it
    int n = 0;
    int64_t sizes[3] = {1, 1, 1}, code_strides[3] = {}, scale_strides[3] = {};
    for (int64_t d = last - 1; d >= 0 && codes.numel() > 0; --d) {
        if (codes.size(d) == 1) continue;
        if (n > 0 && codes.stride(d) == code_strides[n - 1] * sizes[n - 1] && scales.stride(d) == scale_strides[n - 1] * sizes[n - 1]) {
            sizes[n - 1] *= codes.size(d);
            continue;
        }
        TORCH_CHECK(n < 3, op, ": rows in at most three dimensions that do not continue one another expected");
        sizes[n] = codes.size(d);
        code_strides[n] = codes.stride(d);
        scale_strides[n] = scales.stride(d);
        ++n;
    }
    if (codes.numel() == 0) sizes[0] = 0;
    for (int i = 0; i < 3; ++i) {
        r.sizes[2 - i] = sizes[i];
        r.code_strides[2 - i] = code_strides[i];
        r.scale_strides[2 - i] = scale_strides[i];
    }
    const CallDevice device(codes);
    c10::SmallVector<int64_t, 5> shape(codes.sizes().begin(), codes.sizes().end());
    shape.back() = dim;
    Tensor out = device.new_output(shape, type);
    r.codes = codes.data_ptr<uint8_t>();
    r.scales = scales.data_ptr<uint8_t>();
    r.out = out.data_ptr();
    check_status(tde_unpack_fp4(&r, device.stream()), op);
    return out;
}

Tensor unpack_fp4_meta(const Tensor &codes, const Tensor &, c10::optional<at::ScalarType> out_dtype) {
    TORCH_CHECK(codes.dim() >= 1, "unpack_fp4: codes [..., dim / 2] expected");
    c10::SymDimVector shape(codes.sym_sizes().begin(), codes.sym_sizes().end());
    shape.back() = shape.back() * 2;
    return at::empty_symint(shape, codes.options().dtype(out_dtype.value_or(at::kBFloat16)));
}

// ---- update_pages ---------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> update_pages(const Tensor &page_table, const Tensor &kv_lens, const Tensor &new_tokens, const Tensor &free_pages,
                                                const Tensor &free_count, int64_t page_size, int64_t tokens, const c10::optional<Tensor> &keep_lens) {
    constexpr const char *op = "update_pages";
    constexpr int64_t limit = 0x7fffffff;
    TORCH_CHECK(page_table.is_cuda() && page_table.scalar_type() == at::kInt && page_table.dim() == 2 &&
                    (page_table.size(1) <= 1 || page_table.stride(1) == 1),
                op, ": page_table must be an int32 GPU tensor [sequences, pages] with contiguous rows");
    const int64_t seqs = page_table.size(0);
    TORCH_CHECK(seqs <= 1 << 24 && page_table.size(1) <= limit, op, ": too many pages");
    TORCH_CHECK(page_size >= 1 && page_size <= limit, op, ": pages must hold at least one token, and fewer than 2^31");
    TORCH_CHECK(tokens >= 0, op, ": tokens must not be negative");
    tde_page_update u{};
    u.page_table = page_table.data_ptr<int32_t>();
    u.table_stride = stride_of(page_table, 0);
    u.seqs = (int32_t)seqs;
    u.table_pages = (int32_t)page_table.size(1);
    u.page_size = (int32_t)page_size;
    u.tokens = tokens;
    u.kv_lens = const_cast<int32_t *>(ints_of(kv_lens, page_table, seqs, op, "kv_lens"));
    u.new_tokens = ints_of(new_tokens, page_table, seqs, op, "new_tokens");
    const Tensor *keep = given_or_null(keep_lens);
    if (keep != nullptr) u.keep_lens = ints_of(*keep, page_table, seqs, op, "keep_lens");
    TORCH_CHECK(free_pages.dim() == 1 && free_pages.size(0) <= limit, op, ": free_pages must be contiguous int32 [capacity]");
    u.free_pages = const_cast<int32_t *>(ints_of(free_pages, page_table, free_pages.size(0), op, "free_pages"));
    u.free_capacity = (int32_t)free_pages.size(0);
    u.free_count = const_cast<int32_t *>(ints_of(free_count, page_table, 1, op, "free_count"));
    const Spanned written[] = {{page_table, u.page_table}, {kv_lens, u.kv_lens}, {free_pages, u.free_pages}, {free_count, u.free_count}};
    constexpr const char *names[] = {"page_table", "kv_lens", "free_pages", "free_count"};
    for (int i = 0; i < 4; ++i) {
        check_written(written[i], op, names[i]);
        for (int j = i + 1; j < 4; ++j) check_apart(written[i], written[j], op, names[i], names[j]);
        check_apart(written[i], {new_tokens, u.new_tokens}, op, names[i], "new_tokens");
        if (keep != nullptr) check_apart(written[i], {*keep, u.keep_lens}, op, names[i], "keep_lens");
    }
    const CallDevice device(page_table);
    Tensor q_starts = device.new_output({seqs + 1}, at::kInt), positions = device.new_output({tokens}, at::kInt), slots = device.new_output({tokens}, at::kLong);
    u.q_starts = q_starts.data_ptr<int32_t>();
    u.positions = positions.data_ptr<int32_t>();
    u.slots = slots.data_ptr<int64_t>();
    check_status(tde_update_pages(&u, device.stream()), op);
    for (const Spanned &w : written) changed(w.t);
    return {q_starts, positions, slots};
}

std::tuple<Tensor, Tensor, Tensor> update_pages_meta(const Tensor &page_table, const Tensor &, const Tensor &, const Tensor &, const Tensor &, int64_t,
                                                     c10::SymInt tokens, const c10::optional<Tensor> &) {
    return {at::empty_symint({page_table.sym_size(0) + 1}, page_table.options()), at::empty_symint({tokens}, page_table.options()),
            at::empty_symint({tokens}, page_table.options().dtype(at::kLong))};
}

} // namespace

TORCH_LIBRARY_FRAGMENT(torch_dist_ext, m) {
    m.def("append_kv_fp4(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) k_scales, Tensor(c!) v_cache, Tensor(d!) v_scales, Tensor page_table, "
          "Tensor q_starts, Tensor kv_lens, Tensor? cos_sin=None, Tensor? positions=None, Tensor? k_gamma=None, float eps=1e-06, "
          "bool interleaved=False) -> ()");
    m.def("append_kv_fp4.queries(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) k_scales, Tensor(c!) v_cache, Tensor(d!) v_scales, "
          "Tensor page_table, Tensor q_starts, Tensor kv_lens, Tensor q, Tensor? cos_sin=None, Tensor? positions=None, Tensor? q_gamma=None, "
          "Tensor? k_gamma=None, float eps=1e-06, bool interleaved=False) -> Tensor");
    m.def("paged_attention_fp4(Tensor q, Tensor k_cache, Tensor k_scales, Tensor v_cache, Tensor v_scales, Tensor page_table, Tensor q_starts, "
          "Tensor kv_lens, float? scale=None) -> Tensor");
    m.def("paged_attention_fp4_out(Tensor q, Tensor k_cache, Tensor k_scales, Tensor v_cache, Tensor v_scales, Tensor page_table, Tensor q_starts, "
          "Tensor kv_lens, Tensor(a!) out, float? scale=None) -> ()");
    m.def("unpack_fp4(Tensor codes, Tensor scales, ScalarType? out_dtype=None) -> Tensor");
    m.def("update_pages(Tensor(a!) page_table, Tensor(b!) kv_lens, Tensor new_tokens, Tensor(c!) free_pages, Tensor(d!) free_count, int page_size, "
          "SymInt tokens, Tensor? keep_lens=None) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(torch_dist_ext, CUDA, m) {
    m.impl("append_kv_fp4", &append_kv_fp4);
    m.impl("append_kv_fp4.queries", &append_kv_fp4_queries);
    m.impl("paged_attention_fp4", &paged_attention_fp4);
    m.impl("paged_attention_fp4_out", &paged_attention_fp4_out);
    m.impl("unpack_fp4", &unpack_fp4);
    m.impl("update_pages", &update_pages);
}

// Plain outputs, also where an input requires a gradient: these operators serve, they have none.
TORCH_LIBRARY_IMPL(torch_dist_ext, Autograd, m) {
    for (const char *name : {"append_kv_fp4", "append_kv_fp4.queries", "paged_attention_fp4", "paged_attention_fp4_out", "unpack_fp4", "update_pages"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(torch_dist_ext, Meta, m) {
    m.impl("append_kv_fp4", &append_kv_fp4_meta);
    m.impl("append_kv_fp4.queries", &append_kv_fp4_queries_meta);
    m.impl("paged_attention_fp4", &paged_attention_fp4_meta);
    m.impl("paged_attention_fp4_out", &paged_attention_fp4_out_meta);
    m.impl("unpack_fp4", &unpack_fp4_meta);
    m.impl("update_pages", &update_pages_meta);
}
