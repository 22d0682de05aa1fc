// What the registrations of the attention block's operators share: checks of tensors, and their descriptions for the C ABI.
#ifndef TDE_BLOCK_TORCH_H
#define TDE_BLOCK_TORCH_H

#include <cmath>

#include "tde_overlap.h"
#include "tde_torch.h"

namespace {

[[maybe_unused]] const Tensor *given_or_null(const c10::optional<Tensor> &t) { return t.has_value() && t->defined() ? &*t : nullptr; }

[[maybe_unused]] void check_on(const Tensor &t, const Tensor &like, const char *op, const char *name) {
    TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a GPU tensor");
    TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on a different device");
}

[[maybe_unused]] int32_t out_code(at::ScalarType t, const char *op) {
    TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, op, ": out_dtype must be bf16, fp16 or fp32, not ", t);
    return t == at::kBFloat16 ? TDE_BF16 : (t == at::kHalf ? TDE_F16 : TDE_F32);
}

// ---- heads and caches -----------------------------------------------------------------------------------------------

// What separates the elements of a dimension: nothing where there is one at most, whatever stride the tensor names.
[[maybe_unused]] int64_t stride_of(const Tensor &t, int64_t d) { return t.size(d) <= 1 ? 0 : t.stride(d); }

// [rows, heads, dim] with neighbouring channels; any row and head strides.
[[maybe_unused]] tde_heads heads_of(const Tensor &t, const Tensor &like, const char *op, const char *name) {
    check_on(t, like, op, name);
    TORCH_CHECK(t.dim() == 3, op, ": ", name, " must be [tokens, heads, dim]");
    TORCH_CHECK(t.size(1) <= 1 << 16, op, ": at most ", 1 << 16, " heads expected in ", name, ", not ", t.size(1));
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), op, ": ", name, " dtype differs");
    TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, op, ": channels of ", name, " must be contiguous");
    return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1)};
}

// Keys and values: [pages, page_size, heads, dim], any strides but the channels'.
[[maybe_unused]] tde_cache cache_of(const Tensor &t, const Tensor &like, int64_t heads, int64_t dim, const char *op, const char *name) {
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
[[maybe_unused]] void check_written(const Spanned &x, const char *op, const char *name) {
    TORCH_CHECK(x.t.is_contiguous() || !tde::overlaps_itself(x.region()), op, ": elements of ", name, " overlap");
}
[[maybe_unused]] void check_apart(const Spanned &written, const Spanned &other, const char *op, const char *name, const char *other_name) {
    TORCH_CHECK(written.end <= other.begin || other.end <= written.begin || !tde::overlap(written.region(), other.region()), op, ": ", name, " overlaps ",
                other_name);
}

// Counts a change of the tensor, so that a backward pass that saved it before refuses to run on other values.
[[maybe_unused]] void changed(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

[[maybe_unused]] const int32_t *ints_of(const Tensor &t, const Tensor &like, int64_t size, const char *op, const char *name) {
    check_on(t, like, op, name);
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.size(0) == size, op, ": ", name,
                " must be contiguous int32 [", size, "]");
    return t.data_ptr<int32_t>();
}

[[maybe_unused]] tde_paged_batch batch_of(const Tensor &page_table, const Tensor &q_starts, const Tensor &kv_lens, const Tensor &k_cache, const Tensor &v_cache,
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

[[maybe_unused]] const void *gamma_of(const Tensor *t, const Tensor &like, int64_t dim, const char *op, const char *name) {
    if (t == nullptr) return nullptr;
    check_on(*t, like, op, name);
    TORCH_CHECK(t->scalar_type() == like.scalar_type() && t->is_contiguous() && t->numel() == dim, op, ": ", name,
                " must be contiguous, of the heads' dtype, with ", dim, " elements");
    return t->data_ptr();
}

[[maybe_unused]] void rotation_of(tde_head_rows &r, const Tensor *cos_sin, const Tensor *positions, const Tensor &like, int64_t tokens, bool interleaved,
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

[[maybe_unused]] void common_of(tde_head_rows &r, const Tensor &k, double eps, const char *op) {
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

} // namespace

#endif // TDE_BLOCK_TORCH_H
