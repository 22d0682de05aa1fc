// Attention over paged caches in 4 bits: e2m1 codes with a power of two for 32 channels.
#include "tde_paged_attention_kernel.h"

namespace tde {
namespace block {

int plan_attention_fp4(int dim, int64_t tokens, int q_heads, int kv_heads, int seqs, int64_t capacity, AttentionPlan *p) {
    return plan_attention_rows(dim, tokens, q_heads, kv_heads, seqs, capacity, 64, p);
}

int launch_attention_fp4(AttentionFp4Args &a, const AttentionPlan &p, int dtype, hipStream_t s) { return launch_planned<HeldFp4>(a, p, dtype, s); }

} // namespace block
} // namespace tde
