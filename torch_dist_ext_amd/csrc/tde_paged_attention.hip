// Attention over caches that hold keys and values in the queries' type: which kernel takes a call, and its launch.
#include "tde_paged_attention_kernel.h"

namespace tde {
namespace block {

// Which kernel, and whether the keys are split.  capacity: keys that the page table can name for a sequence.  (Times on 256 units.)
//
// Rows of a tile: 16, with every wavefront on keys of its own, where sequences have no more rows than that on average (decode steps:
// bound by the cache's bytes); 128 where they give three workgroups a unit, else 64: a wavefront then has half the work
// between two barriers, which is what few workgroups wait for (mixed batch of 576 workgroups of 128 rows 74 us, of 64 rows 62; one
// chunk of 4096 rows behind 4096, 1024 workgroups, 425 and 630).  Heads of more than 128 channels have registers for one block of
// rows a wavefront: 128 rows are eight wavefronts, two a SIMD, wherever they give every unit a workgroup (12 sequences of up to 800 tokens behind
// 3000, 8 heads, 300 workgroups: 198 us, of 64 rows 235; 2048 tokens behind 2048, 128 workgroups: 191 and 164).
//
// Keys are split where a launch would not give every unit its workgroups (four of 16 rows each, one else), into about as many
// items as that and twice as many of the larger tiles, and none of less than 256 keys (one decode row over 131072 keys 24 us).  Splitting
// beyond that was measured with heads of 256 alone, one wavefront a SIMD (2048 tokens behind 2048 164 us, split 243).  The rule
// sees rows, not lengths, those of no sequence included: one long sequence among many, or decode rows beside chunks that fill the
// units, are walked by one workgroup a key head.
int plan_attention(int dim, int64_t tokens, int q_heads, int kv_heads, int seqs, int64_t capacity, AttentionPlan *p) {
    return plan_attention_rows(dim, tokens, q_heads, kv_heads, seqs, capacity, 16, 128, p);
}

// least_rows, most_rows: of a tile.
int plan_attention_rows(int dim, int64_t tokens, int q_heads, int kv_heads, int seqs, int64_t capacity, int least_rows, int most_rows, AttentionPlan *p) {
    *p = AttentionPlan{};
    p->wide_dim = dim <= 64 ? 64 : (dim <= 128 ? 128 : 256);
    const int64_t group = q_heads / kv_heads, rows_all = tokens * group, cus = device_compute_units();
    if (rows_all > 0x7fffff00) return TDE_ETOOBIG;
    if (rows_all <= (int64_t)seqs * 16 && least_rows == 16) p->rows = 16;
    else p->rows = most_rows >= 128 && rows_all / 128 * kv_heads >= (p->wide_dim <= 128 ? 3 : 1) * cus ? 128 : 64;
    const int64_t tiles = rows_all / p->rows + seqs + 2; // at most: one part tile a sequence, one in front of them and one behind
    const int64_t likely = std::max<int64_t>(1, std::max(rows_all / p->rows, std::min<int64_t>(seqs, tokens))); // rather
    p->min_chunk = 256;
    p->split = p->rows < 128 && likely * kv_heads < (p->rows == 16 ? 4 : 1) * cus && capacity > p->min_chunk;
    p->target = std::max<int64_t>(1, (p->rows == 16 ? 4 : 2) * cus / kv_heads);
    p->tiles = tiles;
    p->items = tiles + (p->split ? p->target : 0);
    if (p->items > 0x7fffff00 / kv_heads || (p->split && tiles > 0x7fffff00 / kv_heads / p->rows)) return TDE_ETOOBIG;
    // of a row: where it may have many parts, and a launch holds them for as many tiles as there may be
    p->join_waves = p->target / likely >= 32 && fits_launch(tiles * kv_heads * p->rows, 1024) ? 16 : 1;
    // eight wavefronts are the most that a tile has
    if (!fits_launch(p->items * kv_heads, p->wide_dim == 256 && p->rows == 128 ? 512 : 256)) return TDE_ETOOBIG;
    if (p->split && !fits_launch(tiles * kv_heads * (p->rows / 4), 256)) return TDE_ETOOBIG;
    if (p->split)
        p->workspace_bytes = p->tiles * (int64_t)sizeof(JoinItem) + p->items * kv_heads * p->rows * (int64_t)(p->wide_dim + 4) * 4;
    return TDE_OK;
}

int launch_attention(AttentionArgs &a, const AttentionPlan &p, int dtype, hipStream_t s) { return launch_planned<Held16>(a, p, dtype, s); }

} // namespace block
} // namespace tde
