// Arguments and plan of the paged attention kernels (tde_paged_attention.hip).  Strides are in bytes.
#ifndef TDE_PAGED_ATTENTION_H
#define TDE_PAGED_ATTENTION_H

#include "tde_block.h"

namespace tde {
namespace block {

// What joining the parts of a tile needs; chunks 0: nothing to join.
struct JoinItem {
    int32_t chunks, item; // their number, and the first one's item
    int32_t tile, begin, count, len;
};

struct AttentionArgs {
    const char *q, *k, *v;
    char *out;
    int64_t q_token, q_head, k_head, v_head, out_token, out_head;
    uint32_t k_page, k_slot, v_page, v_slot;
    PagedBatch batch;
    Divisor32 group;       // query heads a key head
    Divisor32 kv_heads;
    int64_t tokens;
    int64_t target;        // items that the split of the keys aims at, for each key head (split calls)
    int32_t items, tiles;  // at most; grids: items x key heads, and of the second launch tiles x key heads x rows
    int32_t min_chunk;     // keys of an item at least
    int32_t capacity;      // keys that a row of the page table can name
    int32_t dim;
    float scale_log2;      // scale * log2(e)
    float *partial;        // [items, kv_heads, rows of a tile, D + 4]: sums, their maximum and weight
    JoinItem *joins;       // [tiles]
    bool zero_tail;        // rows of no sequence become zeros
};

struct AttentionPlan {
    int wide_dim;   // 64, 128, 256: what the head is padded to in registers and LDS
    int rows;       // rows (token x query head of a group) of a tile
    bool split;     // the keys of a tile go to several workgroups, whose results a second launch joins
    int64_t items, tiles;
    int64_t target;
    int32_t min_chunk;
    int join_waves; // wavefronts that join a row
    int64_t workspace_bytes;
};

int plan_attention(int dim, int64_t tokens, int q_heads, int kv_heads, int seqs, int64_t capacity, AttentionPlan *p);
int launch_attention(AttentionArgs &a, const AttentionPlan &p, int dtype, hipStream_t s);

} // namespace block
} // namespace tde

#endif // TDE_PAGED_ATTENTION_H
