// Arguments of the head-row kernels (tde_head_rows.hip).  Index 0 is queries, 1 keys, 2 values; strides are in bytes.
#ifndef TDE_HEAD_ROWS_H
#define TDE_HEAD_ROWS_H

#include "tde_block.h"

namespace tde {
namespace block {

struct HeadRowsArgs {
    const char *in[3];
    int64_t in_token[3], in_head[3];
    char *out[3];
    int64_t out_token[3], out_head[3]; // keys and values of a paged call: a cache's slot and head strides
    int64_t out_page[3];
    const char *gamma[2]; // null: not normed
    const float *cos_sin; // [table_rows, 2 * half]
    int64_t table_rows, table_stride;
    const void *positions; // null: from the batch
    int64_t tokens;
    PagedBatch batch;
    Divisor32 waves_per_token;
    int32_t heads[3]; // 0: absent
    int32_t dim, half, lanes_log2;
    float eps;
    bool positions_wide, interleaved, paged;
};

// The token's place: its sequence's cache position and the slot's page.  position < 0: the row belongs to no sequence's range (it
// lies in front of the first one or behind the last, or its sequence is shorter than its new tokens).
struct Place {
    int64_t position;
    int32_t page, slot; // page < 0: not in the cache
};

__device__ __forceinline__ Place place_of(const PagedBatch &b, int64_t token, int lane) {
    Place p{-1, -1, 0};
    const int seq = __builtin_amdgcn_readfirstlane(sequence_of(b, token, lane));
    if (seq >= b.seqs) return p;
    const int64_t begin = b.starts[seq], end = b.starts[seq + 1], len = b.lens[seq];
    if (token < begin) return p;
    p.position = len - (end - begin) + (token - begin);
    if (p.position < 0) return p;
    if (p.position > 0x7fffffff) return p; // only where starts do not ascend
    const uint32_t at = b.page.quotient((uint32_t)p.position);
    p.slot = (int32_t)((uint32_t)p.position - at * b.page.d);
    p.page = page_number(b, b.table + seq * b.table_stride, at);
    return p;
}

__device__ __forceinline__ int64_t explicit_position(const HeadRowsArgs &a, int64_t token) {
    return a.positions_wide ? ((const int64_t *)a.positions)[token] : (int64_t)((const int32_t *)a.positions)[token];
}

// VE floats of the table; NaN where the position is not in it.
template <int N>
__device__ __forceinline__ void load_floats(const float *p, bool known, float (&x)[N]) {
    Words<N * 4> w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.w[i] = 0x7fc00000u;
    if (known) w = load_words<N * 4>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __builtin_bit_cast(float, w.w[i]);
}

struct HeadRowsPlan {
    int chunk_bytes; // a lane's part of a row; 0: elements
    int rows;        // rows a lane takes part in
    int lanes_log2;
    uint32_t waves_per_token, blocks;
};

// Keys and values into caches in 4 bits: out[1] and out[2] are codes, their scales beside them.
struct HeadRowsFp4Args : HeadRowsArgs {
    char *scales[2];
    int64_t scale_page[2], scale_slot[2], scale_head[2];
    int32_t most_exponent;
    int32_t rounds[3]; // as many rows as a wavefront has at once
    int32_t turns;     // times that a wavefront takes rows
};

int plan_head_rows(int elem, int dim, int half, bool interleaved, int64_t tokens, int64_t heads_all, HeadRowsPlan *p);
int launch_head_rows(HeadRowsArgs &a, int dtype, hipStream_t s);
int launch_head_rows_fp4(HeadRowsFp4Args &a, int dtype, hipStream_t s);

} // namespace block
} // namespace tde

#endif // TDE_HEAD_ROWS_H
