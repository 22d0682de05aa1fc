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

struct HeadRowsPlan {
    int chunk_bytes; // a lane's part of a row; 0: elements
    int rows;        // rows a lane takes part in
    int lanes_log2;
    uint32_t waves_per_token, blocks;
};

int plan_head_rows(int elem, int dim, int half, bool interleaved, int64_t tokens, int64_t heads_all, HeadRowsPlan *p);
int launch_head_rows(HeadRowsArgs &a, int dtype, hipStream_t s);

} // namespace block
} // namespace tde

#endif // TDE_HEAD_ROWS_H
