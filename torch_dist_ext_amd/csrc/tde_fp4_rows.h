// Arguments of the kernel that turns codes and scales into numbers (tde_fp4_rows.hip).  Strides are in bytes.
#ifndef TDE_FP4_ROWS_H
#define TDE_FP4_ROWS_H

#include "tde_block.h"

namespace tde {
namespace block {

struct UnpackArgs {
    const char *codes, *scales;
    char *out;
    int64_t code_stride[3], scale_stride[3];
    Divisor32 pieces;       // of 8 channels a row
    Divisor32 inner, middle; // sizes of the last dimension of rows and of the one before
    uint32_t total;         // pieces of all rows
};

int launch_unpack_fp4(const UnpackArgs &a, int out_dtype, hipStream_t s);

} // namespace block
} // namespace tde

#endif // TDE_FP4_ROWS_H
