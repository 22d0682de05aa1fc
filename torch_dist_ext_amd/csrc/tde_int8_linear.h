// Arguments and plan of the int8 product (tde_int8_linear.hip).
#ifndef TDE_INT8_LINEAR_H
#define TDE_INT8_LINEAR_H

#include "tde_block.h"

namespace tde {
namespace block {

struct LinearArgs {
    const int8_t *codes, *weight;
    const float *scales, *weight_scales, *bias; // bias may be null
    char *out;
    int64_t tokens, k, n;
};

int launch_int8_linear(const LinearArgs &a, int out_dtype, hipStream_t s);

} // namespace block
} // namespace tde

#endif // TDE_INT8_LINEAR_H
