// Arguments of the kernels that move pages between sequences (tde_page_update.hip).
#ifndef TDE_PAGE_UPDATE_H
#define TDE_PAGE_UPDATE_H

#include "tde_block.h"

namespace tde {
namespace block {

struct PageUpdateArgs {
    int32_t *table, *lens;
    const int32_t *added, *kept; // kept may be null
    int32_t *stack, *count, *starts, *positions;
    int64_t *slots;
    int64_t table_stride;
    int32_t tokens, seqs, width, capacity;
    Divisor32 page;
};

int launch_page_update(const PageUpdateArgs &a, hipStream_t s);

} // namespace block
} // namespace tde

#endif // TDE_PAGE_UPDATE_H
