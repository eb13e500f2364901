// Attention over i8 paged caches (attend_kernel.h).
#include "attend_kernel.h"

namespace ep {

void attend_i8(const AttendArgs &a, int q_dtype, int mt, unsigned grid, hipStream_t st)
{
    if (q_dtype == EP_BF16)
        attend_by_rows<OpBf16, EP_I8>(a, mt, grid, st);
    else
        attend_by_rows<OpF16, EP_I8>(a, mt, grid, st);
}

}  // namespace ep
