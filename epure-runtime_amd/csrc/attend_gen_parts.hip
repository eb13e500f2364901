// Attention over the tables' common pages and those behind them (attend_kernel.h).
#include "attend_kernel.h"

namespace ep {

void attend_parts(const AttendParts &a, int q_dtype, int mt, unsigned grid, hipStream_t st)
{
    if (a.c.dtype == EP_BF16)
        attend_other_by_size<OpBf16, EP_BF16>(a, mt, grid, st);
    else if (a.c.dtype == EP_F16)
        attend_other_by_size<OpF16, EP_F16>(a, mt, grid, st);
    else if (a.c.dtype == EP_I8)
        attend_other_by_query<EP_I8>(a, q_dtype, mt, grid, st);
    else
        attend_other_by_query<EP_E4M3>(a, q_dtype, mt, grid, st);
}

}  // namespace ep
