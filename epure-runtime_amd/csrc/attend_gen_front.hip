// Attention over the tables' common pages, many rows (attend_front.h).
#include "attend_front.h"

namespace ep {

void attend_front(const FrontArgs &a, int q_dtype, unsigned grid, hipStream_t st)
{
    if (a.c.dtype == EP_BF16)
        front_by_size<OpBf16, EP_BF16>(a, grid, st);
    else if (a.c.dtype == EP_F16)
        front_by_size<OpF16, EP_F16>(a, grid, st);
    else if (a.c.dtype == EP_I8 && q_dtype == EP_BF16)
        front_by_size<OpBf16, EP_I8>(a, grid, st);
    else if (a.c.dtype == EP_I8)
        front_by_size<OpF16, EP_I8>(a, grid, st);
    else if (q_dtype == EP_BF16)
        front_by_size<OpBf16, EP_E4M3>(a, grid, st);
    else
        front_by_size<OpF16, EP_E4M3>(a, grid, st);
}

}  // namespace ep
