// Attention over the tables' common pages, many rows, and those behind them (attend_front.h).
#include "attend_front.h"

namespace ep {

void attend_front_tails(const FrontTails &a, int q_dtype, unsigned grid, hipStream_t st)
{
    if (a.front.c.dtype == EP_BF16)
        front_tails_by_size<OpBf16, EP_BF16>(a, grid, st);
    else if (a.front.c.dtype == EP_F16)
        front_tails_by_size<OpF16, EP_F16>(a, grid, st);
    else if (a.front.c.dtype == EP_I8 && q_dtype == EP_BF16)
        front_tails_by_size<OpBf16, EP_I8>(a, grid, st);
    else if (a.front.c.dtype == EP_I8)
        front_tails_by_size<OpF16, EP_I8>(a, grid, st);
    else if (q_dtype == EP_BF16)
        front_tails_by_size<OpBf16, EP_E4M3>(a, grid, st);
    else
        front_tails_by_size<OpF16, EP_E4M3>(a, grid, st);
}

}  // namespace ep
