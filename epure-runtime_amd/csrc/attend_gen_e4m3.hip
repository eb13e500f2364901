// Attention over e4m3 paged caches (attend_kernel.h).
#include "attend_kernel.h"

namespace ep {

void attend_e4m3(const AttendWhole &a, int q_dtype, int mt, unsigned grid, hipStream_t st)
{
    if (q_dtype == EP_BF16)
        attend_by_rows<OpBf16, EP_E4M3>(a, mt, grid, st);
    else
        attend_by_rows<OpF16, EP_E4M3>(a, mt, grid, st);
}

}  // namespace ep
