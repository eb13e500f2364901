// Attention over 16-bit paged caches (attend_kernel.h).
#include "attend_kernel.h"

namespace ep {

void attend_bf16(const AttendArgs &a, int mt, unsigned grid, hipStream_t st)
{
    attend_by_rows<OpBf16, EP_BF16>(a, mt, grid, st);
}
void attend_f16(const AttendArgs &a, int mt, unsigned grid, hipStream_t st)
{
    attend_by_rows<OpF16, EP_F16>(a, mt, grid, st);
}

}  // namespace ep
