// Attention over caches of 4 bits.
#include "cached_attention.h"

namespace taac {

void attend_4(const AttendParams& p, int d, bool f16, int rows, bool alone, uint32_t groups, hipStream_t s) { dispatch_attend<4>(p, d, f16, rows, alone, groups, s); }

}  // namespace taac
