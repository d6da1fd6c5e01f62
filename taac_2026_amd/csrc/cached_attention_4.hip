// Attention over caches of 4 bits.
#include "cached_attention.h"

namespace taac {

void attend_4(const AttendParams& p, int d, bool f16, int rows, int waves, uint32_t groups, hipStream_t s) { dispatch_attend<4>(p, d, f16, rows, waves, groups, s); }

}  // namespace taac
