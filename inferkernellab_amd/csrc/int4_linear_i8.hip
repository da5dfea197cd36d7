// Products of rows in 8 bits with 4-bit weights.
#include "int4_linear_kernels.h"

namespace ikl {

void launch_int4_i8(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s) {
  launch_group<i8_tag>(p, group, plan, s);
}

}  // namespace ikl
