// Products of bf16 rows with 4-bit weights.
#include "int4_linear_kernels.h"

namespace ikl {

void launch_int4_bf16(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s) {
  launch_group<bf16_tag>(p, group, plan, s);
}

}  // namespace ikl
