// Products of fp16 rows with 4-bit weights.
#include "int4_linear_kernels.h"

namespace ikl {

void launch_int4_f16(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s) {
  launch_group<f16_tag>(p, group, plan, s);
}

}  // namespace ikl
