// The norms around a residual add for bf16 elements.
#include "cascmm_gated_launch.h"

namespace cascmm {
CASCMM_GATED_OF(, CASCMM_DT_BF16)
}  // namespace cascmm
