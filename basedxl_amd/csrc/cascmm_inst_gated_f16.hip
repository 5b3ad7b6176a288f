// The norms around a residual add for f16 elements.
#include "cascmm_gated_launch.h"

namespace cascmm {
CASCMM_GATED_OF(, CASCMM_DT_F16)
}  // namespace cascmm
