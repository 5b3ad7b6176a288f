// The norms around a residual add for f32 elements.
#include "cascmm_gated_launch.h"

namespace cascmm {
CASCMM_GATED_OF(, CASCMM_DT_F32)
}  // namespace cascmm
