// Instantiations of the run-time-shaped kernel with the fused epilogue for the
// block-scaled kinds (see kernels_fixed.cuh), in the order of their variant numbers.
#include "kernels_fixed.cuh"

namespace og {

extern const FixedKernel FUSED_SCALED[] = {
    OG_FUSED_KERNEL(8, KIND_MXF8F6F4, 1, 2), OG_FUSED_KERNEL(9, KIND_MXF8F6F4, 2, 2),
    OG_FUSED_KERNEL(10, KIND_MXF4, 1, 2),    OG_FUSED_KERNEL(11, KIND_MXF4, 2, 2),
    OG_FUSED_KERNEL(12, KIND_NVF4, 1, 2),    OG_FUSED_KERNEL(13, KIND_NVF4, 2, 2),
};
extern const int FUSED_SCALED_COUNT = sizeof(FUSED_SCALED) / sizeof(FUSED_SCALED[0]);

}  // namespace og
