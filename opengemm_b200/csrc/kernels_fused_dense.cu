// Instantiations of the run-time-shaped kernel with the fused epilogue for the
// dense float kinds (see kernels_fixed.cuh), in the order of their variant numbers.
#include "kernels_fixed.cuh"

namespace og {

extern const FixedKernel FUSED_DENSE[] = {
    OG_FUSED_KERNEL(0, KIND_F16, 1, 4),     OG_FUSED_KERNEL(1, KIND_F16, 2, 4),
    OG_FUSED_KERNEL(2, KIND_TF32, 1, 4),    OG_FUSED_KERNEL(3, KIND_TF32, 2, 4),
    OG_FUSED_KERNEL(6, KIND_F8F6F4, 1, 4),  OG_FUSED_KERNEL(7, KIND_F8F6F4, 2, 4),
    OG_FUSED_KERNEL(14, KIND_F16, 1, 2),    OG_FUSED_KERNEL(15, KIND_F16, 2, 2),
    OG_FUSED_KERNEL(16, KIND_TF32, 1, 2),   OG_FUSED_KERNEL(17, KIND_TF32, 2, 2),
    OG_FUSED_KERNEL(18, KIND_F8F6F4, 1, 2), OG_FUSED_KERNEL(19, KIND_F8F6F4, 2, 2),
};
extern const int FUSED_DENSE_COUNT = sizeof(FUSED_DENSE) / sizeof(FUSED_DENSE[0]);

}  // namespace og
