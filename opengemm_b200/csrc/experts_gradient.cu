// The gradients of products of 16-bit operands, of experts and of plain ones (experts.cuh).
#include "experts_launch.h"

namespace og {

extern const ExpertKernel EXPERT_GRADIENT[] = {
    OG_EXPERT_KERNEL(KIND_F16, 1, MODE_DX, 0, 0, 2), OG_EXPERT_KERNEL(KIND_F16, 2, MODE_DX, 0, 0, 2),
    OG_EXPERT_KERNEL(KIND_F16, 1, MODE_DX, 0, 0, 4), OG_EXPERT_KERNEL(KIND_F16, 2, MODE_DX, 0, 0, 4),
    OG_EXPERT_KERNEL(KIND_F16, 1, MODE_DW, 0, 0, 2), OG_EXPERT_KERNEL(KIND_F16, 2, MODE_DW, 0, 0, 2),
    OG_EXPERT_KERNEL(KIND_F16, 1, MODE_DW, 0, 0, 4), OG_EXPERT_KERNEL(KIND_F16, 2, MODE_DW, 0, 0, 4),
};
extern const int EXPERT_GRADIENT_COUNT = sizeof(EXPERT_GRADIENT) / sizeof(EXPERT_GRADIENT[0]);

}  // namespace og
