// The forward experts' products of 16-bit operands (experts.cuh).
#include "experts_launch.h"

namespace og {

extern const ExpertKernel EXPERT_FORWARD16[] = {
    OG_EXPERT_KERNEL(KIND_F16, 1, MODE_FORWARD, 0, 0, 2), OG_EXPERT_KERNEL(KIND_F16, 2, MODE_FORWARD, 0, 0, 2),
    OG_EXPERT_KERNEL(KIND_F16, 1, MODE_FORWARD, 0, 1, 2), OG_EXPERT_KERNEL(KIND_F16, 2, MODE_FORWARD, 0, 1, 2),
    OG_EXPERT_KERNEL(KIND_F16, 1, MODE_FORWARD, 1, 0, 2), OG_EXPERT_KERNEL(KIND_F16, 1, MODE_FORWARD, 1, 1, 2),
};
extern const int EXPERT_FORWARD16_COUNT = sizeof(EXPERT_FORWARD16) / sizeof(EXPERT_FORWARD16[0]);

}  // namespace og
