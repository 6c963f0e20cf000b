// The forward experts' products of 8-bit operands (experts.cuh).
#include "experts_launch.h"

namespace og {

extern const ExpertKernel EXPERT_FORWARD8[] = {
    OG_EXPERT_KERNEL(KIND_F8F6F4, 1, MODE_FORWARD, 0, 0, 2), OG_EXPERT_KERNEL(KIND_F8F6F4, 2, MODE_FORWARD, 0, 0, 2),
    OG_EXPERT_KERNEL(KIND_F8F6F4, 1, MODE_FORWARD, 0, 1, 2), OG_EXPERT_KERNEL(KIND_F8F6F4, 2, MODE_FORWARD, 0, 1, 2),
    OG_EXPERT_KERNEL(KIND_F8F6F4, 1, MODE_FORWARD, 1, 0, 2), OG_EXPERT_KERNEL(KIND_F8F6F4, 1, MODE_FORWARD, 1, 1, 2),
};
extern const int EXPERT_FORWARD8_COUNT = sizeof(EXPERT_FORWARD8) / sizeof(EXPERT_FORWARD8[0]);

}  // namespace og
