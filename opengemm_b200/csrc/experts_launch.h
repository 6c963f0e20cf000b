// The compiled kernels of the experts' products (experts.cuh) and their table.
#pragma once

#include <atomic>

#include "dependent_launch.h"
#include "experts.cuh"

namespace og {

struct ExpertKernel {
  int kind, cta_group, mode, gather, glu, out_bytes;
  cudaError_t (*configure)(int smem_bytes);
  cudaError_t (*launch)(const ExpertParams& params, int grid, int smem_bytes, cudaStream_t stream);
};

template <int KIND, int CTA_GROUP, int MODE, bool GATHER, bool GLU, int OUT_BYTES>
cudaError_t expert_configure(int smem_bytes) {
  return cudaFuncSetAttribute(expert_kernel<KIND, CTA_GROUP, MODE, GATHER, GLU, OUT_BYTES>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
}

template <int KIND, int CTA_GROUP, int MODE, bool GATHER, bool GLU, int OUT_BYTES>
cudaError_t expert_launch(const ExpertParams& params, int grid, int smem_bytes, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid, 1, 1);
  config.blockDim = dim3(xp_threads(MODE), 1, 1);
  config.dynamicSmemBytes = size_t(smem_bytes);
  config.stream = stream;
  cudaLaunchAttribute attrs[2];
  int count = 0;
  if (CTA_GROUP > 1) {
    attrs[count].id = cudaLaunchAttributeClusterDimension;
    attrs[count].val.clusterDim.x = CTA_GROUP;
    attrs[count].val.clusterDim.y = 1;
    attrs[count].val.clusterDim.z = 1;
    ++count;
  }
  attrs[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[count].val.programmaticStreamSerializationAllowed = dependent_launches();
  ++count;
  config.attrs = attrs;
  config.numAttrs = count;
  return cudaLaunchKernelEx(&config, expert_kernel<KIND, CTA_GROUP, MODE, GATHER, GLU, OUT_BYTES>, params);
}

#define OG_EXPERT_KERNEL(KIND, GROUP, MODE, GATHER, GLU, OUT)           \
  ExpertKernel { KIND, GROUP, MODE, GATHER, GLU, OUT,                   \
                 expert_configure<KIND, GROUP, MODE, GATHER, GLU, OUT>, \
                 expert_launch<KIND, GROUP, MODE, GATHER, GLU, OUT> }

}  // namespace og
