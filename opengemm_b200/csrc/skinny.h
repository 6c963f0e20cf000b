// The fused product of a few rows without matrix instructions (skinny.cu).
#pragma once

#include "launch_common.h"

namespace og {

constexpr int SKINNY_MAX_M = 4;

// Whether a fused launch goes there; its pointers have passed check_pointers.
bool skinny_serves(const OgGemm& g, const Format& f, const LaunchPointers& io);
cudaError_t launch_skinny(const OgGemm& g, const Format& f, const LaunchPointers& io, const float* alpha, bool pdl, int sm_count, cudaStream_t stream);

}  // namespace og
