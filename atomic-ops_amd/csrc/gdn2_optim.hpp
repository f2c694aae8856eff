// Launches of gdn2_optim.hip; arguments as include/gdn2.h's, checked.
#pragma once
#include "../../include/gdn2.h"
#include "gdn2_kernels.hpp"

namespace gdn2 {
size_t adamw_workspace_bytes(const gdn2_adamw_tensor* t, int n);
hipError_t launch_adamw(const gdn2_adamw_tensor* t, int n, int bits, double max_norm, float* norm, void* workspace, hipStream_t s);
hipError_t launch_adamw_unpack(const gdn2_adamw_tensor* t, int n, float* const* m_out, float* const* v_out, hipStream_t s);
}  // namespace gdn2
