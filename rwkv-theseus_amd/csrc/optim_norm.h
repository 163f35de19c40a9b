// The gradients' norm, clip factor and non-finite flag in device memory (optim_adamw.hip), shared
// by the optimizers' steps.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/theseus_optim.h"

namespace optim {

// Adds the tensors' sums of squared gradients (their grad and numel are read) to partial, one double for
// every THESEUS_ADAMW_CHUNK elements, from place `chunks` on, which is moved past them.  Chunks from
// keep_from on are loaded so that they stay cached.
void launch_sumsq(const theseus_adamw_tensor* tensors, int count, long long& chunks, long long keep_from, double* partial,
                  hipStream_t stream);
// result[0 .. 2] as theseus_adamw_step documents them.
void launch_norm(const double* partial, long long chunks, float grad_scale, float max_norm, float* result, hipStream_t stream);

}  // namespace optim
