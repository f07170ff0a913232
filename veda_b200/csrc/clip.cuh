// The global-norm clip factor shared by the optimiser kernels (src/libs/optim/Clip.cpp:35-60).
#pragma once

#include "common.cuh"

namespace veda::cuda
{

// total = sqrt(sumsq) * grad_scale: the norm of the gradient after the grad_scale factor (the
// 1/world average of data-parallel training) has been applied.
__device__ __forceinline__ float clip_scale(const double* sumsq, float max_norm,
                                            float grad_scale = 1.0f)
{
    if (sumsq == nullptr)
    {
        return 1.0f;
    }
    double total = sqrt(*sumsq);
    if (grad_scale != 1.0f)
    {
        total *= fabs(static_cast<double>(grad_scale));
    }
    if (!isfinite(total) || total <= static_cast<double>(max_norm))
    {
        return 1.0f;
    }
    return static_cast<float>(static_cast<double>(max_norm) / total);
}

// Whether VEDA_ADAMW_SKIP_NONFINITE drops the step.
__device__ __forceinline__ bool skipped_step(int flags, const double* sumsq, float grad_scale)
{
    return (flags & 2) && sumsq != nullptr &&
           !isfinite(static_cast<float>(sqrt(*sumsq) * fabs(static_cast<double>(grad_scale))));
}

} // namespace veda::cuda
