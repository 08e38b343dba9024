// What the operators of include/dgnn_ops.h share: the launch descriptions that ops.cpp fills and the kernel files launch from.
#pragma once

#include "../../include/dgnn_ops.h"

#include <hip/hip_runtime.h>

namespace dgnn {
namespace ops {

// Launches `kernel` and returns what the launch itself said (hipGetLastError would also return, and clear, what others left there).
// `shared`: bytes of LDS beyond what the kernel declares; both together kMaxShared at most (each caller asserts its own bound).
constexpr size_t kMaxShared = 160 * 1024;
template <typename... Params>
hipError_t launch_as(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared, hipStream_t stream, Params... args)
{
    void* pointers[] = {const_cast<void*>(static_cast<const void*>(&args))...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, pointers, shared, stream);
}
template <typename... Params, typename... Args>
hipError_t launch_shared(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared, hipStream_t stream, Args... args)
{
    return launch_as<Params...>(kernel, grid, block, shared, stream, args...);
}
template <typename... Params, typename... Args>
hipError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, hipStream_t stream, Args... args)
{
    return launch_as<Params...>(kernel, grid, block, 0, stream, args...);
}

// A grid dimension times the workgroup's has to stay below 2^32; kernels loop over what a capped grid leaves.
constexpr int64_t kMaxGrid = 1 << 20;

// How far a vector of `width` channels from channel c on reaches beyond the last of them.  (c + width may be more than 32 bits hold.)
__host__ __device__ constexpr int overhang(int c, int width, int channels) { return c > channels - width ? c - (channels - width) : 0; }

int64_t dense_workspace(const dgnn_dense_args& a);
hipError_t launch_dense(const dgnn_dense_args& a, hipStream_t stream);
int64_t group_norm_workspace(const dgnn_group_norm_args& a);
hipError_t launch_group_norm(const dgnn_group_norm_args& a, hipStream_t stream);
hipError_t launch_adjust_logits(const dgnn_logits_args& a, hipStream_t stream);

}  // namespace ops
}  // namespace dgnn
