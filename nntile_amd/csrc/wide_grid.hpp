// Grids of more workgroups than one direction of a launch takes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nntile_hip
{

// A direction of a launch has less than 2^32 threads; what is past them is not run, without
// an error.  Workgroups of up to 256 threads are numbered through x and z instead.
constexpr int64_t kGridRun = 1 << 23;
constexpr int64_t kGridMost = kGridRun * 65535;

inline dim3 wide_grid(int64_t blocks, unsigned y = 1)
{
    const int64_t x = blocks < kGridRun ? blocks : kGridRun;
    return dim3((unsigned)x, y, (unsigned)((blocks + x - 1) / x));
}

__device__ __forceinline__ int64_t wide_block()
{
    return (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
}

} // namespace nntile_hip
