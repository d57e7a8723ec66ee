// Division by a number that is fixed for a launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nntile_hip
{

// Quotients of numbers below 2^31 by a fixed divisor: a multiplication by
// 2^32 (2^shift - by) / by + 1, rounded down, an addition and a shift, exact
// for every such number (Granlund and Montgomery 1994, theorem 4.2 with N = 32).
struct FixedDivide
{
    uint32_t by, factor, shift;
    explicit FixedDivide(uint32_t d) : by(d), factor(0), shift(0)
    {
        while((1ull << shift) < d)
        {
            ++shift;
        }
        factor = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t t) const
    {
        return (__umulhi(t, factor) + t) >> shift;
    }
};

} // namespace nntile_hip
