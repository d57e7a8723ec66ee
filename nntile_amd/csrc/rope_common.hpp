// Tile types and the rotation of a pair, shared by the rotary kernels.
#pragma once

#include "sdpa_common.hpp"

namespace nntile_hip
{

struct RopeF32
{
    typedef float storage;
    static __device__ __forceinline__ float to_float(float v) { return v; }
    static __device__ __forceinline__ float from_float(float v) { return v; }
};
struct RopeBf16
{
    typedef uint16_t storage;
    static __device__ __forceinline__ float to_float(uint16_t v) { return Bf16::to_float(v); }
    static __device__ __forceinline__ uint16_t from_float(float v) { return Bf16::from_float(v); }
};
struct RopeFp16
{
    typedef uint16_t storage;
    static __device__ __forceinline__ float to_float(uint16_t v) { return Fp16::to_float(v); }
    static __device__ __forceinline__ uint16_t from_float(float v) { return Fp16::from_float(v); }
};

template<bool BACKWARD>
__device__ __forceinline__ void rotate(float c, float s, float a, float b, float &x, float &y)
{
    if(BACKWARD)
    {
        x = fmaf(c, a, s * b);
        y = fmaf(c, b, -(s * a));
    }
    else
    {
        x = fmaf(c, a, -(s * b));
        y = fmaf(s, a, c * b);
    }
}

} // namespace nntile_hip
