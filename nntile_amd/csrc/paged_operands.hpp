// Loads, matrix instructions and operands that the attention over pages and what reads its keys share.
#pragma once

#include "paged.hpp"

namespace nntile_hip
{

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

// What the pages hold: 16-bit values, 8-bit codes, 4-bit codes, fp32 values
enum PagedKind { kPaged16, kPaged8, kPaged32, kPaged4 };

// Share w of `all` blocks: [begin(w), begin(w + 1)); the share that has a block.
struct PagedSplit
{
    uint32_t base, rest;    // the first `rest` shares take one block more
    __device__ __forceinline__ PagedSplit(uint32_t all, uint32_t shares)
        : base(shares != 0 ? all / shares : 0), rest(shares != 0 ? all % shares : 0) {}
    __device__ __forceinline__ uint32_t begin(uint32_t w) const { return w * base + min(w, rest); }
    __device__ __forceinline__ uint32_t of(uint32_t block) const
    {
        const uint32_t longer = rest * (base + 1);
        return block < longer ? block / (base + 1) : rest + (block - longer) / base;
    }
};

// A load that is the same for the whole wavefront, through the scalar cache.
template<typename W>
__device__ __forceinline__ W scalar_load(const void *base, int64_t byte)
{
    typedef const __attribute__((address_space(4))) W *ptr;
    return *reinterpret_cast<ptr>(reinterpret_cast<uintptr_t>(base) + byte);
}

// x, of which the compiler knows nothing: what follows from it is not worked out in front of a loop, to be kept
// there in registers that the loop has other use for
__device__ __forceinline__ int fresh(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ int uniform(int x)
{
    return __builtin_amdgcn_readfirstlane(x);
}

// Sums over the wavefront's lanes up to this one, by moves between the vector unit's lanes (through LDS each of the six
// steps waits for a round trip).
__device__ __forceinline__ uint32_t wave_scan(uint32_t x)
{
    // one, two, four and eight lanes up in each row of 16, then the last lane of a row to the rows behind it
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
    return x;
}

template<int N> __device__ __forceinline__ void paged_wait_loads()
{
    static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ void paged_wait_lds()
{
    // lgkmcnt(0)
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
    asm volatile("" ::: "memory");
}

// Over the four lanes that share a query row: lane, lane ^ 16, lane ^ 32, lane ^ 48.
__device__ __forceinline__ float quad_max(float x)
{
    typedef __attribute__((ext_vector_type(2))) uint32_t pair;
    const uint32_t u = __float_as_uint(x);
    const pair r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return max_across_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

__device__ __forceinline__ float quad_sum(float x)
{
    typedef __attribute__((ext_vector_type(2))) uint32_t pair;
    const uint32_t u = __float_as_uint(x);
    const pair r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return sum_across_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// exponent of a scale byte
__device__ __forceinline__ float scale_of(uint32_t bytes, int i)
{
    return __uint_as_float(((bytes >> (8 * i)) & 255u) << 23);
}

// Matrix instructions and operands of the three kinds.
template<typename T> __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr(__is_same(T, Bf16))
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    else
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

template<typename T> __device__ __forceinline__ f32x4 mfma16(u32x2 a, u32x2 b, f32x4 c)
{
    if constexpr(__is_same(T, Bf16))
    {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    }
    else
    {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
    }
}

// Four e4m3 codes times a power of two as four values of T
template<typename T> __device__ __forceinline__ u32x2 widen4(uint32_t codes, float scale)
{
    if constexpr(__is_same(T, Bf16))
    {
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
    }
    else
    {
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false)),
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true))};
    }
}

// Eight e2m1 codes times a power of two as eight values of T (a scale with the exponent of NaN: all NaN)
template<typename T> __device__ __forceinline__ u32x4 widen8_of_4(uint32_t codes, float scale)
{
    u32x4 w;
    if constexpr(__is_same(T, Bf16))
    {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    }
    else
    {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3));
    }
    return w;
}

// Two bf16 numbers, not below 0, at most 1 and taken down by 127 << 7, times 2^byte each (what falls below the
// smallest number becomes 0): the exponents are integers above the seven bits of the mantissa.
__device__ __forceinline__ uint32_t add_exponents(uint32_t lowered, uint32_t two_bytes)
{
    typedef __attribute__((ext_vector_type(2))) int16_t i16x2;
    uint32_t sum;
    asm("v_pk_mad_u16 %0, %1, %2, %3" : "=v"(sum) : "v"(two_bytes), "s"(0x00800080u), "v"(lowered));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(i16x2, sum), i16x2{0, 0}));
}

// ... and down by 127 << 7
__device__ __forceinline__ uint32_t lower_exponents(uint32_t x)
{
    typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, x) - (uint16_t)(127 << 7));
}

// Eight fp16 values as sums of two bf16 numbers: the first 8 bits, and what they leave, exactly.
__device__ __forceinline__ void two_bf16(const u32x4 &x, u32x4 &first, u32x4 &rest)
{
    u32x4 head, tail;
#pragma unroll
    for(int e = 0; e < 4; ++e)
    {
        const float a = Fp16::to_float((uint16_t)(x[e] & 0xffffu)), b = Fp16::to_float((uint16_t)(x[e] >> 16));
        const uint32_t a1 = __float_as_uint(a) & 0xffff0000u, b1 = __float_as_uint(b) & 0xffff0000u;
        // (an infinity leaves nothing)
        const float a2 = (a1 & 0x7f800000u) == 0x7f800000u ? 0.0f : a - __uint_as_float(a1);
        const float b2 = (b1 & 0x7f800000u) == 0x7f800000u ? 0.0f : b - __uint_as_float(b1);
        head[e] = a1 >> 16 | b1;
        tail[e] = __float_as_uint(a2) >> 16 | (__float_as_uint(b2) & 0xffff0000u);
    }
    first = head;
    rest = tail;
}

} // namespace nntile_hip
