// Rotary embedding, forward and backward, with angles that follow from positions of one
// or several axes (time, rows, columns):
//
//   angle[i] = positions[axes[i]] * freqs[i],  i = 0 .. head/2 - 1
//
// and the pair (2i, 2i+1) of every head of the token is turned by it (rope_common.hpp).
// The queries and the keys of a layer go through one launch.
//
// The angle is taken in 64 bits and reduced there to less than half a turn: at position
// 100000 its fp32 product would be off by 0.004 radians.  What is left of it, up to one turn,
// loses 2^-25 of a turn in fp32 at most; sine and cosine of it are those of the device
// library (the hardware's own, less exact, took as long).  A thread takes
// four pairs of a token (16 bytes of a 16-bit tensor, 32 of an fp32 one) of HEADS heads and
// computes their sines and cosines once; tokens are numbered through all sequences, whose rows of a
// head lie behind each other.
//
// Bound by HBM where it is large: 4096 tokens of 32 + 8 heads of 128 in bf16, 84 MB, 16.0 us = 5.2 TB/s
// (17.9 with four heads a thread, 24.1 with two: the sines and cosines are a thread's larger part then);
// 8192 tokens 28.4 us = 5.9 TB/s.
#include "fixed_divide.hpp"
#include "paged.hpp"
#include "rope_common.hpp"
#include "wide_grid.hpp"

namespace nntile_hip
{

// Sine and cosine of 2 pi times the broken part of position * freq / (2 pi).
__device__ __forceinline__ void turn_of(int64_t position, double freq, float &s, float &c)
{
    const double turns = (double)position * (freq * 0.15915494309189533577);
    const float half = (float)(2.0 * (turns - rint(turns)));        // in half turns, [-1, 1]
    sincospif(half, &s, &c);
}

__device__ __forceinline__ int64_t position_on(const RopeAxesParams &p, int axis, int64_t at)
{
    return axis >= 0 && axis < p.n_axes ? p.positions[axis * p.pos_axis_stride + at] : 0;
}

// Four pairs a thread; blockIdx.y over groups of HEADS heads.  STREAM: loads that leave the caches alone.
template<typename S, bool BACKWARD, int HEADS, bool STREAM>
__global__ __launch_bounds__(256)
void rope_axes_vec_kernel(const RopeAxesParams p, const FixedDivide per_row, const FixedDivide per_seq)
{
    typedef typename S::storage E;
    constexpr int NV = (int)sizeof(E) / 2;      // 16-byte pieces of four pairs
    const uint32_t tokens = per_seq.by * (uint32_t)p.n_batch;
    const uint32_t t = blockIdx.x * 256u + threadIdx.x;
    const uint32_t token = per_row.quotient(t);
    if(token >= tokens)
    {
        return;
    }
    const int i = 4 * (int)(t - token * per_row.by);
    const uint32_t at = p.pos_batch_stride != 0 ? token : token - per_seq.quotient(token) * per_seq.by;
    const int h0 = (int)blockIdx.y * HEADS;
    const int heads = (int)(p.heads_q + p.heads_k);
    const int64_t of_head = (int64_t)tokens * p.head;
    const int64_t in_head = (int64_t)token * p.head + 2 * i;
    u32x4 raw[HEADS][NV];
#pragma unroll
    for(int j = 0; j < HEADS; ++j)
    {
        // (heads past the last re-read it)
        const int h = min(h0 + j, heads - 1);
        const bool key = h >= p.heads_q;
        const u32x4 *from = reinterpret_cast<const u32x4 *>(static_cast<const E *>(key ? p.k : p.q)
                + (key ? h - p.heads_q : h) * of_head + in_head);
#pragma unroll
        for(int v = 0; v < NV; ++v)
        {
            raw[j][v] = STREAM ? __builtin_nontemporal_load(from + v) : from[v];
        }
    }
    float s[4], c[4];
#pragma unroll
    for(int k = 0; k < 4; ++k)
    {
        turn_of(position_on(p, p.axes[i + k], at), p.freqs[i + k], s[k], c[k]);
    }
#pragma unroll
    for(int j = 0; j < HEADS; ++j)
    {
        __attribute__((aligned(16))) E in[8];
        __attribute__((aligned(16))) E out[8];
#pragma unroll
        for(int v = 0; v < NV; ++v)
        {
            reinterpret_cast<u32x4 *>(in)[v] = raw[j][v];
        }
#pragma unroll
        for(int k = 0; k < 4; ++k)
        {
            float x, y;
            rotate<BACKWARD>(c[k], s[k], S::to_float(in[2 * k]), S::to_float(in[2 * k + 1]), x, y);
            out[2 * k] = S::from_float(x);
            out[2 * k + 1] = S::from_float(y);
        }
        const int h = h0 + j;
        if(h < heads)
        {
            const bool key = h >= p.heads_q;
            E *to = static_cast<E *>(key ? p.k_out : p.q_out) + (key ? h - p.heads_q : h) * of_head + in_head;
#pragma unroll
            for(int v = 0; v < NV; ++v)
            {
                __builtin_nontemporal_store(reinterpret_cast<const u32x4 *>(out)[v],
                        reinterpret_cast<u32x4 *>(to) + v);
            }
        }
    }
}

// One pair a thread: heads that are no multiple of 8, addresses that are not aligned.
template<typename S, bool BACKWARD>
__global__ __launch_bounds__(256)
void rope_axes_pair_kernel(const RopeAxesParams p, int64_t pairs)
{
    typedef typename S::storage E;
    const int64_t t = wide_block() * 256 + threadIdx.x;
    if(t >= pairs)
    {
        return;
    }
    const int64_t half = p.head / 2;
    const int64_t row = t / half;
    const int i = (int)(t - row * half);
    const int64_t entry = row / p.seq;
    const int64_t token = row - entry * p.seq;
    const int64_t n = entry % p.n_batch;
    const int64_t q_entries = p.heads_q * p.n_batch;
    const bool key = entry >= q_entries;
    const int64_t at = (row - (key ? q_entries * p.seq : 0)) * p.head + 2 * i;
    const E *from = static_cast<const E *>(key ? p.k : p.q) + at;
    E *to = static_cast<E *>(key ? p.k_out : p.q_out) + at;
    float s, c, x, y;
    turn_of(position_on(p, p.axes[i], n * p.pos_batch_stride + token), p.freqs[i], s, c);
    rotate<BACKWARD>(c, s, S::to_float(from[0]), S::to_float(from[1]), x, y);
    to[0] = S::from_float(x);
    to[1] = S::from_float(y);
}

template<typename S, bool BACKWARD, int HEADS, bool STREAM>
static int launch_vec(hipStream_t stream, const RopeAxesParams &p, int64_t blocks_x)
{
    const int64_t heads = p.heads_q + p.heads_k;
    hipLaunchKernelGGL((rope_axes_vec_kernel<S, BACKWARD, HEADS, STREAM>),
            dim3((unsigned)blocks_x, (unsigned)((heads + HEADS - 1) / HEADS)), dim3(256), 0, stream, p,
            FixedDivide((uint32_t)(p.head / 8)), FixedDivide((uint32_t)p.seq));
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

template<typename S, bool BACKWARD>
static int launch_typed(hipStream_t stream, const RopeAxesParams &p)
{
    auto aligned = [](const void *x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    constexpr int64_t E = sizeof(typename S::storage);
    const int64_t heads = p.heads_q + p.heads_k;
    // (a thread's number fits 31 bits)
    if(p.head % 8 == 0 && aligned(p.q) && aligned(p.q_out) && aligned(p.k) && aligned(p.k_out)
            && heads <= 2 * 65535 && p.n_batch <= 0x7fffff00 / p.seq / (p.head / 8))
    {
        const int64_t blocks_x = (p.n_batch * p.seq * (p.head / 8) + 255) / 256;
        // Eight heads a thread where that leaves every CU a workgroup, else two (one token of eight
        // sequences 4.7 us, so 3.7; 64 of them 5.6 and 3.8).
        if(blocks_x * ((heads + 7) / 8) < 256)
        {
            return launch_vec<S, BACKWARD, 2, false>(stream, p, blocks_x);
        }
        // Large fp32 tensors: four, past the caches.  (49 MB of 24 heads 10.2 us with eight, 12.2 so;
        // 201 MB 56 and 43: eight streams in and eight out, 4 MB apart.)
        if constexpr(E == 4)
        {
            if(p.n_batch * p.seq * p.head * heads * E * 2 >= 128ll << 20)
            {
                return launch_vec<S, BACKWARD, 4, true>(stream, p, blocks_x);
            }
        }
        return launch_vec<S, BACKWARD, 8, false>(stream, p, blocks_x);
    }
    const int64_t pairs = heads * p.n_batch * p.seq * (p.head / 2), blocks = (pairs + 255) / 256;
    if(blocks > kGridMost)
    {
        return NNTILE_HIP_EINVAL;
    }
    hipLaunchKernelGGL((rope_axes_pair_kernel<S, BACKWARD>), wide_grid(blocks), dim3(256), 0, stream, p, pairs);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

int launch_rope_axes(hipStream_t stream, int dtype, bool backward, const RopeAxesParams &p)
{
    switch(dtype * 2 + (backward ? 1 : 0))
    {
        case 0: return launch_typed<RopeBf16, false>(stream, p);
        case 1: return launch_typed<RopeBf16, true>(stream, p);
        case 2: return launch_typed<RopeFp16, false>(stream, p);
        case 3: return launch_typed<RopeFp16, true>(stream, p);
        case 4: return launch_typed<RopeF32, false>(stream, p);
        case 5: return launch_typed<RopeF32, true>(stream, p);
        default: return NNTILE_HIP_EINVAL;
    }
}

} // namespace nntile_hip
