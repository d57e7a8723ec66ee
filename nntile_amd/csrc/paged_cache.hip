// Writing new keys and values into the pages of a cache, as they are or in 8 bits, and
// reading rows of it back into dense tiles.
//
// An 8-bit row is e4m3 codes and one power of two 2^k, kept as the byte k + 127: with a the largest
// absolute value of the row, k is the smallest integer from -126 on with a <= 448 * 2^k.
// A power of two costs a floating-point code no precision (all but the subnormal codes
// carry four bits whatever the scale), and the division by it is exact, so a code is one
// rounding of its value, to nearest even, and the value read back is exact in bf16.
//
// Both directions are bound by HBM (long prompts) or by the launch (single tokens).  A
// thread moves 16 bytes of the dense side; the threads of a row are neighbours in a
// wavefront and take its maximum by exchanges.
#include "paged.hpp"

namespace nntile_hip
{

struct PagedMoveParams
{
    PagedView c;
    const char *src[2];     // append: k_new, v_new
    char *dst[2];           // read: k_out, v_out
    int64_t first;          // read: the first row
    int32_t rows;
    int64_t pieces;         // per tensor: entries * rows * pieces of a row
};

// Address of row `pos` of sequence n, head h, in a pool of `row_bytes` a row; null: no page.
// at: the row's place among the scales.
__device__ __forceinline__ char *paged_row(const PagedView &c, char *pages, int n, int h, int pos,
        int row_bytes, int64_t &at)
{
    const int page = c.table[(int64_t)n * c.max_pages + (pos >> c.page_shift)];
    if((unsigned)page >= (unsigned)c.n_pages)
    {
        return nullptr;
    }
    const int64_t in_page = ((int64_t)h << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
    at = page * c.scale_stride + in_page;
    return pages + page * c.page_stride + in_page * row_bytes;
}

// TPR threads a row.
template<int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t x)
{
#pragma unroll
    for(int o = TPR / 2; o >= 1; o >>= 1)
    {
        x = max(x, (uint32_t)__shfl_xor((int)x, o, TPR));
    }
    return x;
}

// T: Bf16 or Fp16 with codes; void: the bytes as they are (row_bytes / 16 threads a row).
template<typename T, int TPR>
__global__ __launch_bounds__(256)
void paged_append_kernel(const PagedMoveParams p)
{
    constexpr bool PACK = !__is_same(T, void);
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if(t >= p.pieces)
    {
        return;         // (whole rows: pieces is a multiple of TPR)
    }
    const int which = blockIdx.y;
    const int64_t row = t / TPR;
    const int piece = (int)(t % TPR);
    const int entry = (int)(row / p.rows);
    const int r = (int)(row - (int64_t)entry * p.rows);
    const int n = entry % p.c.n_batch, h = entry / p.c.n_batch;
    const u32x4 raw = *reinterpret_cast<const u32x4 *>(p.src[which] + t * 16);
    const int given = paged_new(p.c, n, p.rows);
    const int pos = paged_len(p.c, n) - given + r;
    if(r >= given || pos < 0)
    {
        return;
    }
    int64_t at;
    constexpr int row_bytes = PACK ? TPR * 8 : TPR * 16;
    char *to = paged_row(p.c, which ? p.c.v_pages : p.c.k_pages, n, h, pos, row_bytes, at);
    if(to == nullptr)
    {
        return;
    }
    if constexpr(!PACK)
    {
        *reinterpret_cast<u32x4 *>(to + piece * 16) = raw;
    }
    else
    {
        float x[8];
        uint32_t top = 0;
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            x[i] = T::to_float((uint16_t)(raw[i / 2] >> (16 * (i % 2))));
            top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        }
        // (as integers: an infinity is larger than every number, a NaN than an infinity)
        top = row_max<TPR>(top);
        u32x2 codes = {0x7f7f7f7fu, 0x7f7f7f7fu};
        int k = 0;
        if(top < 0x7f800000u)
        {
            // 448 = 1.75 * 2^8
            k = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
            const float scale = __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
            for(int j = 0; j < 2; ++j)
            {
                int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * scale, x[4 * j + 1] * scale, 0, false);
                c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * scale, x[4 * j + 3] * scale, c, true);
                codes[j] = (uint32_t)c;
            }
        }
        *reinterpret_cast<u32x2 *>(to + piece * 8) = codes;
        if(piece == 0)
        {
            (which ? p.c.v_scales : p.c.k_scales)[at] = (uint8_t)(k + 127);
        }
    }
}

template<typename T, int TPR>
__global__ __launch_bounds__(256)
void paged_read_kernel(const PagedMoveParams p)
{
    constexpr bool PACK = !__is_same(T, void);
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if(t >= p.pieces)
    {
        return;
    }
    const int which = blockIdx.y;
    const int64_t row = t / TPR;
    const int piece = (int)(t % TPR);
    const int entry = (int)(row / p.rows);
    const int64_t pos = p.first + (row - (int64_t)entry * p.rows);
    const int n = entry % p.c.n_batch, h = entry / p.c.n_batch;
    u32x4 out = {0, 0, 0, 0};
    if(pos < paged_len(p.c, n))
    {
        int64_t at;
        constexpr int row_bytes = PACK ? TPR * 8 : TPR * 16;
        const char *from = paged_row(p.c, which ? p.c.v_pages : p.c.k_pages, n, h, (int)pos, row_bytes, at);
        if(from != nullptr)
        {
            if constexpr(!PACK)
            {
                out = *reinterpret_cast<const u32x4 *>(from + piece * 16);
            }
            else
            {
                const u32x2 codes = *reinterpret_cast<const u32x2 *>(from + piece * 8);
                const float scale = __uint_as_float(
                        (uint32_t)(which ? p.c.v_scales : p.c.k_scales)[at] << 23);
                float x[8];
#pragma unroll
                for(int j = 0; j < 2; ++j)
                {
                    typedef __attribute__((ext_vector_type(2))) float f32x2;
                    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[j], false);
                    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[j], true);
                    x[4 * j] = lo[0] * scale;
                    x[4 * j + 1] = lo[1] * scale;
                    x[4 * j + 2] = hi[0] * scale;
                    x[4 * j + 3] = hi[1] * scale;
                }
                if constexpr(__is_same(T, Fp16))
                {
                    // 65504 itself has the code of 65536
#pragma unroll
                    for(int i = 0; i < 8; ++i)
                    {
                        x[i] = x[i] > 65504.0f ? 65504.0f : (x[i] < -65504.0f ? -65504.0f : x[i]);
                    }
                }
#pragma unroll
                for(int i = 0; i < 4; ++i)
                {
                    if constexpr(PACK)
                    {
                        out[i] = T::pack2(x[2 * i], x[2 * i + 1]);
                    }
                }
            }
        }
    }
    *reinterpret_cast<u32x4 *>(p.dst[which] + t * 16) = out;
}

template<typename T, int TPR>
static int launch_move(hipStream_t stream, PagedMoveParams &p, bool read)
{
    p.pieces = (int64_t)p.c.n_batch * p.c.n_head_kv * p.rows * TPR;
    const int64_t blocks = (p.pieces + 255) / 256;
    if(blocks > 0x7fffffff)
    {
        return NNTILE_HIP_EINVAL;
    }
    const dim3 grid((unsigned)blocks, 2);
    if(read)
    {
        hipLaunchKernelGGL((paged_read_kernel<T, TPR>), grid, dim3(256), 0, stream, p);
    }
    else
    {
        hipLaunchKernelGGL((paged_append_kernel<T, TPR>), grid, dim3(256), 0, stream, p);
    }
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

static int launch_any(hipStream_t stream, int dtype, PagedMoveParams &p, int head, bool read)
{
    if(p.c.k_scales != nullptr)
    {
        // eight values a thread
        switch(dtype * 2 + (head == 128 ? 1 : 0))
        {
            case 0: return launch_move<Bf16, 8>(stream, p, read);
            case 1: return launch_move<Bf16, 16>(stream, p, read);
            case 2: return launch_move<Fp16, 8>(stream, p, read);
            case 3: return launch_move<Fp16, 16>(stream, p, read);
            default: return NNTILE_HIP_EUNSUPPORTED;
        }
    }
    switch(head * (dtype == 2 ? 4 : 2) / 16)
    {
        case 8: return launch_move<void, 8>(stream, p, read);
        case 16: return launch_move<void, 16>(stream, p, read);
        case 32: return launch_move<void, 32>(stream, p, read);
        default: return NNTILE_HIP_EUNSUPPORTED;
    }
}

int launch_paged_append(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t rows,
        const void *k_new, const void *v_new)
{
    PagedMoveParams p = {};
    p.c = c;
    p.src[0] = static_cast<const char *>(k_new);
    p.src[1] = static_cast<const char *>(v_new);
    p.rows = (int32_t)rows;
    return launch_any(stream, dtype, p, head, false);
}

int launch_paged_read(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t first,
        int64_t rows, void *k_out, void *v_out)
{
    PagedMoveParams p = {};
    p.c = c;
    p.dst[0] = static_cast<char *>(k_out);
    p.dst[1] = static_cast<char *>(v_out);
    p.first = first;
    p.rows = (int32_t)rows;
    return launch_any(stream, dtype, p, head, true);
}

} // namespace nntile_hip
