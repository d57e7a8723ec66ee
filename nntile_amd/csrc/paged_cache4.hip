// Writing new keys and values into pages of 4-bit codes, and reading rows of such pages back into
// dense tiles.
//
// A row is e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two a byte, the lower half first, and one power of
// two 2^k for every 32 values, kept as the byte k + 127: with a the largest absolute value of the 32, k is the
// smallest integer from -125 to 125 with a <= 7 * 2^k (or 125: what lies above becomes 6 * 2^125).  What lies
// between 6 and 7 rounds to 6, by no more than what lies between 4 and 6 is rounded by; on normal values the codes
// then err by 11.2 % (root mean square), by 11.5 % with the power that leaves nothing above 6 or with that of the
// largest value's exponent.  Every value that a code stands for is a normal, finite number of bf16.  The division
// is exact, so a code is one rounding of its value, to nearest even, and what is read back is exact in bf16.  A
// block with a NaN or an infinity has the byte 255.
//
// Like the moves of 8-bit rows: a thread has 16 bytes of the dense side, eight values, of a row or of a few at
// once; the four threads of a block are neighbours.  Bound by HBM, the dense side's bytes: 4 x 4096 rows, 8 heads of 128,
// 67 MB and 19 MB of pages, appended in 17 us = 5.1 TB/s, read back in 14.9 = 5.8.
#include "paged_rows.hpp"
#include "paged_operands.hpp"

namespace nntile_hip
{

// Two values of T divided by a power of two, as the codes of byte AT of a word, to nearest even
template<typename T, int AT>
__device__ __forceinline__ uint32_t narrow2_to_4(uint32_t word, uint32_t x, float scale)
{
    if constexpr(__is_same(T, Fp16))
    {
        typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(f16x2, x), scale, AT);
    }
    else
    {
        typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(bf16x2, x), scale, AT);
    }
}

template<typename T>
__device__ __forceinline__ uint32_t narrow8_to_4(const u32x4 &x, float scale)
{
    return narrow2_to_4<T, 3>(narrow2_to_4<T, 2>(narrow2_to_4<T, 1>(narrow2_to_4<T, 0>(0u, x[0], scale), x[1], scale),
                x[2], scale), x[3], scale);
}

// TPR threads a row, LINES rows a thread, 256 / TPR rows apart.
template<typename T, int TPR, int LINES>
__global__ __launch_bounds__(256)
void paged4_append_kernel(const PagedMoveParams p)
{
    constexpr int row_bytes = TPR * 4, SB = TPR / 4;
    const int which = blockIdx.y;
    const int piece = (int)(threadIdx.x % TPR);
    const uint32_t row0 = blockIdx.x * (uint32_t)(LINES * 256 / TPR) + threadIdx.x / TPR;
    u32x4 raw[LINES];
    int n[LINES], h[LINES], pos[LINES], page[LINES];
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        // (behind the last row: it again, not written)
        const uint32_t row = min(row0 + k * (256u / TPR), p.all_rows - 1);
        int r;
        dense_row(p, row, n[k], h[k], r);
        const int given = paged_new(p.c, n[k], p.rows);
        pos[k] = paged_len(p.c, n[k]) - given + r;
        if(r >= given || row0 + k * (256u / TPR) >= p.all_rows)
        {
            pos[k] = -1;
        }
        raw[k] = u32x4{0, 0, 0, 0};
        if(pos[k] >= 0)
        {
            raw[k] = *(reinterpret_cast<const u32x4 *>(p.src[which] + (int64_t)row * (TPR * 16)) + piece);
        }
    }
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        page[k] = pos[k] >= 0 ? page_of(p.c, n[k], pos[k]) : -1;
    }
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        // Largest sizes, as integers: an infinity is larger than every number, a NaN than an infinity.
        uint32_t x = 0;
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            x = max_halves(x, raw[k][i] & 0x7fff7fffu);
        }
        const uint32_t top = row_max<4>(max(x & 0xffffu, x >> 16));
        if(page[k] < 0)
        {
            continue;       // (the same for all threads of the row)
        }
        const int64_t at = row_in_page(p.c, h[k], pos[k]);
        uint32_t codes = 0, byte = 255;
        const uint32_t bits = __float_as_uint(T::to_float((uint16_t)top));
        if(bits < 0x7f800000u)
        {
            // 7 = 1.75 * 2^2
            const int e = min(max((int)(bits >> 23) - 127 - 2 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -125), 125);
            byte = (uint32_t)(e + 127);
            codes = narrow8_to_4<T>(raw[k], __uint_as_float(byte << 23));
        }
        char *const to = (which ? p.c.v_pages : p.c.k_pages) + page[k] * p.c.page_stride + at * row_bytes;
        // (codes stay in the caches, for whoever reads the prompt back next: 4 x 4096 rows, 8 heads of 128, read 22.6 us
        // behind non-temporal stores, 14.9 behind these)
        reinterpret_cast<uint32_t *>(to)[piece] = codes;
        if(piece % 4 == 0)
        {
            (which ? p.c.v_scales : p.c.k_scales)[page[k] * p.c.scale_stride + at * SB + piece / 4] = (uint8_t)byte;
        }
    }
}

template<typename T, int TPR, int LINES, bool STREAM>
__global__ __launch_bounds__(256)
void paged4_read_kernel(const PagedMoveParams p)
{
    constexpr int row_bytes = TPR * 4, SB = TPR / 4;
    const int which = blockIdx.y;
    const int piece = (int)(threadIdx.x % TPR);
    const uint32_t row0 = blockIdx.x * (uint32_t)(LINES * 256 / TPR) + threadIdx.x / TPR;
    int n[LINES], h[LINES], pos[LINES], page[LINES];
    uint32_t codes[LINES], byte[LINES];
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        int r;
        dense_row(p, min(row0 + k * (256u / TPR), p.all_rows - 1), n[k], h[k], r);
        pos[k] = p.first + r;
        if(pos[k] >= paged_len(p.c, n[k]))
        {
            pos[k] = -1;
        }
    }
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        page[k] = pos[k] >= 0 ? page_of(p.c, n[k], pos[k]) : -1;
    }
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        codes[k] = 0;
        byte[k] = 127;
        if(page[k] >= 0)
        {
            const int64_t at = row_in_page(p.c, h[k], pos[k]);
            const char *const from = (which ? p.c.v_pages : p.c.k_pages) + page[k] * p.c.page_stride + at * row_bytes;
            codes[k] = load_piece<STREAM>(reinterpret_cast<const uint32_t *>(from) + piece);
            byte[k] = (which ? p.c.v_scales : p.c.k_scales)[page[k] * p.c.scale_stride + at * SB + piece / 4];
        }
    }
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        const uint32_t row = row0 + k * (256u / TPR);
        if(row >= p.all_rows)
        {
            return;
        }
        u32x4 out = widen8_of_4<T>(codes[k], __uint_as_float(byte[k] << 23));
        if constexpr(__is_same(T, Fp16))
        {
            // past the type's range its largest value: 65504 itself has the code of 65536
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                out[i] -= ((out[i] & 0x7fffu) == 0x7c00u ? 1u : 0u) + ((out[i] & 0x7fff0000u) == 0x7c000000u ? 0x10000u : 0u);
            }
        }
        __builtin_nontemporal_store(out, reinterpret_cast<u32x4 *>(p.dst[which] + (int64_t)row * (TPR * 16)) + piece);
    }
}

template<int ROWS>
static int64_t move_blocks(const PagedMoveParams &p)
{
    return ((int64_t)p.all_rows + ROWS - 1) / ROWS;
}

template<typename T, int TPR, int LINES>
static int launch_append(hipStream_t stream, const PagedMoveParams &p)
{
    const int64_t blocks = move_blocks<LINES * 256 / TPR>(p);
    if(blocks > kMoveBlocks)
    {
        return NNTILE_HIP_EINVAL;
    }
    hipLaunchKernelGGL((paged4_append_kernel<T, TPR, LINES>), dim3((unsigned)blocks, 2), dim3(256), 0, stream, p);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

template<typename T, int TPR, int LINES, bool STREAM>
static int launch_read(hipStream_t stream, const PagedMoveParams &p)
{
    const int64_t blocks = move_blocks<LINES * 256 / TPR>(p);
    if(blocks > kMoveBlocks)
    {
        return NNTILE_HIP_EINVAL;
    }
    hipLaunchKernelGGL((paged4_read_kernel<T, TPR, LINES, STREAM>), dim3((unsigned)blocks, 2), dim3(256), 0, stream, p);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

template<typename T, int TPR>
static int launch_move(hipStream_t stream, const PagedMoveParams &p, bool read)
{
    // Several rows a thread, and what is read past the caches, from the sizes on from which that pays for the moves of
    // 8-bit rows (here 4 x 4096 rows, 8 heads of 128, bf16: appended by one row a thread 17.7 us, two 16.9, four 17.6;
    // read by one 16.6, two 15.2, four 14.9, eight 23).
    const int64_t bytes = (int64_t)p.all_rows * TPR * 16 * 2;       // of the dense side
    const bool many = bytes >= 16ll * 256 * 256 * 8 * 2;
    if(!read)
    {
        return many ? launch_append<T, TPR, 2>(stream, p) : launch_append<T, TPR, 1>(stream, p);
    }
    return bytes >= 128ll << 20 ? launch_read<T, TPR, 4, true>(stream, p)
        : many ? launch_read<T, TPR, 4, false>(stream, p) : launch_read<T, TPR, 1, false>(stream, p);
}

static int launch_any(hipStream_t stream, int dtype, const PagedMoveParams &p, int head, bool read)
{
    switch(dtype * 2 + (head == 128 ? 1 : 0))
    {
        case 0: return launch_move<Bf16, 8>(stream, p, read);
        case 1: return launch_move<Bf16, 16>(stream, p, read);
        case 2: return launch_move<Fp16, 8>(stream, p, read);
        case 3: return launch_move<Fp16, 16>(stream, p, read);
        default: return NNTILE_HIP_EUNSUPPORTED;
    }
}

int launch_paged4_append(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t rows,
        const void *k_new, const void *v_new)
{
    const PagedMoveParams p = {c, {static_cast<const char *>(k_new), static_cast<const char *>(v_new)},
        {nullptr, nullptr}, 0, (int32_t)rows, (uint32_t)(rows * c.n_batch * c.n_head_kv),
        FixedDivide((uint32_t)rows), FixedDivide((uint32_t)c.n_batch)};
    return launch_any(stream, dtype, p, head, false);
}

int launch_paged4_read(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t first,
        int64_t rows, void *k_out, void *v_out)
{
    const PagedMoveParams p = {c, {nullptr, nullptr}, {static_cast<char *>(k_out), static_cast<char *>(v_out)},
        (int32_t)first, (int32_t)rows, (uint32_t)(rows * c.n_batch * c.n_head_kv),
        FixedDivide((uint32_t)rows), FixedDivide((uint32_t)c.n_batch)};
    return launch_any(stream, dtype, p, head, true);
}

} // namespace nntile_hip
