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
// thread moves 16 bytes of the dense side of a row, or of a few rows at once; the threads of
// a row are neighbours in a wavefront and take its maximum by exchanges.  Lengths, table and pages are
// three loads that depend on each other, which is what more rows a thread hide.  Stores are non-temporal
// (4 x 4096 rows of 16 bits 26.8 us without, 20.9 with).  What they reach: 8 x 8192 rows of 8 bits to
// 16 bits, 403 MB, 72 us = 5.6 TB/s; 4 x 4096 rows of 16 bits appended, 134 MB, 20.9 us = 6.4 TB/s.
#include "fixed_divide.hpp"
#include "paged.hpp"

namespace nntile_hip
{

struct PagedMoveParams
{
    PagedView c;
    const char *src[2];     // append: k_new, v_new
    char *dst[2];           // read: k_out, v_out
    int32_t first;          // read: the first row
    int32_t rows;
    uint32_t all_rows;      // entries * rows, of each tensor
    FixedDivide by_rows, by_batch;
};

// Row `row` of a dense tile [entries][rows]: its sequence, head and place among the rows.
__device__ __forceinline__ void dense_row(const PagedMoveParams &p, uint32_t row, int &n, int &h, int &r)
{
    const uint32_t entry = p.by_rows.quotient(row);
    r = (int)(row - entry * p.by_rows.by);
    h = (int)p.by_batch.quotient(entry);
    n = (int)(entry - (uint32_t)h * p.by_batch.by);
}

// Address of row `pos` of sequence n, head h, in `page`; at: the row's place among the scales.
__device__ __forceinline__ char *paged_row(const PagedView &c, char *pages, int page, int h, int pos,
        int row_bytes, int64_t &at)
{
    const int64_t in_page = ((int64_t)h << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
    at = page * c.scale_stride + in_page;
    return pages + page * c.page_stride + in_page * row_bytes;
}

// The page of row `pos` of sequence n, or -1
__device__ __forceinline__ int page_of(const PagedView &c, int n, int pos)
{
    const int page = c.table[(int64_t)n * c.max_pages + (pos >> c.page_shift)];
    return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}

// The larger of each half, as unsigned 16-bit integers.
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b)
{
    typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                __builtin_bit_cast(u16x2, b)));
}

// Over the TPR threads of a row, each half on its own.
template<int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t x)
{
#pragma unroll
    for(int o = TPR / 2; o >= 1; o >>= 1)
    {
        x = max_halves(x, (uint32_t)__shfl_xor((int)x, o, TPR));
    }
    return x;
}

// Two values of T divided by a power of two, as codes of one half of a word, to nearest even.
template<typename T, bool HIGH>
__device__ __forceinline__ uint32_t narrow2(uint32_t word, uint32_t x, float scale)
{
    typedef __attribute__((ext_vector_type(2))) short s16x2;
    const s16x2 old = __builtin_bit_cast(s16x2, word);
    if constexpr(__is_same(T, Fp16))
    {
        typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
        return __builtin_bit_cast(uint32_t,
                __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, __builtin_bit_cast(f16x2, x), scale, HIGH));
    }
    else
    {
        typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
        return __builtin_bit_cast(uint32_t,
                __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, __builtin_bit_cast(bf16x2, x), scale, HIGH));
    }
}

// T: Bf16 or Fp16 with codes; void: the bytes as they are (row_bytes / 16 threads a row).  A thread
// takes its 16 bytes of LINES rows, 256 / TPR rows apart.  AT_ONCE: all of them are on their way beside the
// lengths, also those that turn out not to be new.
template<typename T, int TPR, int LINES, bool AT_ONCE>
__global__ __launch_bounds__(256)
void paged_append_kernel(const PagedMoveParams p)
{
    constexpr bool PACK = !__is_same(T, void);
    constexpr int row_bytes = PACK ? TPR * 8 : TPR * 16;
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
        const u32x4 *const from = reinterpret_cast<const u32x4 *>(p.src[which] + (int64_t)row * (TPR * 16)) + piece;
        if constexpr(AT_ONCE)
        {
            raw[k] = *from;
        }
        int r;
        dense_row(p, row, n[k], h[k], r);
        const int given = paged_new(p.c, n[k], p.rows);
        pos[k] = paged_len(p.c, n[k]) - given + r;
        if(r >= given || row0 + k * (256u / TPR) >= p.all_rows)
        {
            pos[k] = -1;
        }
        if constexpr(!AT_ONCE)
        {
            raw[k] = pos[k] >= 0 ? *from : u32x4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        page[k] = pos[k] >= 0 ? page_of(p.c, n[k], pos[k]) : -1;
    }
    // Largest sizes, as integers: an infinity is larger than every number, a NaN than an infinity.  Two rows
    // share a word.
    uint32_t top[LINES];
    if constexpr(PACK)
    {
#pragma unroll
        for(int k = 0; k < LINES; ++k)
        {
            uint32_t x = 0;
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                x = max_halves(x, raw[k][i] & 0x7fff7fffu);
            }
            top[k] = max(x & 0xffffu, x >> 16);
        }
        if constexpr(LINES == 2)
        {
            const uint32_t both = row_max<TPR>(top[0] | top[1] << 16);
            top[0] = both & 0xffffu;
            top[1] = both >> 16;
        }
        else
        {
            static_assert(LINES == 1, "one or two rows a thread");
            top[0] = row_max<TPR>(top[0]);
        }
    }
#pragma unroll
    for(int k = 0; k < LINES; ++k)
    {
        if(page[k] < 0)
        {
            continue;       // (the same for all threads of the row)
        }
        int64_t at;
        char *to = paged_row(p.c, which ? p.c.v_pages : p.c.k_pages, page[k], h[k], pos[k], row_bytes, at);
        if constexpr(!PACK)
        {
            __builtin_nontemporal_store(raw[k], reinterpret_cast<u32x4 *>(to + piece * 16));
        }
        else
        {
            u32x2 codes = {0x7f7f7f7fu, 0x7f7f7f7fu};
            int e = 0;
            const uint32_t bits = __float_as_uint(T::to_float((uint16_t)top[k]));
            if(bits < 0x7f800000u)
            {
                // 448 = 1.75 * 2^8
                e = max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
                const float scale = __uint_as_float((uint32_t)(127 + e) << 23);
                codes[0] = narrow2<T, true>(narrow2<T, false>(0u, raw[k][0], scale), raw[k][1], scale);
                codes[1] = narrow2<T, true>(narrow2<T, false>(0u, raw[k][2], scale), raw[k][3], scale);
            }
            __builtin_nontemporal_store(codes, reinterpret_cast<u32x2 *>(to + piece * 8));
            if(piece == 0)
            {
                (which ? p.c.v_scales : p.c.k_scales)[at] = (uint8_t)(e + 127);
            }
        }
    }
}

template<bool STREAM, typename W>
__device__ __forceinline__ W load_piece(const W *from)
{
    if constexpr(STREAM)
    {
        return __builtin_nontemporal_load(from);
    }
    return *from;
}

template<typename T, int TPR, int LINES, bool STREAM>
__global__ __launch_bounds__(256)
void paged_read_kernel(const PagedMoveParams p)
{
    constexpr bool PACK = !__is_same(T, void);
    constexpr int row_bytes = PACK ? TPR * 8 : TPR * 16;
    const int which = blockIdx.y;
    const int piece = (int)(threadIdx.x % TPR);
    const uint32_t row0 = blockIdx.x * (uint32_t)(LINES * 256 / TPR) + threadIdx.x / TPR;
    int n[LINES], h[LINES], pos[LINES], page[LINES];
    u32x4 raw[LINES];
    uint32_t byte[LINES];
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
        raw[k] = u32x4{0, 0, 0, 0};
        byte[k] = 0;
        if(page[k] >= 0)
        {
            int64_t at;
            const char *from = paged_row(p.c, which ? p.c.v_pages : p.c.k_pages, page[k], h[k], pos[k],
                    row_bytes, at);
            if constexpr(PACK)
            {
                const u32x2 codes = load_piece<STREAM>(reinterpret_cast<const u32x2 *>(from) + piece);
                raw[k][0] = codes[0];
                raw[k][1] = codes[1];
                byte[k] = (which ? p.c.v_scales : p.c.k_scales)[at];
            }
            else
            {
                raw[k] = load_piece<STREAM>(reinterpret_cast<const u32x4 *>(from) + piece);
            }
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
        u32x4 out = raw[k];
        if constexpr(PACK)
        {
            const float scale = __uint_as_float(byte[k] << 23);
            float x[8];
#pragma unroll
            for(int j = 0; j < 2; ++j)
            {
                typedef __attribute__((ext_vector_type(2))) float f32x2;
                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[k][j], false);
                const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[k][j], true);
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
                out[i] = T::pack2(x[2 * i], x[2 * i + 1]);
            }
        }
        __builtin_nontemporal_store(out, reinterpret_cast<u32x4 *>(p.dst[which] + (int64_t)row * (TPR * 16)) + piece);
    }
}

// Workgroups of 256 threads that a direction of a launch takes: it has less than 2^32 threads
constexpr int64_t kMoveBlocks = (1 << 24) - 1;

template<typename T, int TPR, int LINES, bool AT_ONCE>
static int launch_append(hipStream_t stream, const PagedMoveParams &p)
{
    constexpr int64_t ROWS = LINES * 256 / TPR;
    const int64_t blocks = (p.all_rows + ROWS - 1) / ROWS;
    if(blocks > kMoveBlocks)
    {
        return NNTILE_HIP_EINVAL;
    }
    hipLaunchKernelGGL((paged_append_kernel<T, TPR, LINES, AT_ONCE>), dim3((unsigned)blocks, 2), dim3(256), 0, stream, p);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

template<typename T, int TPR, int LINES, bool STREAM>
static int launch_read(hipStream_t stream, const PagedMoveParams &p)
{
    constexpr int64_t ROWS = LINES * 256 / TPR;
    const int64_t blocks = (p.all_rows + ROWS - 1) / ROWS;
    if(blocks > kMoveBlocks)
    {
        return NNTILE_HIP_EINVAL;
    }
    hipLaunchKernelGGL((paged_read_kernel<T, TPR, LINES, STREAM>), dim3((unsigned)blocks, 2), dim3(256), 0, stream, p);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

template<typename T, int TPR>
static int launch_move(hipStream_t stream, const PagedMoveParams &p, bool read)
{
    // Several rows a thread once that leaves every CU eight workgroups, as many as keep 32 bytes of the
    // pages on their way: appending 4 x 8 x 4096 rows in 8 bits 17.2 us with one, 16.6 with two, 17.6 with four;
    // reading 8 x 8192 rows of 8 bits 78.6 with two, 72.1 with four, 8 x 4096 of 16 bits 44.2 and 47.3.
    constexpr int LINES = __is_same(T, void) ? 2 : 4;
    const int64_t bytes = (int64_t)p.all_rows * TPR * 16 * 2;       // of the dense side
    const bool many = bytes >= 16ll * 256 * 256 * 8 * 2;
    if(!read)
    {
        // Rows that are not new are not fetched where there are many (4 x 8 x 4096 rows, of which three fifths are
        // new, 16.5 -> 15.4 us; where all are new, that order costs 18.9 -> 20.0).
        return !many ? launch_append<T, TPR, 1, true>(stream, p)
            : p.c.new_rows == nullptr ? launch_append<T, TPR, 2, true>(stream, p)
            : launch_append<T, TPR, 2, false>(stream, p);
    }
    // What is read stays out of the caches (non-temporal) where it would not stay in the 256 MB of the
    // last level anyway: 34 MB in all 7.2 us, 8.4 non-temporal; 403 MB 78.6 and 72.1.
    return bytes >= 128ll << 20 ? launch_read<T, TPR, LINES, true>(stream, p)
        : many ? launch_read<T, TPR, LINES, false>(stream, p) : launch_read<T, TPR, 1, false>(stream, p);
}

static int launch_any(hipStream_t stream, int dtype, const PagedMoveParams &p, int head, bool read)
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
    const PagedMoveParams p = {c, {static_cast<const char *>(k_new), static_cast<const char *>(v_new)},
        {nullptr, nullptr}, 0, (int32_t)rows, (uint32_t)(rows * c.n_batch * c.n_head_kv),
        FixedDivide((uint32_t)rows), FixedDivide((uint32_t)c.n_batch)};
    return launch_any(stream, dtype, p, head, false);
}

int launch_paged_read(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t first,
        int64_t rows, void *k_out, void *v_out)
{
    const PagedMoveParams p = {c, {nullptr, nullptr}, {static_cast<char *>(k_out), static_cast<char *>(v_out)},
        (int32_t)first, (int32_t)rows, (uint32_t)(rows * c.n_batch * c.n_head_kv),
        FixedDivide((uint32_t)rows), FixedDivide((uint32_t)c.n_batch)};
    return launch_any(stream, dtype, p, head, true);
}

} // namespace nntile_hip
