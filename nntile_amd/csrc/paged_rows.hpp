// Rows between dense tiles and the pages of a cache: what the kernels that move them share.
#pragma once

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

// The place of row `pos` of head h among the rows of its page
__device__ __forceinline__ int64_t row_in_page(const PagedView &c, int h, int pos)
{
    return ((int64_t)h << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}

// Address of row `pos` of sequence n, head h, in `page`; at: the row's place among the scales.
__device__ __forceinline__ char *paged_row(const PagedView &c, char *pages, int page, int h, int pos,
        int row_bytes, int64_t &at)
{
    const int64_t in_page = row_in_page(c, h, pos);
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

template<bool STREAM, typename W>
__device__ __forceinline__ W load_piece(const W *from)
{
    if constexpr(STREAM)
    {
        return __builtin_nontemporal_load(from);
    }
    return *from;
}

// Workgroups of 256 threads that a direction of a launch takes: it has less than 2^32 threads
constexpr int64_t kMoveBlocks = (1 << 24) - 1;

} // namespace nntile_hip
