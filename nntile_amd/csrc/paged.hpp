// What the kernels on a paged key/value cache share.
#pragma once

#include "fixed_divide.hpp"
#include "sdpa_common.hpp"

namespace nntile_hip
{

// nntile_hip_paged_cache as the kernels take it.  Strides in bytes.
struct PagedView
{
    char *k_pages, *v_pages;
    uint8_t *k_scales, *v_scales;       // null: the pages hold the tile type
    const int32_t *table, *lens, *new_rows;
    int64_t page_stride, scale_stride;
    int32_t n_batch, n_head_kv, n_pages, max_pages;
    int32_t page_shift;                 // log2 of the rows of a page
    int32_t max_rows;                   // max_pages * rows of a page
};

// Rows of a sequence, whatever stands in lens.
__device__ __forceinline__ int paged_len(const PagedView &c, int n)
{
    return min(max(c.lens[n], 0), c.max_rows);
}

// New tokens of a sequence, of `rows` in the call.
__device__ __forceinline__ int paged_new(const PagedView &c, int n, int rows)
{
    return c.new_rows == nullptr ? rows : min(max(c.new_rows[n], 0), rows);
}

struct PagedAttendParams
{
    PagedView c;
    const void *Q;
    float *lse;
    void *A;
    int32_t q_seq, kv_group, rows;      // rows = kv_group * q_seq, of a key/value head
    int32_t causal, overwrite;
    float scale;                        // 1/sqrt(head)
    int32_t row_groups;                 // of as many rows as a workgroup takes
    int32_t units;                      // n_head_kv * row_groups, of a sequence
    int32_t shares;                     // workgroups that the key blocks are shared out to
    unsigned long long *counts;         // workspace: of a shared unit's shares that are done
    float *part_o;                      // workspace: [share][2][rows of a workgroup][head]
    float *part_ml;                     // workspace: [share][2][rows of a workgroup][2]
};

struct PagedWeightsParams
{
    PagedView c;                        // (the values are not read)
    const void *Q;
    const float *lse;
    float *weights;                     // [entry][columns]
    int64_t columns;
    int32_t q_seq, kv_group, rows;      // rows = kv_group * q_seq, of a key/value head
    int32_t causal;
    float decay;
    float scale;                        // 1/sqrt(head)
    int32_t shares;                     // workgroups
    FixedDivide by_seq;                 // by q_seq
};

struct PagedEvictParams
{
    PagedView c;
    const float *weights;               // [entry][columns]
    float *weights_out;                 // may be the same
    int32_t *kept;                      // [entry][keep]
    int64_t columns;
    int32_t keep, recent;
};

struct RopeAxesParams
{
    int64_t head, seq, n_batch, heads_q, heads_k;
    int64_t pos_batch_stride, pos_axis_stride;
    int32_t n_axes;
    const int64_t *positions;
    const double *freqs;
    const int32_t *axes;
    const void *q, *k;
    void *q_out, *k_out;
};

// dtype: 0 bf16, 1 fp16, 2 fp32
int launch_paged_append(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t rows,
        const void *k_new, const void *v_new);
int launch_paged_read(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t first,
        int64_t rows, void *k_out, void *v_out);
int launch_paged_attend(hipStream_t stream, int dtype, PagedAttendParams &p, int head,
        void *workspace);
// Pages of 4-bit codes
int launch_paged4_append(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t rows,
        const void *k_new, const void *v_new);
int launch_paged4_read(hipStream_t stream, int dtype, const PagedView &c, int head, int64_t first,
        int64_t rows, void *k_out, void *v_out);
int launch_paged4_attend(hipStream_t stream, int dtype, PagedAttendParams &p, int head, void *workspace);
// bits: of a page's values, 4, 8 or those of the tile type
int launch_paged_weights(hipStream_t stream, int dtype, int bits, PagedWeightsParams &p, int head);
int launch_paged_evict(hipStream_t stream, int bits, const PagedEvictParams &p, int head);
// Bytes of workspace for `rows` = kv_group * q_seq query rows of a key/value head.
size_t paged_attend_workspace_bytes(int64_t rows, int64_t head);
int launch_rope_axes(hipStream_t stream, int dtype, bool backward, const RopeAxesParams &p);

} // namespace nntile_hip
