// C ABI of the paged key/value cache, of the weights its rows receive and their eviction, and of the rotary
// embedding with positions of several axes: argument checks and dispatch to the kernels.
#include "paged.hpp"

using namespace nntile_hip;

namespace
{

bool on16(const void *p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

int elem_bytes(int dtype)
{
    return dtype == 2 ? 4 : 2;
}

constexpr int64_t kMost = 0x7fffffff;
// Rows of a sequence that the walks over 4-bit keys, weights and rows that move number with room to the next step
constexpr int64_t kLongest = 1 << 30;

// a * b, or -1 where that is past 2^31 - 1 (both at least 0)
int64_t small_product(int64_t a, int64_t b)
{
    return a < 0 || b < 0 || (b != 0 && a > kMost / b) ? -1 : a * b;
}

// four: pages of 4-bit codes.  values: the call looks at the values, too.
int paged_view(const nntile_hip_paged_cache *c, int dtype, PagedView &v, bool four = false, bool values = true)
{
    if(c == nullptr || c->k_pages == nullptr || (values && c->v_pages == nullptr) || c->table == nullptr
            || c->lens == nullptr || (values && (c->k_scales == nullptr) != (c->v_scales == nullptr))
            || (four && c->k_scales == nullptr)
            || c->head <= 0 || c->page_rows <= 0 || c->n_head_kv <= 0 || c->n_pages <= 0
            || c->max_pages <= 0 || c->n_batch <= 0 || c->n_pages > kMost)
    {
        return NNTILE_HIP_EINVAL;
    }
    if((c->head != 64 && c->head != 128) || c->page_rows < 16 || c->page_rows > 65536
            || (c->page_rows & (c->page_rows - 1)) != 0)
    {
        return NNTILE_HIP_EUNSUPPORTED;
    }
    const bool packed = c->k_scales != nullptr;
    if(packed && dtype == 2)
    {
        return NNTILE_HIP_EUNSUPPORTED;
    }
    const int64_t max_rows = small_product(c->max_pages, c->page_rows);
    const int64_t page_of_heads = small_product(c->page_rows, c->n_head_kv);
    if(max_rows < 0 || page_of_heads < 0 || small_product(c->n_batch, c->n_head_kv) < 0)
    {
        return NNTILE_HIP_EINVAL;
    }
    // half bytes of a value; scale bytes of a page, of 32 values or of a row
    const int64_t e2 = four ? 1 : packed ? 2 : 2 * elem_bytes(dtype);
    const int64_t scales = page_of_heads * (four ? c->head / 32 : 1);
    constexpr int64_t kStride = (int64_t)1 << 55;       // (times the number of pages it stays an address)
    if(c->page_stride < page_of_heads * c->head || c->page_stride > kStride / c->n_pages
            || c->page_stride * e2 % 32 != 0 || !on16(c->k_pages)
            || (values && !on16(c->v_pages)) || (reinterpret_cast<uintptr_t>(c->table) & 3u) != 0
            || (reinterpret_cast<uintptr_t>(c->lens) & 3u) != 0
            || (reinterpret_cast<uintptr_t>(c->new_rows) & 3u) != 0)
    {
        return NNTILE_HIP_EINVAL;
    }
    if(packed && (c->scale_stride < scales || c->scale_stride > kStride / c->n_pages
                || c->scale_stride % 16 != 0 || !on16(c->k_scales) || (values && !on16(c->v_scales))))
    {
        return NNTILE_HIP_EINVAL;
    }
    v.k_pages = static_cast<char *>(c->k_pages);
    v.v_pages = static_cast<char *>(c->v_pages);
    v.k_scales = c->k_scales;
    v.v_scales = c->v_scales;
    v.table = c->table;
    v.lens = c->lens;
    v.new_rows = c->new_rows;
    v.page_stride = c->page_stride * e2 / 2;
    v.scale_stride = packed ? c->scale_stride : 0;
    v.n_batch = (int32_t)c->n_batch;
    v.n_head_kv = (int32_t)c->n_head_kv;
    v.n_pages = (int32_t)c->n_pages;
    v.max_pages = (int32_t)c->max_pages;
    v.page_shift = __builtin_ctzll((unsigned long long)c->page_rows);
    v.max_rows = (int32_t)max_rows;
    return NNTILE_HIP_OK;
}

int append_call(int dtype, bool four, void *stream, const nntile_hip_paged_cache *c, int64_t rows,
        const void *k_new, const void *v_new)
{
    PagedView v;
    const int rc = paged_view(c, dtype, v, four);
    if(rc != NNTILE_HIP_OK)
    {
        return rc;
    }
    if(rows < 0 || small_product(c->n_batch * c->n_head_kv, rows) < 0)
    {
        return NNTILE_HIP_EINVAL;
    }
    if(rows == 0)
    {
        return NNTILE_HIP_OK;
    }
    if(k_new == nullptr || v_new == nullptr || !on16(k_new) || !on16(v_new))
    {
        return NNTILE_HIP_EINVAL;
    }
    return (four ? launch_paged4_append : launch_paged_append)(static_cast<hipStream_t>(stream), dtype, v,
            (int)c->head, rows, k_new, v_new);
}

int read_call(int dtype, bool four, void *stream, const nntile_hip_paged_cache *c, int64_t first, int64_t rows,
        void *k_out, void *v_out)
{
    PagedView v;
    const int rc = paged_view(c, dtype, v, four);
    if(rc != NNTILE_HIP_OK)
    {
        return rc;
    }
    if(rows < 0 || first < 0 || first > kMost - rows
            || small_product(c->n_batch * c->n_head_kv, rows) < 0)
    {
        return NNTILE_HIP_EINVAL;
    }
    if(rows == 0)
    {
        return NNTILE_HIP_OK;
    }
    if(k_out == nullptr || v_out == nullptr || !on16(k_out) || !on16(v_out))
    {
        return NNTILE_HIP_EINVAL;
    }
    return (four ? launch_paged4_read : launch_paged_read)(static_cast<hipStream_t>(stream), dtype, v, (int)c->head,
            first, rows, k_out, v_out);
}

// kv_group * q_seq, or -1
int64_t query_rows(const nntile_hip_paged_cache &c, int64_t q_seq, int64_t kv_group)
{
    if(q_seq <= 0 || kv_group <= 0 || c.n_batch <= 0 || c.n_head_kv <= 0)
    {
        return -1;
    }
    const int64_t rows = small_product(q_seq, kv_group);
    const int64_t entries = small_product(c.n_batch, c.n_head_kv);
    return rows < 0 || entries < 0 || small_product(rows, entries) < 0 ? -1 : rows;
}

// What the attention over pages refuses of masks
int mask_check(int32_t mode)
{
    return mode == NNTILE_HIP_MASK_CAUSAL || mode == NNTILE_HIP_MASK_NONE ? NNTILE_HIP_OK
        : mode == NNTILE_HIP_MASK_ADDITIVE || mode == NNTILE_HIP_MASK_BOOL ? NNTILE_HIP_EUNSUPPORTED
        : NNTILE_HIP_EINVAL;
}

int attend_call(int dtype, bool four, void *stream, const nntile_hip_sdpa_paged_args *a, void *workspace,
        size_t workspace_bytes)
{
    if(a == nullptr)
    {
        return NNTILE_HIP_EINVAL;
    }
    PagedAttendParams p = {};
    const int rc = paged_view(&a->cache, dtype, p.c, four);
    if(rc != NNTILE_HIP_OK)
    {
        return rc;
    }
    const int64_t rows = query_rows(a->cache, a->q_seq, a->kv_group);
    if((four && p.c.max_rows > kLongest) || rows < 0 || a->Q == nullptr || a->lse == nullptr || a->A == nullptr
            || !on16(a->Q) || !on16(a->A) || (reinterpret_cast<uintptr_t>(a->lse) & 3u) != 0
            || (a->flags & ~NNTILE_HIP_SDPA_OVERWRITE) != 0)
    {
        return NNTILE_HIP_EINVAL;
    }
    if(mask_check(a->mask_mode) != NNTILE_HIP_OK)
    {
        return mask_check(a->mask_mode);
    }
    if(workspace == nullptr || !on16(workspace)
            || workspace_bytes < paged_attend_workspace_bytes(rows, a->cache.head))
    {
        return NNTILE_HIP_EWORKSPACE;
    }
    p.Q = a->Q;
    p.lse = a->lse;
    p.A = a->A;
    p.q_seq = (int32_t)a->q_seq;
    p.kv_group = (int32_t)a->kv_group;
    p.rows = (int32_t)rows;
    p.causal = a->mask_mode == NNTILE_HIP_MASK_CAUSAL;
    p.overwrite = (a->flags & NNTILE_HIP_SDPA_OVERWRITE) != 0;
    p.scale = 1.0f / sqrtf((float)a->cache.head);
    return (four ? launch_paged4_attend : launch_paged_attend)(static_cast<hipStream_t>(stream), dtype, p,
            (int)a->cache.head, workspace);
}

int page_bits(const nntile_hip_paged_cache &c, int dtype, bool four)
{
    return four ? 4 : c.k_scales != nullptr ? 8 : 8 * elem_bytes(dtype);
}

int weights_call(int dtype, bool four, void *stream, const nntile_hip_paged_weights_args *a)
{
    if(a == nullptr)
    {
        return NNTILE_HIP_EINVAL;
    }
    PagedView view;
    const int rc = paged_view(&a->cache, dtype, view, four, false);
    if(rc != NNTILE_HIP_OK)
    {
        return rc;
    }
    const int64_t rows = query_rows(a->cache, a->q_seq, a->kv_group);
    if(rows < 0 || a->Q == nullptr || a->lse == nullptr || a->weights == nullptr || !on16(a->Q)
            || (reinterpret_cast<uintptr_t>(a->lse) & 3u) != 0 || (reinterpret_cast<uintptr_t>(a->weights) & 3u) != 0
            || view.max_rows > kLongest || a->columns < view.max_rows || a->columns > kMost
            || !(a->decay >= 0.0f && a->decay <= 1.0f))
    {
        return NNTILE_HIP_EINVAL;
    }
    if(mask_check(a->mask_mode) != NNTILE_HIP_OK)
    {
        return mask_check(a->mask_mode);
    }
    PagedWeightsParams p = {view, a->Q, a->lse, a->weights, a->columns, (int32_t)a->q_seq, (int32_t)a->kv_group,
        (int32_t)rows, a->mask_mode == NNTILE_HIP_MASK_CAUSAL, a->decay, 1.0f / sqrtf((float)a->cache.head), 0,
        FixedDivide((uint32_t)a->q_seq)};
    return launch_paged_weights(static_cast<hipStream_t>(stream), dtype, page_bits(a->cache, dtype, four), p,
            (int)a->cache.head);
}

int evict_call(int dtype, bool four, void *stream, const nntile_hip_paged_evict_args *a)
{
    if(a == nullptr)
    {
        return NNTILE_HIP_EINVAL;
    }
    PagedEvictParams p = {};
    const int rc = paged_view(&a->cache, dtype, p.c, four);
    if(rc != NNTILE_HIP_OK)
    {
        return rc;
    }
    if(p.c.max_rows > kLongest || a->keep <= 0 || a->keep > kLongest || a->recent < 0 || a->recent > a->keep
            || a->weights == nullptr || a->weights_out == nullptr || a->kept == nullptr || (reinterpret_cast<uintptr_t>(a->weights) & 3u) != 0
            || (reinterpret_cast<uintptr_t>(a->weights_out) & 3u) != 0
            || (reinterpret_cast<uintptr_t>(a->kept) & 3u) != 0 || a->columns < p.c.max_rows || a->columns > kMost)
    {
        return NNTILE_HIP_EINVAL;
    }
    p.weights = a->weights;
    p.weights_out = a->weights_out;
    p.kept = a->kept;
    p.columns = a->columns;
    p.keep = (int32_t)a->keep;
    p.recent = (int32_t)a->recent;
    return launch_paged_evict(static_cast<hipStream_t>(stream), page_bits(a->cache, dtype, four), p, (int)a->cache.head);
}

int rope_axes_call(int dtype, void *stream, const nntile_hip_rope_axes_args *a)
{
    if(a == nullptr || a->head < 0 || a->seq < 0 || a->n_batch < 0 || a->heads_q < 0 || a->heads_k < 0
            || a->n_axes <= 0 || a->n_axes > kMost || a->head % 2 != 0
            || (a->pos_batch_stride != 0 && a->pos_batch_stride != a->seq) || a->heads_k > kMost - a->heads_q)
    {
        return NNTILE_HIP_EINVAL;
    }
    // all sizes together stay addresses
    const int64_t heads = a->heads_q + a->heads_k;
    if(a->head == 0 || a->seq == 0 || a->n_batch == 0 || heads == 0)
    {
        return NNTILE_HIP_OK;
    }
    int64_t elements = a->head;
    for(int64_t d : {a->seq, a->n_batch, heads > a->n_axes ? heads : a->n_axes})
    {
        if(d > ((int64_t)1 << 58) / elements)
        {
            return NNTILE_HIP_EINVAL;
        }
        elements *= d;
    }
    const uintptr_t e = (uintptr_t)elem_bytes(dtype) - 1;
    if(a->positions == nullptr || a->freqs == nullptr || a->axes == nullptr
            || (a->heads_q != 0 && (a->q == nullptr || a->q_out == nullptr))
            || (a->heads_k != 0 && (a->k == nullptr || a->k_out == nullptr))
            || (reinterpret_cast<uintptr_t>(a->positions) & 7u) != 0
            || (reinterpret_cast<uintptr_t>(a->freqs) & 7u) != 0
            || (reinterpret_cast<uintptr_t>(a->axes) & 3u) != 0
            || ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out)
                    | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->k_out)) & e) != 0)
    {
        return NNTILE_HIP_EINVAL;
    }
    RopeAxesParams p = {};
    p.head = a->head;
    p.seq = a->seq;
    p.n_batch = a->n_batch;
    p.heads_q = a->heads_q;
    p.heads_k = a->heads_k;
    p.pos_batch_stride = a->pos_batch_stride;
    p.pos_axis_stride = a->pos_batch_stride == 0 ? a->seq : a->seq * a->n_batch;
    p.n_axes = (int32_t)a->n_axes;
    p.positions = a->positions;
    p.freqs = a->freqs;
    p.axes = a->axes;
    p.q = a->q;
    p.k = a->k;
    p.q_out = a->q_out;
    p.k_out = a->k_out;
    return launch_rope_axes(static_cast<hipStream_t>(stream), dtype, a->backward != 0, p);
}

} // namespace

extern "C"
{

size_t nntile_hip_sdpa_fwd_paged_workspace_bytes(const nntile_hip_sdpa_paged_args *args)
{
    const int64_t rows = args == nullptr ? -1 : query_rows(args->cache, args->q_seq, args->kv_group);
    return rows < 0 || args->cache.head <= 0 || args->cache.head > 128 ? 0
        : paged_attend_workspace_bytes(rows, args->cache.head);
}

#define NNTILE_HIP_PAGED_ENTRY(suffix, dt, ctype) \
    int nntile_hip_paged_kv_append_##suffix(void *stream, const nntile_hip_paged_cache *cache, \
            int64_t rows, const ctype *k_new, const ctype *v_new) \
    { \
        return append_call(dt, false, stream, cache, rows, k_new, v_new); \
    } \
    int nntile_hip_paged_kv_read_##suffix(void *stream, const nntile_hip_paged_cache *cache, \
            int64_t first, int64_t rows, ctype *k_out, ctype *v_out) \
    { \
        return read_call(dt, false, stream, cache, first, rows, k_out, v_out); \
    } \
    int nntile_hip_sdpa_fwd_paged_##suffix(void *stream, const nntile_hip_sdpa_paged_args *args, \
            void *workspace, size_t workspace_bytes) \
    { \
        return attend_call(dt, false, stream, args, workspace, workspace_bytes); \
    } \
    int nntile_hip_paged_attn_weights_##suffix(void *stream, const nntile_hip_paged_weights_args *args) \
    { \
        return weights_call(dt, false, stream, args); \
    } \
    int nntile_hip_paged_kv_evict_##suffix(void *stream, const nntile_hip_paged_evict_args *args) \
    { \
        return evict_call(dt, false, stream, args); \
    } \
    int nntile_hip_rope_axes_##suffix(void *stream, const nntile_hip_rope_axes_args *args) \
    { \
        return rope_axes_call(dt, stream, args); \
    }
NNTILE_HIP_PAGED_ENTRY(bf16, 0, uint16_t)
NNTILE_HIP_PAGED_ENTRY(fp16, 1, uint16_t)
NNTILE_HIP_PAGED_ENTRY(fp32, 2, float)
#undef NNTILE_HIP_PAGED_ENTRY

#define NNTILE_HIP_PAGED4_ENTRY(suffix, dt) \
    int nntile_hip_paged4_kv_append_##suffix(void *stream, const nntile_hip_paged_cache *cache, \
            int64_t rows, const uint16_t *k_new, const uint16_t *v_new) \
    { \
        return append_call(dt, true, stream, cache, rows, k_new, v_new); \
    } \
    int nntile_hip_paged4_kv_read_##suffix(void *stream, const nntile_hip_paged_cache *cache, \
            int64_t first, int64_t rows, uint16_t *k_out, uint16_t *v_out) \
    { \
        return read_call(dt, true, stream, cache, first, rows, k_out, v_out); \
    } \
    int nntile_hip_sdpa_fwd_paged4_##suffix(void *stream, const nntile_hip_sdpa_paged_args *args, \
            void *workspace, size_t workspace_bytes) \
    { \
        return attend_call(dt, true, stream, args, workspace, workspace_bytes); \
    } \
    int nntile_hip_paged4_attn_weights_##suffix(void *stream, const nntile_hip_paged_weights_args *args) \
    { \
        return weights_call(dt, true, stream, args); \
    } \
    int nntile_hip_paged4_kv_evict_##suffix(void *stream, const nntile_hip_paged_evict_args *args) \
    { \
        return evict_call(dt, true, stream, args); \
    }
NNTILE_HIP_PAGED4_ENTRY(bf16, 0)
NNTILE_HIP_PAGED4_ENTRY(fp16, 1)
#undef NNTILE_HIP_PAGED4_ENTRY

} // extern "C"
