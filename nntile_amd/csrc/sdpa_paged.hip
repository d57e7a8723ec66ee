// The attention over pages of the tile type and of 8-bit codes.
#include "sdpa_paged.hpp"

namespace nntile_hip
{

size_t paged_attend_workspace_bytes(int64_t rows, int64_t head)
{
    return sizeof(unsigned long long) * kPagedShares * kPagedCountStride + share_rows(rows) * (size_t)(head + 2) * 4;
}

int launch_paged_attend(hipStream_t stream, int dtype, PagedAttendParams &p, int head, void *workspace)
{
    place_workspace(p, head, workspace);
    if(p.c.k_scales != nullptr)
    {
        return dtype == 0 ? launch_kind<Bf16, kPaged8>(stream, p, head)
            : dtype == 1 ? launch_kind<Fp16, kPaged8>(stream, p, head) : NNTILE_HIP_EUNSUPPORTED;
    }
    return dtype == 0 ? launch_kind<Bf16, kPaged16>(stream, p, head)
        : dtype == 1 ? launch_kind<Fp16, kPaged16>(stream, p, head)
        : launch_kind<float, kPaged32>(stream, p, head);
}

} // namespace nntile_hip
