// The attention over pages of 4-bit codes.
#include "sdpa_paged.hpp"

namespace nntile_hip
{

int launch_paged4_attend(hipStream_t stream, int dtype, PagedAttendParams &p, int head, void *workspace)
{
    place_workspace(p, head, workspace);
    return dtype == 0 ? launch_kind<Bf16, kPaged4>(stream, p, head)
        : dtype == 1 ? launch_kind<Fp16, kPaged4>(stream, p, head) : NNTILE_HIP_EUNSUPPORTED;
}

} // namespace nntile_hip
