// Eviction from a cache in pages: of every sequence and head the rows that received most of the attention stay,
// and move together.
//
// Of a sequence with more rows than `keep` stay its last `recent` ones and, of those in front, the heaviest; of equal
// ones the lower row.  They keep their order: row d of what is left is row kept[d] of what was there, kept[d] >= d,
// and moves down in place.  Two launches:
//
//  * selection, a workgroup for every (sequence, head): the threshold by counting the weights' bits from the top, 11,
//    11 and 10 of them, in LDS; then one walk over the rows that numbers those that stay.
//  * the moves, a workgroup for every (sequence, head), K or V, and 64 bytes of the rows: some thousand rows at a
//    time are read into registers, and when all of them are there, written.  A row's new place lies at or in front of
//    its old one, so rows that are read later are never in the way.  What is kept and where it lies is looked up a step
//    ahead, and the first rows, which stay where they are, are skipped (64 of 8192 bf16 rows of 128 values, 8128 kept at
//    random 143 -> 123 us, 1088 of 8128 behind the first that goes 27.9 -> 17).
//
// Bound by latency where little moves: 12 heads of 1024 fp32 rows down to 512 take 9.3 us, half of it the launches,
// the rest the chain of loads, counts and barriers of the selection, and length, kept, table and row of a move.  64 of
// 700 to 8192 4-bit rows down to 1024, 57 MB, 25 us with what reads the pages back; the selection is 8.6 us of them (12.5
// with the weights read again in every pass), the moves 6.6.  With much to move by HBM and the last-level cache: those 8128
// of 8192 rows are 525 MB read and written, 4.7 TB/s in the moves alone.  Slices of 64 bytes of a row: with whole rows a
// workgroup there were a quarter as many to have loads on their way.
#include "paged_operands.hpp"
#include "paged_rows.hpp"

namespace nntile_hip
{

// A weight as an integer of the same order: -0 as 0, a NaN above all
__device__ __forceinline__ uint32_t weight_key(float w)
{
    const uint32_t u = __float_as_uint(w + 0.0f);
    return w != w ? ~0u : (u >> 31) != 0 ? ~u : u | 0x80000000u;
}

// The sums of `x` over the threads in front of this one, and over all.  wave_sum is the call's until the second barrier
// from here.
template<int WAVES>
__device__ __forceinline__ uint32_t workgroup_scan(uint32_t x, uint32_t *wave_sum, uint32_t &all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t upto = wave_scan(x);
    if(lane == 63)
    {
        wave_sum[wave] = upto;
    }
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for(int w = 0; w < WAVES; ++w)
    {
        before += w < wave ? wave_sum[w] : 0;
        all += wave_sum[w];
    }
    return before + upto - x;
}

// A step of the walk over the weights is four of them a thread.  HELD: steps whose weights stay in registers from the
// first look at them to the last; 0: as many as there are rows for, from memory each time.
template<int THREADS, int HELD>
__global__ __launch_bounds__(THREADS)
void paged_select_kernel(const PagedEvictParams p)
{
    constexpr int STEP = 4 * THREADS, WAVES = THREADS / 64, BINS = 2048, MINE = BINS / THREADS;
    constexpr int KEPT = HELD > 0 ? HELD : 1;
    __shared__ uint32_t bins[BINS];
    __shared__ uint32_t wave_sum[2][WAVES];
    __shared__ uint32_t found[3];
    const int tid = threadIdx.x;
    const uint32_t entries = (uint32_t)p.c.n_batch * (uint32_t)p.c.n_head_kv;
    for(uint32_t entry = blockIdx.x; entry < entries; entry += gridDim.x)
    {
        const int n = (int)(entry % (uint32_t)p.c.n_batch);
        const int len = uniform(paged_len(p.c, n));
        const float *const w_in = p.weights + (int64_t)entry * p.columns;
        float *const w_out = p.weights_out + (int64_t)entry * p.columns;
        int32_t *const kept = p.kept + (int64_t)entry * p.keep;
        const int stay = min(len, p.keep);
        for(int d = stay + tid; d < p.keep; d += THREADS)
        {
            kept[d] = -1;
        }
        if(len <= p.keep)
        {
            for(int d = tid; d < len; d += THREADS)
            {
                kept[d] = d;
                if(w_out != w_in)
                {
                    w_out[d] = w_in[d];
                }
            }
            continue;
        }
        const int old = len - p.recent;             // rows that are chosen from (recent <= keep < len)
        const int steps = (len + STEP - 1) / STEP;
        // the thread's weights of step s: rows s * STEP + 4 * tid and on; behind the last: 0
        float held[KEPT][4];
        auto look = [&](int s, float (&w)[4])
        {
            const int at = s * STEP + 4 * tid;
            if(at + 3 < len)
            {
                __builtin_memcpy(w, w_in + at, 16);
            }
            else
            {
#pragma unroll
                for(int k = 0; k < 4; ++k)
                {
                    w[k] = at + k < len ? w_in[at + k] : 0.0f;
                }
            }
        };
        // f(s, weights of step s) for all steps, in order
        auto walk = [&](auto f)
        {
            if constexpr(HELD > 0)
            {
#pragma unroll
                for(int s = 0; s < HELD; ++s)
                {
                    if(s < steps)
                    {
                        f(s, held[s]);
                    }
                }
            }
            else
            {
                for(int s = 0; s < steps; ++s)
                {
                    look(s, held[0]);
                    f(s, held[0]);
                }
            }
        };
        if constexpr(HELD > 0)
        {
#pragma unroll
            for(int s = 0; s < HELD; ++s)
            {
                if(s < steps)
                {
                    look(s, held[s]);
                }
            }
        }
        // ---- the key of the wanted-th heaviest row ------------------------------------
        // All rows with a key above `key` stay, and the first `wanted` that have it.
        uint32_t wanted = (uint32_t)(p.keep - p.recent), key = ~0u;
        if(wanted != 0)
        {
            uint32_t prefix = 0;
            for(int pass = 0; pass < 3; ++pass)
            {
                const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 1024 : 2048;
#pragma unroll
                for(int b = 0; b < MINE; ++b)
                {
                    bins[tid + b * THREADS] = 0;
                }
                __syncthreads();
                walk([&](int s, const float (&w)[4])
                {
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                    {
                        const uint32_t of = weight_key(w[k]);
                        if(s * STEP + 4 * tid + k < old && (pass == 0 || (of >> (pass == 1 ? 21 : 10)) == prefix))
                        {
                            atomicAdd(&bins[(of >> shift) & (width - 1)], 1u);
                        }
                    }
                });
                __syncthreads();
                // the largest bits first, some a thread
                uint32_t count[MINE], sum = 0;
#pragma unroll
                for(int b = 0; b < MINE; ++b)
                {
                    count[b] = bins[BINS - 1 - MINE * tid - b];
                    sum += count[b];
                }
                uint32_t all, before = workgroup_scan<WAVES>(sum, wave_sum[pass & 1], all);
#pragma unroll
                for(int b = 0; b < MINE; ++b)
                {
                    if(before < wanted && wanted <= before + count[b])
                    {
                        found[0] = (uint32_t)(BINS - 1 - MINE * tid - b);
                        found[1] = wanted - before;
                        found[2] = count[b];
                    }
                    before += count[b];
                }
                __syncthreads();
                prefix = prefix << (pass == 2 ? 10 : 11) | found[0];
                wanted = found[1];
                key = prefix << shift;
                if(wanted == found[2] && key != 0)
                {
                    // all rows with these bits stay, whatever the bits below
                    key -= 1;
                    wanted = 0;
                    break;
                }
            }
        }
        // ---- the rows that stay, in order ------------------------------------------------
        uint32_t above_before = 0, equal_before = 0;
        __syncthreads();        // (found and wave_sum have been read)
        walk([&](int s, const float (&w)[4])
        {
            const int at = s * STEP + 4 * tid;
            uint32_t above = 0, equal = 0;          // a bit for each of the four
#pragma unroll
            for(int k = 0; k < 4; ++k)
            {
                const uint32_t of = weight_key(w[k]);
                above |= (at + k < old ? of > key : at + k < len) ? 1u << k : 0u;
                equal |= at + k < old && of == key ? 1u << k : 0u;
            }
            // (at most 4096 of each in a step)
            uint32_t all;
            const uint32_t before = workgroup_scan<WAVES>((uint32_t)__popc(above) | (uint32_t)__popc(equal) << 16,
                    wave_sum[s & 1], all);
            uint32_t a = above_before + (before & 0xffffu), e = equal_before + (before >> 16);
#pragma unroll
            for(int k = 0; k < 4; ++k)
            {
                if((above >> k & 1) != 0 || ((equal >> k & 1) != 0 && e < wanted))
                {
                    const uint32_t d = a + min(e, wanted);
                    kept[d] = at + k;
                    w_out[d] = w[k];
                }
                a += above >> k & 1;
                e += equal >> k & 1;
            }
            above_before += all & 0xffffu;
            equal_before += all >> 16;
        });
        // (the last step's weights have been read by all: the barrier in its scan)
        for(int d = p.keep + tid; d < len; d += THREADS)
        {
            w_out[d] = 0.0f;
        }
        __syncthreads();        // the next entry's bins and sums
    }
}

constexpr int kEvictThreads = 1024;

// The scale bytes of a row, 1, 2 or 4
template<int SB> __device__ __forceinline__ uint32_t load_scales(const uint8_t *from)
{
    if constexpr(SB == 4)
    {
        return *reinterpret_cast<const uint32_t *>(from);
    }
    return SB == 2 ? *reinterpret_cast<const uint16_t *>(from) : *from;
}

template<int SB> __device__ __forceinline__ void store_scales(uint8_t *to, uint32_t x)
{
    if constexpr(SB == 4)
    {
        *reinterpret_cast<uint32_t *>(to) = x;
    }
    else if constexpr(SB == 2)
    {
        *reinterpret_cast<uint16_t *>(to) = (uint16_t)x;
    }
    else
    {
        *to = (uint8_t)x;
    }
}

// SB: scale bytes of a row.  LANES threads have 16 bytes each of a row's slice.
template<int ROW_BYTES, int SB>
__global__ __launch_bounds__(kEvictThreads)
void paged_evict_kernel(const PagedEvictParams p)
{
    constexpr int SLICE = ROW_BYTES < 64 ? ROW_BYTES : 64, SLICES = ROW_BYTES / SLICE, LANES = SLICE / 16;
    constexpr int ROWS = kEvictThreads / LANES, AT_ONCE = 4;
    const int piece = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const uint32_t entries = (uint32_t)p.c.n_batch * (uint32_t)p.c.n_head_kv;
    for(uint32_t work = blockIdx.x; work < entries * (2 * SLICES); work += gridDim.x)
    {
        // (the slices of a row, halves of the same cache lines, have equal index modulo 8 where the pairs are a multiple of 4:
        // one XCD)
        const uint32_t slice = work / (2 * entries), pair = work - slice * (2 * entries), entry = pair / 2, which = pair % 2;
        const int n = (int)(entry % (uint32_t)p.c.n_batch), h = (int)(entry / (uint32_t)p.c.n_batch);
        const int len = uniform(paged_len(p.c, n));
        if(len <= p.keep)
        {
            continue;
        }
        const int32_t *const kept = p.kept + (int64_t)entry * p.keep;
        char *const pages = (which ? p.c.v_pages : p.c.k_pages) + slice * SLICE + piece * 16;
        uint8_t *const scales = which ? p.c.v_scales : p.c.k_scales;
        constexpr int MOVES = ROWS * AT_ONCE;       // of a step
        int d0 = 0;
        if(p.keep > MOVES)
        {
            // rows in front of the first that goes stay where they are: looked for at every `apart`-th
            const int apart = (p.keep + kEvictThreads - 1) / kEvictThreads, d = (int)threadIdx.x * apart;
            d0 = max(__syncthreads_count(d < p.keep && kept[d] == d) - 1, 0) * apart;
        }
        // What is kept in places d0 + slot .. and, for rows that move, the pages they come from and go to.
        auto places = [&](int d0, int (&src)[AT_ONCE])
        {
#pragma unroll
            for(int k = 0; k < AT_ONCE; ++k)
            {
                const int d = d0 + k * ROWS + slot;
                src[k] = d < p.keep ? kept[d] : -1;
            }
        };
        auto look_up = [&](int d0, int (&src)[AT_ONCE], int (&from)[AT_ONCE], int (&to)[AT_ONCE])
        {
#pragma unroll
            for(int k = 0; k < AT_ONCE; ++k)
            {
                const int d = d0 + k * ROWS + slot;
                src[k] = src[k] > d && src[k] < len ? src[k] : -1;      // (a row that stays where it is)
                from[k] = src[k] >= 0 ? page_of(p.c, n, src[k]) : -1;
                to[k] = src[k] >= 0 ? page_of(p.c, n, d) : -1;
            }
        };
        int src[AT_ONCE], from[AT_ONCE], to[AT_ONCE];
        places(d0, src);
        look_up(d0, src, from, to);
        for(; d0 < p.keep; d0 += MOVES)
        {
            u32x4 x[AT_ONCE];
            uint32_t size[AT_ONCE];
            int next[AT_ONCE], next_from[AT_ONCE], next_to[AT_ONCE];
            places(d0 + MOVES, next);
#pragma unroll
            for(int k = 0; k < AT_ONCE; ++k)
            {
                // (a row without a page: zeros)
                x[k] = u32x4{0, 0, 0, 0};
                size[k] = 0x7f7f7f7fu;
                if(from[k] >= 0)
                {
                    const int64_t at = row_in_page(p.c, h, src[k]);
                    x[k] = *reinterpret_cast<const u32x4 *>(pages + from[k] * p.c.page_stride + at * ROW_BYTES);
                    if constexpr(SB != 0)
                    {
                        if(slice == 0 && piece == 0)
                        {
                            size[k] = load_scales<SB>(scales + from[k] * p.c.scale_stride + at * SB);
                        }
                    }
                }
            }
            // all rows of the step are read before the first is written
            paged_wait_loads<0>();
            __syncthreads();
            look_up(d0 + MOVES, next, next_from, next_to);
#pragma unroll
            for(int k = 0; k < AT_ONCE; ++k)
            {
                if(to[k] >= 0)
                {
                    const int64_t at = row_in_page(p.c, h, d0 + k * ROWS + slot);
                    *reinterpret_cast<u32x4 *>(pages + to[k] * p.c.page_stride + at * ROW_BYTES) = x[k];
                    if constexpr(SB != 0)
                    {
                        if(slice == 0 && piece == 0)
                        {
                            store_scales<SB>(scales + to[k] * p.c.scale_stride + at * SB, size[k]);
                        }
                    }
                }
                src[k] = next[k];
                from[k] = next_from[k];
                to[k] = next_to[k];
            }
        }
    }
}

template<int ROW_BYTES, int SB>
static int launch_evict(hipStream_t stream, const PagedEvictParams &p)
{
    constexpr int SLICES = ROW_BYTES < 64 ? 1 : ROW_BYTES / 64;
    const int64_t entries = (int64_t)p.c.n_batch * p.c.n_head_kv, work = entries * 2 * SLICES;
    if(work > 0x7fffffff)
    {
        return NNTILE_HIP_EINVAL;
    }
    // (a direction of a launch has less than 2^32 threads)
    constexpr int64_t MOST = 1 << 20;
    const dim3 grid((unsigned)(entries < MOST ? entries : MOST));
    if(p.c.max_rows <= 4096)
    {
        hipLaunchKernelGGL((paged_select_kernel<256, 4>), grid, dim3(256), 0, stream, p);
    }
    else if(p.c.max_rows <= 8192)
    {
        hipLaunchKernelGGL((paged_select_kernel<1024, 2>), grid, dim3(1024), 0, stream, p);
    }
    else if(p.c.max_rows <= 32768)
    {
        hipLaunchKernelGGL((paged_select_kernel<1024, 8>), grid, dim3(1024), 0, stream, p);
    }
    else
    {
        hipLaunchKernelGGL((paged_select_kernel<1024, 0>), grid, dim3(1024), 0, stream, p);
    }
    if(hipGetLastError() != hipSuccess)
    {
        return NNTILE_HIP_ELAUNCH;
    }
    hipLaunchKernelGGL((paged_evict_kernel<ROW_BYTES, SB>), dim3((unsigned)(work < MOST ? work : MOST)), dim3(kEvictThreads), 0,
            stream, p);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

int launch_paged_evict(hipStream_t stream, int bits, const PagedEvictParams &p, int head)
{
    switch(bits * 256 + head)
    {
        case 4 * 256 + 64: return launch_evict<32, 2>(stream, p);
        case 4 * 256 + 128: return launch_evict<64, 4>(stream, p);
        case 8 * 256 + 64: return launch_evict<64, 1>(stream, p);
        case 8 * 256 + 128: return launch_evict<128, 1>(stream, p);
        case 16 * 256 + 64: return launch_evict<128, 0>(stream, p);
        case 16 * 256 + 128: return launch_evict<256, 0>(stream, p);
        case 32 * 256 + 64: return launch_evict<256, 0>(stream, p);
        case 32 * 256 + 128: return launch_evict<512, 0>(stream, p);
        default: return NNTILE_HIP_EUNSUPPORTED;
    }
}

} // namespace nntile_hip
