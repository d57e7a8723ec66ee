// What cached rows receive of attention: with s = q.k / sqrt(head) and the queries' logsumexp,
//
//   weights = decay * weights + sum over the queries that see the key of exp(s - lse)
//
// for every key of a sequence, over the kv_group query heads of a key/value head and its newest tokens.  One pass
// over the keys in HBM; every key's sum is taken by one wavefront in a fixed order, so the same call gives the same
// bits.
//
//  * The keys of a sequence are cut into blocks, the blocks of all (sequence, head) pairs are numbered through and
//    every workgroup takes an equal run of them, whatever the lengths (which live on the device).
//  * S = Q K^T with matrix instructions of 16 x 16: a lane has one key and four queries, so that a key's sum stays in
//    the lane but for the last two steps, across the four lanes that share it.
//  * A wavefront's keys stay in registers while the queries, 64 rows at a time, come from LDS.
#include <type_traits>

#include "paged_operands.hpp"

namespace nntile_hip
{

constexpr int kWeightsCUs = 256;

// Where a workgroup stands: block `block` of `blocks` of head h of sequence n
struct WeightsPlace
{
    int n, h, len, block, blocks;
};

// GK: groups of 16 keys of a wavefront.
template<typename T, int KIND, int HEAD, int GK>
__global__ __launch_bounds__(256)
void paged_weights_kernel(const PagedWeightsParams p)
{
    constexpr int RB = KIND == kPaged32 ? HEAD * 4 : KIND == kPaged8 ? HEAD : KIND == kPaged4 ? HEAD / 2 : HEAD * 2;
    constexpr int KEYS = 16 * GK, BLOCK = 4 * KEYS;     // keys of a wavefront's step, of a workgroup's
    constexpr int ROWS = 64;                            // query rows that lie in LDS
    // registers of 16 bytes of a row's operand, for keys and queries
    constexpr int QREGS = KIND == kPaged32 ? HEAD / 16 : HEAD / 32;
    // keys of 4 bits become bf16 numbers, and an fp16 query the sum of two
    constexpr bool TWO_Q = KIND == kPaged4 && __is_same(T, Fp16);
    constexpr int QPARTS = TWO_Q ? 2 : 1;
    typedef typename std::conditional<KIND == kPaged4, Bf16, T>::type QK;
    constexpr int QB = HEAD * (KIND == kPaged32 ? 4 : 2), PIECES = QB / 16;
    __shared__ __attribute__((aligned(16))) char q_rows[QPARTS * ROWS * QB];
    __shared__ __attribute__((aligned(16))) float off_of[ROWS];     // -lse in log2 units; -inf: the row counts nothing
    __shared__ __attribute__((aligned(16))) int last_of[ROWS];      // the last key the row sees

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    auto swizzled = [](int r, int piece) { return piece ^ (r % (PIECES < 16 ? PIECES : 16)); };
    // the 16-byte piece of a query row that goes with a lane's operand i
    auto q_piece = [&](int i)
    {
        return KIND == kPaged16 ? 4 * i + quad : KIND == kPaged8 ? 8 * (i / 2) + 2 * quad + i % 2
            : KIND == kPaged4 ? HEAD / 32 * quad + i : 4 * i + quad;
    };

    // ---- the workgroup's run of blocks ----------------------------------------------
    auto blocks_of = [&](int len) { return (len + BLOCK - 1) / BLOCK; };
    int mine = 0;
    for(int n = lane; n < p.c.n_batch; n += 64)
    {
        mine += blocks_of(paged_len(p.c, n));
    }
#pragma unroll
    for(int o = 32; o >= 1; o >>= 1)
    {
        mine += __shfl_xor(mine, o);
    }
    const uint32_t all = (uint32_t)uniform(mine) * (uint32_t)p.c.n_head_kv;
    const uint32_t shares = min((uint32_t)p.shares, all);
    if(blockIdx.x >= shares)
    {
        return;
    }
    const PagedSplit split(all, shares);
    const uint32_t at = split.begin(blockIdx.x);
    int left = (int)(split.begin(blockIdx.x + 1) - at);
    WeightsPlace place = {};
    {
        uint32_t before = 0;
        for(;; ++place.n)
        {
            place.len = uniform(paged_len(p.c, place.n));
            place.blocks = blocks_of(place.len);
            const uint32_t here = (uint32_t)place.blocks * (uint32_t)p.c.n_head_kv;
            if(at < before + here)
            {
                break;      // (at < all: there is one)
            }
            before += here;
        }
        place.h = uniform((int)((at - before) / (uint32_t)place.blocks));
        place.block = uniform((int)((at - before) % (uint32_t)place.blocks));
    }
    const float c_log2 = p.scale * kLog2e;

    bool staged = false;        // the pair's queries lie in LDS, all of them
    bool dead = false;          // a query of those in LDS counts nothing, whatever its scores are
    for(;;)
    {
        const int given = uniform(paged_new(p.c, place.n, p.q_seq));
        const int key0 = place.block * BLOCK + wave * KEYS;
        const bool here = key0 < place.len;

        // ---- keys ----------------------------------------------------------------------
        u32x4 kf[GK][QREGS];
        float s_scale[GK];
        uint32_t hidden = 0;        // groups without a page
#pragma unroll
        for(int g = 0; g < GK; ++g)
        {
            s_scale[g] = 1.0f;
            // (groups behind the last row: the last one's rows, not written)
            const int row = max(min(key0 + 16 * g, place.len - 1), 0) & ~15;
            const int page_in = scalar_load<int>(p.c.table, 4 * ((int64_t)place.n * p.c.max_pages + (row >> p.c.page_shift)));
            const bool real = (unsigned)page_in < (unsigned)p.c.n_pages;
            hidden |= real ? 0u : 1u << g;
            const int64_t page = real ? page_in : 0;
            const int64_t in_page = ((int64_t)place.h << p.c.page_shift) + (row & ((1 << p.c.page_shift) - 1)) + col;
            const char *const from = p.c.k_pages + page * p.c.page_stride + in_page * RB;
            if constexpr(KIND == kPaged4)
            {
                constexpr int W = HEAD / 32;        // words of a lane
                const float scale = __uint_as_float((uint32_t)p.c.k_scales[page * p.c.scale_stride + in_page * W
                        + quad * W / 4] << 23);
#pragma unroll
                for(int i = 0; i < W; ++i)
                {
                    kf[g][i] = widen8_of_4<Bf16>(*reinterpret_cast<const uint32_t *>(from + 4 * (W * quad + i)), scale);
                }
            }
            else if constexpr(KIND == kPaged8)
            {
                const float scale = __uint_as_float((uint32_t)p.c.k_scales[page * p.c.scale_stride + in_page] << 23);
                s_scale[g] = __is_same(T, Bf16) ? 1.0f : scale;
#pragma unroll
                for(int i = 0; i < QREGS / 2; ++i)
                {
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(from + 16 * (4 * i + quad));
#pragma unroll
                    for(int j = 0; j < 2; ++j)
                    {
                        const u32x2 a = widen4<T>(x[2 * j], __is_same(T, Bf16) ? scale : 1.0f),
                            b = widen4<T>(x[2 * j + 1], __is_same(T, Bf16) ? scale : 1.0f);
                        kf[g][2 * i + j] = u32x4{a[0], a[1], b[0], b[1]};
                    }
                }
            }
            else
            {
#pragma unroll
                for(int i = 0; i < QREGS; ++i)
                {
                    kf[g][i] = *reinterpret_cast<const u32x4 *>(from + 16 * (4 * i + quad));
                }
            }
        }

        // ---- sums over the queries -------------------------------------------------------
        float sum[GK];
#pragma unroll
        for(int g = 0; g < GK; ++g)
        {
            sum[g] = 0.0f;
        }
        // below it every row sees every key
        const int all_see = p.causal ? place.len - given : place.len - 1;
        const bool partly = key0 + KEYS - 1 > all_see || hidden != 0;
        for(int row0 = 0; row0 < (given > 0 ? p.rows : 0); row0 += ROWS)
        {
            const int rows = min(p.rows - row0, ROWS);
            if(!staged)
            {
                __syncthreads();        // the rows before these are done with
                bool counts_not = false;
                for(int t = tid; t < ROWS * PIECES; t += 256)
                {
                    const int r = t / PIECES, piece = t % PIECES, rr = row0 + r;
                    const int g = rr / p.q_seq, tok = rr % p.q_seq;
                    const bool ok = r < rows && tok < given;
                    const int64_t row = (place.n + (int64_t)p.c.n_batch * (g + (int64_t)p.kv_group * place.h)) * p.q_seq + tok;
                    u32x4 x = {0, 0, 0, 0};
                    if(ok)
                    {
                        x = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(p.Q) + row * QB + piece * 16);
                    }
                    char *const to = q_rows + r * QB + swizzled(r, piece) * 16;
                    if constexpr(TWO_Q)
                    {
                        u32x4 rest;
                        two_bf16(x, x, rest);
                        *reinterpret_cast<u32x4 *>(to + ROWS * QB) = rest;
                    }
                    *reinterpret_cast<u32x4 *>(to) = x;
                    if(piece == 0)
                    {
                        const float lse = ok ? p.lse[row] : neg_inf();
                        counts_not = counts_not || (ok && lse == neg_inf());
                        off_of[r] = lse == neg_inf() ? neg_inf() : -lse * kLog2e;
                        last_of[r] = lse == neg_inf() ? -1 : p.causal ? place.len - given + tok : place.len - 1;
                    }
                }
                dead = __syncthreads_or(counts_not);
                staged = p.rows <= ROWS;
            }
            if(!here)
            {
                continue;
            }
            for(int rb = 0; rb < rows; rb += 16)
            {
                const f32x4 off = *reinterpret_cast<const f32x4 *>(off_of + rb + 4 * quad);
                f32x4 s[GK];
#pragma unroll
                for(int g = 0; g < GK; ++g)
                {
                    s[g] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for(int i = 0; i < QREGS; ++i)
                {
                    const char *const q_at = q_rows + (rb + col) * QB + swizzled(col, q_piece(i)) * 16;
                    const u32x4 q = *reinterpret_cast<const u32x4 *>(q_at);
#pragma unroll
                    for(int g = 0; g < GK; ++g)
                    {
                        if constexpr(KIND == kPaged32)
                        {
#pragma unroll
                            for(int e = 0; e < 4; ++e)
                            {
                                s[g] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(q[e]),
                                        __uint_as_float(kf[g][i][e]), s[g], 0, 0, 0);
                            }
                        }
                        else
                        {
                            s[g] = mfma32<QK>(q, kf[g][i], s[g]);
                        }
                    }
                    if constexpr(TWO_Q)
                    {
                        const u32x4 rest = *reinterpret_cast<const u32x4 *>(q_at + ROWS * QB);
#pragma unroll
                        for(int g = 0; g < GK; ++g)
                        {
                            s[g] = mfma32<QK>(rest, kf[g][i], s[g]);
                        }
                    }
                }
                if(partly || dead)
                {
                    typedef __attribute__((ext_vector_type(4))) int i32x4;
                    const i32x4 last = *reinterpret_cast<const i32x4 *>(last_of + rb + 4 * quad);
#pragma unroll
                    for(int g = 0; g < GK; ++g)
                    {
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            const float x = fast_exp2(fmaf(s[g][e] * s_scale[g], c_log2, off[e]));
                            sum[g] += key0 + 16 * g + col <= ((hidden >> g) & 1 ? -1 : last[e]) ? x : 0.0f;
                        }
                    }
                }
                else
                {
#pragma unroll
                    for(int g = 0; g < GK; ++g)
                    {
                        const float c = KIND == kPaged8 ? c_log2 * s_scale[g] : c_log2;
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            sum[g] += fast_exp2(fmaf(s[g][e], c, off[e]));
                        }
                    }
                }
            }
        }
        if(here)
        {
            float *const to = p.weights + (place.n + (int64_t)p.c.n_batch * place.h) * p.columns + key0;
#pragma unroll
            for(int g = 0; g < GK; ++g)
            {
                const float x = quad_sum(sum[g]);
                if(quad == 0 && key0 + 16 * g + col < place.len)
                {
                    float *const w = to + 16 * g + col;
                    *w = p.decay == 0.0f ? x : fmaf(p.decay, *w, x);
                }
            }
        }
        if(--left == 0)
        {
            return;
        }
        if(++place.block == place.blocks)
        {
            place.block = 0;
            staged = false;
            if(++place.h == p.c.n_head_kv)
            {
                place.h = 0;
                do
                {
                    ++place.n;
                    place.len = uniform(paged_len(p.c, place.n));
                    place.blocks = blocks_of(place.len);
                } while(place.blocks == 0);     // (there is a block left)
            }
        }
    }
}

template<typename T, int KIND, int HEAD, int GK>
static int launch_form(hipStream_t stream, PagedWeightsParams &p)
{
    constexpr int BLOCK = 64 * GK;
    const int64_t most = (int64_t)p.c.n_batch * p.c.n_head_kv * ((p.c.max_rows - 1) / BLOCK + 1);
    if(most > 0x7fffffffll)
    {
        return NNTILE_HIP_EINVAL;
    }
    const int64_t places = kWeightsCUs * (GK == 1 ? 4 : 2);
    p.shares = (int32_t)(most < places ? most : places);
    hipLaunchKernelGGL((paged_weights_kernel<T, KIND, HEAD, GK>), dim3((unsigned)p.shares), dim3(256), 0, stream, p);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

template<typename T, int KIND>
static int launch_kind(hipStream_t stream, PagedWeightsParams &p, int head)
{
    if(p.rows > 32)
    {
        return head == 64 ? launch_form<T, KIND, 64, 4>(stream, p)
            : launch_form<T, KIND, 128, KIND == kPaged32 ? 2 : 4>(stream, p);
    }
    return head == 64 ? launch_form<T, KIND, 64, 1>(stream, p) : launch_form<T, KIND, 128, 1>(stream, p);
}

int launch_paged_weights(hipStream_t stream, int dtype, int bits, PagedWeightsParams &p, int head)
{
    switch(bits * 4 + dtype)
    {
        case 4 * 4: return launch_kind<Bf16, kPaged4>(stream, p, head);
        case 4 * 4 + 1: return launch_kind<Fp16, kPaged4>(stream, p, head);
        case 8 * 4: return launch_kind<Bf16, kPaged8>(stream, p, head);
        case 8 * 4 + 1: return launch_kind<Fp16, kPaged8>(stream, p, head);
        case 16 * 4: return launch_kind<Bf16, kPaged16>(stream, p, head);
        case 16 * 4 + 1: return launch_kind<Fp16, kPaged16>(stream, p, head);
        case 32 * 4 + 2: return launch_kind<float, kPaged32>(stream, p, head);
        default: return NNTILE_HIP_EUNSUPPORTED;
    }
}

} // namespace nntile_hip
