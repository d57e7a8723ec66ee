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
//  * A wavefront's keys stay in registers while the queries, up to 128 rows at a time, come from LDS; the next
//    block's keys, and the pages of the one behind it, are on their way meanwhile.
//  * Up to 32 rows a wavefront has 16 keys and a CU four workgroups, for HBM; 32 sequences of up to 2000 bf16 rows, 4
//    query rows, 50 MB, 11.3 us = 4.5 TB/s.  More rows: 64 keys (fp32 of 128 values 32), two blocks of 16 rows side by
//    side, since the products of one wait for each other, and two workgroups a CU; bound by vector instructions, of each
//    score an fma, an exponential and an addition: 4-bit fp16 pages of 16384 rows in all, 8 heads of 128, 128 query rows,
//    4.3 GFLOP, 11.6 us, of which 5 are that issue and 3 the launch (every query as the sum of two bf16 numbers 14.4, one
//    block of rows at a time and keys fetched where they are used as well 16.8).
#include <type_traits>

#include "fixed_divide.hpp"
#include "paged_operands.hpp"

namespace nntile_hip
{

constexpr int kWeightsCUs = 256;

// Where a workgroup stands: block `block` of `blocks` of head h of sequence n, which has `given` new tokens
struct WeightsPlace
{
    int n, h, len, given, block, blocks;
};

// GK: groups of 16 keys of a wavefront.
template<typename T, int KIND, int HEAD, int GK>
__global__ __launch_bounds__(256, (GK == 1 ? 4 : 2))
void paged_weights_kernel(const PagedWeightsParams p)
{
    constexpr int RB = KIND == kPaged32 ? HEAD * 4 : KIND == kPaged8 ? HEAD : KIND == kPaged4 ? HEAD / 2 : HEAD * 2;
    constexpr int KEYS = 16 * GK, BLOCK = 4 * KEYS;     // keys of a wavefront's step, of a workgroup's
    constexpr int ROWS = GK == 1 ? 32 : 128;            // query rows that lie in LDS
    constexpr int BLOCKS = GK == 1 ? 1 : 2;             // blocks of 16 of them side by side: one's sums wait for each other
    // registers of 16 bytes: of a row's operand, for keys and queries, and of a key row as it lies in its page
    constexpr int QREGS = KIND == kPaged32 ? HEAD / 16 : HEAD / 32, RAW = RB < 64 ? 1 : RB / 64;
    // Keys of 4 bits become numbers of the tile type exactly, those of fp16 tiles while their powers of two lie from 2^-13
    // to 2^13: a wavefront that has others makes bf16 numbers of its keys, and of a query the sum of two.
    constexpr bool NARROW = KIND == kPaged4 && __is_same(T, Fp16);
    constexpr int QB = HEAD * (KIND == kPaged32 ? 4 : 2), PIECES = QB / 16;
    constexpr bool CODES = KIND == kPaged4 || KIND == kPaged8;
    __shared__ __attribute__((aligned(16))) char q_rows[ROWS * QB];
    __shared__ __attribute__((aligned(16))) float off_of[ROWS];     // -lse in log2 units; -inf: the row counts nothing
    __shared__ __attribute__((aligned(16))) int last_of[ROWS];      // the last key the row sees

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    auto swizzled = [](int r, int piece) { return piece ^ (r % (PIECES < 16 ? PIECES : 16)); };
    // the 16-byte piece of a query row that goes with a lane's operand i
    auto q_piece = [&](int i)
    {
        return KIND == kPaged8 ? 8 * (i / 2) + 2 * quad + i % 2 : KIND == kPaged4 ? HEAD / 32 * quad + i : 4 * i + quad;
    };

    // ---- the workgroup's run of blocks ----------------------------------------------
    auto blocks_of = [&](int len) { return (len + BLOCK - 1) / BLOCK; };
    auto len_of = [&](int n) { return n < p.c.n_batch ? paged_len(p.c, n) : 0; };
    auto scan = [&](int len) { return wave_scan((uint32_t)blocks_of(len)); };      // blocks of the lanes up to this one
    auto last_lane = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); };
    int len_of_lane = len_of(lane);
    uint32_t upto = scan(len_of_lane), all = last_lane(upto);
    if(p.c.n_batch > 64)
    {
        uint32_t more = 0;
        for(int n = lane + 64; n < p.c.n_batch; n += 64)
        {
            more += (uint32_t)blocks_of(paged_len(p.c, n));
        }
        all += last_lane(wave_scan(more));
    }
    all *= (uint32_t)p.c.n_head_kv;
    const uint32_t shares = min((uint32_t)p.shares, all);
    if(blockIdx.x >= shares)
    {
        return;
    }
    const PagedSplit split(all, shares);
    uint32_t at = split.begin(blockIdx.x);
    int left = (int)(split.begin(blockIdx.x + 1) - at);
    WeightsPlace place = {};
    // 64 sequences at a time
    for(int n0 = 0;;)
    {
        const uint32_t here = last_lane(upto) * (uint32_t)p.c.n_head_kv;
        if(at < here)           // (there is one)
        {
            // the first sequence that ends behind the block
            const int t = __popcll(__ballot(upto * (uint32_t)p.c.n_head_kv <= at));
            place.n = n0 + t;
            place.len = __builtin_amdgcn_readlane(len_of_lane, t);
            place.blocks = blocks_of(place.len);
            at -= ((uint32_t)__builtin_amdgcn_readlane((int)upto, t) - (uint32_t)place.blocks) * (uint32_t)p.c.n_head_kv;
            break;
        }
        at -= here;
        n0 += 64;
        len_of_lane = len_of(n0 + lane);
        upto = scan(len_of_lane);
    }
    place.given = uniform(paged_new(p.c, place.n, p.q_seq));
    place.h = uniform((int)(at / (uint32_t)place.blocks));
    place.block = uniform((int)(at % (uint32_t)place.blocks));
    const float c_log2 = p.scale * kLog2e;

    auto next_of = [&](WeightsPlace x)
    {
        if(++x.block == x.blocks)
        {
            x.block = 0;
            if(++x.h == p.c.n_head_kv)
            {
                x.h = 0;
                do
                {
                    ++x.n;
                    x.len = uniform(paged_len(p.c, x.n));
                    x.blocks = blocks_of(x.len);
                } while(x.blocks == 0);     // (there is a block left)
                x.given = uniform(paged_new(p.c, x.n, p.q_seq));
            }
        }
        return x;
    };

    // ---- keys: the pages of the block after the next, the next one's rows, and this one's operands ------------
    // (groups behind the last row: the last one's rows, not written)
    auto group_row = [&](const WeightsPlace &x, int g)
    {
        return max(min(x.block * BLOCK + wave * KEYS + 16 * g, x.len - 1), 0) & ~15;
    };
    auto look_up = [&](const WeightsPlace &x, int (&page)[GK])
    {
#pragma unroll
        for(int g = 0; g < GK; ++g)
        {
            page[g] = scalar_load<int>(p.c.table, 4 * ((int64_t)x.n * p.c.max_pages + (group_row(x, g) >> p.c.page_shift)));
        }
    };
    auto weights_at = [&](const WeightsPlace &x)
    {
        return p.weights + (x.n + (int64_t)p.c.n_batch * x.h) * p.columns + x.block * BLOCK + wave * KEYS + col;
    };
    auto load = [&](const WeightsPlace &x, const int (&page)[GK], u32x4 (&raw)[GK][RAW], uint32_t (&byte)[GK], float (&old)[GK],
            uint32_t &hidden)
    {
        hidden = 0;
#pragma unroll
        for(int g = 0; g < GK; ++g)
        {
            const bool real = (unsigned)page[g] < (unsigned)p.c.n_pages;
            hidden |= real ? 0u : 1u << g;
            const int64_t pg = real ? page[g] : 0;
            const int64_t in_page = ((int64_t)x.h << p.c.page_shift) + (group_row(x, g) & ((1 << p.c.page_shift) - 1)) + col;
            const char *const from = p.c.k_pages + pg * p.c.page_stride + in_page * RB;
            if constexpr(RB < 64)
            {
                const u32x2 two = *reinterpret_cast<const u32x2 *>(from + 8 * quad);
                raw[g][0] = u32x4{two[0], two[1], 0, 0};
            }
            else
            {
#pragma unroll
                for(int i = 0; i < RAW; ++i)
                {
                    raw[g][i] = *reinterpret_cast<const u32x4 *>(from + 16 * (4 * i + quad));
                }
            }
            if constexpr(CODES)
            {
                constexpr int SB = KIND == kPaged4 ? HEAD / 32 : 1;
                byte[g] = p.c.k_scales[pg * p.c.scale_stride + in_page * SB + quad * SB / 4];
            }
            if(p.decay != 0.0f && quad == 0 && x.block * BLOCK + wave * KEYS + 16 * g + col < x.len)
            {
                old[g] = weights_at(x)[16 * g];
            }
        }
    };
    int page[GK];
    u32x4 raw[GK][RAW];
    uint32_t byte[GK] = {}, hidden = 0;
    float old[GK] = {};
    look_up(place, page);
    load(place, page, raw, byte, old, hidden);
    WeightsPlace next = left > 1 ? next_of(place) : place;
    look_up(next, page);

    // Query rows from row0 on into LDS, as many as fill blocks of rows.  True: one of them, or the query that fills the rest
    // up, counts nothing, whatever its scores are.
    auto stage = [&](const WeightsPlace &x, int row0) -> bool
    {
        const int rows = min(p.rows - row0, ROWS), staged_rows = (rows + 16 * BLOCKS - 1) / (16 * BLOCKS) * (16 * BLOCKS);
        const int pieces = staged_rows * PIECES;
        // Row r's place in lse (times head: in Q); of a row that is none: the pair's first, whose scores are numbers wherever
        // a row that counts has one (those of a row of zeros are NaN for a key with an infinity).
        auto place_of = [&](int r, int &tok, bool &ok)
        {
            const int rr = min(row0 + r, p.rows - 1), g = (int)p.by_seq.quotient((uint32_t)rr);
            tok = rr - g * p.q_seq;
            ok = r < rows && tok < x.given;
            return (x.n + (int64_t)p.c.n_batch * ((ok ? g : 0) + (int64_t)p.kv_group * x.h)) * p.q_seq + (ok ? tok : 0);
        };
        int my_tok;
        bool my_ok;
        const int64_t my_row = place_of(min(tid, staged_rows - 1), my_tok, my_ok);
        const float lse_there = p.lse[my_row], lse = my_ok ? lse_there : neg_inf();
        __syncthreads();        // the rows before these are done with
        // (several loads on their way at a time)
        constexpr int AT_ONCE = 4;
        for(int t0 = 0; t0 < pieces; t0 += 256 * AT_ONCE)
        {
            u32x4 v[AT_ONCE];
#pragma unroll
            for(int k = 0; k < AT_ONCE; ++k)
            {
                const int t = min(t0 + 256 * k + tid, pieces - 1);
                int tok;
                bool ok;
                const int64_t row = place_of(t / PIECES, tok, ok);
                v[k] = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(p.Q) + row * QB + t % PIECES * 16);
            }
#pragma unroll
            for(int k = 0; k < AT_ONCE; ++k)
            {
                const int t = t0 + 256 * k + tid, r = t / PIECES;
                if(t < pieces)
                {
                    *reinterpret_cast<u32x4 *>(q_rows + r * QB + swizzled(r, t % PIECES) * 16) = v[k];
                }
            }
        }
        if(tid < staged_rows)
        {
            off_of[tid] = lse == neg_inf() ? neg_inf() : -lse * kLog2e;
            last_of[tid] = lse == neg_inf() ? -1 : p.causal ? x.len - x.given + my_tok : x.len - 1;
        }
        return __syncthreads_or(lse_there == neg_inf());
    };
    bool staged = false;        // the pair's queries lie in LDS, all of them
    bool dead = false;
    for(;;)
    {
        // (the queries in front of the wait for the keys)
        if(!staged && p.rows <= ROWS && place.given > 0)
        {
            dead = stage(place, 0);
            staged = true;
        }
        // this block's operands
        u32x4 kf[GK][QREGS];
        float s_scale[GK], kept[GK];
        const uint32_t without = hidden;
        bool far = false;
        if constexpr(NARROW)
        {
            // (what lies in rows that are none has no say)
            const int rows_there = place.len - place.block * BLOCK - wave * KEYS;
#pragma unroll
            for(int g = 0; g < GK; ++g)
            {
                far = far || (16 * g + col < ((hidden >> g) & 1 ? 0 : rows_there) && byte[g] - (127u - 13u) > 26u);
            }
            far = __any(far);
        }
#pragma unroll
        for(int g = 0; g < GK; ++g)
        {
            const float scale = CODES ? __uint_as_float(byte[g] << 23) : 1.0f;
            s_scale[g] = KIND == kPaged8 && !__is_same(T, Bf16) ? scale : 1.0f;
            kept[g] = old[g];
#pragma unroll
            for(int i = 0; i < QREGS; ++i)
            {
                if constexpr(KIND == kPaged4)
                {
                    if(!NARROW || far)
                    {
                        kf[g][i] = widen8_of_4<Bf16>(raw[g][0][i], scale);
                    }
                    else
                    {
                        kf[g][i] = widen8_of_4<T>(raw[g][0][i], scale);
                    }
                }
                else if constexpr(KIND == kPaged8)
                {
                    const float of_codes = __is_same(T, Bf16) ? scale : 1.0f;
                    const u32x2 a = widen4<T>(raw[g][i / 2][2 * (i % 2)], of_codes),
                        b = widen4<T>(raw[g][i / 2][2 * (i % 2) + 1], of_codes);
                    kf[g][i] = u32x4{a[0], a[1], b[0], b[1]};
                }
                else
                {
                    kf[g][i] = raw[g][i];
                }
            }
        }
        // the next block's rows are on their way meanwhile
        const WeightsPlace now = place;
        if(left > 1)
        {
            load(next, page, raw, byte, old, hidden);
            place = next;
            if(left > 2)
            {
                next = next_of(next);
                look_up(next, page);
            }
        }
        const int key0 = now.block * BLOCK + wave * KEYS;
        const bool here = key0 < now.len;

        // scores of the rows from rb on
        auto scores = [&](int rb, f32x4 (&s)[BLOCKS][GK], auto two)
        {
            constexpr bool TWO = decltype(two)::value;
#pragma unroll
            for(int k = 0; k < BLOCKS; ++k)
            {
#pragma unroll
                for(int g = 0; g < GK; ++g)
                {
                    s[k][g] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
#pragma unroll
            for(int i = 0; i < QREGS; ++i)
            {
#pragma unroll
                for(int k = 0; k < BLOCKS; ++k)
                {
                    u32x4 q = *reinterpret_cast<const u32x4 *>(q_rows + (rb + 16 * k + col) * QB + swizzled(col, q_piece(i)) * 16);
                    u32x4 rest = q;
                    if constexpr(TWO)
                    {
                        two_bf16(q, q, rest);
                    }
#pragma unroll
                    for(int g = 0; g < GK; ++g)
                    {
                        if constexpr(KIND == kPaged32)
                        {
#pragma unroll
                            for(int e = 0; e < 4; ++e)
                            {
                                s[k][g] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(q[e]),
                                        __uint_as_float(kf[g][i][e]), s[k][g], 0, 0, 0);
                            }
                        }
                        else if constexpr(TWO)
                        {
                            s[k][g] = mfma32<Bf16>(q, kf[g][i], s[k][g]);
                            s[k][g] = mfma32<Bf16>(rest, kf[g][i], s[k][g]);
                        }
                        else
                        {
                            s[k][g] = mfma32<T>(q, kf[g][i], s[k][g]);
                        }
                    }
                }
            }
        };

        // ---- sums over the queries -------------------------------------------------------
        float sum[GK];
#pragma unroll
        for(int g = 0; g < GK; ++g)
        {
            sum[g] = 0.0f;
        }
        // below it every row sees every key
        const int all_see = p.causal ? now.len - now.given : now.len - 1;
        const bool partly = key0 + KEYS - 1 > all_see || without != 0;
        for(int row0 = 0; row0 < (now.given > 0 ? p.rows : 0); row0 += ROWS)
        {
            const int rows = min(p.rows - row0, ROWS);
            if(!staged)
            {
                dead = stage(now, row0);
                staged = p.rows <= ROWS;
            }
            if(!here)
            {
                continue;
            }
            for(int rb = 0; rb < rows; rb += 16 * BLOCKS)
            {
                f32x4 s[BLOCKS][GK];
                if(NARROW && far)
                {
                    scores(rb, s, std::bool_constant<NARROW>());
                }
                else
                {
                    scores(rb, s, std::false_type());
                }
                if(partly || dead)
                {
#pragma unroll
                    for(int k = 0; k < BLOCKS; ++k)
                    {
                        typedef __attribute__((ext_vector_type(4))) int i32x4;
                        const f32x4 off = *reinterpret_cast<const f32x4 *>(off_of + rb + 16 * k + 4 * quad);
                        const i32x4 last = *reinterpret_cast<const i32x4 *>(last_of + rb + 16 * k + 4 * quad);
#pragma unroll
                        for(int g = 0; g < GK; ++g)
                        {
#pragma unroll
                            for(int e = 0; e < 4; ++e)
                            {
                                const float x = fast_exp2(fmaf(s[k][g][e] * s_scale[g], c_log2, off[e]));
                                sum[g] += key0 + 16 * g + col <= ((without >> g) & 1 ? -1 : last[e]) ? x : 0.0f;
                            }
                        }
                    }
                }
                else
                {
#pragma unroll
                    for(int k = 0; k < BLOCKS; ++k)
                    {
                        const f32x4 off = *reinterpret_cast<const f32x4 *>(off_of + rb + 16 * k + 4 * quad);
#pragma unroll
                        for(int g = 0; g < GK; ++g)
                        {
                            const float c = KIND == kPaged8 ? c_log2 * s_scale[g] : c_log2;
#pragma unroll
                            for(int e = 0; e < 4; ++e)
                            {
                                sum[g] += fast_exp2(fmaf(s[k][g][e], c, off[e]));
                            }
                        }
                    }
                }
            }
        }
        if(here)
        {
            float *const to = weights_at(now);
#pragma unroll
            for(int g = 0; g < GK; ++g)
            {
                const float x = quad_sum(sum[g]);
                if(quad == 0 && key0 + 16 * g + col < now.len)
                {
                    to[16 * g] = p.decay == 0.0f ? x : fmaf(p.decay, kept[g], x);
                }
            }
        }
        if(--left == 0)
        {
            return;
        }
        staged = staged && place.n == now.n && place.h == now.h;
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
