// A wavefront's walk over its keys in pages of 4-bit codes: what a step of the attention over pages does there.
//
//  * A step is 64 keys: 16 bytes a lane of four rows of each of the four 16-key groups, so that a lane's group, and
//    page, is the same in all loads.  Addresses are the vector unit's, a lane's own: the scalar unit took a fifth of a
//    step's time for those of four groups.
//  * A key row's fourth is what a lane widens: 32 codes (head 128) with one power of two.  The four groups' sums are
//    formed side by side, since the products of one wait for each other.
//  * Values come through the transposing reads as codes, sixteen keys of a column, and their powers of two go into the
//    probabilities, for every 32 columns anew: as bf16 numbers those take them by an addition to their exponents.
//  * What bounds it is the issue of vector instructions, some 400 a step with one row block, 560 with two, beside what
//    a unit's begin and end take: 64 sequences of 17 to 16384 rows, 8 heads of 128, 4 query rows a head, bf16, 173 MB,
//    43.2 us = 4.0 TB/s (loads alone 37); 8 of 8192 rows, 64 query rows, 73 MB and 17 GFLOP, 40.7 us, of which 26 are the
//    issue of these instructions, 6 the beginning, 2 the wavefronts' results and 4 the join.  Probabilities widened in
//    fp32 and scalar addresses took 2.7 us more of the first and 0.6 less of the second.  Half the LDS, each half of a
//    step fetched as soon as it was read, and three workgroups a CU for it: 2.9 more.  Values widened row by row and
//    written back to LDS to be read transposed as bf16 numbers: 3.8 more.
#pragma once

#include <type_traits>

#include "sdpa_paged_shape.hpp"

namespace nntile_hip
{

// The segment's results of the lane's query rows: o unnormalised, m_run, l_run as the other kinds leave them.
// ring: the workgroup's LDS.  All wavefronts of the workgroup run it (there is a barrier).
template<typename T, int HEAD, int NR>
__device__ __forceinline__ void paged4_walk(const PagedAttendParams &p, const PagedSegment &seg, int h, int rg, int given,
        int my_first, int n_mine, int all_see, const int (&last)[NR], char *ring,
        f32x4 (&o)[NR][HEAD / 16], float (&m_run)[NR], float (&l_run)[NR])
{
    typedef PagedShape<kPaged4, HEAD, NR, 1> Shape;
    constexpr int RB = Shape::RB, SB = Shape::SB, CPR = Shape::CPR, KEYS = Shape::KEYS, GROUPS = Shape::GROUPS;
    constexpr int LOADS = Shape::LOADS, K_BYTES = Shape::K_BYTES, STREAMS = Shape::STREAMS, QROWS = Shape::QROWS, QB = Shape::QB;
    constexpr int DBLOCKS = HEAD / 16, QREGS = HEAD / 32;
    // Keys become numbers of the tile type exactly; where a query sees powers of two below 2^-13 or above 2^13 in a step, for
    // which fp16 has no exponents, bf16 numbers, and an fp16 query is the sum of two of them then (11 bits in 8 and 3, exactly).
    // Rows that it does not see have no say in that: they leave every bit of its result as it is.
    // (64 sequences of 2048 rows, 8 heads of 128, 32, 64 and 256 query rows 69, 132 and 512 us with sums of two always, 58,
    // 102 and 361 now; 8 of 8192, 32 query rows, 39.7 and 38.6.)
    // Probabilities of fp16 tiles are always the sum of two bf16 numbers (16 bits), with products of their own each.
    constexpr bool TWO = __is_same(T, Fp16);
    // Rows that another workgroup reads, too, may stay in the caches: 8 sequences of 8192 rows, 8 heads of 128, bf16, 32 and
    // 64 query rows 33.1 -> 31.6 and 42.4 -> 40.8 us (fp16, while it kept its addresses, 38.8 -> 40.3 and 62.2 -> 63.3:
    // not there).
    constexpr bool PAST_CACHES = NR == 1 || TWO;
    // With two row blocks of fp16 tiles addresses that follow from one by an exclusive or are formed where they are used: kept,
    // they are nine registers more than there are, and a reload waits for the loads on their way, too (64 sequences of 2048
    // rows, 8 heads of 128, 32 and 256 query rows 65 and 457 us kept, 53 and 367 formed; one row block or bf16, which have the
    // registers: 1 to 2 % slower formed).
    constexpr bool FORMED = TWO && NR == 2;
    constexpr int SLANES = GROUPS * SB;         // lanes that have the scale bytes of a step's keys, 16 each
    constexpr int STEP_LOADS = 2 * LOADS + 1;   // load instructions of a step
    const int tid = fresh(threadIdx.x), lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    constexpr int SCALES = 2 * KEYS * SB;       // of a step
    char *const slots = ring + wave * (2 * Shape::STAGE);
    char *const scale_slots = ring + STREAMS * 2 * Shape::STAGE + wave * (2 * SCALES);
    char *const q_rows = ring + STREAMS * 2 * (Shape::STAGE + SCALES);
    const float c_log2 = p.scale * kLog2e, slack = kPagedSlack / c_log2;

    // ---- pages and loads ----------------------------------------------------------------
    // Where a page holds a step, its groups lie behind each other in one page: one look-up.
    const int64_t table_row = (int64_t)seg.n * p.c.max_pages;
    const bool one_page = (1 << p.c.page_shift) >= KEYS;
    auto look_up = [&](int i, int (&page)[GROUPS])
    {
        const int row0 = my_first + i * Shape::BLOCK;
        page[0] = scalar_load<int>(p.c.table, 4 * (table_row + (row0 >> p.c.page_shift)));
        if(!one_page)
        {
#pragma unroll
            for(int g = 1; g < GROUPS; ++g)
            {
                // (groups behind the last row take the page of the last)
                const int row = min(row0 + 16 * g, seg.len - 1);
                page[g] = scalar_load<int>(p.c.table, 4 * (table_row + (row >> p.c.page_shift)));
            }
        }
    };
    // (a page that is none is read as page 0 and hidden)
    auto real_page = [&](int page) { return (unsigned)page < (unsigned)p.c.n_pages ? page : 0; };
    // The first row of group g, among those of its page's heads, and the page
    auto group_row = [&](int i, int g)
    {
        const int row = min(my_first + i * Shape::BLOCK + 16 * g, seg.len - 1) & ~15;
        return ((int64_t)h << p.c.page_shift) + (row & ((1 << p.c.page_shift) - 1));
    };
    auto group_page = [&](const int (&page)[GROUPS], int g)
    {
        int mine = real_page(page[0]);
        if(!one_page)
        {
#pragma unroll
            for(int j = 1; j < GROUPS; ++j)
            {
                mine = g == j ? real_page(page[j]) : mine;
            }
        }
        return mine;
    };
    // the lane's place in every load: row in its group, chunk
    uint32_t off[FORMED ? 1 : LOADS];
#pragma unroll
    for(int i = 0; i < (FORMED ? 1 : LOADS); ++i)
    {
        const int r = i * Shape::RPG + lane % 16 / CPR;
        off[i] = (uint32_t)(r * RB + ((lane ^ i ^ quad) & (CPR - 1)) * 16);
    }
    auto load_off = [&](uint32_t first, int i)
    {
        return FORMED ? (first ^ (uint32_t)((i & (CPR - 1)) * 16)) + (uint32_t)(i * Shape::RPG * RB) : off[FORMED ? 0 : i];
    };
    const uint8_t *const scales_of_lane = (lane < SLANES ? p.c.k_scales : p.c.v_scales) + 16 * (lane % SB);
    auto fetch = [&](int i, const int (&page)[GROUPS])
    {
        const int64_t from = group_page(page, quad) * p.c.page_stride + group_row(i, quad) * RB;
        const char *const k_from = p.c.k_pages + from, *const v_from = p.c.v_pages + from;
        char *const slot = slots + (i & 1) * Shape::STAGE;
        const uint32_t first = FORMED ? (uint32_t)fresh((int)off[0]) : 0;
#pragma unroll
        for(int ld = 0; ld < LOADS; ++ld)
        {
            load_to_lds16<0, PAST_CACHES>(k_from + load_off(first, ld), slot + ld * 1024);
        }
#pragma unroll
        for(int ld = 0; ld < LOADS; ++ld)
        {
            load_to_lds16<0, PAST_CACHES>(v_from + load_off(first, ld), slot + K_BYTES + ld * 1024);
        }
        const int g = lane % SLANES / SB;
        const uint8_t *const scale_from = scales_of_lane + group_page(page, g) * p.c.scale_stride + group_row(i, g) * SB;
        if(lane < 2 * SLANES)
        {
            load_to_lds16<0, false>(scale_from, scale_slots + (i & 1) * SCALES);
        }
    };
    int page[GROUPS], page_next[GROUPS];
    if(n_mine > 0)
    {
        look_up(0, page);
        fetch(0, page);
        look_up(min(1, n_mine - 1), page_next);
    }

    // ---- the query rows, of all wavefronts ---------------------------------------------------
    {
        constexpr int PIECES = QB / 16;
        for(int t = tid; t < QROWS * PIECES; t += Shape::THREADS)
        {
            const int r = t / PIECES, piece = t % PIECES, rr = rg * QROWS + r;
            u32x4 x = {0, 0, 0, 0};
            if(rr < p.rows && rr % p.q_seq < given)
            {
                x = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(p.Q)
                        + paged_query_row(p, seg.n, h, rr) * QB + piece * 16);
            }
            *reinterpret_cast<u32x4 *>(q_rows + r * QB + (piece ^ Shape::q_swizzle(r)) * 16) = x;
        }
        __syncthreads();
    }
    // a lane's operands begin at (head/4)*quad + 8i of its row
    auto q_operand = [&](int nr, int i)
    {
        return *reinterpret_cast<const u32x4 *>(q_rows + (nr * 16 + col) * QB
                + ((HEAD / 32 * quad + i) ^ Shape::q_swizzle(col)) * 16);
    };

    // the lane's addresses of a step's operands
    uint32_t k_at[FORMED ? 1 : GROUPS], v_at[FORMED ? 1 : CPR];
#pragma unroll
    for(int g = 0; g < (FORMED ? 1 : GROUPS); ++g)
    {
        k_at[g] = RB < 64 ? (uint32_t)(Shape::place4(16 * g + col, quad >> 1) + 8 * (quad & 1))
            : (uint32_t)Shape::place4(16 * g + col, quad);
    }
#pragma unroll
    for(int c = 0; c < (FORMED ? 1 : CPR); ++c)
    {
        // lane i of a quad gives the address of row i, sixteen values; rows 4g .. 4g + 3 are the 16-key group g's
        v_at[c] = (uint32_t)Shape::place4(16 * (col >> 2) + 4 * quad + (col & 3), c);
    }

    auto without_page = [&]()       // groups of the step
    {
        uint32_t hidden = (unsigned)page[0] < (unsigned)p.c.n_pages ? 0u : one_page ? ~0u : 1u;
        if(!one_page)
        {
#pragma unroll
            for(int g = 1; g < GROUPS; ++g)
            {
                hidden |= (unsigned)page[g] < (unsigned)p.c.n_pages ? 0u : 1u << g;
            }
        }
        return hidden;
    };
    // One step; PARTLY: some of its keys may be hidden from some row.
    auto take_step = [&](int i, auto partly)
    {
        constexpr bool PARTLY = decltype(partly)::value;
        const uint32_t hidden = PARTLY ? without_page() : 0;
        const int key0 = my_first + i * Shape::BLOCK;
        const char *const k_slot = slots + (i & 1) * Shape::STAGE, *const v_slot = k_slot + K_BYTES;
        const char *const k_scales = scale_slots + (i & 1) * SCALES, *const v_scales = k_scales + KEYS * SB;
        // the reads of the slot that is filled next have returned
        paged_wait_lds();
        if(i + 1 < n_mine)
        {
            fetch(i + 1, page_next);
#pragma unroll
            for(int g = 0; g < GROUPS; ++g)
            {
                page[g] = page_next[g];
            }
            look_up(min(i + 2, n_mine - 1), page_next);
            paged_wait_loads<STEP_LOADS>();
        }
        else
        {
            paged_wait_loads<0>();
        }
        // ---- scores ----------------------------------------------------------------------
        f32x4 s[NR][GROUPS];
        uint32_t codes[GROUPS][QREGS];
        float scale[GROUPS];
        const uint32_t k_first = FORMED ? (uint32_t)fresh((int)k_at[0]) : 0;
        // The first key of the step that bf16 numbers are taken for, among those that some query sees (where all queries see
        // all keys: 0 if there is one).
        int first_far = KEYS;
        bool far = false;
#pragma unroll
        for(int g = 0; g < GROUPS; ++g)
        {
            // the power of two of the lane's fourth of its key row
            const uint32_t byte = *reinterpret_cast<const uint8_t *>(k_scales + (16 * g + col) * SB + quad * SB / 4);
            scale[g] = __uint_as_float(byte << 23);
            const uint32_t k_at_g = FORMED ? (k_first ^ (uint32_t)((g & (CPR - 1)) * 16)) + 256u * g : k_at[FORMED ? 0 : g];
            far = far || (TWO && byte - (127u - 13u) > 26u);
#pragma unroll
            for(int i = 0; i < QREGS; ++i)
            {
                codes[g][i] = *reinterpret_cast<const uint32_t *>(k_slot + k_at_g + 4 * i);
            }
#pragma unroll
            for(int nr = 0; nr < NR; ++nr)
            {
                s[nr][g] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        if(TWO && __any(far))
        {
            first_far = PARTLY ? KEYS : 0;
            if constexpr(PARTLY)
            {
#pragma unroll
                for(int g = GROUPS - 1; g >= 0; --g)
                {
                    // (a key in each of 16 lanes, a fourth of it in each 16)
                    const bool there = key0 + 16 * g + col < seg.len && ((hidden >> g) & 1) == 0;
                    const unsigned long long lanes = __ballot(there && (__float_as_uint(scale[g]) >> 23) - (127u - 13u) > 26u);
                    const uint32_t half = (uint32_t)lanes | (uint32_t)(lanes >> 32), keys = (half | half >> 16) & 0xffffu;
                    first_far = keys != 0 ? 16 * g + __builtin_ctz(keys) : first_far;
                }
            }
        }
        // (the groups' sums side by side: a sum's products wait for each other)
        if(!TWO || first_far == KEYS)
        {
#pragma unroll
            for(int i = 0; i < QREGS; ++i)
            {
                u32x4 q[NR];
#pragma unroll
                for(int nr = 0; nr < NR; ++nr)
                {
                    q[nr] = q_operand(nr, i);
                }
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
                    const u32x4 wide = widen8_of_4<T>(codes[g][i], scale[g]);
#pragma unroll
                    for(int nr = 0; nr < NR; ++nr)
                    {
                        s[nr][g] = mfma32<T>(wide, q[nr], s[nr][g]);
                    }
                }
            }
        }
        else if constexpr(TWO)
        {
#pragma unroll
            for(int i = 0; i < QREGS; ++i)
            {
                u32x4 wide[GROUPS];
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
                    wide[g] = widen8_of_4<Bf16>(codes[g][i], scale[g]);
                }
#pragma unroll
                for(int nr = 0; nr < NR; ++nr)
                {
                    u32x4 q = q_operand(nr, i), rest;
                    two_bf16(q, q, rest);
#pragma unroll
                    for(int g = 0; g < GROUPS; ++g)
                    {
                        s[nr][g] = mfma32<Bf16>(wide[g], q, s[nr][g]);
                        s[nr][g] = mfma32<Bf16>(wide[g], rest, s[nr][g]);
                    }
                }
            }
            if constexpr(PARTLY)
            {
                // Queries that see only keys in front of it have the scores that they have without it.
#pragma unroll
                for(int nr = 0; nr < NR; ++nr)
                {
                    const bool sees = last[nr] - key0 >= first_far;
                    if(__all(sees))
                    {
                        continue;
                    }
#pragma unroll
                    for(int g = 0; g < GROUPS; ++g)
                    {
                        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for(int i = 0; i < QREGS; ++i)
                        {
                            x = mfma32<T>(widen8_of_4<T>((uint32_t)fresh((int)codes[g][i]), scale[g]), q_operand(nr, i), x);
                        }
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            s[nr][g][e] = sees ? s[nr][g][e] : x[e];
                        }
                    }
                }
            }
        }
        // ---- probabilities -----------------------------------------------------------------
        // (as of the other kinds of pages)
#pragma unroll
        for(int nr = 0; nr < NR; ++nr)
        {
            float top = neg_inf();
#pragma unroll
            for(int g = 0; g < GROUPS; ++g)
            {
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    if constexpr(PARTLY)
                    {
                        s[nr][g][e] = 4 * quad + e > ((hidden >> g) & 1 ? -1 : last[nr] - key0 - 16 * g) ? neg_inf() : s[nr][g][e];
                    }
                    top = fmaxf(top, s[nr][g][e]);
                }
            }
            top = quad_max(top);
            if(__any(top > m_run[nr] + slack))
            {
                const float m_new = top > m_run[nr] + slack ? top : m_run[nr];
                const float fade = fast_exp2(m_run[nr] * c_log2 - (m_new == neg_inf() ? 0.0f : m_new * c_log2));
                l_run[nr] *= fade;
                m_run[nr] = m_new;
#pragma unroll
                for(int db = 0; db < DBLOCKS; ++db)
                {
                    o[nr][db] *= fade;
                }
            }
            const float down = -kPagedSlack - (m_run[nr] == neg_inf() ? 0.0f : m_run[nr] * c_log2);
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for(int g = 0; g < GROUPS; ++g)
            {
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    s[nr][g][e] = fast_exp2(fmaf(s[nr][g][e], c_log2, down));
                    sum[e] += s[nr][g][e];
                }
            }
            l_run[nr] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }

        // ---- output --------------------------------------------------------------------------
        // the lane's column of every 16: codes of sixteen keys
        u32x2 v[DBLOCKS];
        const uint32_t v_first = FORMED ? (uint32_t)fresh((int)v_at[0]) : 0;
#pragma unroll
        for(int db = 0; db < DBLOCKS; ++db)
        {
            typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
            const uint32_t v_at_c = FORMED ? v_first ^ (uint32_t)(db / 2 * 16) : v_at[FORMED ? 0 : db / 2];
            v[db] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                        (lds_i32x2 *)(v_slot + v_at_c + 8 * (db & 1))));
        }
        // scale bytes of the lane's four value rows of each group
        uint32_t vs[GROUPS][SB];
#pragma unroll
        for(int g = 0; g < GROUPS; ++g)
        {
#pragma unroll
            for(int w = 0; w < SB; ++w)
            {
                vs[g][w] = *reinterpret_cast<const uint32_t *>(v_scales + (16 * g + 4 * quad) * SB + 4 * w);
            }
        }
        // probabilities as the matrix instruction takes them: for TWO the first 8 bits as they are, the next 8 rounded
        auto narrow = [&](const f32x4 &x, uint32_t (&first)[2], uint32_t (&more)[2])
        {
            if constexpr(TWO)
            {
                const u32x4 bits = __builtin_bit_cast(u32x4, x);
                const f32x4 rest = x - __builtin_bit_cast(f32x4, bits & 0xffff0000u);
                first[0] = __builtin_amdgcn_perm(bits[1], bits[0], 0x07060302u);
                first[1] = __builtin_amdgcn_perm(bits[3], bits[2], 0x07060302u);
                more[0] = Bf16::pack2(rest[0], rest[1]);
                more[1] = Bf16::pack2(rest[2], rest[3]);
            }
            else
            {
                first[0] = Bf16::pack2(x[0], x[1]);
                first[1] = Bf16::pack2(x[2], x[3]);
            }
        };
        constexpr int NT = TWO ? NR : 1, GT = TWO ? GROUPS : 1;
        // products of 32 columns, b, with probabilities that have their powers of two
        auto columns = [&](int b, const uint32_t (&first)[NR][GROUPS][2], const uint32_t (&rest)[NT][GT][2])
        {
#pragma unroll
            for(int t = 0; t < GROUPS / 2; ++t)
            {
#pragma unroll
                for(int db = 2 * b; db < 2 * b + 2; ++db)
                {
                    // (widened here, not once for both ways of this step, in front of them)
                    const u32x4 w = widen8_of_4<Bf16>((uint32_t)fresh((int)v[db][t]), 1.0f);
#pragma unroll
                    for(int nr = 0; nr < NR; ++nr)
                    {
                        o[nr][db] = mfma32<Bf16>(w, u32x4{first[nr][2 * t][0], first[nr][2 * t][1],
                                first[nr][2 * t + 1][0], first[nr][2 * t + 1][1]}, o[nr][db]);
                        if constexpr(TWO)
                        {
                            o[nr][db] = mfma32<Bf16>(w, u32x4{rest[nr][2 * t][0], rest[nr][2 * t][1],
                                    rest[nr][2 * t + 1][0], rest[nr][2 * t + 1][1]}, o[nr][db]);
                        }
                    }
                }
            }
        };
        // A power of two that is that of NaN, or 2^65 and more?
        bool odd = false;
        if constexpr(!PARTLY)
        {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(v_scales + 4 * (lane % (16 * SB)));
            odd = __any((w & w << 1 & 0x80808080u) != 0);
        }
        if(!PARTLY && !odd)
        {
            // As bf16 numbers probabilities take a power of two by an addition to their exponents (what falls below the
            // smallest number becomes 0; a probability of 0 counts as 2^-127, 2^-119 of the sum: of values up to
            // 6 * 2^64 that is 2^-52).
            uint32_t pw[NR][GROUPS][2], pw_rest[NT][GT][2];
#pragma unroll
            for(int nr = 0; nr < NR; ++nr)
            {
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
                    narrow(s[nr][g], pw[nr][g], pw_rest[TWO ? nr : 0][TWO ? g : 0]);
#pragma unroll
                    for(int e2 = 0; e2 < 2; ++e2)
                    {
                        pw[nr][g][e2] = lower_exponents(pw[nr][g][e2]);
                        if constexpr(TWO)
                        {
                            pw_rest[nr][g][e2] = lower_exponents(pw_rest[nr][g][e2]);
                        }
                    }
                }
            }
#pragma unroll
            for(int b = 0; b < SB; ++b)
            {
                uint32_t first[NR][GROUPS][2], rest[NT][GT][2];
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
#pragma unroll
                    for(int e2 = 0; e2 < 2; ++e2)
                    {
                        // byte b of two keys as 16-bit integers
                        const uint32_t two = SB == 4
                            ? __builtin_amdgcn_perm(vs[g][2 * e2 + (SB == 4 ? 1 : 0)], vs[g][2 * e2 % SB],
                                    0x0c040c00u + 0x00010001u * (uint32_t)b)
                            : __builtin_amdgcn_perm(0u, vs[g][e2], 0x0c020c00u + 0x00010001u * (uint32_t)b);
#pragma unroll
                        for(int nr = 0; nr < NR; ++nr)
                        {
                            first[nr][g][e2] = add_exponents(pw[nr][g][e2], two);
                            if constexpr(TWO)
                            {
                                rest[nr][g][e2] = add_exponents(pw_rest[nr][g][e2], two);
                            }
                        }
                    }
                }
                columns(b, first, rest);
            }
        }
        else
        {
            // Probabilities that have to be exactly 0, of rows that are hidden or none or whose values are that large, and
            // powers of two that are those of NaN: the product in fp32.
#pragma unroll
            for(int b = 0; b < SB; ++b)
            {
                uint32_t first[NR][GROUPS][2], rest[NT][GT][2];
#pragma unroll
                for(int nr = 0; nr < NR; ++nr)
                {
#pragma unroll
                    for(int g = 0; g < GROUPS; ++g)
                    {
                        f32x4 x;
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            x[e] = s[nr][g][e] * scale_of(vs[g][e * SB / 4], (e * SB + b) % 4);
                            if constexpr(PARTLY)
                            {
                                // (whatever the power of two of a row that is not seen, also none)
                                x[e] = 4 * quad + e > ((hidden >> g) & 1 ? -1 : last[nr] - key0 - 16 * g) ? 0.0f : x[e];
                            }
                        }
                        narrow(x, first[nr][g], rest[TWO ? nr : 0][TWO ? g : 0]);
                    }
                }
                columns(b, first, rest);
            }
        }
    };
    // (the steps without hidden keys on their own: two forms behind each other cost fewer registers than a choice
    // between them)
    int i = 0;
    for(; i < n_mine && my_first + i * Shape::BLOCK + KEYS - 1 <= all_see && without_page() == 0; ++i)
    {
        take_step(i, std::false_type());
    }
    for(; i < n_mine; ++i)
    {
        take_step(i, std::true_type());
    }
}

} // namespace nntile_hip
