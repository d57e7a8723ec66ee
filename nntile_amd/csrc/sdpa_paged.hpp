// Attention of a few new tokens per sequence over a key/value cache in pages, for sequences of
// any lengths, gfx950.  With s = q.k / sqrt(head) over the keys a query sees:
//
//   lse = log sum exp(s),   A = sum exp(s - lse) v
//
// merged into the running pair (lse, A) or written over it.  Bound by the one pass over
// the keys and values in HBM.
//
//  * The kv_group query heads of a key/value head are taken together, rows = kv_group * q_seq in blocks
//    of 16: one or two of them a wavefront, up to four a workgroup (more rows: several workgroups read the
//    keys, each up to the last one that its rows see, on one XCD, so that all but the first read them from its L2).
//  * The keys of a sequence are cut into blocks of 4 * KEYS, the blocks of all (sequence, head, row
//    group) units are numbered through, and every workgroup takes an equal run of them, whatever the
//    lengths: it finds its first unit by a scan of the lengths (they live on the device, so a captured
//    launch follows them).  Equally long units are cut into whole shares instead, where that is as even.
//  * Units that lie within one workgroup are finished there.  Of the others every share leaves its
//    result (unnormalised output, maximum, sum, all fp32) and counts itself done; the one that counts
//    last joins them in the order of the keys.  Nobody waits, so it does not matter which workgroups run
//    at once, and the same call gives the same bits.  (A second launch for it cost 6 us.)
//  * A wavefront streams KEYS keys at a time, its own ones, through its own two slots of LDS
//    (global_load_lds, 16 bytes a lane): no barrier within a unit, 8 KB in flight per wavefront while
//    8 KB are worked on, eight wavefronts a CU.  The pages of the next keys are looked up by scalar
//    loads meanwhile.  More than 32 rows: two wavefronts share the keys, one loads K and one V.
//  * S^T = K Q^T and O^T += V^T P^T with matrix instructions of 16 x 16; P^T is the accumulator of
//    S^T as it stands (the keys of an instruction are numbered so), V^T comes through the transposing
//    LDS reads (fp32: single values).  A lane has one query row.
//    What bounds 64 rows is the issue of the softmax's vector instructions.
//  * 8-bit pages: codes become values of the tile type exactly in front of the matrix instructions.
//    The power of two of a key row goes into its codes (bf16) or into the score (fp16), that of a value
//    row into the probability: as a bf16 number over bf16 tiles, as the sum of two over fp16 tiles, so that it
//    has fp32's exponents and more bits than fp16, whatever the powers of two of other rows are.
//
// What it reaches, 8 heads of 128, bytes of the cache alone: 64 sequences of 1024 bf16 rows, 4 query rows a
// head 5.9 TB/s, 32 rows 5.7, 64 rows 4.4; 64 of 2048 8-bit rows (bf16) 5.8, 5.2 and 3.5.  8 of 8192 bf16 rows, 64
// query rows, 270 MB: 54.7 us = 4.9 TB/s.  A single sequence of 1001 rows, 4 MB: 8.7 us, the chain from
// the lengths over the table and the keys to the join, a memory latency each.
//
// Probabilities of 16-bit tiles are rounded for the matrix instruction, as in the other attention kernels: to
// the tile type, over 8-bit pages of fp16 to 16 bits.  The sum of the softmax takes them unrounded.
#pragma once

#include <type_traits>

#include "sdpa_paged4_walk.hpp"

namespace nntile_hip
{

// Whether a word of a page - two 16-bit values, four codes or an fp32 value - holds a NaN or an infinity
template<typename T, int KIND> __device__ __forceinline__ bool not_numbers(uint32_t w)
{
    if constexpr(KIND == kPaged32)
    {
        return (w & 0x7f800000u) == 0x7f800000u;
    }
    else if constexpr(KIND == kPaged8)
    {
        // a code of all ones behind its sign: adding 1 to it carries into the sign's place
        return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
    }
    else
    {
        constexpr uint32_t E = __is_same(T, Bf16) ? 0x7f80u : 0x7c00u;
        return (w & E) == E || ((w >> 16) & E) == E;
    }
}

// Partial results go from one workgroup to another of the same launch, on any XCD: stores and
// loads that the device serves, not a CU's or an XCD's own cache.
__device__ __forceinline__ void put2(float *to, f32x2 v)
{
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(to), __builtin_bit_cast(unsigned long long, v),
            __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ f32x2 get2(const float *from)
{
    return __builtin_bit_cast(f32x2, __hip_atomic_load(
                reinterpret_cast<unsigned long long *>(const_cast<float *>(from)), __ATOMIC_RELAXED,
                __HIP_MEMORY_SCOPE_AGENT));
}

// The folded row of a unit: (m, l) in log2 units, v unnormalised; into the running pair.
// TPR threads a row, thread t of them with the value pairs 2 * (t + TPR * k), so that neighbours' accesses lie
// side by side.  The threads of a row run in one wavefront, in lock step: every one has read lse before the
// first writes it.
template<typename T, int TPR, int PAIRS>
__device__ __forceinline__ void paged_finish_row(const PagedAttendParams &p, int64_t row, int t, float m, float l,
        const f32x2 (&o)[PAIRS])
{
    constexpr int HEAD = 2 * TPR * PAIRS;
    const bool none = m == neg_inf() && l == 0.0f;
    float lse_out = neg_inf(), w_old = 0.0f, sc = 0.0f;
    if(none)
    {
        if(!p.overwrite)
        {
            return;
        }
    }
    else
    {
        const float lse_new = (m == neg_inf() ? 0.0f : m) * kLn2 + __builtin_amdgcn_logf(l) * kLn2;
        float w_new;
        merge_weights(p.overwrite ? neg_inf() : p.lse[row], lse_new, w_old, w_new, lse_out);
        sc = w_new / l;
    }
#pragma unroll
    for(int k = 0; k < PAIRS; ++k)
    {
        f32x2 v = none ? f32x2{0.0f, 0.0f} : o[k] * sc;
        const int64_t at = row * HEAD + 2 * (t + TPR * k);
        if constexpr(__is_same(T, float))
        {
            f32x2 *dst = reinterpret_cast<f32x2 *>(static_cast<float *>(p.A) + at);
            if(w_old != 0.0f)
            {
                v += w_old * *dst;
            }
            *dst = v;
        }
        else
        {
            uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.A) + at);
            if(w_old != 0.0f)
            {
                const uint32_t old = *dst;
                v[0] += w_old * T::to_float((uint16_t)(old & 0xffffu));
                v[1] += w_old * T::to_float((uint16_t)(old >> 16));
            }
            *dst = T::pack2(v[0], v[1]);
        }
    }
    if(t == 0)
    {
        p.lse[row] = lse_out;
    }
}

// Joins the shares w0 .. w0 + parts - 1 of a unit, in this order, and finishes its rows.
// HEAD/4 threads a row; where the rows leave threads over, they take turns at the
// shares and the sums are added up through LDS.  A thread has PARTS shares of LINES rows on their way
// at a time: the round trips are what the join costs.
template<typename T, int HEAD, int THREADS, int QROWS, int PARTS, int LINES>
__device__ __forceinline__ void paged_join_by(const PagedAttendParams &p, int n, int h, int rg, int rows_here,
        int w0, int parts, float *lds, int tid)
{
    constexpr int TPR = HEAD / 4, ROWS = THREADS / TPR;
    int turns = 1;
    while(2 * turns * rows_here <= ROWS && 2 * turns <= parts)
    {
        turns *= 2;
    }
    const int t = tid % TPR, slot = tid / TPR;      // pairs 2t and 2t + HEAD/2 of the row
    const int turn = slot % turns, step = ROWS / turns;
    // (with more than one turn all rows fit beside each other: one round of one line)
    for(int r0 = slot / turns; r0 - slot / turns < rows_here; r0 += LINES * step)
    {
        float top[LINES], sum[LINES];
        f32x2 v[LINES][2];
#pragma unroll
        for(int k = 0; k < LINES; ++k)
        {
            top[k] = neg_inf();
            sum[k] = 0.0f;
            v[k][0] = v[k][1] = f32x2{0.0f, 0.0f};
        }
        for(int i0 = turn; i0 < parts; i0 += PARTS * turns)
        {
            f32x2 ml[LINES][PARTS], x[LINES][PARTS][2];
#pragma unroll
            for(int k = 0; k < LINES; ++k)
            {
#pragma unroll
                for(int j = 0; j < PARTS; ++j)
                {
                    // (behind the last share or row: it again, with no weight)
                    const int i = min(i0 + j * turns, parts - 1);
                    const int r = min(r0 + k * step, rows_here - 1);
                    const int64_t place = ((int64_t)(w0 + i) * 2 + (i == 0 ? 1 : 0)) * QROWS + r;
                    ml[k][j] = get2(p.part_ml + 2 * place);
                    x[k][j][0] = get2(p.part_o + place * HEAD + 2 * t);
                    x[k][j][1] = get2(p.part_o + place * HEAD + 2 * t + HEAD / 2);
                }
            }
#pragma unroll
            for(int k = 0; k < LINES; ++k)
            {
                float next = top[k];
#pragma unroll
                for(int j = 0; j < PARTS; ++j)
                {
                    next = i0 + j * turns < parts ? fmaxf(next, ml[k][j][0]) : next;
                }
                const float safe = next == neg_inf() ? 0.0f : next;
                const float old = fast_exp2(top[k] - safe);
                sum[k] *= old;
                v[k][0] *= old;
                v[k][1] *= old;
#pragma unroll
                for(int j = 0; j < PARTS; ++j)
                {
                    if(i0 + j * turns < parts)
                    {
                        const float f = fast_exp2(ml[k][j][0] - safe);
                        sum[k] += ml[k][j][1] * f;
                        v[k][0] += x[k][j][0] * f;
                        v[k][1] += x[k][j][1] * f;
                    }
                }
                top[k] = next;
            }
        }
        if(turns > 1)
        {
            float *const at = lds + slot * (HEAD + 4);
            *reinterpret_cast<f32x2 *>(at + 2 * t) = v[0][0];
            *reinterpret_cast<f32x2 *>(at + 2 * t + HEAD / 2) = v[0][1];
            if(t == 0)
            {
                at[HEAD] = top[0];
                at[HEAD + 1] = sum[0];
            }
            __syncthreads();
            if(turn == 0 && r0 < rows_here)
            {
                float next = neg_inf();
                for(int j = 0; j < turns; ++j)
                {
                    next = fmaxf(next, at[j * (HEAD + 4) + HEAD]);
                }
                const float safe = next == neg_inf() ? 0.0f : next;
                sum[0] = 0.0f;
                v[0][0] = v[0][1] = f32x2{0.0f, 0.0f};
                for(int j = 0; j < turns; ++j)
                {
                    const float *const of = at + j * (HEAD + 4);
                    const float f = fast_exp2(of[HEAD] - safe);
                    sum[0] += f * of[HEAD + 1];
                    v[0][0] += f * *reinterpret_cast<const f32x2 *>(of + 2 * t);
                    v[0][1] += f * *reinterpret_cast<const f32x2 *>(of + 2 * t + HEAD / 2);
                }
                top[0] = next;
            }
        }
#pragma unroll
        for(int k = 0; k < LINES; ++k)
        {
            const int r = r0 + k * step;
            if(turn == 0 && r < rows_here)
            {
                paged_finish_row<T, TPR, 2>(p, paged_query_row(p, n, h, rg * QROWS + r), t, top[k], sum[k], v[k]);
            }
        }
    }
}

template<typename T, int HEAD, int THREADS, int QROWS>
__device__ __forceinline__ void paged_join(const PagedAttendParams &p, int n, int h, int rg, int rows_here,
        int w0, int parts, float *lds, int tid)
{
    if(rows_here > THREADS / (HEAD / 4) && parts <= 4)
    {
        paged_join_by<T, HEAD, THREADS, QROWS, 4, 4>(p, n, h, rg, rows_here, w0, parts, lds, tid);
    }
    else if(rows_here > THREADS / (HEAD / 4))
    {
        paged_join_by<T, HEAD, THREADS, QROWS, 8, 2>(p, n, h, rg, rows_here, w0, parts, lds, tid);
    }
    else
    {
        paged_join_by<T, HEAD, THREADS, QROWS, 8, 1>(p, n, h, rg, rows_here, w0, parts, lds, tid);
    }
}

template<typename T, int KIND, int HEAD, int NR, int HALVES>
__global__ __launch_bounds__((PagedShape<KIND, HEAD, NR, HALVES>::THREADS), (PagedShape<KIND, HEAD, NR, HALVES>::MIN_WAVES))
void sdpa_paged_kernel(const PagedAttendParams p)
{
    typedef PagedShape<KIND, HEAD, NR, HALVES> Shape;
    constexpr int RB = Shape::RB, CPR = Shape::CPR, KEYS = Shape::KEYS, GROUPS = Shape::GROUPS;
    constexpr int LOADS = Shape::LOADS, K_BYTES = Shape::K_BYTES, STAGE = Shape::STAGE;
    constexpr int WAVES = Shape::WAVES, STREAMS = Shape::STREAMS, THREADS = Shape::THREADS;
    constexpr int DBLOCKS = HEAD / 16;
    // registers of a row block's query operand: 16 bytes each
    constexpr int QREGS = KIND == kPaged32 ? HEAD / 16 : HEAD / 32;
    constexpr int QROWS = Shape::QROWS;
    constexpr bool Q_IN_LDS = NR > 1 && KIND != kPaged4;
    // the type of the probabilities and values as the matrix instruction takes them (fp32 pages: neither)
    typedef typename std::conditional<KIND == kPaged16, T, Bf16>::type PV;
    // 8-bit pages: the scale of a key row goes into its codes (exact in bf16; fp16 has not the range: into the
    // scores), that of a value row into its probabilities, which are bf16 numbers then and the codes exact in
    // bf16.  For fp16 tiles 8 bits are too few: what the first number leaves of a probability is a second one,
    // with products of its own (64 of 2048 rows, 8 heads of 128: 47 us with 4 query rows, 55 with 32, 94 with 64;
    // as one fp16 number against the largest power of two so far 47, 54 and 84, but then a row that is not seen, or
    // has no weight, takes the bits of smaller ones).
    constexpr bool KSCALE_IN_CODES = KIND == kPaged8 && __is_same(T, Bf16);
    constexpr bool TWO_PARTS = KIND == kPaged8 && __is_same(T, Fp16);
    // the power of two that the probabilities, and so their sum, carry: where they have fp32's exponents, they
    // stay below 1, so that products with the largest values do not overflow
    constexpr float kLift = KIND == kPaged16 && __is_same(T, Fp16) ? kPagedLift : -kPagedSlack;

    constexpr int MERGE_LD = HEAD + 4;
    static_assert(STREAMS * 16 * HALVES * (MERGE_LD + 2) * 4 <= Shape::RING,
            "the wavefronts' results of a row block share the ring");
    constexpr int JOIN_ROWS = THREADS / (HEAD / 4);     // rows that are joined at a time
    static_assert(JOIN_ROWS * (HEAD + 4) * 4 <= Shape::RING, "... and so do the shares' sums");
    __shared__ __attribute__((aligned(1024))) char ring[Shape::RING];
    __shared__ __attribute__((aligned(16))) char q_rows[KIND == kPaged4 ? 16 : Shape::Q_BYTES];
    // 8-bit pages: the scale bytes of a wavefront's step and of the next, keys' and values'
    __shared__ __attribute__((aligned(16))) char scale_bytes[KIND == kPaged8 ? WAVES * 2 * 2 * KEYS : 16];
    __shared__ int scan_of[THREADS], wave_sum[WAVES], found;

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    // Up to 64 rows: two wavefronts read the same keys at about the same time, the second
    // through the L2, for 32 rows each (one with all 64 has too few registers).
    const int stream = wave % STREAMS, half = wave / STREAMS;

    // ---- the workgroup's run of key blocks ----------------------------------------
    // A scan over the sequences' blocks; every lane adds up a few neighbouring sequences.  A unit counts
    // as a block more than it has: its begin and end cost about as much (64 sequences of 17 to 16384
    // 8-bit rows 82 -> 73 us).  Where all sequences have as many blocks it does not, so that
    // shares and units end together.  Up to 64 sequences every wavefront scans for itself,
    // without LDS and barriers.
    const bool in_wave = p.c.n_batch <= 64;
    const int scanner = in_wave ? lane : tid, scanners = in_wave ? 64 : THREADS;
    const int chunk = (p.c.n_batch + scanners - 1) / scanners;
    const int n_lo = min(scanner * chunk, p.c.n_batch), n_hi = min(n_lo + chunk, p.c.n_batch);
    auto blocks_of_rows = [&](int rows) { return (rows + Shape::BLOCK - 1) / Shape::BLOCK; };
    // Up to 64 sequences: a lane has one's length and new tokens, for whoever asks later.
    int len_of_lane = 0, given_of_lane = 0;
    if(in_wave && lane < p.c.n_batch)
    {
        len_of_lane = paged_len(p.c, lane);
        given_of_lane = paged_new(p.c, lane, p.q_seq);
    }
    auto len_of = [&](int n)
    {
        return in_wave ? __builtin_amdgcn_readlane(len_of_lane, n) : uniform(paged_len(p.c, n));
    };
    int unit_cost = kPagedUnitCost;
    auto cost_of = [&](int blocks) { return blocks == 0 ? 0 : blocks + unit_cost; };
    const int blocks_0 = blocks_of_rows(len_of(0));
    int mine = 0;
    bool same = true;
    if(in_wave)
    {
        const int b = blocks_of_rows(len_of_lane);
        mine = cost_of(b);
        same = lane >= p.c.n_batch || b == blocks_0;
    }
    else
    {
        for(int n = n_lo; n < n_hi; ++n)
        {
            const int b = blocks_of_rows(paged_len(p.c, n));
            mine += cost_of(b);
            same = same && b == blocks_0;
        }
    }
    same = __all(same);
    int upto = (int)wave_scan((uint32_t)mine);
    int total = __builtin_amdgcn_readlane(upto, 63);
    if(!in_wave)
    {
        if(lane == 63)
        {
            wave_sum[wave] = same ? upto : ~upto;
        }
        __syncthreads();
        total = 0;
#pragma unroll
        for(int w = 0; w < WAVES; ++w)
        {
            const int sum = uniform(wave_sum[w]);
            same = same && sum >= 0;
            upto += w < wave ? (sum < 0 ? ~sum : sum) : 0;
            total += sum < 0 ? ~sum : sum;
        }
    }
    int in_front = upto - mine;         // of the lane's first sequence
    if(same)
    {
        unit_cost = 0;
        total = p.c.n_batch * blocks_0;
        in_front = n_lo * blocks_0;
    }
    const uint32_t all = (uint32_t)total * (uint32_t)p.units;
    // Where all units are equally long and not more than the workgroups, every unit gets shares of its own, as
    // few as keep the longest as short as it can be (four sequences of 1024 fp32 rows, 48 units, 15.9 -> 13.5
    // us); else an even run of blocks is a share.  (Shares of whole units for unequal lengths as well, where
    // that made the longest no more than two blocks longer: 16 of 500 to 8000 rows 38.0 -> 39.1 us.)
    const uint32_t n_units = (uint32_t)p.c.n_batch * (uint32_t)p.units;
    // The workgroup that joins a unit reads `rows` sums of `head` from every share, alone, while a share
    // reads its part of the keys: with more shares than about sqrt(keys / rows) a unit the join costs more
    // than the shorter shares save (one sequence, 8 units, of 4096 16-bit rows, 64 query rows 42.7 us with 32
    // shares a unit, 26.7 with 8; 4 query rows 16.5 and 11.7).
    const float keys = (float)all / (float)n_units * (float)Shape::BLOCK;
    const float most = fmaxf(sqrtf(keys / (float)min(p.rows, QROWS)), 1.0f);
    const uint32_t places = (uint32_t)uniform((int)fminf((float)p.shares, (float)n_units * most));
    // Equal units whose steps wait for memory more than for instructions: a workgroup a CU, where that leaves
    // none of eight CUs without one (8 heads of 128; 16-bit pages, 32 sequences of 1024, 32 query rows 34.2 ->
    // 28.0 us, 4 query rows 27.8 -> 25.6, but 20 sequences of 2000, 160 units, 33.4 -> 40.2; 8-bit pages, 32
    // query rows 26.4 -> 20.9, 4 query rows over 2048 30.4 -> 36.0).  32 query rows over 16-bit pages are better
    // off in any case (those 160 units 40.7 -> 36.3), unequal units in none (64 of 17 to 8192, 32 query rows
    // 99 -> 137).
    // 4-bit pages, whose joins weigh more beside their keys: where a share of two workgroups a CU has two blocks at most,
    // any rows (8 heads; of 128, 32 of 1024 rows, 4, 16 and 32 query rows 14.5, 15.6, 23.5 -> 12.7, 12.8, 17.9, 4 of 2048, 64
    // query rows 20.7 -> 16.3, of 8192, 4 and 16 query rows 14.5, 19.9 -> 15.0, 16.3; of 64, 32 of 1024, 4 query rows 12.3 ->
    // 9.8), not with more (8 of 8192, 64 query rows 40.7 -> 45.8).
    constexpr bool ONE_A_CU = KIND == kPaged16 || (KIND == kPaged8 && NR == 2);
    const bool one_a_cu = KIND == kPaged4 ? all <= 2 * (uint32_t)p.shares : ONE_A_CU && p.row_groups == 1;
    const uint32_t cus_filled = n_units <= kPagedCUs ? kPagedCUs / n_units * n_units : 0;
    const uint32_t equal_places = one_a_cu
        && (8 * cus_filled >= 7 * kPagedCUs || (KIND == kPaged16 && NR == 2 && cus_filled != 0))
        ? min(places, (uint32_t)kPagedCUs) : places;
    const bool aligned = same && n_units <= equal_places && blocks_0 != 0;
    uint32_t of_unit = 1;
    if(aligned)
    {
        const uint32_t each = equal_places / n_units, longest = ((uint32_t)blocks_0 + each - 1) / each;
        of_unit = ((uint32_t)blocks_0 + longest - 1) / longest;
    }
    const uint32_t shares = aligned ? n_units * of_unit : min(places, all);
    const PagedSplit split(all, shares);
    // sequences without rows: shared out, too, for the rows of their queries, some at a time
    if(p.overwrite && !(same && blocks_0 != 0))
    {
        constexpr int SIDE_BY_SIDE = THREADS / (HEAD / 4), PIECE = 8 * SIDE_BY_SIDE;
        const int rows = p.c.n_head_kv * p.rows, pieces = (rows - 1) / PIECE + 1;
        for(uint32_t piece = blockIdx.x; piece < (uint32_t)p.c.n_batch * (uint32_t)pieces; piece += gridDim.x)
        {
            const int n = (int)(piece / (uint32_t)pieces);
            if(len_of(n) == 0)
            {
                const int first = (int)(piece - (uint32_t)n * (uint32_t)pieces) * PIECE;
                const int here = min(rows - first, PIECE);
                for(int k = tid / (HEAD / 4); k < here; k += SIDE_BY_SIDE)
                {
                    const f32x2 zero[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
                    paged_finish_row<T, HEAD / 4, 2>(p, paged_query_row(p, n, (first + k) / p.rows,
                                (first + k) % p.rows), tid % (HEAD / 4), neg_inf(), 0.0f, zero);
                }
            }
        }
    }
    if(blockIdx.x >= shares)
    {
        return;
    }
    // The workgroup's share.  Where a head's row groups read the same keys, neighbouring shares go to workgroups of equal
    // index modulo 8, to one XCD and its L2.
    uint32_t me = blockIdx.x;
    if(p.row_groups > 1 && me < (shares & ~7u))
    {
        me = me % 8 * (shares / 8) + me / 8;
    }
    uint32_t at = split.begin(me);
    const uint32_t end = split.begin(me + 1);
    PagedSegment seg;
    uint32_t first_share = me;
    if(aligned)
    {
        const uint32_t unit = me / of_unit, part = me - unit * of_unit;
        const PagedSplit of_blocks((uint32_t)blocks_0, of_unit);
        first_share = me - part;
        seg.n = (int)(unit / (uint32_t)p.units);
        seg.u = (int)(unit - (uint32_t)seg.n * (uint32_t)p.units);
        seg.len = len_of(seg.n);
        seg.blocks = blocks_0;
        seg.step = (int)of_blocks.begin(part);
        seg.steps = (int)of_blocks.begin(part + 1) - seg.step;
    }
    else
    {
        // the last lane whose sequences begin at or before the block, then sequence by sequence
        const int block = (int)(at / (uint32_t)p.units);
        int t, before;
        if(in_wave)
        {
            t = __popcll(__ballot(scanner * chunk < p.c.n_batch && in_front <= block)) - 1;
            before = __builtin_amdgcn_readlane(in_front, t);
        }
        else
        {
            scan_of[tid] = in_front;
            __syncthreads();
            const bool here = tid * chunk < p.c.n_batch && in_front <= block
                && (tid == THREADS - 1 || (tid + 1) * chunk >= p.c.n_batch || scan_of[tid + 1] > block);
            if(here)
            {
                found = tid;
            }
            __syncthreads();
            t = uniform(found);
            before = uniform(scan_of[t]);
        }
        seg.n = t * chunk;
        for(;;)
        {
            seg.len = len_of(seg.n);
            seg.blocks = (seg.len + Shape::BLOCK - 1) / Shape::BLOCK;
            if(before + cost_of(seg.blocks) > block || seg.n + 1 >= p.c.n_batch)
            {
                break;
            }
            before += cost_of(seg.blocks);
            ++seg.n;
        }
        const uint32_t rest = at - (uint32_t)before * (uint32_t)p.units;
        seg.u = uniform((int)(rest / (uint32_t)cost_of(seg.blocks)));
        seg.step = uniform((int)(rest % (uint32_t)cost_of(seg.blocks)));
    }
    uint32_t unit_begin = at - (uint32_t)seg.step;      // of the unit's first block among all

    char *const slots = ring + stream * 2 * STAGE;
    // lane's place in every load instruction: row of the 16-row group, chunk.  Of two wavefronts that
    // share their keys, one loads K and one V.
    constexpr bool PAIRED = HALVES == 2;
    uint32_t k_off[LOADS], v_off[PAIRED ? 1 : LOADS];
#pragma unroll
    for(int i = 0; i < LOADS; ++i)
    {
        const int r = i * Shape::ROWS_PER_LOAD + lane / CPR;
        const int k_swizzle = PAIRED && half == 1 ? Shape::v_swizzle(r) : Shape::k_swizzle(r);
        k_off[i] = (uint32_t)((r & 15) * RB + ((lane % CPR) ^ k_swizzle) * 16);
        if constexpr(!PAIRED)
        {
            v_off[i] = (uint32_t)((r & 15) * RB + ((lane % CPR) ^ Shape::v_swizzle(r)) * 16);
        }
    }
    // lane's addresses of the operands in a slot; the 16-key groups lie 16 * RB apart
    // (the swizzles have a period of 16 rows)
    constexpr int KREADS = RB < 64 ? 1 : RB / 64;       // 16-byte reads of a key row by its four lanes
    uint32_t k_at[KREADS];
#pragma unroll
    for(int i = 0; i < KREADS; ++i)
    {
        k_at[i] = (uint32_t)(col * RB + ((4 * i + quad) ^ Shape::k_swizzle(col)) * 16);
    }
    uint32_t v_at[DBLOCKS];
#pragma unroll
    for(int db = 0; db < DBLOCKS; ++db)
    {
        if constexpr(KIND == kPaged16)
        {
            // transposing read: lane i of a quad gives the address of row i / 4, four values
            // from 4 * (i % 4) on
            const int r = 4 * quad + (col >> 2), c = 2 * db + ((col >> 1) & 1);
            v_at[db] = (uint32_t)(K_BYTES + r * RB + (c ^ Shape::v_swizzle(r)) * 16 + 8 * (col & 1));
        }
        else if constexpr(KIND == kPaged8)
        {
            // ... of row i / 2, eight values from 8 * (i % 2) on; rows 4 .. 7 are the
            // next 16-key group's
            const int j = col >> 1, r = 4 * quad + (j & 3) + 16 * (j >> 2);
            v_at[db] = (uint32_t)(K_BYTES + r * RB + (db ^ Shape::v_swizzle(r)) * 16 + 8 * (col & 1));
        }
        else
        {
            // single values of row 4 * quad (+ i: the swizzle is the same for the four)
            const int r = 4 * quad, d = 16 * db + col;
            v_at[db] = (uint32_t)(K_BYTES + r * RB + ((d >> 2) ^ Shape::v_swizzle(r)) * 16 + 4 * (d & 3));
        }
    }
    const float c_log2 = p.scale * kLog2e, slack = kPagedSlack / c_log2;

    for(;;)
    {
        uint32_t taken = 0;
        if(!aligned)
        {
            // (the last place of a unit has no block: seg.steps may be 0)
            seg.steps = (int)min((uint32_t)max(seg.blocks - seg.step, 0), end - at);
            taken = min((uint32_t)(cost_of(seg.blocks) - seg.step), end - at);
        }
        if(seg.steps > 0)
        {
        // (the row groups of a head from both ends in turn: where the last ones see more keys than the first,
        // shares of some units have equally much to do)
        const int h = seg.u / p.row_groups, in_turn = seg.u - h * p.row_groups;
        const int rg = (in_turn & 1) != 0 ? p.row_groups - 1 - (in_turn >> 1) : in_turn >> 1;
        const int given = in_wave ? __builtin_amdgcn_readlane(given_of_lane, seg.n) : uniform(paged_new(p.c, seg.n, p.q_seq));
        const int key_lo = seg.step * Shape::BLOCK;
        // the keys that some row of the group sees, of the tokens of one head: those in front of the newest one's
        int seen = seg.len;
        if(p.row_groups > 1)
        {
            const int first = rg * QROWS, last_row = min(first + QROWS, p.rows) - 1;
            const int head_of = uniform(first / p.q_seq);
            if(last_row < (head_of + 1) * p.q_seq)
            {
                const int newest = min(last_row - head_of * p.q_seq, given - 1);
                seen = first - head_of * p.q_seq >= given ? 0 : p.causal ? max(seg.len - given + newest + 1, 0) : seen;
            }
        }
        const int key_hi = max(min(key_lo + seg.steps * Shape::BLOCK, min(seg.len, seen)), key_lo);
        const int my_first = key_lo + stream * KEYS;
        const int n_mine = my_first < key_hi ? (key_hi - my_first + Shape::BLOCK - 1) / Shape::BLOCK : 0;

        // ---- the lane's query rows ---------------------------------------------------
        // 16-byte pieces of an operand begin at head values: 16-bit 32i + 8*quad; 8-bit pages, whose
        // 16-byte reads hold 16 values, 64(i/2) + 16*quad + 8(i%2); fp32 16i + 4*quad
        constexpr int E = KIND == kPaged32 ? 4 : 2;
        auto q_piece = [&](int i)
        {
            return (KIND == kPaged16 ? 32 * i + 8 * quad : KIND == kPaged8 ? 64 * (i / 2) + 16 * quad + 8 * (i % 2)
                    : 16 * i + 4 * quad) * E / 16;
        };
        u32x4 qf[Q_IN_LDS ? 1 : QREGS];
        int last[NR];           // the last key the row sees
        int token[NR];
        bool row_ok[NR];
#pragma unroll
        for(int nr = 0; nr < NR; ++nr)
        {
            const int rr = rg * QROWS + (half * NR + nr) * 16 + col;
            token[nr] = rr % p.q_seq;
            row_ok[nr] = rr < p.rows && token[nr] < given;
            last[nr] = min(p.causal ? seg.len - given + token[nr] : seg.len - 1, seg.len - 1);
        }
        if constexpr(Q_IN_LDS)
        {
            constexpr int PIECES = Shape::QB / 16;
            for(int t = tid; t < QROWS * PIECES; t += THREADS)
            {
                const int r = t / PIECES, piece = t % PIECES, rr = rg * QROWS + r;
                u32x4 x = {0, 0, 0, 0};
                if(rr < p.rows && rr % p.q_seq < given)
                {
                    x = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(p.Q)
                            + paged_query_row(p, seg.n, h, rr) * Shape::QB + piece * 16);
                }
                *reinterpret_cast<u32x4 *>(q_rows + r * Shape::QB + (piece ^ Shape::q_swizzle(r)) * 16) = x;
            }
            __syncthreads();
        }
        else if constexpr(KIND != kPaged4)
        {
            const char *src = static_cast<const char *>(p.Q)
                + paged_query_row(p, seg.n, h, row_ok[0] ? rg * 16 + col : 0) * Shape::QB;
#pragma unroll
            for(int i = 0; i < QREGS; ++i)
            {
                qf[i] = row_ok[0] ? *reinterpret_cast<const u32x4 *>(src + q_piece(i) * 16) : u32x4{0, 0, 0, 0};
            }
        }
        auto q_operand = [&](int nr, int i) -> u32x4
        {
            if constexpr(Q_IN_LDS)
            {
                return *reinterpret_cast<const u32x4 *>(q_rows + ((half * NR + nr) * 16 + col) * Shape::QB
                        + (q_piece(i) ^ Shape::q_swizzle(col)) * 16);
            }
            else
            {
                return qf[i];
            }
        };
        // below it every row sees every key
        const int all_see = p.causal ? seg.len - given : seg.len - 1;

        f32x4 o[NR][DBLOCKS];
        float m_run[NR], l_run[NR];
#pragma unroll
        for(int nr = 0; nr < NR; ++nr)
        {
            m_run[nr] = neg_inf();
            l_run[nr] = 0.0f;
#pragma unroll
            for(int db = 0; db < DBLOCKS; ++db)
            {
                o[nr][db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }

        // The count of the unit's shares that are done, at the place of its first share (every share is the
        // first of one shared unit at most).  It has kPagedNone between calls; if it holds something else,
        // the workspace is new, which is seen to where the count is needed.
        const bool whole = seg.step == 0 && seg.steps == seg.blocks;
        const uint32_t w0 = aligned || whole ? first_share : split.of(unit_begin);
        unsigned long long *const count = p.counts + w0 * kPagedCountStride;
        unsigned long long held = kPagedNone;
        auto count_so_far = [&]() -> unsigned long long
        {
            return tid == 0 && !whole ? __hip_atomic_load(count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : kPagedNone;
        };
        if constexpr(KIND == kPaged4)
        {
            held = count_so_far();
            paged4_walk<T, HEAD, NR>(p, seg, h, rg, given, my_first, n_mine, all_see, last, ring, o, m_run, l_run);
        }
        else
        {
        // ---- pages and loads ------------------------------------------------------------
        const int64_t table_row = (int64_t)seg.n * p.c.max_pages;
        // Where a page holds a step, its groups lie behind each other in one page: one look-up, one address.
        const bool one_page = (1 << p.c.page_shift) >= KEYS;
        auto look_up = [&](int i, int (&page)[GROUPS])
        {
            const int row0 = my_first + i * Shape::BLOCK;
            page[0] = scalar_load<int>(p.c.table, 4 * (table_row + (row0 >> p.c.page_shift)));
            if(GROUPS > 1 && !one_page)
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
        // the row of group g among those of the pages' heads
        auto in_page = [&](int i, int g)
        {
            const int row = min(my_first + i * Shape::BLOCK + 16 * g, seg.len - 1) & ~15;
            return ((int64_t)h << p.c.page_shift) + (row & ((1 << p.c.page_shift) - 1));
        };
        // (a page that is none is read as page 0 and hidden)
        auto real_page = [&](int page) { return (unsigned)page < (unsigned)p.c.n_pages ? page : 0; };
        // where the groups of a step lie in a pool of rows of `bytes`, `stride` from page to page
        auto places = [&](int i, const int (&page)[GROUPS], int64_t stride, int bytes, int64_t (&from)[GROUPS])
        {
            from[0] = real_page(page[0]) * stride + in_page(i, 0) * bytes;
            if(GROUPS == 1 || one_page)
            {
#pragma unroll
                for(int g = 1; g < GROUPS; ++g)
                {
                    from[g] = from[0] + 16 * g * bytes;
                }
            }
            else
            {
#pragma unroll
                for(int g = 1; g < GROUPS; ++g)
                {
                    from[g] = real_page(page[g]) * stride + in_page(i, g) * bytes;
                }
            }
        };
        auto fetch = [&](int i, const int (&page)[GROUPS], char *slot)
        {
            int64_t from[GROUPS];
            places(i, page, p.c.page_stride, RB, from);
            const char *const first = PAIRED && half == 1 ? p.c.v_pages : p.c.k_pages;
            char *const to = PAIRED && half == 1 ? slot + K_BYTES : slot;
#pragma unroll
            for(int ld = 0; ld < LOADS; ++ld)
            {
                load_to_lds16<0, true>(first + from[ld * Shape::ROWS_PER_LOAD / 16], k_off[ld], to + ld * 1024);
            }
            if constexpr(!PAIRED)
            {
#pragma unroll
                for(int ld = 0; ld < LOADS; ++ld)
                {
                    load_to_lds16<0, true>(p.c.v_pages + from[ld * Shape::ROWS_PER_LOAD / 16], v_off[ld],
                            slot + K_BYTES + ld * 1024);
                }
            }
        };
        // The scale bytes of a step go to LDS like the rows, 16 a lane: lane g < GROUPS has those of the keys of
        // group g, lane GROUPS + g those of the values.  (Through the scalar cache they take more scalar
        // registers than there are: 64 sequences of 17 to 16384 rows, 8 heads of 64, 46.9 -> 42.5 us.)
        char *const scale_slots = scale_bytes + (KIND == kPaged8 ? wave * 4 * KEYS : 0);
        const char *const scales_of_lane = reinterpret_cast<const char *>(lane < GROUPS ? p.c.k_scales : p.c.v_scales);
        auto fetch_scales = [&](int i, const int (&page)[GROUPS])
        {
            int64_t from[GROUPS];
            places(i, page, p.c.scale_stride, 1, from);
            const int g = lane % GROUPS;
            int64_t mine = from[0] + 16 * g;
            if(GROUPS > 1 && !one_page)
            {
                mine = from[0];
#pragma unroll
                for(int j = 1; j < GROUPS; ++j)
                {
                    mine = g == j ? from[j] : mine;
                }
            }
            if(lane < 2 * GROUPS)
            {
                load_to_lds16<0, false>(scales_of_lane + mine, scale_slots + (i & 1) * 2 * KEYS);
            }
        };

        int page[GROUPS], page_next[GROUPS];
        constexpr int STEP_LOADS = (PAIRED ? LOADS : 2 * LOADS) + (KIND == kPaged8 ? 1 : 0);
        if(n_mine > 0)
        {
            look_up(0, page);
            fetch(0, page, slots);
            if constexpr(KIND == kPaged8)
            {
                fetch_scales(0, page);
            }
            look_up(min(1, n_mine - 1), page_next);
        }
        held = count_so_far();
        const int n_steps = PAIRED ? (key_hi - key_lo + Shape::BLOCK - 1) / Shape::BLOCK : n_mine;
        auto without_page = [&]()       // groups of the step
        {
            uint32_t hidden = (unsigned)page[0] < (unsigned)p.c.n_pages ? 0u : GROUPS == 1 || one_page ? ~0u : 1u;
            if(GROUPS > 1 && !one_page)
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
            char *const slot = slots + (i & 1) * STAGE;
            const uint32_t hidden = PARTLY ? without_page() : 0;
            // the reads of the slot that is filled next have returned (to both)
            paged_wait_lds();
            if constexpr(PAIRED)
            {
                __syncthreads();
            }
            if(i + 1 < n_mine)
            {
                fetch(i + 1, page_next, slots + ((i + 1) & 1) * STAGE);
                if constexpr(KIND == kPaged8)
                {
                    fetch_scales(i + 1, page_next);
                }
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
            if constexpr(PAIRED)
            {
                __syncthreads();        // both have loaded their half of this step
            }
            if(PARTLY && PAIRED && i >= n_mine)
            {
                return;
            }
            const int key0 = my_first + i * Shape::BLOCK;
            if(PARTLY && (key0 + KEYS > seg.len || hidden != 0))
            {
                // values of rows that are none: zeros, so that what lies there does not
                // get into the products (their probabilities are exactly 0)
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
                    const int rows_there = (hidden >> g) & 1 ? 0 : min(max(seg.len - key0 - 16 * g, 0), 16);
                    for(int b = rows_there * RB + lane * 16; b < 16 * RB; b += 64 * 16)
                    {
                        *reinterpret_cast<u32x4 *>(slot + K_BYTES + g * 16 * RB + b) = u32x4{0, 0, 0, 0};
                    }
                }
                paged_wait_lds();
            }

            // scale bytes of four keys of each group: the keys', of those around the lane's key row where they go
            // into its codes, else of the lane's scores; the values', of the lane's probabilities
            uint32_t ks[GROUPS], vs[GROUPS];
            if constexpr(KIND == kPaged8)
            {
                const char *const bytes = scale_slots + (i & 1) * 2 * KEYS;
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
                    ks[g] = *reinterpret_cast<const uint32_t *>(bytes + 16 * g + 4 * (KSCALE_IN_CODES ? col >> 2 : quad));
                    vs[g] = *reinterpret_cast<const uint32_t *>(bytes + KEYS + 16 * g + 4 * quad);
                }
            }

            // ---- scores --------------------------------------------------------------
            f32x4 s[NR][GROUPS];
#pragma unroll
            for(int g = 0; g < GROUPS; ++g)
            {
                u32x4 kf[KREADS];
#pragma unroll
                for(int r = 0; r < KREADS; ++r)
                {
                    kf[r] = *reinterpret_cast<const u32x4 *>(slot + k_at[r] + g * 16 * RB);
                }
                u32x4 wide[KIND == kPaged8 ? 2 * KREADS : 1];
                // (of the lane's key row)
                const float k_scale = KSCALE_IN_CODES ? scale_of(ks[g], col & 3) : 1.0f;
                if constexpr(KIND == kPaged8)
                {
#pragma unroll
                    for(int r = 0; r < 2 * KREADS; ++r)
                    {
                        const u32x2 a = widen4<T>(kf[r / 2][2 * (r % 2)], k_scale),
                        b = widen4<T>(kf[r / 2][2 * (r % 2) + 1], k_scale);
                        wide[r] = u32x4{a[0], a[1], b[0], b[1]};
                    }
                }
#pragma unroll
                for(int nr = 0; nr < NR; ++nr)
                {
                    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for(int i = 0; i < QREGS; ++i)
                    {
                        const u32x4 q = q_operand(nr, i);
                        if constexpr(KIND == kPaged32)
                        {
#pragma unroll
                            for(int e = 0; e < 4; ++e)
                            {
                                x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[i][e]),
                                        __uint_as_float(q[e]), x, 0, 0, 0);
                            }
                        }
                        else
                        {
                            x = mfma32<T>(KIND == kPaged8 ? wide[i % (2 * KREADS)] : kf[i % KREADS], q, x);
                        }
                    }
                    s[nr][g] = x;
                }
            }

            // ---- probabilities -------------------------------------------------------
            // 8-bit pages: what a probability is multiplied by for its value row's power of two
            f32x4 of_scale[GROUPS];
            if constexpr(KIND == kPaged8)
            {
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        // (a row that does not exist: whatever its byte, times a probability of 0)
                        const bool there = !PARTLY || 4 * quad + e < ((hidden >> g) & 1 ? 0 : seg.len - key0 - 16 * g);
                        of_scale[g][e] = there ? scale_of(vs[g], e) : 0.0f;
                    }
                }
            }
            uint32_t pw[NR][GROUPS][2];                 // 16-bit pairs
            uint32_t pw_rest[TWO_PARTS ? NR : 1][TWO_PARTS ? GROUPS : 1][2];        // what they leave
            f32x4 pf[NR][GROUPS];                       // fp32
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
                        float x = s[nr][g][e];
                        if constexpr(KIND == kPaged8 && !KSCALE_IN_CODES)
                        {
                            x *= scale_of(ks[g], e);
                        }
                        if constexpr(PARTLY)
                        {
                            x = 4 * quad + e > ((hidden >> g) & 1 ? -1 : last[nr] - key0 - 16 * g) ? neg_inf() : x;
                        }
                        s[nr][g][e] = x;
                        top = fmaxf(top, x);
                    }
                }
                // p = 2^(c * score - c * reference): c is positive, and the product with the
                // reference is rounded the same way wherever it is taken.  The reference is a
                // maximum that is replaced once the scores are 2^kPagedSlack past it, so that sums and
                // products are seldom scaled.
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
                const float off = kLift - (m_run[nr] == neg_inf() ? 0.0f : m_run[nr] * c_log2);
                float sum = 0.0f;
#pragma unroll
                for(int g = 0; g < GROUPS; ++g)
                {
                    f32x4 x;
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        x[e] = fast_exp2(fmaf(s[nr][g][e], c_log2, off));
                        sum += x[e];
                    }
                    if constexpr(KIND == kPaged8)
                    {
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                        {
                            x[e] *= of_scale[g][e];
                        }
                    }
                    if constexpr(KIND == kPaged32)
                    {
                        pf[nr][g] = x;
                    }
                    else if constexpr(TWO_PARTS)
                    {
                        // the first 8 bits as they are, the next 8 rounded: 2^-16 of a probability is lost at most
                        const u32x4 bits = __builtin_bit_cast(u32x4, x);
                        const f32x4 rest = x - __builtin_bit_cast(f32x4, bits & 0xffff0000u);
                        pw[nr][g][0] = __builtin_amdgcn_perm(bits[1], bits[0], 0x07060302u);
                        pw[nr][g][1] = __builtin_amdgcn_perm(bits[3], bits[2], 0x07060302u);
                        pw_rest[nr][g][0] = PV::pack2(rest[0], rest[1]);
                        pw_rest[nr][g][1] = PV::pack2(rest[2], rest[3]);
                    }
                    else
                    {
                        pw[nr][g][0] = PV::pack2(x[0], x[1]);
                        pw[nr][g][1] = PV::pack2(x[2], x[3]);
                    }
                }
                l_run[nr] += sum;
            }

            // ---- output ----------------------------------------------------------------
            auto value_words = [&](int db, int t, u32x4 &w)
            {
                typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
                // keys 32t + {4*quad + 0..3, 16 + 4*quad + 0..3}
                if constexpr(KIND == kPaged16)
                {
                    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (lds_s16x4 *)(slot + v_at[db] + 32 * t * RB)));
                    const u32x2 b = GROUPS == 1 ? u32x2{0, 0}
                        : __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (lds_s16x4 *)(slot + v_at[db] + (32 * t + 16) * RB)));
                    w = u32x4{a[0], a[1], b[0], b[1]};
                }
                else if constexpr(KIND == kPaged8)
                {
                    const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                (lds_i32x2 *)(slot + v_at[db] + 32 * t * RB)));
                    const u32x2 a = widen4<PV>(v[0], 1.0f), b = widen4<PV>(v[1], 1.0f);
                    w = u32x4{a[0], a[1], b[0], b[1]};
                }
                else
                {
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        // key 16t + 4*quad + e
                        w[e] = *reinterpret_cast<const uint32_t *>(slot + v_at[db] + (16 * t + e) * RB);
                    }
                }
            };
            // products of the value words of step t (32 keys, fp32: 16)
            auto multiply = [&](const u32x4 &w, int t, int nr, f32x4 c) -> f32x4
            {
                if constexpr(KIND == kPaged32)
                {
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[e]), pf[nr][t][e], c, 0, 0, 0);
                    }
                    return c;
                }
                else if constexpr(GROUPS == 1)
                {
                    return mfma16<PV>(u32x2{w[0], w[1]}, u32x2{pw[nr][0][0], pw[nr][0][1]}, c);
                }
                else
                {
                    c = mfma32<PV>(w, u32x4{pw[nr][2 * t][0], pw[nr][2 * t][1], pw[nr][2 * t + 1][0],
                            pw[nr][2 * t + 1][1]}, c);
                    if constexpr(TWO_PARTS)
                    {
                        c = mfma32<PV>(w, u32x4{pw_rest[nr][2 * t][0], pw_rest[nr][2 * t][1],
                                pw_rest[nr][2 * t + 1][0], pw_rest[nr][2 * t + 1][1]}, c);
                    }
                    return c;
                }
            };
            constexpr int TSTEPS = KIND == kPaged32 ? GROUPS : (GROUPS + 1) / 2;
            // Where a value is no number, a probability of 0 does not hide it (0 * NaN).  That matters in the
            // rows behind all_see, which are hidden from some query: are there any?
            bool odd = false;
            if(PARTLY && p.causal && given > 1)
            {
                bool any = false;
                for(int b = max(all_see + 1 - key0, 0) * RB + lane * 16; b < K_BYTES; b += 64 * 16)
                {
                    const u32x4 w = *reinterpret_cast<const u32x4 *>(slot + K_BYTES + b);
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        any = any || not_numbers<T, KIND>(w[e]);
                    }
                }
                odd = __any(any);
            }
            // (in one form with the others where there are many registers to keep, see below)
            if(!PARTLY || (NR == 1 && !odd))
            {
#pragma unroll
                for(int db = 0; db < DBLOCKS; ++db)
                {
#pragma unroll
                    for(int t = 0; t < TSTEPS; ++t)
                    {
                        u32x4 w;
                        value_words(db, t, w);
#pragma unroll
                        for(int nr = 0; nr < NR; ++nr)
                        {
                            o[nr][db] = multiply(w, t, nr, o[nr][db]);
                        }
                    }
                }
            }
            else if constexpr(PARTLY)
            {
                // If so, token by token, with the values behind what the token sees taken out and only the
                // rows of the token taken over.
                const int rounds = odd ? given : 1;
                for(int tok = 0; tok < rounds; ++tok)
                {
                    // (nothing is read ahead of the loop: the registers are the other form's)
                    asm volatile("" ::: "memory");
#pragma unroll
                    for(int db = 0; db < DBLOCKS; ++db)
                    {
                        f32x4 fresh[NR];
#pragma unroll
                        for(int nr = 0; nr < NR; ++nr)
                        {
                            fresh[nr] = o[nr][db];
                        }
#pragma unroll
                        for(int t = 0; t < TSTEPS; ++t)
                        {
                            u32x4 w;
                            value_words(db, t, w);
                            if(odd)
                            {
                                // the values of this step's first keys that the token sees
                                const int seen = all_see + tok + 1 - key0 - (KIND == kPaged32 ? 16 : 32) * t - 4 * quad;
#pragma unroll
                                for(int e = 0; e < 4; ++e)
                                {
                                    if constexpr(KIND == kPaged32)
                                    {
                                        w[e] = e < seen ? w[e] : 0u;
                                    }
                                    else
                                    {
                                        const int at_key = 16 * (e >> 1) + 2 * (e & 1);
                                        w[e] &= (at_key < seen ? 0xffffu : 0u) | (at_key + 1 < seen ? 0xffff0000u : 0u);
                                    }
                                }
                            }
#pragma unroll
                            for(int nr = 0; nr < NR; ++nr)
                            {
                                fresh[nr] = multiply(w, t, nr, fresh[nr]);
                            }
                        }
#pragma unroll
                        for(int nr = 0; nr < NR; ++nr)
                        {
                            const bool take = !odd || token[nr] == tok;
#pragma unroll
                            for(int e = 0; e < 4; ++e)
                            {
                                o[nr][db][e] = take ? fresh[nr][e] : o[nr][db][e];
                            }
                        }
                    }
                }
            }
        };
        // (the steps without hidden keys on their own: two forms behind each other cost fewer
        // registers than a choice between them)
        int i = 0;
        for(; i < n_mine && my_first + i * Shape::BLOCK + KEYS - 1 <= all_see && without_page() == 0; ++i)
        {
            take_step(i, std::false_type());
        }
        for(; i < n_steps; ++i)
        {
            take_step(i, std::true_type());
        }
        }

        // ---- the wavefronts' results, then the unit's or the share's ---------------------
        const int my_tid = KIND == kPaged4 ? fresh(tid) : tid, my_wave = KIND == kPaged4 ? uniform(my_tid >> 6) : wave;
        const int my_col = KIND == kPaged4 ? my_tid & 15 : col, my_quad = KIND == kPaged4 ? (my_tid & 63) >> 4 : quad;
        const bool begins = seg.step == 0;
        const int rows_here = min(p.rows - rg * QROWS, QROWS);
        float *const merge_o = reinterpret_cast<float *>(ring);
        float *const merge_ml = merge_o + STREAMS * 16 * HALVES * MERGE_LD;
#pragma unroll
        for(int nr = 0; nr < NR; ++nr)
        {
            __syncthreads();        // every wavefront is done with the ring, or with the last row block
            const int mine = my_wave * 16 + my_col;
            float m = m_run[nr] * c_log2 - kLift, l = quad_sum(l_run[nr]);
            if(!row_ok[nr])
            {
                m = neg_inf();
                l = 0.0f;
            }
#pragma unroll
            for(int db = 0; db < DBLOCKS; ++db)
            {
                *reinterpret_cast<f32x4 *>(merge_o + mine * MERGE_LD + 16 * db + 4 * my_quad)
                    = row_ok[nr] ? o[nr][db] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            if(my_quad == 0)
            {
                merge_ml[2 * mine] = m;
                merge_ml[2 * mine + 1] = l;
            }
            __syncthreads();
            // 16 threads a row; the row of stream w lies at (w + STREAMS * half) * 16 + row
            constexpr int PAIRS = HEAD / 32;
            const int row = (my_tid / 16) % 16, its_half = my_tid / 256, t = my_tid % 16;
            const int in_group = (its_half * NR + nr) * 16 + row, rr = rg * QROWS + in_group;
            if(rr < p.rows)
            {
                const int from = its_half * STREAMS * 16 + row;
                float top = neg_inf(), sum = 0.0f;
                f32x2 v[PAIRS];
#pragma unroll
                for(int w = 0; w < STREAMS; ++w)
                {
                    top = fmaxf(top, merge_ml[2 * (from + w * 16)]);
                }
                const float safe = top == neg_inf() ? 0.0f : top;
#pragma unroll
                for(int k = 0; k < PAIRS; ++k)
                {
                    v[k] = f32x2{0.0f, 0.0f};
                }
#pragma unroll
                for(int w = 0; w < STREAMS; ++w)
                {
                    const float f = fast_exp2(merge_ml[2 * (from + w * 16)] - safe);
                    sum += f * merge_ml[2 * (from + w * 16) + 1];
#pragma unroll
                    for(int k = 0; k < PAIRS; ++k)
                    {
                        v[k] += f * *reinterpret_cast<const f32x2 *>(merge_o + (from + w * 16) * MERGE_LD
                                + 2 * (t + 16 * k));
                    }
                }
                if(whole)
                {
                    paged_finish_row<T, 16, PAIRS>(p, paged_query_row(p, seg.n, h, rr), t, top, sum, v);
                }
                else
                {
                    const int64_t place = ((int64_t)me * 2 + (begins ? 1 : 0)) * QROWS + in_group;
#pragma unroll
                    for(int k = 0; k < PAIRS; ++k)
                    {
                        put2(p.part_o + place * HEAD + 2 * (t + 16 * k), v[k]);
                    }
                    if(t == 0)
                    {
                        put2(p.part_ml + 2 * place, f32x2{top, sum});
                    }
                }
            }
        }
        if(!whole)
        {
            // The share's results are with the device once its stores are acknowledged, every
            // wavefront's in front of the barrier.  The workgroup that counts last joins.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const uint32_t parts = aligned ? of_unit : split.of(unit_begin + (uint32_t)seg.blocks - 1) - w0 + 1;
            if(tid == 0)
            {
                if((held & ~kPagedCountMask) != kPagedNone)
                {
                    // (one of the shares that saw this gets its value in, before any of them counts)
                    __hip_atomic_compare_exchange_strong(count, &held, kPagedNone, __ATOMIC_RELAXED,
                            __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                const unsigned long long old = __hip_atomic_fetch_add(count, 1ull, __ATOMIC_RELAXED,
                        __HIP_MEMORY_SCOPE_AGENT);
                found = (uint32_t)(old & kPagedCountMask) == parts - 1;
            }
            __syncthreads();
            if(uniform(found) != 0)
            {
                if(tid == 0)
                {
                    __hip_atomic_store(count, kPagedNone, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                paged_join<T, HEAD, THREADS, QROWS>(p, seg.n, h, rg, rows_here, (int)w0, (int)parts,
                        reinterpret_cast<float *>(ring), my_tid);
            }
        }
        }
        at += taken;
        if(aligned || at >= end)
        {
            return;
        }
        // the next unit, of this sequence or of the next that has rows
        __syncthreads();
        seg.step = 0;
        unit_begin = at;
        if(++seg.u == p.units)
        {
            seg.u = 0;
            do
            {
                ++seg.n;
                seg.len = len_of(seg.n);
                seg.blocks = (seg.len + Shape::BLOCK - 1) / Shape::BLOCK;
            } while(seg.blocks == 0);       // (`end` lies behind a block that exists)
        }
    }
}

// Blocks of 16 rows that a workgroup takes: 1, 2, or 4 by two wavefronts a key; 1 also where that leaves no
// more than 64 units, which then have more shares, and joins, between them (8 units of 4096 rows, 64 query
// rows, 26.7 us with 4 blocks a workgroup, 21.4 with 1; 64 units of 2048 29.2 and 51.9).
static int row_blocks(bool two_at_most, int64_t entries, int64_t rows)
{
    return rows <= 16 || entries * ((rows + 15) / 16) <= 64 ? 1 : rows <= 32 || two_at_most ? 2 : 4;
}

// The workspace: the counts, then the shares' results (the larger size of the types', which differ in
// the rows of a workgroup).
static size_t share_rows(int64_t rows)
{
    return (size_t)kPagedShares * 2 * 16 * (size_t)row_blocks(false, 64, rows);
}

static void place_workspace(PagedAttendParams &p, int head, void *workspace)
{
    p.counts = static_cast<unsigned long long *>(workspace);
    p.part_o = reinterpret_cast<float *>(p.counts + kPagedShares * kPagedCountStride);
    p.part_ml = p.part_o + share_rows(p.rows) * (size_t)head;
}

template<typename T, int KIND, int HEAD, int NR, int HALVES>
static int launch_form(hipStream_t stream, PagedAttendParams &p)
{
    typedef PagedShape<KIND, HEAD, NR, HALVES> Shape;
    p.row_groups = (p.rows + Shape::QROWS - 1) / Shape::QROWS;
    p.units = p.c.n_head_kv * p.row_groups;
    // at most as many shares as there can be blocks
    const int64_t most = (int64_t)p.c.n_batch * p.units * (p.c.max_rows / Shape::BLOCK + 1 + kPagedUnitCost);
    if(most > 0x7fffffffll)
    {
        return NNTILE_HIP_EINVAL;
    }
    const int64_t places = kPagedCUs * Shape::WGS_PER_CU;
    p.shares = (int32_t)(most < places ? most : places);
    hipLaunchKernelGGL((sdpa_paged_kernel<T, KIND, HEAD, NR, HALVES>), dim3((unsigned)p.shares),
            dim3(Shape::THREADS), 0, stream, p);
    return hipGetLastError() == hipSuccess ? NNTILE_HIP_OK : NNTILE_HIP_ELAUNCH;
}

template<typename T, int KIND>
static int launch_kind(hipStream_t stream, PagedAttendParams &p, int head)
{
    switch(row_blocks(KIND == kPaged32 || KIND == kPaged4, (int64_t)p.c.n_batch * p.c.n_head_kv, p.rows) * 256 + head)
    {
        case 256 + 64: return launch_form<T, KIND, 64, 1, 1>(stream, p);
        case 256 + 128: return launch_form<T, KIND, 128, 1, 1>(stream, p);
        case 512 + 64: return launch_form<T, KIND, 64, 2, 1>(stream, p);
        case 512 + 128: return launch_form<T, KIND, 128, 2, 1>(stream, p);
        default: break;
    }
    if constexpr(KIND != kPaged32 && KIND != kPaged4)
    {
        return head == 64 ? launch_form<T, KIND, 64, 2, 2>(stream, p) : launch_form<T, KIND, 128, 2, 2>(stream, p);
    }
    return NNTILE_HIP_EUNSUPPORTED;
}

} // namespace nntile_hip
