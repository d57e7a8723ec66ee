// Sizes of the attention over pages: what a wavefront and a workgroup take at a time.
#pragma once

#include "paged_operands.hpp"

namespace nntile_hip
{

constexpr int kPagedCUs = 256;
// Workgroups that the keys are shared out to at most: two a CU
constexpr int kPagedShares = 2 * kPagedCUs;
// What a unit costs beside its key blocks, in blocks
constexpr int kPagedUnitCost = 1;
// How far, in powers of two, probabilities may grow past the first before they are taken against a new maximum
constexpr float kPagedSlack = 8.0f;
// fp16 probabilities of 16-bit pages are kept times 2^7: they stay below 2^15, and 2^-21 still has all of its bits
constexpr float kPagedLift = 7.0f;
// Counts of shares in the workspace: in the low bits, above them a fixed word by which a count is told
// from what else memory may hold; a cache line each.
constexpr unsigned long long kPagedCountMask = 4095;
constexpr unsigned long long kPagedNone = 0x9e3779b97f4a7000ull;
constexpr int kPagedCountStride = 8;
static_assert(kPagedShares < (int)kPagedCountMask, "counts stay below the word");

template<int KIND, int HEAD, int NR, int HALVES>
struct PagedShape
{
    static constexpr int STREAMS = 4;                       // wavefronts that take different keys
    static constexpr int WAVES = STREAMS * HALVES;
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int QROWS = 16 * NR * HALVES;          // query rows of a workgroup
    static constexpr int RB = KIND == kPaged32 ? HEAD * 4 : KIND == kPaged8 ? HEAD : KIND == kPaged4 ? HEAD / 2
        : HEAD * 2;                                         // bytes of a row
    static constexpr int SB = KIND == kPaged4 ? HEAD / 32 : 1;      // scale bytes of a row, where there are any
    static constexpr int CPR = RB / 16;                     // 16-byte chunks of a row
    static constexpr int RPL = RB >= 256 ? 1 : 256 / RB;    // rows per 256-byte line of LDS banks
    // keys of a wavefront's step: 8 KB of K and V; twice that where two wavefronts share them and the pages hold
    // 16 bits (8 sequences of 8192 rows, 8 heads of 128, 64 query rows 54.8 us, 58.7 with 8 KB; 8-bit pages, whose
    // widened operands are more registers, 51.7 and 47.7)
    static constexpr int ALONE = 4096 / RB > 16 ? 4096 / RB : 16;
    static constexpr int KEYS = KIND == kPaged8 ? ALONE : HALVES * ALONE < 64 ? HALVES * ALONE : 64;
    static_assert(KIND != kPaged4 || (KEYS == 64 && HALVES == 1), "a transposing read of 4-bit values takes 64 keys");
    static constexpr int BLOCK = STREAMS * KEYS;        // keys of a workgroup's step
    static constexpr int GROUPS = KEYS / 16;
    static constexpr int K_BYTES = KEYS * RB;
    static constexpr int STAGE = 2 * K_BYTES;
    static constexpr int LOADS = K_BYTES / 1024;            // load instructions of a step's K
    static constexpr int ROWS_PER_LOAD = 1024 / RB;
    // (what a row block of all wavefronts takes at the end, too)
    static constexpr int MERGE_BYTES = STREAMS * 16 * HALVES * (HEAD + 4 + 2) * 4;
    // the query rows: the operands of one block of 16 stay in registers, those of two in LDS
    static constexpr int QB = HEAD * (KIND == kPaged32 ? 4 : 2);
    static constexpr int Q_BYTES = NR > 1 ? QROWS * QB : 16;
    // 4-bit pages: two steps' keys, values and scales of every wavefront, and the query rows behind them
    static constexpr int WALK = STREAMS * 2 * (STAGE + 2 * KEYS * SB) + QROWS * QB;
    static constexpr int FILL = KIND == kPaged4 ? WALK : STREAMS * 2 * STAGE;
    static constexpr int RING = FILL > MERGE_BYTES ? FILL : MERGE_BYTES;
    // (4-bit pages, head 64, one row block, as many as LDS has room for, four: 64 sequences of 1024 rows, 4 query rows,
    // 12.2 -> 16.6 us, of 4096 32 -> 37; two row blocks, three: 16 of 300 to 4096 fp16 rows 19 -> 26, by spills)
    static constexpr int WGS_PER_CU = KIND == kPaged4 ? 2
        : RING > 72 * 1024 || WAVES > 4 ? 1 : 2;
    static_assert(KIND != kPaged4 || RING <= 79 * 1024, "room for two workgroups a CU");
    static constexpr int MIN_WAVES = WAVES * WGS_PER_CU / 4;        // of a SIMD
    static __host__ __device__ constexpr int q_swizzle(int r) { return r % (QB / 16 < 16 ? QB / 16 : 16); }

    // 4-bit pages: a load takes RPG rows of each of the four groups, so that a lane has the same group, and page, in
    // all loads.  Where chunk c of row r lies then: rows that one instruction reads are on different banks, but for two
    // lanes each of the transposing reads.
    static constexpr int RPG = KIND == kPaged4 ? 16 / LOADS : 1;
    static __host__ __device__ constexpr int place4(int r, int c)
    {
        return r % 16 / RPG * 1024 + r / 16 * 256 + r % RPG * RB + ((c ^ (r / RPG) ^ (r / 16)) & (CPR - 1)) * 16;
    }

    // Where chunk c of row r lies: chunk position c ^ swizzle(r) of the row, so that the
    // rows one LDS instruction reads fall on different banks.
    static __host__ __device__ constexpr int k_swizzle(int r) { return (r / RPL) % CPR; }
    static __host__ __device__ constexpr int v_swizzle(int r)
    {
        return KIND == kPaged16 ? 2 * ((r / RPL) % (CPR / 2))
            : KIND == kPaged8 ? k_swizzle(r) : 4 * ((r >> 2) & 3);
    }
};

// What a workgroup works on at a time: key blocks [step, step + steps) of unit u (head and row
// group) of sequence n.
struct PagedSegment
{
    int n, len, blocks;     // sequence, its rows, their key blocks
    int u, step, steps;
};

// Row of lse (times head: of Q and A) of query row rr of key/value head h of sequence n
__device__ __forceinline__ int64_t paged_query_row(const PagedAttendParams &p, int n, int h, int rr)
{
    const int g = rr / p.q_seq, tok = rr % p.q_seq;
    return (n + (int64_t)p.c.n_batch * (g + (int64_t)p.kv_group * h)) * p.q_seq + tok;
}

} // namespace nntile_hip
