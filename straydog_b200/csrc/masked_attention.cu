// Attention of many query rows under masks and score rules, on the 5th-generation tensor cores (tcgen05.mma, accumulators in TMEM): packed
// documents over 16-bit keys and values (sdx_masked_attention), and prompt chunks over 8-bit states (the codes unpacked to 16 bits first).
//
// Row i of a sequence with n keys and r rows sits at p = n - r + i and sees key j < n when j <= p and j > p - window, or when j < prefix.
//   s = scale * q . k;  s = cap * tanh(s / cap);  s -= slope[head] * |p - j|;  out = softmax over the seen keys . v, zeros where none is seen
//
// A unit is 256 M-rows of one K/V head as two tiles of 128 (one tile for 256 columns): 128 / group consecutive rows times the `group` query heads, so
// K and V are fetched once for all of them and the diagonal is thin. Its work is the union of its rows' keys in tiles of 128, in steps of 64 keys:
//   S[128 x 64]  = Q . K^T    D / 16 tcgen05.mma, K in shared memory (TMA, 128-byte swizzle), Q there too (256 columns: in TMEM), S FP32 in TMEM
//   O[128 x D]  += P . V      4 tcgen05.mma, P in TMEM over the columns of its S, V in shared memory
// S has two buffers a query tile: while the softmax works on one, the next S and the last value product are under way, of the other query tile too.
// What bounds it: the softmax's issue slots and the tensor pipe, almost evenly. 128 columns: 64 keys of two tiles take 1780 cycles, of which the
// products fill about 1000 (half the rate: a product of 64 keys reads Q from shared memory twice as often for its flops as one of 128) and
// a softmax warp 1480 (64 scores a thread: load, maximum, exponential, sum, rounding, store), the rest is hand-over. Steps of 128 keys with
// one buffer a tile left softmax and products in turn: 285 us for a chunk of 2048 rows over 8192 keys (32 / 8 heads of 128), 241 us now (1.0
// PFLOP/s; 20 us of it unpacking codes and bringing queries to FP16); 4096 rows over 16384 keys of 16 / 2 heads of 256 under a cap 812 us (1.18 PFLOP/s), 7 documents of up to 2100 rows 131 us. A distance
// bias or a cap adds FMA work to the softmax: 4096 rows over 8192 keys of 32 / 8 heads of 128 take 370 us, 404 with a bias, 451 to 467 with a cap of 50, 1265 with a cap
// that most scores are past a quarter of (the slow pass).
// Persistent blocks, one an SM: the units' steps laid end to end are cut into equal runs (a unit counts three steps more, for its first products, its masked
// tiles and its output). A block walks its run without stopping: the next unit's first products are issued while the last one's output is written. A unit that
// two or more blocks share leaves FP32 partials for a second kernel. (A block a unit left the last of 1.7 waves a third empty for a chunk of 2048
// rows, 285 us, and spent half of 184 us on first loads and outputs for packed documents of 8 tiles a unit.)
// Warps: 0-3 and 4-7 softmax, a thread a row (half a row with 256 columns); 8 and 9 issue the products of a query tile each; 10 the TMA loads; 11
// looks after values that some row may not see (below).
//
// Roundings: scores, maxima, sums and O are FP32. P is rounded to the operands' type once (FP16 or BF16), at 2^7 times its size so that FP16 keeps
// 11 bits down to 2^-21 of the largest weight. (The two operands of a product have one type, and FP16 does not hold what values in BF16 may be: there P has
// 8 bits. Codes are FP16 whatever the rows are, queries brought to FP16.) O is multiplied in TMEM only when a row's maximum grew by more than 2^8. The keys' scales of an 8-bit
// state multiply the scores, a block of 32 a factor; the values' scales join the exponent of P, and the running maximum is that of a weight times its
// value's scale, so that P has its bits for what the row sees, however large the values are that it does not see or gives no weight. (The maximum of the
// weights alone, with scales relative to the head's largest: a block of values 2^23 times the others, behind a row's window, left the row's FP16 P nothing.)
//
// A weight of 0 times a value that is infinite or NaN is NaN. In tiles where some row does not see some key (the diagonal, a border), a warp
// replaces such values by 0 before the product reads them; the rows that do see them get them back at the end. What no row sees does not reach it.
#include "kv8.cuh"
#include "masked_attention.cuh"
#include "../../include/straydog_gpu_b200.h"

#include <cuda.h>
#include <type_traits>

namespace sdb {
namespace attn {

constexpr int kThreads = 384, kM = 128, kStep = 64;   // kStep: keys of a step, what the softmax works on at a time
constexpr int kIssueWarp = 8, kLoadWarp = 10, kLookWarp = 11;   // (one or two issuing warps, a query tile each)
constexpr float kLift = 7.0f, kRescale = 8.0f;
constexpr unsigned kSequences = 64;   // sequences a launch
constexpr int kFlagged = 16;          // slots of one piece that are looked at for values that are not finite (borders: at most a dozen)

template<int D> struct Shape {
    static constexpr int kTiles = D == 256 ? 1 : 2;                   // query tiles a unit
    static constexpr int kKSlots = D == 256 ? 3 : 5, kVSlots = D == 256 ? 4 : 5;   // two rings in shared memory, a step's keys or values a slot
    static constexpr int kSlotBytes = kStep * D * 2, kQueryBytes = kM * D * 2;
    static constexpr bool kQInTmem = D == 256;                        // (64 KB that K and V need more; and it is read twice as fast there)
    static constexpr int kOffK = kQInTmem ? 0 : kTiles * kQueryBytes, kOffV = kOffK + kKSlots * kSlotBytes, kOffBars = kOffV + kVSlots * kSlotBytes;
    static constexpr int kOffFlags = kOffBars + 512, kOffStats = kOffFlags + kFlagged * 32;
    static constexpr int kSlack = kTiles == 1 ? 0 : 1024;             // to align the base to 1024 bytes where there is room (the runtime aligns it anyway)
    static constexpr size_t kSmem = kOffStats + (kTiles == 1 ? 2 * 2 * kM * 4 : 0) + kSlack;
    static_assert(kSmem <= 227 * 1024, "shared memory");
    static constexpr int kO = 256, kQ = 128;                          // TMEM columns: two S buffers a tile from 0, Q of 256 columns at 128, O of tile t at 256 + D t
    static __device__ __forceinline__ uint32_t scores(int tile, int buffer) { return tile * 128 + buffer * kStep; }
};

struct KernelSequence {
    uint32_t rows, length, prefix, first_row, first_key, first_unit, blocks, first_block;   // blocks of rows; first_block: of the unpacked blocks of 32 keys
};
constexpr unsigned kMostBlocks = 160;   // blocks of a launch (one an SM)
struct Cut { uint32_t unit, tile; };                   // where a block's run begins
struct Shared { uint32_t unit, first, pieces; };       // a unit that blocks first .. first + pieces - 1 share
struct Args {
    CUtensorMap q_map, k_map, v_map;
    KernelSequence sequence[kSequences];
    uint32_t sequences, heads, kv_heads, group, tokens;   // tokens: rows of a query tile
    uint32_t window, shares;
    Cut cut[kMostBlocks + 1];
    Shared share[kMostBlocks];
    void* out;
    size_t out_stride;
    const float* slopes;
    const float* block_table;    // 8-bit states: [kv_heads][tiles of four blocks of 32 keys][12]: four key scales, log2 of four value scales (from a floor up), the rests below it
    uint32_t table_blocks;
    const uint16_t* queries;     // the query rows again, where they do not come through the map
    const float* query_factors;  // 8-bit states under BF16 rows: [row][head] what a lifted query is to be multiplied by
    size_t query_stride;
    uint32_t first_query;        // the row that queries, their map and their factors begin with
    const uint16_t* values;      // 16-bit rows: the values again, for the rows that see one that is not finite
    size_t value_stride;
    float scale_log2, cap, scale_over_cap;
    float* partial;              // [2 * block + (the unit goes on in the next block)][M-rows][D]: a block shares its first and its last unit at most
    float* sums;                 // the same [M-rows][2]
    int* status;
};

// Barriers: S, P and the value product of (tile, buffer), values looked at, Q, O of a tile, the rings' slots. A barrier tells a phase from its
// neighbours only: whoever waits for one has to know that the phase before is over and that the one after cannot be.
enum { kQFull = 0, kSFull = 1, kPFull = 5, kPvDone = 9, kLook = 13, kClean = 14, kQFree = 15, kOFree = 16, kKFull = 18, kKFree = 23, kVFull = 28, kVFree = 33, kBars = 38 };

constexpr uint32_t kDescHigh = 0x40004040u;   // 128-byte swizzle, 1024 bytes between groups of 8 rows (see csrc/qsa_prompt_tc.cu)
__device__ __forceinline__ uint32_t desc_low(uint32_t address, uint32_t leading_bytes) { return ((address & 0x3ffffu) >> 4) | ((leading_bytes >> 4) << 16); }
__device__ __forceinline__ uint64_t desc_of(uint32_t low) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(kDescHigh));
    return d;
}
// kind::f16: FP32 accumulator; A and B both FP16 or both BF16; A K-major, B K-major or MN-major
__device__ __forceinline__ uint32_t instr_desc(int m, int n, bool bf16, bool b_mn_major) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(uint32_t(accumulate)) : "memory");
}
__device__ __forceinline__ void umma_a_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(uint32_t(accumulate)) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
    return pred != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define SDB_R8(r, b) "=r"(r[b]), "=r"(r[b + 1]), "=r"(r[b + 2]), "=r"(r[b + 3]), "=r"(r[b + 4]), "=r"(r[b + 5]), "=r"(r[b + 6]), "=r"(r[b + 7])
#define SDB_I8(r, b) "r"(r[b]), "r"(r[b + 1]), "r"(r[b + 2]), "r"(r[b + 3]), "r"(r[b + 4]), "r"(r[b + 5]), "r"(r[b + 6]), "r"(r[b + 7])
__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t* r) {   // (the values are there after tmem_load_wait of the same registers)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : SDB_R8(r, 0), SDB_R8(r, 8), SDB_R8(r, 16), SDB_R8(r, 24) : "r"(address) : "memory");
}
#define SDB_B8(r, b) "+r"(r[b]), "+r"(r[b + 1]), "+r"(r[b + 2]), "+r"(r[b + 3]), "+r"(r[b + 4]), "+r"(r[b + 5]), "+r"(r[b + 6]), "+r"(r[b + 7])
// (the registers are operands: no use of them may be scheduled ahead of the wait)
__device__ __forceinline__ void tmem_load_wait(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : SDB_B8(r, 0), SDB_B8(r, 8), SDB_B8(r, 16), SDB_B8(r, 24) :: "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t address, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(address), SDB_I8(r, 0), SDB_I8(r, 8), SDB_I8(r, 16), SDB_I8(r, 24) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(address), SDB_I8(r, 0), SDB_I8(r, 8) : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// (plain loads: see where the table is read)
__device__ __forceinline__ void load_factors(const float* from, float (&v)[1]) { asm volatile("ld.global.f32 %0, [%1];" : "=f"(v[0]) : "l"(from) : "memory"); }
__device__ __forceinline__ void load_factors(const float* from, float (&v)[2]) { asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "l"(from) : "memory"); }
__device__ __forceinline__ void store32(void* to, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), SDB_I8(w, 0) : "memory");
}
// A tile of a packed array: x (columns) on a 16-byte boundary always (a multiple of 64 elements); rows past the array read as zeros.
__device__ __forceinline__ void tma_load(void* to, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(to)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}

// two FP32 operations an instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
    return p;
}
__device__ __forceinline__ void unpair(uint64_t p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t both(float x) { return pair(x, x); }
// of two pairs of 16-bit floats, the larger magnitudes; a NaN if either is
template<bool BF16> __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) {
    uint32_t d;
    a &= 0x7fff7fffu; b &= 0x7fff7fffu;
    if (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// lanes whose bit BIT is 0 give y for the other's x, the others x for the other's y: a transposition in steps
template<int BIT> __device__ __forceinline__ void trade(uint32_t& x, uint32_t& y, int lane) {
    const bool high = lane & BIT;
    const uint32_t other = __shfl_xor_sync(0xffffffffu, high ? x : y, BIT);
    if (high) x = other; else y = other;
}
// the low `count` bits set (none below 0, all from 32 on)
__device__ __forceinline__ uint32_t first_bits(int count) { return count <= 0 ? 0u : count >= 32 ? 0xffffffffu : (1u << count) - 1u; }
__device__ __forceinline__ float max3(float a, float b, float c) {   // (as fmaxf: a NaN is no maximum)
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// A unit: its rows and the key tiles that any of them sees, the same for every role (and on the host, which cuts the runs).
struct Unit {
    uint32_t s, kv, row;                 // sequence, K/V head, first row
    int first, last, length, prefix;     // positions of the first and the last row; the sequence's
    uint32_t head_tiles, jump, tiles;    // tiles from head_tiles on are `jump` tiles further on
    __host__ __device__ __forceinline__ void find(const Args& a, uint32_t unit, uint32_t rows_a_unit) {
        s = 0;
        uint32_t high = a.sequences;
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_unit <= unit) s = mid; else high = mid; }
        const uint32_t inside = unit - a.sequence[s].first_unit;
        kv = inside % a.kv_heads;
        row = inside / a.kv_heads * rows_a_unit;
        fill(a, rows_a_unit);
    }
    __device__ __forceinline__ void next(const Args& a, uint32_t rows_a_unit) {
        if (++kv < a.kv_heads) return;   // (the same rows: the same tiles)
        kv = 0;
        row += rows_a_unit;
        if (row >= a.sequence[s].rows) { ++s; row = 0; }
        fill(a, rows_a_unit);
    }
    __host__ __device__ __forceinline__ void fill(const Args& a, uint32_t rows_a_unit) {
        const KernelSequence& q = a.sequence[s];
        length = int(q.length); prefix = int(q.prefix);
        const uint32_t end = q.rows < row + rows_a_unit ? q.rows : row + rows_a_unit;
        first = length - int(q.rows) + int(row);
        last = length - int(q.rows) + int(end) - 1;
        const int causal = last + 1, reach = causal > prefix ? causal : prefix;
        const uint32_t low = a.window && first >= int(a.window) ? uint32_t(first - int(a.window) + 1) : 0u;
        const uint32_t all = uint32_t((reach > 0 ? reach : 0) + kStep - 1) / kStep;
        head_tiles = uint32_t(prefix + kStep - 1) / kStep;
        uint32_t body = low / kStep > head_tiles ? low / kStep : head_tiles;
        if (body > all) body = all;
        jump = body - head_tiles;
        tiles = all - jump;
    }
    // The last keys come first: where scores fall off with the distance, the maximum then stands after the first tiles. (From the first key on, slopes of
    // 0.001 to 0.01 made most steps of 4096 rows over 8192 keys move the maximum.)
    __device__ __forceinline__ uint32_t key(uint32_t tile) const {
        const uint32_t at = tiles - 1 - tile;
        return (at < head_tiles ? at : at + jump) * kStep;
    }
    // whether every row of the unit sees every key of the tile at key0
    __device__ __forceinline__ bool open(const Args& a, uint32_t key0) const {
        const int end_key = int(key0) + kStep - 1;
        return (end_key <= first && end_key < length && (!a.window || int(key0) > last - int(a.window))) || end_key < prefix;
    }
};

// A block's run, piece by piece: a piece is the part of a unit's tiles that lies in the run.
template<int ROWS> struct Run {
    uint32_t unit, begin, end;   // the piece's tiles
    Cut to;
    bool whole;
    Unit u;
    __device__ __forceinline__ bool start(const Args& a) {
        const Cut from = a.cut[blockIdx.x];
        to = a.cut[blockIdx.x + 1];
        unit = from.unit;
        if (done()) return false;
        u.find(a, unit, ROWS * a.tokens);
        set(from.tile);
        return true;
    }
    __device__ __forceinline__ bool next(const Args& a) {
        ++unit;
        if (done()) return false;
        u.next(a, ROWS * a.tokens);
        set(0);
        return true;
    }
    __device__ __forceinline__ bool done() const { return unit > to.unit || (unit == to.unit && !to.tile); }
    __device__ __forceinline__ void set(uint32_t from) {
        begin = from;
        end = unit == to.unit ? to.tile : u.tiles;
        whole = !begin && end == u.tiles;
    }
};

// BF16: the type of the rows, queries and outputs. KV8: keys and values are codes with scales beside (one kernel that asks took 1349 us for
// 4096 rows over 8192 16-bit keys past a quarter of their cap, 1240 the one without).
template<int D, bool BF16, bool RULE, bool KV8>
__global__ void __launch_bounds__(kThreads, 1) masked_attention_kernel(const __grid_constant__ Args a) {
    using S = Shape<D>;
    constexpr int T = S::kTiles, kGroups = T;   // a softmax thread's groups of 32 columns of S
    constexpr bool kBf16 = BF16 && !KV8, kLifted = BF16 && KV8;   // the products' operands; codes are FP16, and BF16 queries are brought there
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    if (!S::kSlack && smem_u32(smem_raw) % 1024) {   // (no operand layout without it: reported, not computed)
        if (threadIdx.x == 0) atomicExch(a.status, 1);
        return;
    }
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBars);
    static_assert(kBars * 8 + 16 <= S::kOffFlags - S::kOffBars, "barriers");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* flagged_piece = tmem_slot + 2;                       // the piece (counted from 1) that `flagged` belongs to
    uint32_t* flagged = reinterpret_cast<uint32_t*>(smem + S::kOffFlags);   // [slot looked at]: its first key, then four words of keys

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < kBars; ++i)
            mbar_init(&bars[i], (i >= kPFull && i < kPFull + 4) || i == kOFree || i == kOFree + 1 ? (T == 2 ? 4 : 8) : i == kQFull ? (S::kQInTmem ? 8 : 1) :
                                i == kLook || i == kQFree || (i >= kKFree && i < kVFull) || i >= kVFree ? T : 1);
        *abort_flag = 0;
        *flagged_piece = 0;
    }
    fence_barrier_init();
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (everything read from here on may be the kernel's before)

    auto wait = [&](int bar, uint32_t parity) -> bool {   // bounded, and ended by another role's giving up
        if (mbar_try_wait(&bars[bar], parity)) return true;
        const uint64_t start = global_timer_ns();
        for (;;) {
            #pragma unroll 1
            for (int spin = 0; spin < 32; ++spin)
                if (mbar_try_wait(&bars[bar], parity)) return true;
            if (*abort_flag) return false;
            if (global_timer_ns() - start > 2000000000ull) { *abort_flag = 1; atomicExch(a.status, 1); return false; }
        }
    };
    Run<T> run;
    bool alive = true;
    uint32_t done = 0;            // steps of the pieces before (each role counts for itself: the barriers' parities follow these)
    uint32_t used[2] = {0, 0};    // uses of the two S buffers by the pieces before (a piece's step i takes buffer i % 2)
    uint32_t piece = 0;           // pieces with steps before

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");   // (8 warps x 208 and 4 x 88: what 12 are launched with at 168)
        // ================= softmax: a thread a row (T 2: a warpgroup a query tile), or half a row (T 1: a warpgroup a half of the columns) =================
        uint32_t next_queries = 0;
        const int tile_of = T == 2 ? warp / 4 : 0, half = T == 2 ? 0 : warp / 4, m = (warp & 3) * 32 + lane;
        const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
        constexpr int kOColumns = T == 2 ? D : D / 2;                          // a thread's columns of O
        const uint32_t o_base = lane_base + S::kO + tile_of * D + half * kOColumns;
        float* stats = reinterpret_cast<float*>(smem + S::kOffStats) + m;      // T 1: [turn's parity][half][row], what the two threads of a row tell each other
        auto other_half = [&](float mine, uint32_t turn) -> float {
            if (T == 2) return mine;
            stats[((turn & 1) * 2 + half) * kM] = mine;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
            return stats[((turn & 1) * 2 + (half ^ 1)) * kM];
        };
        auto any_of_rows = [&](bool mine) -> bool {   // of the warp's rows (T 1: of the two warps that share them)
            if (T == 2) return __any_sync(0xffffffffu, mine);
            uint32_t any;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                         : "=r"(any) : "r"(uint32_t(mine)), "r"(1 + (warp & 3)) : "memory");
            return any != 0;
        };
        uint32_t turn = 0;
        // 256 columns: the queries of the next piece that has steps go to TMEM as soon as the scores before are done, ahead of the outputs
        auto bring_queries = [&](Run<T> next, bool more) {
            while (more && next.begin == next.end) more = next.next(a);
            if (!more || !alive) return;
            if (next_queries && !wait(kQFree, (next_queries - 1) & 1)) { alive = false; return; }
            ++next_queries;
            fence_after();
            const KernelSequence& sequence = a.sequence[next.u.s];
            const uint32_t token = next.u.row + m / a.group, head = next.u.kv * a.group + m % a.group;
            const bool real = token < sequence.rows && uint32_t(m) < a.tokens * a.group;
            const uint4* from = reinterpret_cast<const uint4*>(a.queries + (real ? (size_t(sequence.first_row - a.first_query) + token) * a.query_stride + size_t(head) * D + half * (D / 2) : 0));
            #pragma unroll 1
            for (int b = 0; b < D / 2 / 64; ++b) {
                uint32_t w[32];
                #pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const uint4 v = real ? from[8 * b + n] : make_uint4(0, 0, 0, 0);   // (plain: they may be the kernel's before)
                    w[4 * n] = v.x; w[4 * n + 1] = v.y; w[4 * n + 2] = v.z; w[4 * n + 3] = v.w;
                }
                tmem_store32(lane_base + S::kQ + half * (D / 4) + 32 * b, w);
            }
            tmem_store_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[kQFull]);
        };
        bool more = run.start(a);
        if (S::kQInTmem) bring_queries(run, more);
        for (; more && alive; more = run.next(a)) {
            const Unit& u = run.u;
            const KernelSequence& sequence = a.sequence[u.s];
            const uint32_t tiles = run.end - run.begin;
            const uint32_t token = u.row + tile_of * a.tokens + m / a.group, head = u.kv * a.group + m % a.group;
            const bool valid = token < sequence.rows && uint32_t(m) < a.tokens * a.group;
            const int position = u.length - int(sequence.rows) + int(token);
            const float slope = RULE && a.slopes && valid ? a.slopes[head] * 1.4426950408889634f : 0.0f;
            // 8-bit states: a tile's factors are 12 floats, [scores' | weights' log2 | rests] x [four groups of 32 keys]
            const float* table_at = KV8 ? a.block_table + (size_t(u.kv) * a.table_blocks + sequence.first_block) * 3 + half : nullptr;
            float scale_log2 = a.scale_log2, scale_over_cap = a.scale_over_cap;
            if (kLifted && tiles) {
                float factor[1] = {0.0f};   // (M-rows without a query hold others' lifted ones: at a factor of 1 their scores made most steps take the slow pass)
                if (valid) load_factors(a.query_factors + (size_t(sequence.first_row - a.first_query) + token) * a.heads + head, factor);
                scale_log2 *= factor[0]; scale_over_cap *= factor[0];
            }
            float top_run = -INFINITY, sum_run = 0.0f;
            #pragma unroll 1
            for (uint32_t i = 0; i < tiles; ++i) {
                const uint32_t key0 = u.key(run.begin + i);
                const int buffer = int(i & 1), ready = 2 * tile_of + buffer;
                float to_score[kGroups], shift[kGroups], to_sum[kGroups], rest[kGroups];
                bool rests = false;
                #pragma unroll
                for (int g = 0; g < kGroups; ++g) { to_score[g] = 1.0f; shift[g] = 0.0f; to_sum[g] = 1.0f; rest[g] = 1.0f; }
                if (KV8) {
                    // (plain loads: the kernel before this one, whose programmatic dependent it is, may still have been writing the table when it was launched)
                    const float* table = table_at + key0 / 128 * 12 + key0 / 64 % 2 * 2;
                    load_factors(table, to_score); load_factors(table + 4, shift); load_factors(table + 8, rest);
                    #pragma unroll
                    for (int g = 0; g < kGroups; ++g) { to_sum[g] = fast_exp2(-shift[g]); rests |= rest[g] != 1.0f; }
                    if (T == 1) {   // (the two threads of a row go the same way: they meet at barriers)
                        float other[1];
                        load_factors(table + 8 + 1 - 2 * half, other);
                        rests |= other[0] != 1.0f;
                    }
                }
                if (!wait(kSFull + ready, (used[buffer] + (i >> 1)) & 1)) { alive = false; break; }
                fence_after();
                const uint32_t s_base = lane_base + S::scores(tile_of, buffer) + half * 32;
                const bool open = u.open(a, key0);
                // Weights are computed from the maximum so far, in one pass over the scores that finds the tile's own on the way. Where that is above by
                // more than 2^8, where there is none yet, and in tiles with a mask, a cap or a bias, the scores are finished and the maximum found
                // first, O is multiplied, and the pass runs over what went back to TMEM. (So it does where a value scale lies below the table's floor.)
                bool first = i == 0 || !open || rests;
                // all keys on one side of all rows: the distance is linear in the key, and its bias starts in the exponent's offset
                float lean = 0.0f;
                if (RULE && a.slopes && open) {
                    if (int(key0) + kStep - 1 <= u.first) lean = slope;
                    else if (int(key0) >= u.last) lean = -slope;
                    else first = true;
                }
                if (!first) {
                    const float under = top_run == -INFINITY ? 0.0f : top_run - kLift;
                    uint32_t loaded[kGroups][32], packed[16 * kGroups];
                    float top = -INFINITY, sum = 0.0f;
                    bool steep = false;
                    #pragma unroll
                    for (int g = 0; g < kGroups; ++g) tmem_load32(s_base + 32 * g, loaded[g]);
                    #pragma unroll
                    for (int g = 0; g < kGroups; ++g) tmem_load_wait(loaded[g]);
                    #pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        uint32_t (&bits)[32] = loaded[g];
                        float most = -INFINITY;
                        uint64_t sums = both(0.0f);
                        auto pass = [&](auto cap_too, auto bias_too) {
                            constexpr bool kCap = decltype(cap_too)::value, kBias = decltype(bias_too)::value;
                            float d = shift[g] - under;
                            if (kBias) d = fmaf(-lean, float(position - int(key0) - half * 32 - 32 * g), d);
                            uint64_t d2 = kBias ? pair(d, d + lean) : both(d);
                            const float c = scale_log2 * to_score[g], inner = kCap ? scale_over_cap * to_score[g] : 0.0f;
                            const uint64_t c1 = both(kCap ? c * kTanh1 : c), c3 = both(c * inner * inner * kTanh3), c5 = both(c * inner * inner * (inner * inner) * kTanh5);
                            const uint64_t step = both(2.0f * lean);
                            float farthest = 0.0f;
                            auto exponents = [&](int n) -> uint64_t {
                                const uint64_t score = pair(__uint_as_float(bits[2 * n]), __uint_as_float(bits[2 * n + 1]));
                                uint64_t x;
                                if (kCap) {   // (the cap and the scale are in the series' coefficients)
                                    farthest = max3(farthest, fabsf(__uint_as_float(bits[2 * n])), fabsf(__uint_as_float(bits[2 * n + 1])));
                                    const uint64_t z = mul2(score, score);
                                    x = fma2(score, fma2(fma2(z, c5, c3), z, c1), d2);
                                } else {
                                    x = fma2(score, c1, d2);
                                }
                                if (kBias) d2 = add2(d2, step);
                                return x;
                            };
                            auto weights = [&](int n, float x0, float x1) {
                                x0 = fast_exp2(x0); x1 = fast_exp2(x1);
                                sums = add2(sums, pair(x0, x1));
                                packed[16 * g + n] = kBf16 ? pack_bf16x2(x0, x1) : pack_half2(x0, x1);
                            };
                            // (exponents first and weights then, where the exponents are chains: 428 us against 495 with a bias; plain ones are 2 % faster in one go)
                            #pragma unroll
                            for (int n = 0; n < 16; ++n) {
                                float x0, x1;
                                unpair(exponents(n), x0, x1);
                                most = max3(most, x0, x1);
                                if (kCap || kBias) { bits[2 * n] = __float_as_uint(x0); bits[2 * n + 1] = __float_as_uint(x1); }
                                else weights(n, x0, x1);
                            }
                            if (kCap || kBias) {
                                #pragma unroll
                                for (int n = 0; n < 16; ++n) weights(n, __uint_as_float(bits[2 * n]), __uint_as_float(bits[2 * n + 1]));
                            }
                            // scores past the series, or so large that its coefficients may have left the normal numbers
                            if (kCap) steep |= !(fabsf(inner) < 1e4f && farthest <= 1e6f && farthest * fabsf(inner) <= kSmallTanh);
                        };
                        using No = std::false_type;
                        if (!RULE) pass(No{}, No{});
                        else if (a.cap > 0.0f && a.slopes) pass(std::bool_constant<RULE>{}, std::bool_constant<RULE>{});
                        else if (a.cap > 0.0f) pass(std::bool_constant<RULE>{}, No{});
                        else pass(No{}, std::bool_constant<RULE>{});
                        float sum0, sum1;
                        unpair(sums, sum0, sum1);
                        top = fmaxf(top, most);
                        sum = fmaf(sum0 + sum1, to_sum[g], sum);
                    }
                    first = any_of_rows(top > (top_run == -INFINITY ? -INFINITY : kLift + kRescale) || (RULE && steep));
                    if (!first) {
                        sum_run += sum;
                        // (over scores that have been read)
                        if constexpr (T == 2) tmem_store32(s_base, packed); else tmem_store16(s_base, packed);
                    }
                }
                if (first) {
                    auto of = [&](const float (&v)[kGroups], int g) -> float {   // (no register is addressed by a variable)
                        float r = v[0];
                        #pragma unroll
                        for (int x = 1; x < kGroups; ++x) r = g == x ? v[x] : r;
                        return r;
                    };
                    // (a block of zero keys has a scale of 0, which a masked score of -inf must not be multiplied by)
                    auto score_factor = [&](float key_scale) -> float { return fmaxf(scale_log2 * key_scale, FLT_TRUE_MIN); };
                    const bool finish = !open || RULE;
                    float top = -INFINITY;
                    #pragma unroll 1
                    for (int g = 0; g < kGroups; ++g) {
                        uint32_t bits[32];
                        tmem_load32(s_base + 32 * g, bits);
                        tmem_load_wait(bits);
                        float c = of(to_score, g);
                        if (RULE && a.cap > 0.0f) {   // cap * tanh(s / cap): the cap (in the exp2 domain) stays outside
                            c *= scale_over_cap;
                            float most = 0.0f;
                            #pragma unroll
                            for (int n = 0; n < 32; n += 2) most = max3(most, fabsf(__uint_as_float(bits[n])), fabsf(__uint_as_float(bits[n + 1])));
                            if (__all_sync(0xffffffffu, most * c <= kSmallTanh)) {   // (the usual case, scores well below the cap: the series to y^7, on the FMA pipe)
                                #pragma unroll
                                for (int n = 0; n < 32; ++n) {
                                    const float y = __uint_as_float(bits[n]) * c, z = y * y;
                                    bits[n] = __float_as_uint(fmaf(fmaf(fmaf(z, -17.0f / 315.0f, 2.0f / 15.0f), z, -1.0f / 3.0f) * z, y, y));
                                }
                            } else if (a.cap <= kFineCap) {
                                #pragma unroll
                                for (int n = 0; n < 32; ++n) bits[n] = __float_as_uint(any_tanh(__uint_as_float(bits[n]) * c));
                            } else {
                                #pragma unroll
                                for (int n = 0; n < 32; ++n) bits[n] = __float_as_uint(either_tanh(__uint_as_float(bits[n]) * c));
                            }
                            c = a.cap;
                        } else {
                            c = score_factor(c);
                        }
                        if (RULE && a.slopes) {
                            const float from = float(position - int(key0) - half * 32 - 32 * g);
                            #pragma unroll
                            for (int n = 0; n < 32; ++n) bits[n] = __float_as_uint(fmaf(-slope, fabsf(from - float(n)), __uint_as_float(bits[n]) * c));
                            c = 1.0f;
                        }
                        if (!open) {
                            // a bit a column: keys up to `to` and above `low`, or below `prefix`, relative to the group
                            const int base = int(key0) + half * 32 + 32 * g;
                            const int to = min(position, u.length - 1) - base, low = a.window ? position - int(a.window) - base : -1, prefix = u.prefix - base;
                            uint32_t seen = (first_bits(to + 1) & ~first_bits(low + 1)) | first_bits(prefix);
                            if (!valid) seen = 0;
                            #pragma unroll
                            for (int n = 0; n < 32; ++n)
                                if (!(seen & (1u << n))) bits[n] = 0xff800000u;
                        }
                        if (finish) tmem_store32(s_base + 32 * g, bits);
                        float t = __uint_as_float(bits[0]);
                        #pragma unroll
                        for (int n = 1; n < 31; n += 2) t = max3(t, __uint_as_float(bits[n]), __uint_as_float(bits[n + 1]));
                        const float d = of(shift, g);
                        top = max3(top, fmaf(t, c, d), fmaf(__uint_as_float(bits[31]), c, d));
                    }
                    if (finish) tmem_store_wait();
                    top = fmaxf(top, other_half(top, turn++));
                    const bool grow = top > top_run + kRescale || (top_run == -INFINITY && top > -INFINITY);
                    const float use = grow ? top : top_run;
                    if (i > 0 && __any_sync(0xffffffffu, grow && top_run != -INFINITY)) {
                        // (the products two steps back were over before these scores were made)
                        if (!wait(kPvDone + 2 * tile_of + (buffer ^ 1), (used[buffer ^ 1] + ((i - 1) >> 1)) & 1)) { alive = false; break; }
                        fence_after();
                        const float factor = grow && top_run != -INFINITY ? fast_exp2(top_run - use) : 1.0f;
                        #pragma unroll 1
                        for (int b = 0; b < kOColumns / 32; ++b) {
                            uint32_t o[32];
                            tmem_load32(o_base + 32 * b, o);
                            tmem_load_wait(o);
                            #pragma unroll
                            for (int n = 0; n < 32; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * factor);
                            tmem_store32(o_base + 32 * b, o);
                        }
                        tmem_store_wait();
                        sum_run *= factor;
                    }
                    top_run = use;
                    const float under = use == -INFINITY ? 0.0f : use - kLift;
                    #pragma unroll 1
                    for (int g = 0; g < kGroups; ++g) {
                        uint32_t bits[32];
                        tmem_load32(s_base + 32 * g, bits);
                        const float c = RULE && a.slopes ? 1.0f : RULE && a.cap > 0.0f ? a.cap : score_factor(of(to_score, g)), d = of(shift, g) - under;
                        tmem_load_wait(bits);
                        float sum0 = 0.0f, sum1 = 0.0f;
                        #pragma unroll
                        for (int n = 0; n < 16; ++n) {
                            const float p0 = fast_exp2(fmaf(__uint_as_float(bits[2 * n]), c, d)), p1 = fast_exp2(fmaf(__uint_as_float(bits[2 * n + 1]), c, d));
                            bits[n] = kBf16 ? pack_bf16x2(p0, p1) : pack_half2(p0, p1);
                            sum0 += p0; sum1 += p1;
                        }
                        if (KV8 && rests) {   // (rare: once more, for the products alone)
                            const float down = of(rest, g);
                            tmem_load32(s_base + 32 * g, bits);
                            tmem_load_wait(bits);
                            #pragma unroll
                            for (int n = 0; n < 16; ++n) {
                                const float p0 = fast_exp2(fmaf(__uint_as_float(bits[2 * n]), c, d)) * down, p1 = fast_exp2(fmaf(__uint_as_float(bits[2 * n + 1]), c, d)) * down;
                                bits[n] = kBf16 ? pack_bf16x2(p0, p1) : pack_half2(p0, p1);
                            }
                        }
                        sum_run = fmaf(sum0 + sum1, of(to_sum, g), sum_run);
                        tmem_store16(s_base + 16 * g, bits);
                    }
                }
                tmem_store_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[kPFull + ready]);
            }
            if (!alive) break;
            // ---- O / sum ----
            if (S::kQInTmem && tiles) {
                Run<T> next = run;
                const bool any = next.next(a);
                bring_queries(next, any);
                if (!alive) break;
            }
            // (the last product is over when all are)
            if (tiles && !wait(kPvDone + 2 * tile_of + int(tiles - 1 & 1), (used[tiles - 1 & 1] + ((tiles - 1) >> 1)) & 1)) { alive = false; break; }
            fence_after();
            if (T == 1) sum_run += other_half(sum_run, turn++);
            const float inverse = !run.whole ? 1.0f : sum_run > 0.0f ? 1.0f / sum_run : sum_run == 0.0f ? 0.0f : sum_run;
            const size_t slot = (2 * size_t(blockIdx.x) + (run.begin ? 0 : 1)) * T + tile_of;
            // A thread has a row: four threads trade 16-byte pieces and store four rows' runs of 64 bytes, a lane of theirs a piece. (A row a thread, 32
            // lines a store, took 5000 cycles a unit, and its partials, written the same way, 12000.)
            uint16_t* row_at[4];
            {
                const uint64_t mine = run.whole && valid ? reinterpret_cast<uint64_t>(static_cast<uint16_t*>(a.out) + (size_t(sequence.first_row) + token) * a.out_stride + size_t(head) * D) : 0;
                #pragma unroll
                for (int r = 0; r < 4; ++r) row_at[r] = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, mine, (lane & 28) + r));
            }
            const bool patches = !KV8 && tiles && *flagged_piece == piece + 1;
            if (patches) {
                // values that were taken out of a tile: back for the rows that see them (rare: nothing here is fast)
                #pragma unroll 1
                for (int b = 0; b < kOColumns / 32; ++b) {
                    uint32_t bits[32];
                    tmem_load32(o_base + 32 * b, bits);
                    tmem_load_wait(bits);
                    const int column = half * kOColumns + 32 * b;
                    #pragma unroll 1
                    for (int p = 0; valid && p < kFlagged; ++p) {
                        const int base = int(flagged[8 * p]);
                        #pragma unroll 1
                        for (int n = 0; n < kStep; ++n) {
                            if (!(flagged[8 * p + 1 + n / 32] >> (n % 32) & 1)) continue;
                            const int key = base + n;
                            const bool seen = key < u.length && ((key <= position && (!a.window || key > position - int(a.window))) || key < u.prefix);
                            if (!seen) continue;
                            const uint16_t* v = a.values + (size_t(sequence.first_key) + key) * a.value_stride + u.kv * D + column;
                            #pragma unroll 1
                            for (int x = 0; x < 32; ++x) {
                                const float f = BF16 ? __uint_as_float(uint32_t(v[x]) << 16) : __half2float(__ushort_as_half(v[x]));
                                if (fabsf(f) <= FLT_MAX) continue;
                                #pragma unroll
                                for (int y = 0; y < 32; ++y) if (y == x) bits[y] = __float_as_uint(__uint_as_float(bits[y]) + f);   // (no register is addressed by a variable)
                            }
                        }
                    }
                    __syncwarp();
                    tmem_store32(o_base + 32 * b, bits);
                    tmem_store_wait();
                }
            }
            #pragma unroll 1
            for (int b = 0; b < kOColumns / 32; ++b) {
                uint32_t bits[32];
                if (tiles) {
                    tmem_load32(o_base + 32 * b, bits);
                    tmem_load_wait(bits);
                    if (b + 1 == kOColumns / 32) {   // O (and `flagged`) may be written again
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bars[kOFree + tile_of]);
                    }
                }
                float o[32];
                #pragma unroll
                for (int n = 0; n < 32; ++n) o[n] = tiles ? __uint_as_float(bits[n]) * inverse : 0.0f;
                const int column = half * kOColumns + 32 * b;
                if (!run.whole) {
                    // [eight columns][row][column]: a warp's stores lie one behind the other
                    float* to = a.partial + (slot * (D / 8) + column / 8) * (kM * 8) + m * 8;
                    #pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        uint32_t w[8];
                        #pragma unroll
                        for (int x = 0; x < 8; ++x) w[x] = __float_as_uint(o[8 * n + x]);
                        store32(to + n * (kM * 8), w);
                    }
                } else {
                    uint32_t w[16];
                    #pragma unroll
                    for (int n = 0; n < 16; ++n) w[n] = BF16 ? pack_bf16x2(o[2 * n], o[2 * n + 1]) : pack_half2(o[2 * n], o[2 * n + 1]);
                    #pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        trade<1>(w[x], w[4 + x], lane); trade<1>(w[8 + x], w[12 + x], lane);
                        trade<2>(w[x], w[8 + x], lane); trade<2>(w[4 + x], w[12 + x], lane);
                    }
                    #pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (row_at[r]) *reinterpret_cast<uint4*>(row_at[r] + column + (lane & 3) * 8) = make_uint4(w[4 * r], w[4 * r + 1], w[4 * r + 2], w[4 * r + 3]);
                }
            }
            if (!run.whole && valid && half == 0) *reinterpret_cast<float2*>(a.sums + (slot * kM + m) * 2) = make_float2(top_run, sum_run);
            if (tiles) {
                ++piece;
                used[0] += (tiles + 1) / 2; used[1] += tiles / 2;
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        constexpr uint32_t kAhead = 2;   // score products issued ahead of the value products
        if (warp == kIssueWarp || (T == 2 && warp == kIssueWarp + 1)) {
            // ================= the products of a query tile =================
            // The whole warp walks, one elected lane issues: addresses and descriptors stay in uniform registers, which the instruction takes. (One
            // thread walking alone moved every operand there, 70 cycles a product, and was what bound the kernel.)
            const int tile = warp - kIssueWarp;
            const bool leader = elect_one();
            const uint32_t idesc_o = instr_desc(kM, D, kBf16, true);
            const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem, 0), base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
            const uint32_t queries = desc_low(base + tile * S::kQueryBytes, 16);
            uint32_t looked = 0;
            const uint32_t idesc_s = instr_desc(kM, kStep, kBf16, false);
            auto score = [&](uint32_t i, uint32_t tiles) -> bool {
                const uint32_t at = done + i, slot = at % S::kKSlots;
                if (!wait(kKFull + slot, (at / S::kKSlots) & 1)) return false;
                fence_after();
                const int buffer = int(i & 1);
                const uint32_t k = desc_low(base + S::kOffK + slot * S::kSlotBytes, 16), d = tmem_base + S::scores(tile, buffer);
                if (leader) {
                    #pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint64_t k_desc = desc_of(k + (((kk / 4) * (kStep * 128) + (kk % 4) * 32) >> 4));
                        if (S::kQInTmem) umma_a_tmem(d, tmem_base + S::kQ + kk * 8, k_desc, idesc_s, kk > 0);
                        else umma(d, desc_of(queries + (((kk / 4) * (kM * 128) + (kk % 4) * 32) >> 4)), k_desc, idesc_s, kk > 0);
                    }
                    umma_commit(&bars[kSFull + 2 * tile + buffer]);
                    umma_commit(&bars[kKFree + slot]);
                    if (i + 1 == tiles) umma_commit(&bars[kQFree]);
                }
                return true;
            };
            for (bool more = run.start(a); more && alive; more = run.next(a)) {
                const uint32_t tiles = run.end - run.begin;
                if (!tiles) continue;
                if (!wait(kQFull, piece & 1)) { alive = false; break; }
                fence_after();
                for (uint32_t f = 0; f < kAhead && f < tiles && alive; ++f) alive = score(f, tiles);
                #pragma unroll 1
                for (uint32_t i = 0; i < tiles && alive; ++i) {
                    const bool look = !KV8 && !run.u.open(a, run.u.key(run.begin + i));
                    const uint32_t at = done + i, slot = at % S::kVSlots;
                    const int buffer = int(i & 1);
                    // the outputs of the piece before have left O (and `flagged`)
                    if (i == 0 && piece && !wait(kOFree + tile, (piece - 1) & 1)) { alive = false; break; }
                    if (!wait(kVFull + slot, (at / S::kVSlots) & 1)) { alive = false; break; }
                    if (look && leader) mbar_arrive(&bars[kLook]);   // (the step's values are looked at while the softmax runs)
                    if (!wait(kPFull + 2 * tile + buffer, (used[buffer] + (i >> 1)) & 1)) { alive = false; break; }
                    if (look && !wait(kClean, looked++ & 1)) { alive = false; break; }
                    fence_after();
                    const uint32_t v = desc_low(base + S::kOffV + slot * S::kSlotBytes, kStep * 128), p = tmem_base + S::scores(tile, buffer), o = tmem_base + S::kO + tile * D;
                    if (leader) {
                        #pragma unroll
                        for (int kk = 0; kk < kStep / 16; ++kk)
                            umma_a_tmem(o, p + (T == 2 ? kk * 8 : kk / 2 * 32 + kk % 2 * 8), desc_of(v + ((kk * (16 * 128)) >> 4)), idesc_o, i > 0 || kk > 0);
                        umma_commit(&bars[kPvDone + 2 * tile + buffer]);
                        umma_commit(&bars[kVFree + slot]);
                    }
                    if (i + kAhead < tiles) alive = score(i + kAhead, tiles);
                }
                done += tiles;
                used[0] += (tiles + 1) / 2; used[1] += tiles / 2;
                ++piece;
            }
        } else if (warp == kLoadWarp) {
            // ================= the loads =================
            if (lane == 0) {
                for (bool more = run.start(a); more && alive; more = run.next(a)) {
                    const uint32_t tiles = run.end - run.begin;
                    if (!tiles) continue;
                    const KernelSequence& sequence = a.sequence[run.u.s];
                    if (!S::kQInTmem) {
                        if (piece && !wait(kQFree, (piece - 1) & 1)) { alive = false; break; }
                        mbar_expect_tx(&bars[kQFull], uint32_t(T * (D / 64)) * a.tokens * a.group * 128);
                        #pragma unroll 1
                        for (int tile = 0; tile < T; ++tile)
                            for (int x = 0; x < D / 64; ++x)
                                tma_load(smem + tile * S::kQueryBytes + x * (kM * 128), &a.q_map, 64 * x, int(run.u.kv * a.group),
                                         int(sequence.first_row - a.first_query + run.u.row + tile * a.tokens), &bars[kQFull]);
                    }
                    auto key_of = [&](uint32_t i) -> int { return int(sequence.first_key + run.u.key(run.begin + i)); };
                    auto load_k = [&](uint32_t i) {
                        const uint32_t at = done + i, slot = at % S::kKSlots;
                        if (at >= uint32_t(S::kKSlots) && !wait(kKFree + slot, (at / S::kKSlots - 1) & 1)) { alive = false; return; }
                        mbar_expect_tx(&bars[kKFull + slot], S::kSlotBytes);
                        for (int x = 0; x < D / 64; ++x)
                            tma_load(smem + S::kOffK + slot * S::kSlotBytes + x * (kStep * 128), &a.k_map, 64 * x, int(run.u.kv), key_of(i), &bars[kKFull + slot]);
                    };
                    for (uint32_t i = 0; i < kAhead && i < tiles && alive; ++i) load_k(i);
                    #pragma unroll 1
                    for (uint32_t i = 0; i < tiles && alive; ++i) {
                        const uint32_t at = done + i, slot = at % S::kVSlots;
                        if (at >= uint32_t(S::kVSlots) && !wait(kVFree + slot, (at / S::kVSlots - 1) & 1)) { alive = false; break; }
                        mbar_expect_tx(&bars[kVFull + slot], S::kSlotBytes);
                        for (int x = 0; x < D / 64; ++x)
                            tma_load(smem + S::kOffV + slot * S::kSlotBytes + x * (kStep * 128), &a.v_map, 64 * x, int(run.u.kv), key_of(i), &bars[kVFull + slot]);
                        if (i + kAhead < tiles) load_k(i + kAhead);
                    }
                        done += tiles;
                    ++piece;
                }
            }
        } else if (warp == kLookWarp && !KV8) {
            // ================= masked values that are not finite =================
            uint32_t looked = 0;   // steps looked at (the next is not asked for before this one is done: the barriers' parities cannot be missed)
            for (bool more = run.start(a); more && alive; more = run.next(a)) {
                const uint32_t tiles = run.end - run.begin;
                if (!tiles) continue;
                int edge = 0;      // the piece's steps looked at: the entry of `flagged` is the step's own
                #pragma unroll 1
                for (uint32_t i = 0; i < tiles; ++i) {
                    const uint32_t key0 = run.u.key(run.begin + i), at = done + i, slot = at % S::kVSlots;
                    if (run.u.open(a, key0)) continue;
                    if (!wait(kLook, looked & 1) || !wait(kVFull + slot, (at / S::kVSlots) & 1)) { alive = false; break; }
                    ++looked;
                    if (!edge) {   // (the outputs of the piece before are done: the issuing warps have waited for them)
                        for (int e = lane; e < kFlagged * 8; e += 32) flagged[e] = 0;
                        __syncwarp();
                    }
                    uint4* rows = reinterpret_cast<uint4*>(smem + S::kOffV + slot * S::kSlotBytes);   // [64 columns of ..][key][8 pieces of 16 bytes]
                    constexpr uint32_t kExponent = BF16 ? 0x7f807f80u : 0x7c007c00u, kCarry = BF16 ? 0x00800080u : 0x04000400u;
                    uint32_t most = 0;   // the largest magnitude of either half, as a NaN if there is one
                    #pragma unroll 8
                    for (int at_piece = lane; at_piece < S::kSlotBytes / 16; at_piece += 32) {
                        const uint4 v = rows[at_piece];
                        most = largest<BF16>(largest<BF16>(largest<BF16>(most, v.x), largest<BF16>(v.y, v.z)), v.w);
                    }
                    if (__any_sync(0xffffffffu, ((most & kExponent) + kCarry) & 0x80008000u) && edge < kFlagged) {
                        #pragma unroll 1
                        for (int at_piece = lane; at_piece < S::kSlotBytes / 16; at_piece += 32) {
                            const uint4 v = rows[at_piece];
                            uint32_t w[4] = {v.x, v.y, v.z, v.w}, hit = 0;
                            #pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const uint32_t bad = (w[x] & kExponent) + kCarry;
                                hit |= bad & 0x80008000u;
                                if (bad & 0x8000u) w[x] &= 0xffff0000u;
                                if (bad & 0x80000000u) w[x] &= 0x0000ffffu;
                            }
                            if (!hit) continue;
                            rows[at_piece] = make_uint4(w[0], w[1], w[2], w[3]);
                            const int n = at_piece / 8 % kStep;
                            flagged[8 * edge] = key0;
                            atomicOr(&flagged[8 * edge + 1 + n / 32], 1u << (n % 32));
                            *flagged_piece = piece + 1;
                        }
                    }
                    ++edge;
                    fence_proxy_async();   // (the tensor core reads the slot through the async proxy)
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars[kClean]);
                }
                done += tiles;
                ++piece;
            }
        }
    }
    __syncwarp();
    if (*abort_flag) drain_delay();   // (copies that were in flight when a role gave up)
    fence_before();
    __syncthreads();
    if (warp == kIssueWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the pieces of the shared units, in the order the blocks took them: four threads an M-row, eight columns at a time each.
template<int D, bool BF16>
__global__ void __launch_bounds__(256) masked_attention_join_kernel(const __grid_constant__ Args a) {
    constexpr int T = Shape<D>::kTiles, kRuns = D / 32;
    const uint32_t index = (blockIdx.x * 256 + threadIdx.x) / 4, quarter = threadIdx.x % 4, tile = index / kM % T, m = index % kM;
    const Shared share = a.share[index / (T * kM)];
    Unit u;
    u.find(a, share.unit, T * a.tokens);
    const KernelSequence& sequence = a.sequence[u.s];
    const uint32_t token = u.row + tile * a.tokens + m / a.group, head = u.kv * a.group + m % a.group;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (token >= sequence.rows || m >= a.tokens * a.group) return;
    auto slot = [&](uint32_t p) -> size_t { return (2 * (size_t(share.first) + p) + (p == 0 ? 1 : 0)) * T + tile; };
    auto sums_of = [&](uint32_t p) -> float2 { return *reinterpret_cast<const float2*>(a.sums + (slot(p) * kM + m) * 2); };
    auto load = [&](uint32_t p, float4 (&o)[2 * kRuns]) {
        const float4* from = reinterpret_cast<const float4*>(a.partial + (slot(p) * (D / 8) + quarter) * (kM * 8) + m * 8);
        #pragma unroll
        for (int e = 0; e < kRuns; ++e) { o[2 * e] = from[e * kM * 8]; o[2 * e + 1] = from[e * kM * 8 + 1]; }
    };
    // (two pieces at least, most often just two: both are asked for before the maximum is known)
    const float2 first = sums_of(0), second = sums_of(1);
    float4 total[2 * kRuns], other[2 * kRuns];
    load(0, total);
    load(1, other);
    float top = fmaxf(first.x, second.x);
    for (uint32_t p = 2; p < share.pieces; ++p) top = fmaxf(top, sums_of(p).x);
    auto factor_of = [&](float2 v) -> float { return v.x == -INFINITY ? (v.y == 0.0f ? 0.0f : 1.0f) : fast_exp2(v.x - top); };   // (scores that are all NaN leave a NaN sum)
    const float factor = factor_of(first);
    float weight = factor * first.y;
    #pragma unroll
    for (int e = 0; e < 2 * kRuns; ++e) { total[e].x *= factor; total[e].y *= factor; total[e].z *= factor; total[e].w *= factor; }
    auto add = [&](float2 v) {
        const float f = factor_of(v);
        weight = fmaf(f, v.y, weight);
        #pragma unroll
        for (int e = 0; e < 2 * kRuns; ++e) {
            total[e].x = fmaf(f, other[e].x, total[e].x); total[e].y = fmaf(f, other[e].y, total[e].y);
            total[e].z = fmaf(f, other[e].z, total[e].z); total[e].w = fmaf(f, other[e].w, total[e].w);
        }
    };
    add(second);
    for (uint32_t p = 2; p < share.pieces; ++p) { load(p, other); add(sums_of(p)); }
    const float inverse = weight > 0.0f ? 1.0f / weight : weight == 0.0f ? 0.0f : weight;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (size_t(sequence.first_row) + token) * a.out_stride + size_t(head) * D + quarter * 8;
    auto both_of = [&](float x, float y) -> uint32_t { return BF16 ? pack_bf16x2(x * inverse, y * inverse) : pack_half2(x * inverse, y * inverse); };
    #pragma unroll
    for (int e = 0; e < kRuns; ++e)
        *reinterpret_cast<uint4*>(out + 32 * e) = make_uint4(both_of(total[2 * e].x, total[2 * e].y), both_of(total[2 * e].z, total[2 * e].w),
                                                            both_of(total[2 * e + 1].x, total[2 * e + 1].y), both_of(total[2 * e + 1].z, total[2 * e + 1].w));
}

// ---- 8-bit states: codes to 16 bits, exactly, and the blocks' scales in the form the kernel uses ----

struct UnpackSequence {
    const uint8_t* state;
    uint32_t context, length, first_block, blocks;   // blocks of 32 keys, a multiple of four
};
struct UnpackArgs {
    UnpackSequence sequence[kSequences];
    uint32_t sequences, kv_heads, blocks;
    uint16_t* rows;       // [2 * kv_heads][blocks * 32][D]
    float* table;
    const uint16_t* queries;   // BF16 rows to lift, or null
    size_t query_stride;
    uint64_t lifts;            // rows x heads
    uint32_t heads;
    uint16_t* lifted;          // [row][head][D]
    float* factors;            // [row][head]
};

template<int CODE> __device__ __forceinline__ void unpack4(uint32_t w, uint32_t (&out)[2]) {
    float f[4];
    #pragma unroll
    for (int b = 0; b < 4; ++b) {
        if (CODE == kv8::kInt8) f[b] = __uint_as_float(prmt(w ^ 0x80808080u, 0x4b000000u, 0x7440u | b)) - 8388736.0f;   // 2^23 + 128 + c
        else f[b] = __uint_as_float(((w >> (8 * b)) & 0x80u) << 24 | ((w >> (8 * b)) & 0x7fu) << 20) * 1.329227995784916e36f;   // (at 2^-120 of its value)
    }
    out[0] = pack_half2(f[0], f[1]);
    out[1] = pack_half2(f[2], f[3]);
}

// BF16 queries in FP16: a warp a row and head. The whole of it is multiplied by the power of two that brings its largest value to 2^8 (exact, and what lies below
// 2^-25 of that loses its last bits), undone on the scores. So the products of a chunk over 8-bit rows are FP16 ones, whose weights have eleven bits: in BF16
// they had eight, and single tokens eleven. (To 2^14, as there, scores before their factor would leave the range the capped ones' polynomial is for.)
template<int D> __device__ __forceinline__ void lift_queries(const UnpackArgs& a, uint64_t first, uint64_t step) {
    constexpr int kWords = D / 64;
    const int lane = threadIdx.x % 32;
    for (uint64_t at = first; at < a.lifts; at += step) {
        const uint32_t* from = reinterpret_cast<const uint32_t*>(a.queries + at / a.heads * a.query_stride + at % a.heads * D) + lane * kWords;
        uint32_t w[kWords], top = 0;   // magnitudes of BF16 values compare as their bits do
        if constexpr (kWords == 4) { const uint4 v = *reinterpret_cast<const uint4*>(from); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
        else if constexpr (kWords == 2) { const uint2 v = *reinterpret_cast<const uint2*>(from); w[0] = v.x; w[1] = v.y; }
        else w[0] = *from;
        #pragma unroll
        for (int i = 0; i < kWords; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        top = __reduce_max_sync(0xffffffffu, top);
        const int exponent = int(top >> 7);   // biased; 255: an infinity or a NaN among them, left as they are
        const int lift = exponent == 255 || exponent == 0 ? 0 : min(100, 127 + 8 - exponent);
        const float up = __uint_as_float(uint32_t(127 + lift) << 23);
        #pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = pack_half2(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
        uint32_t* to = reinterpret_cast<uint32_t*>(a.lifted + at * D) + lane * kWords;
        if constexpr (kWords == 4) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (kWords == 2) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        else *to = w[0];
        if (lane == 0) a.factors[at] = __uint_as_float(uint32_t(127 - lift) << 23);
    }
}

template<int D, int CODE>
__global__ void __launch_bounds__(128) kv8_unpack_kernel(const __grid_constant__ UnpackArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t planes = 2 * a.kv_heads;
    if (blockIdx.y >= planes + a.kv_heads) {
        const uint64_t block = uint64_t(blockIdx.y - planes - a.kv_heads) * gridDim.x + blockIdx.x, all = uint64_t(gridDim.y - planes - a.kv_heads) * gridDim.x;
        lift_queries<D>(a, block * 4 + threadIdx.x / 32, all * 4);
        return;
    }
    if (blockIdx.y >= planes) {
        // the table of one (sequence, K/V head)
        if (blockIdx.x >= a.sequences) return;
        const UnpackSequence& q = a.sequence[blockIdx.x];
        const uint32_t kv = blockIdx.y - planes, real = (q.length + 31) / 32;
        const float* scales = reinterpret_cast<const float*>(q.state + size_t(planes) * q.context * D);
        const float* k = scales + size_t(kv) * (q.context / 32);
        const float* v = scales + size_t(a.kv_heads + kv) * (q.context / 32);
        float top = 0.0f;
        for (uint32_t i = threadIdx.x; i < real; i += 128) top = fmaxf(top, v[i]);
        #pragma unroll
        for (int offset = 16; offset; offset /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
        __shared__ float tops[4];
        if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
        __syncthreads();
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float floor = fmaxf(log2f(top) - kv8::kScaleRange, kv8::kLowestScale);   // (what is missing below it, `rest`, multiplies P)
        float* to = a.table + (size_t(kv) * a.blocks + q.first_block) * 3;
        for (uint32_t i = threadIdx.x; i < q.blocks; i += 128) {
            const float scale = i < real ? v[i] : 0.0f, exponent = log2f(scale);   // (-inf for a block of zeros: any rest serves)
            float* at = to + i / 4 * 12 + i % 4;
            at[0] = i < real ? k[i] : 0.0f; at[4] = fmaxf(exponent, floor); at[8] = scale > 0.0f && exponent < floor ? exp2f(exponent - floor) : 1.0f;
        }
        return;
    }
    if (blockIdx.x >= a.blocks) return;   // (more sequences than blocks: the grid is as wide as either)
    uint32_t s = 0;
    {
        uint32_t high = a.sequences;
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_block <= blockIdx.x) s = mid; else high = mid; }
    }
    const UnpackSequence& q = a.sequence[s];
    constexpr int kPieces = D / 16, kRows = 128 / kPieces, kPasses = 32 / kRows;
    const uint32_t row = threadIdx.x / kPieces, piece = threadIdx.x % kPieces, key0 = (blockIdx.x - q.first_block) * 32;
    const uint8_t* from = q.state + (size_t(blockIdx.y) * q.context + key0) * D + piece * 16;
    uint16_t* to = a.rows + (size_t(blockIdx.y) * a.blocks * 32 + size_t(blockIdx.x) * 32) * D + piece * 16;
    #pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const uint32_t r = p * kRows + row;
        const uint4 v = key0 + r < q.length ? *reinterpret_cast<const uint4*>(from + size_t(r) * D) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t out[4][2];
        #pragma unroll
        for (int i = 0; i < 4; ++i) unpack4<CODE>(w[i], out[i]);
        uint4* at = reinterpret_cast<uint4*>(to + size_t(r) * D);
        at[0] = make_uint4(out[0][0], out[0][1], out[1][0], out[1][1]);
        at[1] = make_uint4(out[2][0], out[2][1], out[3][0], out[3][1]);
    }
}

// ---- host ----

void check_rule(uint64_t heads, uint64_t kv_heads, uint64_t dim, float scale, float cap, int type) {
    if (!heads || !kv_heads || heads % kv_heads || heads / kv_heads > kM || heads > 65535 || (dim != 64 && dim != 128 && dim != 256))
        throw std::runtime_error("invalid Straydog attention dimensions");
    // (scale / cap is what scores are multiplied by under a cap: an infinity would make a score of 0 a NaN)
    if (!(scale > 0.0f) || !(scale < 1e30f) || !(cap >= 0.0f) || !(cap < 1e30f) || (cap > 0.0f && !(scale / cap < 1e30f))) throw std::runtime_error("invalid Straydog attention scale or cap");
    if (type != kv8::kF16 && type != kv8::kBf16) throw std::runtime_error("masked attention takes F16 (1) or BF16 (30) rows");
}

void check_rows(Device& d, const void* pointer, uint64_t rows, uint64_t stride, uint64_t width, const char* what) {
    if (rows >= uint64_t(1) << 31 || stride < width || stride >= uint64_t(1) << 32) throw std::runtime_error(std::string("invalid rows or row stride of ") + what);
    if (reinterpret_cast<uintptr_t>(pointer) % 16 || stride % 8) throw std::runtime_error(std::string(what) + " lie on 16-byte boundaries");
    if (rows) span(d, pointer, (checked_product({rows - 1, stride}) + width) * 2, what);
}

void check_slopes(Device& d, const float* slopes, uint64_t heads) {
    if (!slopes) return;
    if (reinterpret_cast<uintptr_t>(slopes) % 4) throw std::runtime_error("attention slopes must be 4-byte aligned");
    span(d, slopes, checked_product({heads, 4}), "attention slopes");
}

static CUtensorMap tensor_map(const void* base, bool bf16, uint64_t dim, uint64_t heads, uint64_t rows, uint64_t head_stride, uint64_t row_stride,
                              uint32_t box_heads, uint32_t box_rows) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult found;
        SDB_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !entry) throw std::runtime_error("the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<Encode>(entry);
    }();
    CUtensorMap map;
    const cuuint64_t sizes[3] = {dim, heads, rows}, strides[2] = {head_stride * 2, row_stride * 2};
    const cuuint32_t box[3] = {64, box_heads, box_rows}, steps[3] = {1, 1, 1};
    const CUresult result = encode(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), sizes, strides, box,
                                   steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (result != CUDA_SUCCESS) throw std::runtime_error("no tensor map for the attention rows (driver error " + std::to_string(int(result)) + ")");
    return map;
}

template<int D, bool BF16, bool KV8> static void launch(Device& d, Args& args, bool behind) {
    using S = Shape<D>;
    static bool configured[64] = {};
    if (!configured[d.ordinal & 63]) {
        SDB_CHECK(cudaFuncSetAttribute(masked_attention_kernel<D, BF16, false, KV8>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::kSmem)));
        SDB_CHECK(cudaFuncSetAttribute(masked_attention_kernel<D, BF16, true, KV8>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::kSmem)));
        configured[d.ordinal & 63] = true;
    }
    uint32_t units = 0;
    const uint32_t rows_a_unit = S::kTiles * args.tokens;
    for (uint32_t s = 0; s < args.sequences; ++s) {
        KernelSequence& q = args.sequence[s];
        q.blocks = (q.rows + rows_a_unit - 1) / rows_a_unit;
        q.first_unit = units;
        if (uint64_t(units) + uint64_t(q.blocks) * args.kv_heads >= uint64_t(1) << 30) throw std::runtime_error("too many attention rows in one call");
        units += q.blocks * args.kv_heads;
    }
    // The runs: a unit weighs its tiles and kUnitTiles more. The units of a block of rows, one a K/V head, are alike.
    // (7 documents of up to 2100 rows, 32/8 heads of 128: 2 steps 141.8 us, 3 130.1, 4 133.1, 6 137.4; 12 of 1500, 16/16 heads of 64: 85.4, 81.3, 78.7, 78.6;
    // 9 of 1800, 16/2 heads of 256: 207, 183, 170, 154; 30 of 400, 24/2 heads of 256: 100, 95.4, 95.4, 97.2. Wide heads, whose unit is one tile, would gain by more.)
    constexpr uint32_t kUnitTiles = 3;   // what a unit's first products, masked steps and output cost more, in steps
    uint64_t weight = 0;
    auto each_block = [&](auto&& act) {   // act(first unit, tiles of each of its kv_heads units); false ends
        for (uint32_t s = 0; s < args.sequences; ++s)
            for (uint32_t b = 0; b < args.sequence[s].blocks; ++b) {
                Unit u;
                u.find(args, args.sequence[s].first_unit + b * args.kv_heads, rows_a_unit);
                if (!act(args.sequence[s].first_unit + b * args.kv_heads, u.tiles)) return;
            }
    };
    each_block([&](uint32_t, uint32_t tiles) { weight += uint64_t(tiles + kUnitTiles) * args.kv_heads; return true; });
    // What a run weighs at least, unless there are units enough: fewer and longer runs leave SMs idle, more and shorter ones join more. 4 / 8 / 16: one document
    // of 300 rows, 16/2 heads of 256, 19.1 / 22.6 / 22.6 us; 4 of 100, 32/8 heads of 128, 9.8 / 12.8 / 12.7; one row over 8192 keys 29.4 / 29.7 / 30.8; 16 single rows
    // over 2048 keys 33.7 each; long documents do not notice.
    constexpr uint64_t kLeast = 8;
    const uint32_t blocks = uint32_t(std::max<uint64_t>(1, std::min<uint64_t>(std::min<uint64_t>(uint64_t(d.sms), kMostBlocks), std::max<uint64_t>(weight / kLeast, std::min<uint64_t>(units, weight / 2)))));
    uint64_t passed = 0;
    uint32_t next = 1;
    args.cut[0] = Cut{0, 0};
    each_block([&](uint32_t first, uint32_t tiles) {
        const uint64_t each = tiles + kUnitTiles, end = passed + each * args.kv_heads;
        for (; next < blocks; ++next) {
            const uint64_t target = weight * next / blocks;
            if (target >= end) break;
            const uint64_t inside = (target - passed) / each, offset = (target - passed) % each;   // (offset 0 is the unit's own start)
            // a piece of less than two tiles is left to the neighbour
            const uint32_t tile = offset <= kUnitTiles + 1 ? 0 : uint32_t(offset) - kUnitTiles;
            args.cut[next] = tile && tile + 2 <= tiles ? Cut{first + uint32_t(inside), tile} : Cut{first + uint32_t(inside) + (tile ? 1 : 0), 0};
        }
        passed = end;
        return next < blocks;
    });
    for (; next <= blocks; ++next) args.cut[next] = Cut{units, 0};
    args.shares = 0;
    for (uint32_t b = 1; b < blocks; ++b) {
        if (!args.cut[b].tile) continue;
        if (args.shares && args.share[args.shares - 1].unit == args.cut[b].unit) ++args.share[args.shares - 1].pieces;
        else args.share[args.shares++] = Shared{args.cut[b].unit, b - 1, 2};
    }
    args.status = status_word(d);
    if (args.shares) {
        const size_t rows = size_t(2) * blocks * S::kTiles * kM;
        args.partial = static_cast<float*>(workspace(d, d.kv8_partial, rows * (D + 2) * 4));
        args.sums = args.partial + rows * D;
    }
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = S::kSmem;
    config.stream = d.stream;
    config.attrs = &attribute;
    config.numAttrs = behind ? 1 : 0;
    SDB_CHECK(cudaLaunchKernelEx(&config, args.slopes || args.cap > 0.0f ? masked_attention_kernel<D, BF16, true, KV8> : masked_attention_kernel<D, BF16, false, KV8>, args));
    ++d.launches;
    if (args.shares) {
        config.gridDim = dim3(args.shares * S::kTiles * kM / 64);
        config.blockDim = dim3(256);
        config.dynamicSmemBytes = 0;
        config.numAttrs = 1;
        SDB_CHECK(cudaLaunchKernelEx(&config, masked_attention_join_kernel<D, BF16>, args));
        ++d.launches;
    }
}

template<bool KV8> static void launch_dim(Device& d, uint64_t dim, int type, Args& args, bool behind) {
    const bool bf16 = type == kv8::kBf16;
    if (dim == 64) bf16 ? launch<64, true, KV8>(d, args, behind) : launch<64, false, KV8>(d, args, behind);
    else if (dim == 128) bf16 ? launch<128, true, KV8>(d, args, behind) : launch<128, false, KV8>(d, args, behind);
    else bf16 ? launch<256, true, KV8>(d, args, behind) : launch<256, false, KV8>(d, args, behind);
}

static Args rule_args(uint64_t heads, uint64_t kv_heads, uint64_t dim, float scale, float cap, const float* slopes, uint64_t window, const void* q,
                      uint64_t total_rows, uint64_t q_stride, void* out, uint64_t out_stride, int type) {
    Args args{};
    args.heads = uint32_t(heads); args.kv_heads = uint32_t(kv_heads); args.group = uint32_t(heads / kv_heads); args.tokens = uint32_t(kM / args.group);
    args.window = uint32_t(std::min<uint64_t>(window, uint64_t(1) << 30));
    args.out = out; args.out_stride = out_stride; args.slopes = slopes;
    args.queries = static_cast<const uint16_t*>(q); args.query_stride = q_stride;
    args.scale_log2 = scale * 1.4426950408889634f;
    args.cap = cap * 1.4426950408889634f;
    args.scale_over_cap = cap > 0.0f ? scale / cap : 0.0f;
    args.q_map = tensor_map(q, type == kv8::kBf16, dim, heads, total_rows, dim, q_stride, args.group, args.tokens);
    return args;
}

void attend_kv8(Device& d, const std::vector<Sequence>& sequences, uint64_t heads, uint64_t kv_heads, uint64_t dim, int code, float scale,
                float cap, const float* slopes, uint64_t window, const void* q, uint64_t q_stride, void* out, uint64_t out_stride, int type) {
    const uint64_t total_rows = sequences.back().first_row + sequences.back().rows;
    Args args = rule_args(heads, kv_heads, dim, scale, cap, slopes, window, q, total_rows, q_stride, out, out_stride, type);
    uint64_t lifts = 0;   // (row, head) pairs that the first unpacking launch has to lift
    if (type == kv8::kBf16) {
        args.first_query = uint32_t(sequences.front().first_row);
        lifts = (total_rows - args.first_query) * heads;
        const size_t bytes = checked_product({lifts, dim, 2});
        auto* space = static_cast<uint8_t*>(workspace(d, d.kv8_queries, bytes + lifts * 4));
        args.queries = reinterpret_cast<const uint16_t*>(space); args.query_stride = heads * dim;
        args.query_factors = reinterpret_cast<const float*>(space + bytes);
        args.q_map = tensor_map(space, false, dim, heads, total_rows - args.first_query, dim, heads * dim, args.group, args.tokens);
    }
    constexpr uint64_t kMostBytes = uint64_t(1) << 31;   // unpacked rows a launch, unless one sequence alone has more
    for (size_t at = 0; at < sequences.size();) {
        UnpackArgs unpack{};
        unpack.kv_heads = uint32_t(kv_heads);
        args.sequences = 0;
        uint64_t blocks = 0;
        for (; at < sequences.size() && args.sequences < kSequences; ++at) {
            const Sequence& q = sequences[at];
            const uint64_t more = (q.length + 127) / 128 * 4;
            if (args.sequences && (blocks + more) * 32 * dim * 4 * kv_heads > kMostBytes) break;
            unpack.sequence[args.sequences] = UnpackSequence{q.state, uint32_t(q.context), uint32_t(q.length), uint32_t(blocks), uint32_t(more)};
            KernelSequence& to = args.sequence[args.sequences++];
            to = KernelSequence{uint32_t(q.rows), uint32_t(q.length), uint32_t(q.prefix), uint32_t(q.first_row), uint32_t(blocks * 32), 0, 0, uint32_t(blocks)};
            blocks += more;
        }
        unpack.sequences = args.sequences;
        unpack.blocks = uint32_t(blocks);
        args.block_table = nullptr;
        if (blocks) {
            const size_t row_bytes = checked_product({2 * kv_heads, blocks, 32, dim, 2}), table_bytes = checked_product({kv_heads, blocks, 12});
            auto* space = static_cast<uint8_t*>(workspace(d, d.kv8_rows, row_bytes + table_bytes));
            unpack.rows = reinterpret_cast<uint16_t*>(space);
            unpack.table = reinterpret_cast<float*>(space + row_bytes);
            dim3 grid{unsigned(std::max<uint64_t>(blocks, args.sequences)), unsigned(3 * kv_heads)};
            if (lifts) {
                unpack.queries = static_cast<const uint16_t*>(q) + args.first_query * q_stride; unpack.query_stride = q_stride;
                unpack.lifts = lifts; unpack.heads = uint32_t(heads);
                unpack.lifted = const_cast<uint16_t*>(args.queries); unpack.factors = const_cast<float*>(args.query_factors);
                const uint64_t lifting = (lifts + 15) / 16;   // blocks: four rows and heads a warp, more where the grid would not hold them
                grid.y += unsigned(std::min<uint64_t>((lifting + grid.x - 1) / grid.x, 32768));
                lifts = 0;
            }
            const bool int8 = code == kv8::kInt8;
            auto go = [&](auto* kernel) { kernel<<<grid, 128, 0, d.stream>>>(unpack); };
            if (dim == 64) go(int8 ? kv8_unpack_kernel<64, 0> : kv8_unpack_kernel<64, 1>);
            else if (dim == 128) go(int8 ? kv8_unpack_kernel<128, 0> : kv8_unpack_kernel<128, 1>);
            else go(int8 ? kv8_unpack_kernel<256, 0> : kv8_unpack_kernel<256, 1>);
            ++d.launches;
            const uint64_t keys = blocks * 32;
            args.k_map = tensor_map(unpack.rows, false, dim, kv_heads, keys, keys * dim, dim, 1, kStep);
            args.v_map = tensor_map(unpack.rows + kv_heads * keys * dim, false, dim, kv_heads, keys, keys * dim, dim, 1, kStep);
            args.block_table = unpack.table;
            args.table_blocks = uint32_t(blocks);
        } else {
            args.k_map = args.v_map = args.q_map;   // (no keys: nothing is loaded through them)
        }
        launch_dim<true>(d, dim, type, args, blocks != 0);
    }
}

static void masked(Device& d, const void* q, uint64_t q_stride, const void* k, uint64_t k_stride, const void* v, uint64_t v_stride, const uint64_t* rows,
                   const uint64_t* lengths, uint64_t documents, uint64_t heads, uint64_t kv_heads, uint64_t dim, int type, float scale, float cap,
                   const float* slopes, uint64_t window, const uint64_t* prefixes, void* out, uint64_t out_stride) {
    check_rule(heads, kv_heads, dim, scale, cap, type);
    if (!rows || !lengths || !documents || documents > (uint64_t(1) << 24)) throw std::runtime_error("invalid Straydog attention dimensions");
    if (!q_stride) q_stride = heads * dim;
    if (!out_stride) out_stride = heads * dim;
    if (!k_stride) k_stride = kv_heads * dim;
    if (!v_stride) v_stride = kv_heads * dim;
    uint64_t total = 0, keys = 0;
    for (uint64_t s = 0; s < documents; ++s) {
        if (rows[s] > (uint64_t(1) << 24) || lengths[s] > (uint64_t(1) << 24)) throw std::runtime_error("invalid Straydog attention dimensions");
        total += rows[s]; keys += lengths[s];
    }
    if (!total) return;
    check_rows(d, q, total, q_stride, heads * dim, "attention queries");
    check_rows(d, out, total, out_stride, heads * dim, "an attention output");
    if (keys) check_rows(d, k, keys, k_stride, kv_heads * dim, "attention keys");
    if (keys) check_rows(d, v, keys, v_stride, kv_heads * dim, "attention values");
    check_slopes(d, slopes, heads);
    const size_t out_bytes = ((total - 1) * out_stride + heads * dim) * 2;
    if (kv8::overlap(out, out_bytes, q, ((total - 1) * q_stride + heads * dim) * 2) ||
        (keys && (kv8::overlap(out, out_bytes, k, ((keys - 1) * k_stride + kv_heads * dim) * 2) || kv8::overlap(out, out_bytes, v, ((keys - 1) * v_stride + kv_heads * dim) * 2))))
        throw std::runtime_error("an attention output lies over its queries, keys or values");
    if (slopes && kv8::overlap(out, out_bytes, slopes, heads * 4)) throw std::runtime_error("an attention output lies over the slopes");
    Args args = rule_args(heads, kv_heads, dim, scale, cap, slopes, window, q, total, q_stride, out, out_stride, type);
    args.k_map = keys ? tensor_map(k, type == kv8::kBf16, dim, kv_heads, keys, dim, k_stride, 1, kStep) : args.q_map;
    args.v_map = keys ? tensor_map(v, type == kv8::kBf16, dim, kv_heads, keys, dim, v_stride, 1, kStep) : args.q_map;
    args.values = static_cast<const uint16_t*>(v);
    args.value_stride = v_stride;
    uint64_t row = 0, key = 0;
    for (uint64_t at = 0; at < documents;) {
        args.sequences = 0;
        for (; at < documents && args.sequences < kSequences; ++at) {
            if (rows[at])
                args.sequence[args.sequences++] = KernelSequence{uint32_t(rows[at]), uint32_t(lengths[at]),
                                                                 uint32_t(prefixes ? std::min(prefixes[at], lengths[at]) : 0), uint32_t(row), uint32_t(key), 0, 0, 0};
            row += rows[at]; key += lengths[at];
        }
        if (args.sequences) launch_dim<false>(d, dim, type, args, false);
    }
}

}  // namespace attn
}  // namespace sdb

using namespace sdb;

extern "C" int sdx_masked_attention(void* handle, const void* q, uint64_t q_stride, const void* k, uint64_t k_stride, const void* v, uint64_t v_stride,
                                    const uint64_t* rows, const uint64_t* lengths, uint64_t documents, uint64_t heads, uint64_t kv_heads, uint64_t dim,
                                    int type, float scale, float cap, const float* slopes, uint64_t window, const uint64_t* prefixes, void* out,
                                    uint64_t out_stride) {
    SDB_OP_BEGIN
    attn::masked(value, q, q_stride, k, k_stride, v, v_stride, rows, lengths, documents, heads, kv_heads, dim, type, scale, cap, slopes, window, prefixes, out,
                 out_stride);
    SDB_OP_END
}
