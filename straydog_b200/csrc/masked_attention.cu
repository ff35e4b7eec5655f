// Attention of many query rows under masks and score rules, on the 5th-generation tensor cores (tcgen05.mma, accumulators in TMEM): packed
// documents over 16-bit keys and values (sdx_masked_attention), and prompt chunks over 8-bit states (the codes unpacked to 16 bits first).
//
// Row i of a sequence with n keys and r rows sits at p = n - r + i and sees key j < n when j <= p and j > p - window, or when j < prefix.
//   s = scale * q . k;  s = cap * tanh(s / cap);  s -= slope[head] * |p - j|;  out = softmax over the seen keys . v, zeros where none is seen
//
// A block owns 256 M-rows as two tiles of 128 (one tile for 256 columns): 128 / group consecutive rows times the `group` query heads of one K/V
// head, so K and V are fetched once for all of them and the diagonal is thin. It walks the union of its rows' keys in tiles of 128:
//   S[128 x 128] = Q . K^T    D / 16 tcgen05.mma, Q and K in shared memory (TMA, 128-byte swizzle), FP32 in TMEM
//   O[128 x D]  += P . V      8 tcgen05.mma, P in TMEM over the columns of its S, V in shared memory
// Two tiles a block: while one tile's softmax runs, the tensor pipe works on the other's products. With 256 columns TMEM holds one O and two S,
// and the softmax of one key tile runs beside the products of the next.
// Warps: 0-3 and 4-7 softmax, a thread a row; 8 issues the products; 9 the TMA loads; 10-11 look after values that no row may see (below).
//
// Roundings: scores, maxima, sums and O are FP32. P is rounded to the operands' type once (FP16 or BF16), at 2^7 times its size so that FP16 keeps
// 11 bits down to 2^-21 of the largest weight. O is multiplied in TMEM only when a row's maximum grew by more than 2^8. The keys' scales of an 8-bit
// state multiply the scores, a block of 32 a factor; the values' scales, relative to the largest of the K/V head, join the exponent of P.
//
// A weight of 0 times a value that is infinite or NaN is NaN. In tiles where some row does not see some key (the diagonal, a border), two warps
// replace such values by 0 before the product reads them; the rows that do see them get them back at the end. What no row sees does not reach it.
#include "kv8.cuh"
#include "masked_attention.cuh"
#include "../../include/straydog_gpu_b200.h"

#include <cuda.h>
#include <mutex>

namespace sdb {
namespace attn {

constexpr int kThreads = 384, kTileKeys = 128, kM = 128;
constexpr float kLift = 7.0f, kRescale = 8.0f;
constexpr unsigned kSequences = 64;   // sequences a launch
constexpr int kFlagged = 32;          // tiles of one block with masked values that are not finite (borders: at most a dozen)

template<int D> struct Shape {
    static constexpr int kTiles = D == 256 ? 1 : 2;                  // query tiles a block
    static constexpr int kSlotKeys = D == 256 ? 64 : 128;            // keys of a ring slot: 32 KB (16 KB for 64 columns)
    static constexpr int kHalves = kTileKeys / kSlotKeys;            // slots of a key tile
    static constexpr int kSlots = D == 256 ? 5 : 4;
    static constexpr int kSlotBytes = kSlotKeys * D * 2, kQueryBytes = kM * D * 2;
    static constexpr int kOffRing = kTiles * kQueryBytes, kOffBars = kOffRing + kSlots * kSlotBytes;
    static constexpr int kOffFlags = kOffBars + 512;
    static constexpr size_t kSmem = kOffFlags + kFlagged * 32 + 1024;   // + slack to align the base to 1024 bytes
    static constexpr int kS = 0, kO = 256;                           // TMEM columns: S of tile (or buffer) b at 128 b, O of tile b at 256 + D b
};

struct KernelSequence {
    uint32_t rows, length, prefix, first_row, first_key, first_unit, blocks, first_block;   // first_block: of the unpacked blocks of 32 keys
};
struct Args {
    CUtensorMap q_map, k_map, v_map;
    KernelSequence sequence[kSequences];
    uint32_t sequences, heads, kv_heads, group, tokens;   // tokens: rows of a query tile
    uint32_t splits, window;
    void* out;
    size_t out_stride;
    const float* slopes;
    const float4* block_table;   // 8-bit states: [kv_heads][blocks of 32 keys] key scale, log2 and inverse of the value scale over the head's largest
    const float* value_top;      // 8-bit states: [sequence][kv_heads] the largest value scale
    uint32_t table_blocks;
    const uint16_t* values;      // 16-bit rows: the values again, for the rows that see one that is not finite
    size_t value_stride;
    float scale_log2, cap, scale_over_cap;
    float* partial;              // [unit][split][M-rows][D], then [unit][split][M-rows][2]
    float* sums;
    int* status;
};

enum { kQFull = 0, kSFull = 1, kPFull = 3, kPvDone = 5, kLook = 7, kClean = 8, kRing = 9 };   // barriers: then full and free of every slot

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

// A tile of a packed array: x (columns) on a 16-byte boundary always (a multiple of 64 elements); rows past the array read as zeros.
__device__ __forceinline__ void tma_load(void* to, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(to)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The walk of a block (and split) over its key tiles, the same for every role.
struct Walk {
    uint32_t s, unit, kv, block, split;
    int first, last;                     // positions of the block's first and last row
    uint32_t head_tiles, jump, begin, end;
    template<int TILES> __device__ __forceinline__ void find(const Args& a) {
        unit = blockIdx.x / a.splits;
        split = blockIdx.x % a.splits;
        s = 0;
        uint32_t high = a.sequences;
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_unit <= unit) s = mid; else high = mid; }
        const KernelSequence& q = a.sequence[s];
        const uint32_t inside = unit - q.first_unit;
        kv = inside % a.kv_heads;
        block = q.blocks - 1 - inside / a.kv_heads;   // the longest first
        const uint32_t row = block * TILES * a.tokens;
        first = int(q.length) - int(q.rows) + int(row);
        last = int(q.length) - int(q.rows) + int(min(q.rows, row + TILES * a.tokens)) - 1;
        const uint32_t reach = max(uint32_t(max(last + 1, 0)), q.prefix), low = a.window ? uint32_t(max(0, first - int(a.window) + 1)) : 0u;
        const uint32_t all = (reach + kTileKeys - 1) / kTileKeys;
        head_tiles = (q.prefix + kTileKeys - 1) / kTileKeys;
        const uint32_t body = min(all, max(head_tiles, low / kTileKeys));
        jump = body - head_tiles;
        const uint32_t total = all - jump;
        begin = uint32_t(uint64_t(split) * total / a.splits);
        end = uint32_t(uint64_t(split + 1) * total / a.splits);
    }
    __device__ __forceinline__ uint32_t key(uint32_t tile) const { return (tile < head_tiles ? tile : tile + jump) * kTileKeys; }
    // whether every row of the block sees every key of the tile at key0
    __device__ __forceinline__ bool open(const Args& a, uint32_t key0) const {
        const KernelSequence& q = a.sequence[s];
        const int end_key = int(key0) + kTileKeys - 1;
        return (end_key <= first && end_key < int(q.length) && (!a.window || int(key0) > last - int(a.window))) || end_key < int(q.prefix);
    }
};

template<int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) masked_attention_kernel(const __grid_constant__ Args a) {
    using S = Shape<D>;
    constexpr int T = S::kTiles;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBars);
    constexpr int kFull = kRing, kFree = kRing + S::kSlots, kBars = kRing + 2 * S::kSlots;
    static_assert(kBars * 8 + 16 <= 512, "barriers");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint32_t* flagged_count = tmem_slot + 2;
    uint32_t* flagged = reinterpret_cast<uint32_t*>(smem + S::kOffFlags);   // [entry]: key of the slot, then 4 words of keys

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < kBars; ++i) mbar_init(&bars[i], i == kPFull || i == kPFull + 1 ? 4 : i == kClean ? 2 : 1);
        *abort_flag = 0;
        *flagged_count = 0;
    }
    for (int i = tid; i < kFlagged * 8; i += kThreads) flagged[i] = 0;
    fence_barrier_init();
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    Walk walk;
    walk.find<T>(a);
    const KernelSequence& sequence = a.sequence[walk.s];
    const uint32_t tiles = walk.end - walk.begin;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (unpacked rows are the kernel's before)

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

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int tile_of = T == 2 ? warp / 4 : 0;
        if (warp < 4 * T) {
            // ================= softmax: a thread a row =================
            const int m = (warp & 3) * 32 + lane;
            const uint32_t token = (walk.block * T + tile_of) * a.tokens + m / a.group, head = walk.kv * a.group + m % a.group;
            const bool valid = token < sequence.rows && uint32_t(m) < a.tokens * a.group;
            const int position = int(sequence.length) - int(sequence.rows) + int(token);
            const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
            const uint32_t o_base = lane_base + S::kO + tile_of * D;
            const float slope = a.slopes && valid ? a.slopes[head] * 1.4426950408889634f : 0.0f;
            float top_run = -INFINITY, sum_run = 0.0f;
            bool alive = true;
            #pragma unroll 1
            for (uint32_t i = 0; i < tiles && alive; ++i) {
                const uint32_t key0 = walk.key(walk.begin + i);
                const int buffer = T == 2 ? tile_of : int(i & 1);
                float4 table[4];
                if (a.block_table) {
                    #pragma unroll
                    for (int g = 0; g < 4; ++g) table[g] = __ldg(a.block_table + size_t(walk.kv) * a.table_blocks + sequence.first_block + key0 / 32 + g);
                }
                if (!wait(kSFull + buffer, T == 2 ? i & 1 : (i >> 1) & 1)) { alive = false; break; }
                fence_after();
                const uint32_t s_base = lane_base + S::kS + buffer * 128;
                uint32_t bits[128];
                #pragma unroll
                for (int g = 0; g < 4; ++g) tmem_load32(s_base + 32 * g, bits + 32 * g);
                #pragma unroll
                for (int g = 0; g < 4; ++g) tmem_load_wait(bits + 32 * g);
                float s[128];
                #pragma unroll
                for (int n = 0; n < 128; ++n) s[n] = __uint_as_float(bits[n]);
                float c[4];
                #pragma unroll
                for (int g = 0; g < 4; ++g) c[g] = a.scale_log2 * (a.block_table ? table[g].x : 1.0f);
                if (a.cap > 0.0f) {   // cap * tanh(s / cap), tanh(y) = 1 - 2 / (1 + e^(2 y)): off by 2^-23 of the cap at most
                    #pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float inner = a.scale_over_cap * 2.8853900817779268f * (a.block_table ? table[g].x : 1.0f);
                        #pragma unroll
                        for (int n = 32 * g; n < 32 * g + 32; ++n) s[n] = fmaf(-2.0f * a.cap, fast_rcp(1.0f + fast_exp2(s[n] * inner)), a.cap);
                        c[g] = 1.0f;
                    }
                }
                if (a.slopes) {
                    const float from = float(position - int(key0));
                    #pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        #pragma unroll
                        for (int n = 32 * g; n < 32 * g + 32; ++n) s[n] = fmaf(-slope, fabsf(from - float(n)), s[n] * c[g]);
                        c[g] = 1.0f;
                    }
                }
                if (!walk.open(a, key0)) {
                    // relative to the tile: keys up to `to`, above `low`, or below `prefix` are seen
                    const int to = valid ? min(position, int(sequence.length) - 1) - int(key0) : -1;
                    const int low = a.window ? position - int(a.window) - int(key0) : -1, prefix = valid ? int(sequence.prefix) - int(key0) : 0;
                    #pragma unroll
                    for (int n = 0; n < 128; ++n)
                        if (!((n <= to && n > low) || n < prefix)) s[n] = -INFINITY;
                }
                float top = -INFINITY;
                #pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float t0 = s[32 * g], t1 = s[32 * g + 1];
                    #pragma unroll
                    for (int n = 32 * g + 2; n < 32 * g + 32; n += 2) { t0 = fmaxf(t0, s[n]); t1 = fmaxf(t1, s[n + 1]); }
                    top = fmaxf(top, fmaxf(t0, t1) * c[g]);
                }
                // the old maximum serves while the new one is within 2^8 of it: no pass over O
                const bool grow = top > top_run + kRescale || (top_run == -INFINITY && top > -INFINITY);
                const float use = grow ? top : top_run;
                if (__any_sync(0xffffffffu, grow && top_run != -INFINITY)) {
                    if (!wait(kPvDone + tile_of, (i - 1) & 1)) { alive = false; break; }
                    fence_after();
                    const float factor = grow && top_run != -INFINITY ? fast_exp2(top_run - use) : 1.0f;
                    #pragma unroll 1
                    for (int b = 0; b < D / 32; ++b) {
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
                #pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float shift = (a.block_table ? table[g].y : 0.0f) - under;
                    uint32_t packed[16];
                    float sums[2] = {0.0f, 0.0f};
                    #pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        const float p0 = fast_exp2(fmaf(s[32 * g + 2 * n], c[g], shift)), p1 = fast_exp2(fmaf(s[32 * g + 2 * n + 1], c[g], shift));
                        packed[n] = BF16 ? pack_bf16x2(p0, p1) : pack_half2(p0, p1);
                        sums[0] += p0; sums[1] += p1;
                    }
                    sum_run += (sums[0] + sums[1]) * (a.block_table ? table[g].z : 1.0f);
                    tmem_store16(s_base + 16 * g, packed);
                }
                tmem_store_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[kPFull + buffer]);
            }
            // ---- O / sum ----
            // (the last scores were issued behind all products but the last two of one tile: both are waited for in turn, a barrier's parity
            //  tells neighbouring phases apart only)
            if (T == 1 && alive && tiles > 1 && !wait(kPvDone, (tiles - 2) & 1)) alive = false;
            if (alive && tiles && !wait(kPvDone + tile_of, (tiles - 1) & 1)) alive = false;
            fence_after();
            if (alive) {
                const float lift = a.value_top ? a.value_top[walk.s * a.kv_heads + walk.kv] : 1.0f;
                const float inverse = a.splits > 1 ? lift : sum_run > 0.0f ? lift / sum_run : sum_run == 0.0f ? 0.0f : sum_run;
                const size_t slot = (size_t(blockIdx.x) * T + tile_of) * kM + m;
                const uint32_t patches = min(*reinterpret_cast<volatile uint32_t*>(flagged_count), uint32_t(kFlagged));
                #pragma unroll 1
                for (int b = 0; b < D / 32; ++b) {
                    uint32_t bits[32];
                    float o[32];
                    if (tiles) { tmem_load32(o_base + 32 * b, bits); tmem_load_wait(bits); }
                    #pragma unroll
                    for (int n = 0; n < 32; ++n) o[n] = tiles ? __uint_as_float(bits[n]) : 0.0f;
                    if (!valid) continue;
                    for (uint32_t p = 0; p < patches; ++p) {
                        // values that were taken out of a tile: back for the rows that see them (rare: nothing here is fast)
                        const int base = int(flagged[8 * p]);
                        for (int n = 0; n < S::kSlotKeys; ++n) {
                            if (!(flagged[8 * p + 1 + n / 32] >> (n % 32) & 1)) continue;
                            const int key = base + n;
                            const bool seen = key < int(sequence.length) && ((key <= position && (!a.window || key > position - int(a.window))) || key < int(sequence.prefix));
                            if (!seen) continue;
                            const uint16_t* v = a.values + (size_t(sequence.first_key) + key) * a.value_stride + walk.kv * D + 32 * b;
                            for (int x = 0; x < 32; ++x) {
                                const float f = BF16 ? __uint_as_float(uint32_t(v[x]) << 16) : __half2float(__ushort_as_half(v[x]));
                                if (!(fabsf(f) <= FLT_MAX)) o[x] += f;
                            }
                        }
                    }
                    if (a.splits > 1) {
                        float4* to = reinterpret_cast<float4*>(a.partial + slot * D + 32 * b);
                        #pragma unroll
                        for (int n = 0; n < 8; ++n) to[n] = make_float4(o[4 * n] * inverse, o[4 * n + 1] * inverse, o[4 * n + 2] * inverse, o[4 * n + 3] * inverse);
                    } else {
                        uint4* to = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (size_t(sequence.first_row) + token) * a.out_stride + size_t(head) * D + 32 * b);
                        #pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            uint32_t w[4];
                            #pragma unroll
                            for (int x = 0; x < 4; ++x)
                                w[x] = BF16 ? pack_bf16x2(o[8 * n + 2 * x] * inverse, o[8 * n + 2 * x + 1] * inverse) : pack_half2(o[8 * n + 2 * x] * inverse, o[8 * n + 2 * x + 1] * inverse);
                            to[n] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                if (a.splits > 1 && valid) *reinterpret_cast<float2*>(a.sums + slot * 2) = make_float2(top_run, sum_run);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const uint32_t ring = smem_u32(smem + S::kOffRing);
        // The ring's order, for all roles below: K of the first tile (of two tiles with 256 columns), then V of tile i and K of the next.
        constexpr int kAhead = T == 2 ? 1 : 2;
        if (warp == 8) {
            // ================= the products =================
            if (lane == 0 && tiles) {
                const uint32_t idesc_s = instr_desc(kM, S::kSlotKeys, BF16, false), idesc_o = instr_desc(kM, D, BF16, true);
                const uint32_t queries = smem_u32(smem);
                uint32_t item = 0, looked = 0;
                bool alive = wait(kQFull, 0);
                auto score = [&](int tile, int buffer, uint32_t first_item) -> bool {
                    for (int h = 0; h < S::kHalves; ++h) {
                        const uint32_t at = first_item + h, slot = at % S::kSlots;
                        if (!wait(kFull + slot, (at / S::kSlots) & 1)) return false;
                        fence_after();
                        const uint32_t b = desc_low(ring + slot * S::kSlotBytes, 16), q = desc_low(queries + tile * S::kQueryBytes, 16);
                        #pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            umma(tmem + S::kS + buffer * 128 + h * S::kSlotKeys, desc_of(q + (((kk / 4) * (kM * 128) + (kk % 4) * 32) >> 4)),
                                 desc_of(b + (((kk / 4) * (S::kSlotKeys * 128) + (kk % 4) * 32) >> 4)), idesc_s, kk > 0);
                        if (T == 1 || tile == 1) umma_commit(&bars[kFree + slot]);
                    }
                    umma_commit(&bars[kSFull + buffer]);
                    return true;
                };
                // K tiles: the first kAhead at items 0 .., K(i) for i >= kAhead behind V(i - kAhead)
                auto k_item = [&](uint32_t i) -> uint32_t { return i < uint32_t(kAhead) ? i * S::kHalves : (kAhead + 2 * (i - kAhead) + 1) * S::kHalves; };
                auto v_item = [&](uint32_t i) -> uint32_t {
                    const uint32_t ahead = min(uint32_t(kAhead), tiles);   // (K tiles before V(0); the last V tiles have no K between them)
                    const uint32_t k_before = min(i, tiles - ahead);
                    return (ahead + i + k_before) * S::kHalves;
                };
                for (int f = 0; f < kAhead && uint32_t(f) < tiles && alive; ++f) {
                    if (T == 2) { alive = alive && score(0, 0, 0); alive = alive && score(1, 1, 0); }
                    else alive = alive && score(0, f, k_item(f));
                }
                #pragma unroll 1
                for (uint32_t i = 0; i < tiles && alive; ++i) {
                    const bool look = a.values && !walk.open(a, walk.key(walk.begin + i));
                    item = v_item(i);
                    if (look) {   // (the tile's values are there: they are looked at while the softmax runs)
                        for (int h = 0; h < S::kHalves && alive; ++h) alive = wait(kFull + (item + h) % S::kSlots, ((item + h) / S::kSlots) & 1);
                        if (!alive) break;
                        mbar_arrive(&bars[kLook]);
                    }
                    #pragma unroll 1
                    for (int tile = 0; tile < T && alive; ++tile) {
                        const int buffer = T == 2 ? tile : int(i & 1);
                        if (!wait(kPFull + buffer, T == 2 ? i & 1 : (i >> 1) & 1)) { alive = false; break; }
                        for (int h = 0; h < S::kHalves && alive; ++h) {
                            const uint32_t slot = (item + h) % S::kSlots;
                            if (tile == 0) {
                                if (!wait(kFull + slot, ((item + h) / S::kSlots) & 1)) { alive = false; break; }
                                if (look && h == 0) {
                                    if (!wait(kClean, looked & 1)) { alive = false; break; }
                                    ++looked;
                                }
                            }
                            fence_after();
                            const uint32_t v = desc_low(ring + slot * S::kSlotBytes, S::kSlotKeys * 128);
                            #pragma unroll
                            for (int kk = 0; kk < S::kSlotKeys / 16; ++kk)
                                umma_a_tmem(tmem + S::kO + tile * D, tmem + S::kS + buffer * 128 + h * (S::kSlotKeys / 2) + kk * 8,
                                            desc_of(v + ((kk * (16 * 128)) >> 4)), idesc_o, i > 0 || h > 0 || kk > 0);
                            if (T == 1 || tile == 1) umma_commit(&bars[kFree + slot]);
                        }
                        if (!alive) break;
                        umma_commit(&bars[kPvDone + tile]);
                        if (i + kAhead < tiles) alive = score(tile, buffer, k_item(i + kAhead));
                    }
                }
            }
        } else if (warp == 9) {
            // ================= the loads =================
            if (lane == 0 && tiles) {
                mbar_expect_tx(&bars[kQFull], uint32_t(T * (D / 64)) * a.tokens * a.group * 128);
                #pragma unroll 1
                for (int tile = 0; tile < T; ++tile)
                    for (int x = 0; x < D / 64; ++x)
                        tma_load(smem + tile * S::kQueryBytes + x * (kM * 128), &a.q_map, 64 * x, int(walk.kv * a.group),
                                 int(sequence.first_row + (walk.block * T + tile) * a.tokens), &bars[kQFull]);
                uint32_t item = 0;
                bool alive = true;
                auto load = [&](const CUtensorMap& map, uint32_t i) {
                    const int key = int(sequence.first_key + walk.key(walk.begin + i));
                    for (int h = 0; h < S::kHalves && alive; ++h, ++item) {
                        const uint32_t slot = item % S::kSlots;
                        if (item >= uint32_t(S::kSlots) && !wait(kFree + slot, (item / S::kSlots - 1) & 1)) { alive = false; return; }
                        mbar_expect_tx(&bars[kFull + slot], S::kSlotBytes);
                        for (int x = 0; x < D / 64; ++x)
                            tma_load(smem + S::kOffRing + slot * S::kSlotBytes + x * (S::kSlotKeys * 128), &map, 64 * x, int(walk.kv), key + h * S::kSlotKeys, &bars[kFull + slot]);
                    }
                };
                for (uint32_t i = 0; i < uint32_t(kAhead) && i < tiles; ++i) load(a.k_map, i);
                #pragma unroll 1
                for (uint32_t i = 0; i < tiles && alive; ++i) {
                    load(a.v_map, i);
                    if (alive && i + kAhead < tiles) load(a.k_map, i + kAhead);
                }
            }
        } else if (a.values) {
            // ================= masked values that are not finite =================
            const int t = (warp - 10) * 32 + lane;
            const uint32_t ahead = min(uint32_t(kAhead), tiles);
            int edge = 0;          // slots looked at: the entry of `flagged` is the slot's own
            uint32_t looked = 0;   // tiles looked at (the next is not asked for before this one is done: the barriers' parities cannot be missed)
            bool alive = true;
            #pragma unroll 1
            for (uint32_t i = 0; i < tiles && alive; ++i) {
                const uint32_t key0 = walk.key(walk.begin + i);
                if (walk.open(a, key0)) continue;
                if (!wait(kLook, looked & 1)) break;
                ++looked;
                for (int h = 0; h < S::kHalves; ++h) {
                    const uint32_t at = (ahead + i + min(i, tiles - ahead)) * S::kHalves + h, slot = at % S::kSlots;
                    if (!wait(kFull + slot, (at / S::kSlots) & 1)) { alive = false; break; }
                    uint4* rows = reinterpret_cast<uint4*>(smem + S::kOffRing + slot * S::kSlotBytes);   // [64 columns of ..][key][8 pieces of 16 bytes]
                    constexpr uint32_t kExponent = BF16 ? 0x7f807f80u : 0x7c007c00u, kCarry = BF16 ? 0x00800080u : 0x04000400u;
                    #pragma unroll 1
                    for (int piece = t; piece < S::kSlotBytes / 16 && edge < kFlagged; piece += 64) {
                        const uint4 v = rows[piece];
                        uint32_t w[4] = {v.x, v.y, v.z, v.w}, hit = 0;
                        #pragma unroll
                        for (int x = 0; x < 4; ++x) hit |= (w[x] & kExponent) + kCarry;
                        if (!(hit & 0x80008000u)) continue;
                        #pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t bad = (w[x] & kExponent) + kCarry;
                            if (bad & 0x8000u) w[x] &= 0xffff0000u;
                            if (bad & 0x80000000u) w[x] &= 0x0000ffffu;
                        }
                        rows[piece] = make_uint4(w[0], w[1], w[2], w[3]);
                        const int n = piece / 8 % S::kSlotKeys;
                        flagged[8 * edge] = key0 + h * S::kSlotKeys;
                        atomicOr(&flagged[8 * edge + 1 + n / 32], 1u << (n % 32));
                        atomicMax(flagged_count, uint32_t(edge) + 1);
                    }
                    ++edge;
                }
                fence_proxy_async();   // (the tensor core reads the slots through the async proxy)
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[kClean]);
            }
        }
    }
    __syncwarp();
    if (*abort_flag) drain_delay();   // (copies that were in flight when a role gave up)
    fence_before();
    __syncthreads();
    if (warp == 8) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Warp = M-row: joins the splits of a block's key range.
template<int D, bool BF16>
__global__ void __launch_bounds__(256) masked_attention_join_kernel(const __grid_constant__ Args a) {
    constexpr int T = Shape<D>::kTiles, kEach = D / 32;
    const uint32_t lane = threadIdx.x % 32, index = blockIdx.x * 8 + threadIdx.x / 32, unit = index / (T * kM), tile = index / kM % T, m = index % kM;
    uint32_t s = 0;
    {
        uint32_t high = a.sequences;
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_unit <= unit) s = mid; else high = mid; }
    }
    const KernelSequence& sequence = a.sequence[s];
    const uint32_t inside = unit - sequence.first_unit, kv = inside % a.kv_heads, block = sequence.blocks - 1 - inside / a.kv_heads;
    const uint32_t token = (block * T + tile) * a.tokens + m / a.group, head = kv * a.group + m % a.group;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (token >= sequence.rows || m >= a.tokens * a.group) return;
    float top = -INFINITY, weight = 0.0f, total[kEach];
    #pragma unroll
    for (int e = 0; e < kEach; ++e) total[e] = 0.0f;
    const size_t first = (size_t(unit) * a.splits * T + tile) * kM + m, step = size_t(T) * kM;
    for (uint32_t p = 0; p < a.splits; ++p) top = fmaxf(top, a.sums[(first + p * step) * 2]);
    #pragma unroll 2
    for (uint32_t p = 0; p < a.splits; ++p) {
        const float2 v = *reinterpret_cast<const float2*>(a.sums + (first + p * step) * 2);
        const float factor = v.x == -INFINITY ? (v.y == 0.0f ? 0.0f : 1.0f) : fast_exp2(v.x - top);   // (scores that are all NaN leave a NaN sum)
        weight = fmaf(factor, v.y, weight);
        const float* from = a.partial + (first + p * step) * D;
        #pragma unroll
        for (int e = 0; e < kEach; e += 2) {
            const float2 o = *reinterpret_cast<const float2*>(from + (e / 2 * 32 + lane) * 2);
            total[e] = fmaf(factor, o.x, total[e]); total[e + 1] = fmaf(factor, o.y, total[e + 1]);
        }
    }
    const float inverse = weight > 0.0f ? 1.0f / weight : weight == 0.0f ? 0.0f : weight;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (size_t(sequence.first_row) + token) * a.out_stride + size_t(head) * D;
    #pragma unroll
    for (int e = 0; e < kEach; e += 2)
        *reinterpret_cast<uint32_t*>(out + (e / 2 * 32 + lane) * 2) = BF16 ? pack_bf16x2(total[e] * inverse, total[e + 1] * inverse) : pack_half2(total[e] * inverse, total[e + 1] * inverse);
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
    float4* table;
    float* top;
};

template<int CODE, bool BF16> __device__ __forceinline__ void unpack4(uint32_t w, uint32_t (&out)[2]) {
    float f[4];
    #pragma unroll
    for (int b = 0; b < 4; ++b) {
        if (CODE == kv8::kInt8) f[b] = __uint_as_float(prmt(w ^ 0x80808080u, 0x4b000000u, 0x7440u | b)) - 8388736.0f;   // 2^23 + 128 + c
        else f[b] = __uint_as_float(((w >> (8 * b)) & 0x80u) << 24 | ((w >> (8 * b)) & 0x7fu) << 20) * 1.329227995784916e36f;   // (at 2^-120 of its value)
    }
    out[0] = BF16 ? pack_bf16x2(f[0], f[1]) : pack_half2(f[0], f[1]);
    out[1] = BF16 ? pack_bf16x2(f[2], f[3]) : pack_half2(f[2], f[3]);
}

template<int D, int CODE, bool BF16>
__global__ void __launch_bounds__(128) kv8_unpack_kernel(const __grid_constant__ UnpackArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t planes = 2 * a.kv_heads;
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
        if (!(top > 0.0f)) top = 1.0f;
        if (threadIdx.x == 0) a.top[size_t(blockIdx.x) * a.kv_heads + kv] = top;
        float4* to = a.table + size_t(kv) * a.blocks + q.first_block;
        for (uint32_t i = threadIdx.x; i < q.blocks; i += 128) {
            // (a block of zeros counts as one of scale `top`: its values add nothing. Below 2^-64 of the largest a value scale is taken as that.)
            const float ratio = i < real && v[i] > 0.0f ? fmaxf(v[i] / top, 5.421010862427522e-20f) : 1.0f, down = log2f(ratio);
            to[i] = make_float4(i < real ? fmaxf(k[i], 1e-30f) : 1e-30f, down, 1.0f / fast_exp2(down), 0.0f);
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
        for (int i = 0; i < 4; ++i) unpack4<CODE, BF16>(w[i], out[i]);
        uint4* at = reinterpret_cast<uint4*>(to + size_t(r) * D);
        at[0] = make_uint4(out[0][0], out[0][1], out[1][0], out[1][1]);
        at[1] = make_uint4(out[2][0], out[2][1], out[3][0], out[3][1]);
    }
}

// ---- host ----

void check_rule(uint64_t heads, uint64_t kv_heads, uint64_t dim, float scale, float cap, int type) {
    if (!heads || !kv_heads || heads % kv_heads || heads / kv_heads > kM || heads > 65535 || (dim != 64 && dim != 128 && dim != 256))
        throw std::runtime_error("invalid Straydog attention dimensions");
    if (!(scale > 0.0f) || !(scale < 1e30f) || !(cap >= 0.0f) || !(cap < 1e30f)) throw std::runtime_error("invalid Straydog attention scale or cap");
    if (type != kv8::kF16 && type != kv8::kBf16) throw std::runtime_error("masked attention takes F16 (1) or BF16 (30) rows");
}

void check_rows(Device& d, const void* pointer, uint64_t rows, uint64_t stride, uint64_t width, const char* what) {
    if (rows >= uint64_t(1) << 31 || stride < width || stride >= uint64_t(1) << 32) throw std::runtime_error(std::string("invalid rows or row stride of ") + what);
    if (reinterpret_cast<uintptr_t>(pointer) % 16 || stride % 8) throw std::runtime_error(std::string(what) + " lie on 16-byte boundaries");
    if (rows) span(d, pointer, (checked_product({rows - 1, stride}) + width) * 2, what);
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

template<int D, bool BF16> static void launch(Device& d, Args& args, bool behind) {
    using S = Shape<D>;
    static bool configured[64] = {};
    if (!configured[d.ordinal & 63]) {
        SDB_CHECK(cudaFuncSetAttribute(masked_attention_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::kSmem)));
        configured[d.ordinal & 63] = true;
    }
    uint32_t units = 0, longest = 0;
    for (uint32_t s = 0; s < args.sequences; ++s) {
        KernelSequence& q = args.sequence[s];
        const uint32_t tokens = S::kTiles * args.tokens;
        q.blocks = (q.rows + tokens - 1) / tokens;
        q.first_unit = units;
        if (uint64_t(units) + uint64_t(q.blocks) * args.kv_heads >= uint64_t(1) << 30) throw std::runtime_error("too many attention rows in one call");
        units += q.blocks * args.kv_heads;
        const uint32_t seen = args.window ? std::min(q.length, args.window + tokens + q.prefix) : q.length;
        longest = std::max(longest, (seen + kTileKeys - 1) / kTileKeys);
    }
    // Few blocks: the key range is cut, so that every SM has one; a cut of fewer than four tiles would be mostly prologue
    args.splits = std::max<uint32_t>(1, std::min<uint32_t>(uint32_t(d.sms) / units, longest / 4));
    args.status = status_word(d);
    if (args.splits > 1) {
        const size_t rows = size_t(units) * args.splits * S::kTiles * kM;
        args.partial = static_cast<float*>(workspace(d, d.kv8_partial, rows * (D + 2) * 4));
        args.sums = args.partial + rows * D;
    }
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(units * args.splits);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = S::kSmem;
    config.stream = d.stream;
    config.attrs = &attribute;
    config.numAttrs = behind ? 1 : 0;
    SDB_CHECK(cudaLaunchKernelEx(&config, masked_attention_kernel<D, BF16>, args));
    ++d.launches;
    if (args.splits > 1) {
        config.gridDim = dim3(units * S::kTiles * kM / 8);
        config.blockDim = dim3(256);
        config.dynamicSmemBytes = 0;
        config.numAttrs = 1;
        SDB_CHECK(cudaLaunchKernelEx(&config, masked_attention_join_kernel<D, BF16>, args));
        ++d.launches;
    }
}

static void launch_dim(Device& d, uint64_t dim, int type, Args& args, bool behind) {
    const bool bf16 = type == kv8::kBf16;
    if (dim == 64) bf16 ? launch<64, true>(d, args, behind) : launch<64, false>(d, args, behind);
    else if (dim == 128) bf16 ? launch<128, true>(d, args, behind) : launch<128, false>(d, args, behind);
    else bf16 ? launch<256, true>(d, args, behind) : launch<256, false>(d, args, behind);
}

static Args rule_args(uint64_t heads, uint64_t kv_heads, uint64_t dim, float scale, float cap, const float* slopes, uint64_t window, const void* q,
                      uint64_t total_rows, uint64_t q_stride, void* out, uint64_t out_stride, int type) {
    Args args{};
    args.heads = uint32_t(heads); args.kv_heads = uint32_t(kv_heads); args.group = uint32_t(heads / kv_heads); args.tokens = uint32_t(kM / args.group);
    args.window = uint32_t(std::min<uint64_t>(window, uint64_t(1) << 30));
    args.out = out; args.out_stride = out_stride; args.slopes = slopes;
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
    constexpr uint64_t kMostBytes = uint64_t(1) << 31;   // unpacked rows a launch, unless one sequence alone has more
    for (size_t at = 0; at < sequences.size();) {
        UnpackArgs unpack{};
        unpack.kv_heads = uint32_t(kv_heads);
        args.sequences = 0;
        uint64_t blocks = 0;
        for (; at < sequences.size() && args.sequences < kSequences; ++at) {
            const Sequence& q = sequences[at];
            const uint64_t more = (q.length + kTileKeys - 1) / kTileKeys * 4;
            if (args.sequences && (blocks + more) * 32 * dim * 4 * kv_heads > kMostBytes) break;
            unpack.sequence[args.sequences] = UnpackSequence{q.state, uint32_t(q.context), uint32_t(q.length), uint32_t(blocks), uint32_t(more)};
            KernelSequence& to = args.sequence[args.sequences++];
            to = KernelSequence{uint32_t(q.rows), uint32_t(q.length), uint32_t(q.prefix), uint32_t(q.first_row), uint32_t(blocks * 32), 0, 0, uint32_t(blocks)};
            blocks += more;
        }
        unpack.sequences = args.sequences;
        unpack.blocks = uint32_t(blocks);
        args.block_table = nullptr; args.value_top = nullptr;
        if (blocks) {
            const size_t row_bytes = checked_product({2 * kv_heads, blocks, 32, dim, 2}), table_bytes = checked_product({kv_heads, blocks, 16});
            auto* space = static_cast<uint8_t*>(workspace(d, d.kv8_rows, row_bytes + table_bytes + args.sequences * kv_heads * 4));
            unpack.rows = reinterpret_cast<uint16_t*>(space);
            unpack.table = reinterpret_cast<float4*>(space + row_bytes);
            unpack.top = reinterpret_cast<float*>(space + row_bytes + table_bytes);
            const dim3 grid{unsigned(std::max<uint64_t>(blocks, args.sequences)), unsigned(3 * kv_heads)};
            const bool bf16 = type == kv8::kBf16, int8 = code == kv8::kInt8;
            auto go = [&](auto* kernel) { kernel<<<grid, 128, 0, d.stream>>>(unpack); };
            if (dim == 64) go(int8 ? (bf16 ? kv8_unpack_kernel<64, 0, true> : kv8_unpack_kernel<64, 0, false>) : (bf16 ? kv8_unpack_kernel<64, 1, true> : kv8_unpack_kernel<64, 1, false>));
            else if (dim == 128) go(int8 ? (bf16 ? kv8_unpack_kernel<128, 0, true> : kv8_unpack_kernel<128, 0, false>) : (bf16 ? kv8_unpack_kernel<128, 1, true> : kv8_unpack_kernel<128, 1, false>));
            else go(int8 ? (bf16 ? kv8_unpack_kernel<256, 0, true> : kv8_unpack_kernel<256, 0, false>) : (bf16 ? kv8_unpack_kernel<256, 1, true> : kv8_unpack_kernel<256, 1, false>));
            ++d.launches;
            const uint64_t keys = blocks * 32;
            args.k_map = tensor_map(unpack.rows, bf16, dim, kv_heads, keys, keys * dim, dim, 1, dim == 256 ? Shape<256>::kSlotKeys : kTileKeys);
            args.v_map = tensor_map(unpack.rows + kv_heads * keys * dim, bf16, dim, kv_heads, keys, keys * dim, dim, 1, dim == 256 ? Shape<256>::kSlotKeys : kTileKeys);
            args.block_table = unpack.table;
            args.value_top = unpack.top;
            args.table_blocks = uint32_t(blocks);
        } else {
            args.k_map = args.v_map = args.q_map;   // (no keys: nothing is loaded through them)
        }
        launch_dim(d, dim, type, args, blocks != 0);
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
    if (slopes) span(d, slopes, checked_product({heads, 4}), "attention slopes");
    const size_t out_bytes = ((total - 1) * out_stride + heads * dim) * 2;
    if (kv8::overlap(out, out_bytes, q, ((total - 1) * q_stride + heads * dim) * 2) ||
        (keys && (kv8::overlap(out, out_bytes, k, ((keys - 1) * k_stride + kv_heads * dim) * 2) || kv8::overlap(out, out_bytes, v, ((keys - 1) * v_stride + kv_heads * dim) * 2))))
        throw std::runtime_error("an attention output lies over its queries, keys or values");
    Args args = rule_args(heads, kv_heads, dim, scale, cap, slopes, window, q, total, q_stride, out, out_stride, type);
    const uint32_t slot_keys = dim == 256 ? Shape<256>::kSlotKeys : kTileKeys;
    args.k_map = keys ? tensor_map(k, type == kv8::kBf16, dim, kv_heads, keys, dim, k_stride, 1, slot_keys) : args.q_map;
    args.v_map = keys ? tensor_map(v, type == kv8::kBf16, dim, kv_heads, keys, dim, v_stride, 1, slot_keys) : args.q_map;
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
        if (args.sequences) launch_dim(d, dim, type, args, false);
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
