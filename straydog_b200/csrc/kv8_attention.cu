// Attention of a few query rows a sequence (decode, verification) over states of 8-bit rows with block scales, and the entry that sends
// longer chunks to the prompt kernel (csrc/masked_attention.cu). csrc/kv8.cuh has the layout.
//
//   s(r, j) = scale * q_r . (code_j * key scale of j's block), capped, biased by distance, masked;   out_r = sum_j softmax(s)_j * v_j
//
// The query rows of one K/V head (rows x heads a K/V head: up to 16 at a time, 8 of 256 columns) read its K and V once: 2 * dim bytes a position,
// 8 to 32 flops a byte, so memory binds this. The work of a batch is every sequence's (K/V head, tile of keys) laid end to end and cut into equal
// runs, one a warp (a block of eight warps an SM): ragged lengths balance to within a tile. A warp's run is one piece a (sequence, K/V head) it
// crosses. No warp waits for another: each has a ring of tiles in shared memory filled by its own 16-byte asynchronous copies, two or more tiles
// ahead, pieces' borders not minded. (With the pieces cut a block and the eight warps' sums joined in shared memory, every piece cost its block
// about 5 us of barriers and first loads: 78 us for 16 sequences of 4 rows and 167 MB.) The arithmetic is on mma.sync (16 keys x 8 queries x
// 16 columns): int8 and E4M3 codes become FP16 exactly by byte permutes; the keys' scales multiply the scores in FP32, the values' scales join the weights' exponent. Softmax is
// online, in the exp2 domain. Queries enter as FP16: BF16 rows are multiplied by a power of two that brings their largest value to 2^14 (exact),
// undone on the scores. Weights (times their value scale) enter the value product as FP16 at 2^10 times their size (the running maximum has 2^10):
// 11 bits down to 2^-24 of the largest. A piece that is all of its (sequence, K/V head) writes the output, the others leave FP32 partials that a second kernel joins in
// order. Where a piece is cut depends on the batch, the order of the sums inside it does not.
#include "kv8.cuh"
#include "masked_attention.cuh"
#include "../../include/straydog_gpu_b200.h"

namespace sdb {
namespace kv8 {

using attn::any_tanh;
using attn::either_tanh;
using attn::kFineCap;
using attn::kSmallTanh;
using attn::small_tanh;

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr float kLift = 10.0f;   // log2 of what weights are multiplied by on their way to FP16

// Query rows a K/V head up to which the decode kernel takes a sequence. It reads the codes again for every sixteen (eight) query rows, the prompt kernel
// unpacks them once to 16 bits. Decode / prompt kernel, int8, BF16 rows: 8 heads of 128, 8192 keys, 32 rows 16.8 / 40.0 us, 64 27.9 / 42.2, 128 38.2 / 48.3, 256 61.3 / 49.2;
// 16 sequences of 4096 keys, 32 rows 67 / 159, 64 123 / 161, 96 171 / 161, 128 224 / 161; 4 heads of 64 alike (64 rows 50 / 69, 96 70 / 69), 2 of 256: 48 rows
// 68 / 78, 64 87 / 81. One sequence of 1024 keys stays ahead to 256 rows (18.0 / 23.0 us), which a second rule would gain.
constexpr uint64_t kFewQueries = 64;

struct AttentionSequence {
    const uint8_t* state;
    float* weights;          // [kv_heads][context] or null
    uint32_t context, length, rows, first_row, prefix;
    uint32_t tiles;          // tiles a (K/V head, part)
    uint32_t head_tiles, jump;   // tiles below head_tiles are at their place, the others `jump` tiles further on (keys no row sees are passed over)
    uint32_t first_unit;
    uint32_t parts;          // how often a K/V head's rows are read: query rows over queries a unit
    uint32_t score_queries;  // queries of a tile's scores (a multiple of four)
    uint64_t first_tile;     // of all sequences' tiles
    uint64_t first_score;    // of all sequences' scores
};
struct AttentionArgs {
    AttentionSequence sequence[kSequences];
    uint32_t sequences, heads, kv_heads, group, units;
    uint64_t tiles, tiles_a_warp;
    const void* q;
    void* out;
    const float* slopes;
    size_t q_stride, out_stride;
    float scale_log2, cap, scale_over_cap;
    uint32_t window;
    int bf16;
    float* partial;          // [warp + unit][queries][D]: a run's next piece has the next unit, a unit's next piece the next warp
    float* sums;             // [warp + unit][queries][2]: maximum (exp2 domain, lifted), denominator
    float* scores;           // [tile][keys][score_queries] or null
    float* stats;            // [unit][queries]: final maximum and log2 of the sum, added, for the weights
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// the first `bytes` (16 or 0) of them, zeros in place of the rest
__device__ __forceinline__ void copy16_or_zeros(uint32_t to, const void* from, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
// 1 / a row's sum of weights; 0 for a row that has seen nothing, NaN for one of NaN scores
__device__ __forceinline__ float inverse_of(float sum) { return sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum; }
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// The four codes of a word as two FP16 pairs, exactly: columns (0, 1) and (2, 3) of a key, or columns 0 and 1 of two keys (bytes (0, 2) and
// (1, 3)) of values. int8: a byte behind 0x64 is 1024 + 128 + c of the word xor 0x80808080, less 1152; E4M3: the conversion instruction.
template<int CODE, bool KEYS> __device__ __forceinline__ void pairs_of(uint32_t x, uint32_t& first, uint32_t& second) {
    if (CODE == kInt8) {
        x ^= 0x80808080u;
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t h0 = prmt(x, 0x64646464u, KEYS ? 0x4140u : 0x4240u), h1 = prmt(x, 0x64646464u, KEYS ? 0x4342u : 0x4341u);
        const __half2 r0 = __hsub2(*reinterpret_cast<const __half2*>(&h0), bias), r1 = __hsub2(*reinterpret_cast<const __half2*>(&h1), bias);
        first = *reinterpret_cast<const uint32_t*>(&r0); second = *reinterpret_cast<const uint32_t*>(&r1);
    } else {
        if (!KEYS) x = prmt(x, 0u, 0x3120u);
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(first), "=r"(second) : "r"(x));
    }
}

__device__ __forceinline__ float fast_log2(float x) {   // (-inf for subnormal numbers too: scales of values below 2^-117)
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template<int D, int NT> struct Shape {
    static constexpr int kTile = D == 256 ? 16 : 32;                  // keys a tile: 8 KB of keys and values for D 128 and 256, 4 KB for 64
    static constexpr int kQueries = 8 * NT;
    static constexpr int kPlane = kTile * D, kSlot = 2 * kPlane;      // bytes
    static constexpr int kStages = D == 64 ? 6 : 3;
    static constexpr int kRing = kWarps * kStages * kSlot, kSmem = kRing + kWarps * kStages * 8;
};

// A walk over the tiles of a warp's run: the (sequence, unit) a tile belongs to, without divisions after the first.
struct Place {
    uint32_t s, unit;        // unit: counted over all sequences
    uint64_t begin, end;     // tiles of the unit
    __device__ __forceinline__ void find(const AttentionArgs& a, uint64_t tile) {
        s = 0;
        uint32_t high = a.sequences;
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_tile <= tile) s = mid; else high = mid; }
        const AttentionSequence& q = a.sequence[s];
        const uint32_t inside = uint32_t((tile - q.first_tile) / q.tiles);
        unit = q.first_unit + inside;
        begin = q.first_tile + uint64_t(inside) * q.tiles;
        end = begin + q.tiles;
    }
    __device__ __forceinline__ void next(const AttentionArgs& a) {
        ++unit;
        while (s + 1 < a.sequences && a.sequence[s + 1].first_tile <= end) unit = a.sequence[++s].first_unit;   // (one without tiles shares the next one's first tile)
        begin = end;
        end = begin + a.sequence[s].tiles;
    }
};

template<int D, int NT, int CODE>
__global__ void __launch_bounds__(kThreads, 1) kv8_decode_kernel(const __grid_constant__ AttentionArgs a) {
    using S = Shape<D, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    uint8_t* ring = smem + warp * (S::kStages * S::kSlot);
    float* ring_scales = reinterpret_cast<float*>(smem + S::kRing) + warp * (S::kStages * 2);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const uint64_t run = uint64_t(warp) * gridDim.x + blockIdx.x;   // (few warps are spread over many SMs rather than filling one)
    const uint64_t run_begin = run * a.tiles_a_warp, run_end = min(run_begin + a.tiles_a_warp, a.tiles);
    if (run_begin >= run_end) return;

    // ---- the copies ----
    Place at;
    at.find(a, run_begin);
    Place ahead = at;
    uint64_t ahead_tile = run_begin;
    // Rows are laid in a slot as they lie in memory, their 16-byte pieces exchanged so that the reads below meet in no bank: keys by the
    // row's parity (a read takes 64 bytes of each of two neighbouring rows), values by the row's low bits (a transposing read takes one
    // piece of each of eight rows).
    constexpr int kPieces = D / 16, kStepRows = 32 / kPieces;   // pieces a row, rows a copy instruction of the warp
    const int row0 = lane / kPieces, piece0 = lane % kPieces;
    const uint32_t ring_address = smem_u32(ring), scales_address = smem_u32(ring_scales);
    auto fetch = [&](int slot) {
        if (ahead_tile < run_end) {
            if (ahead_tile >= ahead.end) ahead.next(a);
            const AttentionSequence& q = a.sequence[ahead.s];
            uint32_t tile = uint32_t(ahead_tile - ahead.begin);
            if (tile >= q.head_tiles) tile += q.jump;
            const uint32_t kv = (ahead.unit - q.first_unit) / q.parts, key = tile * S::kTile;
            const size_t k_row = size_t(kv) * q.context + key, v_row = size_t(a.kv_heads + kv) * q.context + key;
            const uint8_t* k_from = q.state + k_row * D + lane * 16;
            const uint8_t* v_from = q.state + v_row * D + lane * 16;
            const uint32_t k_to = ring_address + slot * S::kSlot, v_to = k_to + S::kPlane;
            #pragma unroll
            for (int i = 0; i < S::kTile / kStepRows; ++i) {
                const int row = row0 + i * kStepRows;
                const int k_piece = D == 64 ? piece0 : piece0 ^ (4 * (row & 1));
                copy16(k_to + row * D + k_piece * 16, k_from + i * 512);
            }
            #pragma unroll
            for (int i = 0; i < S::kTile / kStepRows; ++i) {
                const int row = row0 + i * kStepRows;
                const int v_piece = D == 64 ? piece0 ^ ((row >> 1) & 3) : piece0 ^ (row & 7);
                // Rows behind the last one hold whatever was there: a weight of 0 times a code that is a NaN in E4M3 (0x7f, 0xff) would be a NaN
                if (CODE == kE4m3) copy16_or_zeros(v_to + row * D + v_piece * 16, v_from + i * 512, key + row < q.length ? 16u : 0u);
                else copy16(v_to + row * D + v_piece * 16, v_from + i * 512);
            }
            if (lane < 2) {
                const float* scales = reinterpret_cast<const float*>(q.state + size_t(2 * a.kv_heads) * q.context * D);
                copy4(scales_address + slot * 8 + lane * 4, scales + (lane ? v_row : k_row) / kBlock);
            }
            ++ahead_tile;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    #pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) fetch(i);

    const uint32_t v_lane = uint32_t(lane % 8 + 8 * ((lane / 8) & 1));   // the key row this lane's address names in a transposing read
    int slot = 0, fill = S::kStages - 1;
    uint64_t tile_id = run_begin;

    for (;;) {
        // ---- a piece: the part of the run that lies in one (sequence, K/V head, part) ----
        const AttentionSequence& sequence = a.sequence[at.s];
        const uint64_t piece_end = min(at.end, run_end);
        const uint32_t inside = at.unit - sequence.first_unit, kv = inside / sequence.parts, part = inside % sequence.parts;
        const uint32_t first_query = part * S::kQueries, queries = sequence.rows * a.group;

        // the queries as B fragments: lane (g, t) holds query 8n + g, of each 64 columns the sixteen from 16 t
        uint32_t qf[NT][D / 8];
        float unscale[NT][2], slope[NT][2];
        int position[NT][2], low[NT][2];
        uint32_t prefix[NT][2];
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t query = first_query + 8 * n + g, row = query / a.group, head = kv * a.group + query % a.group;
            const bool real = query < queries;
            const uint8_t* from = static_cast<const uint8_t*>(a.q) +
                                  (real ? (size_t(sequence.first_row + row) * a.q_stride + size_t(head) * D + 16 * t) * 2 : 0);
            #pragma unroll
            for (int c = 0; c < D / 64; ++c)
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 v = real ? *reinterpret_cast<const uint4*>(from + c * 128 + i * 16) : make_uint4(0, 0, 0, 0);
                    qf[n][c * 8 + i * 4] = v.x; qf[n][c * 8 + i * 4 + 1] = v.y; qf[n][c * 8 + i * 4 + 2] = v.z; qf[n][c * 8 + i * 4 + 3] = v.w;
                }
            float down = 1.0f;
            if (a.bf16) {
                uint32_t top = 0;   // magnitudes of BF16 values compare as their bits do
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) { top = max(top, qf[n][i] & 0x7fffu); top = max(top, (qf[n][i] >> 16) & 0x7fffu); }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int exponent = int(top >> 7);   // biased; 255: an infinity or a NaN among them, left as they are
                const int lift = exponent == 255 || exponent == 0 ? 0 : min(100, 127 + 14 - exponent);   // (-113 at least)
                const float up = __uint_as_float(uint32_t(127 + lift) << 23);
                down *= __uint_as_float(uint32_t(127 - lift) << 23);
                #pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    qf[n][i] = pack_half2(__uint_as_float(qf[n][i] << 16) * up, __uint_as_float(qf[n][i] & 0xffff0000u) * up);
            }
            #pragma unroll
            for (int i = 0; i < 2; ++i) {   // the queries whose scores this lane will hold
                const uint32_t other = first_query + 8 * n + 2 * t + i, other_row = other / a.group;
                const bool there = other < queries;
                unscale[n][i] = __shfl_sync(0xffffffffu, down, (2 * t + i) * 4);
                position[n][i] = there ? int(sequence.length) - int(sequence.rows) + int(other_row) : -1;
                low[n][i] = a.window ? position[n][i] - int(a.window) : -1;   // keys above this one
                prefix[n][i] = there ? sequence.prefix : 0;
                slope[n][i] = there && a.slopes ? a.slopes[kv * a.group + other % a.group] * 1.4426950408889634f : 0.0f;
            }
        }
        // tiles that every row sees whole need no mask: keys up to `open_to`, above `open_from`, or below `open_prefix`
        const int first_position = int(sequence.length) - int(sequence.rows);
        const int open_to = min(first_position, int(sequence.length) - 1), open_from = a.window ? int(sequence.length) - 1 - int(a.window) : -1;
        const int open_prefix = int(sequence.prefix);
        float o[D / 16][NT][4], m[NT][2], l[NT][2], v_floor = kLowestScale;
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY; l[n][0] = l[n][1] = 0.0f;
            #pragma unroll
            for (int i = 0; i < D / 16; ++i)
                #pragma unroll
                for (int c = 0; c < 4; ++c) o[i][n][c] = 0.0f;
        }

        for (; tile_id < piece_end; ++tile_id) {
            __syncwarp();   // (all lanes are past their reads of the slot to fill)
            fetch(fill);
            fill = fill + 1 == S::kStages ? 0 : fill + 1;
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
            __syncwarp();
            uint32_t tile = uint32_t(tile_id - at.begin);
            if (tile >= sequence.head_tiles) tile += sequence.jump;
            const int key0 = int(tile * S::kTile);
            const uint8_t* kt = ring + slot * S::kSlot;
            const uint32_t vt = ring_address + slot * S::kSlot + S::kPlane;
            const float k_scale = ring_scales[slot * 2], v_scale = ring_scales[slot * 2 + 1];
            // The values' scale joins the weights' exponent: the products with the codes then need no scaling of their own, and the sum of the plain
            // weights is the tile's sum over the scale (a scale of 0 stands over zero codes: any other serves).
            // Below 2^-88, or 2^-64 of the largest the piece has had, it counts as that, and what is missing comes off the weights' exponents on their way to FP16: the sum of
            // plain weights, at 2^10 over the scale each, stays finite with 2^24 keys, and blocks of almost nothing keep their weight in it. So do blocks of
            // zeros, whose maximum must not stand in the way of the others' weights (at a scale of 1 it took all bits of values of 1e-8).
            const float v_true = fast_log2(v_scale), v_log = fmaxf(v_true, v_floor), v_inverse = fast_exp2(-v_log);
            v_floor = fmaxf(v_floor, v_true - kScaleRange);

            // ---- scores ----
            float x[S::kTile / 16][NT][4];
            #pragma unroll
            for (int h = 0; h < S::kTile / 16; ++h) {
                float acc[NT][4];
                #pragma unroll
                for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
                #pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const int piece = D == 64 ? t : (4 * c + t) ^ (4 * (g & 1));
                    const uint4 r0 = *reinterpret_cast<const uint4*>(kt + (16 * h + g) * D + piece * 16);
                    const uint4 r1 = *reinterpret_cast<const uint4*>(kt + (16 * h + g + 8) * D + piece * 16);
                    const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t af[4];
                        pairs_of<CODE, true>(w0[i], af[0], af[2]);
                        pairs_of<CODE, true>(w1[i], af[1], af[3]);
                        #pragma unroll
                        for (int n = 0; n < NT; ++n) mma_f16(acc[n], af, qf[n][c * 8 + 2 * i], qf[n][c * 8 + 2 * i + 1]);
                    }
                }
                #pragma unroll
                for (int n = 0; n < NT; ++n)
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) x[h][n][c] = acc[n][c];
            }
            const float to_score = k_scale * (a.cap > 0.0f ? a.scale_over_cap : a.scale_log2);
            #pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float factor[2] = {to_score * unscale[n][0], to_score * unscale[n][1]};
                #pragma unroll
                for (int h = 0; h < S::kTile / 16; ++h)
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) x[h][n][c] = fmaf(x[h][n][c], factor[c & 1], a.cap > 0.0f ? 0.0f : v_log);
            }
            if (a.cap > 0.0f) {   // (the cap is in the exp2 domain too)
                bool small = true;
                #pragma unroll
                for (int h = 0; h < S::kTile / 16; ++h)
                    #pragma unroll
                    for (int n = 0; n < NT; ++n)
                        #pragma unroll
                        for (int c = 0; c < 4; ++c) small &= fabsf(x[h][n][c]) <= kSmallTanh;
                auto capped = [&](auto&& tanh_of) {
                    #pragma unroll
                    for (int h = 0; h < S::kTile / 16; ++h)
                        #pragma unroll
                        for (int n = 0; n < NT; ++n)
                            #pragma unroll
                            for (int c = 0; c < 4; ++c) x[h][n][c] = fmaf(a.cap, tanh_of(x[h][n][c]), v_log);
                };
                if (__all_sync(0xffffffffu, small)) capped([](float y) { return small_tanh(y); });   // (the usual case: scores well below the cap)
                else if (a.cap <= kFineCap) capped([](float y) { return any_tanh(y); });
                else capped([](float y) { return either_tanh(y); });
            }
            if (a.slopes) {
                #pragma unroll
                for (int h = 0; h < S::kTile / 16; ++h)
                    #pragma unroll
                    for (int n = 0; n < NT; ++n)
                        #pragma unroll
                        for (int c = 0; c < 4; ++c)
                            x[h][n][c] = fmaf(-slope[n][c & 1], fabsf(float(position[n][c & 1] - (key0 + 16 * h + g + 8 * (c >> 1)))), x[h][n][c]);
            }
            if (!((key0 + S::kTile - 1 <= open_to && key0 > open_from) || key0 + S::kTile <= open_prefix)) {
                #pragma unroll
                for (int h = 0; h < S::kTile / 16; ++h)
                    #pragma unroll
                    for (int n = 0; n < NT; ++n)
                        #pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int i = c & 1, key = key0 + 16 * h + g + 8 * (c >> 1);
                            const bool seen = ((key <= position[n][i] && key > low[n][i]) || uint32_t(key) < prefix[n][i]) && key < int(sequence.length);
                            if (!seen) x[h][n][c] = -INFINITY;
                        }
            }
            if (a.scores) {
                const uint32_t queries_kept = sequence.score_queries;
                float* to = a.scores + sequence.first_score + (tile_id - sequence.first_tile) * (S::kTile * queries_kept);
                #pragma unroll
                for (int h = 0; h < S::kTile / 16; ++h)
                    #pragma unroll
                    for (int n = 0; n < NT; ++n)
                        #pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (8 * n + 2 * t < int(queries_kept))
                                *reinterpret_cast<float2*>(to + (16 * h + g + 8 * i) * queries_kept + 8 * n + 2 * t) = make_float2(x[h][n][2 * i] - v_log, x[h][n][2 * i + 1] - v_log);
            }
            // ---- the running maximum (lifted) and the weights ----
            bool grew = false;
            float now[NT][2];
            #pragma unroll
            for (int n = 0; n < NT; ++n)
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = fmaxf(x[0][n][i], x[0][n][i + 2]);
                    #pragma unroll
                    for (int h = 1; h < S::kTile / 16; ++h) top = fmaxf(top, fmaxf(x[h][n][i], x[h][n][i + 2]));
                    #pragma unroll
                    for (int offset = 4; offset < 32; offset *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
                    now[n][i] = fmaxf(m[n][i], top - kLift);
                    grew |= now[n][i] > m[n][i];
                }
            if (__any_sync(0xffffffffu, grew)) {
                #pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // (the sum in two steps: from a block of zeros to one of large values the factor alone may be too small for FP32, the sum is not)
                    const float h0 = m[n][0] == -INFINITY ? 0.0f : fast_exp2(0.5f * (m[n][0] - now[n][0])), h1 = m[n][1] == -INFINITY ? 0.0f : fast_exp2(0.5f * (m[n][1] - now[n][1]));
                    const float f0 = h0 * h0, f1 = h1 * h1;
                    l[n][0] = l[n][0] * h0 * h0; l[n][1] = l[n][1] * h1 * h1; m[n][0] = now[n][0]; m[n][1] = now[n][1];
                    #pragma unroll
                    for (int i = 0; i < D / 16; ++i) { o[i][n][0] *= f0; o[i][n][1] *= f1; o[i][n][2] *= f0; o[i][n][3] *= f1; }
                }
            }
            uint32_t pf[S::kTile / 16][NT][2];
            #pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float u0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], u1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];   // (nothing seen so far: every weight 0)
                float sum0 = 0.0f, sum1 = 0.0f;
                #pragma unroll
                for (int h = 0; h < S::kTile / 16; ++h) {
                    const float p0 = fast_exp2(x[h][n][0] - u0), p1 = fast_exp2(x[h][n][1] - u1), p2 = fast_exp2(x[h][n][2] - u0), p3 = fast_exp2(x[h][n][3] - u1);
                    sum0 += p0 + p2; sum1 += p1 + p3;
                    pf[h][n][0] = movmatrix_trans(pack_half2(p0, p1));
                    pf[h][n][1] = movmatrix_trans(pack_half2(p2, p3));
                }
                l[n][0] = fmaf(sum0, v_inverse, l[n][0]); l[n][1] = fmaf(sum1, v_inverse, l[n][1]);
            }
            if (v_true < v_log) {
                #pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float u0 = (m[n][0] == -INFINITY ? 0.0f : m[n][0]) + (v_log - v_true), u1 = (m[n][1] == -INFINITY ? 0.0f : m[n][1]) + (v_log - v_true);
                    #pragma unroll
                    for (int h = 0; h < S::kTile / 16; ++h) {
                        pf[h][n][0] = movmatrix_trans(pack_half2(fast_exp2(x[h][n][0] - u0), fast_exp2(x[h][n][1] - u1)));
                        pf[h][n][1] = movmatrix_trans(pack_half2(fast_exp2(x[h][n][2] - u0), fast_exp2(x[h][n][3] - u1)));
                    }
                }
            }
            // ---- O^T += V^T P^T ----
            #pragma unroll
            for (int b = 0; b < D / 32; ++b)
                #pragma unroll
                for (int h = 0; h < S::kTile / 16; ++h) {
                    const uint32_t row = v_lane + 16 * h, piece = (2 * b + lane / 16) ^ (D == 64 ? (row >> 1) & 3 : row & 7);
                    uint32_t w[4];   // w[0], w[1]: columns 32b + 2g, + 1 of keys (2t, 2t + 1) and (2t + 8, 2t + 9); w[2], w[3]: columns 32b + 16 + 2g, + 1
                    ldmatrix_x4_trans(w, vt + row * D + piece * 16);
                    uint32_t af[4], ag[4];
                    pairs_of<CODE, false>(w[0], af[0], af[1]);
                    pairs_of<CODE, false>(w[1], af[2], af[3]);
                    pairs_of<CODE, false>(w[2], ag[0], ag[1]);
                    pairs_of<CODE, false>(w[3], ag[2], ag[3]);
                    #pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_f16(o[2 * b][n], af, pf[h][n][0], pf[h][n][1]);
                        mma_f16(o[2 * b + 1][n], ag, pf[h][n][0], pf[h][n][1]);
                    }
                }
            if (++slot == S::kStages) slot = 0;
        }

        // ---- the piece's sums: o[i][n][c] is query 8n + 2t + (c & 1), column 16i + 2g + (c >> 1) ----
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int i = 0; i < 2; ++i)
                #pragma unroll
                for (int offset = 4; offset < 32; offset *= 2) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], offset);
        const bool whole = piece_end - max(at.begin, run_begin) == sequence.tiles;   // the piece is all of its unit
        const size_t mine = size_t(run) + at.unit;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int query = 8 * n + 2 * t + i;
                const uint32_t global = first_query + query;
                if (global >= queries) continue;
                if (whole) {
                    const float inverse = inverse_of(l[n][i]);
                    uint16_t* to = static_cast<uint16_t*>(a.out) + size_t(sequence.first_row + global / a.group) * a.out_stride + size_t(kv * a.group + global % a.group) * D + 2 * g;
                    #pragma unroll
                    for (int b = 0; b < D / 16; ++b) {
                        const float v0 = o[b][n][i] * inverse, v1 = o[b][n][i + 2] * inverse;
                        *reinterpret_cast<uint32_t*>(to + 16 * b) = a.bf16 ? pack_bf16x2(v0, v1) : pack_half2(v0, v1);
                    }
                    if (a.scores && g == 0) a.stats[size_t(at.unit) * S::kQueries + query] = m[n][i] + log2f(l[n][i]);
                } else {
                    float* to = a.partial + (mine * S::kQueries + query) * D + 2 * g;
                    #pragma unroll
                    for (int b = 0; b < D / 16; ++b) *reinterpret_cast<float2*>(to + 16 * b) = make_float2(o[b][n][i], o[b][n][i + 2]);
                    if (g == 0) *reinterpret_cast<float2*>(a.sums + (mine * S::kQueries + query) * 2) = make_float2(m[n][i], l[n][i]);
                }
            }
        if (piece_end == run_end) break;
        at.next(a);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Block = (unit, query): joins the partials of a unit that several warps worked on, and zeroes the rows of a sequence without keys.
// Few partials (a batch of many sequences): 128 threads, so that all blocks run at once (4 verification rows of 16 sequences: 55.3 us against 65.6 with
// 512; 64 sequences of up to 32768 keys: 196 against 203); many (one long sequence): 512. Where those are few blocks with long sums, four (two) of them share a row's columns: one
// row of 8192 keys, 16/2 heads of 256 11.8 us against 17.9, 32768 keys 17.2 against 23.2; with 64 partials (1024 keys) 8.3 against 7.6, with 64 query rows
// 22.0 against 20.0, so from more than 64 partials on, and up to two blocks an SM.
constexpr int kMostWarps = 2048, kFewPieces = 32;   // warps of a launch (eight an SM)
template<int D, int kJoinThreads, int kColumns>   // kColumns: how many of a row's D / 4 pieces a block joins
__global__ void __launch_bounds__(kJoinThreads) kv8_decode_join_kernel(const __grid_constant__ AttentionArgs a, uint32_t queries_a_unit) {
    constexpr int kRow = D / 4, kGroups = kJoinThreads / kColumns;   // partials at a time
    constexpr int kMost = kJoinThreads == 128 ? kFewPieces : kMostWarps, kSums = (kMost + kJoinThreads - 1) / kJoinThreads;
    __shared__ float factors[kMost];
    __shared__ float tops[kJoinThreads / 32], weights[kJoinThreads / 32];
    __shared__ float4 totals[kGroups][kColumns];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t unit = blockIdx.x, query = blockIdx.y;
    uint32_t s = 0;
    {
        uint32_t high = a.sequences;
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_unit <= unit) s = mid; else high = mid; }
    }
    const AttentionSequence& sequence = a.sequence[s];
    const uint32_t inside = unit - sequence.first_unit, kv = inside / sequence.parts, global = inside % sequence.parts * queries_a_unit + query;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (in every block: what is launched behind this one counts on the decode's end too)
    if (global >= sequence.rows * a.group) return;
    uint16_t* out = static_cast<uint16_t*>(a.out) + size_t(sequence.first_row + global / a.group) * a.out_stride + size_t(kv * a.group + global % a.group) * D;
    if (!sequence.tiles) {
        if (threadIdx.x < kColumns) *reinterpret_cast<uint2*>(out + 4 * (blockIdx.z * kColumns + threadIdx.x)) = make_uint2(0, 0);
        return;
    }
    const uint64_t begin = sequence.first_tile + uint64_t(inside) * sequence.tiles, end = begin + sequence.tiles;
    const uint32_t first = uint32_t(begin / a.tiles_a_warp), pieces = uint32_t((end - 1) / a.tiles_a_warp) - first + 1;
    if (pieces == 1) return;
    const float2* sums = reinterpret_cast<const float2*>(a.sums) + (size_t(first) + unit) * queries_a_unit + query;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, column = threadIdx.x % kColumns, group = threadIdx.x / kColumns, from_column = blockIdx.z * kColumns;
    const float4* partial = reinterpret_cast<const float4*>(a.partial + ((size_t(first) + unit) * queries_a_unit + query) * D) + from_column + column;
    // the first partials are asked for before the maximum is known
    constexpr int kAhead = 4;
    float4 v[kAhead];
    #pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const uint32_t p = group + i * kGroups;
        v[i] = p < pieces ? partial[size_t(p) * queries_a_unit * kRow] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float2 mine[kSums];
    float top = -INFINITY;
    #pragma unroll
    for (int i = 0; i < kSums; ++i) {
        const uint32_t p = threadIdx.x + i * kJoinThreads;
        mine[i] = p < pieces ? sums[size_t(p) * queries_a_unit] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, mine[i].x);
    }
    #pragma unroll
    for (int offset = 16; offset; offset /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    top = tops[0];
    #pragma unroll
    for (int w = 1; w < kJoinThreads / 32; ++w) top = fmaxf(top, tops[w]);
    float weight = 0.0f;
    #pragma unroll
    for (int i = 0; i < kSums; ++i) {
        const uint32_t p = threadIdx.x + i * kJoinThreads;
        // (nothing seen in a piece: no weight; scores that are all NaN leave a NaN sum, which stays)
        const float root = mine[i].y == 0.0f ? 0.0f : mine[i].x == -INFINITY ? 1.0f : fast_exp2(0.5f * (mine[i].x - top));
        if (p < pieces) factors[p] = root * root;
        weight = fmaf(root * mine[i].y, root, weight);   // (in two steps, as in the decode kernel)
    }
    #pragma unroll
    for (int offset = 16; offset; offset /= 2) weight += __shfl_xor_sync(0xffffffffu, weight, offset);
    if (lane == 0) weights[warp] = weight;
    __syncthreads();
    weight = 0.0f;
    #pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) weight += weights[w];
    float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t from = group; from < pieces; from += kAhead * kGroups) {
        float4 next[kAhead];
        #pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t p = from + (kAhead + i) * kGroups;
            next[i] = p < pieces ? partial[size_t(p) * queries_a_unit * kRow] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        #pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t p = from + i * kGroups;
            const float factor = p < pieces ? factors[p] : 0.0f;
            total.x = fmaf(factor, v[i].x, total.x); total.y = fmaf(factor, v[i].y, total.y);
            total.z = fmaf(factor, v[i].z, total.z); total.w = fmaf(factor, v[i].w, total.w);
            v[i] = next[i];
        }
    }
    totals[group][column] = total;
    __syncthreads();
    const float inverse = inverse_of(weight);
    if (a.scores && threadIdx.x == 0 && blockIdx.z == 0) a.stats[size_t(unit) * queries_a_unit + query] = top + log2f(weight);
    if (threadIdx.x >= kColumns) return;
    #pragma unroll
    for (int i = 1; i < kGroups; ++i) {
        const float4 other = totals[i][column];
        total.x += other.x; total.y += other.y; total.z += other.z; total.w += other.w;
    }
    *reinterpret_cast<uint2*>(out + 4 * (from_column + column)) = a.bf16 ? make_uint2(pack_bf16x2(total.x * inverse, total.y * inverse), pack_bf16x2(total.z * inverse, total.w * inverse))
                                                       : make_uint2(pack_half2(total.x * inverse, total.y * inverse), pack_half2(total.z * inverse, total.w * inverse));
}

// Thread = a seen key of the block's (sequence, K/V head): its weights over the K/V head's query rows, from the scores the attention left, added to the
// running sums. Launched behind the join as its programmatic dependent.
template<int TILE, int QUERIES>
__global__ void __launch_bounds__(256) kv8_weights_kernel(const __grid_constant__ AttentionArgs a) {
    const AttentionSequence& sequence = a.sequence[blockIdx.y];
    const uint32_t kv = blockIdx.z, at = blockIdx.x * 256 + threadIdx.x, keys = sequence.tiles * TILE;
    uint32_t tile = at / TILE;
    if (tile >= sequence.head_tiles) tile += sequence.jump;
    const uint32_t key = tile * TILE + at % TILE, kept = sequence.score_queries;
    const bool there = at < keys && key < sequence.length;
    __shared__ float stat[kFewQueries];
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (in every block, as in the join)
    if (blockIdx.x * 256 >= keys) return;
    const uint32_t all = sequence.rows * a.group;
    if (threadIdx.x < all)
        stat[threadIdx.x] = a.stats[size_t(sequence.first_unit + kv * sequence.parts + threadIdx.x / QUERIES) * QUERIES + threadIdx.x % QUERIES];
    __syncthreads();
    if (!there) return;
    float total = 0.0f;
    for (uint32_t part = 0; part < sequence.parts; ++part) {
        const uint32_t queries = min(uint32_t(QUERIES), all - part * QUERIES);
        const float4* scores = reinterpret_cast<const float4*>(a.scores + sequence.first_score + (uint64_t(kv * sequence.parts + part) * sequence.tiles * TILE + at) * kept);
        #pragma unroll
        for (int i = 0; i < QUERIES / 4; ++i) {
            if (uint32_t(4 * i) >= queries) break;
            const float4 v = scores[i];
            const float x[4] = {v.x, v.y, v.z, v.w};
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (uint32_t(4 * i + c) >= queries) continue;
                if (x[c] != -INFINITY) total += fast_exp2(x[c] - stat[part * QUERIES + 4 * i + c]);
            }
        }
    }
    sequence.weights[size_t(kv) * sequence.context + key] += total;
}

template<int D, int NT, int CODE> static void launch_decode(Device& d, AttentionArgs& args, bool weights) {
    using S = Shape<D, NT>;
    args.units = 0; args.tiles = 0;
    uint64_t most_keys = 0, score_floats = 0, joined = 0;   // joined: query rows a unit, over the units
    bool empty = false;
    for (uint32_t s = 0; s < args.sequences; ++s) {
        AttentionSequence& q = args.sequence[s];
        const uint64_t low = args.window && q.length + 1 > uint64_t(q.rows) + args.window ? q.length + 1 - q.rows - args.window : 0;   // the first row's first key
        const uint32_t all = uint32_t((q.length + S::kTile - 1) / S::kTile);
        q.head_tiles = uint32_t((q.prefix + S::kTile - 1) / S::kTile);
        const uint32_t body = std::min(all, std::max(q.head_tiles, uint32_t(low / S::kTile)));
        q.jump = body - std::min(body, q.head_tiles);
        q.tiles = all - q.jump;
        q.parts = (q.rows * args.group + S::kQueries - 1) / S::kQueries;
        q.first_unit = args.units;
        q.first_tile = args.tiles;
        q.score_queries = std::min<uint32_t>(S::kQueries, (q.rows * args.group + 3) / 4 * 4);
        q.first_score = score_floats;
        score_floats += uint64_t(args.kv_heads) * q.parts * q.tiles * S::kTile * q.score_queries;
        args.units += args.kv_heads * q.parts;
        joined += uint64_t(args.kv_heads) * q.rows * args.group;
        args.tiles += uint64_t(args.kv_heads) * q.parts * q.tiles;
        most_keys = std::max(most_keys, uint64_t(q.tiles) * S::kTile);
        empty |= !q.tiles;
    }
    // One block an SM; a warp takes a tile at least
    const uint64_t warps = std::max<uint64_t>(1, std::min<uint64_t>(std::min<uint64_t>(uint64_t(d.sms) * kWarps, kMostWarps), args.tiles));
    const uint64_t blocks = std::min<uint64_t>(uint64_t(d.sms), warps);
    args.tiles_a_warp = std::max<uint64_t>(1, (args.tiles + warps - 1) / warps);
    const size_t slots = blocks * kWarps + args.units;
    uint64_t pieces = 0;   // of the unit that most warps work on
    for (uint32_t s = 0; s < args.sequences; ++s) {
        const AttentionSequence& q = args.sequence[s];
        for (uint32_t u = 0; u < args.kv_heads * q.parts && q.tiles; ++u) {
            const uint64_t begin = q.first_tile + uint64_t(u) * q.tiles;
            pieces = std::max(pieces, (begin + q.tiles - 1) / args.tiles_a_warp - begin / args.tiles_a_warp + 1);
        }
    }
    const bool cut = pieces > 1;
    const size_t partial_floats = cut ? slots * S::kQueries * D : 0, sums_floats = cut ? slots * S::kQueries * 2 : 0;
    float* partial = cut ? static_cast<float*>(workspace(d, d.kv8_partial, (partial_floats + sums_floats) * 4)) : nullptr;
    args.partial = partial;
    args.sums = partial + partial_floats;
    args.scores = args.stats = nullptr;
    if (weights && args.tiles) {
        args.scores = static_cast<float*>(workspace(d, d.kv8_scores, checked_product({score_floats + uint64_t(args.units) * S::kQueries, 4})));
        args.stats = args.scores + score_floats;
    }
    static bool configured[64] = {};
    if (!configured[d.ordinal & 63]) {
        SDB_CHECK(cudaFuncSetAttribute(kv8_decode_kernel<D, NT, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        configured[d.ordinal & 63] = true;
    }
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    bool behind = false;   // a kernel of this call is ahead in the stream: the next is its programmatic dependent
    if (args.tiles) {
        kv8_decode_kernel<D, NT, CODE><<<unsigned(blocks), kThreads, S::kSmem, d.stream>>>(args);
        ++d.launches;
        behind = true;
    }
    if (cut || empty) {
        const bool few = pieces <= kFewPieces, share = pieces > 64 && joined * (D / 64) <= uint64_t(d.sms) * 2;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(args.units, S::kQueries, share ? D / 64 : 1);
        config.blockDim = dim3(few ? 128 : 512);
        config.stream = d.stream;
        config.attrs = &attribute;
        config.numAttrs = behind ? 1 : 0;
        SDB_CHECK(cudaLaunchKernelEx(&config, few ? kv8_decode_join_kernel<D, 128, D / 4> : share ? kv8_decode_join_kernel<D, 512, 16> : kv8_decode_join_kernel<D, 512, D / 4>,
                                     args, uint32_t(S::kQueries)));
        ++d.launches;
    }
    if (args.scores) {
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(unsigned((most_keys + 255) / 256), args.sequences, args.kv_heads);
        config.blockDim = dim3(256);
        config.stream = d.stream;
        config.attrs = &attribute;
        config.numAttrs = 1;
        SDB_CHECK(cudaLaunchKernelEx(&config, kv8_weights_kernel<S::kTile, S::kQueries>, args));
        ++d.launches;
    }
}

template<int D> static void launch_queries(Device& d, AttentionArgs& args, int code, bool weights, bool two) {
    constexpr int kTwo = D == 256 ? 1 : 2;   // (256 columns: queries and sums of sixteen rows would not fit the registers; they are read in two parts)
    if (two && code == kInt8) launch_decode<D, kTwo, kInt8>(d, args, weights);
    else if (two) launch_decode<D, kTwo, kE4m3>(d, args, weights);
    else if (code == kInt8) launch_decode<D, 1, kInt8>(d, args, weights);
    else launch_decode<D, 1, kE4m3>(d, args, weights);
}

static void attention(Device& d, const void* const* states, const uint64_t* contexts, const uint64_t* lengths, const uint64_t* rows,
                      uint64_t sequences, uint64_t heads, uint64_t kv_heads, uint64_t dim, int code, float scale, float cap, const float* slopes,
                      uint64_t window, const uint64_t* prefixes, const void* q, uint64_t q_stride, float* const* weights, void* out,
                      uint64_t out_stride, int type) {
    check_shape(sequences, kv_heads, dim, code);
    attn::check_rule(heads, kv_heads, dim, scale, cap, type);
    if (!states || !contexts || !lengths || !rows) throw std::runtime_error("invalid Straydog attention dimensions");
    const uint64_t group = heads / kv_heads;
    if (!q_stride) q_stride = heads * dim;
    if (!out_stride) out_stride = heads * dim;
    uint64_t total = 0;
    for (uint64_t s = 0; s < sequences; ++s) {
        check_state(d, states[s], contexts[s], kv_heads, dim);
        if (lengths[s] > contexts[s] || rows[s] > (uint64_t(1) << 24)) throw std::runtime_error("invalid Straydog attention dimensions");
        if (weights) {
            if (rows[s] * group > kFewQueries) throw std::runtime_error("attention weights are added up for at most 64 query rows a K/V head");
            span(d, weights[s], checked_product({kv_heads, contexts[s], 4}), "attention weights");
            if (reinterpret_cast<uintptr_t>(weights[s]) % 4) throw std::runtime_error("attention weights must be 4-byte aligned");
        }
        total += rows[s];
    }
    std::vector<Range> written;
    if (weights) {
        for (uint64_t s = 0; s < sequences; ++s) written.push_back(range(weights[s], kv_heads * contexts[s] * 4));
        check_apart(written, "attention weights of one call overlap, or are listed twice");
    }
    if (!total) return;
    attn::check_rows(d, q, total, q_stride, heads * dim, "attention queries");
    attn::check_rows(d, out, total, out_stride, heads * dim, "an attention output");
    attn::check_slopes(d, slopes, heads);
    if (overlap(q, ((total - 1) * q_stride + heads * dim) * 2, out, ((total - 1) * out_stride + heads * dim) * 2))
        throw std::runtime_error("an attention output lies over its queries");
    const size_t out_bytes = ((total - 1) * out_stride + heads * dim) * 2;
    for (uint64_t s = 0; s < sequences; ++s)
        if (overlap(out, out_bytes, states[s], state_bytes(contexts[s], kv_heads, dim)) || (weights && overlap(out, out_bytes, weights[s], kv_heads * contexts[s] * 4)))
            throw std::runtime_error("an attention output lies over a state or over attention weights");
    if (weights) {
        std::vector<Range> read{range(q, ((total - 1) * q_stride + heads * dim) * 2)};
        if (slopes) read.push_back(range(slopes, heads * 4));
        for (uint64_t s = 0; s < sequences; ++s) read.push_back(range(states[s], state_bytes(contexts[s], kv_heads, dim)));
        check_apart_from(written, read, "attention weights overlap a state, the queries or the slopes");
    }
    if (slopes && overlap(out, out_bytes, slopes, heads * 4)) throw std::runtime_error("an attention output lies over the slopes");

    AttentionArgs args{};
    args.heads = uint32_t(heads); args.kv_heads = uint32_t(kv_heads); args.group = uint32_t(group);
    args.q = q; args.out = out; args.slopes = slopes;
    args.q_stride = q_stride; args.out_stride = out_stride;
    args.scale_log2 = scale * 1.4426950408889634f;
    args.cap = cap * 1.4426950408889634f;
    args.scale_over_cap = cap > 0.0f ? scale / cap : 0.0f;
    args.window = uint32_t(std::min<uint64_t>(window, uint64_t(1) << 25));
    args.bf16 = type == kBf16;
    std::vector<attn::Sequence> chunks;   // what goes to the prompt kernel
    uint64_t row = 0, most = 0;
    auto flush = [&] {
        if (!args.sequences) return;
        const bool two = most > 8;
        if (dim == 64) launch_queries<64>(d, args, code, weights != nullptr, two);
        else if (dim == 128) launch_queries<128>(d, args, code, weights != nullptr, two);
        else launch_queries<256>(d, args, code, weights != nullptr, two);
        args.sequences = 0;
        most = 0;
    };
    for (uint64_t s = 0; s < sequences; ++s) {
        const uint64_t prefix = prefixes ? std::min(prefixes[s], lengths[s]) : 0;
        if (rows[s] && rows[s] * group <= kFewQueries) {
            AttentionSequence& to = args.sequence[args.sequences++];
            to = AttentionSequence{};
            to.state = static_cast<const uint8_t*>(states[s]);
            to.weights = weights ? weights[s] : nullptr;
            to.context = uint32_t(contexts[s]); to.length = uint32_t(lengths[s]); to.rows = uint32_t(rows[s]);
            to.first_row = uint32_t(row); to.prefix = uint32_t(prefix);
            most = std::max(most, rows[s] * group);
            if (args.sequences == kSequences) flush();
        } else if (rows[s]) {
            attn::Sequence to{};
            to.state = static_cast<const uint8_t*>(states[s]);
            to.context = contexts[s]; to.length = lengths[s]; to.rows = rows[s]; to.first_row = row; to.prefix = prefix;
            chunks.push_back(to);
        }
        row += rows[s];
    }
    flush();
    if (!chunks.empty()) attn::attend_kv8(d, chunks, heads, kv_heads, dim, code, scale, cap, slopes, window, q, q_stride, out, out_stride, type);
}

}  // namespace kv8
}  // namespace sdb

using namespace sdb;

extern "C" int sdx_kv8_attention(void* handle, const void* const* states, const uint64_t* contexts, const uint64_t* lengths,
                                 const uint64_t* rows, uint64_t sequences, uint64_t heads, uint64_t kv_heads, uint64_t dim, int code, float scale,
                                 float cap, const float* slopes, uint64_t window, const uint64_t* prefixes, const void* q, uint64_t q_stride,
                                 float* const* weights, void* out, uint64_t out_stride, int type) {
    SDB_OP_BEGIN
    kv8::attention(value, states, contexts, lengths, rows, sequences, heads, kv_heads, dim, code, scale, cap, slopes, window, prefixes, q, q_stride,
                   weights, out, out_stride, type);
    SDB_OP_END
}
