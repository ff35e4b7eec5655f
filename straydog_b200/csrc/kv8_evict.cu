// Eviction from states of 8-bit rows by accumulated attention weight (csrc/kv8.cuh has the layout).
//
// Of a sequence of n > keep positions each K/V head keeps the first `sinks`, the last `recent` and, of those between, the
// keep - sinks - recent with the greatest weights (equal weights: the lower position; a NaN below every number). The kept rows move, in
// their order, to positions 0 .. keep - 1 of another state. A target block takes the largest scale among the blocks its rows come from,
// and rows from a block with a smaller scale have their codes rounded again in it: the rule of an append to a begun block.
//
// kv8_evict_select_kernel: a cluster of 1 to 8 blocks a (sequence, head) finds the weight of the last place in three steps of 11, 11 and 10
// bits, with the weights in registers: a histogram in shared memory of the weights that agree with the bits found so far, summed over the cluster,
// and the bin where the places run out. A warp whose weights are all in one bin (weights of never-attended rows are all 0) adds them with one
// atomic. (Sixteen steps of two bits by compares, without atomics, took 65 us for 16 sequences x 8 heads x 16384: eight issue slots a weight and
// step.) Then ballots give every kept position its place in order. 8192 of 16384 positions of 16 sequences of 8 heads: 23 us, of one sequence 12.
// kv8_evict_move_kernel: 128 threads a (sequence, plane, one or four target blocks of 32 rows), rows of `dim` bytes gathered: bound by memory as long as the
// codes' rounding stays under its issue slots (eleven instructions a code with bit masks for E4M3 and a block a target block: 87 % of all issue slots, 101 us
// for 16 x 16384 positions).
#include "kv8.cuh"
#include "../../include/straydog_gpu_b200.h"

#include <cooperative_groups.h>

namespace sdb {
namespace kv8 {

struct EvictSequence {
    const uint8_t* state;
    uint8_t* target;
    const float* weights;
    float* target_weights;
    uint32_t context, length, target_context, first_unit;
};
struct EvictArgs {
    EvictSequence sequence[kSequences];
    int32_t* kept;      // [sequences of this launch][kv_heads][keep]
    uint32_t sequences, kv_heads, keep, sinks, recent;
    uint32_t each;      // target blocks a thread block moves, one behind the other
};

// and back, but for NaN and -0
__device__ __forceinline__ float weight_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

constexpr int kSelectThreads = 1024, kSelectWarps = 32, kHeld = 16, kFewHeld = 4, kMostCluster = 8;   // weights a thread holds; blocks a head
constexpr int kBins = 2048, kCopies = 4;   // a histogram's bins; copies that a block's warps share out, so that they meet less

// weights in an order of unsigned integers: NaN 0, then -inf .. +inf; the two zeros are equal
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template<int HELD>   // weights a thread holds in registers; 0: read again in every step
__global__ void __launch_bounds__(kSelectThreads, 1) kv8_evict_select_kernel(const __grid_constant__ EvictArgs a, uint32_t ctas) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ __align__(8) uint32_t histogram[kCopies][kBins];
    __shared__ __align__(8) uint32_t groups[kSelectWarps];
    __shared__ uint32_t warp_counts[kSelectWarps][2], block_counts[2], found[2];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t unit = blockIdx.x / ctas, rank = blockIdx.x % ctas, s = unit / a.kv_heads, head = unit % a.kv_heads;
    const EvictSequence& sequence = a.sequence[s];
    const uint32_t length = sequence.length, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const bool all = length <= a.keep;
    const uint32_t sinks = all ? length : a.sinks, recent = all ? 0 : a.recent, want = all ? 0 : a.keep - a.sinks - a.recent;
    const uint32_t between = length - sinks - recent;
    const float* weights = sequence.weights + size_t(head) * sequence.context;
    float* target_weights = sequence.target_weights + size_t(head) * sequence.target_context;
    int32_t* kept = a.kept + (size_t(s) * a.kv_heads + head) * a.keep;
    for (uint32_t i = rank * kSelectThreads + threadIdx.x; i < sinks + recent; i += ctas * kSelectThreads) {
        const uint32_t place = i < sinks ? i : want + i, from = i < sinks ? i : length - recent + (i - sinks);
        kept[place] = int32_t(from);
        target_weights[place] = weights[from];
    }
    // a warp's weights are consecutive: `each` steps of 32
    const uint32_t each = (between + ctas * kSelectThreads - 1) / (ctas * kSelectThreads);
    const uint32_t first = (rank * kSelectWarps + warp) * each * 32;
    const float* mine = weights + sinks;
    uint32_t key[HELD ? HELD : 1];
    auto load = [&](uint32_t j) -> uint32_t { const uint32_t i = first + j * 32 + lane; return i < between ? order_of(__ldg(mine + i)) : 0u; };
    if (HELD) {
        // (one bound for all, so that the loads go out together: 22000 cycles for 16 weights a thread when each waited for the one before)
        const uint32_t end = min(between, first + each * 32);
        #pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const uint32_t i = first + j * 32 + lane;
            key[j] = i < end ? __float_as_uint(__ldg(mine + i)) : 0u;
        }
        #pragma unroll
        for (int j = 0; j < HELD; ++j) key[j] = order_of(__uint_as_float(key[j]));
    }
    auto each_key = [&](auto&& act) {
        if (HELD) {
            #pragma unroll
            for (int j = 0; j < HELD; ++j) {
                if (uint32_t(j) >= each) break;
                act(uint32_t(j), key[j]);
            }
        } else {
            #pragma unroll 4
            for (uint32_t j = 0; j < each; ++j) act(j, load(j));
        }
    };
    uint32_t last = 0, missing = want;   // the key of the last place, its bits from the top; places left among the keys that agree with them
    #pragma unroll 1
    for (int step = 0; want && step < 3; ++step) {
        const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bits = step == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < kCopies * kBins; i += kSelectThreads) (&histogram[0][0])[i] = 0;
        __syncthreads();
        uint32_t* mine_counts = histogram[warp % kCopies];
        each_key([&](uint32_t j, uint32_t k) {
            const bool counts = first + j * 32 + lane < between && (step == 0 || (k >> (shift + bits)) == (last >> (shift + bits)));
            if (step && !__any_sync(0xffffffffu, counts)) return;   // (most steps of 32, once the upper bits are known)
            const uint32_t bin = counts ? (k >> shift) & ((1u << bits) - 1u) : 0xffffffffu;
            const bool same = __all_sync(0xffffffffu, bin == __shfl_sync(0xffffffffu, bin, 0));
            if (counts && (!same || lane == 0)) atomicAdd(&mine_counts[bin], same ? 32u : 1u);
        });
        __syncthreads();
        // the copies' sum, two bins a thread, and the sums of a warp's 64
        uint2 sum = make_uint2(0, 0);
        #pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const uint2 counts = reinterpret_cast<const uint2*>(histogram[c])[threadIdx.x];
            sum.x += counts.x; sum.y += counts.y;
        }
        reinterpret_cast<uint2*>(histogram[0])[threadIdx.x] = sum;
        const uint32_t group = __reduce_add_sync(0xffffffffu, sum.x + sum.y);
        if (lane == 0) groups[warp] = group;
        if (ctas > 1) cluster.sync(); else __syncthreads();
        if (warp == 0) {
            // the group where the places run out, then its bin, each over the cluster from the greatest down. (Every bin of every block read by all threads:
            // 6200 cycles a step with eight blocks.)
            auto over_cluster = [&](uint2* at) -> uint2 {
                if (ctas == 1) return *at;
                uint2 total = make_uint2(0, 0);
                #pragma unroll
                for (uint32_t r = 0; r < kMostCluster; ++r) {
                    const uint2 counts = r < ctas ? *cluster.map_shared_rank(at, r) : make_uint2(0, 0);
                    total.x += counts.x; total.y += counts.y;
                }
                return total;
            };
            auto up_to = [&](uint32_t count) -> uint32_t {   // inclusive sums over the lanes
                #pragma unroll
                for (int offset = 1; offset < 32; offset *= 2) { const uint32_t other = __shfl_up_sync(0xffffffffu, count, offset); if (lane >= uint32_t(offset)) count += other; }
                return count;
            };
            const uint2 two = over_cluster(reinterpret_cast<uint2*>(groups) + (15 - lane / 2));
            const uint32_t mine_group = lane & 1 ? two.x : two.y, above_group = up_to(mine_group);
            const int place = __ffs(__ballot_sync(0xffffffffu, above_group >= missing)) - 1;
            const uint32_t before = __shfl_sync(0xffffffffu, above_group - mine_group, place), base = (31 - place) * 64;
            const uint2 bins = over_cluster(reinterpret_cast<uint2*>(&histogram[0][base + 62 - 2 * lane]));
            const uint32_t above = before + up_to(bins.x + bins.y), before_low = above - bins.x, before_high = before_low - bins.y;
            if (before_high < missing && missing <= above) {   // one lane
                const bool in_high = missing <= before_low;
                found[0] = in_high ? base + 63 - 2 * lane : base + 62 - 2 * lane;
                found[1] = missing - (in_high ? before_high : before_low);
            }
        }
        if (ctas > 1) cluster.sync(); else __syncthreads();   // (also: every block has read the others' counts before they are zeroed)
        last |= found[0] << shift;
        missing = found[1];
    }
    // places: keys above `last` all stay, of those equal to it the first `missing` in order
    {
        uint32_t reach = 0, above = 0;
        if (want) each_key([&](uint32_t j, uint32_t k) {
            const bool real = first + j * 32 + lane < between;
            reach += real && k >= last; above += real && k > last;
        });
        reach = __reduce_add_sync(0xffffffffu, reach);
        above = __reduce_add_sync(0xffffffffu, above);
        if (lane == 0) { warp_counts[warp][0] = reach; warp_counts[warp][1] = above; }
        __syncthreads();
        if (warp == 0) {
            const uint32_t all_reach = __reduce_add_sync(0xffffffffu, warp_counts[lane][0]), all_above = __reduce_add_sync(0xffffffffu, warp_counts[lane][1]);
            if (lane == 0) { block_counts[0] = all_reach; block_counts[1] = all_above; }
        }
        if (ctas > 1) cluster.sync();
        // (a lane a block before this one, and a lane a warp)
        const uint32_t* others = lane < rank ? cluster.map_shared_rank(&block_counts[0], lane) : nullptr;
        reach = __reduce_add_sync(0xffffffffu, (others ? others[0] : 0u) + (lane < warp ? warp_counts[lane][0] : 0u));
        above = __reduce_add_sync(0xffffffffu, (others ? others[1] : 0u) + (lane < warp ? warp_counts[lane][1] : 0u));
        const uint32_t ties = want ? missing : 0;
        uint32_t equal = reach - above;
        uint32_t place = sinks + above + min(equal, ties);
        const uint32_t below = (1u << lane) - 1u;
        if (want) each_key([&](uint32_t j, uint32_t k) {
            const bool real = first + j * 32 + lane < between, tie = real && k == last;
            const uint32_t ties_here = __ballot_sync(0xffffffffu, tie);
            const bool stays = (real && k > last) || (tie && equal + __popc(ties_here & below) < ties);
            const uint32_t staying = __ballot_sync(0xffffffffu, stays);
            if (stays) {
                const uint32_t i = first + j * 32 + lane, at = place + __popc(staying & below);
                kept[at] = int32_t(sinks + i);
                target_weights[at] = k && k != 0x80000000u ? weight_of(k) : mine[i];   // (a NaN and a zero's sign are not in the key)
            }
            equal += __popc(ties_here);
            place += __popc(staying);
        });
    }
    if (ctas > 1) cluster.sync();   // (no block leaves while another may still read its counts)
}

template<int D, int CODE>
__global__ void __launch_bounds__(128) kv8_evict_move_kernel(const __grid_constant__ EvictArgs a) {
    constexpr int kPieces = D / 16, kRows = 128 / kPieces, kPasses = int(kBlock) / kRows;   // threads a row, rows a pass
    uint32_t s = 0;
    {
        uint32_t high = a.sequences;
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_unit <= blockIdx.x) s = mid; else high = mid; }
    }
    const EvictSequence& sequence = a.sequence[s];
    const uint32_t planes = 2 * a.kv_heads, unit = blockIdx.x - sequence.first_unit, plane = unit % planes, first = unit / planes * a.each;
    const uint32_t kept_rows = min(sequence.length, a.keep), end = min(first + a.each, (kept_rows + kBlock - 1) / kBlock);
    const uint32_t row = threadIdx.x / kPieces, piece = threadIdx.x % kPieces;
    const int32_t* kept = a.kept + (size_t(s) * a.kv_heads + plane % a.kv_heads) * a.keep;
    const uint8_t* codes = sequence.state + size_t(plane) * sequence.context * D + piece * 16;
    const float* scales = reinterpret_cast<const float*>(sequence.state + size_t(planes) * sequence.context * D) + size_t(plane) * (sequence.context / kBlock);
    uint8_t* target = sequence.target + size_t(plane) * sequence.target_context * D + piece * 16;
    float* target_scales = reinterpret_cast<float*>(sequence.target + size_t(planes) * sequence.target_context * D) + size_t(plane) * (sequence.target_context / kBlock);
    __shared__ float tops[2][4];
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the positions are the kernel's before
    uint32_t from[kPasses];
    auto positions = [&](uint32_t block) {
        #pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const uint32_t r = block * kBlock + p * kRows + row;
            from[p] = block < end && r < kept_rows ? uint32_t(kept[r]) : 0xffffffffu;
        }
    };
    positions(first);
    #pragma unroll 1
    for (uint32_t block = first; block < end; ++block) {
        uint4 v[kPasses];
        float old[kPasses];
        #pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const bool there = from[p] != 0xffffffffu;
            old[p] = there ? scales[from[p] / kBlock] : 0.0f;
            v[p] = there ? *reinterpret_cast<const uint4*>(codes + size_t(from[p]) * D) : make_uint4(0, 0, 0, 0);
        }
        bool there[kPasses];
        #pragma unroll
        for (int p = 0; p < kPasses; ++p) there[p] = from[p] != 0xffffffffu;
        positions(block + 1);   // (asked for while this block's rows are on their way)
        float top = 0.0f;
        #pragma unroll
        for (int p = 0; p < kPasses; ++p) top = fmaxf(top, old[p]);
        #pragma unroll
        for (int offset = 16; offset >= kPieces; offset /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));   // (a row's threads have one scale)
        if (threadIdx.x % 32 == 0) tops[block & 1][threadIdx.x / 32] = top;
        __syncthreads();
        const float scale = fmaxf(fmaxf(tops[block & 1][0], tops[block & 1][1]), fmaxf(tops[block & 1][2], tops[block & 1][3]));
        #pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            if (!there[p]) continue;
            const float ratio = scale > 0.0f ? __fdiv_rn(old[p], scale) : 0.0f;
            *reinterpret_cast<uint4*>(target + size_t(block * kBlock + p * kRows + row) * D) = recode16<CODE>(v[p], ratio);
        }
        if (threadIdx.x == 0) target_scales[block] = scale;
    }
}

static void launch_move(Device& d, uint64_t dim, int code, const EvictArgs& args, uint32_t units) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(units);
    config.blockDim = dim3(128);
    config.stream = d.stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    const auto kernel = dim == 64    ? (code == kInt8 ? kv8_evict_move_kernel<64, kInt8> : kv8_evict_move_kernel<64, kE4m3>)
                        : dim == 128 ? (code == kInt8 ? kv8_evict_move_kernel<128, kInt8> : kv8_evict_move_kernel<128, kE4m3>)
                                     : (code == kInt8 ? kv8_evict_move_kernel<256, kInt8> : kv8_evict_move_kernel<256, kE4m3>);
    SDB_CHECK(cudaLaunchKernelEx(&config, kernel, args));
    ++d.launches;
}

static void evict(Device& d, const void* const* states, const uint64_t* contexts, const uint64_t* lengths, const float* const* weights,
                  uint64_t sequences, uint64_t keep, uint64_t sinks, uint64_t recent, uint64_t kv_heads, uint64_t dim, int code,
                  void* const* targets, const uint64_t* target_contexts, float* const* target_weights, int32_t* kept) {
    check_shape(sequences, kv_heads, dim, code);
    if (!states || !contexts || !lengths || !weights || !targets || !target_contexts || !target_weights)
        throw std::runtime_error("invalid Straydog eviction");
    if (!keep || keep > (uint64_t(1) << 24) || sinks > keep || recent > keep - sinks)
        throw std::runtime_error("an eviction keeps at least its sinks and its recent positions, at most 2^24");
    std::vector<Range> written, read;
    for (uint64_t s = 0; s < sequences; ++s) {
        check_state(d, states[s], contexts[s], kv_heads, dim);
        check_state(d, targets[s], target_contexts[s], kv_heads, dim);
        if (lengths[s] > contexts[s] || std::min(lengths[s], keep) > target_contexts[s])
            throw std::runtime_error("an eviction's lengths do not fit its states");
        const size_t from = checked_product({kv_heads, contexts[s], 4}), to = checked_product({kv_heads, target_contexts[s], 4});
        span(d, weights[s], from, "attention weights");
        span(d, target_weights[s], to, "an eviction's target weights");
        if (reinterpret_cast<uintptr_t>(weights[s]) % 4 || reinterpret_cast<uintptr_t>(target_weights[s]) % 4)
            throw std::runtime_error("attention weights must be 4-byte aligned");
        read.push_back(range(states[s], state_bytes(contexts[s], kv_heads, dim)));
        read.push_back(range(weights[s], from));
        written.push_back(range(targets[s], state_bytes(target_contexts[s], kv_heads, dim)));
        written.push_back(range(target_weights[s], to));
    }
    if (kept) {
        const size_t bytes = checked_product({sequences, kv_heads, keep, 4});
        span(d, kept, bytes, "an eviction's positions");
        if (reinterpret_cast<uintptr_t>(kept) % 4) throw std::runtime_error("an eviction's positions must be 4-byte aligned");
        written.push_back(range(kept, bytes));
    }
    // what is written lies apart from everything else: rows move between blocks that run in any order
    check_apart(written, "an eviction's targets overlap");
    check_apart_from(written, read, "an eviction's target overlaps what it reads");
    if (!kept) kept = static_cast<int32_t*>(workspace(d, d.kv8_kept, checked_product({sequences, kv_heads, keep, 4})));
    for (uint64_t at = 0; at < sequences;) {
        EvictArgs args{};
        args.kv_heads = uint32_t(kv_heads); args.keep = uint32_t(keep); args.sinks = uint32_t(sinks); args.recent = uint32_t(recent);
        args.kept = kept + at * kv_heads * keep;
        uint64_t units = 0, longest = 0;
        // Four target blocks a thread block where there are enough of them to fill the SMs all the same (sixteen an SM run at once), else one: 1024 kept of
        // 2047 positions 10.8 us by ones, 12.3 by fours; 8192 kept of 16384 of 16 sequences 118.7 by ones, 114.6 by fours
        uint64_t blocks = 0;
        for (uint64_t s = at; s < sequences && s < at + kSequences; ++s) blocks += (std::min(lengths[s], keep) + kBlock - 1) / kBlock * 2 * kv_heads;
        args.each = blocks >= uint64_t(d.sms) * 16 * 4 ? 4 : 1;
        for (; at < sequences && args.sequences < kSequences; ++at) {
            const uint64_t more = (std::min(lengths[at], keep) + args.each * kBlock - 1) / (args.each * kBlock) * 2 * kv_heads;
            if (units + more >= uint64_t(1) << 31) break;
            args.sequence[args.sequences++] = EvictSequence{static_cast<const uint8_t*>(states[at]), static_cast<uint8_t*>(targets[at]), weights[at],
                                                            target_weights[at], uint32_t(contexts[at]), uint32_t(lengths[at]),
                                                            uint32_t(target_contexts[at]), uint32_t(units)};
            units += more;
            longest = std::max(longest, lengths[at]);
        }
        if (!units) continue;   // (every sequence of the group is empty)
        // Blocks a head: enough for the weights to fit the registers, and twice as many again while the heads leave SMs idle (8 heads of 16384 positions
        // 22.2 us against 25.3 without, four such sequences 42.6 against 49.7, before the clusters' sums got faster: 16.9 and 36.8 now)
        uint32_t ctas = 1;
        const uint64_t heads = args.sequences * kv_heads;
        while (ctas < kMostCluster && longest > uint64_t(ctas) * kSelectThreads * kHeld) ctas *= 2;
        while (ctas < kMostCluster && heads * ctas * 2 <= uint64_t(d.sms) && longest > uint64_t(ctas) * kSelectThreads * 4) ctas *= 2;
        // Few weights a thread have a kernel of their own, a quarter of the unrolled code: 1024 kept of 2047 positions 9.6 us against 10.8, 4096 of 16384 16.9 against 18.3
        const uint64_t each = (longest + ctas * kSelectThreads - 1) / (ctas * kSelectThreads);
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(unsigned(heads * ctas));
        config.blockDim = dim3(kSelectThreads);
        config.stream = d.stream;
        cudaLaunchAttribute attribute{};
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = ctas; attribute.val.clusterDim.y = 1; attribute.val.clusterDim.z = 1;
        config.attrs = &attribute;
        config.numAttrs = 1;
        SDB_CHECK(cudaLaunchKernelEx(&config, each <= kFewHeld ? kv8_evict_select_kernel<kFewHeld> : each <= kHeld ? kv8_evict_select_kernel<kHeld> : kv8_evict_select_kernel<0>, args, ctas));
        ++d.launches;
        launch_move(d, dim, code, args, uint32_t(units));
    }
}

}  // namespace kv8
}  // namespace sdb

using namespace sdb;

extern "C" int sdx_kv8_evict(void* handle, const void* const* states, const uint64_t* contexts, const uint64_t* lengths,
                             const float* const* weights, uint64_t sequences, uint64_t keep, uint64_t sinks, uint64_t recent, uint64_t kv_heads,
                             uint64_t dim, int code, void* const* targets, const uint64_t* target_contexts, float* const* target_weights,
                             int32_t* kept) {
    SDB_OP_BEGIN
    kv8::evict(value, states, contexts, lengths, weights, sequences, keep, sinks, recent, kv_heads, dim, code, targets, target_contexts,
               target_weights, kept);
    SDB_OP_END
}
