// New keys and values appended to states of 8-bit rows with block scales (csrc/kv8.cuh has the layout and the codes).
//
// For every block of 32 positions the rows touch, need = max |x| / top over the call's rows in it. A block whose first position is among
// the call's rows takes scale = need. A block with older rows takes scale = max(old, need); where that is more than old, its older codes
// c are rounded again: c * (old / scale). Positions behind the call's rows are not touched (whatever they hold is not counted on: the
// sequence ends there).
//
// One block of 128 or 256 threads does one (sequence, plane, block of 32): the block's new rows stay in registers between the maximum and the
// codes, so each value is read once. Bound by memory for a prompt, by one chain of latencies (row, maximum, store) for a single token:
// then a few threads hold the row and the rest look after the older codes.
// One row each of 32 sequences of 8 heads of 128 (BF16): 3.5 us; 8191 rows of 2 heads of 256 (F16 to E4M3, 25 MB): 11.1 us, of which the copy rate would
// take 3.8: the encoding's issue slots and a tail of one wave are the rest.
#include "kv8.cuh"
#include "../../include/straydog_gpu_b200.h"

namespace sdb {
namespace kv8 {

struct WriteSequence {
    uint8_t* state;
    uint32_t context, base, steps, first_row, first_unit;
};
struct WriteArgs {
    WriteSequence sequence[kSequences];
    uint32_t sequences, kv_heads;
    const void* keys;
    const void* values;
    size_t stride;   // elements between rows of keys and of values
};

template<typename T> struct Load8;
template<> struct Load8<float> {
    static __device__ __forceinline__ void go(const float* at, float (&v)[8]) {
        const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template<> struct Load8<__half> {
    static __device__ __forceinline__ void go(const __half* at, float (&v)[8]) {
        const uint4 a = *reinterpret_cast<const uint4*>(at);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
};
template<> struct Load8<__nv_bfloat16> {
    static __device__ __forceinline__ void go(const __nv_bfloat16* at, float (&v)[8]) {
        const uint4 a = *reinterpret_cast<const uint4*>(at);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
        #pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};

// threads of a block: at most 32 values each
template<int D> constexpr int kWriteThreads = D == 256 ? 256 : 128;

template<int D, typename T, int CODE>
__global__ void __launch_bounds__(kWriteThreads<D>) kv8_write_kernel(const __grid_constant__ WriteArgs a) {
    constexpr int kThreads = kWriteThreads<D>, kColumns = D / 8, kRows = kThreads / kColumns, kPasses = int(kBlock) / kRows;   // threads a row, rows a pass
    uint32_t s = 0;
    {
        uint32_t high = a.sequences;   // the last sequence whose first unit is not behind this block
        while (high - s > 1) { const uint32_t mid = (s + high) / 2; if (a.sequence[mid].first_unit <= blockIdx.x) s = mid; else high = mid; }
    }
    const WriteSequence& sequence = a.sequence[s];
    const uint32_t planes = 2 * a.kv_heads, unit = blockIdx.x - sequence.first_unit, plane = unit % planes;
    const uint32_t block = sequence.base / kBlock + unit / planes, begin = block * kBlock;
    const uint32_t low = max(begin, sequence.base), high = min(begin + kBlock, sequence.base + sequence.steps);   // the call's rows in the block
    uint8_t* codes = sequence.state + (size_t(plane) * sequence.context + begin) * D;
    float* scale_at = reinterpret_cast<float*>(sequence.state + size_t(planes) * sequence.context * D) +
                      size_t(plane) * (sequence.context / kBlock) + block;
    const bool begun = begin < sequence.base;
    const float old = begun ? *scale_at : 0.0f;
    const uint32_t row = threadIdx.x / kColumns, column = threadIdx.x % kColumns * 8;
    const T* source = static_cast<const T*>(plane < a.kv_heads ? a.keys : a.values) + size_t(plane < a.kv_heads ? plane : plane - a.kv_heads) * D + column;

    float x[kPasses][8];
    float top = 0.0f;
    #pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const uint32_t at = begin + p * kRows + row;
        if (at < low || at >= high) continue;
        Load8<T>::go(source + (size_t(sequence.first_row) + (at - sequence.base)) * a.stride, x[p]);
    }
    #pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const uint32_t at = begin + p * kRows + row;
        if (at < low || at >= high) continue;
        #pragma unroll
        for (int i = 0; i < 8; ++i) { const float m = fabsf(x[p][i]); top = fmaxf(top, m <= FLT_MAX ? m : 0.0f); }
    }
    #pragma unroll
    for (int offset = 16; offset; offset /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
    __shared__ float tops[kThreads / 32];
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();   // (also: every thread has read the old scale before one writes the new)
    #pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = fmaxf(top, tops[i]);
    const float scale = fmaxf(old, __fdiv_rn(top, top_code<CODE>()));
    const Reciprocal reciprocal(scale);
    #pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const uint32_t at = begin + p * kRows + row;
        if (at < low || at >= high) continue;
        uint32_t w[2];
        #pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = encode2<CODE>(x[p][4 * i], x[p][4 * i + 1], scale, reciprocal) | encode2<CODE>(x[p][4 * i + 2], x[p][4 * i + 3], scale, reciprocal) << 16;
        *reinterpret_cast<uint2*>(codes + size_t(p * kRows + row) * D + column) = make_uint2(w[0], w[1]);
    }
    if (begun && scale > old) {
        const float ratio = __fdiv_rn(old, scale);
        const uint32_t pieces = (low - begin) * (D / 16);   // the older rows, 16 codes a piece
        for (uint32_t i = threadIdx.x; i < pieces; i += kThreads) {
            uint4* at = reinterpret_cast<uint4*>(codes) + i;
            *at = recode16<CODE>(*at, ratio);
        }
    }
    if (threadIdx.x == 0) *scale_at = scale;
}

template<int D, typename T> static void launch_code(int code, const WriteArgs& args, uint32_t units, cudaStream_t stream) {
    if (code == kInt8) kv8_write_kernel<D, T, kInt8><<<units, kWriteThreads<D>, 0, stream>>>(args);
    else kv8_write_kernel<D, T, kE4m3><<<units, kWriteThreads<D>, 0, stream>>>(args);
}
template<int D> static void launch_type(int code, int type, const WriteArgs& args, uint32_t units, cudaStream_t stream) {
    if (type == kF32) launch_code<D, float>(code, args, units, stream);
    else if (type == kF16) launch_code<D, __half>(code, args, units, stream);
    else launch_code<D, __nv_bfloat16>(code, args, units, stream);
}

static void write(Device& d, void* const* states, const uint64_t* contexts, const uint64_t* bases, const uint64_t* steps, uint64_t sequences,
                  uint64_t kv_heads, uint64_t dim, int code, const void* keys, const void* values, uint64_t stride, int type) {
    check_shape(sequences, kv_heads, dim, code);
    if (type != kF32 && type != kF16 && type != kBf16) throw std::runtime_error("8-bit K/V rows are written from F32 (0), F16 (1) or BF16 (30)");
    if (!states || !contexts || !bases || !steps) throw std::runtime_error("invalid Straydog 8-bit K/V write");
    const size_t size = type == kF32 ? 4 : 2;
    if (!stride) stride = kv_heads * dim;
    if (stride < kv_heads * dim || stride > (uint64_t(1) << 32) || stride * size % 16 || reinterpret_cast<uintptr_t>(keys) % 16 ||
        reinterpret_cast<uintptr_t>(values) % 16)
        throw std::runtime_error("8-bit K/V rows to write lie on 16-byte boundaries, kv_heads * dim elements apart or more");
    uint64_t rows = 0;
    for (uint64_t s = 0; s < sequences; ++s) {
        check_state(d, states[s], contexts[s], kv_heads, dim);
        if (bases[s] > contexts[s] || steps[s] > contexts[s] - bases[s]) throw std::runtime_error("8-bit K/V rows past the state's context");
        rows += steps[s];
    }
    if (!rows) return;
    if (rows >= uint64_t(1) << 31) throw std::runtime_error("too many 8-bit K/V rows in one write");
    std::vector<Range> written;
    for (uint64_t s = 0; s < sequences; ++s) written.push_back(range(states[s], state_bytes(contexts[s], kv_heads, dim)));
    check_apart(written, "8-bit K/V states of one write overlap, or one is listed twice");
    for (const void* from : {keys, values}) {
        span(d, from, (checked_product({rows - 1, stride}) + kv_heads * dim) * size, "8-bit K/V rows to write");
        for (uint64_t s = 0; s < sequences; ++s)
            if (overlap(from, ((rows - 1) * stride + kv_heads * dim) * size, states[s], state_bytes(contexts[s], kv_heads, dim)))
                throw std::runtime_error("8-bit K/V rows to write lie inside a state they are written to");
    }
    uint64_t row = 0;
    for (uint64_t at = 0; at < sequences;) {
        WriteArgs args{};
        args.kv_heads = uint32_t(kv_heads);
        args.keys = keys; args.values = values; args.stride = stride;
        uint64_t units = 0;
        for (; at < sequences && args.sequences < kSequences; ++at) {
            if (!steps[at]) continue;
            const uint64_t blocks = (bases[at] + steps[at] - 1) / kBlock - bases[at] / kBlock + 1, more = blocks * 2 * kv_heads;
            if (units + more >= uint64_t(1) << 31) break;   // (one sequence is at most 2^19 blocks x 2^11 planes: it always fits alone)
            args.sequence[args.sequences++] = WriteSequence{static_cast<uint8_t*>(states[at]), uint32_t(contexts[at]), uint32_t(bases[at]),
                                                            uint32_t(steps[at]), uint32_t(row), uint32_t(units)};
            units += more;
            row += steps[at];
        }
        if (!args.sequences) continue;
        if (dim == 64) launch_type<64>(code, type, args, uint32_t(units), d.stream);
        else if (dim == 128) launch_type<128>(code, type, args, uint32_t(units), d.stream);
        else launch_type<256>(code, type, args, uint32_t(units), d.stream);
        ++d.launches;
    }
}

}  // namespace kv8
}  // namespace sdb

using namespace sdb;

extern "C" uint64_t sdx_kv8_bytes(uint64_t context, uint64_t kv_heads, uint64_t dim) {
    try {
        kv8::check_shape(1, kv_heads, dim, 0);
        if (!context || context % kv8::kBlock || context > (uint64_t(1) << 24))
            throw std::runtime_error("an 8-bit K/V state's context is a multiple of 32, at most 2^24");
        return kv8::state_bytes(context, kv_heads, dim);
    } catch (const std::exception& e) { last_error = e.what(); return 0; }
}

extern "C" int sdx_kv8_write(void* handle, void* const* states, const uint64_t* contexts, const uint64_t* bases, const uint64_t* steps,
                             uint64_t sequences, uint64_t kv_heads, uint64_t dim, int code, const void* keys, const void* values,
                             uint64_t stride, int type) {
    SDB_OP_BEGIN
    kv8::write(value, states, contexts, bases, steps, sequences, kv_heads, dim, code, keys, values, stride, type);
    SDB_OP_END
}
