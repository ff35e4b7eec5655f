// K/V rows in 8 bits whose scale is shared by a block of 32 positions of one head: layout, codecs and the host checks that the
// write, the attention and the eviction over such states have in common.
//
// A state holds 2 * kv_heads planes (keys of head 0 .., then values of head 0 ..). Plane p is `context` rows (a multiple of 32) of `dim`
// one-byte codes at state + p * context * dim; behind the planes lie their block scales, F32, context / 32 a plane. A code c stands for
// c * scale of its block. int8: scale = max |x| / 127, c = x / scale rounded to nearest even; e4m3: scale = max |x| / 448, c = x / scale in
// E4M3 (nearest even). A zero scale means zero rows. Codes are never NaN: an infinity is held as the block's largest magnitude, a NaN as 0
// (one such value must not take its 31 neighbours' scale with it).
#pragma once
#include "common.cuh"

#include <algorithm>
#include <cfloat>
#include <cuda_fp8.h>

namespace sdb {
namespace kv8 {

constexpr unsigned kBlock = 32;        // positions that share a scale
constexpr unsigned kSequences = 64;    // sequences a launch: their descriptors travel as kernel parameters (no table to upload, nothing to keep alive)
constexpr int kInt8 = 0, kE4m3 = 1;
constexpr int kF32 = 0, kF16 = 1, kBf16 = 30;   // element types by their GGML numbers, as sd_op_index_select_proj takes them

// The attention kernels add the log2 of a value scale to the weights' exponents, from 2^-88, and from 2^-64 of the largest, up: so the sum of plain weights
// (at most 2^15 over the scale each, 2^24 of them) stays finite, and a weight beside a small scale, or one of zero, stays in the sum, since the exponential of
// weight times scale is 2^-57 of the row's largest or more.
constexpr float kLowestScale = -88.0f, kScaleRange = 64.0f;

inline size_t state_bytes(uint64_t context, uint64_t kv_heads, uint64_t dim) {
    const size_t raw = checked_product({2 * kv_heads, context, dim}) + checked_product({2 * kv_heads, context / kBlock, 4});
    return (raw + 15) / 16 * 16;
}

inline void check_shape(uint64_t sequences, uint64_t kv_heads, uint64_t dim, int code) {
    if (!sequences || sequences > 65535 || !kv_heads || kv_heads > 1024 || (dim != 64 && dim != 128 && dim != 256))
        throw std::runtime_error("invalid Straydog 8-bit K/V dimensions");
    if (code != kInt8 && code != kE4m3) throw std::runtime_error("an 8-bit K/V code is 0 (int8) or 1 (e4m3)");
}

inline void check_state(Device& d, const void* state, uint64_t context, uint64_t kv_heads, uint64_t dim) {
    if (!context || context % kBlock || context > (uint64_t(1) << 24))
        throw std::runtime_error("an 8-bit K/V state's context is a multiple of 32, at most 2^24");
    span(d, state, state_bytes(context, kv_heads, dim), "an 8-bit K/V state");
    if (reinterpret_cast<uintptr_t>(state) % 16) throw std::runtime_error("an 8-bit K/V state must be 16-byte aligned");
}

// What a launch writes lies apart: blocks run in any order.
using Range = std::pair<uintptr_t, uintptr_t>;
inline Range range(const void* p, size_t bytes) { return {reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes}; }
inline void check_apart(std::vector<Range>& written, const char* message) {
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].first < written[i - 1].second) throw std::runtime_error(message);
}

// (written: sorted and apart, as check_apart leaves them)
inline void check_apart_from(const std::vector<Range>& written, std::vector<Range>& read, const char* message) {
    std::sort(read.begin(), read.end());
    for (size_t i = 0, j = 0; i < read.size(); ++i) {
        while (j < written.size() && written[j].second <= read[i].first) ++j;
        if (j < written.size() && written[j].first < read[i].second) throw std::runtime_error(message);
    }
}

inline bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

#if defined(__CUDACC__)
template<int CODE> constexpr float top_code() { return CODE == kInt8 ? 127.0f : 448.0f; }

// x over scale in the block's code: the IEEE quotient rounded to nearest even. A product with the scale's reciprocal (1 / scale, itself rounded once)
// is within 2^-22 of the quotient; where both ends of that range round to the same code, so does the quotient, and only where they do not
// (about one value in a thousand) is it divided. Scales without a normal number for their reciprocal divide always.
template<int CODE> __device__ __forceinline__ uint32_t round_code(float y) {
    if (CODE == kInt8) {
        int q = __float2int_rn(y);
        q = q > 127 ? 127 : q < -127 ? -127 : q;
        return uint32_t(q) & 0xffu;
    }
    return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
template<int CODE> __device__ __forceinline__ uint32_t encode(float x, float scale) {
    if (!(scale > 0.0f) || x != x) return 0;
    return round_code<CODE>(__fdiv_rn(x, scale));
}
struct Reciprocal {
    float value;
    bool normal;
    __device__ __forceinline__ explicit Reciprocal(float scale) : value(scale > 0.0f ? 1.0f / scale : 0.0f), normal(scale > 1.2e-38f && scale < 8.5e37f) {}
};
// two values; the codes in the low two bytes
template<int CODE> __device__ __forceinline__ uint32_t encode2(float x, float y, float scale, const Reciprocal& r) {
    const float a = __fmul_rn(x, r.value), b = __fmul_rn(y, r.value);
    constexpr float kDown = 1.0f - 3.6e-7f, kUp = 1.0f + 3.6e-7f;   // 1 -+ 3 * 2^-23
    uint32_t low, high;
    if (CODE == kInt8) {
        // a sum with 1.5 * 2^23 rounds to an integer and leaves it in the low byte (clamped before: an infinity is the largest code)
        const float a0 = fminf(fmaxf(a * kDown, -127.0f), 127.0f), a1 = fminf(fmaxf(a * kUp, -127.0f), 127.0f);
        const float b0 = fminf(fmaxf(b * kDown, -127.0f), 127.0f), b1 = fminf(fmaxf(b * kUp, -127.0f), 127.0f);
        low = prmt(__float_as_uint(__fadd_rn(a0, 12582912.0f)), __float_as_uint(__fadd_rn(b0, 12582912.0f)), 0x0040u) & 0xffffu;
        high = prmt(__float_as_uint(__fadd_rn(a1, 12582912.0f)), __float_as_uint(__fadd_rn(b1, 12582912.0f)), 0x0040u) & 0xffffu;
    } else {
        low = __nv_cvt_float2_to_fp8x2(make_float2(a * kDown, b * kDown), __NV_SATFINITE, __NV_E4M3);
        high = __nv_cvt_float2_to_fp8x2(make_float2(a * kUp, b * kUp), __NV_SATFINITE, __NV_E4M3);
    }
    if (low == high && r.normal && x == x && y == y) return low;
    return encode<CODE>(x, scale) | encode<CODE>(y, scale) << 8;
}

// Sixteen codes of a row whose block takes a larger scale: their values in the old scale, rounded again in the new one (ratio = old / new
// <= 1): code times ratio in F32, then one rounding to the code. int8: a byte becomes 2^23 + 128 + c by a byte permute, and a sum with
// 1.5 * 2^23 rounds to nearest even and leaves the code in the low byte. E4M3: two codes a conversion on the way in and out.
template<int CODE> __device__ __forceinline__ uint4 recode16(uint4 v, float ratio) {
    if (ratio == 1.0f) return v;
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (CODE == kInt8) {
            const uint32_t u = w[i] ^ 0x80808080u;
            uint32_t q[4];
            #pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float c = __fsub_rn(__uint_as_float(prmt(u, 0x4b000000u, 0x7440u | b)), 8388736.0f);
                q[b] = __float_as_uint(__fadd_rn(__fmul_rn(c, ratio), 12582912.0f));
            }
            w[i] = prmt(prmt(q[0], q[1], 0x0040u), prmt(q[2], q[3], 0x0040u), 0x5410u);
        } else {
            uint32_t low, high;
            asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(low), "=r"(high) : "r"(w[i]));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&low)), g = __half22float2(*reinterpret_cast<const __half2*>(&high));
            asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
                : "=r"(w[i]) : "f"(__fmul_rn(f.x, ratio)), "f"(__fmul_rn(f.y, ratio)), "f"(__fmul_rn(g.x, ratio)), "f"(__fmul_rn(g.y, ratio)));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
#endif

}  // namespace kv8
}  // namespace sdb
