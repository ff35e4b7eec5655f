// What the attention entries with masks share: the checks of their arguments and the prompt kernel's way in for 8-bit states.
#pragma once
#include "common.cuh"

#include <vector>

namespace sdb {
namespace attn {

// One sequence (or document) of a call.
struct Sequence {
    const uint8_t* state;            // 8-bit state and its context, or null: keys and values are rows of packed arrays
    uint64_t context;
    uint64_t rows, length, prefix;   // query rows, keys, keys every row sees
    uint64_t first_row, first_key;   // in the packed arrays
};

void check_rule(uint64_t heads, uint64_t kv_heads, uint64_t dim, float scale, float cap, int type);
void check_rows(Device& d, const void* pointer, uint64_t rows, uint64_t stride, uint64_t width, const char* what);
void check_slopes(Device& d, const float* slopes, uint64_t heads);

// Sequences over 8-bit states whose query rows are too many for the decode kernel: their codes are unpacked to FP16 (exactly) and BF16
// queries brought to it by powers of two, then the prompt kernel runs over them with the scales beside.
void attend_kv8(Device& d, const std::vector<Sequence>& sequences, uint64_t heads, uint64_t kv_heads, uint64_t dim, int code, float scale,
                float cap, const float* slopes, uint64_t window, const void* q, uint64_t q_stride, void* out, uint64_t out_stride, int type);

#if defined(__CUDACC__)
// tanh(y) in two forms. Up to |y| = 1/4 the odd series to y^9: the next term is below 2^-28 of y, and it runs on the FMA pipe alone. For any y
// 1 - 2 / (1 + e^(2y)): off by 2^-22 at most (an exponential and a reciprocal of 2^-22 and 2^-23 each).
constexpr float kSmallTanh = 0.25f;
// tanh(y) = y (kTanh1 + kTanh3 y^2 + kTanh5 y^4) up to |y| = 1/4, off by 2^-21.1 of it at most: the polynomial of least relative error (by Remez' exchange)
constexpr float kTanh1 = 0.99999958f, kTanh3 = -0.33321908f, kTanh5 = 0.12841614f;
__device__ __forceinline__ float small_tanh(float y) {
    const float z = y * y;
    float p = fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = fmaf(p, z, 2.0f / 15.0f);
    p = fmaf(p, z, -1.0f / 3.0f);
    return fmaf(p * z, y, y);
}
__device__ __forceinline__ float any_tanh(float y) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp2(y * 2.8853900817779268f)));
    return fmaf(-2.0f, r, 1.0f);
}
// One of them by the value, for caps above 64: 2^-22 of the cap is 2^-16 of a weight there and 0.02 of it at 1e5, which a score of a few units must not be off
// because another one lies far from it. Below, the second form is exact enough and faster: 4096 rows over 8192 keys, 32/8 heads of 128, most scores past a
// quarter of their cap of 5: 1275 us by it, 1510 by either; 16384 keys, 16/2 heads of 256: 1697 and 1870.
constexpr float kFineCap = 64.0f * 1.4426950408889634f;   // (caps are held in the exp2 domain)
__device__ __forceinline__ float either_tanh(float y) { return fabsf(y) <= kSmallTanh ? small_tanh(y) : any_tanh(y); }
#endif

}  // namespace attn
}  // namespace sdb
