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

// Sequences over 8-bit states whose query rows are too many for the decode kernel: their codes are unpacked to 16 bits (exactly), then the
// prompt kernel runs over them with the blocks' scales beside.
void attend_kv8(Device& d, const std::vector<Sequence>& sequences, uint64_t heads, uint64_t kv_heads, uint64_t dim, int code, float scale,
                float cap, const float* slopes, uint64_t window, const void* q, uint64_t q_stride, void* out, uint64_t out_stride, int type);

}  // namespace attn
}  // namespace sdb
