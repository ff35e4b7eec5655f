// The 8-bit K/V entries through the C++ wrappers: a state written, attended by a few rows and by a chunk, compared with FP64 over the codes the
// library wrote; an eviction that keeps the rows of greatest weight; refusals that throw.
#include "straydog_b200.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <limits>

using straydog::Backend;
using straydog::Buffer;
using straydog::Error;

namespace {

int failures = 0, checks = 0;
void expect(bool good, const char* what) {
    ++checks;
    if (!good) { ++failures; std::printf("FAILED: %s\n", what); }
}

uint16_t bf16(float x) {
    uint32_t b;
    std::memcpy(&b, &x, 4);
    return uint16_t((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}
float widened(uint16_t h) {
    const uint32_t b = uint32_t(h) << 16;
    float x;
    std::memcpy(&x, &b, 4);
    return x;
}

void attend(Backend& gpu, uint64_t rows) {
    const uint64_t context = 192, length = 150, window = 100;
    const Backend::Shape shape{4, 2, 64, 0, 30};
    std::vector<uint16_t> kv[2], q(rows * shape.heads * shape.dim);
    uint32_t seed = 12345 + uint32_t(rows);
    auto next = [&] { seed = seed * 1664525u + 1013904223u; return bf16(float(int32_t(seed >> 8) % 2000 - 1000) / 500.0f); };
    for (auto& list : kv) {
        list.resize(length * shape.kv_heads * shape.dim);
        for (auto& x : list) x = next();
    }
    for (auto& x : q) x = next();
    Buffer state = gpu.buffer(Backend::kv8_bytes(context, shape.kv_heads, shape.dim)), k = gpu.upload(kv[0]), v = gpu.upload(kv[1]), queries = gpu.upload(q),
           out = gpu.buffer(q.size() * 2);
    gpu.kv8_write({state.pointer}, {context}, {0}, {length}, shape, k.pointer, v.pointer);
    std::vector<int8_t> codes(2 * shape.kv_heads * context * shape.dim);
    std::vector<float> scales(2 * shape.kv_heads * context / 32);
    gpu.read_buffer(state, 0, codes);
    gpu.read_buffer(state, codes.size() / 4, scales);
    auto element = [&](uint64_t plane, uint64_t row, uint64_t d) {
        return double(codes[(plane * context + row) * shape.dim + d]) * double(scales[plane * (context / 32) + row / 32]);
    };
    expect(std::fabs(element(1, 40, 7) - widened(kv[0][(40 * shape.kv_heads + 1) * shape.dim + 7])) <= 2.0 / 127.0, "a written key stands within half a step of its value");
    Backend::Rule rule;
    rule.scale = 0.125f;
    rule.window = window;
    gpu.kv8_attention({state.pointer}, {context}, {length}, {rows}, shape, rule, queries.pointer, out.pointer);
    std::vector<uint16_t> got(q.size());
    gpu.read_buffer(out, 0, got);
    bool close = true;
    for (uint64_t r = 0; r < rows; ++r)
        for (uint64_t h = 0; h < shape.heads; ++h) {
            const uint64_t position = length - rows + r, first = position + 1 > window ? position + 1 - window : 0, kvh = h / (shape.heads / shape.kv_heads);
            std::vector<double> s;
            double top = -std::numeric_limits<double>::infinity(), total = 0.0;
            for (uint64_t j = first; j <= position; ++j) {
                double dot = 0.0;
                for (uint64_t d = 0; d < shape.dim; ++d) dot += double(widened(q[(r * shape.heads + h) * shape.dim + d])) * element(kvh, j, d);
                s.push_back(dot * 0.125);
                top = std::max(top, s.back());
            }
            for (auto& x : s) { x = std::exp(x - top); total += x; }
            for (uint64_t d = 0; d < shape.dim; ++d) {
                double sum = 0.0, size = 0.0;
                for (uint64_t j = first; j <= position; ++j) {
                    const double term = s[j - first] / total * element(shape.kv_heads + kvh, j, d);
                    sum += term; size += std::fabs(term);
                }
                // half a step of the output and of each weight in BF16, 2^-16 for the FP32 arithmetic
                const double bound = std::ldexp(std::fabs(sum), -8) + (std::ldexp(1.0, -8) + std::ldexp(1.0, -16)) * size;
                close = close && std::fabs(widened(got[(r * shape.heads + h) * shape.dim + d]) - sum) <= bound;
            }
        }
    expect(close, "attention over 8-bit rows against FP64 over their codes");
    expect(gpu.decode_status() == 0, "no bounded wait gave up");
    for (Buffer* b : {&state, &k, &v, &queries, &out}) gpu.release(*b);
}

void evict(Backend& gpu) {
    const Backend::Shape shape{1, 1, 64, 0, 1};
    Buffer state = gpu.buffer(Backend::kv8_bytes(64, 1, 64)), target = gpu.buffer(Backend::kv8_bytes(32, 1, 64)), kept = gpu.buffer(8 * 4), moved = gpu.buffer(32 * 4);
    std::vector<float> weights(64);
    for (int i = 0; i < 64; ++i) weights[i] = float((i * 37) % 64);
    Buffer w = gpu.upload(weights);
    gpu.kv8_evict({state.pointer}, {64}, {64}, {w.at<float>()}, 8, 1, 2, shape, {target.pointer}, {32}, {moved.at<float>()}, kept.at<int32_t>());
    std::vector<int32_t> got(8);
    gpu.read_buffer(kept, 0, got);
    std::vector<int32_t> want{0, 62, 63};
    for (int value = 63; want.size() < 8; --value)
        for (int i = 1; i < 62; ++i)
            if ((i * 37) % 64 == value) want.push_back(i);
    std::sort(want.begin(), want.end());
    expect(got == want, "the positions an eviction keeps");
    for (Buffer* b : {&state, &target, &kept, &moved, &w}) gpu.release(*b);
}

void errors(Backend& gpu) {
    bool thrown = false;
    try { Backend::kv8_bytes(33, 1, 64); } catch (const Error& e) { thrown = std::strlen(e.what()) > 0; }
    expect(thrown, "a context that is no multiple of 32 is refused");
    thrown = false;
    try { gpu.kv8_write({nullptr}, {64, 64}, {0}, {1}, {1, 1, 64, 0, 1}, nullptr, nullptr); } catch (const Error&) { thrown = true; }
    expect(thrown, "lists of different lengths are refused");
    thrown = false;
    try { gpu.kv8_write({nullptr}, {64}, {0}, {1}, {1, 1, 64, 0, 1}, nullptr, nullptr); } catch (const Error&) { thrown = true; }
    expect(thrown, "a null state is refused");
}

}  // namespace

int main() {
    try {
        Backend gpu(0, 1ull << 28);
        attend(gpu, 1);
        attend(gpu, 3);
        attend(gpu, 120);
        evict(gpu);
        errors(gpu);
    } catch (const std::exception& e) {
        std::printf("FAILED: %s\n", e.what());
        return 1;
    }
    if (failures) return 1;
    std::printf("ok %d\n", checks);
    return 0;
}
