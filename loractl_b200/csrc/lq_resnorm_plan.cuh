// How the residual norm's work is laid out over threads, blocks and shared memory (lq_resnorm.cu): host arithmetic without CUDA,
// so that it can be checked for every width without a device.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace resnorm_plan {

constexpr int kMaxStages = 8;
constexpr size_t kRingBytes = 216 * 1024;  // shared memory of an SM for the rings of its blocks, at most
// What is there for them: 228 KB an SM, less for each block what the system keeps and its own static part; a block's share
// comes in units of 128 bytes.
constexpr size_t kSmemPerSm = 228 * 1024, kSmemOfSystem = 1024, kRingStatic = 640, kSmemUnit = 128;

inline int threads_of(int64_t h) { return (int)((h + 255) / 256 * 32); }  // 8 columns each

// Blocks of an SM: 1024 threads with the forward's 64 registers, 768 with the backward's 80 (the kernels' launch bounds).
inline int blocks_per_sm(int64_t h, bool backward) { return std::max(1, (backward ? 768 : 1024) / threads_of(h)); }

// ... and of the kernels for any rows: 8 elements a thread in up to 512 threads (128 registers; 64 in the forward), then
// up to 1024 threads, then 16 elements.
inline int scalar_threads(int64_t h) {
    const int64_t e = h <= 8192 ? 8 : 16;
    return (int)(((h + e - 1) / e + 31) / 32 * 32);
}
inline int scalar_blocks_per_sm(int64_t h, bool backward) { return std::max(1, (backward ? 512 : 1024) / scalar_threads(h)); }

// Chunks of one sample, one block each: such that all blocks fill the SMs' places once, or w times where one round
// would leave too many empty (a round beyond the last full one costs as much as a whole one: 448 blocks on 444 places took
// 292 us where 440 take 256, 8 x 4096 x 2048 forward and backward); in the backward four rows or more each where that still
// gives every SM a block (a chunk leaves three partial rows, so a short one costs as much traffic as its rows).
inline int chunks_of(int64_t samples, int64_t tokens, int64_t places, int sms, bool backward) {
    const int64_t one = (sms + samples - 1) / samples;
    const int64_t most = std::max<int64_t>(1, backward ? std::min(tokens, std::max(tokens / 4, one)) : tokens);
    int64_t best = 1, cost = -1;
    for (int64_t w = 1; w <= 4; ++w) {
        const int64_t c = std::min(most, std::max<int64_t>(1, places * w / samples));
        const int64_t t = (samples * c + places - 1) / places * ((tokens + c - 1) / c + 2);
        if (cost < 0 || t < cost) best = c, cost = t;
    }
    return (int)best;
}

// Rows in the ring of a block, 0 when fewer than two fit, such that all blocks_per_sm() blocks are resident.  Equal shares of
// kRingBytes alone let 7 of 8 in at 768 bf16 columns (backward, three inputs), and a last round of blocks ran almost alone: 62500
// rows took 162 us, with one row less in each ring 122.
inline int stages_of(int64_t h, int element_bytes, int inputs, bool backward) {
    const size_t blocks = (size_t)blocks_per_sm(h, backward);
    const size_t share = kSmemPerSm / blocks / kSmemUnit * kSmemUnit - kSmemOfSystem - kRingStatic;
    const size_t stage = (size_t)inputs * h * element_bytes, wanted = kRingBytes / blocks / stage;
    // two rows where that needs the equal share (256 f32 columns, backward with four inputs): 23 of 24 blocks with a ring
    const size_t n = wanted < 3 ? wanted : std::max<size_t>(2, std::min(wanted, share / stage));
    return n < 2 ? 0 : (int)std::min<size_t>(n, kMaxStages);
}

}  // namespace resnorm_plan
