// How a pass of linear attention is cut over a device.  Host arithmetic alone, no CUDA.
//
// A chain (b,h) is a walk over its chunks (or blocks) of tokens with a carried state.  Where there are fewer chains than CTAs that the device holds,
// a chain is cut into segments: a first pass over k and v alone gives what each segment adds to the state, then every
// segment starts from the sum of those before it.  That reads k and v twice (the second time from L2, where they fit) and
// pays as soon as two segments of every chain run at once.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace rwkv7 {
namespace linear_attention_plan {

constexpr int kChunk = 128;   // tokens of a chunk of the tensor-core kernel
constexpr int kResident = 1;  // its CTAs per SM
constexpr int kBlock = 16;    // tokens of a block of the other kernel

struct Cut {
    int64_t segments;   // per chain
    int64_t chunks;     // per segment (the last may have fewer)
};

// As many segments as there are places for them, of `least` chunks at the least, no more than `most` (what a workspace has room for).
inline Cut cut(int64_t chains, int64_t chunks, int64_t places, int64_t least, int64_t most) {
    const int64_t segments = std::min(std::min(chunks / least, most), chains > 0 ? places / chains : 1);
    if (segments < 2) return {1, chunks};
    const int64_t each = (chunks + segments - 1) / segments;
    return {(chunks + each - 1) / each, each};
}

// fp32 states of all segments: what comes before the first, and what each but the last adds.
inline size_t state_bytes(int64_t chains, int64_t segments, int64_t N) {
    return segments < 2 ? 0 : (size_t)chains * (size_t)segments * (size_t)(N * N) * sizeof(float);
}
inline int64_t segments_in(size_t bytes, int64_t chains, int64_t N) {
    return chains > 0 ? (int64_t)(bytes / ((size_t)chains * (size_t)(N * N) * sizeof(float))) : 0;
}

}  // namespace linear_attention_plan
}  // namespace rwkv7
