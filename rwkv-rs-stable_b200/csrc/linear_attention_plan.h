// How a pass of linear attention is cut over a device.  Host arithmetic alone, no CUDA.
//
// A chain (b,h) is a walk over its chunks (or blocks) of tokens with a carried state.  Where there are fewer chains than CTAs that the device holds,
// a chain is cut into segments: a first pass over k and v alone gives what each segment adds to the state, then every
// segment starts from the sum of those before it.  That reads k and v twice (the second time from L2, where they fit), takes three launches
// instead of one, and pays where a segment's two walks and what the launches cost are shorter than the chain's one.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace rwkv7 {
namespace linear_attention_plan {

// Tokens of a chunk of the tensor-core kernel (one CTA per SM), and the chunks that its two launches more are worth.  bf16, one sequence of 32
// heads, in segments and in one piece: 512 tokens 17.1 and 11.9 us, 1024 (two chunks a segment) 19.7 and 18.7, 1500 (three) 23.0 and 26.0; of 4
// heads (one chunk a segment) 768 tokens 15.9 and 15.0, 1024 16.0 and 18.4.
constexpr int kChunk = 128, kChunksOfLaunches = 4;
// Of a block of the other kernel.  fp32, 32 tokens (two blocks) of 32 heads 16.2 us in segments and 13.9 in one piece, 48 15.1 and 19.3, 128 16.4
// and 47.1; 48 of 8 sequences of 32 heads 30.1 and 20.7, for the SMs are busy then, and twice the work takes twice as long.
constexpr int kBlock = 16, kBlocksOfLaunches = 1;

struct Cut {
    int64_t segments;   // per chain
    int64_t chunks;     // per segment (the last may have fewer)
};

// As many segments as there are places for them, no more than `most` (what a workspace has room for), or one.
inline Cut cut(int64_t chains, int64_t chunks, int64_t places, int64_t launches, int64_t most) {
    const int64_t segments = std::min(std::min(chunks, most), chains > 0 ? places / chains : 1);
    if (segments < 2) return {1, chunks};
    const int64_t each = (chunks + segments - 1) / segments;
    if (chunks <= 2 * each + launches) return {1, chunks};
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
