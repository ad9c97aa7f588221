// The cut of a pass of linear attention, for the tests.
#include "linear_attention_plan.h"

using namespace rwkv7::linear_attention_plan;

extern "C" void linear_attention_cut(int64_t chains, int64_t chunks, int64_t places, int64_t launches, int64_t most, int64_t *out) {
    const Cut c = cut(chains, chunks, places, launches, most);
    out[0] = c.segments;
    out[1] = c.chunks;
}
extern "C" int64_t linear_attention_segments_in(int64_t bytes, int64_t chains, int64_t N) { return segments_in((size_t)bytes, chains, N); }
extern "C" int64_t linear_attention_state_bytes(int64_t chains, int64_t segments, int64_t N) { return (int64_t)state_bytes(chains, segments, N); }
