// Beam search over the vocabulary, and the reordering of recurrent states by its result.
//
// A candidate (i, t) of a search is token t behind beam i, with score[i] + x[i][t] - log sum_t exp x[i][t].  The first kernel
// goes once over the beams' rows: the maximum, the sum of exponentials and the K largest logits, among which are all that can be chosen.
// Its floor is the bytes of the logits; it is bound by its instructions, some seven a logit (unpack, maximum, scale, exponential, sum and
// their surroundings).  So nothing else is done to most of them: a bound under the K-th largest is known, the K-th largest of the threads'
// maxima of some 8192 logits, which at least K reach and hardly more, and only a thread whose maximum reaches it puts its logits aside; those
// are gone through from time to time, by all threads, and the bound is raised to the K-th largest of what was kept.  512 rows of 65536 bf16,
// K = 8: 24 us, 10.2 by its bytes (27.8 where the bound stayed where it was).  The second kernel takes the K best of a search from its
// rows' sorted lists; four rows of 65536 fp32 take both kernels 7.5 us (13.5 with every list's head ranked against every other's).
// Masked vocabularies and rows of equal logits stay on that way: a thread without ordinary logits has no sum, equals are bounded by their tokens as well,
// and where fewer logits are above -inf than are chosen the first other tokens fill up (512 rows with nine tenths masked 21 to 44 us, all equal 41).  What
// holds NaN or +inf is gone through once more for the sum and for every choice (370 us).
// Scores are compared in 64 bits: the candidates of different beams lie as close together as their last bits, and a 32-bit score in
// the tens has only four decimals behind the point.  Ties go to the lowest i V + t.  A logit that is NaN counts as -inf, +inf as the
// largest finite number.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cstdint>

#include "elements.cuh"
#include "kernels.h"
#include "launch.h"
#include "rwkv7_b200.h"

namespace rwkv7 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

__device__ __forceinline__ float clean(float x) {
    if (x != x) return -INFINITY;
    return fminf(x, FLT_MAX);
}

template <typename Value, typename Index>
struct Candidate {
    Value value;
    Index index;
};
template <typename C>
__device__ __forceinline__ bool before(const C &a, const C &b) {
    return a.value > b.value || (a.value == b.value && a.index < b.index);
}
// The first of all threads' candidates, for every thread.
template <typename C>
__device__ C block_first(C c, C *shared) {
    auto first_of_warp = [](C x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const C y{__shfl_xor_sync(0xffffffffu, x.value, o), __shfl_xor_sync(0xffffffffu, x.index, o)};
            if (before(y, x)) x = y;
        }
        return x;
    };
    c = first_of_warp(c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = c;
    __syncthreads();
    return first_of_warp(shared[threadIdx.x & (kWarps - 1)]);
}

constexpr int kVectors = 4;                          // 16-byte vectors a thread has in registers, and as many on their way
constexpr int kMostAside = kThreads + 32;            // threads' vectors put aside: gone through when there are more than 32
constexpr int kMostKept = 2048;                      // logits over the bound: room for; it is raised when they are many for K
constexpr int kMostRanked = 256;                     // of them, each against each; more come of many equal ones alone
constexpr float kLowest = -1e38f;                    // where x log2 e is still a number; masks are below
constexpr int kMostSplits = 32;                      // CTAs on a row

// Pieces of a row.  They start on 16 bytes, the first at or (where rows are not whole vectors) before the row's start.
constexpr int64_t pieces(int64_t V, bool bf16) {
    const int64_t vec = bf16 ? 8 : 4, piece = kThreads * kVectors * vec;
    return (V + (V % vec == 0 ? 0 : vec - 1) + piece - 1) / piece;
}

// A float as an unsigned number of the same order.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u ^ ((u & 0x80000000u) ? 0x80000000u : 0xffffffffu)); }

// The lanes' values in falling order.
template <typename U>
__device__ __forceinline__ U warp_sort(U x, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
            const U y = __shfl_xor_sync(0xffffffffu, x, j);
            x = ((lane & j) == 0) == ((lane & k) == 0) ? max(x, y) : min(x, y);
        }
    return x;
}
// The 32 largest of two falling lists, falling.
template <typename U>
__device__ __forceinline__ U warp_merge(U x, U other, int lane) {
    x = max(x, __shfl_sync(0xffffffffu, other, 31 - lane));
#pragma unroll
    for (int j = 16; j > 0; j /= 2) {
        const U y = __shfl_xor_sync(0xffffffffu, x, j);
        x = (lane & j) == 0 ? max(x, y) : min(x, y);
    }
    return x;
}

// Some pieces of one row: (max, sum of exp(x - max)) and the K first of (logit, token); token -1 where there are fewer.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
beam_rows_kernel(const BeamSelectArgs p, int splits, int each, int n_pieces, float2 *sums, float *values, int *tokens) {
    constexpr int VEC = 16 / (int)sizeof(T), NV = kVectors, kPer = NV * VEC, kPiece = kThreads * kPer;
    constexpr float kLog2e = 1.4426950408889634f;
    __shared__ Candidate<float, int> shared[kWarps];
    __shared__ uint32_t tops[kWarps][32];
    __shared__ uint64_t firsts[kWarps][32];
    __shared__ float2 partial[kWarps];
    __shared__ uint64_t kept[kMostKept];
    __shared__ uint64_t best[32];
    __shared__ uint4 aside[kMostAside][kVectors];
    __shared__ int aside_from[kMostAside];   // its first token
    __shared__ int n_kept, n_before, n_aside, full[2];   // `full`, of even and odd pieces: what is aside is to be gone through
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t out = blockIdx.x, row = out / splits;
    const int split = (int)(out - row * splits), stop = min(n_pieces, (split + 1) * each);
    if (tid == 0) n_kept = n_before = n_aside = full[0] = full[1] = 0;
    wait_for_previous();
    let_next_in();
    const T *logits = static_cast<const T *>(p.logits);
    const int64_t begin = row * p.V, end = begin + p.V;
    const int64_t base = begin / VEC * VEC;
    const int V = (int)p.V;

    uint4 raw[NV], coming[NV];
    // Logits outside the row read as -inf; so do they count, wherever one is not picked by its place.
    auto load = [&](uint4 (&raw)[NV], int64_t first) {
        if (first >= begin && first + kPiece <= end) {
            const uint4 *at = reinterpret_cast<const uint4 *>(logits + first) + tid;
#pragma unroll
            for (int i = 0; i < NV; ++i) raw[i] = __ldcs(at + i * kThreads);
            return;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t at = first + (i * kThreads + tid) * VEC;
            constexpr uint32_t kLow = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
            raw[i] = make_uint4(kLow, kLow, kLow, kLow);
            if (at >= begin && at + VEC <= end) {
                raw[i] = __ldcs(reinterpret_cast<const uint4 *>(logits + at));
            } else if (at + VEC > begin && at < end) {   // the row's ends
                uint32_t v[4] = {kLow, kLow, kLow, kLow};
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (at + e < begin || at + e >= end) continue;
                    const uint32_t x = __float_as_uint(ldf(logits + at + e));
                    if constexpr (sizeof(T) == 4) v[e] = x;
                    else v[e / 2] = e & 1 ? (v[e / 2] & 0xffffu) | x : (v[e / 2] & 0xffff0000u) | x >> 16;
                }
                raw[i] = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
    };
    auto value = [&](int j) {   // (static indexes)
        const uint4 &r = raw[j / VEC];
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j % 4]);
        else return __uint_as_float(j & 1 ? w[j % 8 / 2] & 0xffff0000u : w[j % 8 / 2] << 16);
    };
    auto token = [&](int lead, int j) { return lead + (j / VEC * kThreads + tid) * VEC + j % VEC; };
    float top = -INFINITY, sum = 0.f;   // of this thread's logits
    // What is looked at reaches this (-inf never does).  Where K tokens in front of the piece were kept it is above the least of them: of equals they
    // go first.
    float bound = -FLT_MAX;
    // All threads: what is aside and reaches the bound is kept; with much kept the bound is raised.  (Nobody puts aside meanwhile.)
    auto go_through = [&] {
        __syncthreads();
        const int n = n_aside * kPer;
        auto each_aside = [&](auto &&use) {
            for (int i = tid; i < n; i += kThreads) {
                const int e = i / kPer, j = i % kPer;
                const float x = ldf(reinterpret_cast<const T *>(aside[e]) + j);
                // (-0 is 0)
                if (x >= bound) use((uint64_t)ordered(x + 0.f) << 32 | (uint32_t)~(uint32_t)(aside_from[e] + j / VEC * kThreads * VEC + j % VEC));
            }
        };
        auto keep = [&](uint64_t least, int enough) {
            each_aside([&](uint64_t x) {
                if (x < least || *(volatile int *)&n_kept > enough) return;
                const int at = atomicAdd(&n_kept, 1);
                if (at < kMostKept) kept[at] = x;
            });
            __syncthreads();
        };
        keep(0, kMostRanked);
        const bool many = n_kept > kMostRanked;
        if (many) {
            // Again, by the K-th of what is the threads' first: K threads at most have any that reach it, 36 each.
            uint64_t mine = 0;
            each_aside([&](uint64_t x) { mine = max(mine, x); });
            firsts[warp][lane] = warp_sort(mine, lane);
            __syncthreads();
            if (tid == 0) n_kept = n_before;
            uint64_t list = firsts[0][lane];
#pragma unroll 1
            for (int w = 1; w < kWarps; ++w) list = warp_merge(list, firsts[w][lane], lane);
            __syncthreads();
            keep(__shfl_sync(0xffffffffu, list, p.K - 1), kMostKept);
        }
        if (tid == 0) n_aside = 0;
        if (many || n_kept > 2 * p.K + 16) {   // (there are K)
            const int n = n_kept;
            for (int i = tid; i < n; i += kThreads) {
                const uint64_t mine = kept[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += kept[j] > mine;
                if (rank < p.K) best[rank] = mine;
            }
            __syncthreads();
            if (tid < p.K) kept[tid] = best[tid];
            if (tid == 0) n_kept = p.K;
            bound = fmaxf(bound, unordered((uint32_t)(best[p.K - 1] >> 32) + 1));
        }
        __syncthreads();
        if (tid == 0) n_before = n_kept;
    };
    auto sum_of_block = [&](float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        __syncthreads();
        if (lane == 0) partial[warp].y = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) x += partial[w].y;
        return x;
    };

    load(coming, base + (int64_t)split * each * kPiece);
    for (int piece = split * each; piece < stop; ++piece) {
        const int64_t first = base + (int64_t)piece * kPiece;
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = coming[i];
        if (piece + 1 < stop) load(coming, first + kPiece);
        float most;   // (both maxima pass over NaN)
        if constexpr (sizeof(T) == 4) {
            most = -INFINITY;
#pragma unroll
            for (int j = 0; j < kPer; ++j) most = fmaxf(most, value(j));
        } else {
            const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(raw);
            __nv_bfloat162 m = h[0];
#pragma unroll
            for (int j = 1; j < kPer / 2; ++j) m = __hmax2(m, h[j]);
            most = fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);
        }
        // 2^(x log2 e - c), c being the maximum's log2 e rounded; what the rounding takes is put back behind the sum.  (A thread that has seen nothing
        // but masked logits has no sum: beside any other it is nothing, and a row without any other is summed below.)
        if (most > top) {
            sum *= exp2f((top - most) * kLog2e);
            top = most;
        }
        if (top > kLowest) {
            const float c = top * kLog2e;
            float2 part = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < kPer; j += 2) {
                const float2 x = __ffma2_rn(make_float2(value(j), value(j + 1)), make_float2(kLog2e, kLog2e), make_float2(-c, -c));
                float2 e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
                part = __fadd2_rn(part, e);
            }
            sum += (part.x + part.y) * exp2f(fmaf(-top, kLog2e, c));
        }
        // the bound, where more threads than it should reach it
        if (__syncthreads_count(most >= bound) > 2 * 32) {
            tops[warp][lane] = warp_sort(ordered(most), lane);
            __syncthreads();
            uint32_t list = tops[0][lane];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) list = warp_merge(list, tops[w][lane], lane);
            bound = unordered(__shfl_sync(0xffffffffu, list, p.K - 1));
        }
        if (full[(piece + 1) & 1] != 0) {   // (set, if at all, while the piece before was dealt with: the same for all)
            go_through();
            if (tid == 0) full[(piece + 1) & 1] = 0;
        }
        if (most >= bound) {
            const int at = atomicAdd(&n_aside, 1);
#pragma unroll
            for (int i = 0; i < NV; ++i) aside[at][i] = raw[i];
            aside_from[at] = (int)(first - begin) + tid * VEC;   // (not a token yet in front of the row)
            if (at >= kMostAside - kThreads) full[piece & 1] = 1;
        }
    }
    go_through();
    // The block's maximum and sum.
    float block_top = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) block_top = fmaxf(block_top, __shfl_xor_sync(0xffffffffu, block_top, o));
    if (lane == 0) partial[warp].x = block_top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) block_top = fmaxf(block_top, partial[w].x);
    const int from = (int)max((int64_t)0, base + (int64_t)split * each * kPiece - begin);
    const int to = (int)min((int64_t)V, base + (int64_t)stop * kPiece - begin);
    if (block_top == -INFINITY) {   // nothing but -inf and NaN: the first places
        if (tid < p.K) {
            values[out * p.K + tid] = -INFINITY;
            tokens[out * p.K + tid] = from + tid < to ? from + tid : -1;
        }
        if (tid == 0) sums[out] = make_float2(-INFINITY, 0.f);
        return;
    }
    float total = sum_of_block(top == -INFINITY ? sum : sum * exp2f((top - block_top) * kLog2e));
    // (NaN, +inf and numbers near it, which the sum does not stand)
    const bool plain = total < INFINITY && block_top < -kLowest;
    const float top_clean = clean(block_top);
    // Summed again, which is rare: NaN and +inf as what they count for; a row of masks alone; and a row of fewer logits than are chosen, whose terms are
    // the same numbers whichever thread has them, so that equal rows are equal wherever they lie.
    if (!plain || block_top <= kLowest || (n_pieces == 1 && n_kept < p.K)) {
        sum = 0.f;
        for (int piece = split * each; piece < stop; ++piece) {
            load(raw, base + (int64_t)piece * kPiece);
#pragma unroll
            for (int j = 0; j < kPer; ++j) sum += expf(clean(value(j)) - top_clean);
        }
        total = sum_of_block(sum);
    }
    if (tid == 0) sums[out] = make_float2(top_clean, total);
    if (plain) {
        const int n = n_kept;
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t mine = kept[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += kept[j] > mine;
            if (rank < p.K) {
                values[out * p.K + rank] = unordered((uint32_t)(mine >> 32));
                tokens[out * p.K + rank] = (int)~(uint32_t)mine;
            }
        }
        if (n < p.K && warp == 0) {   // all that is above -inf was kept: the first other tokens fill up
            bool other = from + lane < to;
            for (int j = 0; j < n; ++j) other = other && (int)~(uint32_t)kept[j] != from + lane;
            const uint32_t others = __ballot_sync(0xffffffffu, other);
            const int rank = n + (other ? __popc(others & ((1u << lane) - 1)) : __popc(others) + __popc(~others & ((1u << lane) - 1)));
            if (rank < p.K) {
                values[out * p.K + rank] = -INFINITY;
                tokens[out * p.K + rank] = other ? from + lane : -1;
            }
        }
        return;
    }
    // NaN and the like: one choice after the other.
    Candidate<float, int> last{INFINITY, -1};
    for (int k = 0; k < p.K; ++k) {
        Candidate<float, int> found{-INFINITY, INT_MAX};
        for (int piece = split * each; piece < stop; ++piece) {
            if (each > 1) load(raw, base + (int64_t)piece * kPiece);
            const int lead = (int)(base + (int64_t)piece * kPiece - begin);
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const Candidate<float, int> x{clean(value(j)), token(lead, j)};
                if (x.index >= 0 && x.index < V && before(last, x) && before(x, found)) found = x;
            }
        }
        found = block_first(found, shared);
        if (tid == 0) {
            values[out * p.K + k] = found.value;
            tokens[out * p.K + k] = found.index == INT_MAX ? -1 : found.index;
        }
        last = found;
    }
}

__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u ^ ((uint64_t)((int64_t)u >> 63) | (uint64_t)1 << 63);
}
__device__ __forceinline__ double unordered(uint64_t u) {
    return __longlong_as_double((long long)(u ^ (u >> 63 ? (uint64_t)1 << 63 : ~(uint64_t)0)));
}
struct Choice {
    uint64_t score;   // ordered; 0 is none
    int beam, token;
};
__device__ constexpr Choice kNoChoice{0, INT_MAX, INT_MAX};

// One search: the K first of its sorted lists, one of every split of every beam.  They come from the K lists with the first heads, which
// are at most 32: one warp, a list a lane, takes the first of all heads K times.
__global__ void __launch_bounds__(kThreads)
beam_merge_kernel(const BeamSelectArgs p, int splits, const float2 *sums, const float *values, const int *tokens) {
    __shared__ double log_sum[32];   // of a row, behind its maximum
    __shared__ float top[32];
    __shared__ Choice heads[32 * kMostSplits], lists_of[32][32];
    __shared__ uint64_t ranked[32 * kMostSplits];   // heads that may be among the first, in any order
    __shared__ int ranked_list[32 * kMostSplits], n_ranked, chosen[32];
    __shared__ uint32_t tops[kWarps][32];
    const int64_t search = blockIdx.x, first = search * p.I;
    const int lists = p.I * splits, tid = threadIdx.x;
    if (tid == 0) n_ranked = 0;
    wait_for_previous();
    // A list's entry is asked for before what its row adds to it is known.
    auto entry = [&](int l, int k) {
        const int64_t at = (first * splits + l) * p.K + k;
        return Candidate<float, int>{values[at], tokens[at]};
    };
    const Candidate<float, int> mine = tid < lists ? entry(tid, 0) : Candidate<float, int>{0.f, -1};
    {   // eight lanes a row.  The parts' sums are good to 32 bits, and so are the factors; the sum of sums and its logarithm have 64.
        const int i = tid >> 3, lane = tid & 7;
        float2 s[kMostSplits / 8];
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < kMostSplits / 8; ++j) {
            s[j] = i < p.I && lane + 8 * j < splits ? sums[(first + i) * splits + lane + 8 * j] : make_float2(-INFINITY, 0.f);
            most = fmaxf(most, s[j].x);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < kMostSplits / 8; ++j)
            if (s[j].y > 0.f) sum += (double)(s[j].y * expf(s[j].x - most));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (i < p.I && lane == 0) {
            top[i] = most;
            log_sum[i] = sum;
        }
    }
    __syncthreads();
    if (tid < p.I) log_sum[tid] = log(log_sum[tid]);   // (one warp: a double's logarithm is long)
    __syncthreads();
    auto candidate = [&](int l, int k, Candidate<float, int> c) {
        const int i = l / splits;
        const int64_t row = first + i;
        const float score = clean(p.scores[row]), x = c.value;
        const int token = c.index;
        const bool finished = p.finished != nullptr && p.finished[row] != 0;
        if (score == -INFINITY || finished) {
            // -inf whatever the logits; finished: the padding token at no cost, and nothing else
            const int64_t t = score == -INFINITY ? k : k == 0 ? p.pad_token : (k - 1) + (k - 1 >= p.pad_token);
            if (l != i * splits || t >= p.V) return kNoChoice;
            return Choice{ordered(k == 0 ? (double)score : -INFINITY), i, (int)t};
        }
        if (token < 0) return kNoChoice;
        const double lp = x == -INFINITY ? -INFINITY : ((double)x - (double)top[i]) - log_sum[i];
        return Choice{ordered((double)score + lp), i, token};
    };
    for (int l = tid; l < lists; l += kThreads) heads[l] = candidate(l, 0, l == tid ? mine : entry(l, 0));
    __syncthreads();
    const int n = min(lists, p.K);
    if (lists <= p.K) {
        if (tid < lists) chosen[tid] = tid;
    } else {
        // Of many lists only those whose heads reach the K-th largest of the threads' first heads (its upper half) are ranked.
        uint32_t bound = 0;
        if (lists > 64) {
            uint32_t most = 0;
            for (int l = tid; l < lists; l += kThreads) most = max(most, (uint32_t)(heads[l].score >> 32));
            tops[tid >> 5][tid & 31] = warp_sort(most, tid & 31);
            __syncthreads();
            uint32_t list = tops[0][tid & 31];
            for (int w = 1; w < kWarps; ++w) list = warp_merge(list, tops[w][tid & 31], tid & 31);
            bound = __shfl_sync(0xffffffffu, list, p.K - 1);
        }
        for (int l = tid; l < lists; l += kThreads) {
            if ((uint32_t)(heads[l].score >> 32) < bound) continue;
            const int at = atomicAdd(&n_ranked, 1);
            ranked[at] = heads[l].score;
            ranked_list[at] = l;
        }
        __syncthreads();
        for (int e = tid; e < n_ranked; e += kThreads) {
            const uint64_t score = ranked[e];
            const int l = ranked_list[e];
            int rank = 0;   // of equal scores the earlier list has the lower beam, or the lower token
#pragma unroll 8
            for (int j = 0; j < n_ranked; ++j) rank += (ranked[j] > score) | ((ranked[j] == score) & (ranked_list[j] < l));
            if (rank < p.K) chosen[rank] = l;
        }
    }
    __syncthreads();
    for (int e = tid; e < n * p.K; e += kThreads) {
        const int l = e / p.K, k = e - l * p.K;
        lists_of[l][k] = k == 0 ? heads[chosen[l]] : candidate(chosen[l], k, entry(chosen[l], k));
    }
    __syncthreads();
    if (tid >= 32) return;
    int taken = 0;
    Choice head = tid < n ? lists_of[tid][0] : kNoChoice;
    for (int k = 0; k < p.K; ++k) {
        // the largest score; of several the lowest beam, then the lowest token
        constexpr unsigned kAll = 0xffffffffu;
        const uint32_t hi = (uint32_t)(head.score >> 32), lo = (uint32_t)head.score;
        const uint32_t most = __reduce_max_sync(kAll, hi), least = __reduce_max_sync(kAll, hi == most ? lo : 0u);
        bool mine = hi == most && lo == least;
        if (__popc(__ballot_sync(kAll, mine)) > 1) {
            const int beam = __reduce_min_sync(kAll, mine ? head.beam : INT_MAX);
            mine = mine && head.beam == beam;
            const int token = __reduce_min_sync(kAll, mine ? head.token : INT_MAX);
            mine = mine && head.token == token;
        }
        if (mine) {
            const int64_t o = search * p.K + k;
            p.next_scores[o] = (float)unordered(head.score);
            p.parents[o] = head.beam;
            p.tokens[o] = head.token;
            head = ++taken < p.K ? lists_of[tid][taken] : kNoChoice;
        }
    }
}

// A thread moves one 16-byte (4-, 2-byte) piece of all of a search's beams: it holds the parents' pieces before it writes the
// first, so that the states may be reordered where they lie.  What stays in place is neither read nor written then.
template <typename Unit, int K>
__global__ void __launch_bounds__(kThreads)
beam_reorder_kernel(const BeamReorderArgs p) {
    wait_for_previous();
    const auto &t = p.tensors[blockIdx.y];
    const int64_t units = t.row_bytes / (int64_t)sizeof(Unit);
    const bool in_place = t.from == t.to;
    for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < p.B * units; at += (int64_t)gridDim.x * kThreads) {
        const int64_t search = at / units, piece = at % units;
        const Unit *from = static_cast<const Unit *>(t.from) + search * p.I * units + piece;
        Unit *to = static_cast<Unit *>(t.to) + search * p.K * units + piece;
        Unit held[K];
        bool moves[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            moves[j] = false;
            if (j < p.K) {
                const int64_t parent = p.parents_i64 ? static_cast<const int64_t *>(p.parents)[search * p.K + j]
                                                     : (int64_t) static_cast<const int *>(p.parents)[search * p.K + j];
                const bool valid = parent >= 0 && parent < p.I;
                if (!valid && piece == 0) atomicExch(p.status, (int)kDevBadIndex);
                moves[j] = valid && !(in_place && parent == j);
                if (moves[j]) held[j] = from[parent * units];
            }
        }
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (moves[j]) to[j * units] = held[j];
    }
}

template <typename Unit>
cudaError_t launch_reorder(const BeamReorderArgs &p, unsigned blocks, cudaStream_t stream) {
    const auto kernel = p.K <= 4 ? beam_reorder_kernel<Unit, 4> : p.K <= 8 ? beam_reorder_kernel<Unit, 8>
                        : p.K <= 16 ? beam_reorder_kernel<Unit, 16> : beam_reorder_kernel<Unit, 32>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, (unsigned)p.n);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e == cudaSuccess) count_launch();
    return e;
}

size_t align16(size_t x) { return (x + 15) / 16 * 16; }
size_t list_bytes(size_t lists, int K) { return align16(lists * sizeof(float2)) + 2 * align16(lists * (size_t)K * 4); }

// CTAs on a row and the pieces each takes: as many as the device has places for and the workspace room, one at least.
struct RowCut {
    int n, splits, each;   // pieces of a row, CTAs, pieces of a CTA
};
RowCut cut_rows(const BeamSelectArgs &p, size_t room) {
    const int64_t n = pieces(p.V, p.bf16), rows = p.B * p.I;
    int64_t most = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(n, kMostSplits), 4 * (int64_t)p.num_sms / rows));
    while (most > 1 && list_bytes((size_t)(rows * most), p.K) > room) --most;
    const int64_t each = (n + most - 1) / most;
    return {(int)n, (int)((n + each - 1) / each), (int)each};
}

}  // namespace

size_t beam_select_workspace_bytes(const BeamSelectArgs &p) { return list_bytes((size_t)(p.B * p.I * cut_rows(p, SIZE_MAX).splits), p.K); }
size_t beam_select_min_workspace_bytes(const BeamSelectArgs &p) { return list_bytes((size_t)(p.B * p.I), p.K); }

int launch_beam_select(const BeamSelectArgs &p, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    const RowCut cut = cut_rows(p, workspace_bytes);
    const int64_t lists = p.B * p.I * cut.splits;
    char *w = static_cast<char *>(workspace);
    float2 *sums = reinterpret_cast<float2 *>(w);
    float *values = reinterpret_cast<float *>(w + align16((size_t)lists * sizeof(float2)));
    int *tokens = reinterpret_cast<int *>(reinterpret_cast<char *>(values) + align16((size_t)(lists * p.K) * 4));
    const auto kernel = p.bf16 ? beam_rows_kernel<__nv_bfloat16> : beam_rows_kernel<float>;
    cudaError_t e = launch_serialized(kernel, (unsigned)lists, (unsigned)kThreads, 0, stream, p, cut.splits, cut.each, cut.n, sums, values, tokens);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_serialized(beam_merge_kernel, (unsigned)p.B, (unsigned)kThreads, 0, stream, p, cut.splits, (const float2 *)sums,
                                  (const float *)values, (const int *)tokens);
}

int launch_beam_reorder(const BeamReorderArgs &p, int unit, cudaStream_t stream) {
    int64_t most = 0;
    for (int i = 0; i < p.n; ++i) most = std::max(most, p.tensors[i].row_bytes);
    const unsigned blocks = (unsigned)std::min<int64_t>((p.B * (most / unit) + kThreads - 1) / kThreads, (int64_t)p.num_sms * 8);
    if (unit == 16) return (int)launch_reorder<uint4>(p, blocks, stream);
    if (unit == 4) return (int)launch_reorder<uint32_t>(p, blocks, stream);
    return (int)launch_reorder<uint16_t>(p, blocks, stream);
}

}  // namespace rwkv7
