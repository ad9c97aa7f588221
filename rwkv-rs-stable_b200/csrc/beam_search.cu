// Beam search over the vocabulary, and the reordering of recurrent states by its result.
//
// A candidate (i, t) of a search is token t behind beam i, with score[i] + x[i][t] - log sum_t exp x[i][t].  The first kernel
// takes each beam's row: its maximum, its sum of exponentials and its K largest logits, which hold every candidate of the row that can be
// chosen.  The second takes the K best of a search from the rows' candidates.  Scores are compared in 64 bits: the candidates of
// different beams lie as close together as their last bits, and a 32-bit score in the tens has only four decimals behind the point.
// Ties go to the lowest i V + t.  A logit that is NaN counts as -inf, +inf as the largest finite number.
#include <cuda_runtime.h>

#include <cfloat>

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

template <typename Value>
struct Candidate {
    Value value;
    int64_t index;
};
template <typename Value>
__device__ __forceinline__ bool before(const Candidate<Value> &a, const Candidate<Value> &b) {
    return a.value > b.value || (a.value == b.value && a.index < b.index);
}
// The first of all threads' candidates, for every thread.
template <typename Value>
__device__ Candidate<Value> block_first(Candidate<Value> c, Candidate<Value> *shared) {
    auto first_of_warp = [](Candidate<Value> x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Candidate<Value> y{__shfl_xor_sync(0xffffffffu, x.value, o), __shfl_xor_sync(0xffffffffu, x.index, o)};
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

constexpr int64_t kNone = INT64_MAX;   // behind every index: no candidate

// One beam's row: (max, sum of exp) and the K first of (logit, token); token -1 where the row has fewer.
template <typename T>
__global__ void __launch_bounds__(kThreads)
beam_rows_kernel(const BeamSelectArgs p, float2 *sums, float *values, int *tokens) {
    __shared__ Candidate<float> shared[kWarps];
    __shared__ float partial[kWarps];
    const int64_t row = blockIdx.x;
    wait_for_previous();
    const T *x = static_cast<const T *>(p.logits) + row * p.V;
    Candidate<float> last{INFINITY, -1};
    float top = 0.f;
    for (int k = 0; k < p.K; ++k) {
        Candidate<float> best{-INFINITY, kNone};
        for (int64_t t = threadIdx.x; t < p.V; t += kThreads) {
            const Candidate<float> c{clean(ldf(x + t)), t};
            if (before(last, c) && before(c, best)) best = c;
        }
        best = block_first(best, shared);
        if (k == 0) top = best.value;
        if (threadIdx.x == 0) {
            values[row * p.K + k] = best.value;
            tokens[row * p.K + k] = best.index == kNone ? -1 : (int)best.index;
        }
        last = best;
    }
    float sum = 0.f;
    if (top > -INFINITY)
        for (int64_t t = threadIdx.x; t < p.V; t += kThreads) sum += expf(clean(ldf(x + t)) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWarps; ++w) sum += partial[w];
        sums[row] = make_float2(top, sum);
    }
}

// One search: the K first of its rows' candidates.
__global__ void __launch_bounds__(kThreads)
beam_merge_kernel(const BeamSelectArgs p, const float2 *sums, const float *values, const int *tokens) {
    __shared__ Candidate<double> shared[kWarps];
    const int64_t search = blockIdx.x;
    wait_for_previous();
    const int64_t first = search * p.I;
    auto candidate = [&](int e) {
        const int i = e / p.K, k = e % p.K;
        const int64_t row = first + i;
        const float score = clean(p.scores[row]);
        if (score == -INFINITY) return Candidate<double>{-INFINITY, k < p.V ? i * p.V + k : kNone};   // whatever the logits
        if (p.finished != nullptr && p.finished[row] != 0) {   // the padding token at no cost, and nothing else
            const int64_t token = k == 0 ? p.pad_token : (k - 1) + (k - 1 >= p.pad_token);
            return Candidate<double>{k == 0 ? (double)score : -INFINITY, token < p.V ? i * p.V + token : kNone};
        }
        const int token = tokens[row * p.K + k];
        if (token < 0) return Candidate<double>{-INFINITY, kNone};
        const float x = values[row * p.K + k];
        const float2 s = sums[row];
        const double lp = x == -INFINITY ? -INFINITY : ((double)x - (double)s.x) - log((double)s.y);
        return Candidate<double>{(double)score + lp, i * p.V + token};
    };
    Candidate<double> last{INFINITY, -1};
    for (int k = 0; k < p.K; ++k) {
        Candidate<double> best{-INFINITY, kNone};
        for (int e = threadIdx.x; e < p.I * p.K; e += kThreads) {
            const Candidate<double> c = candidate(e);
            if (c.index != kNone && before(last, c) && before(c, best)) best = c;
        }
        best = block_first(best, shared);
        if (threadIdx.x == 0) {
            const int64_t o = search * p.K + k;
            p.next_scores[o] = (float)best.value;
            p.parents[o] = (int)(best.index / p.V);
            p.tokens[o] = (int)(best.index % p.V);
        }
        last = best;
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

}  // namespace

size_t beam_select_workspace_bytes(int64_t B, int64_t I, int64_t K) {
    return align16((size_t)(B * I) * sizeof(float2)) + 2 * align16((size_t)(B * I * K) * 4);
}

int launch_beam_select(const BeamSelectArgs &p, void *workspace, cudaStream_t stream) {
    char *w = static_cast<char *>(workspace);
    float2 *sums = reinterpret_cast<float2 *>(w);
    float *values = reinterpret_cast<float *>(w + align16((size_t)(p.B * p.I) * sizeof(float2)));
    int *tokens = reinterpret_cast<int *>(reinterpret_cast<char *>(values) + align16((size_t)(p.B * p.I * p.K) * 4));
    const auto rows = p.bf16 ? beam_rows_kernel<__nv_bfloat16> : beam_rows_kernel<float>;
    cudaError_t e = launch_serialized(rows, (unsigned)(p.B * p.I), (unsigned)kThreads, 0, stream, p, sums, values, tokens);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_serialized(beam_merge_kernel, (unsigned)p.B, (unsigned)kThreads, 0, stream, p, (const float2 *)sums, (const float *)values,
                                  (const int *)tokens);
}

int launch_beam_reorder(const BeamReorderArgs &p, cudaStream_t stream) {
    int64_t unit = 16, most = 0;
    for (int i = 0; i < p.n; ++i) {
        while (p.tensors[i].row_bytes % unit != 0) unit /= 2;
        if (p.tensors[i].row_bytes > most) most = p.tensors[i].row_bytes;
    }
    if (unit == 8) unit = 4;
    const int64_t wanted = (p.B * (most / unit) + kThreads - 1) / kThreads, cap = (int64_t)p.num_sms * 8;
    const unsigned blocks = (unsigned)(wanted < cap ? wanted : cap);
    if (unit == 16) return (int)launch_reorder<uint4>(p, blocks, stream);
    if (unit == 4) return (int)launch_reorder<uint32_t>(p, blocks, stream);
    return (int)launch_reorder<uint16_t>(p, blocks, stream);
}

}  // namespace rwkv7
