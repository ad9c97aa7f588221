// Linear attention with one decay per head, token by token.
//
//   S_t = d S_{t-1} + c_t b_t^T,   y_t = S_t a_t,   d = exp(log_decay[h])      (S [N rows of c][N columns of b], fp32)
//
// over a sequence, or over the sequence reversed, where the carried matrix is the gradient G of the state behind a token:
//
//   G_t = (t last ? G_T : d G_{t+1}) + c_t b_t^T,   y_t = G_t a_t,   left over: d G_0
//
// With (a, b, c) = (q, k, v) the first is the operator itself, with (dy, v, k) and S0 transposed it is the gradient of q.  The
// second gives the gradient of v from (k, q, dy) and the gradient of k from (v, dy, q) with G_T transposed.
//
// One CTA per chain (b,h).  A thread holds part of one row of S in registers: every TPR-th group of four columns, so that the
// threads of a row read neighbouring 16-byte pieces of a and b.  Tokens are staged in shared memory, sixteen at a time, as fp32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "elements.cuh"
#include "kernels.h"
#include "launch.h"

namespace rwkv7 {
namespace {

constexpr int kBlock = 16;   // tokens staged together

// Threads that share a row of an N x N state.
__host__ __device__ constexpr int threads_per_row(int N) { return N >= 128 ? 4 : 2; }

template <typename T, int N, bool REVERSED>
__global__ void __launch_bounds__(N * threads_per_row(N))
scan_kernel(const LinearAttentionPass p) {
    constexpr int TPR = threads_per_row(N), Q = N / 4 / TPR, THREADS = N * TPR;
    __shared__ __align__(16) float sa[kBlock][N], sb[kBlock][N], sc[kBlock][N], sy[kBlock][N];
    const int64_t chain = blockIdx.x;
    const int64_t bi = chain / p.H, h = chain % p.H;
    const int tid = threadIdx.x, row = tid / TPR, part = tid % TPR;

    wait_for_previous();
    const float d = expf(p.log_decay[h]);
    const int64_t len = p.lens == nullptr ? p.T : min(max((int64_t)p.lens[bi], (int64_t)0), p.T);
    const int64_t base = (bi * p.T * p.H + h) * N;   // of token 0
    const int64_t step = p.H * N;
    const T *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b), *c = static_cast<const T *>(p.c);
    T *y = static_cast<T *>(p.y);

    float4 S[Q];
#pragma unroll
    for (int m = 0; m < Q; ++m) S[m] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.s_in != nullptr) {
        const float *src = p.s_in + chain * N * N;
#pragma unroll
        for (int m = 0; m < Q; ++m) {
            const int col = 4 * (m * TPR + part);
            if (!p.s_in_transposed) {
                S[m] = *reinterpret_cast<const float4 *>(src + row * N + col);
            } else {
                S[m] = make_float4(src[col * N + row], src[(col + 1) * N + row], src[(col + 2) * N + row], src[(col + 3) * N + row]);
            }
        }
    }

    float scale = REVERSED ? 1.f : d;   // of the state before a token is added
    for (int64_t done = 0; done < len; done += kBlock) {
        const int n = (int)min((int64_t)kBlock, len - done);
        const int64_t first = REVERSED ? len - done - n : done;   // the block's tokens are [first, first + n)
        __syncthreads();
        for (int i = tid; i < n * N; i += THREADS) {
            const int t = i / N, j = i % N;
            const int64_t at = base + (first + t) * step + j;
            sa[t][j] = ldf(a + at);
            sb[t][j] = ldf(b + at);
            sc[t][j] = ldf(c + at);
        }
        __syncthreads();
        for (int i = 0; i < n; ++i) {
            const int t = REVERSED ? n - 1 - i : i;
            const float ci = sc[t][row];
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int m = 0; m < Q; ++m) {
                const float4 bv = *reinterpret_cast<const float4 *>(&sb[t][4 * (m * TPR + part)]);
                const float4 av = *reinterpret_cast<const float4 *>(&sa[t][4 * (m * TPR + part)]);
                S[m].x = fmaf(S[m].x, scale, ci * bv.x);
                S[m].y = fmaf(S[m].y, scale, ci * bv.y);
                S[m].z = fmaf(S[m].z, scale, ci * bv.z);
                S[m].w = fmaf(S[m].w, scale, ci * bv.w);
                acc.x = fmaf(S[m].x, av.x, fmaf(S[m].z, av.z, acc.x));
                acc.y = fmaf(S[m].y, av.y, fmaf(S[m].w, av.w, acc.y));
            }
            scale = d;
            float out = acc.x + acc.y;
#pragma unroll
            for (int o = TPR / 2; o > 0; o >>= 1) out += __shfl_xor_sync(0xffffffffu, out, o);
            if (part == 0) sy[t][row] = out;
        }
        __syncthreads();
        for (int i = tid; i < n * N; i += THREADS) stf(y + base + (first + i / N) * step + i % N, sy[i / N][i % N]);
    }
    for (int64_t i = len * N + tid; i < p.T * N; i += THREADS) stf(y + base + i / N * step + i % N, 0.f);

    if (p.s_out != nullptr) {
        float *dst = p.s_out + chain * N * N + row * N;
        const float last = REVERSED && len > 0 ? d : 1.f;
#pragma unroll
        for (int m = 0; m < Q; ++m)
            *reinterpret_cast<float4 *>(dst + 4 * (m * TPR + part)) = make_float4(S[m].x * last, S[m].y * last, S[m].z * last, S[m].w * last);
    }
}

template <typename T, int N>
int launch_scan(const LinearAttentionPass &p, cudaStream_t stream) {
    const auto kernel = p.reversed ? scan_kernel<T, N, true> : scan_kernel<T, N, false>;
    return (int)launch_serialized(kernel, (unsigned)(p.B * p.H), (unsigned)(N * threads_per_row(N)), 0, stream, p);
}

template <typename T>
int launch_scan(const LinearAttentionPass &p, cudaStream_t stream) {
    switch (p.N) {
        case 32: return launch_scan<T, 32>(p, stream);
        case 64: return launch_scan<T, 64>(p, stream);
        default: return launch_scan<T, 128>(p, stream);
    }
}

}  // namespace

bool linear_attention_supported(int64_t N) { return N == 32 || N == 64 || N == 128; }

size_t linear_attention_workspace_bytes(const LinearAttentionPass &p) {
    return linear_attention_chunks_supported(p) ? linear_attention_chunks_workspace_bytes(p) : 0;
}

int launch_linear_attention(const LinearAttentionPass &p, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (linear_attention_chunks_supported(p)) return launch_linear_attention_chunks(p, workspace, workspace_bytes, stream);
    return p.bf16 ? launch_scan<__nv_bfloat16>(p, stream) : launch_scan<float>(p, stream);
}

}  // namespace rwkv7
