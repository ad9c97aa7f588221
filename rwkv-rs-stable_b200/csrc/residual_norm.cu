// What stands between two blocks of a cell, one row of C channels at a time:
//
//   u = norm_post(h) (or h),   x' = x + s (g u),   z = norm_pre(x')
//   norm(v) = (v - mean v) / sqrt(var v + eps) gamma + beta        (layer; rms: without the mean)
//
// and its gradients.  Both are bound by the bytes of the rows: a CTA keeps a row in registers, eight channels a thread, so that every
// element is read once and every result is rounded once, on its way out.  Means and variances are taken in turn (the variance from
// the differences, which a large mean does not spoil), in fp32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "elements.cuh"
#include "kernels.h"
#include "launch.h"

namespace rwkv7 {
namespace {

constexpr int kPer = 8;           // channels a thread
constexpr int kMaxWarps = 32;
constexpr int kParams = 5;        // summed over the rows: scale, post gamma, post beta, pre gamma, pre beta

// Eight channels of a row: neighbours where rows start on 16 bytes (VEC), else every threads-th.
template <typename T, bool VEC>
struct Lane {
    int C, tid, threads;
    __device__ int channel(int i) const { return VEC ? tid * kPer + i : tid + i * threads; }
    __device__ bool any() const { return channel(0) < C; }
    // (what lies outside the row counts as zero)
    __device__ void load(float (&v)[kPer], const T *row) const {
        if constexpr (VEC) {
            if (any()) { ld8(v, row + tid * kPer); return; }
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = !VEC && channel(i) < C ? ldf(row + channel(i)) : 0.f;
    }
    __device__ void store(T *row, const float (&v)[kPer]) const {
        if constexpr (VEC) {
            if (any()) st8(row + tid * kPer, v);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (channel(i) < C) stf(row + channel(i), v[i]);
        }
    }
    __device__ bool inside(int i) const { return VEC ? any() : channel(i) < C; }
};

// The sums of `K` values over the block.  `slot` alternates between calls, so that one barrier a sum is enough.
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float (*shared)[kMaxWarps][2], int &slot, int warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (warps == 1) return;
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) shared[slot][warp][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float x = lane < warps ? shared[slot][lane][k] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        v[k] = x;
    }
    slot ^= 1;
}

// v -> (v - mean) / sqrt(var + eps); returns the reciprocal root.
template <typename L>
__device__ __forceinline__ float normalize(float (&v)[kPer], const L &lane, bool layer, float eps, float (*shared)[kMaxWarps][2], int &slot, int warps) {
    float sum[1];
    const float inv = 1.f / (float)lane.C;
    if (layer) {
        sum[0] = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum[0] += v[i];
        block_sum(sum, shared, slot, warps);
        const float mean = sum[0] * inv;
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = lane.inside(i) ? v[i] - mean : 0.f;
    }
    sum[0] = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum[0] = fmaf(v[i], v[i], sum[0]);
    block_sum(sum, shared, slot, warps);
    const float r = 1.f / sqrtf(fmaf(sum[0], inv, eps));
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] *= r;
    return r;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(1024)
residual_norm_kernel(const ResidualNormArgs p) {
    __shared__ float shared[2][kMaxWarps][2];
    const Lane<T, VEC> lane{(int)p.C, (int)threadIdx.x, (int)blockDim.x};
    const int warps = (int)blockDim.x >> 5;
    int slot = 0;
    wait_for_previous();
    auto param = [&](float (&v)[kPer], const void *q, float absent) {
        if (q != nullptr) lane.load(v, static_cast<const T *>(q));
        else
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] = absent;
    };
    const int64_t at = (int64_t)blockIdx.x * p.C;
    float x[kPer], u[kPer], w[kPer];
    lane.load(x, static_cast<const T *>(p.residual) + at);
    if (p.block_output != nullptr) {
        lane.load(u, static_cast<const T *>(p.block_output) + at);
        float g[kPer];
        param(g, p.gate == nullptr ? nullptr : static_cast<const T *>(p.gate) + at, 1.f);
        if (p.post_gamma != nullptr) {
            normalize(u, lane, p.layer, p.epsilon, shared, slot, warps);
            param(w, p.post_gamma, 1.f);
#pragma unroll
            for (int i = 0; i < kPer; ++i) u[i] *= w[i];
            param(w, p.post_beta, 0.f);
#pragma unroll
            for (int i = 0; i < kPer; ++i) u[i] += w[i];
        }
        param(w, p.residual_scale, 1.f);
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = lane.inside(i) ? fmaf(w[i], g[i] * u[i], x[i]) : 0.f;
        lane.store(static_cast<T *>(p.next_residual) + at, x);
    }
    if (p.normed == nullptr) return;
    normalize(x, lane, p.layer, p.epsilon, shared, slot, warps);
    param(w, p.pre_gamma, 1.f);
    param(u, p.pre_beta, 0.f);
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = fmaf(x[i], w[i], u[i]);
    lane.store(static_cast<T *>(p.normed) + at, x);
}

// (dy gamma) -> the gradient behind the normalisation: r (g - mean g - hat mean(g hat)), rms without the first mean.
template <typename L>
__device__ __forceinline__ void normalize_backward(float (&g)[kPer], const float (&hat)[kPer], float r, const L &lane, bool layer,
                                                   float (*shared)[kMaxWarps][2], int &slot, int warps) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        sum[0] += g[i];
        sum[1] = fmaf(g[i], hat[i], sum[1]);
    }
    block_sum(sum, shared, slot, warps);
    const float inv = 1.f / (float)lane.C;
    const float mean = layer ? sum[0] * inv : 0.f, dot = sum[1] * inv;
#pragma unroll
    for (int i = 0; i < kPer; ++i) g[i] = lane.inside(i) ? r * (g[i] - mean - hat[i] * dot) : 0.f;
}

// Rows in turn; a thread sums the gradients of its channels' parameters over its rows and leaves them to the second kernel.
template <typename T, bool VEC>
__global__ void __launch_bounds__(1024)
residual_norm_backward_kernel(const ResidualNormBackwardArgs p, float *partials) {
    __shared__ float shared[2][kMaxWarps][2];
    const Lane<T, VEC> lane{(int)p.f.C, (int)threadIdx.x, (int)blockDim.x};
    const int warps = (int)blockDim.x >> 5;
    int slot = 0;
    wait_for_previous();
    auto param = [&](float (&v)[kPer], const void *q, float absent) {
        if (q != nullptr) lane.load(v, static_cast<const T *>(q));
        else
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] = absent;
    };
    float sum[kParams][kPer] = {};
    const bool block = p.f.block_output != nullptr, post = p.f.post_gamma != nullptr, pre = p.normed_grad != nullptr;
    for (int64_t r = blockIdx.x; r < p.f.rows; r += gridDim.x) {
        const int64_t at = r * p.f.C;
        float x[kPer], h[kPer], g[kPer], u[kPer], w[kPer], dx[kPer];
        lane.load(x, static_cast<const T *>(p.f.residual) + at);
        float rh = 0.f;
        if (block) {
            lane.load(h, static_cast<const T *>(p.f.block_output) + at);
            param(g, p.f.gate == nullptr ? nullptr : static_cast<const T *>(p.f.gate) + at, 1.f);
            if (post) {
                rh = normalize(h, lane, p.f.layer, p.f.epsilon, shared, slot, warps);
                param(w, p.f.post_gamma, 1.f);
                param(u, p.f.post_beta, 0.f);
#pragma unroll
                for (int i = 0; i < kPer; ++i) u[i] = fmaf(h[i], w[i], u[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i) u[i] = h[i];
            }
            param(w, p.f.residual_scale, 1.f);
#pragma unroll
            for (int i = 0; i < kPer; ++i) x[i] = lane.inside(i) ? fmaf(w[i], g[i] * u[i], x[i]) : 0.f;
        }
        if (pre) {
            const float rx = normalize(x, lane, p.f.layer, p.f.epsilon, shared, slot, warps);
            lane.load(dx, static_cast<const T *>(p.normed_grad) + at);
            param(w, p.f.pre_gamma, 1.f);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                sum[3][i] = fmaf(dx[i], x[i], sum[3][i]);
                sum[4][i] += dx[i];
                dx[i] *= w[i];
            }
            normalize_backward(dx, x, rx, lane, p.f.layer, shared, slot, warps);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) dx[i] = 0.f;
        }
        if (p.next_residual_grad != nullptr) {
            lane.load(w, static_cast<const T *>(p.next_residual_grad) + at);
#pragma unroll
            for (int i = 0; i < kPer; ++i) dx[i] += w[i];
        }
        lane.store(static_cast<T *>(p.residual_grad) + at, dx);
        if (!block) continue;
        param(w, p.f.residual_scale, 1.f);
        float dg[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            sum[0][i] = fmaf(dx[i], g[i] * u[i], sum[0][i]);
            dg[i] = dx[i] * w[i] * u[i];
            dx[i] = dx[i] * w[i] * g[i];   // the gradient of u from here on
        }
        if (p.gate_grad != nullptr) lane.store(static_cast<T *>(p.gate_grad) + at, dg);
        if (post) {
            param(w, p.f.post_gamma, 1.f);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                sum[1][i] = fmaf(dx[i], h[i], sum[1][i]);
                sum[2][i] += dx[i];
                dx[i] *= w[i];
            }
            normalize_backward(dx, h, rh, lane, p.f.layer, shared, slot, warps);
        }
        lane.store(static_cast<T *>(p.block_output_grad) + at, dx);
    }
#pragma unroll
    for (int k = 0; k < kParams; ++k) {
        if (p.param_grads[k] == nullptr) continue;
        float *row = partials + ((int64_t)k * gridDim.x + blockIdx.x) * p.f.C;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (lane.inside(i)) row[lane.channel(i)] = sum[k][i];
    }
}

// Sums the CTAs' parts of the parameters' gradients: one warp for 32 channels of one parameter, in the order of the CTAs.
template <typename T>
__global__ void __launch_bounds__(256)
residual_norm_params_kernel(const ResidualNormBackwardArgs p, const float *partials, int parts) {
    __shared__ float shared[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t groups = (p.f.C + 31) / 32;
    const int k = (int)(blockIdx.x / groups);
    const int64_t c = blockIdx.x % groups * 32 + lane;
    wait_for_previous();
    if (p.param_grads[k] == nullptr) return;
    float sum = 0.f;
    if (c < p.f.C)
        for (int i = warp; i < parts; i += 8) sum += partials[((int64_t)k * parts + i) * p.f.C + c];
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.f.C) {
#pragma unroll
        for (int w = 1; w < 8; ++w) sum += shared[w][lane];
        stf(static_cast<T *>(p.param_grads[k]) + c, sum);
    }
}

unsigned threads_for(int64_t C) { return (unsigned)(((C + kPer - 1) / kPer + 31) / 32 * 32); }

int backward_parts(int64_t rows, int num_sms) {
    const int64_t most = (int64_t)num_sms * 2;
    return (int)(rows < most ? rows : most);
}

template <typename T, bool VEC>
int launch_backward(const ResidualNormBackwardArgs &p, float *partials, cudaStream_t stream) {
    const int parts = backward_parts(p.f.rows, p.f.num_sms);
    cudaError_t e = launch_serialized(residual_norm_backward_kernel<T, VEC>, (unsigned)parts, threads_for(p.f.C), 0, stream, p, partials);
    bool any = false;
    for (void *g : p.param_grads) any = any || g != nullptr;
    if (e != cudaSuccess || !any) return (int)e;
    return (int)launch_serialized(residual_norm_params_kernel<T>, (unsigned)(kParams * ((p.f.C + 31) / 32)), 256u, 0, stream, p,
                                  (const float *)partials, parts);
}

}  // namespace

int64_t residual_norm_max_channels() { return 1024 * kPer; }

size_t residual_norm_backward_workspace_bytes(int64_t rows, int64_t C, int num_sms) {
    return (size_t)backward_parts(rows, num_sms) * (size_t)C * kParams * sizeof(float);
}

int launch_residual_norm(const ResidualNormArgs &p, cudaStream_t stream) {
    const bool vec = p.C % kPer == 0;
    const auto kernel = p.bf16 ? (vec ? residual_norm_kernel<__nv_bfloat16, true> : residual_norm_kernel<__nv_bfloat16, false>)
                               : (vec ? residual_norm_kernel<float, true> : residual_norm_kernel<float, false>);
    return (int)launch_serialized(kernel, (unsigned)p.rows, threads_for(p.C), 0, stream, p);
}

int launch_residual_norm_backward(const ResidualNormBackwardArgs &p, void *workspace, cudaStream_t stream) {
    float *partials = static_cast<float *>(workspace);
    const bool vec = p.f.C % kPer == 0;
    if (p.f.bf16) return vec ? launch_backward<__nv_bfloat16, true>(p, partials, stream) : launch_backward<__nv_bfloat16, false>(p, partials, stream);
    return vec ? launch_backward<float, true>(p, partials, stream) : launch_backward<float, false>(p, partials, stream);
}

}  // namespace rwkv7
