// What stands between two blocks of a cell, one row of C channels at a time:
//
//   u = norm_post(h) (or h),   x' = x + s (g u),   z = norm_pre(x')
//   norm(v) = (v - mean v) / sqrt(var v + eps) gamma + beta        (layer; rms: without the mean)
//
// and its gradients.  Both are bound by the bytes of the rows: a CTA keeps a row in registers, eight channels a thread, so that every
// element is read once and every result is rounded once, on its way out.  It walks over rows with the parameters in registers
// and the next row's loads on their way, for a row is a chain of sums over the block (forward four, backward six) and little else.
// Means and variances are taken in turn (the variance from the differences, which a large mean does not spoil), in fp32.
// Arithmetic goes two channels at a time, which halves the instructions that the backward pass would else be bound by.
// 16380 rows of 2048 bf16 channels: forward 60 us (5.6 TB/s of five rows read and written), backward 145 (3.7 TB/s), which the chains of
// six sums a row and some 480 instructions a warp and row bound.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "elements.cuh"
#include "kernels.h"
#include "launch.h"

namespace rwkv7 {
namespace {

constexpr int kPer = 8, kPairs = kPer / 2;   // channels a thread
constexpr int kMaxWarps = 32;
constexpr int kParams = 5;                   // summed over the rows: scale, post gamma, post beta, pre gamma, pre beta

struct Eight {
    float2 v[kPairs];
};
__device__ __forceinline__ Eight all(float x) {
    Eight r;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) r.v[i] = make_float2(x, x);
    return r;
}
__device__ __forceinline__ Eight operator*(const Eight &a, const Eight &b) {
    Eight r;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) r.v[i] = __fmul2_rn(a.v[i], b.v[i]);
    return r;
}
__device__ __forceinline__ Eight operator+(const Eight &a, const Eight &b) {
    Eight r;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) r.v[i] = __fadd2_rn(a.v[i], b.v[i]);
    return r;
}
__device__ __forceinline__ Eight fma(const Eight &a, const Eight &b, const Eight &c) {
    Eight r;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) r.v[i] = __ffma2_rn(a.v[i], b.v[i], c.v[i]);
    return r;
}
__device__ __forceinline__ float total(const Eight &a) {
    const float2 s = __fadd2_rn(__fadd2_rn(a.v[0], a.v[1]), __fadd2_rn(a.v[2], a.v[3]));
    return s.x + s.y;
}
__device__ __forceinline__ float dot(const Eight &a, const Eight &b) {
    float2 s = __fmul2_rn(a.v[0], b.v[0]);
#pragma unroll
    for (int i = 1; i < kPairs; ++i) s = __ffma2_rn(a.v[i], b.v[i], s);
    return s.x + s.y;
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
    uint32_t r[kPairs];
    __device__ Eight get() const {
        Eight e;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) e.v[i] = make_float2(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u));
        return e;
    }
    __device__ void read(const __nv_bfloat16 *from) {
        const uint4 u = *reinterpret_cast<const uint4 *>(from);
        r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
    }
    __device__ void set(int i, __nv_bfloat16 x) {
        const uint32_t u = __bfloat16_as_ushort(x);
        r[i / 2] = i & 1 ? (r[i / 2] & 0xffffu) | u << 16 : (r[i / 2] & 0xffff0000u) | u;
    }
};
template <>
struct Raw<float> {
    float r[kPer];
    __device__ Eight get() const {
        Eight e;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) e.v[i] = make_float2(r[2 * i], r[2 * i + 1]);
        return e;
    }
    __device__ void read(const float *from) {
        const float4 a = *reinterpret_cast<const float4 *>(from), b = *reinterpret_cast<const float4 *>(from + 4);
        r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
        r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
    }
    __device__ void set(int i, float x) { r[i] = x; }
};

// How much is known when a kernel is built: nothing (kOdd: rows that are not whole vectors, read by single elements); rows of whole
// vectors (kVectors); these, no thread without channels, and every part of the operator there (kFull).  What the last leaves out are
// some sixty branches a row.
enum Form { kOdd, kVectors, kFull };

// Eight channels of a row: neighbours, or, of odd rows, every threads-th.
template <typename T, Form FORM>
struct Lane {
    static constexpr bool VEC = FORM != kOdd;
    int C, tid, threads;
    __device__ Lane(int64_t channels) : C((int)channels), tid((int)threadIdx.x), threads((int)blockDim.x) {}
    __device__ int channel(int i) const { return VEC ? tid * kPer + i : tid + i * threads; }
    __device__ bool inside(int i) const { return FORM == kFull || (VEC ? tid * kPer < C : channel(i) < C); }
    // (what lies outside the row counts as zero)
    __device__ Raw<T> load(const void *at, int64_t offset) const {
        const T *row = static_cast<const T *>(at) + offset;
        Raw<T> v{};
        if constexpr (VEC) {
            if (inside(0)) {
                v.read(row + tid * kPer);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (inside(i)) v.set(i, row[channel(i)]);
        }
        return v;
    }
    __device__ void store(void *at, int64_t offset, const Eight &e) const {
        T *row = static_cast<T *>(at) + offset;
        const float v[kPer] = {e.v[0].x, e.v[0].y, e.v[1].x, e.v[1].y, e.v[2].x, e.v[2].y, e.v[3].x, e.v[3].y};
        if constexpr (VEC) {
            if (inside(0)) st8(row + tid * kPer, v);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (inside(i)) stf(row + channel(i), v[i]);
        }
    }
    // a - x; outside the row zero, or, where a thread is in it as a whole or not at all, anything: what it adds to a sum is taken out there
    __device__ Eight minus(const Eight &a, float x) const {
        Eight r;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            r.v[i] = __fadd2_rn(a.v[i], make_float2(-x, -x));
            if constexpr (!VEC) r.v[i] = make_float2(inside(2 * i) ? r.v[i].x : 0.f, inside(2 * i + 1) ? r.v[i].y : 0.f);
        }
        return r;
    }
    __device__ float counted(float partial_sum) const { return !VEC || inside(0) ? partial_sum : 0.f; }
};

// A parameter's eight channels: kept in registers where there is room for it, else read from L1 for every row.
template <typename T, Form FORM, bool KEPT>
struct Param {
    const Lane<T, FORM> &lane;
    const void *at;
    Raw<T> kept;
    __device__ Param(const Lane<T, FORM> &l, const void *p) : lane(l), at(p), kept{} {
        if (KEPT && at != nullptr) kept = lane.load(at, 0);
    }
    __device__ Eight get() const {
        if constexpr (KEPT) return kept.get();
        else return at == nullptr ? all(0.f) : lane.load(at, 0).get();
    }
};

// Sums over a block of at most MOST threads.  Two sets of slots in turn, so that one barrier a sum is enough.
template <int MOST>
struct Block {
    float (*shared)[2][kMaxWarps];   // [set][value][warp], zero at first
    int set = 0, warps = (int)blockDim.x >> 5;
    __device__ __forceinline__ float of_warps(int k) const {
        const float4 *part = reinterpret_cast<const float4 *>(shared[set][k]);
        float4 s = part[0];
#pragma unroll
        for (int w = 1; w < MOST / 128; ++w) {
            const float4 x = part[w];
            s = make_float4(s.x + x.x, s.y + x.y, s.z + x.z, s.w + x.w);
        }
        return (s.x + s.y) + (s.z + s.w);
    }
    __device__ __forceinline__ float sum(float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (warps == 1) return x;
        if ((threadIdx.x & 31) == 0) shared[set][0][threadIdx.x >> 5] = x;
        __syncthreads();
        x = of_warps(0);
        set ^= 1;
        return x;
    }
    // Two at once: the halves of the warp take one each after the first step.
    __device__ __forceinline__ void sum2(float (&v)[2]) {
        const int lane = threadIdx.x & 31;
        const bool low = lane < 16;
        float x = (low ? v[0] : v[1]) + __shfl_xor_sync(0xffffffffu, low ? v[1] : v[0], 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (warps == 1) {
            v[0] = __shfl_sync(0xffffffffu, x, 0);
            v[1] = __shfl_sync(0xffffffffu, x, 16);
            return;
        }
        if ((lane & 15) == 0) shared[set][lane >> 4][threadIdx.x >> 5] = x;
        __syncthreads();
        v[0] = of_warps(0);
        v[1] = of_warps(1);
        set ^= 1;
    }
};
__device__ __forceinline__ void clear(float (*shared)[2][kMaxWarps]) {
    for (int i = threadIdx.x; i < 2 * 2 * kMaxWarps; i += blockDim.x) (&shared[0][0][0])[i] = 0.f;
    __syncthreads();
}

// v -> (v - mean) / sqrt(var + eps); returns the reciprocal root.
template <typename L, typename B>
__device__ __forceinline__ float normalize(Eight &v, const L &lane, bool layer, float eps, B &block) {
    const float inv = 1.f / (float)lane.C;
    if (layer) v = lane.minus(v, block.sum(lane.counted(total(v))) * inv);
    const float r = rsqrtf(fmaf(block.sum(lane.counted(dot(v, v))), inv, eps));
    v = v * all(r);
    return r;
}

template <typename T, Form FORM, int MOST, int RESIDENT>
__global__ void __launch_bounds__(MOST, RESIDENT)
residual_norm_kernel(const ResidualNormArgs p) {
    __shared__ __align__(16) float shared[2][2][kMaxWarps];
    const Lane<T, FORM> lane(p.C);
    clear(shared);
    Block<MOST> block{shared};
    wait_for_previous();
    let_next_in();
    constexpr bool kAll = FORM == kFull;
    const bool has_block = kAll || p.block_output != nullptr, has_gate = kAll || p.gate != nullptr, post = kAll || p.post_gamma != nullptr,
               has_scale = kAll || p.residual_scale != nullptr, pre = kAll || p.normed != nullptr;
    Raw<T> x_in, h_in{}, g_in{};
    auto load = [&](int64_t row) {
        x_in = lane.load(p.residual, row * p.C);
        if (has_block) h_in = lane.load(p.block_output, row * p.C);
        if (has_gate) g_in = lane.load(p.gate, row * p.C);
    };
    load(blockIdx.x);
    const Param<T, FORM, sizeof(T) == 2> scale(lane, p.residual_scale), post_gamma(lane, p.post_gamma), post_beta(lane, p.post_beta), pre_gamma(lane, p.pre_gamma),
        pre_beta(lane, p.pre_beta);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t at = row * p.C;
        Eight x = x_in.get(), u = h_in.get(), g = g_in.get();
        if (row + gridDim.x < p.rows) load(row + gridDim.x);
        if (has_block) {
            if (post) {
                normalize(u, lane, p.layer, p.epsilon, block);
                u = fma(u, post_gamma.get(), post_beta.get());
            }
            if (has_gate) u = g * u;
            x = has_scale ? fma(scale.get(), u, x) : x + u;
            lane.store(p.next_residual, at, x);
        }
        if (!pre) continue;
        normalize(x, lane, p.layer, p.epsilon, block);
        lane.store(p.normed, at, fma(x, pre_gamma.get(), pre_beta.get()));
    }
}

// (dy gamma) -> the gradient behind the normalisation: r (g - mean g - hat mean(g hat)), rms without the first mean.
template <typename L, typename B>
__device__ __forceinline__ Eight normalize_backward(const Eight &g, const Eight &hat, float r, const L &lane, bool layer, B &block) {
    float sum[2] = {lane.counted(total(g)), lane.counted(dot(g, hat))};
    block.sum2(sum);
    const float inv = 1.f / (float)lane.C;
    return fma(hat, all(-r * sum[1] * inv), lane.minus(g, layer ? sum[0] * inv : 0.f) * all(r));
}

// A thread sums the gradients of its channels' parameters over its rows, in registers, and leaves them to the second kernel.
template <typename T, Form FORM, int MOST, int RESIDENT>
__global__ void __launch_bounds__(MOST, RESIDENT)
residual_norm_backward_kernel(const ResidualNormBackwardArgs p, float *partials) {
    __shared__ __align__(16) float shared[2][2][kMaxWarps];
    const Lane<T, FORM> lane(p.f.C);
    clear(shared);
    Block<MOST> block{shared};
    wait_for_previous();
    let_next_in();
    constexpr bool kAll = FORM == kFull;
    const bool has_block = kAll || p.f.block_output != nullptr, has_gate = kAll || p.f.gate != nullptr, post = kAll || p.f.post_gamma != nullptr,
               has_scale = kAll || p.f.residual_scale != nullptr, pre = kAll || p.normed_grad != nullptr,
               has_grad = kAll || p.next_residual_grad != nullptr;
    Raw<T> x_in, h_in{}, g_in{}, dz_in{}, dx_in{};
    auto load = [&](int64_t row) {
        x_in = lane.load(p.f.residual, row * p.f.C);
        if (has_block) h_in = lane.load(p.f.block_output, row * p.f.C);
        if (has_gate) g_in = lane.load(p.f.gate, row * p.f.C);
        if (pre) dz_in = lane.load(p.normed_grad, row * p.f.C);
        if (has_grad) dx_in = lane.load(p.next_residual_grad, row * p.f.C);
    };
    constexpr bool kAhead = sizeof(T) == 2;   // (five fp32 rows on their way would not leave room for the one at hand)
    if (kAhead) load(blockIdx.x);
    const Param<T, FORM, false> scale_in(lane, p.f.residual_scale), post_gamma(lane, p.f.post_gamma), post_beta(lane, p.f.post_beta),
        pre_gamma(lane, p.f.pre_gamma);
    auto scale = [&] { return has_scale ? scale_in.get() : all(1.f); };
    Eight sum[kParams];
#pragma unroll
    for (int k = 0; k < kParams; ++k) sum[k] = all(0.f);
    for (int64_t row = blockIdx.x; row < p.f.rows; row += gridDim.x) {
        const int64_t at = row * p.f.C;
        if (!kAhead) load(row);
        Eight x = x_in.get(), h = h_in.get();
        const Eight g = has_gate ? g_in.get() : all(1.f);
        Eight dz = dz_in.get(), dx = dx_in.get();   // (zero where there is none)
        if (kAhead && row + gridDim.x < p.f.rows) load(row + gridDim.x);
        Eight u = h;
        float rh = 0.f;
        if (has_block) {
            if (post) {
                rh = normalize(h, lane, p.f.layer, p.f.epsilon, block);
                u = fma(h, post_gamma.get(), post_beta.get());
            }
            x = fma(scale(), g * u, x);
        }
        if (pre) {
            const float rx = normalize(x, lane, p.f.layer, p.f.epsilon, block);
            sum[3] = fma(dz, x, sum[3]);
            sum[4] = sum[4] + dz;
            dx = dx + normalize_backward(dz * pre_gamma.get(), x, rx, lane, p.f.layer, block);
        }
        lane.store(p.residual_grad, at, dx);
        if (!has_block) continue;
        sum[0] = fma(dx, g * u, sum[0]);
        dx = dx * scale();
        if (has_gate) lane.store(p.gate_grad, at, dx * u);
        dx = dx * g;   // the gradient of u
        if (post) {
            sum[1] = fma(dx, h, sum[1]);
            sum[2] = sum[2] + dx;
            dx = normalize_backward(dx * post_gamma.get(), h, rh, lane, p.f.layer, block);
        }
        lane.store(p.block_output_grad, at, dx);
    }
#pragma unroll
    for (int k = 0; k < kParams; ++k) {
        if (p.param_grads[k] == nullptr) continue;
        float *row = partials + ((int64_t)k * gridDim.x + blockIdx.x) * p.f.C;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            if (lane.inside(2 * i)) row[lane.channel(2 * i)] = sum[k].v[i].x;
            if (lane.inside(2 * i + 1)) row[lane.channel(2 * i + 1)] = sum[k].v[i].y;
        }
    }
}

// Sums the CTAs' parts of the parameters' gradients, 32 channels of one parameter a CTA: eight warps in turn, then in their order.
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
    if (c < p.f.C) {
        const float *at = partials + (int64_t)k * parts * p.f.C + c;
        constexpr int kAhead = 8;
        for (int i = warp; i < parts; i += 8 * kAhead) {
            float x[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) x[j] = i + 8 * j < parts ? at[(int64_t)(i + 8 * j) * p.f.C] : 0.f;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) sum += x[j];
        }
    }
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.f.C) {
#pragma unroll
        for (int w = 1; w < 8; ++w) sum += shared[w][lane];
        stf(static_cast<T *>(p.param_grads[k]) + c, sum);
    }
}

unsigned threads_for(int64_t C) { return (unsigned)(((C + kPer - 1) / kPer + 31) / 32 * 32); }

// CTAs of the backward pass: what its 128 registers let an SM hold of blocks of that size, 512 threads.  2048 channels (two CTAs) 145 us for 67 MB a tensor,
// 2560 (one of ten warps) 214, 4096 (one of sixteen) 177, 8192 (64 registers, which spill) 398.
int backward_parts(int64_t rows, int64_t C, int num_sms) {
    const int64_t threads = threads_for(C), resident = std::max<int64_t>(1, 512 / threads);
    return (int)std::min<int64_t>(rows, (int64_t)num_sms * resident);
}

template <typename T, Form FORM>
int launch_forward(const ResidualNormArgs &p, cudaStream_t stream) {
    const unsigned threads = threads_for(p.C);
    // (768 threads of 80 registers an SM: 2048 channels 60 us, 2560 66, 4096, where one CTA is left, 79)
    const unsigned ctas = (unsigned)std::min<int64_t>(p.rows, (int64_t)p.num_sms * std::max(1u, 768 / threads));
    const auto kernel = threads <= 256 ? residual_norm_kernel<T, FORM, 256, 3>
                        : threads <= 512 ? residual_norm_kernel<T, FORM, 512, 1> : residual_norm_kernel<T, FORM, 1024, 1>;
    return (int)launch_serialized(kernel, ctas, threads, 0, stream, p);
}

template <typename T, Form FORM>
int launch_backward(const ResidualNormBackwardArgs &p, float *partials, cudaStream_t stream) {
    const int parts = backward_parts(p.f.rows, p.f.C, p.f.num_sms);
    const unsigned threads = threads_for(p.f.C);
    const auto kernel = threads <= 256 ? residual_norm_backward_kernel<T, FORM, 256, 2>
                        : threads <= 512 ? residual_norm_backward_kernel<T, FORM, 512, 1> : residual_norm_backward_kernel<T, FORM, 1024, 1>;
    const cudaError_t e = launch_serialized(kernel, (unsigned)parts, threads, 0, stream, p, partials);
    bool any = false;
    for (void *g : p.param_grads) any = any || g != nullptr;
    if (e != cudaSuccess || !any) return (int)e;
    return (int)launch_serialized(residual_norm_params_kernel<T>, (unsigned)(kParams * ((p.f.C + 31) / 32)), 256u, 0, stream, p,
                                  (const float *)partials, parts);
}

}  // namespace

int64_t residual_norm_max_channels() { return 1024 * kPer; }

size_t residual_norm_backward_workspace_bytes(int64_t rows, int64_t C, int num_sms) {
    return (size_t)backward_parts(rows, C, num_sms) * (size_t)C * kParams * sizeof(float);
}

int launch_residual_norm(const ResidualNormArgs &p, cudaStream_t stream) {
    const bool full = p.C % (32 * kPer) == 0 && p.block_output != nullptr && p.gate != nullptr && p.residual_scale != nullptr && p.post_gamma != nullptr && p.normed != nullptr;
    if (p.C % kPer != 0) return p.bf16 ? launch_forward<__nv_bfloat16, kOdd>(p, stream) : launch_forward<float, kOdd>(p, stream);
    if (!full) return p.bf16 ? launch_forward<__nv_bfloat16, kVectors>(p, stream) : launch_forward<float, kVectors>(p, stream);
    return p.bf16 ? launch_forward<__nv_bfloat16, kFull>(p, stream) : launch_forward<float, kFull>(p, stream);
}

int launch_residual_norm_backward(const ResidualNormBackwardArgs &p, void *workspace, cudaStream_t stream) {
    float *partials = static_cast<float *>(workspace);
    const ResidualNormArgs &f = p.f;
    const bool full = f.C % (32 * kPer) == 0 && f.block_output != nullptr && f.gate != nullptr && f.residual_scale != nullptr && f.post_gamma != nullptr &&
                      p.normed_grad != nullptr && p.next_residual_grad != nullptr;
    if (f.C % kPer != 0) return f.bf16 ? launch_backward<__nv_bfloat16, kOdd>(p, partials, stream) : launch_backward<float, kOdd>(p, partials, stream);
    if (!full) return f.bf16 ? launch_backward<__nv_bfloat16, kVectors>(p, partials, stream) : launch_backward<float, kVectors>(p, partials, stream);
    return f.bf16 ? launch_backward<__nv_bfloat16, kFull>(p, partials, stream) : launch_backward<float, kFull>(p, partials, stream);
}

}  // namespace rwkv7
