// Linear attention with one decay per head, on the fp32 units: any type and head size, a few tokens or many.
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
// Tokens go in blocks of sixteen, as in linear_attention_chunks.cu:
//   y_i = d^(i+1) S a_i + sum_{j <= i} d^(i-j) (a_i . b_j) c_j,   S' = d^n S + sum_j d^(n-1-j) c_j b_j^T      (reversed: mirrored)
// so that S is scaled once a block and a long memory is not the sum of a rounding for every token.  It takes two multiply-adds per
// element of S and token (three go token by token), and nothing of a token behind another ever meets it, not even times zero.
//
// S is in registers: a thread holds four rows x 16 columns, the columns in groups of four that alternate between the threads of a
// row, so that these read neighbouring pieces.  A token then costs 64 multiply-adds for nine loads from shared memory; one row a
// thread needed sixteen for 32.  For one token it is bound by the bytes of S (512 sequences of 40 heads 112 us, 6.1 TB/s, into a state
// that is there, 119 with its allocation); for many by the chain of a
// block, 5.3 us at N = 64 on two warps, which several CTAs an SM overlap (2 x 1000 tokens of 12 heads in fp32 43 us, three launches of
// segments of two blocks).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "elements.cuh"
#include "kernels.h"
#include "launch.h"
#include "linear_attention_decay.cuh"
#include "linear_attention_plan.h"

namespace rwkv7 {
namespace {

using linear_attention_plan::kBlock;

// How an N x N state lies in a CTA.
template <int N>
struct Shape {
    static constexpr int kRows = N >= 64 ? 4 : 2, kCols = 16;      // of a thread
    static constexpr int kShare = N / kCols;                       // threads of a row
    static constexpr int kThreads = N / kRows * kShare;
    static constexpr int kPitch = N + 4;                           // floats of a staged row
    // CTAs an SM is to hold, which spills a few of 160 registers: one token of 512 sequences of 40 heads 118 -> 112 us, 4 x 1000 fp32 tokens of 32
    // heads 177 -> 157, N = 128 of 16 heads 397 -> 308 (313 with what came since).  The pass that only adds to states spills more than it gains at N = 64.
    static constexpr int resident(bool adds) { return N == 128 ? 2 : N == 64 ? (adds ? 1 : 8) : 16; }
};

struct ScanArgs {
    LinearAttentionPass p;
    float *parts;             // null with one segment
    int64_t segments, tokens; // per chain, per segment
};

// Sums over the `SHARE` threads of a row, one token each: v[t][r] of all -> v[0][r] of token `part`.
template <int SHARE, int ROWS>
__device__ __forceinline__ void scatter_sums(float (&v)[SHARE][ROWS], int part) {
#pragma unroll
    for (int o = SHARE / 2; o > 0; o /= 2) {
        const bool upper = (part & o) != 0;
#pragma unroll
        for (int t = 0; t < o; ++t)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float sent = upper ? v[t][r] : v[t + o][r];
                v[t][r] = (upper ? v[t + o][r] : v[t][r]) + __shfl_xor_sync(0xffffffffu, sent, o);
            }
    }
}

// ADDS: only what a segment adds to the state.
template <typename T, int N, bool REVERSED, bool ADDS>
__global__ void __launch_bounds__(Shape<N>::kThreads, Shape<N>::resident(ADDS))
scan_kernel(const ScanArgs args) {
    using Sh = Shape<N>;
    constexpr int R = Sh::kRows, SHARE = Sh::kShare, THREADS = Sh::kThreads, PITCH = Sh::kPitch;
    __shared__ __align__(16) float sa[ADDS ? 1 : kBlock * PITCH], sb[kBlock * PITCH], sc[kBlock * PITCH], sp[ADDS ? 1 : kBlock * kBlock];
    __shared__ float dec[kBlock + 1];
    __shared__ SteadyPower whole;   // d^16, by which S may be scaled again and again
    __shared__ float scale;         // of the block at hand
    const LinearAttentionPass &p = args.p;
    const int64_t chains = p.B * p.H, chain = blockIdx.x % chains, order = blockIdx.x / chains;
    const int64_t bi = chain / p.H, h = chain % p.H;
    const int tid = threadIdx.x, row0 = tid / SHARE * R, part = tid % SHARE;
    auto column = [&](int m) { return 4 * (m * SHARE + part); };

    wait_for_previous();
    // The state's loads first; everything else is on its way behind them.
    float2 S[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < 8; ++m) S[r][m] = make_float2(0.f, 0.f);
    auto read = [&](const float *src, bool transposed) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int row = row0 + r, col = column(m);
                const float4 x = transposed ? make_float4(src[col * N + row], src[(col + 1) * N + row], src[(col + 2) * N + row], src[(col + 3) * N + row])
                                            : __ldcs(reinterpret_cast<const float4 *>(src + row * N + col));
                S[r][2 * m] = make_float2(x.x, x.y);
                S[r][2 * m + 1] = make_float2(x.z, x.w);
            }
    };
    auto write = [&](float *dst) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < 4; ++m)
                __stcs(reinterpret_cast<float4 *>(dst + (row0 + r) * N + column(m)), make_float4(S[r][2 * m].x, S[r][2 * m].y, S[r][2 * m + 1].x, S[r][2 * m + 1].y));
    };
    float *parts = args.parts + chain * args.segments * (N * N);
    const float *s_in = p.s_in == nullptr ? nullptr : p.s_in + chain * (N * N);
    if (ADDS) {
        if (order == 0) {   // the state in front of everything: s_in may be overwritten before the last segment starts
            if (s_in != nullptr) read(s_in, p.s_in_transposed);
            write(parts);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int m = 0; m < 8; ++m) S[r][m] = make_float2(0.f, 0.f);
        }
    } else if (args.segments > 1) {
        read(parts + order * (N * N), false);
    } else if (s_in != nullptr) {
        read(s_in, p.s_in_transposed);
    }
    const int64_t len = p.lens == nullptr ? p.T : min(max((int64_t)p.lens[bi], (int64_t)0), p.T);
    const int64_t seg = REVERSED ? args.segments - 1 - order : order;
    const int64_t begin = min(p.T, seg * args.tokens), end = min(p.T, begin + args.tokens), stop = max(begin, min(len, end));   // live: [begin, stop)
    // d^k in 64 bits, rounded once; d^0 is 1 for every d.
    const double lambda = (double)p.log_decay[h];
    const int full = stop - begin < kBlock ? (int)(stop - begin) : kBlock;
    static_assert(THREADS > kBlock + 1);
    if (tid <= full || tid == kBlock + 1) {
        const double power = exp(lambda * min(tid, kBlock));
        if (tid <= full) dec[tid] = tid == 0 ? 1.f : (float)power;
        else whole = SteadyPower(power);
    }
    const int64_t step = p.H * N, base = (bi * p.T * p.H + h) * N;   // of token 0
    const T *a = static_cast<const T *>(p.a) + base, *b = static_cast<const T *>(p.b) + base, *c = static_cast<const T *>(p.c) + base;
    T *y = static_cast<T *>(p.y) + base;

    for (int64_t done = begin; done < stop; done += kBlock) {
        // blocks from the segment's first token on, reversed from the last block back
        const int64_t first = REVERSED ? begin + (stop - 1 - done) / kBlock * kBlock : done;
        const int n = (int)min((int64_t)kBlock, stop - first);
        __syncthreads();
        if (tid == 0) scale = n == kBlock ? whole.factor((uint32_t)((done - begin) / kBlock)) : dec[n];
        for (int i = tid; i < n * (N / 4); i += THREADS) {
            const int t = i / (N / 4), j = i % (N / 4) * 4;
            const int64_t at = (first + t) * step + j;
            if (!ADDS) st4(sa + t * PITCH + j, a + at);
            st4(sb + t * PITCH + j, b + at);
            st4(sc + t * PITCH + j, c + at);
        }
        __syncthreads();
        if (!ADDS) {
            // d^gap (a_i . b_j): four j a thread
            for (int e = tid; e < kBlock * kBlock / 4; e += THREADS) {
                const int i = e / (kBlock / 4), j0 = e % (kBlock / 4) * 4;
                if (i >= n || j0 >= n || (REVERSED ? j0 + 3 < i : j0 > i)) continue;
                float2 s[4] = {};
#pragma unroll 4
                for (int k = 0; k < N; k += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(sa + i * PITCH + k);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 z = *reinterpret_cast<const float4 *>(sb + (j0 + q) * PITCH + k);   // (behind n: not used)
                        s[q] = __ffma2_rn(make_float2(x.x, x.y), make_float2(z.x, z.y), s[q]);
                        s[q] = __ffma2_rn(make_float2(x.z, x.w), make_float2(z.z, z.w), s[q]);
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int gap = REVERSED ? j0 + q - i : i - j0 - q;
                    if (gap >= 0 && j0 + q < n) sp[i * kBlock + j0 + q] = (s[q].x + s[q].y) * dec[gap];
                }
            }
            __syncthreads();
            for (int i0 = 0; i0 < n; i0 += SHARE) {
                float v[SHARE][R];
#pragma unroll
                for (int t = 0; t < SHARE; ++t) {
                    float2 s[R] = {};
                    if (i0 + t < n) {
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const float4 x = *reinterpret_cast<const float4 *>(sa + (i0 + t) * PITCH + column(m));
#pragma unroll
                            for (int r = 0; r < R; ++r) {
                                s[r] = __ffma2_rn(S[r][2 * m], make_float2(x.x, x.y), s[r]);
                                s[r] = __ffma2_rn(S[r][2 * m + 1], make_float2(x.z, x.w), s[r]);
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) v[t][r] = s[r].x + s[r].y;
                }
                scatter_sums<SHARE, R>(v, part);
                const int i = i0 + part;
                if (i < n) {
                    const float f = dec[REVERSED ? n - 1 - i : i + 1];
                    float out[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) out[r] = v[0][r] * f;
                    const int j_end = REVERSED ? n : i + 1;
#pragma unroll 4
                    for (int j = REVERSED ? i : 0; j < j_end; ++j) {
                        const float w = sp[i * kBlock + j];
                        float cj[R];
                        ldn(cj, sc + j * PITCH + row0);
#pragma unroll
                        for (int r = 0; r < R; ++r) out[r] = fmaf(w, cj[r], out[r]);
                    }
                    stn<R>(y + (first + i) * step + row0, out);
                }
            }
        }
        // S' (the last block's is not needed where nobody takes it)
        const float dn = scale;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < 8; ++m) S[r][m] = __fmul2_rn(S[r][m], make_float2(dn, dn));
#pragma unroll 2
        for (int j = 0; j < n; ++j) {
            const float w = dec[REVERSED ? j + 1 : n - 1 - j];
            float cw[R];
            ldn(cw, sc + j * PITCH + row0);
#pragma unroll
            for (int r = 0; r < R; ++r) cw[r] *= w;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float4 x = *reinterpret_cast<const float4 *>(sb + j * PITCH + column(m));
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    S[r][2 * m] = __ffma2_rn(make_float2(cw[r], cw[r]), make_float2(x.x, x.y), S[r][2 * m]);
                    S[r][2 * m + 1] = __ffma2_rn(make_float2(cw[r], cw[r]), make_float2(x.z, x.w), S[r][2 * m + 1]);
                }
            }
        }
    }
    if constexpr (ADDS) {
        write(parts + (order + 1) * (N * N));
    } else {
        for (int64_t i = (stop - begin) * (N / 4) + tid; i < (end - begin) * (N / 4); i += THREADS) {   // behind the sequence
            const float zero[4] = {};
            stn<4>(y + (begin + i / (N / 4)) * step + i % (N / 4) * 4, zero);
        }
        if (order == args.segments - 1 && p.s_out != nullptr) write(p.s_out + chain * (N * N));
    }
}

// Four elements a thread; the parts of several segments are on their way at once, and the first of them while the powers are taken.
__global__ void __launch_bounds__(256) segment_states_kernel(const ScanArgs args) {
    wait_for_previous();
    const LinearAttentionPass &p = args.p;
    const int64_t quads = p.N * p.N / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x, chain = i / quads;
    if (chain >= p.B * p.H) return;
    float4 *at = reinterpret_cast<float4 *>(args.parts) + chain * args.segments * quads + i % quads;
    constexpr int kAhead = 8;
    float4 s = *at, part[kAhead];
    auto load = [&](int64_t o) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (o + j < args.segments) part[j] = at[(o + j) * quads];
    };
    load(1);
    const int64_t len = p.lens == nullptr ? p.T : min(max((int64_t)p.lens[chain / p.H], (int64_t)0), p.T);
    const double lambda = (double)p.log_decay[chain % p.H];
    // d^(tokens of a segment): of a whole one, and of the one that the sequence ends in
    const SteadyPower whole(exp(lambda * (double)args.tokens));
    const float last = len % args.tokens == 0 ? 1.f : (float)exp(lambda * (double)(len % args.tokens));
    for (int64_t o = 1; o < args.segments; o += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (o + j >= args.segments) break;
            // s_o = d^(tokens of the segment before) s_(o-1) + what that adds
            const int64_t from = (p.reversed ? args.segments - (o + j) : o + j - 1) * args.tokens;
            const float f = len >= from + args.tokens ? whole.factor((uint32_t)(o + j)) : len > from ? last : 1.f;
            s = make_float4(fmaf(s.x, f, part[j].x), fmaf(s.y, f, part[j].y), fmaf(s.z, f, part[j].z), fmaf(s.w, f, part[j].w));
            at[(o + j) * quads] = s;
        }
        load(o + kAhead);
    }
}

// CTAs of a pass on the device: segments fill them.  fp32: 4 x 1000 tokens of 32 heads at N = 64 184 us with 6 an SM, 170 with 7, 157 with 8; 84, 72 and 67
// at N = 32 with 8, 12 and 16; 64 chains of 1000 at N = 128 514, 399 and 414 with 1, 2 and 3.
int64_t places(const LinearAttentionPass &p) { return (int64_t)p.num_sms * (p.N == 128 ? 2 : p.N == 64 ? 8 : 16); }

template <typename T, int N>
int launch_scan(const ScanArgs &args, cudaStream_t stream) {
    const LinearAttentionPass &p = args.p;
    const int64_t chains = p.B * p.H;
    const unsigned threads = (unsigned)Shape<N>::kThreads;
    if (args.segments > 1) {
        const cudaError_t e = launch_serialized(p.reversed ? scan_kernel<T, N, true, true> : scan_kernel<T, N, false, true>,
                                                (unsigned)(chains * (args.segments - 1)), threads, 0, stream, args);
        if (e != cudaSuccess) return (int)e;
        if (int f = launch_segment_states(p, args.parts, args.segments, args.tokens, stream)) return f;
    }
    return (int)launch_serialized(p.reversed ? scan_kernel<T, N, true, false> : scan_kernel<T, N, false, false>, (unsigned)(chains * args.segments),
                                  threads, 0, stream, args);
}

template <typename T>
int launch_scan(const ScanArgs &args, cudaStream_t stream) {
    switch (args.p.N) {
        case 32: return launch_scan<T, 32>(args, stream);
        case 64: return launch_scan<T, 64>(args, stream);
        default: return launch_scan<T, 128>(args, stream);
    }
}

}  // namespace

bool linear_attention_supported(int64_t N) { return N == 32 || N == 64 || N == 128; }

int launch_segment_states(const LinearAttentionPass &p, float *parts, int64_t segments, int64_t tokens, cudaStream_t stream) {
    return (int)launch_serialized(segment_states_kernel, (unsigned)((p.B * p.H * (p.N * p.N / 4) + 255) / 256), 256u, 0, stream,
                                  ScanArgs{p, parts, segments, tokens});
}

size_t linear_attention_workspace_bytes(const LinearAttentionPass &p) {
    using namespace linear_attention_plan;
    if (linear_attention_chunks_supported(p)) return linear_attention_chunks_workspace_bytes(p);
    const int64_t chains = p.B * p.H;
    return state_bytes(chains, cut(chains, (p.T + kBlock - 1) / kBlock, places(p), kBlocksOfLaunches, INT64_MAX).segments, p.N);
}

int launch_linear_attention(const LinearAttentionPass &p, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    using namespace linear_attention_plan;
    if (linear_attention_chunks_supported(p)) return launch_linear_attention_chunks(p, workspace, workspace_bytes, stream);
    const int64_t chains = p.B * p.H;
    const Cut c = cut(chains, (p.T + kBlock - 1) / kBlock, places(p), kBlocksOfLaunches, workspace == nullptr ? 1 : segments_in(workspace_bytes, chains, p.N));
    const ScanArgs args{p, c.segments > 1 ? static_cast<float *>(workspace) : nullptr, c.segments, c.chunks * kBlock};
    return p.bf16 ? launch_scan<__nv_bfloat16>(args, stream) : launch_scan<float>(args, stream);
}

}  // namespace rwkv7
