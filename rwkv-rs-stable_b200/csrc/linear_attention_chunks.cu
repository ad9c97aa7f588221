// Linear attention with one decay per head on the tensor cores: bf16 tensors, head size 64, chunks of 128 tokens.
//
// In the notation of linear_attention.cu, for a chunk of n tokens with the state S in front of it, forwards:
//
//   y_i = sum_{j <= i} d^(i-j) (a_i . b_j) c_j + d^(i+1) S a_i        S' = d^n S + sum_j d^(n-1-j) c_j b_j^T
//
// and reversed (G, the gradient behind the chunk's last token):
//
//   y_i = sum_{j >= i} d^(j-i) (a_i . b_j) c_j + d^(n-1-i) G a_i      G' = d^n G + sum_j d^(j+1) c_j b_j^T
//
// Four products of a chunk: P = A B^T [128 x 128], Y2 = A S [128 x 64], the sum for S' = B^T (w C) [64 x 64] and, once P carries
// its decays and its mask, Y1 = P C [128 x 64].  A walk over the chunks is bound by HBM (64 KB a chunk, 1.5 us of an SM's share) if
// two CTAs an SM take at most 3 us for one: so the chunk's chain of waits is kept short.  P stays in TMEM: read as fp32, written
// back as the bf16 operand of its own product.  Two threads share a row, which halves what is done between two products; c has two
// buffers, for which the last part of w C takes the place of a as soon as a has been read.
//
// Precision: y is rounded to bf16, and so is P (once); S stays in fp32 registers and enters Y2 as hi + lo (16 bits and a
// sign), because its errors would add up; the sum for S' takes w C as hi + mid + lo, all 24 bits, because S is an fp32 output.
//
// Warps 0-7 own half a row (TMEM lane) a thread, warp 8 issues the products, warp 9 the loads.  The state's rows are those of b, on
// lanes 0-63 forwards and 64-127 reversed: of the two 64-row blocks of that product's A operand the other one is whatever
// tile lies beside b, and its lanes are not read.  (So the warps with the smaller share of the triangle P update S.)
//
// Entries of c that are not finite would reach tokens on the other side of the mask (0 x inf): a chunk that has some takes
// them as zero and sets what they do reach, the column's later tokens and the state's column, to NaN.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

#include "elements.cuh"
#include "kernels.h"
#include "launch.h"
#include "linear_attention_plan.h"
#include "sm100_umma.cuh"

namespace rwkv7 {
namespace {

using namespace sm100;

constexpr int kN = 64, kL = linear_attention_plan::kChunk;
constexpr int kRowThreads = 256, kThreads = kRowThreads + 64;
constexpr uint32_t kTile = kL * 128;           // [128 tokens][64] bf16, 128-byte swizzle
// Shared memory: a (then the last part of w C), b, c twice (in this order, see above), two parts of w C, S in two, tables, barriers.
constexpr uint32_t kA = 0, kB = kTile, kC = 2 * kTile, kW = 4 * kTile, kS = 6 * kTile, kSPart = kN * 128;
constexpr uint32_t kCol = kS + 2 * kSPart;     // d^31 .. d^0 forwards, d^0 .. d^31 reversed
constexpr uint32_t kDec = kCol + 128;          // d^0 .. d^128
constexpr uint32_t kBars = kDec + 520;
constexpr uint32_t kBad = kBars + 120;         // per column the first (reversed: last) token that is not finite
constexpr uint32_t kSmem = kBad + 256;
static_assert(kSmem <= 115712, "two CTAs on an SM");
// TMEM columns: P as fp32 at 0; as bf16 its first half on columns 0-31, its second on 96-127, where the threads that read
// those columns put it; Y1 between them; Y2 and the state's sum.
constexpr uint32_t kP = 0, kY1 = 32, kY2 = 128, kKV = 192;
__host__ __device__ constexpr uint32_t p_operand(int kstep) { return kP + (kstep < 4 ? 0 : 64) + kstep * 8; }

struct Maps {
    CUtensorMap a, b, c, y;
};

struct ChunkArgs {
    __nv_bfloat16 *y;
    const float *log_decay;
    const int *lens;
    const float *s_in;     // or null
    float *s_out;          // or null
    float *parts;          // [chain][segment][c][b]: before the first segment, then what each adds; null with one segment
    int T, H, chains;
    int segments, chunks;  // per chain, per segment
    bool s_in_transposed;
    int *status;
};

enum Bar { kFullA, kFullB, kFullC, kFullC1, kPDone, kADone, kYDone, kKvDone, kSReady, kPReady, kWReady, kYRead, kYStored, kEnd, kBarCount };
static_assert(kBarCount * 8 + 8 <= 120, "room for the barriers");

// 16-byte piece `q` of a 128-byte row.
__device__ __forceinline__ uint32_t piece(int row, int q) { return (uint32_t)row * 128u + (uint32_t)((q ^ (row & 7)) << 4); }
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float2 unpack2(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(float2 v) { return pack_bf2(v.x, v.y); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return __fadd2_rn(a, make_float2(-b.x, -b.y)); }
__device__ __forceinline__ void rows_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// ADDS: only what a segment adds to the state.
template <bool REVERSED, bool ADDS>
__global__ void __launch_bounds__(kThreads, 2)
chunk_kernel(const __grid_constant__ Maps maps, const ChunkArgs p) {
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (smem_u32(smem) & 1023u) {
        if (tid == 0) atomicExch(p.status, (int)kDevInternal);
        return;
    }
    const uint32_t base = smem_u32(smem);
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + kBars);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + kBars + kBarCount * 8);
    float *dec = reinterpret_cast<float *>(smem + kDec), *col = reinterpret_cast<float *>(smem + kCol);
    int *bad_from = reinterpret_cast<int *>(smem + kBad);
    volatile int *bad_chunk = reinterpret_cast<volatile int *>(tmem_slot + 1);   // the last chunk with entries that are not finite
    constexpr uint32_t kColumns = ADDS ? 64 : 256;
    if (tid == 0) {
        for (int i = 0; i < kBarCount; ++i)
            mbar_init(bar + i, i == kSReady ? 2 * kN : i >= kPReady && i <= kYStored ? kRowThreads : 1);
        *bad_chunk = -1;
        mbar_fence_init();
    }
    if (warp == 8) tmem_alloc(tmem_slot, kColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t t_kv = tmem + (ADDS ? 0 : kKV);

    wait_for_previous();
    const int chain = blockIdx.x % p.chains, order = blockIdx.x / p.chains;
    const int bi = chain / p.H, h = chain % p.H;
    const int len = p.lens == nullptr ? p.T : min(max(p.lens[bi], 0), p.T);
    const float lambda = p.log_decay[h];
    // The order-th segment that is worked on, its tokens and chunks.
    const int seg = REVERSED ? p.segments - 1 - order : order;
    const int64_t seg_tokens = (int64_t)p.chunks * kL;
    const int begin = (int)min((int64_t)p.T, seg * seg_tokens), end = (int)min((int64_t)p.T, (seg + 1) * seg_tokens);
    const int live = min(len, end) - begin;   // tokens of this segment (none if not positive)
    const int count = live > 0 ? (live + kL - 1) / kL : 0;
    auto first_token = [&](int it) { return begin + (REVERSED ? count - 1 - it : it) * kL; };
    // d^k; d^0 is 1 for every d
    auto power = [&](int64_t k) { return k == 0 ? 1.f : expf(lambda * (float)k); };
    // Rows wait for one another at barriers, so none leaves early: after a time-out a thread waits no more and walks on to the end.
    bool ok = true;
    auto wait = [&](Bar b, uint32_t parity) {
        if (ok) ok = mbar_wait(bar + b, parity);
    };

    if (warp == 9) {
        // ---- loads: a tile is refilled when the last product that reads it is done
        if (elect_one()) {
            auto load = [&](int it, const CUtensorMap *map, uint32_t tile, int full) {
                mbar_expect_tx(bar + full, kTile);
                tma_load_3d(smem + tile, map, h * kN, first_token(it), bi, bar + full);
            };
            auto load_ab = [&](int it) {
                if (it >= count) return;
                if (!ADDS) load(it, &maps.a, kA, kFullA);
                load(it, &maps.b, kB, kFullB);
            };
            auto load_c = [&](int it) {
                if (it < count) load(it, &maps.c, kC + (it & 1) * kTile, kFullC + (it & 1));
            };
            auto prefetch_ab = [&](int it) {   // (their loads have to wait for this chunk's products, and then find them in L2)
                if (it >= count) return;
                if (!ADDS) tma_prefetch_3d(&maps.a, h * kN, first_token(it), bi);
                tma_prefetch_3d(&maps.b, h * kN, first_token(it), bi);
            };
            load_ab(0);
            load_c(0);
            load_c(1);
            prefetch_ab(1);
            for (int it = 0; it < count; ++it) {
                const uint32_t ph = it & 1;
                if (it + 1 < count) {
                    if (!(ok = mbar_wait(bar + kKvDone, ph))) break;
                    load_ab(it + 1);
                    prefetch_ab(it + 2);
                }
                if (!ADDS) {   // y lies where c was
                    if (!(ok = mbar_wait(bar + kYStored, ph))) break;
                    tma_store_3d(&maps.y, h * kN, first_token(it), bi, smem + kC + (it & 1) * kTile);
                    bulk_commit_group();
                    if (it + 2 < count) bulk_wait_group_read<0>();
                }
                load_c(it + 2);
            }
            bulk_wait_group<0>();
            // (after a time-out what is in flight lands before the CTA leaves: both phases of every tile)
            if (!ok)
                for (int tile = kFullA; tile <= kFullC1; ++tile)
                    for (uint32_t i = 0; i < 2; ++i) mbar_wait(bar + tile, i, 100000u);
        }
    } else if (warp == 8) {
        // ---- products
        if (elect_one()) {
            constexpr uint32_t id_p = make_idesc(kFmtBF16, 128, 128, false, false), id_y = make_idesc(kFmtBF16, 128, 64, false, true),
                               id_kv = make_idesc(kFmtBF16, 128, 64, true, true);
            // one of the three parts of w C
            auto add = [&](uint32_t part, bool first) {
#pragma unroll
                for (int k = 0; k < kL / 16; ++k)
                    umma_f16(t_kv, make_smem_desc(base + (REVERSED ? kA : kB) + k * 2048, kTile, 1024),
                             make_smem_desc(base + part + k * 2048, kTile, 1024), id_kv, !first || k > 0);
            };
            for (int it = 0; it < count; ++it) {
                const uint32_t ph = it & 1;
                if (!ADDS) {
                    ok = mbar_wait(bar + kFullA, ph) && mbar_wait(bar + kFullB, ph) && (it == 0 || mbar_wait(bar + kYRead, ph ^ 1));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kN / 16; ++k)
                        umma_f16(tmem + kP, make_smem_desc(base + kA + k * 32, 16, 1024), make_smem_desc(base + kB + k * 32, 16, 1024), id_p, k > 0);
                    umma_commit(bar + kPDone);
                    if (!(ok = mbar_wait(bar + kSReady, ph))) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 2 * (kN / 16); ++k)   // S hi, S lo
                        umma_f16(tmem + kY2, make_smem_desc(base + kA + (k & 3) * 32, 16, 1024),
                                 make_smem_desc(base + kS + (k >> 2) * kSPart + (k & 3) * 2048, kSPart, 1024), id_y, k > 0);
                    umma_commit(bar + kADone);
                    ok = mbar_wait(bar + kPReady, ph) && mbar_wait(bar + kFullC + (it & 1), (uint32_t)(it >> 1) & 1u);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kL / 16; ++k)
                        umma_f16_ts(tmem + kY1, tmem + p_operand(k), make_smem_desc(base + kC + (it & 1) * kTile + k * 2048, kTile, 1024), id_y, k > 0);
                    umma_commit(bar + kYDone);
                }
                ok = mbar_wait(bar + kWReady, ph) && (!ADDS || mbar_wait(bar + kFullB, ph));
                if (!ok) break;
                tc_fence_after();
                add(kW, true);
                add(kW + kTile, false);
                add(kA, false);
                umma_commit(bar + kKvDone);
            }
            umma_commit(bar + kEnd);
            ok = mbar_wait(bar + kEnd, 0) && ok;
        }
    } else {
        // ---- rows
        const int quarter = warp & 3, half = warp >> 2, row = tid & 127;
        const uint32_t t_lane = (uint32_t)(quarter * 32) << 16;
        const bool has_state = (quarter >= 2) == REVERSED;   // uniform in a warp
        const int bidx = row & 63, c0 = half * (kN / 2);      // the thread's part of S: row bidx, 32 columns
        float2 S[kN / 4];
#pragma unroll
        for (int j = 0; j < kN / 4; ++j) S[j] = make_float2(0.f, 0.f);
        if (tid <= kL) dec[tid] = power(tid);
        if (tid < 32) col[tid] = power(REVERSED ? tid : 31 - tid);
        constexpr int kNoToken = REVERSED ? -1 : kL;
        if (tid < kN) bad_from[tid] = kNoToken;
        float *parts = p.parts + (size_t)chain * p.segments * (kN * kN);
        auto write = [&](float *dst) {
#pragma unroll
            for (int j = 0; j < kN / 4; ++j) {
                dst[(c0 + 2 * j) * kN + bidx] = S[j].x;
                dst[(c0 + 2 * j + 1) * kN + bidx] = S[j].y;
            }
        };
        if (has_state) {
            auto read = [&](const float *src, bool transposed) {
                if (transposed) {
#pragma unroll
                    for (int j = 0; j < kN / 4; j += 2) {
                        const float4 v = *reinterpret_cast<const float4 *>(src + bidx * kN + c0 + 2 * j);
                        S[j] = make_float2(v.x, v.y);
                        S[j + 1] = make_float2(v.z, v.w);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kN / 4; ++j) S[j] = make_float2(src[(c0 + 2 * j) * kN + bidx], src[(c0 + 2 * j + 1) * kN + bidx]);
                }
            };
            const float *s_in = p.s_in == nullptr ? nullptr : p.s_in + (size_t)chain * (kN * kN);
            if (ADDS) {
                if (order == 0) {   // the state in front of everything: s_in may be overwritten before the last segment starts
                    if (s_in != nullptr) read(s_in, p.s_in_transposed);
                    write(parts);
#pragma unroll
                    for (int j = 0; j < kN / 4; ++j) S[j] = make_float2(0.f, 0.f);
                }
            } else if (p.segments > 1) {
                read(parts + (size_t)order * (kN * kN), false);
            } else if (s_in != nullptr) {
                read(s_in, p.s_in_transposed);
            }
        }
        // S as the operand of the next chunk's Y2: row b, columns c, hi and lo
        auto publish = [&] {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 s = S[4 * q + e];
                    hi[e] = pack2(s);
                    lo[e] = pack2(sub2(s, unpack2(hi[e])));
                }
                sts16(base + kS + piece(bidx, half * 4 + q), make_uint4(hi[0], hi[1], hi[2], hi[3]));
                sts16(base + kS + kSPart + piece(bidx, half * 4 + q), make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            fence_proxy_async();
            mbar_arrive(bar + kSReady);
        };
        if (!ADDS && has_state && count > 0) publish();
        rows_sync();   // (the tables)

        for (int it = 0; it < count; ++it) {
            const uint32_t ph = it & 1, tile_c = kC + (it & 1) * kTile;
            const int t0 = first_token(it), n = min(kL, len - t0);   // tokens of the chunk: all but the sequence's last have 128
            uint32_t own[4];   // where this thread's half row lies in a tile
#pragma unroll
            for (int q = 0; q < 4; ++q) own[q] = piece(row, half * 4 + q);

            // c as the products may see it
            wait((Bar)(kFullC + (it & 1)), (uint32_t)(it >> 1) & 1u);
            if (n < kL) {   // (uniform) behind the sequence anything may stand
                wait(kFullB, ph);
                if (row >= n) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        sts16(base + kB + own[q], make_uint4(0u, 0u, 0u, 0u));
                        sts16(base + tile_c + own[q], make_uint4(0u, 0u, 0u, 0u));
                    }
                    fence_proxy_async();
                }
            }
            {
                uint4 in[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) in[q] = lds16(base + tile_c + own[q]);
                uint32_t all = 0;   // sign bits: an exponent of ones in the low or the high half of a word
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    for (uint32_t u : {in[q].x, in[q].y, in[q].z, in[q].w}) all |= ((u & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                if (all != 0u) {
                    for (int j = c0; j < c0 + kN / 2; ++j) {
                        unsigned short *c = reinterpret_cast<unsigned short *>(smem + tile_c + piece(row, j >> 3) + (j & 7) * 2);
                        if ((*c & 0x7f80) != 0x7f80) continue;
                        *c = 0;
                        if (REVERSED) atomicMax(bad_from + j, row);
                        else atomicMin(bad_from + j, row);
                    }
                    *bad_chunk = it;
                    fence_proxy_async();
                }
            }

            if (!ADDS) {
                // P: decays and mask, and bf16.  Each warp takes two blocks of 32 columns, the outer one first (see p_operand).
                wait(kPDone, ph);
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int c = half == 0 ? i : 3 - i;
                    uint32_t out[16];
                    if (REVERSED ? c < quarter : c > quarter) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) out[e] = 0u;
                    } else {
                        uint32_t v[32];
                        tmem_ld32(tmem + kP + t_lane + c * 32, v);
                        tmem_ld_wait();
                        if (c == quarter) {
                            const float *gap0 = dec + (REVERSED ? -lane : lane);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const bool seen = REVERSED ? e >= lane : e <= lane;
                                const float g = seen ? gap0[REVERSED ? e : -e] : 0.f;
                                v[e] = seen ? __float_as_uint(__uint_as_float(v[e]) * g) : 0u;
                            }
#pragma unroll
                            for (int e = 0; e < 16; ++e) out[e] = pack_bf2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
                        } else {
                            // d^gap as a factor of the row and one of the column, neither with a negative power
                            const float f = dec[REVERSED ? 32 * c - row : row - 32 * c - 31];
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 g = *reinterpret_cast<const float4 *>(col + e);
                                out[e / 2] = pack2(__fmul2_rn(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])),
                                                              __fmul2_rn(make_float2(g.x, g.y), make_float2(f, f))));
                                out[e / 2 + 1] = pack2(__fmul2_rn(make_float2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])),
                                                                  __fmul2_rn(make_float2(g.z, g.w), make_float2(f, f))));
                            }
                        }
                        if (REVERSED && 32 * c + 32 > n) {   // (forwards no row of the sequence sees what is behind it)
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                if (32 * c + 2 * e >= n) out[e] = 0u;
                                else if (32 * c + 2 * e + 1 >= n) out[e] &= 0xffffu;
                            }
                        }
                    }
                    tmem_st16(tmem + p_operand(2 * c) + t_lane, out);
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(bar + kPReady);
            }

            // w C in three parts.  (The product that read the previous ones is done, and a has been read.)
            if (it > 0) wait(kKvDone, ph ^ 1);
            if (!ADDS) wait(kADone, ph);
            {
                const float w = row < n ? dec[REVERSED ? row + 1 : n - 1 - row] : 0.f;
                uint4 in[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) in[q] = lds16(base + tile_c + own[q]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t u[4] = {in[q].x, in[q].y, in[q].z, in[q].w};
                    uint32_t hi[4], mid[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float2 x = __fmul2_rn(unpack2(u[e]), make_float2(w, w));
                        hi[e] = pack2(x);
                        x = sub2(x, unpack2(hi[e]));
                        mid[e] = pack2(x);
                        lo[e] = pack2(sub2(x, unpack2(mid[e])));
                    }
                    sts16(base + kW + own[q], make_uint4(hi[0], hi[1], hi[2], hi[3]));
                    sts16(base + kW + kTile + own[q], make_uint4(mid[0], mid[1], mid[2], mid[3]));
                    sts16(base + kA + own[q], make_uint4(lo[0], lo[1], lo[2], lo[3]));
                }
            }
            fence_proxy_async();
            mbar_arrive(bar + kWReady);

            bool any_bad = false;   // (the same for all: every thread has looked at c before the products that are waited for)
            if (!ADDS) {
                // y, to where this thread's c was
                wait(kYDone, ph);
                tc_fence_after();
                any_bad = *bad_chunk == it;
                const float f = dec[REVERSED ? max(n - 1 - row, 0) : row + 1];
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    uint32_t v[16], u[16];
                    tmem_ld16(tmem + kY1 + t_lane + c0 + part * 16, v);
                    tmem_ld16(tmem + kY2 + t_lane + c0 + part * 16, u);
                    tmem_ld_wait();
                    if (part == 1) {
                        tc_fence_before();
                        mbar_arrive(bar + kYRead);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float2 x = __ffma2_rn(make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])), make_float2(f, f),
                                                    make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
                        u[e / 2] = pack2(x);
                    }
                    if (any_bad) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int from = bad_from[c0 + part * 16 + e];
                            if (REVERSED ? row <= from : row >= from) u[e / 2] |= e & 1 ? 0x7fff0000u : 0x7fffu;
                        }
                    }
                    if (row >= n) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) u[e] = 0u;
                    }
                    sts16(base + tile_c + own[2 * part], make_uint4(u[0], u[1], u[2], u[3]));
                    sts16(base + tile_c + own[2 * part + 1], make_uint4(u[4], u[5], u[6], u[7]));
                }
                fence_proxy_async();
                mbar_arrive(bar + kYStored);
            }
            if (has_state) {
                wait(kKvDone, ph);
                tc_fence_after();
                any_bad = *bad_chunk == it;
                const float dn = dec[n];
                uint32_t v[32];
                tmem_ld32(t_kv + t_lane + c0, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < kN / 4; ++j)
                    S[j] = __ffma2_rn(S[j], make_float2(dn, dn), make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])));
                if (any_bad) {
#pragma unroll
                    for (int j = 0; j < kN / 4; ++j) {
                        if ((unsigned)bad_from[c0 + 2 * j] < (unsigned)kL) S[j].x = __uint_as_float(0x7fffffffu);
                        if ((unsigned)bad_from[c0 + 2 * j + 1] < (unsigned)kL) S[j].y = __uint_as_float(0x7fffffffu);
                    }
                }
                tc_fence_before();
                if (!ADDS && it + 1 < count) publish();
            }
            if (ADDS) {
                wait(kKvDone, ph);
                any_bad = *bad_chunk == it;
            }
            if (any_bad) {
                rows_sync();   // (all have read it)
                if (tid < kN) bad_from[tid] = kNoToken;
                rows_sync();
            }
        }
        if (ok && !ADDS) {   // chunks behind the sequence
            const int from = begin + count * kL;
            for (int64_t i = tid; i < (int64_t)(end - from) * 8; i += kRowThreads)
                *reinterpret_cast<uint4 *>(p.y + (((int64_t)bi * p.T + from + i / 8) * p.H + h) * kN + i % 8 * 8) = make_uint4(0u, 0u, 0u, 0u);
        }
        if (ok && has_state) {
            if (ADDS) write(parts + (size_t)(order + 1) * (kN * kN));
            else if (order == p.segments - 1 && p.s_out != nullptr) write(p.s_out + (size_t)chain * (kN * kN));
        }
    }
    __syncwarp();
    if (!ok) atomicExch(p.status, (int)kDevTimeout);
    tc_fence_before();
    __syncthreads();
    if (warp == 8) tmem_dealloc(tmem, kColumns);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(f);
    });
    return fn;
}

// A [B,T,H,64] tensor in tiles of 128 tokens of one head; tokens behind T read as zero.
bool describe(CUtensorMap *map, const void *ptr, const LinearAttentionPass &p) {
    const EncodeTiledFn encode = encode_fn();
    const cuuint64_t dims[3] = {(cuuint64_t)(p.H * kN), (cuuint64_t)p.T, (cuuint64_t)p.B};
    const cuuint64_t strides[2] = {(cuuint64_t)(p.H * kN * 2), (cuuint64_t)(p.T * p.H * kN * 2)};
    const cuuint32_t box[3] = {(cuuint32_t)kN, (cuuint32_t)kL, 1}, step[3] = {1, 1, 1};
    return encode != nullptr && encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr), dims, strides, box, step,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool REVERSED, bool ADDS>
cudaError_t launch(const Maps &maps, const ChunkArgs &args, int64_t ctas, int device, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};   // devices the kernel has its shared memory on
    const uint64_t bit = (uint64_t)1 << (device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(chunk_kernel<REVERSED, ADDS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch_serialized(chunk_kernel<REVERSED, ADDS>, (unsigned)ctas, (unsigned)kThreads, kSmem, stream, maps, args);
}

}  // namespace

bool linear_attention_chunks_supported(const LinearAttentionPass &p) { return p.bf16 && p.N == kN && p.T >= 64; }

size_t linear_attention_chunks_workspace_bytes(const LinearAttentionPass &p) {
    using namespace linear_attention_plan;
    const int64_t chains = p.B * p.H;
    return state_bytes(chains, cut(chains, (p.T + kL - 1) / kL, (int64_t)p.num_sms * kResident, 1, INT64_MAX).segments, kN);
}

int launch_linear_attention_chunks(const LinearAttentionPass &p, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    using namespace linear_attention_plan;
    const int64_t chains = p.B * p.H;
    const Cut c = cut(chains, (p.T + kL - 1) / kL, (int64_t)p.num_sms * kResident, 1, workspace == nullptr ? 1 : segments_in(workspace_bytes, chains, kN));
    Maps maps;
    if (!describe(&maps.a, p.a, p) || !describe(&maps.b, p.b, p) || !describe(&maps.c, p.c, p) || !describe(&maps.y, p.y, p)) return (int)cudaErrorInvalidValue;
    ChunkArgs args{};
    args.y = static_cast<__nv_bfloat16 *>(p.y);
    args.log_decay = p.log_decay;
    args.lens = p.lens;
    args.s_in = p.s_in;
    args.s_out = p.s_out;
    args.parts = c.segments > 1 ? static_cast<float *>(workspace) : nullptr;
    args.T = (int)p.T;
    args.H = (int)p.H;
    args.chains = (int)chains;
    args.segments = (int)c.segments;
    args.chunks = (int)c.chunks;
    args.s_in_transposed = p.s_in_transposed;
    if (int e = device_status_ptr(p.device, &args.status)) return e;
    if (c.segments > 1) {
        const int64_t ctas = chains * (c.segments - 1);
        const cudaError_t e = p.reversed ? launch<true, true>(maps, args, ctas, p.device, stream) : launch<false, true>(maps, args, ctas, p.device, stream);
        if (e != cudaSuccess) return (int)e;
        if (int f = launch_segment_states(p, args.parts, c.segments, c.chunks * kL, stream)) return f;
    }
    const int64_t ctas = chains * c.segments;
    return (int)(p.reversed ? launch<true, false>(maps, args, ctas, p.device, stream) : launch<false, false>(maps, args, ctas, p.device, stream));
}

}  // namespace rwkv7
