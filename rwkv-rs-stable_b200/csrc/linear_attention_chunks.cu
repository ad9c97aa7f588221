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
// Four products of a chunk: P = A B^T [128 x 128], Y2 = A S [128 x 64], the sum for S' = (w C)^T B [64 x 64] and, once P carries
// its decays and its mask, Y1 = P C [128 x 64].  HBM gives an SM a chunk's 64 KB in 1.5 us.  What is scarcer is shared memory's
// 128 bytes a cycle, which the products' operands, the loads and everything else share: so P and w C are operands in TMEM (as operands in
// shared memory they made 160 us of the 129 below).  One CTA an SM runs all of it as a pipeline:
//   warps 0-7         P of a chunk, then y          (two threads a row: a TMEM lane and a half of its columns)
//   warps 8 9 12 13   w C of the chunk behind, transposed and in three parts, put into TMEM when the product of this one has read the last
//                     (where only what a segment adds is wanted, with 0 1 4 5, which take every other chunk)
//   warps 16 17       S behind a chunk from its product, one row of S a thread
//   warp 14           d^128 in 64 bits, for these (its some 0.3 us of code would else stand in front of the first chunk)
//   warp 10           issues the products: P, the sum for S', Y2, Y1
//   warp 11           loads, four chunks ahead, and stores y from where c was
// 8 x 4096 tokens of 32 heads: 129 us, 4.2 TB/s, 2.3 us a chunk and SM.  What bounds it is the chain of a chunk through the roles: its state waits
// for its sum, its sum for w C, y for P's decays, and each of these hands over through a barrier.
//
// Precision: y is rounded to bf16, and so is P (once); S stays in fp32 registers and enters Y2 as hi + lo (16 bits and a
// sign), because its errors would add up; the sum for S' takes w C as hi + mid + lo, all 24 bits, because S is an fp32 output.  The decays inside
// a chunk are fp32 powers (expf); d^128, which a state meets again with every chunk, comes from 64 bits.
//
// Entries of c that are not finite would reach tokens on the other side of the mask (0 x inf): a chunk that has some takes
// them as zero and sets what they do reach, the column's later tokens and the state's column, to NaN.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <mutex>

#include "elements.cuh"
#include "kernels.h"
#include "launch.h"
#include "linear_attention_decay.cuh"
#include "linear_attention_plan.h"
#include "sm100_mma.cuh"
#include "sm100_umma.cuh"

namespace rwkv7 {
namespace {

using namespace sm100;

constexpr int kN = 64, kL = linear_attention_plan::kChunk;
constexpr int kGroup = 256, kThreads = 576, kStages = 4;
constexpr uint32_t kTile = kL * 128;           // [128 tokens][64] bf16, 128-byte swizzle
// Shared memory: a, b, c of every stage, two parts of S, tables, barriers.
constexpr uint32_t kA = 0, kB = kTile, kC = 2 * kTile, kStage = 3 * kTile, kS = kStages * kStage, kSPart = kN * 128;
constexpr uint32_t kCol = kS + 2 * kSPart;     // d^31 .. d^0 forwards, d^0 .. d^31 reversed
constexpr uint32_t kDiag = kCol + 128;         // the same continued by zeros (reversed: behind zeros), four times, each a word further on
constexpr uint32_t kDiagWords = 68;
constexpr uint32_t kDec = kDiag + 4 * kDiagWords * 4;   // d^0 .. d^128
constexpr uint32_t kWhole = kDec + 520;                 // d^128 as the factor of whole chunks
constexpr uint32_t kBars = kWhole + 16;
static_assert(sizeof(SteadyPower) <= 16);
enum Bar {   // [stage], [parity of the chunk], or one
    kFull,                                                // a, b and c are loaded
    kFreeA = kFull + kStages, kFreeB = kFreeA + kStages,  // the last product that reads it is done (without y: and S behind the chunk is known)
    kYStored = kFreeB + kStages,
    kAddDone = kYStored + kStages, kAddRead = kAddDone + 2,   // (the latter without y; with it kSReady says so)
    kWReady = kAddRead + 2,
    kPDone = kWReady + 2, kPReady, kYDone, kYRead, kSReady, kEnd, kBarCount
};
constexpr uint32_t kSlot = kBars + kBarCount * 8;   // TMEM address, then the last chunk in each stage with entries that are not finite
// [stage][column]: 128 x chunk + 127 - the first such token (reversed: + the last)
constexpr uint32_t kBad = kSlot + 24;
constexpr uint32_t kSmem = kBad + kStages * kN * 4;
static_assert(kSmem <= 232448, "shared memory of a CTA");
// TMEM columns.  P as fp32 on 128; as bf16 its first half on columns 0-31, its second on 96-127, where the threads that read those
// columns put it; Y1 between them.  Y2; the sums for S' of even and odd chunks; three parts of w C (lanes 0-63).
constexpr uint32_t kP = 0, kY1 = 32, kY2 = 128, kW = 320;
__host__ __device__ constexpr uint32_t t_add(int it) { return 192 + (it & 1) * 64; }
// (without y there is room for those of two chunks)
template <bool ADDS>
__host__ __device__ constexpr uint32_t t_w(int it) {
    return ADDS && (it & 1) ? kP : kW;
}
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

// 16-byte piece `q` of a 128-byte row.
__device__ __forceinline__ uint32_t piece(int row, int q) { return (uint32_t)row * 128u + (uint32_t)((q ^ (row & 7)) << 4); }
__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float2 unpack2(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(float2 v) { return pack_bf2(v.x, v.y); }
// The part in front of others: bf16's largest number, not infinity, for what lies beyond that, which the last part then has.
__device__ __forceinline__ uint32_t pack2_finite(float2 v) {
    uint32_t u;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(v.y), "f"(v.x));
    return u;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return __fadd2_rn(a, make_float2(-b.x, -b.y)); }
// What is not finite in 16 columns (two pieces) of a token becomes zero, and its place is noted: first + 127 - token (reversed: + token).
// In loops, as all that is rare or can be: a kernel of several roles lives on what the instruction caches hold of each.  Unrolled, with this for
// every register, a chunk took 7300 cycles instead of 4400, most of them waits for instructions.
__device__ __forceinline__ void take_out(unsigned char *tile, int token, int c8, int *bad_from, int first, bool reversed) {
#pragma unroll 1
    for (int j = 0; j < 16; ++j) {
        unsigned short *c = reinterpret_cast<unsigned short *>(tile + piece(token, c8 + j / 8) + j % 8 * 2);
        if ((*c & 0x7f80) != 0x7f80) continue;
        *c = 0;
        atomicMax(bad_from + c8 * 8 + j, first + (reversed ? token : kL - 1 - token));
    }
}
// Half a row of y gets NaN where such an entry reaches it.
__device__ __forceinline__ void put_nan(unsigned char *tile, int token, int half, const int *bad_from, int first, bool reversed) {
#pragma unroll 1
    for (int j = half * 32; j < half * 32 + 32; ++j) {
        const int from = bad_from[j] - first;   // (negative: of an earlier chunk)
        if (from >= 0 && (reversed ? token <= from : token >= kL - 1 - from))
            *reinterpret_cast<unsigned short *>(tile + piece(token, j / 8) + j % 8 * 2) = 0x7fff;
    }
}

// ADDS: only what a segment adds to the state.
template <bool REVERSED, bool ADDS>
__global__ void __launch_bounds__(kThreads, 1)
chunk_kernel(const __grid_constant__ Maps maps, const ChunkArgs p) {
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (smem_u32(smem) & 1023u) {
        if (tid == 0) atomicExch(p.status, (int)kDevInternal);
        return;
    }
    const uint32_t base = smem_u32(smem);
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + kBars);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + kSlot);
    volatile int *bad_chunk = reinterpret_cast<volatile int *>(smem + kSlot + 4);
    int *bad_from = reinterpret_cast<int *>(smem + kBad);
    float *dec = reinterpret_cast<float *>(smem + kDec), *col = reinterpret_cast<float *>(smem + kCol), *diag = reinterpret_cast<float *>(smem + kDiag);
    constexpr int kMmaWarp = 10, kLoadWarp = 11, kPowerWarp = 14, kStateWarp = 16;   // (w C and S are on lanes 0-63: their warps are numbers 0 and 1 of four)
    if (tid == 0) {
        for (int i = 0; i < kBarCount; ++i)
            mbar_init(bar + i, (i >= kYStored && i < kAddDone) || i == kPReady || i == kYRead ? kGroup
                               : i >= kWReady && i < kPDone ? kGroup / 2 : (i >= kAddRead && i < kWReady) || i == kSReady ? kN
                               : i < kFreeA ? (ADDS ? 2 : 3) : ADDS && i >= kFreeB && i < kYStored ? 1 + kN : 1);
        mbar_fence_init();
        for (int i = 0; i < kStages; ++i) bad_chunk[i] = -1;
    }
    if (tid >= kGroup && tid < kGroup + kStages * kN) bad_from[tid - kGroup] = -1;
    if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_previous();
    const int chain = blockIdx.x % p.chains, order = blockIdx.x / p.chains;
    const int bi = chain / p.H, h = chain % p.H;
    const int len = p.lens == nullptr ? p.T : min(max(p.lens[bi], 0), p.T);
    // Tables, by those that use them; the loads start meanwhile.
    if (warp != kMmaWarp && warp != kLoadWarp) {
        const float lambda = p.log_decay[h];
        auto power = [&](int k) { return k == 0 ? 1.f : expf(lambda * (float)k); };   // d^k; d^0 is 1 for every d
        // (reversed, a chunk of fewer than 128 tokens meets powers behind its last one times zero: where d is above one they are kept finite)
        if (tid <= kL) dec[tid] = REVERSED && power(tid) > FLT_MAX ? FLT_MAX : power(tid);
        const int other = (tid < kMmaWarp * 32 ? tid : tid - 64) - (kL + 1);   // threads that have no entry of dec
        if (other >= 0 && other < 32) col[other] = power(REVERSED ? other : 31 - other);
        // diag[shift][k + shift] for k = e - lane + 31: d^(lane - e) where e <= lane (reversed: d^(e - lane) where e >= lane), else 0
        const int i = other - 32;
        static_assert(kThreads - 64 - (kL + 1) - 32 >= (int)(4 * kDiagWords));
        if (i >= 0 && i < (int)(4 * kDiagWords)) {
            const int gap = REVERSED ? i % (int)kDiagWords - i / (int)kDiagWords - 31 : 31 - (i % (int)kDiagWords - i / (int)kDiagWords);
            diag[i] = gap >= 0 && gap < 32 ? power(gap) : 0.f;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 64) : "memory");
    }
    // The order-th segment that is worked on, its tokens and chunks.
    const int seg = REVERSED ? p.segments - 1 - order : order;
    const int64_t seg_tokens = (int64_t)p.chunks * kL;
    const int begin = (int)min((int64_t)p.T, seg * seg_tokens), end = (int)min((int64_t)p.T, (seg + 1) * seg_tokens);
    const int live = min(len, end) - begin;   // tokens of this segment (none if not positive)
    const int count = live > 0 ? (live + kL - 1) / kL : 0;
    auto first_token = [&](int it) { return begin + (REVERSED ? count - 1 - it : it) * kL; };
    auto tokens_of = [&](int it) { return min(kL, len - first_token(it)); };   // all but the sequence's last chunk have 128
    // A barrier of the chunk's stage, or of its parity, in the chunk's turn of it.  A thread whose wait has run out waits no more, and walks
    // on to the end, so that nobody waits for it at a barrier of threads.
    bool ok = true;
    auto wait = [&](int b, uint32_t parity) {
        if (ok) ok = mbar_wait(bar + b, parity);
        return ok;
    };
    auto wait_stage = [&](int b, int it) { return wait(b + it % kStages, (uint32_t)(it / kStages) & 1u); };
    auto wait_turn = [&](int b, int it) { return wait(b + (it & 1), (uint32_t)(it >> 1) & 1u); };

    if (warp == kLoadWarp) {
        // ---- loads, and the stores of y
        if (elect_one()) {
            auto load = [&](int it, const CUtensorMap *map, uint32_t tile) {
                if (it >= count) return;
                mbar_expect_tx(bar + kFull + it % kStages, kTile);
                tma_load_3d(smem + it % kStages * kStage + tile, map, h * kN, first_token(it), bi, bar + kFull + it % kStages);
            };
            for (int it = 0; it < kStages; ++it) {
                if (!ADDS) load(it, &maps.a, kA);
                load(it, &maps.b, kB);
                load(it, &maps.c, kC);
            }
            for (int it = 0; it < count; ++it) {
                if (!wait_stage(kFreeB, it)) break;
                load(it + kStages, &maps.b, kB);
                if (!ADDS) {
                    if (!wait_stage(kFreeA, it)) break;
                    load(it + kStages, &maps.a, kA);
                    if (!wait_stage(kYStored, it)) break;
                    tma_store_3d(&maps.y, h * kN, first_token(it), bi, smem + it % kStages * kStage + kC);
                    bulk_commit_group();
                    if (it + kStages < count) bulk_wait_group_read<0>();
                }
                load(it + kStages, &maps.c, kC);
            }
            bulk_wait_group<0>();
            // (after a time-out what is in flight lands before the CTA leaves: both phases of every stage)
            if (!ok)
                for (int b = kFull; b < kFreeA; ++b)
                    for (uint32_t i = 0; i < 2; ++i) mbar_wait(bar + b, i, 100000u);
        }
    } else if (warp == kMmaWarp) {
        // ---- products
        if (elect_one()) {
            constexpr uint32_t id_p = make_idesc(kFmtBF16, 128, 128, false, false), id_y2 = make_idesc(kFmtBF16, 128, 64, false, false),
                               id_mn = make_idesc(kFmtBF16, 128, 64, false, true);
            // P first, for what waits for it takes longest; while it is given its decays, the sum for S' and Y2 follow.  (A third of the sum in
            // front of P made 135 us of 129, Y2 in front of the sum 144.)
            for (int it = 0; it < count; ++it) {
                const uint32_t at = base + it % kStages * kStage, ph = it & 1;
                if (!ADDS) {
                    if (!wait_stage(kFull, it) || (it > 0 && !wait(kYRead, ph ^ 1))) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kN / 16; ++k)
                        umma_f16(tmem + kP, make_smem_desc(at + kA + k * 32, 16, 1024), make_smem_desc(at + kB + k * 32, 16, 1024), id_p, k > 0);
                    umma_commit(bar + kPDone);
                }
                // (the sum of two chunks ago has been read: S behind it was published before the last Y2)
                if (!wait_turn(kWReady, it) || (ADDS && it >= 2 && !wait_turn(kAddRead, it - 2))) break;
                tc_fence_after();
#pragma unroll 1
                for (int part = 0; part < 3; ++part)
#pragma unroll
                    for (int k = 0; k < kL / 16; ++k)
                        umma_f16_ts(tmem + t_add(it), tmem + t_w<ADDS>(it) + part * 64 + k * 8, make_smem_desc(at + kB + k * 2048, kTile, 1024), id_mn, part > 0 || k > 0);
                umma_commit(bar + kAddDone + ph);
                umma_commit(bar + kFreeB + it % kStages);
                if (ADDS) continue;
                if (!wait(kSReady, ph)) break;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 2 * (kN / 16); ++k)   // S hi, S lo
                    umma_f16(tmem + kY2, make_smem_desc(at + kA + (k & 3) * 32, 16, 1024),
                             make_smem_desc(base + kS + (k >> 2) * kSPart + (k & 3) * 32, 16, 1024), id_y2, k > 0);
                umma_commit(bar + kFreeA + it % kStages);
                if (!wait(kPReady, ph)) break;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < kL / 16; ++k)   // (c is as the products may see it: w C is ready)
                    umma_f16_ts(tmem + kY1, tmem + p_operand(k), make_smem_desc(at + kC + k * 2048, kTile, 1024), id_mn, k > 0);
                umma_commit(bar + kYDone);
            }
            umma_commit(bar + kEnd);
            ok = mbar_wait(bar + kEnd, 0) && ok;
        }
    } else if (warp >= kStateWarp) {
        // ---- the state
        const int row = tid - kStateWarp * 32;   // of S: the thread's column of c
        const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
        float2 S[kN / 2];
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) S[j] = make_float2(0.f, 0.f);
        float *parts = p.parts + (size_t)chain * p.segments * (kN * kN);
        auto write = [&](float *dst) {
#pragma unroll
            for (int j = 0; j < kN / 2; j += 2) *reinterpret_cast<float4 *>(dst + row * kN + 2 * j) = make_float4(S[j].x, S[j].y, S[j + 1].x, S[j + 1].y);
        };
        auto read = [&](const float *src, bool transposed) {
            if (!transposed) {
#pragma unroll
                for (int j = 0; j < kN / 2; j += 2) {
                    const float4 v = *reinterpret_cast<const float4 *>(src + row * kN + 2 * j);
                    S[j] = make_float2(v.x, v.y);
                    S[j + 1] = make_float2(v.z, v.w);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kN / 2; ++j) S[j] = make_float2(src[2 * j * kN + row], src[(2 * j + 1) * kN + row]);
            }
        };
        const float *s_in = p.s_in == nullptr ? nullptr : p.s_in + (size_t)chain * (kN * kN);
        if (ADDS) {
            if (order == 0) {   // the state in front of everything: s_in may be overwritten before the last segment starts
                if (s_in != nullptr) read(s_in, p.s_in_transposed);
                write(parts);
#pragma unroll
                for (int j = 0; j < kN / 2; ++j) S[j] = make_float2(0.f, 0.f);
            }
        } else if (p.segments > 1) {
            read(parts + (size_t)order * (kN * kN), false);
        } else if (s_in != nullptr) {
            read(s_in, p.s_in_transposed);
        }
        // S as the operand of a chunk's Y2: row c, columns b, hi and lo
        auto publish = [&] {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 s = S[4 * q + e];
                    hi[e] = pack2_finite(s);
                    lo[e] = pack2(sub2(s, unpack2(hi[e])));
                }
                sts16(base + kS + piece(row, q), make_uint4(hi[0], hi[1], hi[2], hi[3]));
                sts16(base + kS + kSPart + piece(row, q), make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            fence_proxy_async();
            mbar_arrive(bar + kSReady);
        };
        SteadyPower whole;
        for (int it = 0; it < count; ++it) {
            if (!ADDS) {
                if (it > 0) wait_stage(kFreeA, it - 1);   // the Y2 that reads the last one is done
                publish();
            }
            if (it == 0 && live >= kL) {
                asm volatile("bar.sync 2, 96;" ::: "memory");
                whole = *reinterpret_cast<const SteadyPower *>(smem + kWhole);
            }
            wait_turn(kAddDone, it);
            tc_fence_after();
            float dn = tokens_of(it) == kL ? whole.factor((uint32_t)it) : dec[tokens_of(it)];
            if (bad_chunk[it % kStages] == it && bad_from[it % kStages * kN + row] >= it * kL) dn = __uint_as_float(0x7fffffffu);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t v[16];
                tmem_ld16(tmem + t_add(it) + t_lane + q * 16, v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    S[q * 8 + e] = __ffma2_rn(S[q * 8 + e], make_float2(dn, dn), make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])));
            }
            tc_fence_before();   // (the sum has been read: here for publish's arrival as well)
            if (ADDS) {          // and the note of what is not finite: both places may be written again
                mbar_arrive(bar + kAddRead + (it & 1));
                mbar_arrive(bar + kFreeB + it % kStages);
            }
        }
        if (ok && ADDS) write(parts + (size_t)(order + 1) * (kN * kN));
        if (ok && !ADDS && order == p.segments - 1 && p.s_out != nullptr) write(p.s_out + (size_t)chain * (kN * kN));
    } else if (warp == kPowerWarp) {
        if (live >= kL) {   // (there is a whole chunk: the warps of the state wait for this in front of its sum)
            if (lane == 0) *reinterpret_cast<SteadyPower *>(smem + kWhole) = SteadyPower(exp((double)p.log_decay[h] * kL));
            __syncwarp();
            asm volatile("bar.arrive 2, 96;" ::: "memory");
        }
    } else if ((ADDS || warp >= 8) && (warp & 2) == 0) {
        // ---- w C, transposed and in three parts: 32 columns of c (TMEM lanes) and 64 tokens a warp, in fragments of 8 x 8: a register holds
        // tokens t and t + 1 of a column, two registers columns eight apart
        const int quarter = warp & 1, token0 = (warp >> 2 & 1) * 64;
        const uint32_t t_lane = (uint32_t)(quarter * 32) << 16;
        const int q = lane & 3;
        // the weights of this lane's pairs of tokens, token0 + 8 i + 2 q and the next, of a chunk of n
        float2 w[8];
        auto weigh = [&](int n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = token0 + 8 * i + 2 * q;   // (behind the sequence c is zero)
                w[i] = make_float2(dec[REVERSED ? t + 1 : max(n - 1 - t, 0)], dec[REVERSED ? t + 2 : max(n - 2 - t, 0)]);
            }
        };
        int weighed = 0;
        if (REVERSED) weigh(kL);
        // (without y its warps take the odd chunks)
        for (int it = ADDS && warp < 8 ? 1 : 0; it < count; it += ADDS ? 2 : 1) {
            const int stage = it % kStages, n = tokens_of(it);
            const uint32_t tile_b = stage * kStage + kB, tile_c = stage * kStage + kC;
            if (!REVERSED && n != weighed) weigh(weighed = n);
            wait_stage(kFull, it);
            if (n < kL) {   // (uniform) behind the sequence anything may stand
#pragma unroll 1
                for (int i = lane; i < 64 * 4; i += 32) {
                    const int t = token0 + i / 4;
                    if (t < n) continue;
                    sts16(base + tile_b + piece(t, quarter * 4 + i % 4), make_uint4(0u, 0u, 0u, 0u));
                    sts16(base + tile_c + piece(t, quarter * 4 + i % 4), make_uint4(0u, 0u, 0u, 0u));
                }
                __syncwarp();
            }
#pragma unroll 1
            for (int side = 0; side < 2; ++side) {   // sixteen columns (lanes) at a time
                // sixteen tokens: matrices (tokens, columns), (tokens, columns + 8), (tokens + 8, ..), (tokens + 8, .. + 8)
                const uint32_t src = base + tile_c + piece(token0 + (lane & 7) + (lane >> 4) * 8, quarter * 4 + side * 2 + (lane >> 3 & 1));
                uint32_t in[4][4];
                do {
                    uint32_t not_finite = 0;   // sign bits: an exponent of ones in the low or the high half of a word
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ldsm4_t(in[i], src + i * 16 * 128);   // (sixteen rows on, the swizzle is the same)
#pragma unroll
                        for (int e = 0; e < 4; ++e) not_finite |= ((in[i][e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                    }
                    if (!__any_sync(0xffffffffu, not_finite != 0)) break;
                    for (int t = token0 + lane; t < token0 + 64; t += 32)
                        take_out(smem + tile_c, t, quarter * 4 + side * 2, bad_from + stage * kN, it * kL, REVERSED);
                    bad_chunk[stage] = it;
                    __syncwarp();
                } while (true);
                uint32_t hi[2][8], mid[2][8], lo[2][8];   // of 32 tokens each
#pragma unroll
                for (int i = 0; i < 8; ++i) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = i % 4 * 2 + e;
                        float2 x = __fmul2_rn(unpack2(in[i / 2][i % 2 * 2 + e]), w[i]);
                        hi[i / 4][r] = pack2_finite(x);
                        x = sub2(x, unpack2(hi[i / 4][r]));
                        mid[i / 4][r] = pack2_finite(x);
                        lo[i / 4][r] = pack2(sub2(x, unpack2(mid[i / 4][r])));
                    }
                }
                constexpr int kBehind = ADDS ? 2 : 1;
                if (side == 0 && it >= kBehind) {   // the product that reads what is there is done
                    wait_turn(kAddDone, it - kBehind);
                    tc_fence_after();
                }
                const uint32_t at = tmem + t_w<ADDS>(it) + t_lane + ((uint32_t)(side * 16) << 16) + token0 / 2;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    tmem_st_fragments(at + i * 16, hi[i]);
                    tmem_st_fragments(at + 64 + i * 16, mid[i]);
                    tmem_st_fragments(at + 128 + i * 16, lo[i]);
                }
            }
            tmem_st_wait();
            fence_proxy_async();
            tc_fence_before();
            mbar_arrive(bar + kWReady + (it & 1));
        }
    } else if (!ADDS && warp < 8) {
        // ---- P of a chunk, then y
        const int quarter = warp & 3, half = warp >> 2, row = tid & 127, c0 = half * (kN / 2);
        const uint32_t t_lane = (uint32_t)(quarter * 32) << 16;
        for (int it = 0; it < count; ++it) {
            const int n = tokens_of(it);
            {
                // Each warp takes two blocks of 32 columns, the outer one first (see p_operand).
                wait(kPDone, it & 1);
                tc_fence_after();
#pragma unroll 1
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
                            // lane's factors from word 31 - lane on, in the copy where they start on 16 bytes
                            const int shift = (lane + 1) & 3;
                            const float4 *factor = reinterpret_cast<const float4 *>(diag + shift * kDiagWords + 31 - lane + shift);
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 g = factor[e / 4];
                                const float2 x = __fmul2_rn(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), make_float2(g.x, g.y));
                                const float2 z = __fmul2_rn(make_float2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), make_float2(g.z, g.w));
                                auto seen = [&](int j, float r) { return (REVERSED ? j >= lane : j <= lane) ? r : 0.f; };   // (whatever was there)
                                out[e / 2] = pack_bf2(seen(e, x.x), seen(e + 1, x.y));
                                out[e / 2 + 1] = pack_bf2(seen(e + 2, z.x), seen(e + 3, z.y));
                            }
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
            // Y2 is there before Y1: it is read, and given its decay, while P C is on its way; once Y1 is read, the next P may be.
            const uint32_t tile_c = it % kStages * kStage + kC;
            const float f = dec[REVERSED ? max(n - 1 - row, 0) : row + 1];
            float2 y[kN / 4];
            wait_stage(kFreeA, it);
            tc_fence_after();
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                uint32_t u[16];
                tmem_ld16(tmem + kY2 + t_lane + c0 + part * 16, u);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    y[part * 8 + e] = __fmul2_rn(make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1])), make_float2(f, f));
            }
            wait(kYDone, it & 1);
            tc_fence_after();
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                uint32_t v[16];
                tmem_ld16(tmem + kY1 + t_lane + c0 + part * 16, v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    y[part * 8 + e] = __fadd2_rn(y[part * 8 + e], make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])));
            }
            tc_fence_before();
            mbar_arrive(bar + kYRead);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = row < n ? pack2(y[q * 4 + e]) : 0u;
                sts16(base + tile_c + piece(row, half * 4 + q), make_uint4(u[0], u[1], u[2], u[3]));
            }
            if (bad_chunk[it % kStages] == it && row < n) put_nan(smem + tile_c, row, half, bad_from + it % kStages * kN, it * kL, REVERSED);
            fence_proxy_async();
            mbar_arrive(bar + kYStored + it % kStages);
        }
        const int from = begin + count * kL;   // chunks behind the sequence
        for (int64_t i = tid; ok && i < (int64_t)(end - from) * 8; i += kGroup)
            *reinterpret_cast<uint4 *>(p.y + (((int64_t)bi * p.T + from + i / 8) * p.H + h) * kN + i % 8 * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncwarp();
    if (!ok) atomicExch(p.status, (int)kDevTimeout);
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
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

// A chunk takes a CTA about 6.5 us whatever it holds, one CTA an SM; the other kernel's blocks of sixteen tokens share the SMs.  Prompts of 17, 32
// and 48 tokens, this kernel and the other: 128 chains 8.6, 8.5, 7.5 and 9.5, 13.5, 20.4 us; 384 chains 20.1, 20.3, 20.7 and 12.3, 17.9, 22.1 (of 40);
// 768 chains 37.7, 37.5, 37.9 and 17.6, 25.9, 36.6.
bool linear_attention_chunks_supported(const LinearAttentionPass &p) {
    return p.bf16 && p.N == kN && (p.T >= 48 || (p.T > linear_attention_plan::kBlock && p.B * p.H <= p.num_sms));
}

size_t linear_attention_chunks_workspace_bytes(const LinearAttentionPass &p) {
    using namespace linear_attention_plan;
    const int64_t chains = p.B * p.H;
    return state_bytes(chains, cut(chains, (p.T + kL - 1) / kL, (int64_t)p.num_sms, kChunksOfLaunches, INT64_MAX).segments, kN);
}

int launch_linear_attention_chunks(const LinearAttentionPass &p, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    using namespace linear_attention_plan;
    const int64_t chains = p.B * p.H;
    const Cut c = cut(chains, (p.T + kL - 1) / kL, (int64_t)p.num_sms, kChunksOfLaunches, workspace == nullptr ? 1 : segments_in(workspace_bytes, chains, kN));
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
