// Backward pass of the router: gradients of the routing weights (and, where
// given, of the logits) carried to the tokens and to the router weight.  No
// counterpart in the reference, whose block is forward-only.
//
//   ds[t,k] = w[t,k] (gw[t,k] - sum_j w[t,j] gw[t,j])      softmax over the selected scores
//   d       = grad_logits + scatter of ds to the ids        [T, E], fp32
//   dx      = d W  [T, H], rounded once to bf16             dW = d^T x  [E, H], fp32
//
// Both products are 2 T E H flop of fp32 data.  The tensor cores take bf16, so
// every fp32 operand is split into bf16 parts whose sum is the value: hi =
// bf16(v), mid = bf16(v - hi), lo = bf16(v - hi - mid), each within half a step
// (2^-8) of the rest, so hi + mid + lo is v to 2^-24.  x is bf16 already.  dW
// takes all three parts of d.  dx takes the six products whose parts' ranks add up
// to hi lo or less: what is left out (mid lo, lo mid, lo lo) is 2^-23 |d W|, as much as
// the two splits are off, so dx is an fp32 product before its one rounding to bf16.
// (Three products, without mid mid, hi lo and lo hi, are 2^-16 |d W| off; at 32768 tokens,
// 256 experts, hidden 7168 the splits and dx then take 256 us and not 434.)
//
//   split_kernel           d's parts, [T, 3 E8] bf16 with columns lo | mid | hi (E8: E
//                          rounded up to 8), and W^T's parts,
//                          [H, 3 E8] bf16 with columns hi | mid | lo
//   router_dx_kernel       dx: tcgen05 on CTA pairs, K = E, six MMAs per 16 experts
//   router_dw_kernel, router_dw_pair_kernel  dW: tcgen05 over tokens as K, both
//                          operands MN-major; up to 80 experts, and above
//   add_parts_kernel       adds the token ranges' partial sums in order
//
// Up to kFewExperts experts one kernel does both products from the same parts and reads
// x once (router_few_kernel).
//
// Bound: for few experts by x and dx through memory; for 256 experts by the tensor
// cores (dx six bf16 products per fp32 multiply-add, dW three).
#include "common.cuh"
#include "launch.h"
#include "tcgen05.cuh"

namespace moe {

// gemm_sm100.cu: [rows, cols] bf16 whose rows lie `stride` elements apart (0: cols), in
// boxes of box_rows x 64 columns, 128-byte swizzle.
bool encode_bf16_tensor_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols,
                            uint64_t stride, uint32_t box_rows);

namespace {

__device__ int32_t g_route_backward_status;
constexpr int32_t kStatusRouterBackwardWait = 7;
constexpr uint64_t kWaitLimitNs = 4000000000ull;
constexpr uint64_t kDrainLimitNs = 200000000ull;

// ------------------------------------------------------------------- splits

__device__ __forceinline__ uint32_t bf16_part(float& rest) {
    const __nv_bfloat16 h = __float2bfloat16_rn(rest);
    rest -= __bfloat162float(h);
    return __bfloat16_as_ushort(h);
}

// d's parts of every token.  LANES lanes share a token, eight neighbouring experts each:
// two 16-byte loads of grad_logits (`wide`: rows and pointer on 16 bytes) and a 16-byte
// store per part.  The scatter goes through a row in shared memory, one lane per
// selected expert; where ids repeat they add one after the other, in order.
template <int LANES>
__device__ void split_gradient(const float* __restrict__ grad_logits, const int32_t* __restrict__ ids,
                               const float* __restrict__ weights, const float* __restrict__ grad_weights,
                               __nv_bfloat16* __restrict__ parts, int64_t tokens, int experts, int padded, int topk,
                               bool wide, int block, int blocks) {
    constexpr int kTokens = 32 / LANES;  // per warp
    __shared__ __align__(16) float rows[8][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LANES - 1);
    const int slot = (threadIdx.x & 31) / LANES;
    float* row = rows[warp] + slot * (LANES * 8);
    const int e0 = lane * 8;
    const int64_t stride = static_cast<int64_t>(blocks) * 8 * kTokens;
    for (int64_t first = (block * 8ll + warp) * kTokens; first < tokens; first += stride) {  // same for the warp
        const int64_t t = first + slot;
        const bool live = t < tokens;
        float d[8] = {};
        if (grad_logits && live && e0 < experts) {
            const float* from = grad_logits + t * experts + e0;
            if (wide) {
                const float4 v = *reinterpret_cast<const float4*>(from);
                d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
                if (e0 + 4 < experts) {
                    const float4 u = *reinterpret_cast<const float4*>(from + 4);
                    d[4] = u.x, d[5] = u.y, d[6] = u.z, d[7] = u.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (e0 + j < experts) d[j] = from[j];
            }
        }
        int id = -1;
        float w = 0.0f, g = 0.0f;
        if (live && lane < topk) {
            id = ids[t * topk + lane];
            w = weights[t * topk + lane];
            g = grad_weights[t * topk + lane];
        }
        float dot = w * g;
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
        const float ds = w * (g - dot);
        *reinterpret_cast<float4*>(row + e0) = make_float4(d[0], d[1], d[2], d[3]);
        *reinterpret_cast<float4*>(row + e0 + 4) = make_float4(d[4], d[5], d[6], d[7]);
        const bool mine = id >= 0 && id < experts;
        // one key per expert of this token; lanes without one differ from all others
        const int key = mine ? slot << 16 | id : -1 - static_cast<int>(threadIdx.x & 31);
        const unsigned same = __match_any_sync(0xffffffffu, key);
        if (__any_sync(0xffffffffu, __popc(same) > 1)) {
            for (int k = 0; k < topk; ++k) {
                __syncwarp();
                if (mine && lane == k) row[id] += ds;
            }
        } else {
            __syncwarp();
            if (mine) row[id] += ds;
        }
        __syncwarp();
        const float4 v = *reinterpret_cast<const float4*>(row + e0);
        const float4 u = *reinterpret_cast<const float4*>(row + e0 + 4);
        __syncwarp();  // read before the next token's row is written
        d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
        d[4] = u.x, d[5] = u.y, d[6] = u.z, d[7] = u.w;
        if (live && e0 < padded) {
            __nv_bfloat16* to = parts + t * 3 * padded + e0;
#pragma unroll
            for (int part = 2; part >= 0; --part) {  // hi, mid, lo
                uint32_t piece[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 both = __floats2bfloat162_rn(d[2 * j], d[2 * j + 1]);
                    piece[j] = *reinterpret_cast<const uint32_t*>(&both);
                    d[2 * j] -= __uint_as_float(piece[j] << 16);
                    d[2 * j + 1] -= __uint_as_float(piece[j] & 0xffff0000u);
                }
                *reinterpret_cast<uint4*>(to + part * padded) = make_uint4(piece[0], piece[1], piece[2], piece[3]);
            }
        }
    }
}

// W [E, H] fp32 -> [H, 3 E8] bf16: one 32 x 32 tile through shared memory.
__device__ void split_weight(const float* __restrict__ weight, __nv_bfloat16* __restrict__ out, int experts,
                             int padded, int64_t hidden, int64_t h0, int e0) {
    __shared__ float tile[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int i = y; i < 32; i += 8)
        tile[i][x] = e0 + i < experts && h0 + x < hidden ? weight[(e0 + i) * hidden + h0 + x] : 0.0f;
    __syncthreads();
    if (e0 + x >= padded) return;
    for (int i = y; i < 32; i += 8) {
        if (h0 + i >= hidden) break;
        float v = tile[x][i];
        __nv_bfloat16* row = out + (h0 + i) * 3 * padded + e0 + x;
#pragma unroll
        for (int part = 0; part < 3; ++part) row[part * padded] = __ushort_as_bfloat16(static_cast<unsigned short>(bf16_part(v)));
    }
}

// Both splits in one launch: the first CTAs take a tile of W each (none without dx),
// the others d.
template <int LANES>
__global__ void __launch_bounds__(256)
split_kernel(const float* __restrict__ weight, __nv_bfloat16* __restrict__ weight_parts, int64_t hidden,
             int tiles_h, int tiles,
             const float* __restrict__ grad_logits, const int32_t* __restrict__ ids,
             const float* __restrict__ weights, const float* __restrict__ grad_weights,
             __nv_bfloat16* __restrict__ parts, int64_t tokens, int experts, int padded, int topk, bool wide) {
    pdl_trigger();
    pdl_wait();
    const int block = blockIdx.x;
    if (block < tiles) {
        split_weight(weight, weight_parts, experts, padded, hidden, block % tiles_h * 32ll, block / tiles_h * 32);
    } else {
        split_gradient<LANES>(grad_logits, ids, weights, grad_weights, parts, tokens, experts, padded, topk, wide,
                              block - tiles, gridDim.x - tiles);
    }
}

// ----------------------------------------------------------------------- dW

constexpr int kTileH = 128;   // rows of dW^T per CTA (M)
// Tokens per pipeline stage (K).  With 32 twice as many tile copies bring the same bytes,
// and their number counts: 26 us against 20 at 64 experts, 283 against 238 at 256.
constexpr int kTileT = 64;
constexpr int kBlock = kTileT * 128;  // bytes of 64 columns x kTileT tokens
constexpr int kMaxStages = 8;
constexpr int kDwThreads = 192;  // producer, issuer, four epilogue warps
// The tensor cores cut the sum of 16 products and the accumulator off below its last
// bit, so long sums drift: with 500 MMAs into one accumulator dW of 32768 tokens, 256
// experts was 6.7e-6 of its norm off, where plain fp32 products are 5.8e-7 off.  So in
// every dW kernel an accumulator takes kChunk tokens (16 MMAs per part of d), and is then
// added to an fp32 sum, rounded to nearest.
constexpr int kChunk = 256;
constexpr int kChunkSteps = kChunk / kTileT;
constexpr int kDwSmem = 224 * 1024;

struct DwParams {
    float* out;           // dW [E, H], or the partial sums [ranges, E, H]
    int64_t hidden;
    int tokens, experts, padded;
    int range;            // tokens per CTA or CTA pair (a multiple of kTileT)
    int n;                // MMA N
    int blocks;           // 64-column boxes of d per stage (pair: per part and CTA)
    int stages;
};

// Up to this many (padded) experts d's parts fit side by side into one MMA.
constexpr int kSideBySide = 80;
constexpr int kSideBySide32 = (kSideBySide + 31) / 32 * 32;  // read 32 columns at a time
static_assert(2 * kSideBySide + kSideBySide32 <= 256, "the last part's columns lie in its accumulator");

__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                             uint64_t limit) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t start = global_timer();
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 31) == 0) {
            if (*abort_flag) return false;
            if (global_timer() - start > limit) {
                atomicCAS(&g_route_backward_status, 0, kStatusRouterBackwardWait);
                *abort_flag = 1;
                return false;
            }
        }
    }
}

// MN-major operand, 128-byte swizzle: 64 columns x tokens as rows of 128 bytes;
// 8-token groups 1024 bytes apart (stride offset), 64-column blocks kBlock apart
// (leading offset).
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kBlock >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
           (static_cast<uint64_t>(2) << 61);
}

// dW^T tile [128 h, E] of one range of tokens, up to 80 experts.  Warp 0 loads x
// [64 tokens, 128] and d's parts by TMA, warp 1 issues the MMAs (M = 128, K = 16),
// warps 2-5 add the accumulators into registers (two accumulators in turn, 256 columns of
// tensor memory each; a thread has all experts of one row) and store the tile.  The three
// parts stand side by side in N (3 E8 <= 240): one MMA per 16 tokens, and the epilogue
// adds the three column groups.  Ranges are added in a launch of their own.
__global__ void __launch_bounds__(kDwThreads, 1)
router_dw_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_d,
                 const DwParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h0 = blockIdx.x * kTileH;
    const int t0 = blockIdx.y * p.range;
    const int t1 = min(t0 + p.range, p.tokens);
    const int steps = (t1 - t0 + kTileT - 1) / kTileT;  // >= 1
    const int chunks = (steps + kChunkSteps - 1) / kChunkSteps;
    const int stage_bytes = (2 + p.blocks) * kBlock;

    pdl_trigger();
    if (warp == 0 && lane == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], kDwThreads - 64);  // the epilogue's threads
        }
        mbar_init(&drain, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0 && lane == 0) {
        int stage = 0;
        uint32_t phase = 0, armed = 0, parity = 0;
        for (int i = 0; i < steps; ++i) {
            if (!wait_bounded(&empty[stage], phase ^ 1u, &abort_flag, kWaitLimitNs)) break;
            uint8_t* at = tiles + stage * stage_bytes;
            const int t = t0 + i * kTileT;
            mbar_expect_tx(&full[stage], stage_bytes);
            tma_load_2d(at, &map_x, &full[stage], h0, t);
            tma_load_2d(at + kBlock, &map_x, &full[stage], h0 + 64, t);
            at += 2 * kBlock;
            for (int b = 0; b < p.blocks; ++b, at += kBlock)
                tma_load_2d(at, &map_d, &full[stage], b * 64, t);
            armed |= 1u << stage;
            parity = (parity & ~(1u << stage)) | (phase << stage);
            if (++stage == p.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (abort_flag) {  // every copy in flight lands before the CTA exits
            volatile int never = 0;
            for (int s = 0; s < p.stages; ++s)
                if (armed & (1u << s)) wait_bounded(&full[s], (parity >> s) & 1u, &never, kDrainLimitNs);
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t idesc = make_idesc(kTileH, p.n) | (1u << 15) | (1u << 16);  // both MN-major
        int stage = 0;
        uint32_t phase = 0;
        bool issued = false, ok = true;
        for (int chunk = 0; chunk < chunks && ok; ++chunk) {
            const int acc = chunk & 1;
            if (!wait_bounded(&acc_empty[acc], ((chunk >> 1) & 1) ^ 1u, &abort_flag, kWaitLimitNs)) break;
            tc_fence_after();
            const int here = min(kChunkSteps, steps - chunk * kChunkSteps);
            for (int i = 0; i < here; ++i) {
                if (!wait_bounded(&full[stage], phase, &abort_flag, kWaitLimitNs)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t x_at = smem_u32(tiles + stage * stage_bytes);
                const uint32_t d_at = x_at + 2 * kBlock;
                for (int k = 0; k < kTileT / 16; ++k)
                    umma_bf16(tmem + acc * 256, mn_desc(x_at + k * 2048), mn_desc(d_at + k * 2048), idesc,
                              (i | k) != 0 ? 1u : 0u);
                issued = true;
                umma_commit(&empty[stage]);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok) umma_commit(&acc_full[acc]);
        }
        if (issued) {  // no MMA outlives this wait, whatever the epilogue does
            umma_commit(&drain);
            volatile int never = 0;
            wait_bounded(&drain, 0, &never, kWaitLimitNs);
        }
    } else if (warp >= 2) {
        // TMEM lane = row of the tile (h), column = expert: a warp stores 32 neighbours of one
        // expert's row.  Lanes past H (only in the last tile) store nothing.
        const int quarter = warp & 3;
        const int64_t h = h0 + quarter * 32 + lane;
        const uint32_t row = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        float sum[kSideBySide32];
#pragma unroll
        for (int j = 0; j < kSideBySide32; ++j) sum[j] = 0.0f;
        bool ok = true;
        for (int chunk = 0; chunk < chunks; ++chunk) {
            const int acc = chunk & 1;
            if (!wait_bounded(&acc_full[acc], (chunk >> 1) & 1, &abort_flag, kWaitLimitNs)) {
                ok = false;
                break;
            }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < kSideBySide32; c += 32) {
                if (c < p.experts) {
                    uint32_t v[3][32];
#pragma unroll
                    for (int s = 0; s < 3; ++s) tmem_ld32(row + acc * 256 + s * p.padded + c, v[s]);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; ++j)  // the small parts first: lo + mid + hi
                        sum[c + j] += (__uint_as_float(v[0][j]) + __uint_as_float(v[1][j])) + __uint_as_float(v[2][j]);
                }
            }
            tc_fence_before();
            mbar_arrive(&acc_empty[acc]);
        }
        if (ok && h < p.hidden) {
            float* out = p.out + static_cast<int64_t>(blockIdx.y) * p.experts * p.hidden + h;
#pragma unroll
            for (int j = 0; j < kSideBySide32; ++j)
                if (j < p.experts) out[j * p.hidden] = sum[j];
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// dW^T tile [256 h, E] of one range of tokens on a CTA pair (cta_group::2), more
// than 80 experts: each CTA loads its 128 columns of x and its half of every part's
// E columns, the even CTA issues M = 256, N up to 256, one MMA per part and 16
// tokens.  (One CTA with M = 128 needs 112 KB per 64 tokens and SM instead of 64: 451 us
// at 32768 tokens, 256 experts, hidden 7168 against 283 for the pair, both with stages of
// 32 tokens.)
// While an accumulator takes its kChunk tokens (48 MMAs) the epilogue warps add the
// one before into fp32 registers, 128 columns of one row per thread (7.4e-7 of dW's norm).
constexpr int kPairThreads = 320;  // producer, issuer, eight epilogue warps
constexpr int kPairStages = 3;

__device__ __forceinline__ bool wait_bounded_cluster(uint64_t* bar, uint32_t parity,
                                                     volatile int* abort_flag, uint64_t limit) {
    const uint64_t start = global_timer();
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait_cluster(bar, parity)) return true;
        if ((i & 31) == 0) {
            if (*abort_flag) return false;
            if (global_timer() - start > limit) {
                atomicCAS(&g_route_backward_status, 0, kStatusRouterBackwardWait);
                *abort_flag = 1;
                return false;
            }
        }
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
router_dw_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_d,
                      const DwParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int h0 = blockIdx.x * kTileH;  // the pair's tile: 256 columns of x from the even CTA's on
    const int t0 = blockIdx.y * p.range;
    const int t1 = min(t0 + p.range, p.tokens);
    const int steps = (t1 - t0 + kTileT - 1) / kTileT;  // >= 1
    const int chunks = (steps + kChunkSteps - 1) / kChunkSteps;
    const int stage_bytes = (2 + 3 * p.blocks) * kBlock;  // of one CTA

    pdl_trigger();
    if (warp == 0 && lane == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], 2 * (kPairThreads - 64));  // both CTAs' epilogue threads
        }
        mbar_init(&drain, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are set up
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0 && lane == 0) {
        int stage = 0;
        uint32_t phase = 0, armed = 0, parity = 0;
        for (int i = 0; i < steps; ++i) {
            if (!wait_bounded(&empty[stage], phase ^ 1u, &abort_flag, kWaitLimitNs)) break;
            uint8_t* at = tiles + stage * stage_bytes;
            const int t = t0 + i * kTileT;
            const uint32_t leader_full = map_to_cta(smem_u32(&full[stage]), 0);
            if (leader) mbar_expect_tx(&full[stage], 2 * stage_bytes);
            tma_load_2d_pair(at, &map_x, leader_full, h0, t);
            tma_load_2d_pair(at + kBlock, &map_x, leader_full, h0 + 64, t);
            at += 2 * kBlock;
            for (int s = 0; s < 3; ++s)
                for (int b = 0; b < p.blocks; ++b, at += kBlock)
                    tma_load_2d_pair(at, &map_d, leader_full, s * p.padded + rank * (p.n / 2) + b * 64, t);
            armed |= 1u << stage;
            parity = (parity & ~(1u << stage)) | (phase << stage);
            if (++stage == kPairStages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (abort_flag && leader) {  // every copy in flight lands before the pair exits
            volatile int never = 0;
            for (int s = 0; s < kPairStages; ++s)
                if (armed & (1u << s)) wait_bounded(&full[s], (parity >> s) & 1u, &never, kDrainLimitNs);
        }
    } else if (warp == 1 && lane == 0 && leader) {
        const uint32_t idesc = make_idesc(2 * kTileH, p.n) | (1u << 15) | (1u << 16);  // both MN-major
        int stage = 0;
        uint32_t phase = 0;
        bool issued = false, ok = true;
        for (int chunk = 0; chunk < chunks && ok; ++chunk) {
            const int acc = chunk & 1;
            if (!wait_bounded_cluster(&acc_empty[acc], ((chunk >> 1) & 1) ^ 1u, &abort_flag, kWaitLimitNs)) break;
            tc_fence_after();
            const int here = min(kChunkSteps, steps - chunk * kChunkSteps);
            for (int i = 0; i < here; ++i) {
                if (!wait_bounded(&full[stage], phase, &abort_flag, kWaitLimitNs)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t x_at = smem_u32(tiles + stage * stage_bytes);
                const uint32_t d_at = x_at + 2 * kBlock;
                for (int k = 0; k < kTileT / 16; ++k)
                    for (int s = 0; s < 3; ++s)
                        umma_bf16_pair(tmem + acc * 256, mn_desc(x_at + k * 2048),
                                       mn_desc(d_at + s * p.blocks * kBlock + k * 2048), idesc,
                                       (i | k | s) != 0 ? 1u : 0u);
                issued = true;
                umma_commit_pair(&empty[stage]);
                if (++stage == kPairStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok) umma_commit_pair(&acc_full[acc]);
        }
        if (issued) {  // no MMA outlives this wait, whatever the epilogue does
            umma_commit_pair(&drain);
            volatile int never = 0;
            wait_bounded(&drain, 0, &never, kWaitLimitNs);
        }
    } else if (warp >= 2) {
        // TMEM lane = row of the tile (h), column = expert: each warp takes half of the columns
        // of 32 rows, and stores 32 neighbours of one expert's row at a time
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t row = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * (p.n / 2);
        const uint32_t leader_empty0 = map_to_cta(smem_u32(&acc_empty[0]), 0);
        const uint32_t leader_empty1 = map_to_cta(smem_u32(&acc_empty[1]), 0);
        float sum[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) sum[j] = 0.0f;
        bool ok = true;
        for (int chunk = 0; chunk < chunks; ++chunk) {
            const int acc = chunk & 1;
            if (!wait_bounded(&acc_full[acc], (chunk >> 1) & 1, &abort_flag, kWaitLimitNs)) {
                ok = false;
                break;
            }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 128; c += 32) {
                if (c < p.n / 2) {
                    uint32_t v[32];
                    tmem_ld32(row + acc * 256 + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[c + j] += __uint_as_float(v[j]);
                }
            }
            tc_fence_before();
            mbar_arrive_cluster(acc ? leader_empty1 : leader_empty0);
        }
        const int64_t h = h0 + quarter * 32 + lane;
        if (ok && h < p.hidden) {
            const int e0 = half * (p.n / 2);
            float* out = p.out + (static_cast<int64_t>(blockIdx.y) * p.experts + e0) * p.hidden + h;
            const int mine = min(p.n / 2, p.experts - e0);
#pragma unroll
            for (int j = 0; j < 128; ++j)
                if (j < mine) out[j * p.hidden] = sum[j];
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while its peer may still touch its memory
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ----------------------------------------------------------------------- dx

// dx tile [256 tokens, 256 h] on a CTA pair: each CTA loads the three parts of its 128
// tokens' d and of its 128 rows of W^T, 64 experts at a time (a tensor map per part, so
// that columns past E8 are zeros and not the next part's), the even CTA issues the six
// products, M = 256, N = 256, the small ones of all 64 experts first: what an MMA cuts off
// goes by the sum that it finds.
// The epilogue warps turn 32 tokens x 64 columns at a time into bf16 in shared memory
// and store them as a tile while the next accumulator fills.
// With the splits before it 434 us at 32768 tokens, 256 experts, hidden 7168 (1.7
// PFLOP/s of bf16 products: bound by the tensor cores), and 32 at 16384 tokens, 64
// experts, hidden 2048 (the epilogue and its stores).
constexpr int kDxTile = 128;                        // tokens, and rows of W^T, of a CTA
constexpr int kDxPart = kDxTile * 128;              // bytes of one part's 64 columns
constexpr int kDxStageBytes = 6 * kDxPart;
constexpr int kDxStages = 2;
constexpr int kDxThreads = 320;                     // producer, issuer, eight epilogue warps
constexpr int kDxStaging = 32 * 128;                // bytes per epilogue warp
constexpr int kDxSmem = kDxStages * kDxStageBytes + 8 * kDxStaging + 1024;
constexpr int kDxProducts = 6;

struct DxMaps {
    CUtensorMap d[3], w[3];  // lo, mid, hi of d; hi, mid, lo of W^T
    CUtensorMap out;
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kDxThreads, 1)
router_dx_kernel(const __grid_constant__ DxMaps maps, int tokens, int64_t hidden, int padded) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[kDxStages], empty[kDxStages], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int k_blocks = (padded + 63) / 64;
    const int tiles_h = static_cast<int>((hidden + 2 * kDxTile - 1) / (2 * kDxTile));
    const int all = (tokens + 2 * kDxTile - 1) / (2 * kDxTile) * tiles_h;
    const int first = blockIdx.x / 2, stride = gridDim.x / 2;

    pdl_trigger();
    if (warp == 0 && lane == 0) {
        for (int s = 0; s < kDxStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], 2 * (kDxThreads - 64));  // both CTAs' epilogue threads
        }
        mbar_init(&drain, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are set up
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0 && lane == 0) {
        int stage = 0;
        uint32_t phase = 0, armed = 0, parity = 0;
        bool ok = true;
        for (int tile = first; tile < all && ok; tile += stride) {
            const int t = tile / tiles_h * (2 * kDxTile) + static_cast<int>(rank) * kDxTile;
            const int h = tile % tiles_h * (2 * kDxTile) + static_cast<int>(rank) * kDxTile;
            for (int kb = 0; kb < k_blocks; ++kb) {
                if (!wait_bounded(&empty[stage], phase ^ 1u, &abort_flag, kWaitLimitNs)) {
                    ok = false;
                    break;
                }
                uint8_t* at = tiles + stage * kDxStageBytes;
                const uint32_t leader_full = map_to_cta(smem_u32(&full[stage]), 0);
                if (leader) mbar_expect_tx(&full[stage], 2 * kDxStageBytes);
                for (int part = 0; part < 3; ++part) {  // lo and W's hi first: the first product's
                    tma_load_2d_pair(at + part * kDxPart, &maps.d[part], leader_full, kb * 64, t);
                    tma_load_2d_pair(at + (3 + part) * kDxPart, &maps.w[part], leader_full, kb * 64, h);
                }
                armed |= 1u << stage;
                parity = (parity & ~(1u << stage)) | (phase << stage);
                if (++stage == kDxStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        if (abort_flag && leader) {  // every copy in flight lands before the pair exits
            volatile int never = 0;
            for (int s = 0; s < kDxStages; ++s)
                if (armed & (1u << s)) wait_bounded(&full[s], (parity >> s) & 1u, &never, kDrainLimitNs);
        }
    } else if (warp == 1 && lane == 0 && leader) {
        constexpr uint32_t idesc = make_idesc(2 * kDxTile, 2 * kDxTile);
        int stage = 0, local = 0;
        uint32_t phase = 0;
        bool issued = false, ok = true;
        for (int tile = first; tile < all && ok; tile += stride, ++local) {
            const int acc = local & 1;
            if (!wait_bounded_cluster(&acc_empty[acc], ((local >> 1) & 1) ^ 1u, &abort_flag, kWaitLimitNs)) break;
            tc_fence_after();
            for (int kb = 0; kb < k_blocks; ++kb) {
                if (!wait_bounded(&full[stage], phase, &abort_flag, kWaitLimitNs)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d_at = smem_u32(tiles + stage * kDxStageBytes);
                const uint32_t w_at = d_at + 3 * kDxPart;
                const int steps = (min(64, padded - kb * 64) + 15) / 16;  // the rest is zeros
                // product q: d's part (lo, mid, hi: 0, 1, 2) and W's (hi, mid, lo: 0, 1, 2)
                constexpr int kOfD[kDxProducts] = {0, 1, 2, 1, 2, 2};
                constexpr int kOfW[kDxProducts] = {0, 1, 2, 0, 1, 0};
#pragma unroll
                for (int q = 0; q < kDxProducts; ++q)
                    for (int k = 0; k < steps; ++k)
                        umma_bf16_pair(tmem + acc * 256, smem_desc_sw128(d_at + kOfD[q] * kDxPart + k * 32),
                                       smem_desc_sw128(w_at + kOfW[q] * kDxPart + k * 32), idesc,
                                       (kb | q | k) != 0 ? 1u : 0u);
                issued = true;
                umma_commit_pair(&empty[stage]);
                if (++stage == kDxStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok) umma_commit_pair(&acc_full[acc]);
        }
        if (issued) {  // no MMA outlives this wait, whatever the epilogue does
            umma_commit_pair(&drain);
            volatile int never = 0;
            wait_bounded(&drain, 0, &never, kWaitLimitNs);
        }
    } else if (warp >= 2) {
        // TMEM lane = token; each warp takes 32 tokens and half of the columns, 64 at a time
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint8_t* staging = tiles + kDxStages * kDxStageBytes + (warp - 2) * kDxStaging;
        const uint32_t staged = smem_u32(staging);
        const uint32_t row = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
        const uint32_t leader_empty0 = map_to_cta(smem_u32(&acc_empty[0]), 0);
        const uint32_t leader_empty1 = map_to_cta(smem_u32(&acc_empty[1]), 0);
        int local = 0;
        for (int tile = first; tile < all; tile += stride, ++local) {
            const int acc = local & 1;
            const int t = tile / tiles_h * (2 * kDxTile) + static_cast<int>(rank) * kDxTile + quarter * 32;
            const int h = tile % tiles_h * (2 * kDxTile) + half * 128;
            if (!wait_bounded(&acc_full[acc], (local >> 1) & 1, &abort_flag, kWaitLimitNs)) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 128; c += 64) {
                uint32_t v[2][32];
                tmem_ld32(row + acc * 256 + c, v[0]);
                tmem_ld32(row + acc * 256 + c + 32, v[1]);
                tmem_wait_ld();
                if (c == 64) {  // the accumulator has been read
                    tc_fence_before();
                    mbar_arrive_cluster(acc ? leader_empty1 : leader_empty0);
                }
                // the tile stored before has left the staging
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 8; ++q) {  // 16-byte piece q of this token's 128, swizzled
                    uint32_t piece[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        piece[j] = pack_bf16x2(__uint_as_float(v[q / 4][q % 4 * 8 + 2 * j]),
                                               __uint_as_float(v[q / 4][q % 4 * 8 + 2 * j + 1]));
                    *reinterpret_cast<uint4*>(staging + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                        make_uint4(piece[0], piece[1], piece[2], piece[3]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0 && t < tokens && h + c < hidden) {
                    tma_store_2d(&maps.out, staged, h + c, t);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while its peer may still touch its memory
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ------------------------------------------------------------- few experts

// Both products at once for up to EP (8 or 16) experts, bound by x and dx through
// memory: x is read once, by mma.sync (tcgen05 tiles of 128 rows would be 7/8 empty).
// A CTA has 512 columns of hidden and a range of tokens, a warp 64 of the columns.  The
// warp copies its part of 16 tokens at a time into a ring in shared memory, makes dW
// from it (M = the parts of d^T, K = tokens, N = columns), and dx (M = tokens, K = the
// parts of d, N = columns, against W's parts in registers), which takes x's place in
// the ring on its way out.  d's parts are made for 256 tokens at a time, a row of
// hi | mid | lo per token; the one layout serves both products, transposed and not.
// The sums hi and mid + lo of dW are kept apart; after every batch of d (256 tokens at most,
// see kChunk) they are added to this CTA's fp32 sums in memory, each by the thread that
// wrote it before, and start again from zero.
// (21 us with the ranges' sum at 4096 tokens, 8 experts, hidden 4096, 28 with 16 experts;
// for 8, fp32 multiply-adds on the CUDA cores, two lanes an instruction, took 7 us more,
// the split products of more experts 19 more.)
constexpr int kFewExperts = 16;
constexpr int kFewThreads = 256;
constexpr int kFewCols = 512;     // of a CTA
constexpr int kFewWarpCols = kFewCols / (kFewThreads / 32);
constexpr int kFewTile = 16;      // tokens
constexpr int kFewStages = 3;
constexpr int kFewRow = kFewWarpCols * 2 + 16;  // bytes of a token in a warp's ring; the pad spreads the banks
constexpr int kFewStage = kFewTile * kFewRow;
template <int EP> constexpr int few_d_row() { return 3 * EP * 2 + (EP == 8 ? 32 : 16); }  // 80 or 112: likewise
template <int EP> constexpr int few_tokens() { return EP == 8 ? 256 : 224; }  // of d at a time (224: two CTAs fit an SM)
static_assert(few_tokens<8>() <= kChunk && few_tokens<16>() <= kChunk, "dW's accumulators are emptied after each");
// mid and lo of W's fragments wait in shared memory: of the 128 registers 16 experts' accumulators take 64
template <int EP> constexpr int few_w_bytes() { return kFewThreads * (kFewWarpCols / 8) * EP; }
template <int EP> constexpr int few_smem() {
    return (kFewThreads / 32) * kFewStages * kFewStage + few_tokens<EP>() * few_d_row<EP>() + few_w_bytes<EP>();
}
static_assert(2 * (few_smem<8>() + 1024) <= 228 * 1024 && 2 * (few_smem<16>() + 1024) <= 228 * 1024, "two CTAs an SM");

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_k16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {  // c = 0 before
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int EP>
__global__ void __launch_bounds__(kFewThreads, 2)
router_few_kernel(const __nv_bfloat16* __restrict__ x, const float* __restrict__ weight,
                  const int32_t* __restrict__ ids, const float* __restrict__ weights,
                  const float* __restrict__ grad_weights, const float* __restrict__ grad_logits,
                  __nv_bfloat16* __restrict__ grad_x, float* __restrict__ sums, int tokens,
                  int64_t hidden, int experts, int topk, int range) {
    constexpr int kFrags = kFewWarpCols / 8;  // n8 fragments of a warp
    extern __shared__ __align__(128) uint8_t few_smem_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = smem_u32(few_smem_raw) + warp * kFewStages * kFewStage;
    uint8_t* d_rows = few_smem_raw + (kFewThreads / 32) * kFewStages * kFewStage;
    const uint32_t d_at = smem_u32(d_rows);
    const int64_t h0 = static_cast<int64_t>(blockIdx.x) * kFewCols + warp * kFewWarpCols;
    const int t0 = blockIdx.y * range, t1 = min(t0 + range, tokens);
    const bool active = h0 < hidden;  // this warp has columns
    pdl_trigger();
    pdl_wait();

    // lane: chunk lane % 8 of tokens lane / 8 + 4 j
    const int chunk = lane & 7, row = lane >> 3;
    const bool in_cols = h0 + chunk * 8 < hidden;
    const uint32_t lane_at = row * kFewRow + chunk * 16;
    const int64_t step = 4 * hidden;
    const __nv_bfloat16* from_x = x + (static_cast<int64_t>(t0) + row) * hidden + h0 + chunk * 8;
    __nv_bfloat16* to_dx = grad_x + (static_cast<int64_t>(t0) + row) * hidden + h0 + chunk * 8;
    int load_t = t0 + row;  // this lane's first token of the next load
    auto load = [&](int slot) {
#pragma unroll
        for (int j = 0; j < kFewTile / 4; ++j) {
            const bool in = in_cols && load_t < t1;
            copy16(ring + slot * kFewStage + lane_at + 4 * j * kFewRow, in ? from_x : x, in);
            from_x += step;
            load_t += 4;
        }
    };
#pragma unroll
    for (int s = 0; s < kFewStages - 1; ++s) {
        if (active && sums) load(s);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // W's parts as B fragments: experts k = 2 (lane % 4) and the next (and 8 further), column lane / 4
    uint32_t w_hi[kFrags][EP / 8];
    struct alignas(EP) Staged { uint32_t mid[EP / 8], lo[EP / 8]; };
    Staged* w_staged = reinterpret_cast<Staged*>(d_rows + few_tokens<EP>() * few_d_row<EP>()) + tid;  // [fragment][thread]
    if (grad_x) {
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
            for (int g = 0; g < EP / 8; ++g) {
                const int e = g * 8 + 2 * (lane & 3);
                const int64_t h = h0 + f * 8 + (lane >> 2);
                float a = h < hidden && e < experts ? weight[e * hidden + h] : 0.0f;
                float b = h < hidden && e + 1 < experts ? weight[(e + 1) * hidden + h] : 0.0f;
                w_hi[f][g] = bf16_part(a) | bf16_part(b) << 16;
                w_staged[f * kFewThreads].mid[g] = bf16_part(a) | bf16_part(b) << 16;
                w_staged[f * kFewThreads].lo[g] = bf16_part(a) | bf16_part(b) << 16;
            }
    }

    // dW: EP = 8: rows 0..7 of the fragment are hi, 8..15 mid and lo; EP = 16: one fragment each
    float acc[kFrags][EP / 8][4] = {};
    int slot = 0, load_slot = kFewStages - 1;
    for (int batch = t0; batch < t1; batch += few_tokens<EP>()) {
        if (batch > t0) __syncthreads();  // d of the batch before has been used
        const int count = min(few_tokens<EP>(), t1 - batch);
        for (int i = tid; i < (count + kFewTile - 1) / kFewTile * kFewTile; i += kFewThreads) {
            float d[EP];
#pragma unroll
            for (int e = 0; e < EP; ++e) d[e] = 0.0f;
            if (i < count) {
                const int64_t t = batch + i;
                float dot = 0.0f;
                for (int k = 0; k < topk; ++k) dot = fmaf(weights[t * topk + k], grad_weights[t * topk + k], dot);
                if (grad_logits) {
#pragma unroll
                    for (int e = 0; e < EP; ++e)
                        if (e < experts) d[e] = grad_logits[t * experts + e];
                }
                for (int k = 0; k < topk; ++k) {  // in order: a repeated id adds the same way every time
                    const int id = ids[t * topk + k];
                    const float v = weights[t * topk + k] * (grad_weights[t * topk + k] - dot);
                    if (id >= experts) continue;
#pragma unroll
                    for (int e = 0; e < EP; ++e)
                        if (id == e) d[e] += v;
                }
            }
            uint32_t* out = reinterpret_cast<uint32_t*>(d_rows + i * few_d_row<EP>());
#pragma unroll
            for (int part = 0; part < 3; ++part)
#pragma unroll
                for (int e = 0; e < EP; e += 2)
                    out[(part * EP + e) / 2] = bf16_part(d[e]) | bf16_part(d[e + 1]) << 16;
        }
        __syncthreads();
        if (!active) continue;
        for (int first = batch; first < batch + count; first += kFewTile) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
            __syncwarp();
            if (sums) load(load_slot);  // past the range: zeros
            asm volatile("cp.async.commit_group;" ::: "memory");
            const uint32_t xs = ring + slot * kFewStage;
            const uint32_t ds = d_at + (first - batch) * few_d_row<EP>();
#pragma unroll
            for (int k = 0; k < kFewTile / 16; ++k) {
                // the 8 x 8 blocks (token half, part block) of these 16 tokens; matrix m of an
                // ldmatrix is addressed by lanes 8 m .. 8 m + 7
                const uint32_t at = ds + (k * 16 + (lane & 7)) * few_d_row<EP>();
                const int m = lane >> 3;
                if (sums) {
                    // A = d^T: {rows 0-7, rows 8-15} x {tokens 0-7, tokens 8-15}, transposed on load
                    uint32_t first_a[4], second_a[4], third_a[4];
                    const uint32_t at_t = at + (m >> 1) * 8 * few_d_row<EP>() + (m & 1) * 16;
                    ldmatrix4_trans(at_t, first_a);            // EP 8: hi, mid; EP 16: hi
                    ldmatrix4_trans(at_t + 2 * EP, second_a);  // EP 8: mid, lo; EP 16: mid
                    if constexpr (EP == 16) ldmatrix4_trans(at_t + 4 * EP, third_a);  // lo
#pragma unroll
                    for (int f = 0; f < kFrags; f += 2) {
                        uint32_t bx[4];  // {tokens 0-7, 8-15} of columns 8 f, then of the next eight
                        ldmatrix4_trans(xs + (k * 16 + (lane & 7) + (m & 1) * 8) * kFewRow + (f + (m >> 1)) * 16, bx);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            if constexpr (EP == 8) {
                                mma_k16(acc[f + q][0], 0, second_a[1], 0, second_a[3], bx[2 * q], bx[2 * q + 1]);
                                mma_k16(acc[f + q][0], first_a[0], first_a[1], first_a[2], first_a[3], bx[2 * q],
                                        bx[2 * q + 1]);
                            } else {
                                mma_k16(acc[f + q][1], third_a[0], third_a[1], third_a[2], third_a[3], bx[2 * q],
                                        bx[2 * q + 1]);
                                mma_k16(acc[f + q][1], second_a[0], second_a[1], second_a[2], second_a[3],
                                        bx[2 * q], bx[2 * q + 1]);
                                mma_k16(acc[f + q][0], first_a[0], first_a[1], first_a[2], first_a[3], bx[2 * q],
                                        bx[2 * q + 1]);
                            }
                        }
                    }
                }
                if (grad_x) {
                    // A = d: {tokens 0-7, tokens 8-15} x {k 0-7, k 8-15}
                    uint32_t hi[4], mid[4], lo[4];
                    const uint32_t at_d = at + (m & 1) * 8 * few_d_row<EP>() + (m >> 1) * 16;
                    ldmatrix4(at_d, hi);           // EP 8: hi, mid; EP 16: hi
                    ldmatrix4(at_d + 2 * EP, mid);  // EP 8: mid, lo; EP 16: mid
                    if constexpr (EP == 16) ldmatrix4(at_d + 4 * EP, lo);
                    __syncwarp();  // x of these tokens has been read: dx may take its place
#pragma unroll
                    for (int f = 0; f < kFrags; ++f) {
                        float c[4];
                        // the six products, small ones first
                        const Staged w = w_staged[f * kFewThreads];
                        if constexpr (EP == 8) {
                            mma_k16_first(c, hi[0], hi[1], mid[2], mid[3], w.lo[0], w_hi[f][0]);
                            mma_k16(c, hi[0], hi[1], hi[2], hi[3], w.mid[0], w.mid[0]);
                            mma_k16(c, hi[0], hi[1], hi[2], hi[3], w_hi[f][0], w_hi[f][0]);
                        } else {
                            mma_k16_first(c, hi[0], hi[1], hi[2], hi[3], w.lo[0], w.lo[1]);
                            mma_k16(c, mid[0], mid[1], mid[2], mid[3], w.mid[0], w.mid[1]);
                            mma_k16(c, lo[0], lo[1], lo[2], lo[3], w_hi[f][0], w_hi[f][1]);
                            mma_k16(c, hi[0], hi[1], hi[2], hi[3], w.mid[0], w.mid[1]);
                            mma_k16(c, mid[0], mid[1], mid[2], mid[3], w_hi[f][0], w_hi[f][1]);
                            mma_k16(c, hi[0], hi[1], hi[2], hi[3], w_hi[f][0], w_hi[f][1]);
                        }
                        const uint32_t to = xs + (k * 16 + (lane >> 2)) * kFewRow + f * 16 + (lane & 3) * 4;
                        const __nv_bfloat162 low = __floats2bfloat162_rn(c[0], c[1]);
                        const __nv_bfloat162 high = __floats2bfloat162_rn(c[2], c[3]);
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(*reinterpret_cast<const uint32_t*>(&low)) : "memory");
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 8 * kFewRow), "r"(*reinterpret_cast<const uint32_t*>(&high)) : "memory");
                    }
                }
            }
            if (grad_x) {
                __syncwarp();
                const uint8_t* from = few_smem_raw + (warp * kFewStages + slot) * kFewStage + lane_at;
#pragma unroll
                for (int j = 0; j < kFewTile / 4; ++j) {
                    if (in_cols && first + row + 4 * j < t1)
                        *reinterpret_cast<uint4*>(to_dx) = *reinterpret_cast<const uint4*>(from + 4 * j * kFewRow);
                    to_dx += step;
                }
                __syncwarp();  // the slot is free again
            }
            if (++slot == kFewStages) slot = 0;
            if (++load_slot == kFewStages) load_slot = 0;
        }
        if (sums) {
            float* at = sums + (static_cast<int64_t>(blockIdx.y) * experts + (lane >> 2)) * hidden + h0 + 2 * (lane & 3);
#pragma unroll
            for (int g = 0; g < EP / 8; ++g, at += 8 * hidden) {
                const int e = g * 8 + (lane >> 2);
                const auto here = [&](int f) { return e < experts && h0 + f * 8 < hidden; };  // 8 divides hidden
                float2 before[kFrags];  // all on their way before the first is used
#pragma unroll
                for (int f = 0; f < kFrags; ++f)
                    before[f] = batch > t0 && here(f) ? *reinterpret_cast<const float2*>(at + f * 8) : make_float2(0.0f, 0.0f);
#pragma unroll
                for (int f = 0; f < kFrags; ++f) {
                    // expert e: EP 8: rows e and e + 8; EP 16: the same row of both fragments
                    const float a = EP == 8 ? acc[f][0][0] + acc[f][0][2] : acc[f][0][2 * g] + acc[f][EP / 8 - 1][2 * g];
                    const float b = EP == 8 ? acc[f][0][1] + acc[f][0][3] : acc[f][0][2 * g + 1] + acc[f][EP / 8 - 1][2 * g + 1];
                    if (here(f)) *reinterpret_cast<float2*>(at + f * 8) = make_float2(before[f].x + a, before[f].y + b);
                }
            }
#pragma unroll
            for (int f = 0; f < kFrags; ++f)
#pragma unroll
                for (int g = 0; g < EP / 8; ++g)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[f][g][j] = 0.0f;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// out = the parts' sum, in a fixed order: SLICES threads per vector add a stretch of
// the parts each, the first adds the stretches' sums.
template <int SLICES>
__global__ void __launch_bounds__(256)
add_parts_kernel(const float4* __restrict__ parts, float4* __restrict__ out, int64_t vecs, int ranges) {
    constexpr int kColumns = 256 / SLICES;
    __shared__ float4 sums[SLICES][kColumns];
    pdl_trigger();
    pdl_wait();
    const int column = threadIdx.x % kColumns, slice = threadIdx.x / kColumns;
    const int64_t i = blockIdx.x * static_cast<int64_t>(kColumns) + column;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (i < vecs) {
        const int from = ranges * slice / SLICES, to = ranges * (slice + 1) / SLICES;
#pragma unroll 8
        for (int r = from; r < to; ++r) {
            const float4 v = parts[r * vecs + i];
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
    }
    if constexpr (SLICES > 1) {
        sums[slice][column] = sum;
        __syncthreads();
        if (slice > 0) return;
        for (int s = 1; s < SLICES; ++s) {
            const float4 v = sums[s][column];
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
    }
    if (i < vecs) out[i] = sum;
}

// ------------------------------------------------------------------ host side

int pad8(int experts) { return (experts + 7) / 8 * 8; }

// Ranges of tokens for dW: those that take the least time, as waves of CTAs (or
// pairs) over the SMs, each as long as its tokens and a start of about 64, plus the
// partial sums' way through memory.  A token costs an SM of the first kernel about
// 6 ns (x read at the memory's rate), a pair of the second 12.6 ns at N = 256 (6
// MMAs of 128 cycles per 32 tokens); the partial sums of a range cost
// 8 E H bytes at 6500 bytes/ns.
constexpr int64_t kMinRange = 256;
int token_ranges(int64_t tokens, int64_t hidden, int experts, int sms) {
    const bool pair = pad8(experts) > kSideBySide;
    const int64_t tiles = pair ? (hidden + 2 * kTileH - 1) / (2 * kTileH) : (hidden + kTileH - 1) / kTileH;
    const int64_t slots = pair ? sms / 2 : sms;
    const double token_ns = pair ? 12.6 * experts / 256 : 6.0;
    const double part_tokens = 8.0 * experts * hidden / 6500.0 / token_ns;
    int64_t most = (tokens + kMinRange - 1) / kMinRange;
    if (most > 32) most = 32;
    int64_t best = 1;
    double best_time = 1e30;
    for (int64_t r = 1; r <= most; ++r) {
        const double waves = static_cast<double>((tiles * r + slots - 1) / slots);
        const double time = waves * (static_cast<double>(tokens) / r + 64.0) + (r > 1 ? r * part_tokens : 0.0);
        if (time < best_time) {
            best_time = time;
            best = r;
        }
    }
    return static_cast<int>(best);
}

int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The few-experts kernel: ranges of tokens so that every SM has the two CTAs that it
// holds, of whole tiles.
struct FewShape {
    int columns, range, ranges;
};
FewShape few_shape(int64_t tokens, int64_t hidden, int sms) {
    FewShape f;
    f.columns = static_cast<int>((hidden + kFewCols - 1) / kFewCols);
    const int64_t ranges = 2 * sms / f.columns < 1 ? 1 : 2 * sms / f.columns;
    f.range = static_cast<int>(((tokens + ranges - 1) / ranges + kFewTile - 1) / kFewTile * kFewTile);
    f.ranges = static_cast<int>((tokens + f.range - 1) / f.range);
    return f;
}

struct Layout {
    int64_t parts, weight, sums, total;
};
Layout layout(int64_t tokens, int64_t hidden, int experts, bool dx, bool dw, int sms) {
    const int64_t e8 = pad8(experts);
    Layout l = {};
    if (tokens == 0) return l;  // nothing is launched but a fill
    if (experts <= kFewExperts) {
        const int64_t ranges = few_shape(tokens, hidden, sms).ranges;
        l.total = dw && ranges > 1 ? round256(ranges * experts * hidden * 4) : 0;
        return l;
    }
    l.parts = 0;
    l.weight = round256(tokens * 3 * e8 * 2);
    l.sums = l.weight + (dx ? round256(hidden * 3 * e8 * 2) : 0);
    const int ranges = token_ranges(tokens, hidden, experts, sms);
    l.total = l.sums + (dw && ranges > 1 ? round256(ranges * experts * hidden * 4) : 0);
    return l;
}

cudaError_t device_sms(int* sms) {
    static int cached[64] = {};
    int device = 0;
    MOE_CUDA_TRY(cudaGetDevice(&device));
    if (cached[device & 63] == 0)
        MOE_CUDA_TRY(cudaDeviceGetAttribute(&cached[device & 63], cudaDevAttrMultiProcessorCount, device));
    *sms = cached[device & 63];
    return cudaSuccess;
}

cudaError_t add_parts(const float* parts, float* out, int64_t count, int ranges, cudaStream_t stream) {
    // Eight threads per vector where there are many parts (74 parts of 8 x 4096: 16 us with one).
    const int64_t vecs = count / 4;
    const int columns = ranges >= 16 ? 32 : 256;
    auto kernel = ranges >= 16 ? add_parts_kernel<8> : add_parts_kernel<1>;
    return launch_dependent(kernel, dim3(static_cast<unsigned>((vecs + columns - 1) / columns)), dim3(256), 0,
                            stream, reinterpret_cast<const float4*>(parts), reinterpret_cast<float4*>(out),
                            vecs, ranges);
}

cudaError_t few_experts(const __nv_bfloat16* x, const float* weight, const int32_t* ids,
                        const float* weights, const float* grad_weights, const float* grad_logits,
                        __nv_bfloat16* grad_x, float* grad_weight, float* scratch, int64_t tokens,
                        int64_t hidden, int experts, int topk, int sms, cudaStream_t stream) {
    const FewShape f = few_shape(tokens, hidden, sms);
    float* sums = grad_weight && f.ranges > 1 ? scratch : grad_weight;
    const bool eight = experts <= 8;
    auto kernel = eight ? router_few_kernel<8> : router_few_kernel<16>;
    const int smem = eight ? few_smem<8>() : few_smem<16>();
    static bool configured[2][64] = {};
    int device = 0;
    MOE_CUDA_TRY(cudaGetDevice(&device));
    if (!configured[eight][device & 63]) {
        MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        configured[eight][device & 63] = true;
    }
    MOE_CUDA_TRY(launch_dependent(kernel, dim3(f.columns, f.ranges), dim3(kFewThreads), smem, stream, x, weight,
                                  ids, weights, grad_weights, grad_logits, grad_x, sums, static_cast<int>(tokens),
                                  hidden, experts, topk, f.range));
    if (grad_weight && f.ranges > 1)
        return add_parts(sums, grad_weight, experts * hidden, f.ranges, stream);
    return cudaSuccess;
}

}  // namespace

cudaError_t route_backward_scratch_bytes(int64_t tokens, int64_t hidden, int experts, bool dx, bool dw,
                                         int64_t* bytes) {
    int sms = 0;
    MOE_CUDA_TRY(device_sms(&sms));
    *bytes = layout(tokens, hidden, experts, dx, dw, sms).total;
    return cudaSuccess;
}

cudaError_t launch_route_backward(const void* x, const float* weight, const int32_t* ids,
                                  const float* weights, const float* grad_weights,
                                  const float* grad_logits, void* grad_x, float* grad_weight,
                                  void* scratch, int64_t tokens, int64_t hidden, int experts, int topk,
                                  cudaStream_t stream, const char** error) {
    *error = nullptr;
    if (tokens == 0)
        return grad_weight ? cudaMemsetAsync(grad_weight, 0, experts * hidden * 4, stream) : cudaSuccess;
    int sms = 0;
    MOE_CUDA_TRY(device_sms(&sms));
    const int e8 = pad8(experts);
    const Layout l = layout(tokens, hidden, experts, grad_x != nullptr, grad_weight != nullptr, sms);
    char* base = static_cast<char*>(scratch);
    auto* parts = reinterpret_cast<__nv_bfloat16*>(base + l.parts);

    if (experts <= kFewExperts)
        return few_experts(static_cast<const __nv_bfloat16*>(x), weight, ids, weights, grad_weights, grad_logits,
                           static_cast<__nv_bfloat16*>(grad_x), grad_weight, reinterpret_cast<float*>(base + l.sums),
                           tokens, hidden, experts, topk, sms, stream);

    auto* wt = reinterpret_cast<__nv_bfloat16*>(base + l.weight);
    const int tiles_h = static_cast<int>((hidden + 31) / 32);
    const int weight_tiles = grad_x ? tiles_h * ((e8 + 31) / 32) : 0;
    // as few lanes per token as hold its experts, eight each, and its ids, one each
    const int lanes = experts <= 64 && topk <= 8 ? 8 : (experts <= 128 && topk <= 16 ? 16 : 32);
    const bool wide = experts % 4 == 0 && reinterpret_cast<uintptr_t>(grad_logits) % 16 == 0;
    const int64_t blocks = (tokens * lanes + 255) / 256;
    const int64_t grid = weight_tiles + (blocks < 8ll * sms ? blocks : 8ll * sms);
    auto split = lanes == 8 ? split_kernel<8> : (lanes == 16 ? split_kernel<16> : split_kernel<32>);
    MOE_CUDA_TRY(launch_dependent(split, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, weight, wt, hidden,
                                  tiles_h, weight_tiles, grad_logits, ids, weights, grad_weights,
                                  parts, tokens, experts, e8, topk, wide));
    int device = 0;
    MOE_CUDA_TRY(cudaGetDevice(&device));
    const char* rejected = "cuTensorMapEncodeTiled rejected an operand (pointer alignment or shape)";
    if (grad_x) {
        DxMaps maps;
        bool encoded = encode_bf16_tensor_map(&maps.out, grad_x, tokens, hidden, 0, 32);
        for (int part = 0; part < 3; ++part)
            encoded = encoded && encode_bf16_tensor_map(&maps.d[part], parts + part * e8, tokens, e8, 3 * e8, kDxTile) &&
                      encode_bf16_tensor_map(&maps.w[part], wt + part * e8, hidden, e8, 3 * e8, kDxTile);
        if (!encoded) {
            *error = rejected;
            return cudaErrorInvalidValue;
        }
        static bool configured[64] = {};
        if (!configured[device & 63]) {
            MOE_CUDA_TRY(cudaFuncSetAttribute(router_dx_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDxSmem));
            configured[device & 63] = true;
        }
        const int64_t pairs = ((tokens + 2 * kDxTile - 1) / (2 * kDxTile)) * ((hidden + 2 * kDxTile - 1) / (2 * kDxTile));
        const int64_t ctas = 2 * (pairs < sms / 2 ? pairs : sms / 2);
        MOE_CUDA_TRY(launch_dependent(router_dx_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kDxThreads), kDxSmem,
                                      stream, maps, static_cast<int>(tokens), hidden, e8));
    }
    if (grad_weight) {
        DwParams p;
        p.hidden = hidden;
        p.tokens = static_cast<int>(tokens);
        p.experts = experts;
        p.padded = e8;
        const bool pair = e8 > kSideBySide;
        if (pair) {
            p.n = (experts + 63) / 64 * 64;
            p.blocks = (p.n / 2 + 63) / 64;
            p.stages = kPairStages;
        } else {
            p.n = (3 * e8 + 15) / 16 * 16;
            p.blocks = (3 * e8 + 63) / 64;
            const int fit = kDwSmem / ((2 + p.blocks) * kBlock);
            p.stages = fit < kMaxStages ? fit : kMaxStages;
        }
        const int stage_bytes = (2 + (pair ? 3 : 1) * p.blocks) * kBlock;
        const int ranges = token_ranges(tokens, hidden, experts, sms);
        const int64_t per = (tokens + ranges - 1) / ranges;
        p.range = static_cast<int>((per + kTileT - 1) / kTileT * kTileT);
        const unsigned used = static_cast<unsigned>((tokens + p.range - 1) / p.range);
        p.out = used > 1 ? reinterpret_cast<float*>(base + l.sums) : grad_weight;
        CUtensorMap map_x, map_d;
        if (!encode_bf16_tensor_map(&map_x, x, tokens, hidden, 0, kTileT) ||
            !encode_bf16_tensor_map(&map_d, parts, tokens, 3 * e8, 0, kTileT)) {
            *error = rejected;
            return cudaErrorInvalidValue;
        }
        static bool configured[2][64] = {};
        auto kernel = pair ? router_dw_pair_kernel : router_dw_kernel;
        if (!configured[pair][device & 63]) {
            MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDwSmem + 1024));
            configured[pair][device & 63] = true;
        }
        const int tile = pair ? 2 * kTileH : kTileH;
        const unsigned tiles = static_cast<unsigned>((hidden + tile - 1) / tile * (pair ? 2 : 1));
        MOE_CUDA_TRY(launch_dependent(kernel, dim3(tiles, used), dim3(pair ? kPairThreads : kDwThreads),
                                      p.stages * stage_bytes + 1024, stream, map_x, map_d, p));
        if (used > 1)
            MOE_CUDA_TRY(add_parts(p.out, grad_weight, experts * hidden, static_cast<int>(used), stream));
    }
    return cudaSuccess;
}

cudaError_t read_route_backward_status(int32_t* code, bool clear) {
    MOE_CUDA_TRY(cudaMemcpyFromSymbol(code, g_route_backward_status, sizeof(int32_t)));
    if (clear) {
        const int32_t zero = 0;
        MOE_CUDA_TRY(cudaMemcpyToSymbol(g_route_backward_status, &zero, sizeof(int32_t)));
    }
    return cudaSuccess;
}

}  // namespace moe
