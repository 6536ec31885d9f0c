// Low-rank adapters of many requests beside the experts' shared projections.
// No counterpart in the reference.
//
// Packed row r belongs to expert e (by its place in offsets) and, through its
// request, to adapter p (row_adapters[r]; outside 0..P-1: none):
//   s[r]   = x[r] . A[p,e]^T                              [rank], fp32
//   y[r]   = base[r] + scale[p] s[r] . B[p,e]^T           [n]
//   out[r] = bf16(y[r])    or    bf16(silu(y[r, :I]) * y[r, I:]),  n = 2 I
// base is the projection's bf16 output; the sum and the SwiGLU are fp32 and
// rounded once.  Rows at or past offsets[E] are not touched.
//
// With rank <= 128 both products are thin: the traffic of x, of base and out,
// and of the A and B in use bounds them.  Two forms:
//
// Few rows (decoding): every row reads its own A and B.
//   shrink_rows_kernel  a warp per (row, rank index, 2048 elements of K)
//   expand_rows_kernel  rank/8 lanes per output column, 16 bytes of B each
//
// Many rows: rows that share a pair (p, e) share its weights through tiles.
//   count_kernel, order_kernel  stable counting sort of the rows by adapter.  Rows
//       come expert by expert, so the sorted rows are grouped by (p, e).
//   shrink_tile_kernel  64 sorted rows x rank, K in 64-wide cp.async stages; a
//       tile walks the runs of equal pairs inside it as one pipelined sequence
//   expand_tile_kernel  64 sorted rows x 128 columns; s enters the tensor cores as
//       two bf16 parts (s to 2^-16), base is added in fp32; each run of a tile finishes
//       its own rows, so what is not finite in one adapter stays in its rows
// Both use mma.sync: at rank <= 64 a 64-row tile does at most 64 flop per byte
// moved, far below what the tensor cores need to be the bound.
//
// Nothing depends on where a row lands in a tile: its products are its own, so
// results do not change with the batch around it, except between the two forms
// (their summation orders differ).
#include "common.cuh"
#include "launch.h"

namespace moe {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kNone = -1;     // row without an adapter
constexpr int kOutside = -2;  // row behind the last expert's span

struct Adapter {
    const bf16 *base, *x, *a, *b;
    const float* scale;           // [P] or null
    const int32_t* row_adapters;  // [rows]
    const int32_t* offsets;       // [E+1] or null: one expert, every row
    bf16* out;
    int64_t rows, k, n, cols;     // cols: output columns (n, or n / 2 with SwiGLU)
    int rank, adapters, experts;
    int32_t *table, *order, *keys;
    float* s;                     // [splits][rows][padded rank]
    int splits;
    int64_t split_k;              // K elements per split
};

__device__ __forceinline__ int64_t valid_rows(const Adapter& p) {
    if (!p.offsets) return p.rows;
    const int64_t end = p.offsets[p.experts];
    return end < p.rows ? end : p.rows;
}

// Expert whose span holds the row (offsets ascend; empty spans are passed over).
__device__ __forceinline__ int expert_of(const Adapter& p, int64_t row) {
    if (!p.offsets) return 0;
    int lo = 0, hi = p.experts - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.offsets[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ int row_key(const Adapter& p, int64_t row, int64_t valid) {
    if (row >= valid) return kOutside;
    const int adapter = p.row_adapters[row];
    if (adapter < 0 || adapter >= p.adapters) return kNone;
    return adapter * p.experts + expert_of(p, row);
}

__device__ __forceinline__ float silu_times(float g, float u) { return (g / (1.0f + expf(-g))) * u; }

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float sum) {
    sum = fmaf(bf16_lo(a.x), bf16_lo(b.x), sum);
    sum = fmaf(bf16_hi(a.x), bf16_hi(b.x), sum);
    sum = fmaf(bf16_lo(a.y), bf16_lo(b.y), sum);
    sum = fmaf(bf16_hi(a.y), bf16_hi(b.y), sum);
    sum = fmaf(bf16_lo(a.z), bf16_lo(b.z), sum);
    sum = fmaf(bf16_hi(a.z), bf16_hi(b.z), sum);
    sum = fmaf(bf16_lo(a.w), bf16_lo(b.w), sum);
    return fmaf(bf16_hi(a.w), bf16_hi(b.w), sum);
}

// ------------------------------------------------------------------ few rows

constexpr int kRowsSplitK = 2048;  // K elements per warp: 8 loads of 16 bytes a lane

__global__ void __launch_bounds__(256) shrink_rows_kernel(const Adapter p) {
    const int lane = threadIdx.x & 31;
    pdl_trigger();
    pdl_wait();
    const int64_t row = blockIdx.x;
    const int j = blockIdx.y * 8 + (threadIdx.x >> 5);
    const int key = row_key(p, row, valid_rows(p));
    if (key < 0 || j >= p.rank) return;
    const int64_t k0 = static_cast<int64_t>(blockIdx.z) * kRowsSplitK;
    const int count = static_cast<int>(p.k - k0 < kRowsSplitK ? p.k - k0 : kRowsSplitK);
    const bf16* x = p.x + row * p.k + k0;
    const bf16* a = p.a + (static_cast<int64_t>(key) * p.rank + j) * p.k + k0;
    uint4 xv[8], av[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = (lane + 32 * i) * 8;
        const bool in = c < count;
        av[i] = in ? __ldg(reinterpret_cast<const uint4*>(a + c)) : make_uint4(0, 0, 0, 0);
        xv[i] = in ? __ldg(reinterpret_cast<const uint4*>(x + c)) : make_uint4(0, 0, 0, 0);
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = dot8(xv[i], av[i], sum);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) p.s[(static_cast<int64_t>(blockIdx.z) * p.rows + row) * p.rank + j] = sum;
}

// LANES (a power of two >= rank / 8) lanes per column, kUnroll columns per lane.
template <int LANES, bool SWIGLU>
__global__ void __launch_bounds__(256) expand_rows_kernel(const Adapter p) {
    constexpr int kUnroll = 4, kStep = 256 / LANES;
    pdl_trigger();
    pdl_wait();
    const int64_t row = blockIdx.y;
    const int key = row_key(p, row, valid_rows(p));
    if (key == kOutside) return;
    if (key == kNone && !SWIGLU && p.out == p.base) return;
    const int chunk = threadIdx.x % LANES;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * (kUnroll * kStep) + threadIdx.x / LANES;
    const bf16* base = p.base + row * p.n;
    float d[kUnroll][SWIGLU ? 2 : 1] = {};
    if (key >= 0) {
        const bool in_rank = chunk * 8 < p.rank;
        const bf16* b = p.b + static_cast<int64_t>(key) * p.n * p.rank + chunk * 8;
        uint4 bv[kUnroll][SWIGLU ? 2 : 1];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int h = 0; h < (SWIGLU ? 2 : 1); ++h) {
                const int64_t c = c0 + u * kStep;
                bv[u][h] = in_rank && c < p.cols
                               ? __ldg(reinterpret_cast<const uint4*>(b + (c + h * p.cols) * p.rank))
                               : make_uint4(0, 0, 0, 0);
            }
        float s[8] = {};
        if (in_rank) {
            for (int z = 0; z < p.splits; ++z) {
                const float4* part = reinterpret_cast<const float4*>(
                    p.s + (static_cast<int64_t>(z) * p.rows + row) * p.rank + chunk * 8);
                const float4 lo = part[0], hi = part[1];
                s[0] += lo.x, s[1] += lo.y, s[2] += lo.z, s[3] += lo.w;
                s[4] += hi.x, s[5] += hi.y, s[6] += hi.z, s[7] += hi.w;
            }
        }
        const float scale = p.scale ? p.scale[key / p.experts] : 1.0f;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int h = 0; h < (SWIGLU ? 2 : 1); ++h) {
                const uint4 v = bv[u][h];
                float sum = s[0] * bf16_lo(v.x);
                sum = fmaf(s[1], bf16_hi(v.x), sum);
                sum = fmaf(s[2], bf16_lo(v.y), sum);
                sum = fmaf(s[3], bf16_hi(v.y), sum);
                sum = fmaf(s[4], bf16_lo(v.z), sum);
                sum = fmaf(s[5], bf16_hi(v.z), sum);
                sum = fmaf(s[6], bf16_lo(v.w), sum);
                sum = fmaf(s[7], bf16_hi(v.w), sum);
#pragma unroll
                for (int off = LANES / 2; off > 0; off >>= 1)
                    sum += __shfl_xor_sync(0xffffffffu, sum, off);
                d[u][h] = sum * scale;
            }
    }
    if (chunk != 0) return;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t c = c0 + u * kStep;
        if (c >= p.cols) continue;
        const float g = __bfloat162float(base[c]) + d[u][0];
        float y = g;
        if constexpr (SWIGLU) y = silu_times(g, __bfloat162float(base[c + p.cols]) + d[u][1]);
        p.out[row * p.cols + c] = __float2bfloat16_rn(y);
    }
}

// ---------------------------------------------------- many rows: sorted order

constexpr int kSortThreads = 1024;
constexpr int kMaxChunks = 128;

// Buckets: the adapters, then rows without one, then rows outside every span.
__device__ __forceinline__ int bucket_of(const Adapter& p, int64_t row, int64_t valid) {
    if (row >= valid) return p.adapters + 1;
    const int adapter = p.row_adapters[row];
    return adapter < 0 || adapter >= p.adapters ? p.adapters : adapter;
}

// table[bucket][chunk] = rows of the chunk in the bucket.
__global__ void __launch_bounds__(kSortThreads) count_kernel(const Adapter p, int64_t chunk_rows) {
    extern __shared__ int32_t counts[];
    const int buckets = p.adapters + 2;
    pdl_trigger();
    for (int i = threadIdx.x; i < buckets; i += kSortThreads) counts[i] = 0;
    pdl_wait();
    __syncthreads();
    const int64_t valid = valid_rows(p);
    const int64_t begin = blockIdx.x * chunk_rows;
    const int64_t end = begin + chunk_rows < p.rows ? begin + chunk_rows : p.rows;
    for (int64_t row = begin + threadIdx.x; row < end; row += kSortThreads)
        atomicAdd(&counts[bucket_of(p, row, valid)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < buckets; i += kSortThreads)
        p.table[static_cast<int64_t>(i) * gridDim.x + blockIdx.x] = counts[i];
}

// order[position] = row, keys[position] = its pair; stable inside a bucket.
__global__ void __launch_bounds__(kSortThreads) order_kernel(const Adapter p, int64_t chunk_rows) {
    extern __shared__ int32_t sort_smem[];
    const int buckets = p.adapters + 2;
    const int stride = buckets | 1;
    int32_t* hist = sort_smem;                  // [32 warps][buckets]
    int32_t* next = sort_smem + 32 * stride;    // [buckets] next position of this chunk's rows
    int32_t* total = next + buckets;       // [buckets]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    for (int i = tid; i < 32 * stride; i += kSortThreads) hist[i] = 0;
    pdl_wait();
    const int chunks = gridDim.x, me = blockIdx.x;
    for (int b = warp; b < buckets; b += 32) {
        int all = 0, before = 0;
        for (int c = lane; c < chunks; c += 32) {
            const int v = p.table[static_cast<int64_t>(b) * chunks + c];
            all += v;
            if (c < me) before += v;
        }
        all = __reduce_add_sync(0xffffffffu, all);
        before = __reduce_add_sync(0xffffffffu, before);
        if (lane == 0) {
            total[b] = all;
            next[b] = before;
        }
    }
    __syncthreads();
    if (warp == 0) {  // bucket starts
        int carry = 0;
        for (int b0 = 0; b0 < buckets; b0 += 32) {
            const int b = b0 + lane;
            const int v = b < buckets ? total[b] : 0;
            int inclusive = v;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inclusive, off);
                if (lane >= off) inclusive += y;
            }
            if (b < buckets) next[b] += carry + inclusive - v;
            carry += __shfl_sync(0xffffffffu, inclusive, 31);
        }
    }
    __syncthreads();
    const int64_t valid = valid_rows(p);
    const int64_t begin = me * chunk_rows;
    const int64_t end = begin + chunk_rows < p.rows ? begin + chunk_rows : p.rows;
    for (int64_t row0 = begin; row0 < end; row0 += kSortThreads) {
        const int64_t row = row0 + tid;
        const bool in = row < end;
        const int b = in ? bucket_of(p, row, valid) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, b);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        if (in && rank == 0) hist[warp * stride + b] = __popc(peers);
        __syncthreads();
        // per bucket: the warps' counts become the warps' first positions
        for (int x = warp; x < buckets; x += 32) {
            const int c = hist[lane * stride + x];
            int inclusive = c;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inclusive, off);
                if (lane >= off) inclusive += y;
            }
            const int at = next[x];
            hist[lane * stride + x] = at + inclusive - c;
            __syncwarp();
            if (lane == 31) next[x] = at + inclusive;
        }
        __syncthreads();
        if (in) {
            const int position = hist[warp * stride + b] + rank;
            p.order[position] = static_cast<int32_t>(row);
            p.keys[position] = b < p.adapters ? b * p.experts + expert_of(p, row)
                                              : (b == p.adapters ? kNone : kOutside);
        }
        __syncthreads();
        for (int x = warp; x < buckets; x += 32) hist[lane * stride + x] = 0;
        __syncthreads();
    }
}

// ------------------------------------------------------------ many rows: tiles

constexpr int kTileRows = 64;
constexpr int kTileThreads = 128;  // four warps, 16 rows each

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes, or zeros when !in (the source is not read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix2(uint32_t addr, uint32_t (&r)[2]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];"
                 : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The rows of a tile and the runs of equal pairs among them.  Rows without an
// adapter stand behind all others, so a run ends where the next begins.
struct TileRows {
    int32_t key[kTileRows];
    int32_t row[kTileRows];
    int32_t run[kTileRows + 1];  // first row of each run, then the end of the last
    int32_t runs;
    uint32_t starts[2], has[2];
};

__device__ __forceinline__ void load_tile_rows(const Adapter& p, int64_t tile, TileRows& t) {
    const int tid = threadIdx.x;
    if (tid < kTileRows) {
        const int64_t at = tile * kTileRows + tid;
        const int key = at < p.rows ? p.keys[at] : kOutside;
        t.key[tid] = key;
        t.row[tid] = at < p.rows ? p.order[at] : 0;
    }
    __syncthreads();
    bool start = false;
    if (tid < kTileRows) {
        const int key = t.key[tid];
        start = key >= 0 && (tid == 0 || key != t.key[tid - 1]);
        const uint32_t s = __ballot_sync(0xffffffffu, start), h = __ballot_sync(0xffffffffu, key >= 0);
        if ((tid & 31) == 0) {
            t.starts[tid >> 5] = s;
            t.has[tid >> 5] = h;
        }
    }
    __syncthreads();
    const int runs = __popc(t.starts[0]) + __popc(t.starts[1]);
    if (start) {
        const int before = (tid >= 32 ? __popc(t.starts[0]) : 0) +
                           __popc(t.starts[tid >> 5] & ((1u << (tid & 31)) - 1u));
        t.run[before] = tid;
    }
    if (tid == 0) {
        t.run[runs] = __popc(t.has[0]) + __popc(t.has[1]);
        t.runs = runs;
    }
    __syncthreads();
}

constexpr int kShrinkStages = 4;
template <int RN> constexpr int shrink_stage_bytes() { return (kTileRows + RN) * 128; }

// RN: rank rounded up to 8, 16, 32, 64 or 128; columns past the rank are zero.
template <int RN>
__global__ void __launch_bounds__(kTileThreads) shrink_tile_kernel(const Adapter p) {
    extern __shared__ __align__(128) uint8_t stages[];
    __shared__ TileRows t;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    load_tile_rows(p, blockIdx.x, t);
    const int runs = t.runs;
    if (runs == 0) return;
    const int64_t k0 = blockIdx.y * p.split_k;
    const int64_t k1 = k0 + p.split_k < p.k ? k0 + p.split_k : p.k;
    const int steps = static_cast<int>((k1 - k0 + 63) / 64);
    const int total = runs * steps;

    int load_run = 0, load_step = 0;
    auto load = [&](int slot) {  // one 64-wide K step of one run
        const uint32_t at = smem_addr(stages) + slot * shrink_stage_bytes<RN>();
        const int i0 = t.run[load_run], i1 = t.run[load_run + 1];
        const int64_t kc = k0 + load_step * 64;
#pragma unroll
        for (int j = 0; j < kTileRows * 8 / kTileThreads; ++j) {
            const int i = (tid + j * kTileThreads) >> 3, c = tid & 7;
            if (i < i0 || i >= i1) continue;  // rows of other runs: products nobody stores
            const bool in = kc + c * 8 < k1;
            copy16(at + i * 128 + ((c ^ (i & 7)) << 4),
                   p.x + static_cast<int64_t>(t.row[i]) * p.k + (in ? kc + c * 8 : 0), in);
        }
        const bf16* a = p.a + static_cast<int64_t>(t.key[i0]) * p.rank * p.k;
        for (int i = tid >> 3; i < RN; i += kTileThreads / 8) {
            const int c = tid & 7;
            const bool in = i < p.rank && kc + c * 8 < k1;
            copy16(at + kTileRows * 128 + i * 128 + ((c ^ (i & 7)) << 4),
                   a + (in ? i * p.k + kc + c * 8 : 0), in);
        }
        if (++load_step == steps) {
            load_step = 0;
            ++load_run;
        }
    };
#pragma unroll
    for (int s = 0; s < kShrinkStages - 1; ++s) {
        if (s < total) load(s);
        copy_commit();
    }
    float acc[RN / 8][4] = {};
    int run = 0, step = 0;
    for (int it = 0; it < total; ++it) {
        copy_wait<kShrinkStages - 2>();
        __syncthreads();  // stage `it` has landed everywhere, and stage it - 1 has been read
        if (it + kShrinkStages - 1 < total) load((it + kShrinkStages - 1) % kShrinkStages);
        copy_commit();
        const int i0 = t.run[run], i1 = t.run[run + 1];
        if (warp * 16 < i1 && warp * 16 + 16 > i0) {
            const uint32_t xs = smem_addr(stages) + (it % kShrinkStages) * shrink_stage_bytes<RN>();
            const uint32_t as = xs + kTileRows * 128;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint32_t xf[4];
                const int i = warp * 16 + (lane & 15);
                ldmatrix4(xs + i * 128 + (((kk * 2 + (lane >> 4)) ^ (i & 7)) << 4), xf);
                if constexpr (RN == 8) {
                    uint32_t af[2];
                    const int n = lane & 7;
                    ldmatrix2(as + n * 128 + (((kk * 2 + ((lane >> 3) & 1)) ^ (n & 7)) << 4), af);
                    mma16816(acc[0], xf, af[0], af[1]);
                } else {
#pragma unroll
                    for (int n0 = 0; n0 < RN; n0 += 16) {
                        uint32_t af[4];
                        const int n = n0 + (lane & 7) + ((lane >> 4) << 3);
                        ldmatrix4(as + n * 128 + (((kk * 2 + ((lane >> 3) & 1)) ^ (n & 7)) << 4), af);
                        mma16816(acc[n0 / 8], xf, af[0], af[1]);
                        mma16816(acc[n0 / 8 + 1], xf, af[2], af[3]);
                    }
                }
            }
            if (step == steps - 1) {
                const int64_t first = static_cast<int64_t>(blockIdx.y) * p.rows + blockIdx.x * static_cast<int64_t>(kTileRows);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = warp * 16 + (lane >> 2) + 8 * h;
                    if (i < i0 || i >= i1) continue;
                    float* s = p.s + (first + i) * RN + 2 * (lane & 3);
#pragma unroll
                    for (int n = 0; n < RN / 8; ++n)
                        *reinterpret_cast<float2*>(s + n * 8) = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
                }
#pragma unroll
                for (int n = 0; n < RN / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
            }
        }
        if (++step == steps) {
            step = 0;
            ++run;
        }
    }
    copy_wait<0>();
}

constexpr int kTileCols = 128;                        // rows of B per tile: 128 columns, or 64 gate + 64 up
constexpr int kBaseStride = kTileCols * 2 + 16;       // bytes; the pads keep ldmatrix and row stores conflict-free
template <int RN> constexpr int rank_k() { return RN < 16 ? 16 : RN; }
template <int RN> constexpr int b_stride() { return rank_k<RN>() * 2 + 16; }
template <int RN> constexpr int s_stride() { return rank_k<RN>() + 8; }  // floats
template <int RN> constexpr int expand_smem() {
    return kTileRows * kBaseStride + 2 * kTileCols * b_stride<RN>() + kTileRows * s_stride<RN>() * 4;
}

// Two floats as bf16 hi parts, and the rests' as a second register.
__device__ __forceinline__ void split2(float2 v, uint32_t& hi, uint32_t& lo) {
    const uint32_t a = f32_to_bf16_bits(v.x), b = f32_to_bf16_bits(v.y);
    hi = a | b << 16;
    lo = pack_bf16x2(v.x - bf16_bits_to_f32(a), v.y - bf16_bits_to_f32(b));
}

template <int RN, bool SWIGLU>
__global__ void __launch_bounds__(kTileThreads) expand_tile_kernel(const Adapter p, int blocks) {
    constexpr int RK = rank_k<RN>();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ TileRows t;
    uint8_t* base_s = smem;
    uint8_t* b_s = smem + kTileRows * kBaseStride;
    float* s_s = reinterpret_cast<float*>(b_s + 2 * kTileCols * b_stride<RN>());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t tile = blockIdx.x / blocks;
    constexpr int kOut = SWIGLU ? kTileCols / 2 : kTileCols;  // output columns of the tile
    const int64_t c0 = static_cast<int64_t>(blockIdx.x % blocks) * kOut;
    pdl_trigger();
    pdl_wait();
    load_tile_rows(p, tile, t);
    const int runs = t.runs;
    if (t.key[0] == kOutside) return;  // and so are all behind it
    if (runs == 0 && !SWIGLU && p.out == p.base) return;

    // row c of the tile's B: column c0 + c, or with SwiGLU the gate and up columns
    auto column = [&](int c) -> int64_t {
        return SWIGLU ? c0 + (c & 63) + (c >= 64 ? p.cols : 0) : c0 + c;
    };
    auto inside = [&](int c) { return c0 + (SWIGLU ? c & 63 : c) < p.cols; };
    // base: each warp its own 16 rows
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int i = warp * 16 + j * 2 + (lane >> 4), c = (lane & 15) * 8;
        if (t.key[i] != kOutside && inside(c))
            copy16(smem_addr(base_s) + i * kBaseStride + c * 2,
                   p.base + static_cast<int64_t>(t.row[i]) * p.n + column(c), true);
    }
    auto load_b = [&](int run, int slot) {
        const bf16* b = p.b + static_cast<int64_t>(t.key[t.run[run]]) * p.n * p.rank;
        const uint32_t at = smem_addr(b_s) + slot * kTileCols * b_stride<RN>();
        constexpr int kChunks = RK / 8;
        for (int i = tid; i < kTileCols * kChunks; i += kTileThreads) {
            const int c = i / kChunks, q = i % kChunks;
            const bool in = q * 8 < p.rank && inside(c);
            copy16(at + c * b_stride<RN>() + q * 16, b + (in ? column(c) * p.rank + q * 8 : 0), in);
        }
    };
    if (runs > 0) load_b(0, 0);
    copy_commit();

    // s: the splits' sum, scaled; zero past the rank and in rows without an adapter
    if (runs > 0) {
        const int64_t first = tile * kTileRows;
        for (int i = tid; i < kTileRows * (RK / 4); i += kTileThreads) {
            const int r = i / (RK / 4), q = (i % (RK / 4)) * 4;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int key = t.key[r];
            if (key >= 0 && q < RN) {
                for (int z = 0; z < p.splits; ++z) {
                    const float4 w = *reinterpret_cast<const float4*>(
                        p.s + (static_cast<int64_t>(z) * p.rows + first + r) * RN + q);
                    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                }
                const float scale = p.scale ? p.scale[key / p.experts] : 1.0f;
                v.x *= scale, v.y *= scale, v.z *= scale, v.w *= scale;
            }
            *reinterpret_cast<float4*>(s_s + r * s_stride<RN>() + q) = v;
        }
    }

    // y = base + delta in place, for rows r (one of two per lane; conflict-free)
    float acc[kTileCols / 8][4] = {};
    auto finish = [&](int h) {
        uint8_t* row = base_s + (warp * 16 + (lane >> 2) + 8 * h) * kBaseStride + (lane & 3) * 4;
#pragma unroll
        for (int n = 0; n < kOut / 8; ++n) {
            uint32_t* at = reinterpret_cast<uint32_t*>(row + n * 16);
            const uint32_t g = *at;
            float y0 = bf16_lo(g) + acc[n][2 * h], y1 = bf16_hi(g) + acc[n][2 * h + 1];
            if constexpr (SWIGLU) {
                const uint32_t u = *reinterpret_cast<const uint32_t*>(row + n * 16 + 128);
                y0 = silu_times(y0, bf16_lo(u) + acc[n + 8][2 * h]);
                y1 = silu_times(y1, bf16_hi(u) + acc[n + 8][2 * h + 1]);
            }
            *at = pack_bf16x2(y0, y1);
        }
    };
    const int r0 = warp * 16 + (lane >> 2), r1 = r0 + 8;
    for (int run = 0; run < runs; ++run) {
        __syncthreads();  // the other slot has been read; s is in place
        if (run + 1 < runs) load_b(run + 1, (run + 1) & 1);
        copy_commit();
        copy_wait<1>();
        __syncthreads();
        const int i0 = t.run[run], i1 = t.run[run + 1];
        if (warp * 16 >= i1 || warp * 16 + 16 <= i0) continue;
        const uint32_t bs = smem_addr(b_s) + (run & 1) * kTileCols * b_stride<RN>();
#pragma unroll
        for (int kk = 0; kk < RK / 16; ++kk) {
            uint32_t hi[4], lo[4];
            const float* s0 = s_s + r0 * s_stride<RN>() + kk * 16 + 2 * (lane & 3);
            const float* s1 = s0 + 8 * s_stride<RN>();
            split2(*reinterpret_cast<const float2*>(s0), hi[0], lo[0]);
            split2(*reinterpret_cast<const float2*>(s1), hi[1], lo[1]);
            split2(*reinterpret_cast<const float2*>(s0 + 8), hi[2], lo[2]);
            split2(*reinterpret_cast<const float2*>(s1 + 8), hi[3], lo[3]);
#pragma unroll
            for (int n0 = 0; n0 < kTileCols; n0 += 16) {
                uint32_t bf[4];
                const int n = n0 + (lane & 7) + ((lane >> 4) << 3);
                ldmatrix4(bs + n * b_stride<RN>() + (kk * 2 + ((lane >> 3) & 1)) * 16, bf);
                mma16816(acc[n0 / 8], lo, bf[0], bf[1]);
                mma16816(acc[n0 / 8], hi, bf[0], bf[1]);
                mma16816(acc[n0 / 8 + 1], lo, bf[2], bf[3]);
                mma16816(acc[n0 / 8 + 1], hi, bf[2], bf[3]);
            }
        }
        if (r0 >= i0 && r0 < i1) finish(0);
        if (r1 >= i0 && r1 < i1) finish(1);
#pragma unroll
        for (int n = 0; n < kTileCols / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
    }
    copy_wait<0>();
    __syncwarp();  // base rows are the warp's own
    if constexpr (SWIGLU) {  // rows without an adapter (elsewhere base stands as it is)
        if (t.key[r0] == kNone) finish(0);
        if (t.key[r1] == kNone) finish(1);
    }
    __syncwarp();
    constexpr int kPieces = kOut / 8, kPer = 32 / kPieces;  // 16-byte pieces of a row; rows per step
#pragma unroll
    for (int j = 0; j < 16 / kPer; ++j) {
        const int i = warp * 16 + j * kPer + lane / kPieces, c = (lane % kPieces) * 8;
        if (t.key[i] == kOutside || c0 + c >= p.cols) continue;
        if (!SWIGLU && t.key[i] == kNone && p.out == p.base) continue;
        *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(t.row[i]) * p.cols + c0 + c) =
            *reinterpret_cast<const uint4*>(base_s + i * kBaseStride + c * 2);
    }
}

// ---------------------------------------------------- adapters of packed rows

// row_adapters[inverse[t,k]] = token_adapters[t]; the padding rows of each
// expert's span (from offsets[e] + counts[e] on) get none.
__global__ void __launch_bounds__(256)
adapter_rows_kernel(const int32_t* __restrict__ token_adapters, const int32_t* __restrict__ inverse,
                    const int32_t* __restrict__ counts, const int32_t* __restrict__ offsets,
                    int32_t* __restrict__ row_adapters, int64_t assignments, int topk, int experts,
                    int64_t rows, int64_t blocks) {
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x < blocks) {
        const int64_t i = blockIdx.x * 256ll + threadIdx.x;
        if (i >= assignments) return;
        const int64_t row = inverse[i];
        if (row >= 0 && row < rows) row_adapters[row] = token_adapters[i / topk];
    } else {
        const int e = static_cast<int>(blockIdx.x - blocks);
        const int64_t end = offsets[e + 1] < rows ? offsets[e + 1] : rows;
        for (int64_t r = static_cast<int64_t>(offsets[e]) + counts[e] + threadIdx.x; r < end; r += 256)
            if (r >= 0) row_adapters[r] = kNone;
    }
}

// ------------------------------------------------------------------ host side

int padded_rank(int rank) {
    int r = 8;
    while (r < rank) r *= 2;
    return r;
}

// Which form: see the comment at kFewRows.
constexpr int64_t kFewRows = 256;

struct Shape {
    bool few;
    int splits;
    int64_t split_k, chunk_rows, table, order, keys, s, total;
    int chunks;
};

int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

Shape shape_of(int64_t rows, int64_t k, int rank, int adapters, int sms) {
    Shape f = {};
    f.few = rows <= kFewRows;
    if (f.few) {
        f.split_k = kRowsSplitK;
        f.splits = static_cast<int>((k + kRowsSplitK - 1) / kRowsSplitK);
        f.total = round256(rows * rank * 4 * f.splits);
        return f;
    }
    // K is split until about four CTAs of the shrink kernel stand on every SM, in
    // parts of at least 256 elements.
    const int64_t tiles = (rows + kTileRows - 1) / kTileRows;
    int64_t splits = 4ll * sms / tiles;
    const int64_t most = (k + 255) / 256;
    splits = splits < 1 ? 1 : (splits > most ? most : splits);
    f.split_k = ((k + splits - 1) / splits + 63) / 64 * 64;
    f.splits = static_cast<int>((k + f.split_k - 1) / f.split_k);
    f.chunk_rows = (rows + static_cast<int64_t>(kMaxChunks) * kSortThreads - 1) /
                   (static_cast<int64_t>(kMaxChunks) * kSortThreads) * kSortThreads;
    f.chunks = static_cast<int>((rows + f.chunk_rows - 1) / f.chunk_rows);
    f.table = 0;
    f.order = round256(static_cast<int64_t>(adapters + 2) * f.chunks * 4);
    f.keys = f.order + round256(rows * 4);
    f.s = f.keys + round256(rows * 4);
    f.total = f.s + round256(rows * padded_rank(rank) * 4 * f.splits);
    return f;
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

template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, bool (&configured)[64]) {
    int device = 0;
    MOE_CUDA_TRY(cudaGetDevice(&device));
    if (!configured[device & 63]) {
        MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        configured[device & 63] = true;
    }
    return cudaSuccess;
}

template <int LANES, bool SWIGLU>
cudaError_t expand_rows(const Adapter& p, cudaStream_t stream) {
    constexpr int kCols = 4 * 256 / LANES;
    return launch_dependent(expand_rows_kernel<LANES, SWIGLU>,
                            dim3(static_cast<unsigned>((p.cols + kCols - 1) / kCols), static_cast<unsigned>(p.rows)),
                            dim3(256), 0, stream, p);
}

template <bool SWIGLU>
cudaError_t few_rows(const Adapter& p, cudaStream_t stream) {
    MOE_CUDA_TRY(launch_dependent(shrink_rows_kernel,
                                  dim3(static_cast<unsigned>(p.rows), (p.rank + 7) / 8, p.splits), dim3(256),
                                  0, stream, p));
    if (p.rank <= 8) return expand_rows<1, SWIGLU>(p, stream);
    if (p.rank <= 16) return expand_rows<2, SWIGLU>(p, stream);
    if (p.rank <= 32) return expand_rows<4, SWIGLU>(p, stream);
    if (p.rank <= 64) return expand_rows<8, SWIGLU>(p, stream);
    return expand_rows<16, SWIGLU>(p, stream);
}

template <int RN, bool SWIGLU>
cudaError_t tiles(const Adapter& p, const Shape& f, cudaStream_t stream) {
    static bool order_ok[64] = {}, shrink_ok[64] = {}, expand_ok[64] = {};
    const int buckets = p.adapters + 2;
    const int order_smem = (32 * (buckets | 1) + 2 * buckets) * 4;
    constexpr int kOrderMost = (32 * ((kMaxAdapters + 2) | 1) + 2 * (kMaxAdapters + 2)) * 4;
    constexpr int kShrinkSmem = kShrinkStages * shrink_stage_bytes<RN>();
    MOE_CUDA_TRY(allow_smem(order_kernel, kOrderMost, order_ok));
    MOE_CUDA_TRY(allow_smem(shrink_tile_kernel<RN>, kShrinkSmem, shrink_ok));
    MOE_CUDA_TRY(allow_smem(expand_tile_kernel<RN, SWIGLU>, expand_smem<RN>(), expand_ok));
    MOE_CUDA_TRY(launch_dependent(count_kernel, dim3(f.chunks), dim3(kSortThreads), buckets * 4, stream, p,
                                  f.chunk_rows));
    MOE_CUDA_TRY(launch_dependent(order_kernel, dim3(f.chunks), dim3(kSortThreads), order_smem, stream, p,
                                  f.chunk_rows));
    const unsigned n_tiles = static_cast<unsigned>((p.rows + kTileRows - 1) / kTileRows);
    MOE_CUDA_TRY(launch_dependent(shrink_tile_kernel<RN>, dim3(n_tiles, f.splits), dim3(kTileThreads),
                                  kShrinkSmem, stream, p));
    const int out_cols = SWIGLU ? kTileCols / 2 : kTileCols;
    const int blocks = static_cast<int>((p.cols + out_cols - 1) / out_cols);
    return launch_dependent(expand_tile_kernel<RN, SWIGLU>, dim3(n_tiles * static_cast<unsigned>(blocks)),
                            dim3(kTileThreads), expand_smem<RN>(), stream, p, blocks);
}

template <bool SWIGLU>
cudaError_t many_rows(const Adapter& p, const Shape& f, cudaStream_t stream) {
    switch (padded_rank(p.rank)) {
        case 8: return tiles<8, SWIGLU>(p, f, stream);
        case 16: return tiles<16, SWIGLU>(p, f, stream);
        case 32: return tiles<32, SWIGLU>(p, f, stream);
        case 64: return tiles<64, SWIGLU>(p, f, stream);
        default: return tiles<128, SWIGLU>(p, f, stream);
    }
}

}  // namespace

cudaError_t adapter_scratch_bytes(int64_t rows, int64_t k, int rank, int adapters, int64_t* bytes) {
    int sms = 0;
    MOE_CUDA_TRY(device_sms(&sms));
    *bytes = shape_of(rows, k, rank, adapters, sms).total;
    return cudaSuccess;
}

cudaError_t launch_adapter(const void* base, const void* x, const void* a, const void* b,
                           const float* scale, const int32_t* row_adapters, const int32_t* offsets,
                           void* out, int64_t rows, int64_t k, int64_t n, int rank, int adapters,
                           int experts, bool swiglu, void* scratch, cudaStream_t stream) {
    if (rows == 0) return cudaSuccess;
    int sms = 0;
    MOE_CUDA_TRY(device_sms(&sms));
    const Shape f = shape_of(rows, k, rank, adapters, sms);
    Adapter p;
    p.base = static_cast<const bf16*>(base);
    p.x = static_cast<const bf16*>(x);
    p.a = static_cast<const bf16*>(a);
    p.b = static_cast<const bf16*>(b);
    p.scale = scale;
    p.row_adapters = row_adapters;
    p.offsets = offsets;
    p.out = static_cast<bf16*>(out);
    p.rows = rows;
    p.k = k;
    p.n = n;
    p.cols = swiglu ? n / 2 : n;
    p.rank = rank;
    p.adapters = adapters;
    p.experts = experts;
    char* at = static_cast<char*>(scratch);
    p.table = reinterpret_cast<int32_t*>(at + f.table);
    p.order = reinterpret_cast<int32_t*>(at + f.order);
    p.keys = reinterpret_cast<int32_t*>(at + f.keys);
    p.s = reinterpret_cast<float*>(at + f.s);
    p.splits = f.splits;
    p.split_k = f.split_k;
    if (f.few) return swiglu ? few_rows<true>(p, stream) : few_rows<false>(p, stream);
    return swiglu ? many_rows<true>(p, f, stream) : many_rows<false>(p, f, stream);
}

cudaError_t launch_adapter_rows(const int32_t* token_adapters, const int32_t* inverse,
                                const int32_t* counts, const int32_t* offsets, int32_t* row_adapters,
                                int64_t tokens, int topk, int experts, int64_t rows, cudaStream_t stream) {
    const int64_t blocks = (tokens * topk + 255) / 256;
    return launch_dependent(adapter_rows_kernel, dim3(static_cast<unsigned>(blocks + experts)), dim3(256), 0,
                            stream, token_adapters, inverse, counts, offsets, row_adapters, tokens * topk,
                            topk, experts, rows, blocks);
}

}  // namespace moe
