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
//   tiles_kernel        cuts each group into tiles of up to 64 rows.  (Tiles over 64
//       consecutive sorted rows, whatever groups they touch, were measured first: a
//       few tiles with 26 small groups held everything up, 1080 us against 583 at
//       16384 tokens, 64 experts, top-6, 32 adapters of rank 32.)
//   shrink_tile_kernel  a tile's rows x rank, K in 128-wide cp.async stages
//   expand_tile_kernel  a tile's rows x column blocks of 64; s enters the tensor
//       cores as three bf16 parts (s to 2^-24), base is added in fp32
// Both use mma.sync: at rank <= 64 a 64-row tile does at most 64 flop per byte
// moved, far below what the tensor cores need to be the bound.  A tile holds one
// adapter's rows only, so what is not finite in one adapter or row stays there.
//
// Nothing depends on where a row lands in a tile: its products are its own, so for a
// given number of rows (which decides the form and how K is split) a row's result does
// not change with the rows around it.
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
    int32_t* tile_count;          // [0] tiles, [1] stretches claimed by the expand kernel
    int2* tiles;                  // {first sorted row, rows} of each tile
    float* s;                     // few rows: [splits][rows][rank]; tiles: pieces (s_pieces)
    int splits;                   // of K
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

// Key of one row for a whole warp: the spans that end at or before the row are
// counted, all their ends loaded at once (a search would wait for each).
__device__ __forceinline__ int row_key(const Adapter& p, int64_t row, int lane) {
    const int adapter = p.row_adapters[row];
    int expert = 0;
    if (p.offsets) {
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            expert += __popc(__ballot_sync(0xffffffffu, e < p.experts && p.offsets[e + 1] <= row));
        }
        if (expert >= p.experts) return kOutside;
    }
    return adapter < 0 || adapter >= p.adapters ? kNone : adapter * p.experts + expert;
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

// ------------------------------------------------------------------ few rows

constexpr int kRowsSplitK = 2048;  // K elements per CTA

// CTA: one row, eight rows of its A (a warp each), 2048 elements of K.  Everything is
// copied to shared memory at once, so that all of it is in flight together; loads
// into registers were used one by one (16.8 us against 12.3 at 134 rows of 14336).
__global__ void __launch_bounds__(256) shrink_rows_kernel(const Adapter p) {
    __shared__ uint4 xs[kRowsSplitK / 8];
    __shared__ uint4 as[8][kRowsSplitK / 8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    const int64_t row = blockIdx.x;
    const int key = row_key(p, row, lane);
    if (key < 0) return;
    const int j = blockIdx.y * 8 + warp;  // < rank: rank is a multiple of 8
    const int64_t k0 = static_cast<int64_t>(blockIdx.z) * kRowsSplitK;
    const int vecs = static_cast<int>(p.k - k0 < kRowsSplitK ? p.k - k0 : kRowsSplitK) / 8;
    const bf16* x = p.x + row * p.k + k0;
    const bf16* a = p.a + (static_cast<int64_t>(key) * p.rank + j) * p.k + k0;
    if (static_cast<int>(threadIdx.x) < vecs) copy16(smem_addr(&xs[threadIdx.x]), x + threadIdx.x * 8, true);
#pragma unroll
    for (int i = 0; i < kRowsSplitK / 8; i += 32)
        if (i + lane < vecs) copy16(smem_addr(&as[warp][i + lane]), a + (i + lane) * 8, true);
    copy_commit();
    copy_wait<0>();
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kRowsSplitK / 8; i += 32)
        if (i + lane < vecs) sum = dot8(xs[i + lane], as[warp][i + lane], sum);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) p.s[(static_cast<int64_t>(blockIdx.z) * p.rows + row) * p.rank + j] = sum;
}

// CTA: one row, 1024 / LANES columns (with SwiGLU as many gate and up columns), LANES (a
// power of two >= rank / 8) lanes per column with 16 bytes of B each.  B, base and the
// parts of s are copied to shared memory together, as above.
constexpr int kSplitsAtOnce = 8;

template <int LANES, bool SWIGLU>
__global__ void __launch_bounds__(256) expand_rows_kernel(const Adapter p) {
    constexpr int kUnroll = 4, kStep = 256 / LANES, kHalves = SWIGLU ? 2 : 1, kCols = kUnroll * kStep;
    __shared__ uint4 bs[kHalves][kUnroll][256];
    __shared__ uint4 base_s[kHalves][kCols / 8];
    __shared__ __align__(16) float s_s[kSplitsAtOnce][LANES * 8];
    const int tid = threadIdx.x, chunk = tid % LANES, column = tid / LANES;
    pdl_trigger();
    pdl_wait();
    const int64_t row = blockIdx.y;
    const int key = row_key(p, row, tid & 31);
    if (key == kOutside) return;
    if (key == kNone && !SWIGLU && p.out == p.base) return;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kCols;
    const int cols = static_cast<int>(p.cols - c0 < kCols ? p.cols - c0 : kCols);
    const bool in_rank = key >= 0 && chunk * 8 < p.rank;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        const int64_t first = c0 + h * p.cols;
        if (tid < cols / 8) copy16(smem_addr(&base_s[h][tid]), p.base + row * p.n + first + tid * 8, true);
        const bf16* b = p.b + ((key >= 0 ? static_cast<int64_t>(key) : 0) * p.n + first + column) * p.rank + chunk * 8;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (in_rank && column + u * kStep < cols)
                copy16(smem_addr(&bs[h][u][tid]), b + u * kStep * p.rank, true);
    }
    float s[8] = {};
    for (int z0 = 0; z0 < (key >= 0 ? p.splits : 0); z0 += kSplitsAtOnce) {
        const int count = min(kSplitsAtOnce, p.splits - z0);
        if (z0 > 0) __syncthreads();
        for (int i = tid; i < count * (p.rank / 4); i += 256) {
            const int z = i / (p.rank / 4), q = i % (p.rank / 4) * 4;
            copy16(smem_addr(&s_s[z][q]), p.s + ((z0 + z) * p.rows + row) * p.rank + q, true);
        }
        copy_commit();
        copy_wait<0>();
        __syncthreads();
        if (in_rank)
            for (int z = 0; z < count; ++z)
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += s_s[z][chunk * 8 + i];
    }
    copy_commit();
    copy_wait<0>();
    __syncthreads();  // base has arrived everywhere
    const float scale = key >= 0 && p.scale ? p.scale[key / p.experts] : 1.0f;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int c = column + u * kStep;
        float y[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            float sum = 0.0f;
            if (in_rank && c < cols) {
                const uint4 v = bs[h][u][tid];
                sum = s[0] * bf16_lo(v.x);
                sum = fmaf(s[1], bf16_hi(v.x), sum);
                sum = fmaf(s[2], bf16_lo(v.y), sum);
                sum = fmaf(s[3], bf16_hi(v.y), sum);
                sum = fmaf(s[4], bf16_lo(v.z), sum);
                sum = fmaf(s[5], bf16_hi(v.z), sum);
                sum = fmaf(s[6], bf16_lo(v.w), sum);
                sum = fmaf(s[7], bf16_hi(v.w), sum);
            }
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            y[h] = c < cols ? __bfloat162float(reinterpret_cast<const bf16*>(base_s[h])[c]) : 0.0f;
            if (key >= 0) y[h] += sum * scale;  // without an adapter a zero keeps its sign
        }
        if constexpr (SWIGLU) y[0] = silu_times(y[0], y[1]);
        if (chunk == 0 && c < cols) p.out[row * p.cols + c0 + c] = __float2bfloat16_rn(y[0]);
    }
}

// ---------------------------------------------------- many rows: sorted order

constexpr int kSortThreads = 1024;
constexpr int kMaxChunks = 128;
constexpr int kClusterChunks = 8;                 // the sort as one cluster: up to 8 chunks
constexpr int64_t kClusterChunkRows = kSortThreads;  // of one round of rows
constexpr int kTileRows = 64;

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word of this CTA's shared memory, in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t load_peer(const void* local, int rank) {
    uint32_t address = smem_addr(local), value;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(address), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(value) : "r"(address) : "memory");
    return value;
}

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
    if (blockIdx.x == 0 && threadIdx.x < 2) p.tile_count[threadIdx.x] = 0;
    const int64_t valid = valid_rows(p);
    const int64_t begin = blockIdx.x * chunk_rows;
    const int64_t end = begin + chunk_rows < p.rows ? begin + chunk_rows : p.rows;
    for (int64_t row = begin + threadIdx.x; row < end; row += kSortThreads)
        atomicAdd(&counts[bucket_of(p, row, valid)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < buckets; i += kSortThreads)
        p.table[static_cast<int64_t>(i) * gridDim.x + blockIdx.x] = counts[i];
}

// Cuts the sorted rows' groups of equal keys into tiles.  A thread whose key
// differs from the one before starts a group; where the next start lies in the
// same warp the group's length is known, and the warp searches the end of its
// last group together (32 probes at a time).  Tiles land in any order: each is
// a piece of work of its own.  none: rows without an adapter need tiles too.
// Called by whole warps, lane 0 at a multiple of 32; `at` may be past the rows.
__device__ void cut_tiles(const Adapter& p, bool none, int64_t at) {
    const int lane = threadIdx.x & 31;
    const int key = at < p.rows ? p.keys[at] : kOutside;
    const bool start = at < p.rows && (at == 0 || p.keys[at - 1] != key);
    const uint32_t starts = __ballot_sync(0xffffffffu, start);
    if (starts == 0) return;
    const int last = 31 - __clz(starts);
    const uint32_t later = lane == 31 ? 0 : starts >> (lane + 1);
    int64_t length = start && later ? __ffs(later) : 0;
    const int last_key = __shfl_sync(0xffffffffu, key, last);
    const int64_t last_at = at - lane + last;
    int64_t lo = at - lane + 32, hi = p.rows;  // keys[lo - 1] is last_key; the end lies in [lo, hi]
    if (lo > hi) lo = hi;
    while (lo < hi) {
        const int64_t step = (hi - lo + 31) / 32;
        const int64_t probe = lo + step * (lane + 1) - 1;
        const uint32_t past = __ballot_sync(0xffffffffu, probe >= hi || p.keys[probe] != last_key);
        if (past == 0) {
            lo = hi;
        } else {
            const int f = __ffs(past) - 1;
            const int64_t bound = lo + step * (f + 1) - 1;
            if (bound < hi) hi = bound;
            lo += step * f;
        }
    }
    if (lane == last) length = lo - last_at;
    const bool wanted = start && (key >= 0 || (none && key == kNone));
    const int count = wanted ? static_cast<int>((length + kTileRows - 1) / kTileRows) : 0;
    int inclusive = count;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inclusive, off);
        if (lane >= off) inclusive += y;
    }
    const int total = __shfl_sync(0xffffffffu, inclusive, 31);
    int first = 0;
    if (lane == 0 && total > 0) first = atomicAdd(p.tile_count, total);
    first = __shfl_sync(0xffffffffu, first, 0);
    if (count > 0 && lane != last)  // at most 31 rows: one tile
        p.tiles[first + inclusive - 1] = make_int2(static_cast<int>(at), static_cast<int>(length));
    const int last_count = __shfl_sync(0xffffffffu, count, last);
    for (int i = lane; i < last_count; i += 32) {
        const int64_t row = last_at + static_cast<int64_t>(i) * kTileRows;
        const int64_t rest = lo - row;
        p.tiles[first + total - last_count + i] =
            make_int2(static_cast<int>(row), static_cast<int>(rest < kTileRows ? rest : kTileRows));
    }
}

__global__ void __launch_bounds__(256) tiles_kernel(const Adapter p, bool none) {
    pdl_trigger();
    pdl_wait();
    cut_tiles(p, none, blockIdx.x * 256ll + threadIdx.x);
}

// order[position] = row, keys[position] = its pair; stable inside a bucket.  One CTA
// per chunk.  kCluster: the CTAs are one cluster, count their chunks themselves, learn
// each other's counts from shared memory, and cut the tiles when all rows are placed,
// in one launch instead of three.
template <bool kCluster>
__global__ void __launch_bounds__(kSortThreads) order_kernel(const Adapter p, int64_t chunk_rows, bool none) {
    extern __shared__ int32_t sort_smem[];
    const int buckets = p.adapters + 2;
    const int stride = buckets | 1;
    int32_t* hist = sort_smem;                  // [32 warps][buckets]
    int32_t* next = sort_smem + 32 * stride;    // [buckets] next position of this chunk's rows
    int32_t* total = next + buckets;            // [buckets]
    int32_t* local = total + buckets;           // [buckets] this chunk's counts (cluster form)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int chunks = gridDim.x, me = blockIdx.x;
    // no early trigger: CTAs of the next kernel that start beside this one's end up crowded on
    // the other SMs (1032 rows over 443 pairs: the call 179 us with it, 140 without)
    for (int i = tid; i < 32 * stride; i += kSortThreads) hist[i] = 0;
    if constexpr (kCluster)
        for (int i = tid; i < buckets; i += kSortThreads) local[i] = 0;
    pdl_wait();
    if constexpr (kCluster) {
        __syncthreads();
        if (me == 0 && tid < 2) p.tile_count[tid] = 0;
        const int64_t valid = valid_rows(p);
        const int64_t end = (me + 1) * chunk_rows < p.rows ? (me + 1) * chunk_rows : p.rows;
        for (int64_t row = me * chunk_rows + tid; row < end; row += kSortThreads)
            atomicAdd(&local[bucket_of(p, row, valid)], 1);
        cluster_barrier();
        for (int b = tid; b < buckets; b += kSortThreads) {
            int all = 0, before = 0;
            for (int c = 0; c < chunks; ++c) {
                const int v = static_cast<int>(load_peer(&local[b], c));
                all += v;
                if (c < me) before += v;
            }
            total[b] = all;
            next[b] = before;
        }
    } else {
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
    if constexpr (kCluster) {
        cluster_barrier();  // every row is in its place, and every peer's counts have been read
        for (int64_t at = static_cast<int64_t>(me) * kSortThreads + tid; at - tid < p.rows;
             at += static_cast<int64_t>(chunks) * kSortThreads)
            cut_tiles(p, none, at);
    }
}

// ------------------------------------------------------------ many rows: tiles

constexpr int kTileThreads = 128;  // of the shrink kernel: four warps, 16 rows each

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

constexpr int kShrinkStages = 3;
constexpr int kShrinkK = 128;                   // K elements per stage: 256 bytes of each row
constexpr int kShrinkRow = kShrinkK * 2;
// The tensor cores cut a sum off below the accumulator's last bit at every MMA, so long sums
// drift (s of K = 14336 lost 1e-4 of a sum whose first term is the largest).  After this many
// stages (256 elements, 16 MMAs) an accumulator is added to an fp32 sum, rounded to nearest.
constexpr int kShrinkChunk = 2;
template <int RN> constexpr int shrink_stage_bytes() { return (kTileRows + RN) * kShrinkRow; }

// 16-byte chunk c of row i of a stage: the low three bits are swizzled by the
// row, so the eight rows of an ldmatrix lie in different banks.
__device__ __forceinline__ uint32_t stage_at(int i, int c) { return i * kShrinkRow + ((c ^ (i & 7)) << 4); }

template <int RN> constexpr int rank_k() { return RN < 16 ? 16 : RN; }

// s of a sorted row as the tensor cores take it: three bf16 parts, each the leading eight
// bits of what those before it leave, so their sum is s.  An infinity is the first part alone
// (and its product what the formula says), as no part of a finite s is infinite.  For every 16 of its elements four pieces
// of 16 bytes, piece q = bf16 {hi(2q, 2q + 1), hi(2q + 8, 2q + 9), mid of the same}, and four
// of 8, lo of the same.  A lane's part of an accumulator fragment is a piece of both, and so
// is its part of an operand.
constexpr int kPieceBytes = 96;
template <int RN> __device__ __forceinline__ char* s_pieces(const Adapter& p, int64_t row, int kk) {
    return reinterpret_cast<char*>(p.s) + (row * (rank_k<RN>() / 16) + kk) * kPieceBytes;
}
__device__ __forceinline__ uint4* piece_hi_mid(char* pieces, int q) { return reinterpret_cast<uint4*>(pieces) + q; }
__device__ __forceinline__ uint2* piece_lo(char* pieces, int q) { return reinterpret_cast<uint2*>(pieces + 64) + q; }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Two floats as three bf16 parts.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    const auto take = [&] {
        const uint32_t x = __float_as_uint(a) & 0xffff0000u, y = __float_as_uint(b) & 0xffff0000u;
        a = fabsf(a) < INFINITY ? a - __uint_as_float(x) : 0.0f;
        b = fabsf(b) < INFINITY ? b - __uint_as_float(y) : 0.0f;
        return x >> 16 | y;
    };
    hi = take(), mid = take(), lo = take();
}

// RN: rank rounded up to 8, 16, 32, 64 or 128; columns past the rank are zero.
// Clusters walk the tiles with the grid's stride; K is split over a cluster's CTAs,
// whose sums meet in shared memory: CTA z finishes the rows of the warps w with
// w % CTAs = z, adding the CTAs' fragments in order, scaling and splitting.
template <int RN>
__global__ void __launch_bounds__(kTileThreads) shrink_tile_kernel(const Adapter p) {
    extern __shared__ __align__(128) uint8_t stages[];
    constexpr int kChunks = kShrinkK / 8, kPass = kTileThreads / kChunks;  // rows copied at a time
    constexpr int kRegs = RN / 2;                                          // accumulators of a lane
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c = tid % kChunks, i_first = tid / kChunks;  // this thread copies chunk c of every kPass-th row
    pdl_wait();
    const int splits = p.splits, split = blockIdx.x % splits;  // a cluster's CTAs are neighbours
    const int tile_count = *p.tile_count;
    const int64_t k0 = split * p.split_k;
    const int64_t k1 = k0 + p.split_k < p.k ? k0 + p.split_k : p.k;
    const int steps = static_cast<int>((k1 - k0 + kShrinkK - 1) / kShrinkK);
    for (int item = blockIdx.x / splits; item < tile_count; item += gridDim.x / splits) {
        const int2 tile = p.tiles[item];
        const int key = p.keys[tile.x];
        if (key < 0) continue;  // rows without an adapter: the same for the whole cluster
        const bf16* rows[kTileRows / kPass];
#pragma unroll
        for (int j = 0; j < kTileRows / kPass; ++j) {
            const int i = i_first + j * kPass;
            rows[j] = p.x + static_cast<int64_t>(i < tile.y ? p.order[tile.x + i] : 0) * p.k + k0 + c * 8;
        }
        const bf16* a = p.a + (static_cast<int64_t>(key) * p.rank + i_first) * p.k + k0 + c * 8;
        auto load = [&](int slot, int step) {
            const uint32_t at = smem_addr(stages) + slot * shrink_stage_bytes<RN>();
            const int kc = step * kShrinkK;
            const bool in = k0 + kc + c * 8 < k1;
#pragma unroll
            for (int j = 0; j < kTileRows / kPass; ++j) {
                const int i = i_first + j * kPass;
                if (i < tile.y)  // what stands in the other rows is multiplied, and stored nowhere
                    copy16(at + stage_at(i, c), in ? rows[j] + kc : p.x, in);
            }
#pragma unroll
            for (int j = 0; j < (RN + kPass - 1) / kPass; ++j) {
                const int i = i_first + j * kPass;
                const bool here = in && i < p.rank;
                if (i < RN) copy16(at + kTileRows * kShrinkRow + stage_at(i, c),
                                   here ? a + static_cast<int64_t>(j * kPass) * p.k + kc : p.a, here);
            }
        };
        __syncthreads();  // the item before has read its stages
#pragma unroll
        for (int s = 0; s < kShrinkStages - 1; ++s) {
            if (s < steps) load(s, s);
            copy_commit();
        }
        float acc[RN / 8][4] = {}, sum[RN / 8][4] = {};
        int slot = 0, load_slot = kShrinkStages - 1;
        for (int step = 0; step < steps; ++step) {
            copy_wait<kShrinkStages - 2>();
            __syncthreads();  // this stage has landed everywhere, and the one before has been read
            if (step + kShrinkStages - 1 < steps) load(load_slot, step + kShrinkStages - 1);
            copy_commit();
            if (warp * 16 < tile.y) {
                const uint32_t xs = smem_addr(stages) + slot * shrink_stage_bytes<RN>();
                const uint32_t as = xs + kTileRows * kShrinkRow;
#pragma unroll
                for (int kk = 0; kk < kShrinkK / 16; ++kk) {
                    uint32_t xf[4];
                    ldmatrix4(xs + stage_at(warp * 16 + (lane & 15), kk * 2 + (lane >> 4)), xf);
                    if constexpr (RN == 8) {
                        uint32_t af[2];
                        ldmatrix2(as + stage_at(lane & 7, kk * 2 + ((lane >> 3) & 1)), af);
                        mma16816(acc[0], xf, af[0], af[1]);
                    } else {
#pragma unroll
                        for (int n0 = 0; n0 < RN; n0 += 16) {
                            uint32_t af[4];
                            ldmatrix4(as + stage_at(n0 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)), af);
                            mma16816(acc[n0 / 8], xf, af[0], af[1]);
                            mma16816(acc[n0 / 8 + 1], xf, af[2], af[3]);
                        }
                    }
                }
                if (step % kShrinkChunk == kShrinkChunk - 1) {
#pragma unroll
                    for (int j = 0; j < kRegs; ++j) {
                        sum[j / 4][j % 4] += acc[j / 4][j % 4];
                        acc[j / 4][j % 4] = 0.0f;
                    }
                }
            }
            if (++slot == kShrinkStages) slot = 0;
            if (++load_slot == kShrinkStages) load_slot = 0;
        }
#pragma unroll
        for (int j = 0; j < kRegs; ++j) acc[j / 4][j % 4] += sum[j / 4][j % 4];
        bool mine = warp * 16 < tile.y;
        if (splits > 1) {
            float* partial = reinterpret_cast<float*>(stages) + warp * kRegs * 32 + lane;  // [warp][register][lane]
            __syncthreads();  // the stages have been read
#pragma unroll
            for (int j = 0; j < kRegs; ++j) partial[j * 32] = acc[j / 4][j % 4];
            cluster_barrier();
            mine = mine && warp % splits == split;
            if (mine) {
                for (int z = 0; z < splits; ++z) {
                    float v[kRegs];  // all on their way before the first is added
#pragma unroll
                    for (int j = 0; j < kRegs; ++j) v[j] = __uint_as_float(load_peer(partial + j * 32, z));
#pragma unroll
                    for (int j = 0; j < kRegs; ++j)
                        acc[j / 4][j % 4] = z == 0 ? v[j] : acc[j / 4][j % 4] + v[j];
                }
            }
            cluster_barrier();  // everyone's sums have been read
        }
        if (mine) {
            const float scale = p.scale ? p.scale[key / p.experts] : 1.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = warp * 16 + (lane >> 2) + 8 * h;
                if (i >= tile.y) continue;
#pragma unroll
                for (int kk = 0; kk < rank_k<RN>() / 16; ++kk) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    uint2 lo = make_uint2(0, 0);
                    if (kk * 16 < p.rank)  // past the rank: zeros, not an infinite x times a zero
                        split2(acc[2 * kk][2 * h] * scale, acc[2 * kk][2 * h + 1] * scale, v.x, v.z, lo.x);
                    if constexpr (RN > 8)
                        if (kk * 16 + 8 < p.rank)
                            split2(acc[2 * kk + 1][2 * h] * scale, acc[2 * kk + 1][2 * h + 1] * scale, v.y, v.w, lo.y);
                    char* const to = s_pieces<RN>(p, tile.x + i, kk);
                    *piece_hi_mid(to, lane & 3) = v;
                    *piece_lo(to, lane & 3) = lo;
                }
            }
        }
    }
    copy_wait<0>();
}

constexpr int kExpandThreads = 128;                   // 4 x 16 rows
constexpr int kExpandStages = 2;
constexpr int kTileCols = 64;                         // rows of B per step: 64 columns, or 32 gate + 32 up
constexpr int kBaseStride = kTileCols * 2 + 16;       // bytes; the pads keep ldmatrix and row stores conflict-free
template <int RN> constexpr int b_stride() { return rank_k<RN>() * 2 + 16; }
template <int RN> constexpr int expand_ctas() { return RN <= 32 ? 6 : (RN <= 64 ? 4 : 2); }  // per SM
template <int RN> constexpr int expand_smem() {
    return kExpandStages * (kTileRows * kBaseStride + kTileCols * b_stride<RN>()) + rank_k<RN>() / 16 * kExpandThreads * 16;
}

// Two fp32 lanes in one register pair: one instruction for both.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t x, y, z;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(z) : "l"(x), "l"(y));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(z));
    return a;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t x, y, z;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(z) : "l"(x), "l"(y));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(z));
    return a;
}

// silu(g) u from the hardware's exponential and reciprocal: g log2 e is rounded
// once (|g| 2^-24), both are good to a few steps, so it is within (|g| + 8) 2^-23
// of the value, against 2^-8 of the rounding to bf16.  The sum 1 + e is taken a quarter
// as large: the reciprocal of more than 2^126 would be flushed to zero, for gates between
// -88.72 and -87.33.  Below, where e is infinite, the value is 0, as g / (1 + expf(-g)) is.
// (With expf, a division and single lanes the
// SwiGLU form of the expand kernel was bound by its instructions and took 1.7 times as
// long at 4096 tokens, 8 experts, top-2.)
__device__ __forceinline__ float2 fast_silu_times(float2 g, float2 u) {
    const float2 t = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = fma2(e, make_float2(0.25f, 0.25f), make_float2(0.25f, 0.25f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    return mul2(mul2(mul2(g, make_float2(0.25f, 0.25f)), r), u);
}

// Stretch q of the (tile, column block) pairs: the first gridDim.x stretches cover
// half of the pairs, the next as many half of the rest, and so on, down to
// kLeastStretch pairs (8 at least left a third of the CTAs without work in a small
// call).  Returns its first pair and its end.
constexpr int kLeastStretch = 2;
struct Stretch { int64_t x, y; };
__device__ __forceinline__ Stretch stretch_of(int64_t q, int64_t all) {
    const int64_t round = gridDim.x;
    int64_t first = 0;
    for (;;) {
        int64_t size = (all - first) / (2 * round);
        if (size <= kLeastStretch) {
            size = kLeastStretch;
        } else if (q >= round) {
            first += size * round;
            q -= round;
            continue;
        }
        first += q * size;
        return {min(first, all), min(first + size, all)};
    }
}

// CTAs claim stretches of the (tile, column block) pairs, long ones first, and walk
// them tile by tile: tiles differ in their rows, so equal shares end far apart
// (one share per CTA took 1.6 times as long at 4096 tokens, 8 experts of 14336,
// top-2), and short stretches alone pay for many starts.  A CTA's blocks of one
// tile form one cp.async pipeline whose stages hold the tile's base rows and the
// pair's rows of B; s stays as bf16 fragments in registers (hi and mid) and in shared
// memory (lo, written and read by the same lane: the registers decide how many CTAs an SM
// holds), and the accumulators start from base.
//
// Measured (a call less the same call with 8 columns): 172 us at that size (8192 rows
// -> 2 x 14336, rank 16: 710 MB through memory in this kernel, 108 us), 305 at 98304 rows
// of 2 x 1408, 2048 pairs, rank 32.  No unit is saturated (instruction issue 51-56 %, DRAM
// 42-49 %, tensor cores 13-35 %): the warps wait for their own chains and at the barrier.
// Five CTAs an SM at rank 32 or three at rank 64, with lo in registers' reach: the same or
// slower.  Measured with two parts of s (160 and 280 us): four warps a CTA and six CTAs an
// SM, because a barrier then holds up 64 columns and not 128 (4 and 20 us more with eight
// warps); B in the warps' registers instead of shared memory, with no barrier, 9 and 96
// more; three stages the same as two.
template <int RN, bool SWIGLU>
__global__ void __launch_bounds__(kExpandThreads, expand_ctas<RN>())
expand_tile_kernel(const Adapter p, int blocks) {
    constexpr int RK = rank_k<RN>();
    constexpr int kOut = SWIGLU ? kTileCols / 2 : kTileCols;  // output columns of a block
    constexpr int kHalves = SWIGLU ? 2 : 1;
    constexpr int kStage = kTileRows * kBaseStride + kTileCols * b_stride<RN>();
    constexpr int kChunks = RK / 8, kBRows = kExpandThreads / kChunks, kBCopies = kTileCols / kBRows;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cols = static_cast<int>(p.cols);
    // this thread's share of the base rows: one 16-byte chunk of rows i_first + 16 j
    const int c = (tid & 7) * 8, i_first = tid >> 3;
    const int c_col = SWIGLU ? c & 31 : c;  // its column inside the block
    const int b_q = tid % kChunks, b_n = tid / kChunks;  // and of B: chunk b_q of rows b_n + kBRows j
    const uint32_t base_to = i_first * kBaseStride + c * 2;
    const uint32_t b_to = kTileRows * kBaseStride + b_n * b_stride<RN>() + b_q * 16;
    // this lane's first row of B for ldmatrix, and its first pair of base, inside a stage
    const uint32_t b_lane = kTileRows * kBaseStride +
                            ((lane & 7) + ((lane >> 4) << 3)) * b_stride<RN>() + ((lane >> 3) & 1) * 16;
    const int r0 = warp * 16 + (lane >> 2);
    const int base_lane = r0 * kBaseStride + (lane & 3) * 4;
    constexpr int kPieces = kOut / 8, kPer = 32 / kPieces;  // out: 16-byte pieces of a row; rows at a time
    const int out_row = warp * 16 + lane / kPieces, out_col = (lane % kPieces) * 8;
    const int out_lane = out_row * kBaseStride + out_col * 2;
    uint4* const lo_s = reinterpret_cast<uint4*>(smem + kExpandStages * kStage) + tid;  // [kk][thread]
    if (b_q * 8 >= p.rank) {  // past the rank B is zero: written once, never copied over
#pragma unroll
        for (int s = 0; s < kExpandStages; ++s)
#pragma unroll
            for (int j = 0; j < kBCopies; ++j)
                *reinterpret_cast<uint4*>(smem + s * kStage + b_to + j * kBRows * b_stride<RN>()) = make_uint4(0, 0, 0, 0);
    }
    pdl_trigger();
    pdl_wait();
    __shared__ int claimed[2];
    const int64_t all = static_cast<int64_t>(*p.tile_count) * blocks;
    Stretch stretch = stretch_of(blockIdx.x, all);
    int turn = 0;
    if (tid == 0) claimed[0] = atomicAdd(p.tile_count + 1, 1);
    while (stretch.x < all) {
        const int2 tile = p.tiles[stretch.x / blocks];
        const int first_block = static_cast<int>(stretch.x % blocks);
        const int count = static_cast<int>(min(static_cast<int64_t>(blocks - first_block), stretch.y - stretch.x));
        const int key = p.keys[tile.x];
        // Blocks in which a column of this thread's lies inside the row: its copies and stores
        // stop there, so a step compares step numbers only.
        const int col0 = first_block * kOut, width = cols - col0;
        const auto blocks_with = [&](int column) { return width > column ? (width - column + kOut - 1) / kOut : 0; };
        const int base_blocks = blocks_with(c_col), base_rows = (tile.y - i_first + 15) / 16;
        const bf16* base[kTileRows / 16];
#pragma unroll
        for (int j = 0; j < kTileRows / 16; ++j) {
            const int i = i_first + 16 * j;
            base[j] = p.base + static_cast<int64_t>(i < tile.y ? p.order[tile.x + i] : 0) * p.n + col0 + c_col +
                      (SWIGLU && c >= 32 ? cols : 0);
        }
        const bf16* b[kBCopies];
        int b_blocks[kBCopies];
#pragma unroll
        for (int j = 0; j < kBCopies; ++j) {
            const int n = b_n + kBRows * j, column = SWIGLU ? n & 31 : n;
            b[j] = p.b + (key < 0 ? 0 : (static_cast<int64_t>(key) * p.n + col0 + column + (SWIGLU && n >= 32 ? cols : 0)) *
                                            p.rank + b_q * 8);
            b_blocks[j] = key < 0 || b_q * 8 >= p.rank ? 0 : blocks_with(column);
        }
        auto load = [&](uint32_t stage, int step) {
            const uint32_t at = smem_addr(smem) + stage;
            if (step < base_blocks) {
#pragma unroll
                for (int j = 0; j < kTileRows / 16; ++j)
                    if (j < base_rows) copy16(at + base_to + 16 * j * kBaseStride, base[j], true);
            }
#pragma unroll
            for (int j = 0; j < kTileRows / 16; ++j) base[j] += kOut;
#pragma unroll
            for (int j = 0; j < kBCopies; ++j) {
                if (step < b_blocks[j]) copy16(at + b_to + j * kBRows * b_stride<RN>(), b[j], true);
                b[j] += kOut * p.rank;
            }
        };
        __syncthreads();  // the item before is done with its stages
        load(0, 0);
        copy_commit();

        bf16* out[16 / kPer];
        int out_blocks[16 / kPer];
#pragma unroll
        for (int j = 0; j < 16 / kPer; ++j) {
            const int i = out_row + j * kPer;
            out[j] = p.out + static_cast<int64_t>(i < tile.y ? p.order[tile.x + i] : 0) * p.cols + col0 + out_col;
            out_blocks[j] = i < tile.y ? blocks_with(out_col) : 0;
        }

        // s of this warp's 16 rows as fragments
        uint32_t hi[RK / 16][4] = {}, mid[RK / 16][4] = {};
        if (key >= 0) {
#pragma unroll
            for (int kk = 0; kk < RK / 16; ++kk) {
                uint32_t lo[4] = {};
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (r0 + 8 * h < tile.y) {
                        char* const from = s_pieces<RN>(p, static_cast<int64_t>(tile.x) + r0 + 8 * h, kk);
                        const uint4 v = *piece_hi_mid(from, lane & 3);
                        const uint2 w = *piece_lo(from, lane & 3);
                        hi[kk][h] = v.x, hi[kk][2 + h] = v.y, mid[kk][h] = v.z, mid[kk][2 + h] = v.w;
                        lo[h] = w.x, lo[2 + h] = w.y;
                    }
                lo_s[kk * kExpandThreads] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }

        uint32_t stage = 0;
        for (int step = 0; step < count; ++step) {
            copy_wait<0>();
            __syncthreads();  // this stage has landed everywhere, and the one before is done with
            if (step + 1 < count) load(kStage - stage, step + 1);
            copy_commit();
            uint8_t* const base_s = smem + stage;
            if (warp * 16 < tile.y) {
                if (key >= 0) {
                    // 16 columns at a time (with SwiGLU 16 gate and the matching 16 up columns), so
                    // few accumulators live at once; they start from base and end in its place
                    // (conflict-free)
                    const uint32_t bs = smem_addr(base_s) + b_lane;
                    uint8_t* const mine = base_s + base_lane;
#pragma unroll
                    for (int f = 0; f < kOut; f += 16) {
                        float acc[kHalves][2][4];
                        const auto word = [&](int h, int q) {
                            return reinterpret_cast<uint32_t*>(mine + h * 8 * kBaseStride + (f + q * 8) * 2);
                        };
#pragma unroll
                        for (int g = 0; g < kHalves; ++g)
#pragma unroll
                            for (int q = 0; q < 2; ++q)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const uint32_t v = word(h, q)[g * 16];  // up: 64 bytes further
                                    acc[g][q][2 * h] = bf16_lo(v), acc[g][q][2 * h + 1] = bf16_hi(v);
                                }
#pragma unroll
                        for (int kk = 0; kk < RK / 16; ++kk) {
                            const uint4 w = lo_s[kk * kExpandThreads];
                            const uint32_t lo[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int g = 0; g < kHalves; ++g) {
                                uint32_t bf[4];
                                ldmatrix4(bs + (f + g * 32) * b_stride<RN>() + kk * 32, bf);
                                mma16816(acc[g][0], lo, bf[0], bf[1]);
                                mma16816(acc[g][1], lo, bf[2], bf[3]);
                                mma16816(acc[g][0], mid[kk], bf[0], bf[1]);
                                mma16816(acc[g][1], mid[kk], bf[2], bf[3]);
                                mma16816(acc[g][0], hi[kk], bf[0], bf[1]);
                                mma16816(acc[g][1], hi[kk], bf[2], bf[3]);
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                float2 y = make_float2(acc[0][q][2 * h], acc[0][q][2 * h + 1]);
                                if constexpr (SWIGLU)
                                    y = fast_silu_times(y, make_float2(acc[1][q][2 * h], acc[1][q][2 * h + 1]));
                                *word(h, q) = pack2(y.x, y.y);
                            }
                    }
                } else if constexpr (SWIGLU) {
                    // without an adapter: the bits of swiglu_kernel; two rows, a pair of columns a lane
                    uint8_t* pair = base_s + (warp * 16 + (lane >> 4)) * kBaseStride + (lane & 15) * 4;
#pragma unroll 4
                    for (int i = 0; i < 16; i += 2, pair += 2 * kBaseStride) {
                        uint32_t* at = reinterpret_cast<uint32_t*>(pair);
                        const uint32_t g = *at, u = at[16];
                        *at = pack2(silu_times(bf16_lo(g), bf16_lo(u)), silu_times(bf16_hi(g), bf16_hi(u)));
                    }
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 16 / kPer; ++j) {
                    if (step < out_blocks[j])
                        *reinterpret_cast<uint4*>(out[j]) =
                            *reinterpret_cast<const uint4*>(base_s + out_lane + j * kPer * kBaseStride);
                    out[j] += kOut;
                }
            }
            stage = kStage - stage;
        }
        stretch.x += count;
        if (stretch.x == stretch.y) {  // the claim was made a stretch ago; make the next one now
            stretch = stretch_of(static_cast<int64_t>(gridDim.x) + claimed[turn], all);
            turn ^= 1;
            if (tid == 0) claimed[turn] = atomicAdd(p.tile_count + 1, 1);
        }
    }
    copy_wait<0>();
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

// Which form.  Measured in graphs (us, few-rows form / tiles), 8 experts, rank 16, down
// projection 14336 -> 4096: one adapter, 128 rows 13 / 25, 264 rows 23 / 27, 512 rows
// 40 / 30, 1024 rows 77 / 32; 64 adapters, a row's own each, 264 rows 28 / 83, 512 rows
// 47 / 111, 1024 rows 83 / 137, 2048 rows 156 / 160.  (Rank 8 to 128 and 4096 -> 28672
// cross over near the same places.)  Where the rows are no more than twice the pairs that
// they may fall on, tiles may hold few rows each.
// The rule goes by what the host knows, the rows' capacity and the adapters loaded, not by
// the rows and pairs in use, which only the device knows.  It costs most where many
// adapters are loaded and all rows use one: 64 loaded, 512 rows 40 / 30, 1024 rows 77 / 33;
// and a few tokens over very many experts, whose padded spans count as rows, take tiles.
constexpr int64_t kFewRows = 256;
constexpr int64_t kFewRowsScattered = 1024;
bool few_rows_form(int64_t rows, int adapters, int experts) {
    return rows <= kFewRows ||
           (rows <= kFewRowsScattered && rows <= 2ll * adapters * experts);
}

struct Shape {
    bool few, cluster_sort;
    int splits;
    int64_t split_k, chunk_rows, table, order, keys, tiles, s, total;
    int chunks;
};

int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Twice the SMs: 98 tiles of K = 2048, rank 64: 14.9 us with two CTAs a tile, 18.6 with one,
// 19.7 with four (which no longer fit at once).
constexpr int64_t kSpread = 2;
Shape shape_of(int64_t rows, int64_t k, int rank, int adapters, int experts, int sms) {
    Shape f = {};
    f.few = few_rows_form(rows, adapters, experts);
    if (f.few) {
        f.split_k = kRowsSplitK;
        f.splits = static_cast<int>((k + kRowsSplitK - 1) / kRowsSplitK);
        f.total = round256(rows * rank * 4 * f.splits);
        return f;
    }
    // K is split over clusters of 1, 2 or 4 CTAs: as long as the clusters still find a place
    // on the SMs at once, and each CTA keeps at least 512 elements.
    const int64_t tiles = (rows + kTileRows - 1) / kTileRows;
    int64_t splits = 1;
    while (splits < 4 && tiles * splits * 2 <= kSpread * sms && k >= splits * 2 * 512) splits *= 2;
    f.split_k = ((k + splits - 1) / splits + kShrinkK - 1) / kShrinkK * kShrinkK;
    f.splits = static_cast<int>(splits);  // the last ones may be empty
    // One cluster sorts up to 8192 rows: 5003 rows in 8.6 us against 10.0 in three launches
    // (8256 rows, two rounds a CTA: 11.0 against 10.3).
    f.cluster_sort = rows <= kClusterChunks * kClusterChunkRows;
    const int64_t spread = (f.cluster_sort ? kClusterChunks : kMaxChunks) * static_cast<int64_t>(kSortThreads);
    f.chunk_rows = (rows + spread - 1) / spread * kSortThreads;
    f.chunks = static_cast<int>((rows + f.chunk_rows - 1) / f.chunk_rows);
    f.table = 0;
    f.order = round256(static_cast<int64_t>(adapters + 2) * f.chunks * 4);
    f.keys = f.order + round256(rows * 4);
    f.tiles = f.keys + round256(rows * 4);
    f.s = f.tiles + round256(rows * 8 + 256);  // the count, then at most one tile per row
    f.total = f.s + round256(rows * (padded_rank(rank) < 16 ? 1 : padded_rank(rank) / 16) * kPieceBytes);
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

// A dependent launch of `ctas` CTAs in clusters of `cluster`.  With `fit`, at most as
// many clusters as the device holds at once (looked up once, into *fit): a walk with
// the grid's stride would else leave shares to clusters that start when the others
// are done, which doubled the shrink kernel's time at 443 small tiles.
template <typename... Params, typename... Args>
cudaError_t launch_clusters(void (*kernel)(Params...), int ctas, int cluster, int threads, int smem,
                            cudaStream_t stream, int* fit, Args&&... args) {
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attribute[1].val.clusterDim.y = 1;
    attribute[1].val.clusterDim.z = 1;
    config.gridDim = dim3(static_cast<unsigned>(ctas));
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = static_cast<size_t>(smem);
    config.stream = stream;
    config.attrs = attribute;
    config.numAttrs = 2;
    if (fit) {
        if (*fit == 0) MOE_CUDA_TRY(cudaOccupancyMaxActiveClusters(fit, kernel, &config));
        if (*fit > 0 && ctas > *fit * cluster) config.gridDim = dim3(static_cast<unsigned>(*fit * cluster));
    }
    return cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
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
cudaError_t tiles(const Adapter& p, const Shape& f, int sms, cudaStream_t stream) {
    static bool order_ok[2][64] = {}, shrink_ok[64] = {}, expand_ok[64] = {};
    const int buckets = p.adapters + 2;
    const int order_smem = (32 * (buckets | 1) + 3 * buckets) * 4;
    constexpr int kOrderMost = (32 * ((kMaxAdapters + 2) | 1) + 3 * (kMaxAdapters + 2)) * 4;
    constexpr int kShrinkSmem = kShrinkStages * shrink_stage_bytes<RN>();
    MOE_CUDA_TRY(allow_smem(f.cluster_sort ? order_kernel<true> : order_kernel<false>, kOrderMost,
                            order_ok[f.cluster_sort]));
    MOE_CUDA_TRY(allow_smem(shrink_tile_kernel<RN>, kShrinkSmem, shrink_ok));
    MOE_CUDA_TRY(allow_smem(expand_tile_kernel<RN, SWIGLU>, expand_smem<RN>(), expand_ok));
    const bool none = SWIGLU || p.out != p.base;
    if (f.cluster_sort) {
        MOE_CUDA_TRY(launch_clusters(order_kernel<true>, f.chunks, f.chunks, kSortThreads, order_smem, stream,
                                     nullptr, p, f.chunk_rows, none));
    } else {
        MOE_CUDA_TRY(launch_dependent(count_kernel, dim3(f.chunks), dim3(kSortThreads), buckets * 4, stream, p,
                                      f.chunk_rows));
        MOE_CUDA_TRY(launch_dependent(order_kernel<false>, dim3(f.chunks), dim3(kSortThreads), order_smem, stream,
                                      p, f.chunk_rows, none));
        MOE_CUDA_TRY(launch_dependent(tiles_kernel, dim3(static_cast<unsigned>((p.rows + 255) / 256)), dim3(256),
                                      0, stream, p, none));
    }
    const auto resident = [&](int smem_bytes, int threads_most) {
        const int fit = 227 * 1024 / (smem_bytes + 1024);
        return static_cast<int64_t>(sms) * (fit < threads_most ? fit : threads_most);
    };
    static int shrink_fit[5][64] = {};  // by splits
    int device = 0;
    MOE_CUDA_TRY(cudaGetDevice(&device));
    const int64_t most = resident(kShrinkSmem, 4) / f.splits;
    MOE_CUDA_TRY(launch_clusters(shrink_tile_kernel<RN>, static_cast<int>((p.rows < most ? p.rows : most) * f.splits),
                                 f.splits, kTileThreads, kShrinkSmem, stream, &shrink_fit[f.splits][device & 63], p));
    const int out_cols = SWIGLU ? kTileCols / 2 : kTileCols;
    const int blocks = static_cast<int>((p.cols + out_cols - 1) / out_cols);
    const int64_t expand_most = resident(expand_smem<RN>(), expand_ctas<RN>());
    return launch_dependent(expand_tile_kernel<RN, SWIGLU>, dim3(static_cast<unsigned>(expand_most)),
                            dim3(kExpandThreads), expand_smem<RN>(), stream, p, blocks);
}

template <bool SWIGLU>
cudaError_t many_rows(const Adapter& p, const Shape& f, int sms, cudaStream_t stream) {
    switch (padded_rank(p.rank)) {
        case 8: return tiles<8, SWIGLU>(p, f, sms, stream);
        case 16: return tiles<16, SWIGLU>(p, f, sms, stream);
        case 32: return tiles<32, SWIGLU>(p, f, sms, stream);
        case 64: return tiles<64, SWIGLU>(p, f, sms, stream);
        default: return tiles<128, SWIGLU>(p, f, sms, stream);
    }
}

}  // namespace

cudaError_t adapter_scratch_bytes(int64_t rows, int64_t k, int rank, int adapters, int experts,
                                  int64_t* bytes) {
    int sms = 0;
    MOE_CUDA_TRY(device_sms(&sms));
    *bytes = shape_of(rows, k, rank, adapters, experts, sms).total;
    return cudaSuccess;
}

cudaError_t launch_adapter(const void* base, const void* x, const void* a, const void* b,
                           const float* scale, const int32_t* row_adapters, const int32_t* offsets,
                           void* out, int64_t rows, int64_t k, int64_t n, int rank, int adapters,
                           int experts, bool swiglu, void* scratch, cudaStream_t stream) {
    if (rows == 0) return cudaSuccess;
    int sms = 0;
    MOE_CUDA_TRY(device_sms(&sms));
    const Shape f = shape_of(rows, k, rank, adapters, experts, sms);
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
    p.tile_count = reinterpret_cast<int32_t*>(at + f.tiles);
    p.tiles = reinterpret_cast<int2*>(at + f.tiles + 256);
    p.s = reinterpret_cast<float*>(at + f.s);
    p.splits = f.splits;
    p.split_k = f.split_k;
    if (f.few) return swiglu ? few_rows<true>(p, stream) : few_rows<false>(p, stream);
    return swiglu ? many_rows<true>(p, f, sms, stream) : many_rows<false>(p, f, sms, stream);
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
