// Load-balance loss of a router, its per-expert counts and its gradient.  No
// counterpart in the reference, whose block is forward-only.
//
//   z = logits + bias, p = softmax(z) over the E experts
//   counts[e] = ids equal to e in the V tokens that count, f[e] = counts[e] / (V K)
//   loss = c E sum_e f[e] mean_t p[t,e]
//   dloss/dlogits[t,e] = (c E / V) p[t,e] (f[e] - sum_j f[j] p[t,j])
//
// (f does not depend on the logits.)  A row whose scores are all -inf has
// p = 0; a token that the mask leaves out is not read and has gradient 0.
//
// Both passes are bound by reading (and writing) the logits once.  A token's E
// scores lie in the registers of a group of 8, 16 or 32 lanes; a lane keeps the
// running sum of p for its own experts over all tokens that its group takes, so
// the sum over tokens needs no atomics.  Each CTA takes one fixed, contiguous
// range of tokens; its sums go to its own row of the scratch, and a second,
// dependent launch of one cluster adds the rows in a fixed order: the loss has the
// same bits on every run.  Integer counts are added with shared-memory atomics
// (order-free).
#include "common.cuh"
#include "launch.h"

namespace moe {
namespace {

constexpr int kThreads = 512;
constexpr int kFinishThreads = 1024;

// Lanes per token and scores per lane: VPL * G >= E.
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// Expert of a lane's i-th score: VPL of them, in runs of VEC neighbours that are
// loaded and stored as one vector.
template <int G, int VEC>
__device__ __forceinline__ int expert_at(int lane, int i) {
    return (lane + G * (i / VEC)) * VEC + i % VEC;
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Run { T v[VEC]; };

// One token's scores; experts past E (a multiple of VEC) are -inf.
template <int DT, int G, int VPL, int VEC>
__device__ __forceinline__ void load_scores(const typename Elem<DT>::T* __restrict__ row,
                                            const float (&bias)[VPL], int lane, int experts,
                                            bool valid, float (&z)[VPL]) {
#pragma unroll
    for (int i = 0; i < VPL; i += VEC) {
        const int e = expert_at<G, VEC>(lane, i);
        if (valid && e < experts) {
            const auto run = *reinterpret_cast<const Run<typename Elem<DT>::T, VEC>*>(row + e);
#pragma unroll
            for (int j = 0; j < VEC; ++j) z[i + j] = Elem<DT>::load(run.v[j]) + bias[i + j];
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) z[i + j] = -INFINITY;
        }
    }
}

// z -> softmax(z) in place (all zeros when no score is above -inf; a NaN or
// +inf among the scores makes the row NaN).  With one score a lane, dividing costs
// nothing that shows, and each p is the nearest fp32 value to its quotient.
template <int G, int VPL>
__device__ __forceinline__ void softmax(float (&z)[VPL]) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) top = fmaxf(top, z[i]);
    top = group_max<G>(top);
    if (top == -INFINITY) top = 0.0f;
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        z[i] = expf(z[i] - top);
        total += z[i];
    }
    total = group_sum<G>(total);
    if constexpr (VPL == 1) {
        z[0] = total == 0.0f ? 0.0f : z[0] / total;
    } else {
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < VPL; ++i) z[i] *= inv;
    }
}

// Tokens that a group of lanes works on at once: their loads and shuffles overlap.
template <int VPL> constexpr int tokens_at_once() { return VPL >= 8 ? 2 : 4; }

template <int DT, int G, int VPL, int VEC>
__global__ void __launch_bounds__(kThreads, 2)
balance_forward_kernel(const typename Elem<DT>::T* __restrict__ logits,
                       const float* __restrict__ bias, const int32_t* __restrict__ ids,
                       const uint8_t* __restrict__ mask, float* __restrict__ sums,
                       int32_t* __restrict__ part_counts, int64_t tokens, int experts, int topk,
                       int64_t per_cta) {
    constexpr int kGroups = kThreads / G;       // tokens in flight per CTA
    constexpr int kWarps = kThreads / 32;
    constexpr int kAtOnce = tokens_at_once<VPL>();
    __shared__ float warp_sums[kWarps][G * VPL];
    __shared__ int32_t counts[G * VPL + 1];     // [E] and the tokens that count
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    pdl_trigger();
    for (int e = threadIdx.x; e <= experts; e += kThreads) counts[e] = 0;
    pdl_wait();
    float b[VPL], acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = expert_at<G, VEC>(lane, i);
        b[i] = bias && e < experts ? bias[e] : 0.0f;
        acc[i] = 0.0f;
    }
    __syncthreads();

    const int64_t t0 = blockIdx.x * per_cta;
    const int64_t t1 = t0 + per_cta < tokens ? t0 + per_cta : tokens;
    // the counts first: their loads overlap those of the scores
    const int n = t1 > t0 ? static_cast<int>((t1 - t0) * topk) : 0;
    for (int p0 = threadIdx.x; p0 < n; p0 += 4 * kThreads) {
        int e[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int p = p0 + u * kThreads;
            e[u] = p < n && (!mask || mask[t0 + static_cast<unsigned>(p) / static_cast<unsigned>(topk)])
                       ? ids[t0 * topk + p] : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (e[u] >= 0 && e[u] < experts) atomicAdd(&counts[e[u]], 1);
    }
    // whole warps stay in the loop: the shuffles name every lane
    for (int64_t base = t0; base < t1; base += kGroups * kAtOnce) {
        float z[kAtOnce][VPL];
        int valid_here = 0;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int64_t t = base + u * kGroups + group;
            const bool valid = t < t1 && (!mask || mask[t]);
            load_scores<DT, G, VPL, VEC>(logits + t * experts, b, lane, experts, valid, z[u]);
            valid_here += valid;
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            if (base + u * kGroups >= t1) break;
            softmax<G, VPL>(z[u]);
#pragma unroll
            for (int i = 0; i < VPL; ++i) acc[i] += z[u][i];
        }
        if (valid_here && lane == 0) atomicAdd(&counts[experts], valid_here);
    }

    // The warp's groups, then the CTA's warps, in a fixed order.
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
#pragma unroll
        for (int off = 16; off >= G; off >>= 1)
            acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], off);
        if (threadIdx.x % 32 < G) warp_sums[threadIdx.x / 32][expert_at<G, VEC>(lane, i)] = acc[i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += kThreads) {
        if (e < experts) {
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) total += warp_sums[w][e];
            sums[static_cast<int64_t>(blockIdx.x) * experts + e] = total;
        }
        part_counts[static_cast<int64_t>(blockIdx.x) * (experts + 1) + e] = counts[e];
    }
}

__device__ __forceinline__ uint32_t load_peer(const void* local, uint32_t rank) {
    uint32_t address = static_cast<uint32_t>(__cvta_generic_to_shared(local)), value;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(address), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(value) : "r"(address) : "memory");
    return value;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One cluster (of one CTA for few parts): every CTA adds a stretch of the parts in
// order, the first adds the CTAs' sums in order from their shared memory and writes
// counts[E], counted[0] = V, both once more into kept, and the loss.
__global__ void __launch_bounds__(kFinishThreads)
balance_finish_kernel(const float* __restrict__ sums, const int32_t* __restrict__ part_counts,
                      int parts, int experts, int topk, float coefficient, float* __restrict__ loss,
                      int32_t* __restrict__ counts, int32_t* __restrict__ counted,
                      int32_t* __restrict__ kept) {
    constexpr int kMax = kFinishThreads;
    __shared__ float s_sum[kMax];
    __shared__ int32_t s_count[kMax];
    __shared__ int32_t s_valid;
    pdl_trigger();
    pdl_wait();
    // thread (slice, e) of this CTA's stretch
    const int slices = kMax / (experts + 1);
    const int slice = threadIdx.x / (experts + 1), e = threadIdx.x % (experts + 1);
    const int all_slices = slices * gridDim.x, my_slice = blockIdx.x * slices + slice;
    float total = 0.0f;
    int32_t count = 0;
    if (slice < slices) {
        const int from = static_cast<int>(static_cast<int64_t>(parts) * my_slice / all_slices);
        const int to = static_cast<int>(static_cast<int64_t>(parts) * (my_slice + 1) / all_slices);
#pragma unroll 8
        for (int c = from; c < to; ++c) {
            if (e < experts) total += sums[static_cast<int64_t>(c) * experts + e];
            count += part_counts[static_cast<int64_t>(c) * (experts + 1) + e];
        }
    }
    s_sum[threadIdx.x] = total;
    s_count[threadIdx.x] = count;
    __syncthreads();
    if (slice == 0) {
        for (int s = 1; s < slices; ++s) {
            total += s_sum[s * (experts + 1) + e];
            count += s_count[s * (experts + 1) + e];
        }
        s_sum[e] = total;
        s_count[e] = count;
    }
    cluster_barrier();
    if (blockIdx.x == 0) {
        if (slice == 0) {
            for (unsigned c = 1; c < gridDim.x; ++c) {
                total += __uint_as_float(load_peer(&s_sum[e], c));
                count += static_cast<int32_t>(load_peer(&s_count[e], c));
            }
            kept[e] = count;
            if (e < experts) counts[e] = count;
            else {
                counted[0] = count;
                s_valid = count;
            }
        }
        __syncthreads();
        if (slice == 0 && e < experts) s_sum[e] = total * static_cast<float>(count);
        __syncthreads();
        if (threadIdx.x < 32) {  // sum_e f[e] mean p[e], in expert order per lane
            float v = 0.0f;
            for (int i = threadIdx.x; i < experts; i += 32) v += s_sum[i];
            v = group_sum<32>(v);
            if (threadIdx.x == 0) {
                const float n = static_cast<float>(s_valid);
                loss[0] = s_valid == 0 ? 0.0f
                                       : coefficient * static_cast<float>(experts) *
                                             (v / n / n / static_cast<float>(topk));
            }
        }
    }
    cluster_barrier();  // no CTA leaves while the first may still read its sums
}

template <int DT, int G, int VPL, int VEC>
__global__ void __launch_bounds__(kThreads, 2)
balance_backward_kernel(const typename Elem<DT>::T* __restrict__ logits,
                        const float* __restrict__ bias, const uint8_t* __restrict__ mask,
                        const int32_t* __restrict__ counts, const int32_t* __restrict__ counted,
                        const float* __restrict__ grad_loss, float coefficient,
                        typename Elem<DT>::T* __restrict__ grad, int64_t tokens, int experts,
                        int topk) {
    const int lane = threadIdx.x % G;
    const int64_t groups = static_cast<int64_t>(gridDim.x) * (kThreads / G);
    pdl_trigger();
    pdl_wait();
    const float n = static_cast<float>(counted[0]);
    const float factor = n > 0.0f ? grad_loss[0] * (coefficient * static_cast<float>(experts)) / n : 0.0f;
    float b[VPL], f[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = expert_at<G, VEC>(lane, i);
        b[i] = bias && e < experts ? bias[e] : 0.0f;
        f[i] = e < experts && n > 0.0f ? static_cast<float>(counts[e]) / (n * static_cast<float>(topk)) : 0.0f;
    }
    constexpr int kAtOnce = tokens_at_once<VPL>();
    const int in_warp = (threadIdx.x % 32) / G;
    const int64_t first = (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x) / G - in_warp;
    for (int64_t t0 = first; t0 < tokens; t0 += groups * kAtOnce) {
        float z[kAtOnce][VPL];
        bool inside[kAtOnce], valid[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int64_t t = t0 + in_warp + u * groups;
            inside[u] = t < tokens;
            valid[u] = inside[u] && (!mask || mask[t]);
            load_scores<DT, G, VPL, VEC>(logits + t * experts, b, lane, experts, valid[u], z[u]);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int64_t t = t0 + in_warp + u * groups;
            if (t0 + u * groups >= tokens) break;
            softmax<G, VPL>(z[u]);
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) dot = __fadd_rn(dot, __fmul_rn(z[u][i], f[i]));
            dot = group_sum<G>(dot);
#pragma unroll
            for (int i = 0; i < VPL; i += VEC) {
                const int e = expert_at<G, VEC>(lane, i);
                Run<typename Elem<DT>::T, VEC> run;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    run.v[j] = Elem<DT>::store(
                        valid[u] ? (factor * z[u][i + j]) * (f[i + j] - dot) : 0.0f);
                if (inside[u] && e < experts)
                    *reinterpret_cast<Run<typename Elem<DT>::T, VEC>*>(grad + t * experts + e) = run;
            }
        }
    }
}

cudaError_t sm_count(int* sms) {
    static int cached[64] = {};
    int device = 0;
    MOE_CUDA_TRY(cudaGetDevice(&device));
    if (cached[device & 63] == 0)
        MOE_CUDA_TRY(cudaDeviceGetAttribute(&cached[device & 63], cudaDevAttrMultiProcessorCount, device));
    *sms = cached[device & 63];
    return cudaSuccess;
}

// The scratch: counts and V once more for the backward pass (the caller may change its
// counts before that), then the CTAs' sums and counts.
int64_t kept_bytes(int experts) { return (4 * (experts + 1) + 15) / 16 * 16; }

// CTAs of the forward pass: two per SM at most (each costs the finishing launch a
// row to add), at least one token per group of lanes each.
constexpr int kMaxParts = 512;
int balance_parts(int64_t tokens, int group, int sms) {
    const int64_t rounds = (tokens + kThreads / group - 1) / (kThreads / group);
    const int64_t most = 2 * sms < kMaxParts ? 2 * sms : kMaxParts;
    return static_cast<int>(rounds < 1 ? 1 : (rounds < most ? rounds : most));
}

struct BalanceArgs {
    const void* logits;
    const float* bias;
    const int32_t* ids;
    const uint8_t* mask;
    int64_t tokens;
    int experts, topk;
    float coefficient;
    float* loss;
    int32_t *counts, *counted;
    void* scratch;
    const float* grad_loss;
    void* grad;
    cudaStream_t stream;
};

template <int DT, int G, int VPL, int VEC>
cudaError_t forward(const BalanceArgs& a) {
    using T = typename Elem<DT>::T;
    int sms = 0;
    MOE_CUDA_TRY(sm_count(&sms));
    const int parts = balance_parts(a.tokens, G, sms);
    const int64_t per_cta = (a.tokens + parts - 1) / parts;
    int32_t* kept = static_cast<int32_t*>(a.scratch);
    float* sums = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kept_bytes(a.experts));
    int32_t* part_counts = reinterpret_cast<int32_t*>(sums + static_cast<int64_t>(kMaxParts) * a.experts);
    MOE_CUDA_TRY(launch_dependent(balance_forward_kernel<DT, G, VPL, VEC>, dim3(parts), dim3(kThreads), 0,
                                  a.stream, static_cast<const T*>(a.logits), a.bias, a.ids, a.mask,
                                  sums, part_counts, a.tokens, a.experts, a.topk, per_cta));
    // 148 rows of 256 experts took one CTA 8.8 us; eight take 6.8 for 296.
    const unsigned cluster = static_cast<int64_t>(parts) * a.experts > 2048 ? 8 : 1;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = cluster;
    attribute[1].val.clusterDim.y = 1;
    attribute[1].val.clusterDim.z = 1;
    config.gridDim = dim3(cluster);
    config.blockDim = dim3(kFinishThreads);
    config.stream = a.stream;
    config.attrs = attribute;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, balance_finish_kernel, static_cast<const float*>(sums),
                              static_cast<const int32_t*>(part_counts), parts, a.experts, a.topk,
                              a.coefficient, a.loss, a.counts, a.counted, kept);
}

template <int DT, int G, int VPL, int VEC>
cudaError_t backward(const BalanceArgs& a) {
    using T = typename Elem<DT>::T;
    int sms = 0;
    MOE_CUDA_TRY(sm_count(&sms));
    const int64_t rounds = (a.tokens + kThreads / G - 1) / (kThreads / G);
    const int64_t most = 2 * static_cast<int64_t>(sms);
    return launch_dependent(balance_backward_kernel<DT, G, VPL, VEC>,
                            dim3(static_cast<unsigned>(rounds < most ? rounds : most)), dim3(kThreads),
                            0, a.stream, static_cast<const T*>(a.logits), a.bias, a.mask, a.counts,
                            a.counted, a.grad_loss, a.coefficient, static_cast<T*>(a.grad), a.tokens,
                            a.experts, a.topk);
}

template <int DT, bool kBackward>
cudaError_t by_experts(const BalanceArgs& a) {
    auto run = [&](auto g, auto v, auto w) {
        if constexpr (kBackward) return backward<DT, g(), v(), w()>(a);
        else return forward<DT, g(), v(), w()>(a);
    };
    // Rows of a multiple of four experts on aligned pointers: vectors of four.
    constexpr uintptr_t kRun = 4 * sizeof(typename Elem<DT>::T);
    const bool fours = a.experts % 4 == 0 && reinterpret_cast<uintptr_t>(a.logits) % kRun == 0 &&
                       reinterpret_cast<uintptr_t>(a.grad) % kRun == 0;
#define MOE_INT(n) std::integral_constant<int, n>{}
    if (a.experts <= 8) return run(MOE_INT(8), MOE_INT(1), MOE_INT(1));
    if (a.experts <= 16) return run(MOE_INT(16), MOE_INT(1), MOE_INT(1));
    if (a.experts <= 32) return run(MOE_INT(32), MOE_INT(1), MOE_INT(1));
    if (fours) {
        if (a.experts <= 64) return run(MOE_INT(16), MOE_INT(4), MOE_INT(4));
        if (a.experts <= 128) return run(MOE_INT(32), MOE_INT(4), MOE_INT(4));
        return run(MOE_INT(32), MOE_INT(8), MOE_INT(4));
    }
    if (a.experts <= 64) return run(MOE_INT(32), MOE_INT(2), MOE_INT(1));
    if (a.experts <= 128) return run(MOE_INT(32), MOE_INT(4), MOE_INT(1));
    return run(MOE_INT(32), MOE_INT(8), MOE_INT(1));
#undef MOE_INT
}

template <bool kBackward>
cudaError_t by_dtype(int dtype, const BalanceArgs& a) {
    if (dtype == kF32) return by_experts<kF32, kBackward>(a);
    if (dtype == kF16) return by_experts<kF16, kBackward>(a);
    return by_experts<kBF16, kBackward>(a);
}

}  // namespace

int64_t balance_scratch_bytes(int experts) {
    return kept_bytes(experts) + static_cast<int64_t>(kMaxParts) * (2 * experts + 1) * 4;
}

cudaError_t launch_balance_loss(const void* logits, int dtype, const float* bias,
                                const int32_t* ids, const uint8_t* mask, float coefficient,
                                float* loss, int32_t* counts, int32_t* counted, void* scratch,
                                int64_t tokens, int experts, int topk, cudaStream_t stream) {
    BalanceArgs a = {logits, bias, ids, mask, tokens, experts, topk, coefficient,
                     loss, counts, counted, scratch, nullptr, nullptr, stream};
    return by_dtype<false>(dtype, a);
}

cudaError_t launch_balance_loss_backward(const void* logits, int dtype, const float* bias,
                                         const uint8_t* mask, const int32_t* counts,
                                         const int32_t* counted, const float* grad_loss,
                                         float coefficient, void* grad, int64_t tokens, int experts,
                                         int topk, cudaStream_t stream) {
    if (tokens == 0) return cudaSuccess;
    BalanceArgs a = {logits, bias, nullptr, mask, tokens, experts, topk, coefficient,
                     nullptr, const_cast<int32_t*>(counts), const_cast<int32_t*>(counted), nullptr,
                     grad_loss, grad, stream};
    return by_dtype<true>(dtype, a);
}

}  // namespace moe
