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
// dependent launch of one CTA adds the rows in order: the loss has the same
// bits on every run.  Integer counts are added with shared-memory atomics
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

// One token's scores; lane holds experts lane + G * i.  Experts past E are -inf.
template <int DT, int G, int VPL>
__device__ __forceinline__ void load_scores(const typename Elem<DT>::T* __restrict__ row,
                                            const float (&bias)[VPL], int lane, int experts,
                                            bool valid, float (&z)[VPL]) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + G * i;
        z[i] = valid && e < experts ? Elem<DT>::load(row[e]) + bias[i] : -INFINITY;
    }
}

// z -> softmax(z) in place (all zeros when no score is above -inf; a NaN or
// +inf among the scores makes the row NaN).
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
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < VPL; ++i) z[i] *= inv;
}

template <int DT, int G, int VPL>
__global__ void __launch_bounds__(kThreads)
balance_forward_kernel(const typename Elem<DT>::T* __restrict__ logits,
                       const float* __restrict__ bias, const int32_t* __restrict__ ids,
                       const uint8_t* __restrict__ mask, float* __restrict__ sums,
                       int32_t* __restrict__ part_counts, int64_t tokens, int experts, int topk,
                       int64_t per_cta) {
    constexpr int kGroups = kThreads / G;       // tokens in flight per CTA
    constexpr int kWarps = kThreads / 32;
    __shared__ float warp_sums[kWarps][32 * VPL];
    __shared__ int32_t counts[32 * VPL + 1];    // [E] and the tokens that count
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    pdl_trigger();
    for (int e = threadIdx.x; e <= experts; e += kThreads) counts[e] = 0;
    pdl_wait();
    float b[VPL], acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + G * i;
        b[i] = bias && e < experts ? bias[e] : 0.0f;
        acc[i] = 0.0f;
    }
    __syncthreads();

    const int64_t t0 = blockIdx.x * per_cta;
    const int64_t t1 = t0 + per_cta < tokens ? t0 + per_cta : tokens;
    // whole warps stay in the loop: the shuffles name every lane
    for (int64_t base = t0; base < t1; base += kGroups) {
        const int64_t t = base + group;
        const bool valid = t < t1 && (!mask || mask[t]);
        float z[VPL];
        load_scores<DT, G, VPL>(logits + t * experts, b, lane, experts, valid, z);
        softmax<G, VPL>(z);
#pragma unroll
        for (int i = 0; i < VPL; ++i) acc[i] += z[i];
        if (valid && lane == 0) atomicAdd(&counts[experts], 1);
    }
    for (int64_t p = t0 * topk + threadIdx.x; p < t1 * topk; p += kThreads) {
        const int e = ids[p];
        if (e >= 0 && e < experts && (!mask || mask[p / topk])) atomicAdd(&counts[e], 1);
    }

    // The warp's groups, then the CTA's warps, in a fixed order.
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
#pragma unroll
        for (int off = 16; off >= G; off >>= 1)
            acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], off);
        if (threadIdx.x % 32 < G) warp_sums[threadIdx.x / 32][lane + G * i] = acc[i];
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

// One CTA: adds the CTAs' rows in order, writes counts[E], counted[0] = V, loss.
__global__ void __launch_bounds__(kFinishThreads)
balance_finish_kernel(const float* __restrict__ sums, const int32_t* __restrict__ part_counts,
                      int parts, int experts, int topk, float coefficient, float* __restrict__ loss,
                      int32_t* __restrict__ counts, int32_t* __restrict__ counted) {
    constexpr int kMax = kFinishThreads;
    __shared__ float s_sum[kMax];
    __shared__ int32_t s_count[kMax];
    __shared__ int32_t s_valid;
    pdl_trigger();
    pdl_wait();
    // slices of the parts x experts: thread (slice, e)
    const int slices = kMax / (experts + 1);
    const int slice = threadIdx.x / (experts + 1), e = threadIdx.x % (experts + 1);
    float total = 0.0f;
    int32_t count = 0;
    if (slice < slices) {
        const int from = static_cast<int>(static_cast<int64_t>(parts) * slice / slices);
        const int to = static_cast<int>(static_cast<int64_t>(parts) * (slice + 1) / slices);
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
        if (e < experts) counts[e] = count;
        else {
            counted[0] = count;
            s_valid = count;
        }
    }
    __syncthreads();
    // f[e] * mean p[e], summed by the first warp in expert order per lane
    if (slice == 0 && e < experts) s_sum[e] = total * static_cast<float>(count);
    __syncthreads();
    if (threadIdx.x < 32) {
        float v = 0.0f;
        for (int i = threadIdx.x; i < experts; i += 32) v += s_sum[i];
        v = group_sum<32>(v);
        if (threadIdx.x == 0) {
            const float n = static_cast<float>(s_valid);
            loss[0] = s_valid == 0 ? 0.0f : coefficient * static_cast<float>(experts) * (v / n / n / static_cast<float>(topk));
        }
    }
}

template <int DT, int G, int VPL>
__global__ void __launch_bounds__(kThreads)
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
    const float inv = n > 0.0f ? 1.0f / n : 0.0f;
    const float factor = grad_loss[0] * coefficient * static_cast<float>(experts) * inv;
    float b[VPL], f[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + G * i;
        b[i] = bias && e < experts ? bias[e] : 0.0f;
        f[i] = e < experts ? static_cast<float>(counts[e]) * (inv / static_cast<float>(topk)) : 0.0f;
    }
    const int64_t first = (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x) / G;
    for (int64_t t0 = 0; t0 < tokens; t0 += groups) {
        const int64_t t = t0 + first;
        const bool inside = t < tokens, valid = inside && (!mask || mask[t]);
        float z[VPL];
        load_scores<DT, G, VPL>(logits + t * experts, b, lane, experts, valid, z);
        softmax<G, VPL>(z);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) dot += z[i] * f[i];
        dot = group_sum<G>(dot);
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = lane + G * i;
            if (inside && e < experts)
                grad[t * experts + e] =
                    Elem<DT>::store(valid ? factor * (z[i] * (f[i] - dot)) : 0.0f);
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

// CTAs of the forward pass: one per SM at most (each costs the finishing CTA a
// row to add), at least one round of tokens each.
constexpr int kMaxParts = 256;
int balance_parts(int64_t tokens, int experts, int sms) {
    const int group = experts <= 8 ? 8 : (experts <= 16 ? 16 : 32);
    const int64_t rounds = (tokens + kThreads / group - 1) / (kThreads / group);
    const int64_t most = sms < kMaxParts ? sms : kMaxParts;
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

template <int DT, int G, int VPL>
cudaError_t forward(const BalanceArgs& a) {
    using T = typename Elem<DT>::T;
    int sms = 0;
    MOE_CUDA_TRY(sm_count(&sms));
    const int parts = balance_parts(a.tokens, a.experts, sms);
    const int64_t per_cta = (a.tokens + parts - 1) / parts;
    float* sums = static_cast<float*>(a.scratch);
    int32_t* part_counts = reinterpret_cast<int32_t*>(sums + static_cast<int64_t>(kMaxParts) * a.experts);
    MOE_CUDA_TRY(launch_dependent(balance_forward_kernel<DT, G, VPL>, dim3(parts), dim3(kThreads), 0,
                                  a.stream, static_cast<const T*>(a.logits), a.bias, a.ids, a.mask,
                                  sums, part_counts, a.tokens, a.experts, a.topk, per_cta));
    return launch_dependent(balance_finish_kernel, dim3(1), dim3(kFinishThreads), 0, a.stream, sums,
                            part_counts, parts, a.experts, a.topk, a.coefficient, a.loss, a.counts,
                            a.counted);
}

template <int DT, int G, int VPL>
cudaError_t backward(const BalanceArgs& a) {
    using T = typename Elem<DT>::T;
    int sms = 0;
    MOE_CUDA_TRY(sm_count(&sms));
    const int64_t rounds = (a.tokens + kThreads / G - 1) / (kThreads / G);
    const int64_t most = 4 * static_cast<int64_t>(sms);
    return launch_dependent(balance_backward_kernel<DT, G, VPL>,
                            dim3(static_cast<unsigned>(rounds < most ? rounds : most)), dim3(kThreads),
                            0, a.stream, static_cast<const T*>(a.logits), a.bias, a.mask, a.counts,
                            a.counted, a.grad_loss, a.coefficient, static_cast<T*>(a.grad), a.tokens,
                            a.experts, a.topk);
}

template <int DT, bool kBackward>
cudaError_t by_experts(const BalanceArgs& a) {
    auto run = [&](auto g, auto v) {
        if constexpr (kBackward) return backward<DT, g(), v()>(a);
        else return forward<DT, g(), v()>(a);
    };
#define MOE_INT(n) std::integral_constant<int, n>{}
    if (a.experts <= 8) return run(MOE_INT(8), MOE_INT(1));
    if (a.experts <= 16) return run(MOE_INT(16), MOE_INT(1));
    if (a.experts <= 32) return run(MOE_INT(32), MOE_INT(1));
    if (a.experts <= 64) return run(MOE_INT(32), MOE_INT(2));
    if (a.experts <= 128) return run(MOE_INT(32), MOE_INT(4));
    return run(MOE_INT(32), MOE_INT(8));
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
    return static_cast<int64_t>(kMaxParts) * (2 * experts + 1) * 4;
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
