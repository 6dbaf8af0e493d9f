// The balance loss of a router, its counts and its gradient:
//     counts_e = pairs of expert e,  f_e = counts_e / sum counts
//     p_te     = softmax(logits_t)_e,  or  s_te / sum s_t  with the logistic s of the logits
//     P_e      = mean of p_te over the tokens that have an expert,  loss = c E sum f_e P_e
//     dlogits  = upstream c E / T * w_te (f_e - sum_j p_tj f_j),  w = p (softmax) or p (1 - s)
// (counts are whole numbers, which have no gradient).  f_e - sum_j p_j f_j is formed from f_e - 1 / E,
// which differ from one another as much as f_e do: an even load leaves nothing of the f_e themselves.
//
// A kernel counts, block by block; the other needs all counts (its CTAs add the blocks' up), takes a token
// per warp, logits read once, and keeps sums of p in registers; its last CTA adds those up.
#pragma once

#include "dense_params.h"
#include "norm_kernel.cuh"

#include <cfloat>

namespace b200 {

constexpr int kBalanceWarps = 8;
constexpr int kBalanceThreads = 32 * kBalanceWarps;

// Counts of the tokens [begin, end) into shared memory: counts[0 .. experts), and counts[experts]
// of tokens that have an expert.  All threads of the CTA.
__device__ __forceinline__ void count_pairs(const BalanceParams& p, int begin, int end, int32_t* counts) {
  for (int i = threadIdx.x; i <= p.experts; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  for (int64_t t = begin + static_cast<int>(threadIdx.x); t < end; t += blockDim.x) {
    bool any = false;
    for (int k = 0; k < p.top_k; ++k) {
      const int32_t id = __ldg(p.ids + t * p.top_k + k);
      if (id >= 0 && id < p.experts) {
        atomicAdd(counts + id, 1);  // (whole numbers: the order does not matter)
        any = true;
      }
    }
    if (any) atomicAdd(counts + p.experts, 1);
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kBalanceThreads) balance_count_kernel(const BalanceParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int32_t counts[1025];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
  const int per = (p.tokens + p.count_blocks - 1) / p.count_blocks;
  const int begin = min(static_cast<int>(blockIdx.x) * per, p.tokens);
  count_pairs(p, begin, min(begin + per, p.tokens), counts);
  for (int i = threadIdx.x; i <= p.experts; i += blockDim.x) p.part_counts[static_cast<int64_t>(blockIdx.x) * (p.experts + 1) + i] = counts[i];
}

__device__ __forceinline__ float logit_of(const BalanceParams& p, int64_t token, int e) {
  const int64_t i = token * p.ld + e;
  const float x = p.type == kF32 ? __ldg(static_cast<const float*>(p.logits) + i)
                  : p.type == kF16 ? __half2float(static_cast<const __half*>(p.logits)[i])
                                   : __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[i]);
  return x > FLT_MAX ? FLT_MAX : x;  // (+inf counts as the largest number, as it does in routing)
}
__device__ __forceinline__ void put_gradient(const BalanceParams& p, int64_t token, int e, float v) {
  const int64_t i = token * p.ldg + e;
  if (p.type == kF32) {
    static_cast<float*>(p.dlogits)[i] = v;
  } else if (p.type == kF16) {
    static_cast<__half*>(p.dlogits)[i] = __float2half_rn(v);
  } else {
    static_cast<__nv_bfloat16*>(p.dlogits)[i] = __float2bfloat16_rn(v);
  }
}

// kPer: experts per lane.  p.count_blocks == 0: one CTA, which counts itself.
template <int kPer>
__global__ void __launch_bounds__(kBalanceThreads) balance_kernel(const BalanceParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int32_t counts[32 * kPer + 1];
  __shared__ float share[32 * kPer];             // f_e - 1 / E
  __shared__ float join[kBalanceWarps][32 * kPer <= 256 ? 32 * kPer : 256];
  __shared__ double terms[kBalanceWarps];
  __shared__ int32_t last, all_pairs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, experts = p.experts;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.count_blocks == 0) {
    count_pairs(p, 0, p.tokens, counts);
  } else {
    for (int i = threadIdx.x; i <= experts; i += kBalanceThreads) {
      int32_t sum = 0;
#pragma unroll 8
      for (int b = 0; b < p.count_blocks; ++b) sum += __ldcg(p.part_counts + static_cast<int64_t>(b) * (experts + 1) + i);
      counts[i] = sum;
    }
    __syncthreads();
  }
  if (warp == 0) {
    int32_t sum = 0;
    for (int i = lane; i < experts; i += 32) sum += counts[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) all_pairs = sum;
  }
  __syncthreads();
  const int64_t pairs = all_pairs;
  const int live_tokens = counts[experts];
  for (int i = threadIdx.x; i < experts; i += kBalanceThreads) {
    // a whole number over a whole number: one rounding
    const int64_t above = static_cast<int64_t>(counts[i]) * experts - pairs;
    share[i] = pairs > 0 ? static_cast<float>(static_cast<double>(above) / (static_cast<double>(pairs) * experts)) : 0.0f;
    if (blockIdx.x == 0 && p.counts) p.counts[i] = counts[i];
  }
  __syncthreads();
  const float factor = live_tokens > 0 ? (p.upstream ? __ldg(p.upstream) : 1.0f) * p.coefficient * static_cast<float>(experts) /
                                             static_cast<float>(live_tokens)
                                       : 0.0f;
  float sums[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) sums[j] = 0.0f;
  const int step = gridDim.x * kBalanceWarps;
  for (int64_t t = blockIdx.x * kBalanceWarps + warp; t < p.tokens; t += step) {
    bool any = false;
    for (int k = lane; k < p.top_k; k += 32) {
      const int32_t id = __ldg(p.ids + t * p.top_k + k);
      any |= id >= 0 && id < experts;
    }
    if (!__any_sync(0xffffffffu, any)) {  // a padding token
      if (p.dlogits) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (lane + 32 * j < experts) put_gradient(p, t, lane + 32 * j, 0.0f);
      }
      continue;
    }
    float x[kPer], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      x[j] = lane + 32 * j < experts ? logit_of(p, t, lane + 32 * j) : -INFINITY;
      if (!(x[j] > -INFINITY)) x[j] = -INFINITY;  // (NaN: the expert is out)
      most = fmaxf(most, x[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    // Scores over a common factor: of the logistic exp(x) at far negative logits, whose sum would vanish.
    const float shift = p.sigmoid ? fminf(most, 0.0f) : most;
    float total = 0.0f, along = 0.0f, rest[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const bool out = x[j] == -INFINITY;
      rest[j] = 1.0f;
      float s;
      if (p.sigmoid) {
        const float small = expf(-fabsf(x[j])), d = 1.0f + small;
        s = expf(fminf(x[j], 0.0f) - shift) / d;
        rest[j] = (x[j] >= 0.0f ? small : 1.0f) / d;  // 1 - s
      } else {
        s = expf(x[j] - shift);
      }
      x[j] = out ? 0.0f : s;
      total += x[j];
    }
    total = warp_sum(total);
    const float inverse = total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      x[j] *= inverse;
      sums[j] += x[j];
      if (lane + 32 * j < experts) along = __fmaf_rn(x[j], share[lane + 32 * j], along);
    }
    if (p.dlogits) {
      along = warp_sum(along);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (lane + 32 * j < experts) put_gradient(p, t, lane + 32 * j, factor * (x[j] * rest[j] * (share[lane + 32 * j] - along)));
    }
  }
  if (p.loss == nullptr) return;
  // The CTA's sums of scores, at most 256 experts at a time, warps in turn; into part_scores where there are
  // several CTAs.
  const bool alone = gridDim.x == 1;
  double term = 0.0;  // this thread's part of sum f_e P_e
  constexpr int kAtOnce = kPer <= 8 ? kPer : 8;
  for (int j0 = 0; j0 < kPer; j0 += kAtOnce) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j >= j0 && j < j0 + kAtOnce) join[warp][lane + 32 * (j - j0)] = sums[j];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * kAtOnce; i += kBalanceThreads) {
      const int e = 32 * j0 + i;
      if (e >= experts) continue;
      float s = join[0][i];
#pragma unroll
      for (int w = 1; w < kBalanceWarps; ++w) s += join[w][i];
      if (alone) {
        term += static_cast<double>(counts[e]) * s;
      } else {
        p.part_scores[static_cast<int64_t>(blockIdx.x) * experts + e] = s;
      }
    }
  }
  if (!alone) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1 ? 1 : 0;
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (int e = threadIdx.x; e < experts; e += kBalanceThreads) {
      double s = 0.0;
#pragma unroll 8
      for (int b = 0; b < static_cast<int>(gridDim.x); ++b) s += __ldcg(p.part_scores + static_cast<int64_t>(b) * experts + e);
      term += static_cast<double>(counts[e]) * s;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
  if (lane == 0) terms[warp] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < kBalanceWarps; ++w) sum += terms[w];
    const double scale = pairs > 0 ? static_cast<double>(experts) / (static_cast<double>(pairs) * live_tokens) : 0.0;
    *p.loss = static_cast<float>(static_cast<double>(p.coefficient) * scale * sum);
  }
}

}  // namespace b200
