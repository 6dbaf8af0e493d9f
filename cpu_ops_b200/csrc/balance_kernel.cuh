// The balance loss of a router, its counts and its gradient:
//     counts_e = pairs of expert e,  f_e = counts_e / sum counts
//     p_te     = softmax(logits_t)_e,  or  s_te / sum s_t  with the logistic s of the logits
//     P_e      = mean of p_te over the tokens that have an expert,  loss = c E sum f_e P_e
//     dlogits  = upstream c E / T * w_te (f_e - sum_j p_tj f_j),  w = p (softmax) or p (1 - s)
// (counts are whole numbers, which have no gradient).  f_e - sum_j p_j f_j is formed from f_e - 1 / E,
// which differ from one another as much as f_e do: an even load leaves nothing of the f_e themselves.
//
// A kernel counts, block by block; the other needs all counts (its CTAs add the blocks' up), takes a token
// per warp, logits read once, and keeps sums of p in registers; its last CTA adds those up.  Bound by latencies: two
// launches, two hand-overs through L2, a token's three sums across a warp.  8192 tokens of 256 experts, f32: 16 us of a
// replayed graph (17 MB, 2.6 us at HBM's rate); 1537 of 60, bf16: 8.5; 32 of 64 in one launch: 4.6.  Beyond 512 experts a thread's
// scores, the next token's and its sums do not all fit 128 registers (208 bytes spilled): 8192 of 1024 48 us.
#pragma once

#include "dense_params.h"
#include "norm_kernel.cuh"

#include <cfloat>

namespace b200 {

constexpr int kBalanceCountThreads = 256;
// Warps of a CTA of the main kernel, as many as its registers (a token's scores, its next logits, the sums) leave.
__host__ __device__ constexpr int balance_warps(int per_lane) { return per_lane <= 8 ? 32 : 16; }

// Counts of the tokens [begin, end) into shared memory: counts[0 .. experts), and counts[experts]
// of tokens that have an expert.  All threads of the CTA.
__device__ __forceinline__ void count_pairs(const BalanceParams& p, int64_t begin, int64_t end, int32_t* counts) {
  for (int i = threadIdx.x; i <= p.experts; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  for (int64_t t = begin + threadIdx.x; t < end; t += blockDim.x) {
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

__global__ void __launch_bounds__(kBalanceCountThreads) balance_count_kernel(const BalanceParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int32_t counts[1025];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
  const int64_t tokens = p.tokens, per = (tokens + p.count_blocks - 1) / p.count_blocks;
  const int64_t begin = min(blockIdx.x * per, tokens);
  count_pairs(p, begin, min(begin + per, tokens), counts);
  for (int i = threadIdx.x; i <= p.experts; i += blockDim.x) p.part_counts[static_cast<int64_t>(blockIdx.x) * (p.experts + 1) + i] = counts[i];
}

// exp(v), v <= 0: exp2 of a rounded product, off by |v| eps / 2 of itself, which the sums of the larger terms dwarf.
__device__ __forceinline__ float exp_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}

// kPer: experts per lane.  p.count_blocks == 0: one CTA, which counts itself.
template <typename T, int kPer>
__global__ void __launch_bounds__(32 * balance_warps(kPer)) balance_kernel(const BalanceParams p) {
  constexpr int kWarps = balance_warps(kPer), kThreads = 32 * kWarps;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int32_t counts[32 * kPer + 1];
  __shared__ float share[32 * kPer];             // f_e - 1 / E
  __shared__ float join[kWarps][32 * kPer <= 256 ? 32 * kPer : 256];
  __shared__ double terms[kWarps];
  __shared__ int32_t last, all_pairs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, experts = p.experts;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.count_blocks == 0) {
    count_pairs(p, 0, p.tokens, counts);
  } else {
    // the blocks' counts, each warp its share of the blocks (all of its loads in flight together)
    for (int i = threadIdx.x; i <= experts; i += kThreads) counts[i] = 0;
    __syncthreads();
    int32_t some[kPer + 1];
#pragma unroll
    for (int j = 0; j <= kPer; ++j) some[j] = 0;
#pragma unroll 2
    for (int b = warp; b < p.count_blocks; b += kWarps) {
#pragma unroll
      for (int j = 0; j <= kPer; ++j)
        if (lane + 32 * j <= experts) some[j] += __ldcg(p.part_counts + static_cast<int64_t>(b) * (experts + 1) + lane + 32 * j);
    }
#pragma unroll
    for (int j = 0; j <= kPer; ++j)
      if (some[j] != 0) atomicAdd(counts + lane + 32 * j, some[j]);
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
  for (int i = threadIdx.x; i < experts; i += kThreads) {
    // a whole number over a whole number: nothing cancels behind this difference
    const int64_t above = static_cast<int64_t>(counts[i]) * experts - pairs;
    share[i] = pairs > 0 ? static_cast<float>(above) / (static_cast<float>(pairs) * static_cast<float>(experts)) : 0.0f;
    if (blockIdx.x == 0 && p.counts) p.counts[i] = counts[i];
  }
  __syncthreads();
  const float factor = live_tokens > 0 ? (p.upstream ? __ldg(p.upstream) : 1.0f) * p.coefficient * static_cast<float>(experts) /
                                             static_cast<float>(live_tokens)
                                       : 0.0f;
  float sums[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) sums[j] = 0.0f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  const T* logits = static_cast<const T*>(p.logits);
  T* dlogits = static_cast<T*>(p.dlogits);
  T next[kPer];
  int32_t next_id = -1;
  auto fetch = [&](int64_t t) {  // (top_k is at most 32)
    next_id = lane < p.top_k ? __ldg(p.ids + t * p.top_k + lane) : -1;
#pragma unroll
    for (int j = 0; j < kPer; ++j) next[j] = lane + 32 * j < experts ? logits[t * p.ld + lane + 32 * j] : from_f32<T>(-INFINITY);
  };
  int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (t < p.tokens) fetch(t);
  for (; t < p.tokens; t += step) {
    float x[kPer], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float v = to_f32(next[j]);
      // (NaN: the expert is out; +inf counts as the largest number, as it does in routing)
      x[j] = v > -INFINITY ? fminf(v, FLT_MAX) : -INFINITY;
      most = fmaxf(most, x[j]);
    }
    const bool live = __any_sync(0xffffffffu, next_id >= 0 && next_id < experts);
    if (t + step < p.tokens) fetch(t + step);
    if (!live) {  // a padding token
      if (dlogits) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (lane + 32 * j < experts) dlogits[t * p.ldg + lane + 32 * j] = from_f32<T>(0.0f);
      }
      continue;
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
        const float small = exp_fast(-fabsf(x[j])), r = __fdividef(1.0f, 1.0f + small);
        s = exp_fast(fminf(x[j], 0.0f) - shift) * r;
        rest[j] = (x[j] >= 0.0f ? small : 1.0f) * r;  // 1 - s
      } else {
        s = exp_fast(x[j] - shift);
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
    if (dlogits) {
      along = warp_sum(along);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (lane + 32 * j < experts)
          dlogits[t * p.ldg + lane + 32 * j] = from_f32<T>(factor * (x[j] * rest[j] * (share[lane + 32 * j] - along)));
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
    for (int i = threadIdx.x; i < 32 * kAtOnce; i += kThreads) {
      const int e = 32 * j0 + i;
      if (e >= experts) continue;
      float s = join[0][i];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) s += join[w][i];
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
    float own[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) own[j] = 0.0f;
#pragma unroll 4
    for (int b = warp; b < static_cast<int>(gridDim.x); b += kWarps) {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (lane + 32 * j < experts) own[j] += __ldcg(p.part_scores + static_cast<int64_t>(b) * experts + lane + 32 * j);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (lane + 32 * j < experts) term += static_cast<double>(counts[lane + 32 * j]) * own[j];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
  if (lane == 0) terms[warp] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < kWarps; ++w) sum += terms[w];
    const double scale = pairs > 0 ? static_cast<double>(experts) / (static_cast<double>(pairs) * live_tokens) : 0.0;
    *p.loss = static_cast<float>(static_cast<double>(p.coefficient) * scale * sum);
  }
}

}  // namespace b200
