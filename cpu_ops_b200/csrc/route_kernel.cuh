// Routing to experts, and the row plan that the experts' products read.
//
//   route_kernel        one warp per token: scores of its logits, the groups that stay, the
//                       top_k best experts and their weights
//   count_ids_kernel,   the plan: a stable counting sort of pairs by their id
//   group_rows_kernel
//   route_few_kernel    both, for few tokens
//
// Every choice is that of scores in double precision.  In f32 two experts of a token whose scores
// differ by less than a rounding come out in an order that depends on how exp was rounded, about
// once in a batch of 8192 tokens x 256 experts.  So a token is routed by f32 scores, with a check that
// neighbours in the order are further apart than the scores' errors, and only where they are not (one token in
// some hundred) by double ones (8192 tokens, 256 experts in 8 groups, sigmoid, bias: TBD us, all in double
// precision 42).  Weights are always formed in double precision.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace b200 {

enum : int32_t { kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2 };
constexpr int kMaxGroups = 1024;  // experts of a route call, groups of a plan
constexpr int kMaxTopK = 32;

struct RouteParams {
  const void* logits;
  const float* bias;  // or null
  int32_t* ids;
  float* weights;
  int64_t ld;
  int32_t type, tokens, experts, top_k;
  int32_t sigmoid, n_groups, top_groups, group_best, renormalize;
  float scale;
};

__device__ __forceinline__ float load_float(const void* base, int32_t type, int64_t i) {
  if (type == kTypeF32) return static_cast<const float*>(base)[i];
  if (type == kTypeF16) return __half2float(static_cast<const __half*>(base)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
}

constexpr int kRouteWarps = 8;

// A token is one warp's; experts lane, lane + 32, ... of it belong to a lane.

// The logit that the rules see: NaN is -inf, +inf the largest number; -inf: the expert is out.  (-0 is 0.)
__device__ __forceinline__ float route_logit(const RouteParams& p, int64_t row, int e) {
  const float v = load_float(p.logits, p.type, row + e);
  return v == v ? fminf(v, 3.402823466e38f) + 0.0f : -INFINITY;
}
// e / per for e < 1024 (magic = ceil(2^20 / per)).
__device__ __forceinline__ int group_of(int e, uint32_t magic) { return static_cast<int>((static_cast<uint32_t>(e) * magic) >> 20); }

// The choice by its definition, everything in double precision.  Returns lane j's expert of slot j
// (-1: none).  scratch: experts + n_groups doubles of this warp (n_groups > 1 only).
template <int kPerLane>
__device__ __noinline__ int route_exact(const RouteParams& p, int64_t row, double* scratch) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const double kOut = -INFINITY;  // the choice of an expert that is out (a valid choice is above: score >= 0, bias > -inf)
  double choice[kPerLane];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = lane + 32 * i;
    float x = e < p.experts ? route_logit(p, row, e) : -INFINITY;
    if (p.bias != nullptr && e < p.experts && !(p.bias[e] > -INFINITY)) x = -INFINITY;
    choice[i] = static_cast<double>(x);
    top = fmaxf(top, x);
  }
  for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, s));
  double total = 0.0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    if (choice[i] == kOut) continue;
    choice[i] = p.sigmoid ? 1.0 / (1.0 + exp(-choice[i])) : exp(choice[i] - static_cast<double>(top));
    total += choice[i];
  }
  if (!p.sigmoid) {
    for (int s = 16; s > 0; s >>= 1) total += __shfl_xor_sync(kAll, total, s);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (choice[i] != kOut) choice[i] /= total;
  }
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (choice[i] != kOut) choice[i] += static_cast<double>(p.bias[lane + 32 * i]);
  }
  if (p.n_groups > 1) {
    double* group = scratch + p.experts;
    const int per = p.experts / p.n_groups;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < p.experts) scratch[lane + 32 * i] = choice[i];
    __syncwarp();
    for (int g = lane; g < p.n_groups; g += 32) {
      double best = kOut, second = kOut;
      for (int j = 0; j < per; ++j) {
        const double v = scratch[g * per + j];
        if (v > best) {
          second = best;
          best = v;
        } else if (v > second) {
          second = v;
        }
      }
      group[g] = p.group_best == 2 && second != kOut ? best + second : best;
    }
    __syncwarp();
    // a group stays if fewer than top_groups come before it
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts) {
        const int g = e / per;
        const double v = group[g];
        int ahead = 0;
        for (int j = 0; j < p.n_groups; ++j) ahead += group[j] > v || (group[j] == v && j < g);
        if (ahead >= p.top_groups) choice[i] = kOut;
      }
    }
  }
  // The best expert, top_k times: value first, the lower index of equal ones.
  int my_id = -1;
  for (int j = 0; j < p.top_k; ++j) {
    double best = kOut;
    int at = kMaxGroups;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      if (choice[i] > best) {
        best = choice[i];
        at = lane + 32 * i;
      }
    }
    for (int s = 16; s > 0; s >>= 1) {
      const double other = __shfl_xor_sync(kAll, best, s);
      const int other_at = __shfl_xor_sync(kAll, at, s);
      if (other > best || (other == best && other_at < at)) {
        best = other;
        at = other_at;
      }
    }
    if (best == kOut) break;  // (the same in all lanes)
    if (lane == j) my_id = at;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (at == lane + 32 * i) choice[i] = kOut;
  }
  return my_id;
}

// f32 as whole numbers in the same order (-inf lowest); 0 is below all of them.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The same choice from f32 scores, and whether these settle it.  Two neighbours in the order of choice
// (the first one left out among them) have to be further apart than both scores' errors: `apart`.
// Without a bias the order is that of the logits themselves, which f32 holds exactly.
template <int kPerLane>
__device__ __forceinline__ int route_fast(const RouteParams& p, int64_t row, float* scratch, float& top, bool& settled) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const bool by_logit = p.bias == nullptr && p.n_groups == 1;
  float x[kPerLane];
  uint32_t key[kPerLane];
  top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = lane + 32 * i;
    x[i] = e < p.experts ? route_logit(p, row, e) : -INFINITY;
  }
  float bias[kPerLane], largest_bias = 0.0f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = lane + 32 * i;
    bias[i] = p.bias != nullptr && e < p.experts ? p.bias[e] : 0.0f;
    if (!(bias[i] > -INFINITY)) x[i] = -INFINITY;
    if (x[i] != -INFINITY) largest_bias = fmaxf(largest_bias, fabsf(bias[i]));
    top = fmaxf(top, x[i]);
  }
  if (p.bias != nullptr) largest_bias = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(largest_bias)));
  top = key_value(__reduce_max_sync(kAll, order_key(top)));
  float inverse = 1.0f;
  if (!by_logit) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const float e = x[i] == -INFINITY ? 0.0f : p.sigmoid ? 1.0f / (1.0f + expf(-x[i])) : expf(x[i] - top);
      total += e;
      if (x[i] != -INFINITY) x[i] = e;
    }
    if (!p.sigmoid) {
      for (int s = 16; s > 0; s >>= 1) total += __shfl_xor_sync(kAll, total, s);
      inverse = 1.0f / total;
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (x[i] != -INFINITY) x[i] = x[i] * inverse + bias[i];
  }
  settled = true;
  if (p.n_groups > 1) {
    if (p.n_groups > 32) {  // (a group to a lane below)
      settled = false;
      return -1;
    }
    // per + 1 words to a group in shared memory; the warp's lanes share the groups evenly
    const int per = p.experts / p.n_groups;
    const uint32_t magic = ((1u << 20) + per - 1) / per;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts) scratch[e + group_of(e, magic)] = x[i];
    }
    __syncwarp();
    int share = 1;  // lanes per group
    while (2 * share * p.n_groups <= 32) share *= 2;
    const int g = lane / share, part = lane & (share - 1);
    float best = -INFINITY, second = -INFINITY;
    if (g < p.n_groups)
      for (int j = part; j < per; j += share) {
        const float v = scratch[g * (per + 1) + j];
        second = fmaxf(second, fminf(best, v));
        best = fmaxf(best, v);
      }
    for (int s = 1; s < share; s <<= 1) {
      const float b2 = __shfl_xor_sync(kAll, best, s), s2 = __shfl_xor_sync(kAll, second, s);
      second = fmaxf(fmaxf(second, s2), fminf(best, b2));
      best = fmaxf(best, b2);
    }
    const float score = p.group_best == 2 && second != -INFINITY ? best + second : best;
    int ahead = 0;
    for (int j = 0; j < p.n_groups; ++j) {
      const float other = __shfl_sync(kAll, score, j * share);
      ahead += other > score || (other == score && j < g);
    }
    const bool mine = g < p.n_groups, stays = mine && ahead < p.top_groups;
    // the last group that stays and the first that does not
    const float low = -key_value(__reduce_max_sync(kAll, stays ? order_key(-score) : 0u));
    const float high = key_value(__reduce_max_sync(kAll, mine && !stays ? order_key(score) : order_key(-INFINITY)));
    if (p.top_groups < p.n_groups && !(low - high > 1e-6f * (2.0f + fabsf(low) + fabsf(high))) && high != -INFINITY) settled = false;
    const unsigned kept = __ballot_sync(kAll, stays && part == 0);  // bit g * share
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts && !(kept >> (group_of(e, magic) * share) & 1u)) x[i] = -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) key[i] = order_key(x[i]);
  const uint32_t out = order_key(-INFINITY);
  int my_id = -1;
  float my_value = -INFINITY, after = -INFINITY;  // after: the first one left out
  for (int j = 0; j <= p.top_k; ++j) {
    uint32_t best = out;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(kAll, best);
    if (best == out) break;
    uint32_t at = kMaxGroups;
#pragma unroll
    for (int i = kPerLane - 1; i >= 0; --i) at = key[i] == best ? lane + 32 * i : at;
    at = __reduce_min_sync(kAll, at);
    if (j == p.top_k) {
      after = key_value(best);
      break;
    }
    if (lane == j) {
      my_id = static_cast<int>(at);
      my_value = key_value(best);
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (at == lane + 32 * i) key[i] = out;
  }
  // lane j against slot j + 1 (the last one against the one left out)
  float next = __shfl_down_sync(kAll, my_value, 1);
  if (lane == p.top_k - 1) next = after;
  bool apart = true;
  if (my_id >= 0 && lane < p.top_k) {
    if (by_logit) {
      // equal logits are equal; others differ in double precision too, unless it has run out of digits
      apart = my_value == next || next == -INFINITY || my_value - next > 1e-8f;
      apart = apart && (p.sigmoid ? fabsf(my_value) < 15.0f : my_value - top > -600.0f);
    } else {
      // scores (at most 1, and at most the value and the bias together) are within 1e-6 of themselves,
      // sums within 1.2e-7; twice that for either
      const float size = fabsf(my_value) + fabsf(next);
      const float scores = fminf(size + 2.0f * largest_bias, 2.0f);
      apart = next == -INFINITY || my_value - next > 2e-6f * scores + 4e-7f * size + 1e-37f;
    }
  }
  settled = settled && __all_sync(kAll, apart);
  return my_id;
}

// Shared memory (the grouped case only): experts + n_groups doubles per warp.
template <int kPerLane>
__device__ __forceinline__ void route_token(const RouteParams& p, int token, double* scratch) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(token) * p.ld;
  float top;
  bool settled;
  int my_id = route_fast<kPerLane>(p, row, reinterpret_cast<float*>(scratch), top, settled);
  if (!settled) my_id = route_exact<kPerLane>(p, row, scratch);

  // Weights: the chosen experts' scores in double precision.
  double total = 1.0;
  if (!p.sigmoid && !p.renormalize) {
    total = 0.0;
    for (int e = lane; e < p.experts; e += 32) {
      const float v = route_logit(p, row, e);
      if (v != -INFINITY && (p.bias == nullptr || p.bias[e] > -INFINITY))
        total += exp(static_cast<double>(v) - static_cast<double>(top));
    }
    for (int s = 16; s > 0; s >>= 1) total += __shfl_xor_sync(kAll, total, s);
  }
  double score = 0.0;
  if (my_id >= 0) {
    const double v = static_cast<double>(route_logit(p, row, my_id));
    score = p.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - static_cast<double>(top)) / total;
  }
  if (p.renormalize) {
    double sum = score;
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(kAll, sum, s);
    score = sum > 0.0 ? score / sum : 0.0;
  }
  if (lane < p.top_k) {
    const int64_t at = static_cast<int64_t>(token) * p.top_k + lane;
    p.ids[at] = my_id;
    p.weights[at] = static_cast<float>(score * static_cast<double>(p.scale));
  }
}

__host__ __device__ inline size_t route_smem_bytes(int experts, int n_groups) {
  return n_groups > 1 ? static_cast<size_t>(kRouteWarps) * (experts + n_groups) * sizeof(double) : 0;
}
template <int kPerLane>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ double route_smem[];
  const int warp = threadIdx.x >> 5;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token < p.tokens) route_token<kPerLane>(p, token, route_smem + warp * (p.experts + p.n_groups));
}

// ---- the plan ---------------------------------------------------------------------------
//
// A block of kThreads threads sorts kThreads * kRounds pairs; pairs in no group make up one more group
// behind the last, whose places hold -1.  Ranks are counted warp by warp over ascending pairs (every
// warp owns a contiguous run), so the sort is stable and its result does not depend on which warp came first.

constexpr int kPlanThreads = 1024;
constexpr int kPlanRounds = 4;  // 32-pair steps of a warp
constexpr int kPlanPairs = kPlanThreads * kPlanRounds;

// The bin of pair q: its group, or `groups` for none.
__device__ __forceinline__ int plan_bin(const int32_t* ids, int64_t q, int groups) {
  const int id = ids[q];
  return id >= 0 && id < groups ? id : groups;
}

// counts[b * (groups + 1) + g]: pairs of bin g among block b's.
__global__ void __launch_bounds__(kPlanThreads) count_ids_kernel(const int32_t* ids, int64_t rows, int groups,
                                                                 int32_t* counts) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ int32_t bins[kMaxGroups + 1];
  for (int g = threadIdx.x; g <= groups; g += kPlanThreads) bins[g] = 0;
  __syncthreads();
  for (int i = 0; i < kPlanRounds; ++i) {
    const int64_t q = static_cast<int64_t>(blockIdx.x) * kPlanPairs + i * kPlanThreads + threadIdx.x;
    if (q < rows) atomicAdd(&bins[plan_bin(ids, q, groups)], 1);  // (whole numbers: any order gives the same)
  }
  __syncthreads();
  for (int g = threadIdx.x; g <= groups; g += kPlanThreads)
    counts[static_cast<int64_t>(blockIdx.x) * (groups + 1) + g] = bins[g];
}

// Shared memory: per bin its start, all blocks' pairs, those of the blocks before, the warps' counters.
__host__ __device__ inline int plan_smem_bytes(int groups, int threads = kPlanThreads) {
  return (groups + 1) * (3 * 4 + threads / 32 * 2);
}

// A group's pairs cut into tiles of up to kPlanTileRows, for kernels that work tile by tile.
constexpr int kPlanTileRows = 64;
__host__ __device__ inline int64_t plan_max_tiles(int64_t rows, int groups) {
  return rows / kPlanTileRows + (rows < groups + 1 ? rows : groups + 1);
}

// `counts`: from count_ids_kernel, or null with a single block.  `offsets` may be null.  With `tiles`
// (plan_max_tiles entries) the pairs in no group are kept, as a group behind the last, and the tiles of
// all groups are listed: {group, first place in order, pairs, 0}, then empty ones.
template <int kThreads, int kRounds>
__device__ __forceinline__ void plan_block(const int32_t* ids, int64_t rows, int groups, const int32_t* counts,
                                           int32_t* offsets, int32_t* order, int4* tiles, int32_t* plan_smem) {
  constexpr int kWarps = kThreads / 32;
  const int bins = groups + 1;
  int32_t* start = plan_smem;                                     // [bins]
  int32_t* all = plan_smem + bins;                                // [2][bins]
  uint16_t* seen = reinterpret_cast<uint16_t*>(plan_smem + 3 * bins);  // [kWarps][bins]
  __shared__ int32_t warp_sums[kWarps];
  constexpr unsigned kAll = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kWarps * bins; i += kThreads) seen[i] = 0;
  __syncthreads();
  const int64_t q0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kRounds) + warp * (32 * kRounds);
  int bin[kRounds], rank[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int64_t q = q0 + i * 32 + lane;
    bin[i] = q < rows ? plan_bin(ids, q, groups) : -1;
  }
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const unsigned same = __match_any_sync(kAll, bin[i]);
    const int below = __popc(same & ((1u << lane) - 1u));
    rank[i] = 0;
    if (bin[i] >= 0) rank[i] = seen[warp * bins + bin[i]] + below;
    __syncwarp();
    if (bin[i] >= 0 && below == 0)
      seen[warp * bins + bin[i]] = static_cast<uint16_t>(seen[warp * bins + bin[i]] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  // All blocks' pairs per bin, and those of the blocks before this one.
  if (counts != nullptr) {
    for (int g = threadIdx.x; g < 2 * bins; g += kThreads) all[g] = 0;
    __syncthreads();
    const int n = static_cast<int>(gridDim.x) * bins;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int b = i / bins, g = i - b * bins, c = counts[i];
      if (c != 0) {
        atomicAdd(&all[g], c);
        if (b < static_cast<int>(blockIdx.x)) atomicAdd(&all[bins + g], c);
      }
    }
    __syncthreads();
  }
  // Per bin the warps' counts become the warps' starts within the block.
  constexpr int kPerThread = (kMaxGroups + 1 + kThreads - 1) / kThreads;
  int total[kPerThread], before[kPerThread];
  int sum = 0;  // of this thread's bins: kPerThread neighbouring ones
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int g = static_cast<int>(threadIdx.x) * kPerThread + j;
    total[j] = before[j] = 0;
    if (g < bins) {
      int c[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) c[w] = seen[w * bins + g];
      int in_block = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        seen[w * bins + g] = static_cast<uint16_t>(in_block);
        in_block += c[w];
      }
      total[j] = counts != nullptr ? all[g] : in_block;
      before[j] = counts != nullptr ? all[bins + g] : 0;
      sum += total[j];
    }
  }
  // exclusive scan of the bins' totals
  int scan = sum;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int up = __shfl_up_sync(kAll, scan, s);
    if (lane >= s) scan += up;
  }
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  if (warp == 0) {
    int v = lane < kWarps ? warp_sums[lane] : 0;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int up = __shfl_up_sync(kAll, v, s);
      if (lane >= s) v += up;
    }
    if (lane < kWarps) warp_sums[lane] = v;
  }
  __syncthreads();
  int at = scan - sum + (warp > 0 ? warp_sums[warp - 1] : 0);
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int g = static_cast<int>(threadIdx.x) * kPerThread + j;
    if (g < bins) {
      start[g] = at + before[j];
      // (offsets[groups]: where the pairs in no group begin)
      if (blockIdx.x == 0 && offsets != nullptr) offsets[g] = at;
      at += total[j];
    }
  }
  __syncthreads();
  if (tiles != nullptr && blockIdx.x == 0) {
    // the same scan over the bins' tiles
    int own = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) own += (total[j] + kPlanTileRows - 1) / kPlanTileRows;
    int v = own;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int up = __shfl_up_sync(kAll, v, s);
      if (lane >= s) v += up;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
      int w = lane < kWarps ? warp_sums[lane] : 0;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int up = __shfl_up_sync(kAll, w, s);
        if (lane >= s) w += up;
      }
      if (lane < kWarps) warp_sums[lane] = w;
    }
    __syncthreads();
    int slot = v - own + (warp > 0 ? warp_sums[warp - 1] : 0);
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int g = static_cast<int>(threadIdx.x) * kPerThread + j;
      for (int done = 0; done < total[j]; done += kPlanTileRows)
        tiles[slot++] = make_int4(g, start[g] + done, min(kPlanTileRows, total[j] - done), 0);
    }
    const int listed = warp_sums[kWarps - 1], most = static_cast<int>(plan_max_tiles(rows, groups));
    for (int s = listed + static_cast<int>(threadIdx.x); s < most; s += kThreads) tiles[s] = make_int4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (bin[i] >= 0)
      order[start[bin[i]] + seen[warp * bins + bin[i]] + rank[i]] =
          bin[i] < groups || tiles != nullptr ? static_cast<int32_t>(q0 + i * 32 + lane) : -1;
  }
}

__global__ void __launch_bounds__(kPlanThreads) group_rows_kernel(const int32_t* ids, int64_t rows, int groups,
                                                                  const int32_t* counts, int32_t* offsets,
                                                                  int32_t* order, int4* tiles) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ int32_t plan_smem[];
  plan_block<kPlanThreads, kPlanRounds>(ids, rows, groups, counts, offsets, order, tiles, plan_smem);
}

// Few tokens: routing and plan in one launch of one block.
constexpr int kRouteFewTokens = 16, kRouteFewRounds = 2;
constexpr int kRouteFewPairs = kRouteWarps * 32 * kRouteFewRounds;
template <int kPerLane>
__global__ void __launch_bounds__(kRouteWarps * 32) route_few_kernel(const RouteParams p, int32_t* offsets, int32_t* order) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ double route_smem[];
  const int warp = threadIdx.x >> 5;
  for (int token = warp; token < p.tokens; token += kRouteWarps)
    route_token<kPerLane>(p, token, route_smem + warp * (p.experts + p.n_groups));
  __syncthreads();  // all ids are written; the shared memory is the plan's
  plan_block<kRouteWarps * 32, kRouteFewRounds>(p.ids, static_cast<int64_t>(p.tokens) * p.top_k, p.experts, nullptr, offsets,
                                                order, nullptr, reinterpret_cast<int32_t*>(route_smem));
}
__host__ __device__ inline size_t route_few_smem_bytes(int experts, int n_groups) {
  const size_t plan = static_cast<size_t>(plan_smem_bytes(experts, kRouteWarps * 32)), route = route_smem_bytes(experts, n_groups);
  return plan > route ? plan : route;
}

}  // namespace b200
