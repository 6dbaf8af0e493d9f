// Routing to experts, and the row plan that the experts' products read.
//
//   route_kernel        one warp per token: scores of its logits, the groups that stay, the
//                       top_k best experts and their weights
//   count_ids_kernel,   the plan: a stable counting sort of pairs by their id
//   group_rows_kernel
//
// Every choice is made on scores in double precision.  In f32 two experts of a token whose scores
// differ by less than a rounding come out in an order that depends on how exp was rounded, about
// once in a batch of 8192 tokens x 256 experts; B200 has f64 units at half the f32 rate, so exact
// choices cost little.
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

// Experts lane, lane + 32, ... belong to a lane: kPerLane of them, 32 * kPerLane >= experts.
// Shared memory: one double per expert and per group and warp (the grouped case only).
template <int kPerLane>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ double route_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= p.tokens) return;
  constexpr unsigned kAll = 0xffffffffu;
  const double kOut = -INFINITY;  // the choice of an expert that is out (a valid choice is above: score >= 0, bias > -inf)
  const int64_t row = static_cast<int64_t>(token) * p.ld;

  float x[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = lane + 32 * i;
    x[i] = e < p.experts ? load_float(p.logits, p.type, row + e) : -INFINITY;
    if (x[i] != x[i]) x[i] = -INFINITY;
    if (x[i] == INFINITY) x[i] = 3.402823466e38f;  // FLT_MAX
    if (p.bias != nullptr && e < p.experts) {
      const float b = p.bias[e];
      if (!(b > -INFINITY)) x[i] = -INFINITY;
    }
  }
  float top = -INFINITY;
  double total = 0.0;
  if (!p.sigmoid) {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) top = fmaxf(top, x[i]);
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, s));
  }
  double choice[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    if (x[i] == -INFINITY) {
      choice[i] = kOut;
    } else if (p.sigmoid) {
      choice[i] = 1.0 / (1.0 + exp(-static_cast<double>(x[i])));
    } else {
      choice[i] = exp(static_cast<double>(x[i]) - static_cast<double>(top));
      total += choice[i];
    }
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
    double* mine = route_smem + warp * (p.experts + p.n_groups);
    double* group = mine + p.experts;
    const int per = p.experts / p.n_groups;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < p.experts) mine[lane + 32 * i] = choice[i];
    __syncwarp();
    for (int g = lane; g < p.n_groups; g += 32) {
      double best = kOut, second = kOut;
      for (int j = 0; j < per; ++j) {
        const double v = mine[g * per + j];
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
    uint32_t out = 0;  // bit i: the group of this lane's expert i is out
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts) {
        const int g = e / per;
        const double v = group[g];
        int ahead = 0;
        for (int j = 0; j < p.n_groups; ++j) ahead += group[j] > v || (group[j] == v && j < g);
        if (ahead >= p.top_groups) out |= 1u << i;
      }
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (out >> i & 1u) choice[i] = kOut;
  }

  // The best expert, top_k times: value first, the lower index of equal ones.
  int my_id = -1;  // lane j: the id of slot j
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

  double score = 0.0;
  if (my_id >= 0) {
    float v = load_float(p.logits, p.type, row + my_id);
    if (v == INFINITY) v = 3.402823466e38f;
    score = p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(v)))
                      : exp(static_cast<double>(v) - static_cast<double>(top)) / total;
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

// ---- the plan ---------------------------------------------------------------------------
//
// A block sorts kPlanPairs pairs; pairs in no group make up one more group behind the last,
// whose places hold -1.  Ranks are counted warp by warp over ascending pairs (every warp owns a
// contiguous run), so the sort is stable and its result does not depend on which warp came first.

constexpr int kPlanThreads = 1024;
constexpr int kPlanRounds = 4;                                // 32-pair steps of a warp
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
__host__ __device__ inline int plan_smem_bytes(int groups) { return (groups + 1) * (3 * 4 + 32 * 2); }

// A group's pairs cut into tiles of up to kPlanTileRows, for kernels that work tile by tile.
constexpr int kPlanTileRows = 64;
__host__ __device__ inline int64_t plan_max_tiles(int64_t rows, int groups) {
  return rows / kPlanTileRows + (rows < groups + 1 ? rows : groups + 1);
}

// `counts`: from count_ids_kernel, or null with a single block.  `offsets` may be null.  With `tiles`
// (plan_max_tiles entries) the pairs in no group are kept, as a group behind the last, and the tiles of
// all groups are listed: {group, first place in order, pairs, 0}, then empty ones.
__global__ void __launch_bounds__(kPlanThreads) group_rows_kernel(const int32_t* ids, int64_t rows, int groups,
                                                                  const int32_t* counts, int32_t* offsets,
                                                                  int32_t* order, int4* tiles) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ int32_t plan_smem[];
  const int bins = groups + 1;
  int32_t* start = plan_smem;                                     // [bins]
  int32_t* all = plan_smem + bins;                                // [2][bins]
  uint16_t* seen = reinterpret_cast<uint16_t*>(plan_smem + 3 * bins);  // [32][bins]
  __shared__ int32_t warp_sums[32];
  constexpr unsigned kAll = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < 32 * bins; i += kPlanThreads) seen[i] = 0;
  __syncthreads();
  const int64_t q0 = static_cast<int64_t>(blockIdx.x) * kPlanPairs + warp * (32 * kPlanRounds);
  int bin[kPlanRounds], rank[kPlanRounds];
#pragma unroll
  for (int i = 0; i < kPlanRounds; ++i) {
    const int64_t q = q0 + i * 32 + lane;
    bin[i] = q < rows ? plan_bin(ids, q, groups) : -1;
  }
#pragma unroll
  for (int i = 0; i < kPlanRounds; ++i) {
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
    for (int g = threadIdx.x; g < 2 * bins; g += kPlanThreads) all[g] = 0;
    __syncthreads();
    const int n = static_cast<int>(gridDim.x) * bins;
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
      const int b = i / bins, g = i - b * bins, c = counts[i];
      if (c != 0) {
        atomicAdd(&all[g], c);
        if (b < static_cast<int>(blockIdx.x)) atomicAdd(&all[bins + g], c);
      }
    }
    __syncthreads();
  }
  // Per bin the warps' counts become the warps' starts within the block.
  constexpr int kPerThread = (kMaxGroups + 1 + kPlanThreads - 1) / kPlanThreads;
  int total[kPerThread], before[kPerThread];
  int sum = 0;  // of this thread's bins: kPerThread neighbouring ones
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int g = static_cast<int>(threadIdx.x) * kPerThread + j;
    total[j] = before[j] = 0;
    if (g < bins) {
      int c[32];
#pragma unroll
      for (int w = 0; w < 32; ++w) c[w] = seen[w * bins + g];
      int in_block = 0;
#pragma unroll
      for (int w = 0; w < 32; ++w) {
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
    int v = warp_sums[lane];
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int up = __shfl_up_sync(kAll, v, s);
      if (lane >= s) v += up;
    }
    warp_sums[lane] = v;
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
      int w = warp_sums[lane];
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int up = __shfl_up_sync(kAll, w, s);
        if (lane >= s) w += up;
      }
      warp_sums[lane] = w;
    }
    __syncthreads();
    int slot = v - own + (warp > 0 ? warp_sums[warp - 1] : 0);
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int g = static_cast<int>(threadIdx.x) * kPerThread + j;
      for (int done = 0; done < total[j]; done += kPlanTileRows)
        tiles[slot++] = make_int4(g, start[g] + done, min(kPlanTileRows, total[j] - done), 0);
    }
    const int listed = warp_sums[31], most = static_cast<int>(plan_max_tiles(rows, groups));
    for (int s = listed + static_cast<int>(threadIdx.x); s < most; s += kPlanThreads) tiles[s] = make_int4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kPlanRounds; ++i) {
    if (bin[i] >= 0)
      order[start[bin[i]] + seen[warp * bins + bin[i]] + rank[i]] =
          bin[i] < groups || tiles != nullptr ? static_cast<int32_t>(q0 + i * 32 + lane) : -1;
  }
}

}  // namespace b200
