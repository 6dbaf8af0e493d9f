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
// some hundred) by double ones (8192 tokens, 256 experts in 8 groups, sigmoid, bias: 21 us without the plan, all
// in double precision 44).  Weights are always formed in double precision.
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
// A lane's logits (-inf behind the last expert).
template <int kPerLane>
__device__ __forceinline__ void route_logits(const RouteParams& p, int64_t row, float (&x)[kPerLane]) {
  const int lane = threadIdx.x & 31;
  auto all = [&](auto* base) {
    const auto* from = base + row + lane;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) x[i] = lane + 32 * i < p.experts ? static_cast<float>(from[32 * i]) : -INFINITY;
  };
  if (p.type == kTypeF32) all(static_cast<const float*>(p.logits));
  else if (p.type == kTypeF16) all(static_cast<const __half*>(p.logits));
  else all(static_cast<const __nv_bfloat16*>(p.logits));
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) x[i] = x[i] == x[i] ? fminf(x[i], 3.402823466e38f) + 0.0f : -INFINITY;
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

// Which groups stay, in the precision of T: bit g * share of the result, share lanes to a group (n_groups <=
// 32).  `v`: a lane's choices (-inf: out); scratch: experts + n_groups numbers of this warp.  `near`: the
// last group that stays and the first that does not are no further apart than `slack` times the sizes of the
// choices in them (a group's two may cancel: its score may be far smaller than their roundings) and `least`.
template <typename T, int kPerLane>
__device__ __forceinline__ unsigned groups_kept(const RouteParams& p, const T (&v)[kPerLane], T* scratch, uint32_t magic,
                                                int share, T slack, T least, bool& near) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int per = p.experts / p.n_groups;
  const T kOut = -INFINITY;
  // per + 1 places to a group; the warp's lanes share the groups evenly
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = lane + 32 * i;
    if (e < p.experts) scratch[e + group_of(e, magic)] = v[i];
  }
  __syncwarp();
  const int g = lane / share, part = lane & (share - 1);
  const bool mine = g < p.n_groups;
  T best = kOut, second = kOut;
  if (mine)
    for (int j = part; j < per; j += share) {
      const T w = scratch[g * (per + 1) + j];
      const T less = best < w ? best : w;
      second = second < less ? less : second;
      best = best < w ? w : best;
    }
  for (int s = 1; s < share; s <<= 1) {
    const T b2 = __shfl_xor_sync(kAll, best, s), s2 = __shfl_xor_sync(kAll, second, s);
    const T less = best < b2 ? best : b2, most = second < s2 ? s2 : second;
    second = most < less ? less : most;
    best = best < b2 ? b2 : best;
  }
  const bool both = p.group_best == 2 && second != kOut;
  const T score = both ? best + second : best;
  const T reach = slack * ((best < 0 ? -best : best) + (both ? second < 0 ? -second : second : T(0)));
  int ahead = 0;
  unsigned close = 0;  // groups that are no further away
  for (int j = 0; j < p.n_groups; ++j) {
    const T other = __shfl_sync(kAll, score, j * share), other_reach = __shfl_sync(kAll, reach, j * share);
    ahead += other > score || (other == score && j < g);
    const T gap = other < score ? score - other : other - score;
    if (other != kOut && score != kOut && !(gap > reach + other_reach + least)) close |= 1u << j;
  }
  const bool stays = mine && ahead < p.top_groups;
  const unsigned kept = __ballot_sync(kAll, stays && part == 0);
  bool across = false;  // ... and on the other side
  for (; close != 0; close &= close - 1) across = across || ((kept >> ((__ffs(close) - 1) * share) & 1u) != 0) != stays;
  near = __any_sync(kAll, mine && across);
  return kept;
}

// Lane j's choice of expert `id` in double precision (softmax: `total` is the sum of exponentials).
__device__ __forceinline__ double exact_choice(const RouteParams& p, int64_t row, int id, float top, double total) {
  const double v = static_cast<double>(route_logit(p, row, id));
  const double score = p.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - static_cast<double>(top)) / total;
  return p.bias != nullptr ? score + static_cast<double>(p.bias[id]) : score;
}
__device__ __noinline__ double exact_total(const RouteParams& p, int64_t row, float top) {
  double total = 0.0;
  for (int e = threadIdx.x & 31; e < p.experts; e += 32) {
    const float v = route_logit(p, row, e);
    if (v != -INFINITY && (p.bias == nullptr || p.bias[e] > -INFINITY))
      total += exp(static_cast<double>(v) - static_cast<double>(top));
  }
  for (int s = 16; s > 0; s >>= 1) total += __shfl_xor_sync(0xffffffffu, total, s);
  return total;
}
// The groups that stay, in double precision.
template <int kPerLane>
__device__ __noinline__ unsigned groups_kept_exact(const RouteParams& p, int64_t row, double* scratch, uint32_t magic,
                                                   int share, float top) {
  const int lane = threadIdx.x & 31;
  const double total = p.sigmoid ? 1.0 : exact_total(p, row, top);
  double v[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = lane + 32 * i;
    v[i] = -INFINITY;
    if (e < p.experts && route_logit(p, row, e) != -INFINITY && (p.bias == nullptr || p.bias[e] > -INFINITY))
      v[i] = exact_choice(p, row, e, top, total);
  }
  bool near;
  return groups_kept<double, kPerLane>(p, v, scratch, magic, share, 0.0, 0.0, near);
}

// The choice from f32 scores, with doubles only where those do not settle it: the experts that may be among the
// top_k are those not further below the last of these than both scores' errors; where two neighbours
// are no further apart than that, all of these are put in order in double precision.  list: 32 entries of this warp.
// False: more than 32 are that close (route_exact decides).
// Without a bias the order is that of the logits themselves, which f32 holds exactly.
template <int kPerLane>
__device__ __forceinline__ bool route_fast(const RouteParams& p, int64_t row, double* scratch, uint2* list, float& top, int& my_id) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const bool by_logit = p.bias == nullptr && p.n_groups == 1;
  float x[kPerLane];
  uint32_t key[kPerLane];
  top = -INFINITY;
  my_id = -1;
  route_logits<kPerLane>(p, row, x);
  float bias[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) bias[i] = 0.0f;
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < p.experts) bias[i] = p.bias[lane + 32 * i];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (!(bias[i] > -INFINITY)) x[i] = -INFINITY;
  }
  if (!p.sigmoid) {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) top = fmaxf(top, x[i]);
    top = key_value(__reduce_max_sync(kAll, order_key(top)));
  }
  if (!by_logit) {
    float total = 0.0f, inverse = 1.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const float e = __expf(p.sigmoid ? -x[i] : x[i] - top);  // (of an expert that is out it is not used)
      const float score = p.sigmoid ? __fdividef(1.0f, 1.0f + e) : e;
      const bool in = x[i] != -INFINITY;
      total += in ? score : 0.0f;
      x[i] = in ? score : -INFINITY;
    }
    if (!p.sigmoid) {
      for (int s = 16; s > 0; s >>= 1) total += __shfl_xor_sync(kAll, total, s);
      inverse = __fdividef(1.0f, total);
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) x[i] = x[i] != -INFINITY ? x[i] * inverse + bias[i] : -INFINITY;
  }
  // How far two f32 choices of a summed size have to be apart: slack times it, and least.  u = 2^-24 below.
  // An exponential is within (2 + 1.173 |argument|) 2u of itself (CUDA's bound for __expf), the rounding of
  // an argument of size a moves it by another a u (a < 64: by 2^-19 at most), a quotient is within 4u.
  //   No bias: a softmax's quotient is common to all of a token's scores, so it does not count.  Down to
  //   1e-25 = exp(-57.6), below which `least` holds, a score is within 139 u + 32 u + 2 u = 1.03e-5 of itself.
  //   Bias, softmax: scores are at most 1, and so is the sum of those compared.  The total is common to
  //   them: it counts once, for their difference.  Its terms' errors: at most 5 2u = 5.9e-7 of a largest score
  //   (2 + 1.67 sum of p_j |argument j|, which with 1024 experts is below 1.77 of it); its sum, kPerLane numbers
  //   one after another and five steps across the lanes: kPerLane + 4 roundings; the quotient 2.4e-7.
  //   The exponentials of the scores themselves: 2.5 2u = 2.9e-7, of four scores of two groups 3.0 2u; the products
  //   6e-8.  Together 1.26e-6 + (kPerLane + 4) u.
  //   Bias, sigmoid: s (1 - s) (2 + 1.173 |argument|) 2u + 5u, together 3.8e-7 for each score, which is less.
  //   The sum with the bias: u of the choice, which slack covers.
  const float slack = p.bias == nullptr ? 1.1e-5f : 4e-7f;
  const float least = p.bias == nullptr ? 1e-25f : 1.3e-6f + static_cast<float>(kPerLane + 5) * 6e-8f;
  if (p.n_groups > 1) {
    if (p.n_groups > 32) return false;  // (a group to a lane at least)
    const uint32_t magic = ((1u << 20) + p.experts / p.n_groups - 1) / (p.experts / p.n_groups);
    int share = 1;  // lanes per group
    while (2 * share * p.n_groups <= 32) share *= 2;
    bool near;
    unsigned kept = groups_kept<float, kPerLane>(p, x, reinterpret_cast<float*>(scratch), magic, share, slack, 2.0f * least, near);
    if (near && p.top_groups < p.n_groups) kept = groups_kept_exact<kPerLane>(p, row, scratch, magic, share, top);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int e = lane + 32 * i;
      if (e < p.experts && !(kept >> (group_of(e, magic) * share) & 1u)) x[i] = -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) key[i] = order_key(x[i]);
  const uint32_t out = order_key(-INFINITY);
  // How far a choice has to be below the one before it for their order to be settled.
  auto settled = [&](float above, float value) {
    // equal logits are equal; others differ in double precision too, unless it has run out of digits
    if (by_logit) return above == value || above - value > 1e-8f;
    return above - value > slack * (fabsf(above) + fabsf(value)) + least;
  };
  // ... and, by logit, where scores end at 0 or 1, it has.
  auto in_range = [&](float value) { return !by_logit || (p.sigmoid ? fabsf(value) < 15.0f : value - top > -600.0f); };
  bool apart = true;  // every choice of the top_k settled against the next one
  int picked = 0;
  if (p.top_k < 32) {
    // The lanes' best ones in order: of 32 lanes' maxima the top_k + 1st is no larger than the top_k + 1st
    // of all.  What is not settled below it is listed (a dozen or so, of top_k 8), ranked by counting.
    uint32_t most = out;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) most = max(most, key[i]);
#pragma unroll
    for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
      for (int s = size / 2; s > 0; s /= 2) {
        const uint32_t other = __shfl_xor_sync(kAll, most, s);
        const bool larger = ((lane & s) == 0) == ((lane & size) == 0 || size == 32);
        most = larger ? max(most, other) : min(most, other);
      }
    }
    const float bar = key_value(__shfl_sync(kAll, most, p.top_k));
    const float low = by_logit ? bar - 1e-8f : bar - (slack * 2.0f * fabsf(bar) + least) * 1.01f;
    const uint32_t at_least = max(order_key(low), out + 1);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const bool in = key[i] >= at_least;
      const unsigned who = __ballot_sync(kAll, in);
      const int place = picked + __popc(who & ((1u << lane) - 1u));
      if (in && place < 32) list[place] = make_uint2(key[i], static_cast<uint32_t>(lane + 32 * i));
      picked += __popc(who);
    }
    if (picked > 32) {
      picked = 0;
    } else if (picked > 0) {
      __syncwarp();
      const uint2 mine = lane < picked ? list[lane] : make_uint2(0u, 0u);
      int place = 0;
      for (int j = 0; j < picked; ++j) {
        const uint2 other = list[j];
        place += other.x > mine.x || (other.x == mine.x && other.y < mine.y);
      }
      __syncwarp();
      if (lane < picked) list[place] = mine;
      __syncwarp();
      const uint2 sorted = lane < picked ? list[lane] : make_uint2(out, 0u);
      const float value = key_value(sorted.x);
      const float next = __shfl_down_sync(kAll, value, 1);
      if (lane < picked) my_id = static_cast<int>(sorted.y);
      const bool in = lane < picked && lane < p.top_k;
      if (!__all_sync(kAll, !in || in_range(value))) return false;
      apart = __all_sync(kAll, !in || lane + 1 == picked || settled(value, next));
    }
  }
  if (picked == 0) {  // one after another
    float before = INFINITY, last = INFINITY;  // last: the choice of slot top_k - 1
    while (true) {
      uint32_t best = out;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(kAll, best);
      if (best == out) break;
      const float value = key_value(best);
      if (picked < p.top_k && !in_range(value)) return false;
      if (picked >= p.top_k) {  // left out, if it is far enough below the last one in
        if (by_logit ? settled(before, value) && before != value : settled(last, value)) break;
        if (by_logit && last == value && before == value) break;  // (equal logits: the lower indices are in)
        if (picked == 32) return false;
      }
      if (picked > 0) apart = apart && settled(before, value);
      uint32_t at = kMaxGroups;
#pragma unroll
      for (int i = kPerLane - 1; i >= 0; --i) at = key[i] == best ? lane + 32 * i : at;
      at = __reduce_min_sync(kAll, at);
      if (lane == picked) my_id = static_cast<int>(at);
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (at == lane + 32 * i) key[i] = out;
      before = value;
      if (++picked == p.top_k) last = value;
    }
  }
  if (!apart) {
    const double total = p.sigmoid ? 1.0 : exact_total(p, row, top);
    const double mine = my_id >= 0 ? exact_choice(p, row, my_id, top, total) : 0.0;
    int place = 0;
    for (int j = 0; j < picked; ++j) {
      const double other = __shfl_sync(kAll, mine, j);
      const int other_id = __shfl_sync(kAll, my_id, j);
      place += other > mine || (other == mine && other_id < my_id);
    }
    int sorted = -1;
    for (int j = 0; j < picked; ++j) {
      const int id = __shfl_sync(kAll, my_id, j), at = __shfl_sync(kAll, place, j);
      if (at == lane) sorted = id;
    }
    my_id = sorted;
  }
  if (lane >= p.top_k) my_id = -1;
  return true;
}

// Shared memory (the grouped case only): experts + n_groups doubles per warp.
template <int kPerLane>
__device__ __forceinline__ void route_token(const RouteParams& p, int token, double* scratch) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(token) * p.ld;
  float top;
  int my_id;
  __shared__ uint2 lists[kRouteWarps][32];
  if (!route_fast<kPerLane>(p, row, scratch, lists[threadIdx.x >> 5], top, my_id)) my_id = route_exact<kPerLane>(p, row, scratch);

  // Weights: the chosen experts' scores in double precision.
  const double total = !p.sigmoid && !p.renormalize ? exact_total(p, row, top) : 1.0;
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
constexpr int kPlanRounds = 4;  // 32-pair steps of a warp: of the only block, or of many; of some blocks one step
constexpr int kPlanPairs = kPlanThreads * kPlanRounds;
// Blocks of one step spread the scattered stores of `order` over more SMs (65536 pairs of 256 groups: 12.2 us with
// 16 blocks, 10.7 with 64; 6148 of 60: 9.0, 6.1); each block reads all blocks' counts, so there are not too many of them.
__host__ __device__ inline int plan_rounds(int64_t rows) { return rows > kPlanPairs && rows <= 128 * kPlanThreads ? 1 : kPlanRounds; }
__host__ __device__ inline int64_t plan_blocks(int64_t rows) {
  const int64_t per = static_cast<int64_t>(kPlanThreads) * plan_rounds(rows);
  return rows > 0 ? (rows + per - 1) / per : 1;
}

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
  const int rounds = plan_rounds(rows);
  for (int i = 0; i < rounds; ++i) {
    const int64_t q = (static_cast<int64_t>(blockIdx.x) * rounds + i) * kPlanThreads + threadIdx.x;
    if (q < rows) atomicAdd(&bins[plan_bin(ids, q, groups)], 1);  // (whole numbers: any order gives the same)
  }
  __syncthreads();
  for (int g = threadIdx.x; g <= groups; g += kPlanThreads)
    counts[static_cast<int64_t>(blockIdx.x) * (groups + 1) + g] = bins[g];
}

// Shared memory: per bin its start, all blocks' pairs, those of the blocks before, this block's; the warps'
// counters of 16 bits, plan_row of them to a warp (an odd number of words: the warps' counters of a
// bin lie in different banks).
__host__ __device__ inline int plan_row(int groups) { return 2 * ((groups + 2) / 2 | 1); }
__host__ __device__ inline int plan_smem_bytes(int groups, int threads = kPlanThreads) {
  return (groups + 1) * 4 * 4 + threads / 32 * plan_row(groups) * 2;
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
  int32_t* own = plan_smem + 3 * bins;                            // [bins]
  const int ld = plan_row(groups);
  uint16_t* seen = reinterpret_cast<uint16_t*>(plan_smem + 4 * bins);  // [kWarps][ld]
  __shared__ int32_t warp_sums[kWarps];
  constexpr unsigned kAll = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kWarps * ld / 2; i += kThreads) reinterpret_cast<uint32_t*>(seen)[i] = 0u;
  __syncthreads();
  const int64_t q0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kRounds) + warp * (32 * kRounds);
  int bin[kRounds], rank[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int64_t q = q0 + i * 32 + lane;
    bin[i] = q < rows ? plan_bin(ids, q, groups) : -1;
  }
  const int bits = 33 - __clz(bins);  // (-1, behind the last pair, differs from all bins in the highest)
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    // the lanes with the same bin, bit by bit (the instruction for it takes as long as there are
    // different ones: 4096 pairs of 60 groups 10.2 us, 9.0 so)
    unsigned same = kAll;
    for (int bit = 0; bit < bits; ++bit) {
      const bool one = (bin[i] >> bit & 1) != 0;
      const unsigned ones = __ballot_sync(kAll, one);
      same &= one ? ones : ~ones;
    }
    const int below = __popc(same & ((1u << lane) - 1u));
    rank[i] = 0;
    if (bin[i] >= 0) rank[i] = seen[warp * ld + bin[i]] + below;
    __syncwarp();
    if (bin[i] >= 0 && below == 0)
      seen[warp * ld + bin[i]] = static_cast<uint16_t>(seen[warp * ld + bin[i]] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  // All blocks' pairs per bin, and those of the blocks before this one.
  if (counts != nullptr) {
    for (int g = threadIdx.x; g < 2 * bins; g += kThreads) all[g] = 0;
    __syncthreads();
    for (int b = warp; b < static_cast<int>(gridDim.x); b += kWarps) {
      const int32_t* from = counts + static_cast<int64_t>(b) * bins;
      const bool earlier = b < static_cast<int>(blockIdx.x);
      for (int g0 = lane; g0 < bins; g0 += 32 * 4) {
        int c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = g0 + 32 * j < bins ? from[g0 + 32 * j] : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c[j] != 0) {
            atomicAdd(&all[g0 + 32 * j], c[j]);
            if (earlier) atomicAdd(&all[bins + g0 + 32 * j], c[j]);
          }
      }
    }
    __syncthreads();
  }
  // Per bin the warps' counts become the warps' starts within the block: a warp for every bin in turn, lane
  // w for warp w.
  for (int g = warp; g < bins; g += kWarps) {
    const int c = lane < kWarps ? seen[lane * ld + g] : 0;
    int v = c;
#pragma unroll
    for (int s = 1; s < kWarps; s <<= 1) {
      const int up = __shfl_up_sync(kAll, v, s);
      if (lane >= s) v += up;
    }
    if (lane < kWarps) seen[lane * ld + g] = static_cast<uint16_t>(v - c);
    if (lane == kWarps - 1) own[g] = v;
  }
  __syncthreads();
  constexpr int kPerThread = (kMaxGroups + 1 + kThreads - 1) / kThreads;
  int total[kPerThread], before[kPerThread];
  int sum = 0;  // of this thread's bins: kPerThread neighbouring ones
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int g = static_cast<int>(threadIdx.x) * kPerThread + j;
    total[j] = before[j] = 0;
    if (g < bins) {
      total[j] = counts != nullptr ? all[g] : own[g];
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
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) mine += (total[j] + kPlanTileRows - 1) / kPlanTileRows;
    int v = mine;
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
    int slot = v - mine + (warp > 0 ? warp_sums[warp - 1] : 0);
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
      order[start[bin[i]] + seen[warp * ld + bin[i]] + rank[i]] =
          bin[i] < groups || tiles != nullptr ? static_cast<int32_t>(q0 + i * 32 + lane) : -1;
  }
}

template <int kRounds>
__global__ void __launch_bounds__(kPlanThreads) group_rows_kernel(const int32_t* ids, int64_t rows, int groups,
                                                                  const int32_t* counts, int32_t* offsets,
                                                                  int32_t* order, int4* tiles) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ int32_t plan_smem[];
  plan_block<kPlanThreads, kRounds>(ids, rows, groups, counts, offsets, order, tiles, plan_smem);
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
