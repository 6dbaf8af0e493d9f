// Entry points of the projections whose weights are chosen per row: routing, row plans, the
// experts' products, low-rank adapters.  Included by api.cu only, after its helpers.
#pragma once

#include "adapter_kernel.cuh"
#include "grouped_kernel.cuh"
#include "host_runtime.h"
#include "route_kernel.cuh"
#include "tensor_maps.h"

namespace {

static_assert(kMaxGroups == CPUOPS_B200_MAX_GROUPS && kMaxTopK == CPUOPS_B200_MAX_TOP_K &&
                  kMaxRank == CPUOPS_B200_MAX_RANK,
              "kernels and header agree on the limits");

int refuse(const char* what) {
  set_error("%s", what);
  return CPUOPS_B200_STATUS_INVALID_ARGUMENTS;
}

int row_kernels_ready(DeviceState& st);

// A call on its device: the device's lock and the stream it runs on.
struct RowCall {
  DeviceRestore restore;
  DeviceState* st = nullptr;
  std::unique_lock<std::mutex> lock;
  cudaStream_t stream = nullptr;
  bool async = false;

  template <typename Desc>
  int enter(const Desc& d) {
    if (int rc = init_device(d.device, &st)) return rc;
    lock = std::unique_lock<std::mutex>(st->mu);
    t_tm_cache = st->tm_cache;
    stream = d.stream ? static_cast<cudaStream_t>(d.stream) : st->stream;
    async = (d.flags & CPUOPS_B200_FLAG_ASYNC) != 0;
    // (a synchronous call ends with a wait, which would end the capture)
    if (!async && stream_is_capturing(stream)) return refuse("a call on a stream that is being captured needs FLAG_ASYNC");
    return row_kernels_ready(*st);
  }
  // Every pointer given (nulls apart) is this device's memory.
  int check(int memory_space, std::initializer_list<const void*> pointers) const {
    if (memory_space == CPUOPS_B200_MEM_DEVICE) return 0;
    for (const void* p : pointers) {
      if (!p) continue;
      cudaPointerAttributes attr;
      if (cudaPointerGetAttributes(&attr, p) != cudaSuccess) {
        cudaGetLastError();
        attr.type = cudaMemoryTypeUnregistered;
      }
      if (attr.type == cudaMemoryTypeManaged) continue;
      if (attr.type != cudaMemoryTypeDevice || attr.device != st->device) {
        set_error("pointer %p is not memory of device %d (this call takes device memory only)", p, st->device);
        return CPUOPS_B200_STATUS_INVALID_ARGUMENTS;
      }
    }
    return 0;
  }
  int finish() { return async ? CPUOPS_B200_STATUS_SUCCESS : finish_stream(*st, stream); }
};

// One launch that may become resident while the kernel before it in the stream ends (every kernel
// here waits for that one before it touches memory).
template <typename... Formal, typename... Actual>
int launch_after(void (*kernel)(Formal...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Actual... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));  // (its own error: another call's may still be kept)
  g_launches.fetch_add(1);
  return 0;
}

bool type_ok(int t) { return t == CPUOPS_B200_TYPE_F32 || t == CPUOPS_B200_TYPE_F16 || t == CPUOPS_B200_TYPE_BF16; }

template <typename Desc>
int check_desc(const Desc* d) {
  if (d && d->struct_size == sizeof(Desc)) return 0;
  set_error("descriptor is null or struct_size does not match this library (ABI %d)", CPUOPS_B200_ABI_VERSION);
  return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
}

using RouteKernel = void (*)(RouteParams);
RouteKernel route_kernel_for(int experts) {
  const int per_lane = (experts + 31) / 32;
  return per_lane <= 1 ? route_kernel<1> : per_lane <= 2 ? route_kernel<2> : per_lane <= 4 ? route_kernel<4>
       : per_lane <= 8 ? route_kernel<8> : per_lane <= 16 ? route_kernel<16> : route_kernel<32>;
}
using RouteFewKernel = void (*)(RouteParams, int32_t*, int32_t*);
RouteFewKernel route_few_kernel_for(int experts) {
  const int per_lane = (experts + 31) / 32;
  return per_lane <= 1 ? route_few_kernel<1> : per_lane <= 2 ? route_few_kernel<2> : per_lane <= 4 ? route_few_kernel<4>
       : per_lane <= 8 ? route_few_kernel<8> : per_lane <= 16 ? route_few_kernel<16> : route_few_kernel<32>;
}

using GroupedKernel = void (*)(CUtensorMap, CUtensorMap, GroupedParams);
template <int KIND>
GroupedKernel grouped_kernel_for(bool gated, bool two) {
  if (two) return gated ? grouped_mx_kernel<KIND, true, true> : grouped_mx_kernel<KIND, false, true>;
  return gated ? grouped_mx_kernel<KIND, true, false> : grouped_mx_kernel<KIND, false, false>;
}
GroupedKernel grouped_kernel(int kind, bool gated, bool two) {
  return kind == kKindMxf4 ? grouped_kernel_for<kKindMxf4>(gated, two) : grouped_kernel_for<kKindMxf8>(gated, two);
}

// Tiles of one launch of the experts' kernel.
struct GroupedChoice {
  bool two = false;     // two W tiles per CTA
  bool sorted = false;  // rows of A copied in plan order first
  int BN = 32, stages = 2, tile_cols = 128;
};

// The kernels for many rows: ranks in chunks of 16 or 64.
using AdapterTileKernel = void (*)(AdapterTileParams);
template <typename X, typename W>
AdapterTileKernel adapter_down_for(bool narrow, bool wide, int* smem) {
  *smem = narrow ? down_smem_bytes<X, 16>() : down_smem_bytes<X, 64>();
  if (narrow) return wide ? adapter_down_kernel<X, W, 16, true> : adapter_down_kernel<X, W, 16, false>;
  return wide ? adapter_down_kernel<X, W, 64, true> : adapter_down_kernel<X, W, 64, false>;
}
AdapterTileKernel adapter_down(int x_type, int w_type, bool narrow, bool wide, int* smem) {
  if (x_type == CPUOPS_B200_TYPE_F16) return adapter_down_for<__half, __half>(narrow, wide, smem);
  if (x_type == CPUOPS_B200_TYPE_BF16) return adapter_down_for<__nv_bfloat16, __nv_bfloat16>(narrow, wide, smem);
  return w_type == CPUOPS_B200_TYPE_F16 ? adapter_down_for<float, __half>(narrow, wide, smem)
                                        : adapter_down_for<float, __nv_bfloat16>(narrow, wide, smem);
}
int adapter_up_smem(int w_type, int rank_pad) {
  return up_smem_bytes(rank_pad, w_type == CPUOPS_B200_TYPE_F16 ? UpTerms<__half>::kCount : UpTerms<__nv_bfloat16>::kCount);
}
template <typename W>
AdapterTileKernel adapter_up_for(int rank_pad, bool whole) {
  if (up_stages(rank_pad) == 3) return whole ? adapter_up_kernel<W, 3, true> : adapter_up_kernel<W, 3, false>;
  return whole ? adapter_up_kernel<W, 2, true> : adapter_up_kernel<W, 2, false>;
}
AdapterTileKernel adapter_up(int w_type, int rank_pad, bool whole) {
  return w_type == CPUOPS_B200_TYPE_F16 ? adapter_up_for<__half>(rank_pad, whole) : adapter_up_for<__nv_bfloat16>(rank_pad, whole);
}

// Kernel attributes, once per device (under its lock): the most dynamic shared memory each may take.
int row_kernels_ready(DeviceState& st) {
  static bool ready[64] = {};
  if (ready[st.device]) return 0;
  constexpr auto kMost = cudaFuncAttributeMaxDynamicSharedMemorySize;
  for (int experts = 32; experts <= kMaxGroups; experts *= 2) {
    CUDA_TRY(cudaFuncSetAttribute(route_kernel_for(experts), kMost, static_cast<int>(route_smem_bytes(experts, experts))));
    CUDA_TRY(cudaFuncSetAttribute(route_few_kernel_for(experts), kMost, static_cast<int>(route_few_smem_bytes(experts, experts))));
  }
  CUDA_TRY(cudaFuncSetAttribute(group_rows_kernel<1>, kMost, plan_smem_bytes(kMaxGroups)));
  CUDA_TRY(cudaFuncSetAttribute(group_rows_kernel<kPlanRounds>, kMost, plan_smem_bytes(kMaxGroups)));
  for (int kind : {kKindMxf8, kKindMxf4})
    for (bool gated : {false, true})
      for (bool two : {false, true}) CUDA_TRY(cudaFuncSetAttribute(grouped_kernel(kind, gated, two), kMost, st.smem_optin));
  for (int x_type : {kTypeF32, kTypeF16, kTypeBf16})
    for (int w_type : {kTypeF16, kTypeBf16})
      for (bool narrow : {false, true})
        for (bool wide : {false, true}) {
          int smem = 0;
          AdapterTileKernel down = adapter_down(x_type, w_type, narrow, wide, &smem);
          CUDA_TRY(cudaFuncSetAttribute(down, kMost, smem));
        }
  for (int w_type : {kTypeF16, kTypeBf16})
    for (int rank : {128, kMaxRank})
      for (bool whole : {false, true})
        CUDA_TRY(cudaFuncSetAttribute(adapter_up(w_type, rank, whole), kMost, adapter_up_smem(w_type, rank)));
  ready[st.device] = true;
  return 0;
}

// ---- plans ---------------------------------------------------------------------------------

size_t plan_workspace(int64_t rows, int groups) {
  if (rows <= kPlanPairs) return 0;
  return static_cast<size_t>(plan_blocks(rows)) * (groups + 1) * sizeof(int32_t);
}

// `counts`: plan_workspace() bytes.
int launch_plan(const int32_t* ids, int64_t rows, int groups, int32_t* offsets, int32_t* order,
                int32_t* counts, int4* tiles, cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>(plan_blocks(rows));
  if (blocks > 1) {
    if (int rc = launch_after(count_ids_kernel, dim3(blocks), kPlanThreads, 0, stream, ids, rows, groups, counts)) return rc;
  }
  return launch_after(plan_rounds(rows) == 1 ? group_rows_kernel<1> : group_rows_kernel<kPlanRounds>, dim3(blocks), kPlanThreads, static_cast<size_t>(plan_smem_bytes(groups)), stream, ids, rows, groups,
                      static_cast<const int32_t*>(blocks > 1 ? counts : nullptr), offsets, order, tiles);
}

int group_rows_call(const cpuops_b200_group_rows_desc* d) {
  if (int rc = check_desc(d)) return rc;
  if (d->rows < 0 || d->groups < 0) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (!d->offsets || (d->rows > 0 && (!d->ids || !d->order))) return refuse("group_rows: a buffer is missing");
  if (d->groups > kMaxGroups) {
    set_error("group_rows: %d groups, at most %d are supported", d->groups, kMaxGroups);
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->ids, d->offsets, d->order})) return rc;
  uint8_t* ws = nullptr;
  if (const size_t need = plan_workspace(d->rows, d->groups)) {
    if (int rc = ensure_workspace(*call.st, call.stream, need, &ws)) return rc;
  }
  if (int rc = launch_plan(d->ids, d->rows, d->groups, d->offsets, d->order, reinterpret_cast<int32_t*>(ws),
                           nullptr, call.stream))
    return rc;
  return call.finish();
}

// ---- routing -------------------------------------------------------------------------------

int route_call(const cpuops_b200_route_desc* d) {
  if (int rc = check_desc(d)) return rc;
  if (d->scoring != CPUOPS_B200_SCORE_SOFTMAX && d->scoring != CPUOPS_B200_SCORE_SIGMOID) {
    set_error("unknown scoring %d", d->scoring);
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  if (!type_ok(d->logits_type)) {
    set_error("unknown logits type %d", d->logits_type);
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  if (d->tokens < 0 || d->experts < 1 || d->top_k < 1) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (d->top_k > d->experts) return refuse("route: top_k exceeds the number of experts");
  if (d->n_groups < 1 || d->experts % d->n_groups != 0 || d->top_groups < 1 || d->top_groups > d->n_groups ||
      (d->group_best != 1 && d->group_best != 2))
    return refuse("route: n_groups must divide experts, top_groups lie in 1 .. n_groups, group_best be 1 or 2");
  if (d->experts > kMaxGroups || d->top_k > kMaxTopK) {
    set_error("route: %d experts, top_k %d; at most %d and %d are supported", d->experts, d->top_k, kMaxGroups, kMaxTopK);
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  const int64_t pairs = static_cast<int64_t>(d->tokens) * d->top_k;
  if (pairs > INT32_MAX) return refuse("route: tokens * top_k must fit 31 bits");
  if (!d->offsets != !d->order && pairs > 0) return refuse("route: a plan is both offsets and order");
  if (d->tokens > 0) {
    if (!d->logits || !d->ids || !d->weights) return refuse("route: logits, ids or weights missing");
    if (d->ld_logits < d->experts) return refuse("route: ld_logits is less than the number of experts");
  }
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->logits, d->bias, d->ids, d->weights, d->offsets, d->order})) return rc;
  uint8_t* ws = nullptr;
  if (d->offsets) {
    if (const size_t need = plan_workspace(pairs, d->experts)) {
      if (int rc = ensure_workspace(*call.st, call.stream, need, &ws)) return rc;
    }
  }
  if (d->tokens > 0) {
    RouteParams p;
    p.logits = d->logits;
    p.bias = d->bias;
    p.ids = d->ids;
    p.weights = d->weights;
    p.ld = d->ld_logits;
    p.type = d->logits_type;
    p.tokens = d->tokens;
    p.experts = d->experts;
    p.top_k = d->top_k;
    p.sigmoid = d->scoring == CPUOPS_B200_SCORE_SIGMOID ? 1 : 0;
    p.n_groups = d->n_groups;
    p.top_groups = d->top_groups;
    p.group_best = d->group_best;
    p.renormalize = d->renormalize ? 1 : 0;
    p.scale = d->scale;
    if (d->offsets && d->tokens <= kRouteFewTokens && pairs <= kRouteFewPairs) {
      if (int rc = launch_after(route_few_kernel_for(d->experts), dim3(1), kRouteWarps * 32,
                                route_few_smem_bytes(d->experts, d->n_groups), call.stream, p, d->offsets, d->order))
        return rc;
      return call.finish();
    }
    const unsigned blocks = static_cast<unsigned>((d->tokens + kRouteWarps - 1) / kRouteWarps);
    if (int rc = launch_after(route_kernel_for(d->experts), dim3(blocks), kRouteWarps * 32,
                              route_smem_bytes(d->experts, d->n_groups), call.stream, p))
      return rc;
  }
  if (d->offsets) {
    if (int rc = launch_plan(d->ids, pairs, d->experts, d->offsets, d->order, reinterpret_cast<int32_t*>(ws),
                             nullptr, call.stream))
      return rc;
  }
  return call.finish();
}

// ---- the experts' products -----------------------------------------------------------------

int grouped_stages(int smem_optin, int BN, int ka, int groups, bool two) {
  return std::min(kGroupedMaxStages, (smem_optin - grouped_smem_bytes(BN, 0, ka, groups, two)) /
                                         (grouped_stage_bytes(BN, two) + grouped_atoms(BN, ka, two) * 512));
}

// The host knows how many pairs there are, not how they spread: it plans for equal groups.
//   * Few pairs per group (below 48): one W tile, room for twice the average, rows gathered.  Such calls are bound
//     by reading W, and the width does not matter to that.
//   * Many: the width and the tile count whose estimated time is least: rounds of items over the SMs
//     x (k-blocks x cycles per k-block + a fixed part).  A k-block takes its loads' time at 44 bytes a
//     cycle, what an SM was seen to get out of L2 beside all others, or its MMAs' (2 cycles per pair
//     and W tile); with one set of accumulators D's stores, 100 cycles per pair, are not hidden.
//     (us, 8192 rows x 4096 x 4096 e4m3, one group: two tiles of 112 pairs 171, 144 214, 192 190; one
//     tile of 112 271, 192 232.)
GroupedChoice choose_grouped(const DeviceState& st, int rows, int n, int groups, int k_blocks, int ka, bool gated) {
  GroupedChoice best;
  const int average = rows / std::max(1, groups), sms = st.sms();
  if (average < 48) {
    static_assert(2 * 47 <= kGroupedMaxGathered && kGroupedMaxGathered % 32 == 0, "twice the average, in steps of 32");
    best.BN = std::max(32, (std::min(rows, 2 * average) + 31) / 32 * 32);
    best.stages = grouped_stages(st.smem_optin, best.BN, ka, groups, false);
    best.tile_cols = gated ? 64 : 128;
    return best;
  }
  double least = 0.0;
  for (bool two : {true, false}) {
    for (int BN = 64; BN <= kGroupedMaxBN; BN += 16) {
      GroupedChoice c;
      c.two = two;
      c.sorted = true;
      c.BN = BN;
      c.tile_cols = (gated ? 64 : 128) * (two ? 2 : 1);
      c.stages = grouped_stages(st.smem_optin, BN, ka, groups, two);
      if (c.stages < 3) continue;  // (longer than a run of the scale writers)
      const int wide = average + average / 8;  // (groups differ: cuts for a somewhat larger one)
      const int cuts = (wide + BN - 1) / BN, width = ((average + cuts - 1) / cuts + 15) / 16 * 16;
      const int64_t items = static_cast<int64_t>(groups) * cuts * ((n + c.tile_cols - 1) / c.tile_cols);
      const double rounds = static_cast<double>((items + sms - 1) / sms);
      const double block = std::max(2.0 * width * (two ? 2 : 1), (16384.0 * (two ? 2 : 1) + 128.0 * BN) / 44.0);
      const double drain = grouped_acc_sets(BN, ka, two) == 2 ? 1000.0 : 1000.0 + 100.0 * width;
      const double cycles = rounds * (k_blocks * block + drain);
      if (least == 0.0 || cycles < least) {
        least = cycles;
        best = c;
      }
    }
  }
  return best;
}

int gemm_grouped_call(const cpuops_b200_gemm_grouped_desc* d) {
  if (int rc = check_desc(d)) return rc;
  auto ok_fmt = [](int f) { return f == CPUOPS_B200_FMT_E4M3 || f == CPUOPS_B200_FMT_E5M2 || f == CPUOPS_B200_FMT_E2M1; };
  if (!ok_fmt(d->a_format) || !ok_fmt(d->b_format)) {
    set_error("MX operands must be e4m3, e5m2 or e2m1");
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  const bool fp4_a = d->a_format == CPUOPS_B200_FMT_E2M1, fp4_b = d->b_format == CPUOPS_B200_FMT_E2M1;
  if (fp4_a && !fp4_b) {
    set_error("gemm_grouped: e2m1 rows under 8-bit weights are not built");
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  const bool mixed = fp4_b && !fp4_a;
  const int rows = d->rows, n = d->n, k = d->k, groups = d->groups;
  if (rows < 0 || n < 0 || k < 0 || groups < 0) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (rows == 0 || n == 0) return CPUOPS_B200_STATUS_SUCCESS;
  if (k == 0) return refuse("gemm_grouped: k must be positive");
  if (groups > kMaxGroups) {
    set_error("gemm_grouped: %d groups, at most %d are supported", groups, kMaxGroups);
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  if (d->pairs_per_a_row < 1 || d->pairs_per_d_row < 1 || rows % d->pairs_per_d_row != 0)
    return refuse("gemm_grouped: pairs_per_a_row and pairs_per_d_row must be positive, the latter divide rows");
  if (d->a_rows < 1 || static_cast<int64_t>(d->a_rows) * d->pairs_per_a_row < rows)
    return refuse("gemm_grouped: A has fewer rows than the pairs need");
  const bool summed = d->pairs_per_d_row > 1;
  if (!d->a || !d->b || !d->a_scales || !d->b_scales || !d->offsets || !d->order || !d->d || (summed && !d->ids))
    return refuse("gemm_grouped: a buffer is missing");
  const int64_t n_b = d->gated ? 2 * static_cast<int64_t>(n) : n;
  const int blocks32 = static_cast<int>((static_cast<int64_t>(k) + 31) / 32);
  if (d->lda < k || d->ldb < k || d->ld_scales_a < blocks32 || d->ld_scales_b < blocks32 || d->ldd < n ||
      d->b_group_rows < n_b)
    return refuse("gemm_grouped: a leading dimension (or b_group_rows) is too small");
  const int64_t b_rows = (groups > 0 ? static_cast<int64_t>(groups - 1) * d->b_group_rows : 0) + n_b;
  if (b_rows > INT32_MAX - 256) return refuse("gemm_grouped: groups * b_group_rows must fit 31 bits");
  // operand rows as TMA takes them
  const int64_t a_pitch = fp4_a ? d->lda / 2 : d->lda, b_pitch = fp4_b ? d->ldb / 2 : d->ldb;
  auto on = [](const void* ptr, int64_t pitch, int to) { return reinterpret_cast<uintptr_t>(ptr) % to == 0 && pitch % to == 0; };
  if ((fp4_a && (d->lda & 1)) || (fp4_b && (d->ldb & 1)) || (fp4_b && (k & 1)))
    return refuse("gemm_grouped: e2m1 operands need an even k and even leading dimensions");
  if (!on(d->a, a_pitch, 16) || !on(d->b, b_pitch, mixed ? 32 : 16) || (mixed && k % 128 != 0))
    return refuse("gemm_grouped: A and B must be 16-byte aligned with rows a multiple of 16 bytes apart (e2m1 weights "
                  "under 8-bit rows: 32 bytes, and k a multiple of 128)");
  const int kind = fp4_a ? kKindMxf4 : kKindMxf8;
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  DeviceState& st = *call.st;
  if (int rc = call.check(d->memory_space, {d->a, d->b, d->a_scales, d->b_scales, d->offsets, d->order, d->ids,
                                            d->row_weights, d->d}))
    return rc;

  GroupedParams p;
  memset(&p, 0, sizeof(p));
  p.sw = static_cast<const uint8_t*>(d->b_scales);
  p.sx = static_cast<const uint8_t*>(d->a_scales);
  p.offsets = d->offsets;
  p.order = d->order;
  p.row_weights = d->row_weights;
  p.ld_sw = d->ld_scales_b;
  p.ld_sx = d->ld_scales_a;
  p.rows = rows;
  p.groups = groups;
  p.n = n;
  p.b_group_rows = d->b_group_rows;
  p.a_rows = d->a_rows;
  p.pairs_per_a_row = d->pairs_per_a_row;
  const int ka = kind == kKindMxf4 ? 2 : 1;
  p.k_blocks = static_cast<int>((static_cast<int64_t>(k) + (kind == kKindMxf4 ? 255 : 127)) / (kind == kKindMxf4 ? 256 : 128));
  p.kblocks32 = blocks32;
  const GroupedChoice choice = choose_grouped(st, rows, n, groups, p.k_blocks, ka, d->gated != 0);
  p.BN = choice.BN;
  p.stages = choice.stages;
  p.sorted = choice.sorted ? 1 : 0;
  p.tiles = static_cast<int>((static_cast<int64_t>(n) + choice.tile_cols - 1) / choice.tile_cols);
  auto alignment = [&](const void* ptr, int64_t ld) { return on(ptr, ld, 16) ? 16 : on(ptr, ld, 4) ? 4 : 1; };
  p.align_w = alignment(d->b_scales, d->ld_scales_b);
  p.align_x = alignment(d->a_scales, d->ld_scales_a);
  p.w_tile_bytes = (choice.two ? 2 : 1) * kTileM * (mixed ? 64 : 128);
  {
    auto code = [](int f) { return f == CPUOPS_B200_FMT_E5M2 ? 1u : f == CPUOPS_B200_FMT_E2M1 ? 5u : 0u; };
    p.idesc = kind == kKindMxf4 ? make_idesc_block_scaled(1u, 1u, kTileM, 0)
                                : make_idesc_block_scaled(code(d->b_format), code(d->a_format), kTileM, 0);
  }
  p.wait_budget_us = g_wait_budget_us.load();
  p.error = st.error_dev;

  const int64_t most_items = (static_cast<int64_t>(std::min(groups, rows)) + rows / p.BN) * p.tiles;
  if (most_items > INT32_MAX) return refuse("gemm_grouped: the problem has more tiles than fit 31 bits");
  const unsigned row_blocks = static_cast<unsigned>(std::min<int64_t>((static_cast<int64_t>(rows) + 7) / 8, 8 * st.sm_count));
  if (!summed && d->ids) {  // rows without a group are zeros, as in a sum
    if (int rc = launch_after(zero_rows_kernel, dim3(row_blocks), 256, 0, call.stream, d->ids, groups, rows, n, d->d,
                              static_cast<int64_t>(d->ldd)))
      return rc;
  }
  const int row_bytes = fp4_a ? k / 2 : k;
  const int64_t x_pitch = align_up(row_bytes, 16), sx_pitch = align_up(blocks32, 16);
  Plan plan;
  const size_t off_x = plan.take(p.sorted ? static_cast<size_t>(rows) * x_pitch : 0);
  const size_t off_sx = plan.take(p.sorted ? static_cast<size_t>(rows) * sx_pitch : 0);
  const size_t off_sum = plan.take(summed ? static_cast<size_t>(rows) * n * sizeof(float) : 0);
  uint8_t* ws = nullptr;
  if (plan.total > 0) {
    if (int rc = ensure_workspace(st, call.stream, plan.total, &ws)) return rc;
  }
  if (p.sorted) {
    p.sx = ws + off_sx;
    p.ld_sx = sx_pitch;
    p.align_x = 16;
    if (int rc = launch_after(gather_rows_kernel, dim3(row_blocks), 256, 0, call.stream, static_cast<const uint8_t*>(d->a), a_pitch,
                              static_cast<const uint8_t*>(d->a_scales), static_cast<int64_t>(d->ld_scales_a), d->order, rows,
                              d->a_rows, d->pairs_per_a_row, row_bytes, blocks32, ws + off_x, x_pitch, ws + off_sx, sx_pitch))
      return rc;
  }
  p.d = summed ? reinterpret_cast<float*>(ws + off_sum) : d->d;
  p.ldd = summed ? n : d->ldd;

  if (groups > 0) {
    CUtensorMap tmW, tmX;
    const uint32_t box = d->gated && !choice.two ? 16 : 128;
    if (mixed) {
      if (int rc = make_tensor_map_fp4_padded(&tmW, d->b, k, b_rows, b_pitch, box)) return rc;
    } else {
      if (int rc = make_tensor_map(&tmW, d->b, fp4_b ? k / 2 : k, b_rows, b_pitch, box)) return rc;
    }
    if (p.sorted) {
      if (int rc = make_tensor_map(&tmX, ws + off_x, row_bytes, rows, x_pitch, static_cast<uint32_t>(p.BN / 2))) return rc;
    } else {
      if (int rc = make_tensor_map(&tmX, d->a, row_bytes, d->a_rows, a_pitch, 1)) return rc;
    }
    // (one CTA per SM: it takes all of tensor memory)
    const int smem = std::max(grouped_smem_bytes(p.BN, p.stages, ka, groups, choice.two), 120 * 1024);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(most_items, st.sms()));
    if (int rc = launch_after(grouped_kernel(kind, d->gated != 0, choice.two), dim3(grid), grouped_threads(choice.two),
                              static_cast<size_t>(smem), call.stream, tmW, tmX, p))
      return rc;
  }
  if (summed) {
    const int64_t d_rows = rows / d->pairs_per_d_row;
    const dim3 grid(static_cast<unsigned>((n + 255) / 256), static_cast<unsigned>(std::min<int64_t>(d_rows, 65535)));
    if (int rc = launch_after(sum_pairs_kernel, grid, 256, 0, call.stream, static_cast<const float*>(p.d), d->ids, groups,
                              d->pairs_per_d_row, d_rows, n, d->d, static_cast<int64_t>(d->ldd)))
      return rc;
  }
  return call.finish();
}

// ---- adapters ------------------------------------------------------------------------------

using AdapterKernel = void (*)(AdapterParams);
AdapterKernel adapter_rows(int x_type, int w_type) {
  if (x_type == CPUOPS_B200_TYPE_F16) return adapter_rows_kernel<__half, __half>;
  if (x_type == CPUOPS_B200_TYPE_BF16) return adapter_rows_kernel<__nv_bfloat16, __nv_bfloat16>;
  return w_type == CPUOPS_B200_TYPE_F16 ? adapter_rows_kernel<float, __half> : adapter_rows_kernel<float, __nv_bfloat16>;
}

// Rows sorted by adapter, then both products tile by tile.
int adapters_by_tiles(RowCall& call, const AdapterParams& p, int x_type, int w_type) {
  AdapterTileParams t;
  t.a = p;
  t.rank_pad = (p.rank + 15) / 16 * 16;
  const int64_t tiles = plan_max_tiles(p.m, p.adapters);
  const bool narrow = p.rank <= 16;
  const int chunks = narrow ? 1 : (p.rank + 63) / 64;
  // parts of k: as many as fit the SMs at once with three CTAs each, at least four stages to a part
  int parts = static_cast<int>(std::min<int64_t>(3 * call.st->sms() / (tiles * chunks), 16));
  parts = std::max(1, std::min(parts, (p.k + 4 * kDownDepth - 1) / (4 * kDownDepth)));
  t.depth = ((p.k + parts - 1) / parts + kDownDepth - 1) / kDownDepth * kDownDepth;
  t.splits = (p.k + t.depth - 1) / t.depth;
  // Columns per CTA of the up kernel, two CTAs of which share an SM: of the counts that fill up to four
  // rounds of them, the one that leaves the fewest idle in the last round (of equal ones the least, since
  // every CTA reads u anew): 8192 rows, rank 64, n 4096: 2 CTAs per tile 70 us, 7 took 78.
  const int64_t steps = (p.n + kUpCols - 1) / kUpCols, slots = 2 * call.st->sms();
  int64_t ctas = 1;
  double best = 0.0;
  for (int64_t c = 1; c <= steps && (c == 1 || c * tiles <= 4 * slots); ++c) {
    const int64_t per = (steps + c - 1) / c, rounds = (tiles * c + slots - 1) / slots;
    const double busy = static_cast<double>(tiles * steps) / static_cast<double>(rounds * slots * per);
    if (busy > best + 0.02) {
      best = busy;
      ctas = c;
    }
  }
  t.up_cols = static_cast<int>((steps + ctas - 1) / ctas) * kUpCols;
  Plan plan;
  const size_t off_counts = plan.take(plan_workspace(p.m, p.adapters));
  const size_t off_order = plan.take(static_cast<size_t>(p.m) * sizeof(int32_t));
  const size_t off_tiles = plan.take(static_cast<size_t>(tiles) * sizeof(int4));
  const size_t off_u = plan.take(static_cast<size_t>(t.splits) * p.m * t.rank_pad * sizeof(float));
  uint8_t* ws = nullptr;
  if (int rc = ensure_workspace(*call.st, call.stream, plan.total, &ws)) return rc;
  int32_t* order = reinterpret_cast<int32_t*>(ws + off_order);
  int4* table = reinterpret_cast<int4*>(ws + off_tiles);
  t.order = order;
  t.tiles = table;
  t.u = reinterpret_cast<float*>(ws + off_u);
  if (int rc = launch_plan(p.ids, p.m, p.adapters, nullptr, order, reinterpret_cast<int32_t*>(ws + off_counts), table,
                           call.stream))
    return rc;
  int smem = 0;
  AdapterTileKernel down = adapter_down(x_type, w_type, narrow, p.align_k == 16, &smem);
  if (int rc = launch_after(down, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(t.splits), static_cast<unsigned>(chunks)),
                            128, static_cast<size_t>(smem), call.stream, t))
    return rc;
  const bool whole = p.align_r == 16 && p.align_c == 16 && p.align_d == 16 && p.n % kUpCols == 0 && p.rank % 8 == 0;
  return launch_after(adapter_up(w_type, t.rank_pad, whole), dim3(static_cast<unsigned>((p.n + t.up_cols - 1) / t.up_cols),
                                               static_cast<unsigned>(tiles)),
                      256, static_cast<size_t>(adapter_up_smem(w_type, t.rank_pad)), call.stream, t);
}

// Whether rows are taken tile by tile.  By themselves they read their adapters anew, row by row, from L2 where rows
// share one: 3.3 TB/s of that were seen.  A step of a tile (64 columns, or 64 elements of k) takes its time
// however few rows the tile has, and an adapter in use has a tile at least.  us, tiles / rows by themselves:
//   rank 16, 4096 x 4096, 16 adapters: 128 rows 21 / 11.5, 256 22 / 23, 1024 30 / 82
//   the same of 128 adapters: 256 rows 63 / 27, 512 64 / 48, 1024 65 / 86
//   rank 64, 2048 x 2048, 64 adapters: 128 rows 35 / 28, 256 36 / 49
bool adapters_want_tiles(const AdapterParams& p, int sms) {
  const int64_t tiles = plan_max_tiles(p.m, p.adapters);
  if (p.adapters > kMaxGroups || tiles > 65535) return false;
  const double rows_us = 4.0 + 2.0 * p.m * static_cast<double>(p.rank) * (static_cast<double>(p.n) + p.k) / 3.3e6;
  const double up = static_cast<double>(tiles) * ((p.n + kUpCols - 1) / kUpCols) / (2.0 * sms);
  const double down = static_cast<double>(tiles) * ((p.k + kDownDepth - 1) / kDownDepth) * ((p.rank + 63) / 64) / (3.0 * sms);
  return 12.0 + 1.2 * (1.0 + p.rank / 64.0) * up + 0.5 * down < rows_us;
}

int adapters_call(const cpuops_b200_adapters_desc* d) {
  if (int rc = check_desc(d)) return rc;
  if (!type_ok(d->x_type) || !type_ok(d->w_type)) {
    set_error("unknown element type");
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  if (d->w_type == CPUOPS_B200_TYPE_F32 || (d->x_type != CPUOPS_B200_TYPE_F32 && d->x_type != d->w_type)) {
    set_error("adapters: A and B are f16 or bf16, X is f32 or of their type");
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  if (d->m < 0 || d->n < 0 || d->k < 0 || d->rank < 0 || d->adapters < 0) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (d->m == 0 || d->n == 0) return CPUOPS_B200_STATUS_SUCCESS;
  if (d->n > (1 << 30) || d->k > (1 << 30)) return refuse("adapters: n and k are at most 2^30");
  if (d->rank > kMaxRank) {
    set_error("adapters: rank %d, at most %d is supported", d->rank, kMaxRank);
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  // an empty product adds nothing: every row goes without
  const bool any = d->k > 0 && d->rank > 0 && d->adapters > 0;
  if (!d->ids || !d->c || !d->d || (any && (!d->x || !d->a || !d->b))) return refuse("adapters: a buffer is missing");
  if (d->ldc < d->n || d->ldd < d->n) return refuse("adapters: a leading dimension is too small");
  if (any && (d->ldx < d->k || d->lda < d->k || d->ldb < d->rank || d->a_stride < 0 || d->b_stride < 0))
    return refuse("adapters: a leading dimension is too small");
  if (d->c == d->d && d->ldc != d->ldd) return refuse("adapters: in place, C and D have the same leading dimension");
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->x, d->a, d->b, d->ids, d->scales, d->c, d->d})) return rc;
  AdapterParams p;
  memset(&p, 0, sizeof(p));
  p.x = d->x;
  p.a = d->a;
  p.b = d->b;
  p.ids = d->ids;
  p.scales = d->scales;
  p.c = d->c;
  p.d = d->d;
  p.ldx = d->ldx;
  p.lda = d->lda;
  p.ldb = d->ldb;
  p.a_stride = d->a_stride;
  p.b_stride = d->b_stride;
  p.ldc = d->ldc;
  p.ldd = d->ldd;
  p.m = d->m;
  p.n = d->n;
  p.k = d->k;
  p.rank = d->rank;
  p.adapters = any ? d->adapters : 0;
  const int x_size = d->x_type == CPUOPS_B200_TYPE_F32 ? 4 : 2;
  auto align = [](const void* ptr, int64_t ld, int64_t stride, int size) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(ptr) | static_cast<uint64_t>(ld * size) | static_cast<uint64_t>(stride * size);
    return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
  };
  p.align_k = std::min(align(d->x, d->ldx, 0, x_size), align(d->a, d->lda, d->a_stride, 2));
  p.align_r = align(d->b, d->ldb, d->b_stride, 2);
  p.align_c = align(d->c, d->ldc, 0, 4);
  p.align_d = align(d->d, d->ldd, 0, 4);
  if (any && adapters_want_tiles(p, call.st->sms())) {
    if (int rc = adapters_by_tiles(call, p, d->x_type, d->w_type)) return rc;
    return call.finish();
  }
  if (static_cast<int64_t>(d->m) * kAdapterCluster > INT32_MAX) return refuse("adapters: too many rows");
  if (int rc = launch_after(adapter_rows(d->x_type, d->w_type), dim3(static_cast<unsigned>(d->m) * kAdapterCluster),
                            kAdapterThreads, 0, call.stream, p))
    return rc;
  return call.finish();
}

}  // namespace

extern "C" {

CPUOPS_B200_API int cpuops_b200_route(const cpuops_b200_route_desc* d) { return route_call(d); }
CPUOPS_B200_API int cpuops_b200_group_rows(const cpuops_b200_group_rows_desc* d) { return group_rows_call(d); }
CPUOPS_B200_API int cpuops_b200_gemm_grouped(const cpuops_b200_gemm_grouped_desc* d) { return gemm_grouped_call(d); }
CPUOPS_B200_API int cpuops_b200_adapters(const cpuops_b200_adapters_desc* d) { return adapters_call(d); }

}  // extern "C"
