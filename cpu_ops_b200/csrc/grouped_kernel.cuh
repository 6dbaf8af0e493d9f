// The experts' products: for every pair q of group g in a row plan, D[q] = A[row of q] * B_g^T on MX
// operands (OCP MX fp8 / fp4, one E8M0 scale per 32 k-elements), f32 sums, optionally
// silu(gate) * up of two such products and a weight per pair.
//
// Kernel view, as in the small-m kernel (decode_kernel.cuh): the weights W (B_g, 128-row tiles)
// sit on the MMA M side, the pairs' rows X on the N side.  A work item is one tile of W times up
// to BN pairs of its group, over all of k.  Which groups have pairs, and how many, is known on
// the device only: every CTA reads the plan's offsets at its start, makes the prefix sum of the
// groups' item counts in shared memory, and takes items blockIdx.x, + gridDim.x, ...  Items of one
// group are neighbours, those of one W tile next to each other, so what runs at the same time
// shares W and X in L2 and W leaves HBM once.
//
//   * The N of an item is what its pairs need (a group's pairs are cut evenly, in steps of 16):
//     groups of any size waste less than 16 columns of tensor-core time per tile.
//   * X rows are gathered by TMA (tile::gather4, four rows by their numbers per instruction), one
//     lane of a warp for every four rows; their scales by the scale-writer warps, which read them by
//     row anyway.  A gather costs the TMA unit about 38 cycles whatever its rows, which W's own time hides
//     while items have few pairs.  With many, gather_rows_kernel copies the rows in plan order once,
//     and X comes in boxes of BN / 2 rows (2048 rows x 4 of 32 experts, 4096 x 4096 e4m3: 650 us
//     gathered, 275 copied, the copy's 10 included).
//   * Gated: a tile holds 64 gate rows and their 64 up rows, 16 and 16 in each warp's lane quarter, so
//     that the two accumulators of an output meet in one warp (lane l and l + 16): one exchange
//     between lanes, and D is written once, at its final size.
//   * A thread holds one W row (a column of D), so the lanes of a warp write 128 (gated 64)
//     contiguous bytes of one row of D at a time: rows go wherever the plan says, with no
//     staging.
//
// Roles (512 threads, kTwo 640): warp 0 TMA producer of W, warp 1 MMA issuer (owns tensor memory), warps
// 2-9 scale writers (two sets of four in turn), warps 10-11 load X (in turn), warps 12-15 (kTwo: -19)
// epilogue (one TMEM lane quarter each).  What a role does for a k-block is a chain of latencies of
// some 600 cycles (wait, a few operations, fence, arrival), which with one warp or set was longer
// than the k-block's loads took: hence the turns.
// Every wait is bounded, as in the other kernels.
#pragma once

#include "decode_kernel.cuh"
#include "route_kernel.cuh"

namespace b200 {

// Warps: 0 loads W, 1 issues MMAs, 2-9 write scales, 10-11 load X, from 12 on the epilogue.
constexpr int kGroupedEpilogueWarp = 12;
__host__ __device__ constexpr int grouped_threads(bool two) { return 32 * (kGroupedEpilogueWarp + (two ? 8 : 4)); }
constexpr int kGroupedMaxStages = 8;
constexpr int kGroupedMaxBN = 192;   // two accumulators and four slots of scales fit tensor memory
constexpr int kGroupedMaxGathered = 96;  // ... of launches that gather X row by row
// 16-byte scale chunks that each of the two sets of scale writers has in flight: of two k-blocks for e2m1
// (ka = 2 atoms), of four else.  (One token, 8 of 64 experts, 2048 x 4096 e2m1: with half as many 13.1 us, so 12.6.)
__host__ __device__ constexpr int grouped_fetch_ahead(bool two, int ka) { return (two ? 1 : 2) * ka; }

struct GroupedParams {
  const uint8_t* sw;          // W's scales, row-major
  const uint8_t* sx;          // X's
  const int32_t* offsets;     // the plan
  const int32_t* order;
  const float* row_weights;   // or null
  float* d;
  int32_t ldd;
  int64_t ld_sw, ld_sx;
  int32_t rows, groups;       // pairs; groups of the plan
  int32_t n;                  // columns of D
  int32_t b_group_rows;       // rows of W from one group to the next
  int32_t a_rows, pairs_per_a_row;
  int32_t tiles;              // W tiles of a group
  int32_t k_blocks, kblocks32;
  int32_t BN, stages;
  int32_t w_tile_bytes;       // what the loads of a W tile credit to the barrier
  int32_t align_w, align_x;   // scale rows start on multiples of 16, 4 or 1 bytes
  int32_t sorted;             // 1: X (and sx) hold a row per pair, in plan order
  uint32_t idesc;             // without N
  uint32_t wait_budget_us;
  int32_t* error;
};

// W tiles of a CTA: one, or (kTwo) two that share X.
__host__ __device__ inline int grouped_stage_bytes(int BN, bool two) { return (two ? 2 : 1) * kTileM * 128 + BN * 128; }
__host__ __device__ inline int grouped_atoms(int BN, int ka, bool two) { return ka * ((two ? 2 : 1) + (BN > 128 ? 2 : 1)); }
__host__ __device__ inline int grouped_staging_bytes(int BN, int ka, bool two) {
  return 2 * grouped_fetch_ahead(two, ka) * ((two ? 2 : 1) * kTileM + BN) * 16;
}
// Tensor memory: accumulators of BN columns (two sets of them, where they fit), four slots of scales.
__host__ __device__ inline int grouped_acc_sets(int BN, int ka, bool two) {
  return 2 * (two ? 2 : 1) * BN + kDecodeSfSlots * 4 * grouped_atoms(BN, ka, two) <= 512 ? 2 : 1;
}
// The first items of a CTA are worked out once, by all threads, and looked up by the roles.
constexpr int kGroupedTable = 64;
// Then the epilogue's list of an item's pairs and weights, for two items.
__host__ __device__ inline int grouped_table_bytes(int groups) {
  return (2 * (groups + 1) * 4 + 15) / 16 * 16 + kGroupedTable * 16 + 2 * kGroupedMaxBN * 8;
}
constexpr int kGroupedBarrierBytes = 256;
__host__ __device__ inline int grouped_smem_bytes(int BN, int stages, int ka, int groups, bool two) {
  return 1024 + stages * (grouped_stage_bytes(BN, two) + grouped_atoms(BN, ka, two) * 512) + grouped_staging_bytes(BN, ka, two) +
         grouped_table_bytes(groups) + kGroupedBarrierBytes;
}

// One item: a tile of a group's W times pairs order[p0 .. p0 + count).
struct GroupedItem {
  int group, tile, p0, count;
};

// Item `it` from the prefix sums (first[g] = items of the groups before g) and the groups' starts.
__device__ __forceinline__ GroupedItem grouped_item(const int32_t* first, const int32_t* start, int groups, int tiles,
                                                    int BN, int it) {
  int lo = 0, hi = groups;  // first[lo] <= it < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= it) lo = mid; else hi = mid;
  }
  const int pairs = start[lo + 1] - start[lo];
  const int cuts = (pairs + BN - 1) / BN;
  const int width = ((pairs + cuts - 1) / cuts + 15) & ~15;  // <= BN, a multiple of 16
  const int local = it - first[lo];
  GroupedItem item;
  item.group = lo;
  item.tile = local / cuts;
  const int cut = local - item.tile * cuts;
  item.p0 = start[lo] + cut * width;
  item.count = min(width, pairs - cut * width);  // (at least 1: all cuts but one hold width <= BN each)
  return item;
}

// Four rows of a 128-byte wide box, by their numbers (tile::gather4).
__device__ __forceinline__ void tma_gather4(uint32_t smem_dst, const CUtensorMap* tm, uint32_t bar, int32_t x,
                                            int32_t r0, int32_t r1, int32_t r2, int32_t r3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      :
      : "r"(smem_dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
      : "memory");
}

// 16 bytes of a scale row into this thread's own staging slot: `valid` of them exist, the others
// become zero.  Rows that start on 16- or 4-byte boundaries are copied asynchronously.
__device__ __forceinline__ void fetch_scales(uint32_t dst, const uint8_t* src, int valid, int align) {
  if (align == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
  } else if (align == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int left = min(4, max(0, valid - 4 * j));
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * j), "l"(src + (left > 0 ? 4 * j : 0)),
                   "r"(left)
                   : "memory");
    }
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < valid) w[j >> 2] |= static_cast<uint32_t>(src[j]) << (8 * (j & 3));
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                 : "memory");
  }
}

// kGated: silu(gate) * up.  KIND: kKindMxf8 (also fp4 weights under fp8 rows) or kKindMxf4.
// kTwo: two W tiles share a stage's X (gated: the gate's and the up projection's 128 rows).  A stage's
// loads take some 2000 cycles from the moment it is free, so the ring has to hold that much work:
// with one tile five stages of 144 pairs hold 1440 cycles of it, with two four stages hold 2300, and every
// role has twice the time for a k-block.  (275 -> 193 us, 2048 rows x 4 of 32 experts, 4096 x 4096 e4m3.)
template <int KIND, bool kGated, bool kTwo>
__global__ void __launch_bounds__(grouped_threads(kTwo), 1)
    grouped_mx_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                      const GroupedParams p) {
  constexpr int kSfBytes = KIND == kKindMxf4 ? 8 : 4;  // scale bytes per row and k-block
  constexpr int kKa = kSfBytes / 4;                    // atoms along k per operand
  constexpr int kUnitsPerChunk = 16 / kSfBytes;        // k-blocks served by one 16-byte fetch of a scale row
  constexpr int kTiles = kTwo ? 2 : 1;
  constexpr int kTileCols = 128 * kTiles / (kGated ? 2 : 1);  // columns of D per item
  constexpr int kThreads = grouped_threads(kTwo), kFetchAhead = grouped_fetch_ahead(kTwo, kKa);
  constexpr uint32_t kWBytes = kTiles * kTileM * 128;
  constexpr unsigned kAll = 0xffffffffu;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = ((raw_addr + 1023u) & ~1023u) - raw_addr;
  uint8_t* smem = smem_raw + pad;
  const uint32_t smem_base = raw_addr + pad;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = p.stages, BN = p.BN;
  const int x_halves = BN > 128 ? 2 : 1;
  const uint32_t stage_bytes = static_cast<uint32_t>(grouped_stage_bytes(BN, kTwo));
  const uint32_t atoms = static_cast<uint32_t>(grouped_atoms(BN, kKa, kTwo));
  const uint32_t atom_bytes = atoms * 512u;
  const uint32_t atom_base = smem_base + stages * stage_bytes;
  const uint32_t staging_base = atom_base + stages * atom_bytes;
  const uint32_t table_off = staging_base + static_cast<uint32_t>(grouped_staging_bytes(BN, kKa, kTwo)) - smem_base;
  int4* table = reinterpret_cast<int4*>(smem + table_off);        // [kGroupedTable]
  int2* lists = reinterpret_cast<int2*>(table + kGroupedTable);   // [2][kGroupedMaxBN]: pair, weight
  int32_t* first = reinterpret_cast<int32_t*>(lists + 2 * kGroupedMaxBN);  // [groups + 1]
  int32_t* start = first + p.groups + 1;                          // [groups + 1]
  const uint32_t bar_base = smem_base + table_off + static_cast<uint32_t>(grouped_table_bytes(p.groups));
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kGroupedMaxStages + s); };
  auto acc_full_bar = [&](int b) { return bar_base + 8u * (2 * kGroupedMaxStages + b); };
  auto acc_empty_bar = [&](int b) { return bar_base + 8u * (2 * kGroupedMaxStages + 2 + b); };
  const uint32_t drain_bar = bar_base + 8u * (2 * kGroupedMaxStages + 4);
  constexpr int kBarriers = 2 * kGroupedMaxStages + 5;
  static_assert(8 * kBarriers + 8 <= kGroupedBarrierBytes, "barrier region too small");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (bar_base - smem_base) + 8 * kBarriers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint64_t budget_ns = static_cast<uint64_t>(p.wait_budget_us) * 1000ull;
  const int acc_sets = grouped_acc_sets(BN, kKa, kTwo), acc_cols = kTiles * BN;

  if (warp == 2) {
    if (lane < kBarriers) {
      // full: the two producers' arrive.expect_tx and one arrival per scale-writer warp; empty,
      // accumulator full, drain: one tcgen05.commit; accumulator empty: the epilogue warps
      uint32_t count = 1u;
      if (lane < kGroupedMaxStages) count = 6u;
      if (lane == 2 * kGroupedMaxStages + 2 || lane == 2 * kGroupedMaxStages + 3) count = 4u * kTiles;
      mbar_init(bar_base + 8u * static_cast<uint32_t>(lane), count);
    }
    if (lane == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512u);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmW);
    prefetch_tensormap(&tmX);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // Whatever the array holds, the starts become an ascending sequence within 0 .. rows: no item
  // reaches outside `order`, and there are no more items than the launcher allowed for.
  for (int g = threadIdx.x; g <= p.groups; g += kThreads) start[g] = min(max(p.offsets[g], 0), p.rows);
  __syncthreads();
  if (warp == 2) {
    int sum = 0, high = start[0];  // items and highest start so far
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      const int g = g0 + lane;
      int end = g < p.groups ? start[g + 1] : 0;
      if (lane == 0) end = max(end, high);
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int up = __shfl_up_sync(kAll, end, s);
        if (lane >= s) end = max(end, up);
      }
      int begin = __shfl_up_sync(kAll, end, 1);
      if (lane == 0) begin = high;
      const int own = (end - begin + BN - 1) / BN * p.tiles;
      int v = own;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int up = __shfl_up_sync(kAll, v, s);
        if (lane >= s) v += up;
      }
      if (g < p.groups) {
        first[g] = sum + v - own;
        start[g + 1] = end;
      }
      sum += __shfl_sync(kAll, v, 31);
      high = __shfl_sync(kAll, end, 31);
    }
    if (lane == 0) first[p.groups] = sum;
  }
  __syncthreads();
  if (threadIdx.x < kGroupedTable) {
    const int64_t it = blockIdx.x + static_cast<int64_t>(threadIdx.x) * gridDim.x;
    if (it < first[p.groups]) {
      const GroupedItem item = grouped_item(first, start, p.groups, p.tiles, BN, static_cast<int>(it));
      table[threadIdx.x] = make_int4(item.group, item.tile, item.p0, item.count);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int step = static_cast<int>(gridDim.x), n_all = first[p.groups];
  const int n_items = n_all > static_cast<int>(blockIdx.x) ? (n_all - 1 - static_cast<int>(blockIdx.x)) / step + 1 : 0;
  // This CTA's item j: work item blockIdx.x + j gridDim.x.  (Worked out anew it is a search and three
  // divisions, some 700 cycles of every role.)
  auto item_at = [&](int j) {
    if (j < kGroupedTable) {
      const int4 v = table[j];
      return GroupedItem{v.x, v.y, v.z, v.w};
    }
    return grouped_item(first, start, p.groups, p.tiles, BN, static_cast<int>(blockIdx.x) + j * step);
  };
  // The pair at place p0 + r of an item's run, or -1.
  auto pair_at = [&](const GroupedItem& item, int r) {
    if (r >= item.count) return -1;
    const int q = p.order[item.p0 + r];
    return q >= 0 && q < p.rows ? q : -1;
  };
  // What finds the row of X behind the pair at place p0 + r of item j: fetched an item ahead ...
  auto x_pair = [&](int j, int r) {
    if (j >= n_items) return -1;
    const GroupedItem item = item_at(j);
    if (p.sorted) return r < item.count ? item.p0 + r : -1;
    return pair_at(item, r);
  };
  // ... and the row itself, or -1.
  auto x_row = [&](int q) { return p.sorted || q < 0 ? q : min(q / p.pairs_per_a_row, p.a_rows - 1); };
  auto columns_of = [&](const GroupedItem& item) { return max(16, (item.count + 15) & ~15); };

  if (warp == 0) {
    // ------------------------------ W producer ------------------------------
    const uint32_t el = elect_one() ? 1u : 0u;
    int s = 0;
    uint32_t ph = 0;
    bool alive = true;
    for (int it = 0; it < n_items && alive; ++it) {
      const GroupedItem item = item_at(it);
      const int base = item.group * p.b_group_rows;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        if (!__all_sync(kAll, mbar_wait_bounded(empty_bar(s), ph ^ 1u, abort_flag, budget_ns))) {
          if (el) {
            leave_error(p.error, kErrProducerWait);
            *abort_flag = 1;
          }
          alive = false;
          break;
        }
        mbar_expect_tx_p(full_bar(s), static_cast<uint32_t>(p.w_tile_bytes), el);
        const uint32_t dst = smem_base + s * stage_bytes;
        if constexpr (kTwo) {
          const int row = base + item.tile * (kGated ? kTileM : 2 * kTileM);
          tma_load_2d_g<false>(dst, &tmW, full_bar(s), kb * 128, row, el);
          tma_load_2d_g<false>(dst + kTileM * 128, &tmW, full_bar(s), kb * 128, row + (kGated ? p.n : kTileM), el);
        } else if constexpr (kGated) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int row = base + item.tile * 64 + 16 * q;
            tma_load_2d_g<false>(dst + (32 * q) * 128, &tmW, full_bar(s), kb * 128, row, el);
            tma_load_2d_g<false>(dst + (32 * q + 16) * 128, &tmW, full_bar(s), kb * 128, row + p.n, el);
          }
        } else {
          tma_load_2d_g<false>(dst, &tmW, full_bar(s), kb * 128, base + item.tile * kTileM, el);
        }
        if (++s == stages) { s = 0; ph ^= 1u; }
      }
    }
    if (*abort_flag != 0 && el) {
      // give the copies already issued time to land before the CTA exits
      const uint64_t t_end = global_timer_ns() + 200000;
      while (global_timer_ns() < t_end) __nanosleep(1000);
    }
    __syncwarp();
  } else if (warp == 10 || warp == 11) {
    // ------------------------------ X ------------------------------
    // Two warps, k-blocks in turn (as for the scale writers' runs, a ring of two stages or more keeps the
    // parities apart).  Rows in plan order: one or two boxes of BN / 2 rows.  Otherwise lane l
    // gathers rows 4 l .. 4 l + 3 of the item's X (which is kGroupedMaxGathered wide at most); rows that do
    // not exist inside a group of four are read as the group's first one.  What is not loaded is left
    // as it is (its columns are computed and never read).
    const uint32_t el = elect_one() ? 1u : 0u;
    int s = 0, turn = 0;
    uint32_t ph = 0;
    bool alive = true;
    static_assert(kGroupedMaxGathered <= 128, "four rows to a lane");
    int pairs[4];
    auto fetch_pairs = [&](int j) {
      if (p.sorted) return;
#pragma unroll
      for (int i = 0; i < 4; ++i) pairs[i] = x_pair(j, 4 * lane + i);
    };
    fetch_pairs(0);
    for (int it = 0; it < n_items && alive; ++it) {
      const GroupedItem item = item_at(it);
      const bool mine = !p.sorted && 4 * lane < item.count;
      int row[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) row[j] = p.sorted ? -1 : x_row(pairs[j]);
      if (row[0] < 0) row[0] = 0;
#pragma unroll
      for (int j = 1; j < 4; ++j)
        if (row[j] < 0) row[j] = row[0];
      fetch_pairs(it + 1);
      const bool second = item.count > BN / 2;
      const uint32_t bytes = p.sorted ? static_cast<uint32_t>(BN / 2 * 128 * (second ? 2 : 1))
                                      : static_cast<uint32_t>((item.count + 3) >> 2) * 512u;
      for (int kb = 0; kb < p.k_blocks; kb += 2) {
        // of two k-blocks the first or the second is this warp's (the second may not be there)
        const bool later = turn != warp - 10;
        int mine_s = s;
        uint32_t mine_ph = ph;
        if (later && ++mine_s == stages) { mine_s = 0; mine_ph ^= 1u; }
        const int x_kb = kb + (later ? 1 : 0);
        if (x_kb < p.k_blocks) {
          if (!__all_sync(kAll, mbar_wait_bounded(empty_bar(mine_s), mine_ph ^ 1u, abort_flag, budget_ns))) {
            if (el) {
              leave_error(p.error, kErrProducerWait);
              *abort_flag = 1;
            }
            alive = false;
            break;
          }
          mbar_expect_tx_p(full_bar(mine_s), bytes, el);
          const uint32_t x_base = smem_base + mine_s * stage_bytes + kWBytes;
          if (p.sorted) {
            tma_load_2d_g<false>(x_base, &tmX, full_bar(mine_s), x_kb * 128, item.p0, el);
            tma_load_2d_g<false>(x_base + BN / 2 * 128, &tmX, full_bar(mine_s), x_kb * 128, item.p0 + BN / 2, second ? el : 0u);
          } else {
            __syncwarp();  // (the bytes are announced before any can arrive)
            const uint32_t dst = x_base + static_cast<uint32_t>(lane) * 512u;
            if (mine) tma_gather4(dst, &tmX, full_bar(mine_s), x_kb * 128, row[0], row[1], row[2], row[3]);
          }
        }
        const int done = min(2, p.k_blocks - kb);
        turn = (turn + done) & 1;
        s += done;
        if (s >= stages) { s -= stages; ph ^= 1u; }
      }
    }
    if (*abort_flag != 0) {
      const uint64_t t_end = global_timer_ns() + 200000;
      while (global_timer_ns() < t_end) __nanosleep(1000);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------- MMA issuer -------------------------------
    const uint32_t el = elect_one() ? 1u : 0u;
    const uint64_t op_hi64 = make_smem_desc_hi(16, 1024, 2);  // K-major, 128-byte swizzle
    const uint32_t op_hi = static_cast<uint32_t>(op_hi64 >> 32);
    const uint32_t a_lo0 = static_cast<uint32_t>(op_hi64) | (smem_base >> 4);
    const uint32_t b_lo0 = static_cast<uint32_t>(op_hi64) | ((smem_base + kWBytes) >> 4);
    const uint64_t sf_hi64 = make_smem_desc_hi(0, 128, 0);
    const uint32_t sf_hi = static_cast<uint32_t>(sf_hi64 >> 32);
    const uint32_t sf_lo0 = static_cast<uint32_t>(sf_hi64) | (atom_base >> 4);
    const uint32_t sf_t0 = tmem_base + static_cast<uint32_t>(acc_sets * acc_cols);
    const uint32_t sf_cols = 4u * atoms;
    const uint32_t sfb_half = 4u * static_cast<uint32_t>(x_halves);
    int s = 0, buf = 0, sf_q = 0;
    uint32_t ph = 0, acc_ph = 0;
    bool ok = true;
    for (int it = 0; it < n_items && ok; ++it) {
      const GroupedItem item = item_at(it);
      const uint32_t idesc = p.idesc | (static_cast<uint32_t>(columns_of(item)) >> 3) << 17;
      if (!__all_sync(kAll, mbar_wait_bounded(acc_empty_bar(buf), acc_ph ^ 1u, abort_flag, budget_ns))) {
        if (el) {
          leave_error(p.error, kErrMmaWaitAcc);
          *abort_flag = 1;
        }
        break;
      }
      tc_fence_after_sync();
      const uint32_t d_tmem0 = tmem_base + static_cast<uint32_t>(buf * acc_cols);
      uint32_t accumulate = 0;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        if (!__all_sync(kAll, mbar_wait_bounded(full_bar(s), ph, abort_flag, budget_ns))) {
          if (el) {
            leave_error(p.error, kErrMmaWaitFull);
            *abort_flag = 1;
          }
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t b_lo = b_lo0 + s * (stage_bytes >> 4);
        const uint32_t sf_t = sf_t0 + static_cast<uint32_t>(sf_q) * sf_cols, sfb_t = sf_t + 4u * kKa * kTiles;
        {
          uint32_t src = sf_lo0 + s * (atom_bytes >> 4), dst = sf_t;
          for (uint32_t a = 0; a < atoms; ++a, src += 32, dst += 4) tmem_cp_atom_g<false>(dst, src, sf_hi, el);
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const uint32_t a_lo = a_lo0 + s * (stage_bytes >> 4) + t * (kTileM * 128 / 16);
          const uint32_t d_tmem = d_tmem0 + static_cast<uint32_t>(t * BN), sfa_t = sf_t + 4u * kKa * t;
          if constexpr (KIND == kKindMxf8) {
            mma_mxf8f6f4_g<false>(d_tmem, a_lo, op_hi, b_lo, op_hi, idesc, sfa_t, sfb_t, accumulate, el);
            mma_mxf8f6f4_g<false>(d_tmem, a_lo + 2, op_hi, b_lo + 2, op_hi, idesc_with_sf_ids(idesc, 1, 1), sfa_t, sfb_t, 1u, el);
            mma_mxf8f6f4_g<false>(d_tmem, a_lo + 4, op_hi, b_lo + 4, op_hi, idesc_with_sf_ids(idesc, 2, 2), sfa_t, sfb_t, 1u, el);
            mma_mxf8f6f4_g<false>(d_tmem, a_lo + 6, op_hi, b_lo + 6, op_hi, idesc_with_sf_ids(idesc, 3, 3), sfa_t, sfb_t, 1u, el);
          } else {
            const uint32_t id2 = idesc_with_sf_ids(idesc, 2, 2);
            mma_mxf4_g<false>(d_tmem, a_lo, op_hi, b_lo, op_hi, idesc, sfa_t, sfb_t, accumulate, el);
            mma_mxf4_g<false>(d_tmem, a_lo + 2, op_hi, b_lo + 2, op_hi, id2, sfa_t, sfb_t, 1u, el);
            mma_mxf4_g<false>(d_tmem, a_lo + 4, op_hi, b_lo + 4, op_hi, idesc, sfa_t + 4u, sfb_t + sfb_half, 1u, el);
            mma_mxf4_g<false>(d_tmem, a_lo + 6, op_hi, b_lo + 6, op_hi, id2, sfa_t + 4u, sfb_t + sfb_half, 1u, el);
          }
        }
        accumulate = 1u;
        tc_commit_g<false>(empty_bar(s), el);  // frees the stage once these MMAs and copies have read it
        if (++sf_q == kDecodeSfSlots) sf_q = 0;
        if (++s == stages) { s = 0; ph ^= 1u; }
      }
      if (!ok) break;
      tc_commit_g<false>(acc_full_bar(buf), el);
      if (++buf == acc_sets) { buf = 0; acc_ph ^= 1u; }
    }
    // nothing may still be executing when tensor memory is released
    tc_commit_g<false>(drain_bar, el);
    if (!__all_sync(kAll, mbar_drain(drain_bar, 0)) && el) {
      leave_error(p.error, kErrDrainWait);
      *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp < 10) {
    // ------------------------------ scale writers ------------------------------
    // Two sets of four warps that take runs of kRun k-blocks in turn.  Thread r (0..127) of a set owns
    // row r of each W tile and rows r and r + 128 of X.  As in the small-m kernel it fetches its rows'
    // scale bytes 16 at a time, ahead, and turns them into the atoms of its k-blocks among those that
    // share the fetch.
    // A set waits for its own stages only, and a parity wait tells a phase from the one two before it only
    // if that one is known to be over.  It is: the set has seen the stage of the k-block in front of
    // the other's run free, hence (MMAs end in order) all k-blocks up to a ring's length before that
    // one done; the phase in question is two ring lengths back, no later than that while a
    // run is shorter than the ring.
    constexpr int kRun = kUnitsPerChunk / 2;
    const int set = (warp - 2) >> 2;
    const int r = ((warp - 2) & 3) * 32 + lane;
    const uint32_t slot_off = static_cast<uint32_t>((r & 31) * 16 + (r >> 5) * 4);
    const uint32_t kStagingSlot = static_cast<uint32_t>(kTiles * kTileM + BN) * 16u, x_slot = kTiles * kTileM * 16u;
    const uint32_t stage_w = staging_base + static_cast<uint32_t>(r) * 16u + static_cast<uint32_t>(set * kFetchAhead) * kStagingSlot;
    // (BN need not reach 128 or 256: threads beyond it have no slot)
    const bool slot0 = r < BN, slot1 = r + 128 < BN;
    const bool aligned = p.align_w == 16 && p.align_x == 16;
    int f_it = 0, f_kb = 0;
    const uint8_t *f_w[kTiles], *f_x0 = nullptr, *f_x1 = nullptr;  // rows of the item being fetched, or null
    int next0 = x_pair(0, r), next1 = slot1 ? x_pair(0, r + 128) : -1;  // of the item entered next
    auto enter = [&]() {  // the item at the fetch cursor
      f_x0 = f_x1 = nullptr;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) f_w[t] = nullptr;
      if (f_it >= n_items) return;
      const GroupedItem item = item_at(f_it);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        int col, row;
        if constexpr (kTwo) {
          col = item.tile * kTileCols + (kGated ? 0 : t * kTileM) + r;
          row = col + (kGated && t == 1 ? p.n : 0);
        } else if constexpr (kGated) {
          col = item.tile * kTileCols + (r >> 5) * 16 + (r & 15);
          row = col + ((r & 16) ? p.n : 0);
        } else {
          col = row = item.tile * kTileCols + r;
        }
        if (col < p.n) f_w[t] = p.sw + (static_cast<int64_t>(item.group) * p.b_group_rows + row) * p.ld_sw;
      }
      const int a0 = x_row(next0), a1 = x_row(next1);
      if (a0 >= 0) f_x0 = p.sx + a0 * p.ld_sx;
      if (a1 >= 0) f_x1 = p.sx + a1 * p.ld_sx;
      next0 = x_pair(f_it + 1, r);
      if (slot1) next1 = x_pair(f_it + 1, r + 128);
    };
    auto fetch = [&](int slot) {
      if (f_it < n_items) {
        const int col = (f_kb * kSfBytes) & ~15;
        const int valid = min(16, p.kblocks32 - col);
        const uint32_t dst = stage_w + slot * kStagingSlot;
        if (aligned) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + t * kTileM * 16u),
                         "l"(f_w[t] != nullptr ? f_w[t] + col : p.sw), "r"(f_w[t] != nullptr ? valid : 0)
                         : "memory");
          if (slot0)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + x_slot),
                         "l"(f_x0 != nullptr ? f_x0 + col : p.sx), "r"(f_x0 != nullptr ? valid : 0)
                         : "memory");
          if (slot1)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + x_slot + kTileM * 16u),
                         "l"(f_x1 != nullptr ? f_x1 + col : p.sx), "r"(f_x1 != nullptr ? valid : 0)
                         : "memory");
        } else {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            fetch_scales(dst + t * kTileM * 16u, f_w[t] != nullptr ? f_w[t] + col : p.sw, f_w[t] != nullptr ? valid : 0, p.align_w);
          if (slot0) fetch_scales(dst + x_slot, f_x0 != nullptr ? f_x0 + col : p.sx, f_x0 != nullptr ? valid : 0, p.align_x);
          if (slot1)
            fetch_scales(dst + x_slot + kTileM * 16u, f_x1 != nullptr ? f_x1 + col : p.sx, f_x1 != nullptr ? valid : 0, p.align_x);
        }
        f_kb += kUnitsPerChunk;
        if (f_kb >= p.k_blocks) {
          f_kb = 0;
          ++f_it;
          enter();
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");  // always: the group count stays in step
    };
    enter();
    for (int j = 0; j < kFetchAhead; ++j) fetch(j);
    int s = 0, kb = 0, c_slot = 0, run = 0;  // run: k-blocks so far, modulo two runs
    uint32_t ph = 0;
    bool alive = true;
    for (int it = 0; it < n_items && alive;) {
      const int in_chunk = min(kUnitsPerChunk, p.k_blocks - kb);
      asm volatile("cp.async.wait_group %0;" ::"n"(kFetchAhead - 1) : "memory");
      uint4 cw[kTiles], cx0 = make_uint4(0, 0, 0, 0), cx1 = make_uint4(0, 0, 0, 0);
      const uint32_t from = stage_w + c_slot * kStagingSlot;
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(cw[t].x), "=r"(cw[t].y), "=r"(cw[t].z), "=r"(cw[t].w)
                     : "r"(from + t * kTileM * 16u));
      if (slot0)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(cx0.x), "=r"(cx0.y), "=r"(cx0.z), "=r"(cx0.w)
                     : "r"(from + x_slot));
      if (slot1)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(cx1.x), "=r"(cx1.y), "=r"(cx1.z), "=r"(cx1.w)
                     : "r"(from + x_slot + kTileM * 16u));
      if (in_chunk == kUnitsPerChunk && run == 0) {
        // the usual case, a whole chunk of two whole runs, without the bookkeeping of the general one below
        int s1 = s;
        uint32_t ph1 = ph;
        if (set == 1) {
          s1 += kRun;
          if (s1 >= stages) { s1 -= stages; ph1 ^= 1u; }
        }
        const int first_s = s1;
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
          if (!__all_sync(kAll, mbar_wait_bounded(empty_bar(s1), ph1 ^ 1u, abort_flag, budget_ns))) alive = false;
          if (!alive) break;
          const uint32_t aw = atom_base + s1 * atom_bytes + slot_off, ax = aw + kTiles * kKa * 512u;
#pragma unroll
          for (int a = 0; a < kKa; ++a) {
            const int lo = u * kKa + a, hi = lo + kRun * kKa;  // this set's word: one of two
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(aw + 512u * (t * kKa + a)),
                           "r"(set == 0 ? pick_word(cw[t], lo) : pick_word(cw[t], hi))
                           : "memory");
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(ax + 512u * (a * x_halves)),
                         "r"(set == 0 ? pick_word(cx0, lo) : pick_word(cx0, hi))
                         : "memory");
            if (x_halves == 2)
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(ax + 512u * (a * 2 + 1)),
                           "r"(set == 0 ? pick_word(cx1, lo) : pick_word(cx1, hi))
                           : "memory");
          }
          if (++s1 == stages) { s1 = 0; ph1 ^= 1u; }
        }
        if (!alive) {
          if (lane == 0) {
            leave_error(p.error, kErrProducerWait);
            *abort_flag = 1;
          }
          break;
        }
        fence_proxy_async_shared_cta();
        __syncwarp();
        if (lane < kRun) {
          const int mine = first_s + lane;
          mbar_arrive(full_bar(mine >= stages ? mine - stages : mine));
        }
        s += kUnitsPerChunk;
        while (s >= stages) { s -= stages; ph ^= 1u; }
        fetch(c_slot);
        if (++c_slot == kFetchAhead) c_slot = 0;
        kb += kUnitsPerChunk;
        if (kb == p.k_blocks) {
          kb = 0;
          ++it;
        }
        continue;
      }
      int first_s = s, pending = 0;  // stages written and not yet handed over
      for (int u = 0; u < in_chunk; ++u) {
        if (run / kRun == set) {
          // the stage's previous atoms have been copied to tensor memory (its MMAs are done)
          if (!__all_sync(kAll, mbar_wait_bounded(empty_bar(s), ph ^ 1u, abort_flag, budget_ns))) {
            if (lane == 0) {
              leave_error(p.error, kErrProducerWait);
              *abort_flag = 1;
            }
            alive = false;
            break;
          }
          const int sub = u * kKa;
          const uint32_t aw = atom_base + s * atom_bytes + slot_off, ax = aw + kTiles * kKa * 512u;
#pragma unroll
          for (int a = 0; a < kKa; ++a) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(aw + 512u * (t * kKa + a)), "r"(pick_word(cw[t], sub + a)) : "memory");
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(ax + 512u * (a * x_halves)), "r"(pick_word(cx0, sub + a)) : "memory");
            if (x_halves == 2)
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(ax + 512u * (a * 2 + 1)), "r"(pick_word(cx1, sub + a)) : "memory");
          }
          if (pending++ == 0) first_s = s;
        }
        if (++run == 2 * kRun) run = 0;
        if (++s == stages) { s = 0; ph ^= 1u; }
        // a run (or chunk) has ended: hand its stages over (one proxy fence for all)
        if (pending > 0 && (u + 1 == in_chunk || run / kRun != set)) {
          fence_proxy_async_shared_cta();  // these writes -> visible to tcgen05.cp
          __syncwarp();
          if (lane == 0) {
            for (int j = 0; j < pending; ++j) {
              mbar_arrive(full_bar(first_s));
              if (++first_s == stages) first_s = 0;
            }
          }
          pending = 0;
        }
      }
      if (!alive) break;
      fetch(c_slot);
      if (++c_slot == kFetchAhead) c_slot = 0;
      kb += in_chunk;
      if (kb == p.k_blocks) {
        kb = 0;
        ++it;
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    // -------------------------------- epilogue --------------------------------
    // 16 columns (pairs) at a time.  The item's pairs and weights are put into a list in shared memory before its
    // accumulator is waited for (fetched step by step they took most of the epilogue's time).  kTwo: two
    // warps to a lane quarter; gated they take the steps in turn, else a W tile each.
    const int quarter = warp & 3;  // the TMEM lane quarter this warp can read
    const int half = (warp - kGroupedEpilogueWarp) >> 2;
    constexpr bool kTurns = kTwo && kGated;
    constexpr int kStep = kTurns ? 32 : 16;
    const bool weighted = p.row_weights != nullptr;
    bool alive = true;
    int buf = 0;
    uint32_t acc_ph = 0;
    for (int it = 0; it < n_items; ++it) {
      const GroupedItem item = item_at(it);
      int2* list = lists + (it & 1) * kGroupedMaxBN;
      const uint32_t list_at = smem_u32(list);
      for (int r = static_cast<int>(threadIdx.x) - 32 * kGroupedEpilogueWarp; r < ((item.count + 15) & ~15); r += 128 * kTiles) {
        const int q = pair_at(item, r);
        list[r] = make_int2(q, __float_as_int(weighted && q >= 0 ? p.row_weights[q] : 1.0f));
      }
      // the list is complete (and everyone is done with the one before the last); a warp that gave up
      // waiting takes the others along here, none waits for one that has left
      uint32_t all_alive;
      asm volatile(
          "{\n\t"
          ".reg .pred p, q;\n\t"
          "setp.ne.b32 p, %1, 0;\n\t"
          "bar.red.and.pred q, 1, %2, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t"
          "}\n"
          : "=r"(all_alive)
          : "r"(alive ? 1u : 0u), "n"(128 * kTiles)
          : "memory");
      if (!all_alive) break;
      const bool got = mbar_wait_bounded(acc_full_bar(buf), acc_ph, abort_flag, budget_ns);
      if (!__all_sync(kAll, got)) {
        if (lane == 0) {
          leave_error(p.error, kErrEpilogueWait);
          *abort_flag = 1;
        }
        alive = false;
        continue;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(buf * acc_cols + (kTwo && !kGated ? half * BN : 0));
      int col = item.tile * kTileCols;
      if constexpr (kTwo) col += (kGated ? 0 : half * kTileM) + quarter * 32 + lane;
      else col += kGated ? quarter * 16 + (lane & 15) : quarter * 32 + lane;
      float* const d_col = p.d + col;
      const bool in = col < p.n;
      for (int c = kTurns ? 16 * half : 0; c < item.count; c += kStep) {
        uint32_t acc[16];
        tmem_ld_32x16(taddr + static_cast<uint32_t>(c), acc);
        if constexpr (kTurns) {
          uint32_t up[16];
          tmem_ld_32x16(taddr + static_cast<uint32_t>(BN + c), up);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[j] = __float_as_uint(silu_f32(__uint_as_float(acc[j])) * __uint_as_float(up[j]));
        } else {
          tmem_ld_wait();
        }
#pragma unroll
        for (int j0 = 0; j0 < 16; j0 += 8) {
          if (c + j0 >= item.count) break;
          // eight pairs and weights, before any store (behind one the compiler would have to load them again)
          int q[8];
          float w[8];
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(q[j]), "=f"(w[j]), "=r"(q[j + 1]), "=f"(w[j + 1])
                         : "r"(list_at + static_cast<uint32_t>(c + j0 + j) * 8u));
#pragma unroll
          for (int j = 0; j < 8; j += kGated && !kTwo ? 2 : 1) {
            float y = __uint_as_float(acc[j0 + j]);
            int to = q[j];
            float weight = w[j];
            if constexpr (kGated && !kTwo) {
              // lanes 0-15 hold the gate, 16-31 the up product: the lower lanes finish the even columns,
              // the upper ones the odd
              const bool upper = lane >= 16;
              const float other = __shfl_xor_sync(kAll, upper ? y : __uint_as_float(acc[j0 + j + 1]), 16);
              const float kept = upper ? __uint_as_float(acc[j0 + j + 1]) : y;
              y = silu_f32(upper ? other : kept) * (upper ? kept : other);
              to = upper ? q[j + 1] : to;
              weight = upper ? w[j + 1] : weight;
            }
            if (weighted) y *= weight;
            if (in && to >= 0) d_col[static_cast<int64_t>(to) * p.ldd] = y;
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty_bar(buf));
      if (++buf == acc_sets) { buf = 0; acc_ph ^= 1u; }
    }
  }

  tc_fence_before_sync();
  __syncwarp();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 512u);
}

// Rows of A (elements, then scales) in plan order: row p of `x` and `sx` belongs to pair order[p].  A warp
// for every place in turn; places without a pair are left as they are.
__global__ void __launch_bounds__(256) gather_rows_kernel(const uint8_t* a, int64_t a_pitch, const uint8_t* sa,
                                                          int64_t sa_pitch, const int32_t* order, int rows, int a_rows,
                                                          int pairs_per_a_row, int row_bytes, int scale_bytes, uint8_t* x,
                                                          int64_t x_pitch, uint8_t* sx, int64_t sx_pitch) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int place = blockIdx.x * 8 + static_cast<int>(threadIdx.x >> 5); place < rows; place += static_cast<int>(gridDim.x) * 8) {
    const int lane = threadIdx.x & 31;
    const int q = order[place];
    if (q < 0 || q >= rows) continue;
    const int64_t row = min(q / pairs_per_a_row, a_rows - 1);
    const uint8_t* from = a + row * a_pitch;
    uint8_t* to = x + place * x_pitch;
    int i = lane * 16;
    for (; i + 1552 <= row_bytes; i += 2048) {  // four pieces on their way at a time
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(from + i + 512 * j);
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(to + i + 512 * j) = v[j];
    }
    for (; i + 16 <= row_bytes; i += 512) *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(from + i);
    for (int j = (row_bytes & ~15) + lane; j < row_bytes; j += 32) to[j] = from[j];
    const uint8_t* sfrom = sa + row * sa_pitch;
    uint8_t* sto = sx + place * sx_pitch;
    for (int j = lane; j < scale_bytes; j += 32) sto[j] = sfrom[j];
  }
}

// Zeros in the rows of D whose only pair is in no group.  A warp for every row in turn.
__global__ void __launch_bounds__(256) zero_rows_kernel(const int32_t* ids, int groups, int rows, int n, float* d, int64_t ldd) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t row = blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8) {
    const int id = ids[row];
    if (id >= 0 && id < groups) continue;
    for (int64_t col = threadIdx.x & 31; col < n; col += 32) d[row * ldd + col] = 0.0f;
  }
}

// D[t] = the sum of row t's `per` pairs, ascending; pairs in no group add nothing.
__global__ void __launch_bounds__(256) sum_pairs_kernel(const float* pairs, const int32_t* ids, int groups, int per,
                                                        int64_t rows, int n, float* d, int64_t ldd) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t t = blockIdx.y; t < rows; t += gridDim.y) {
    for (int col = blockIdx.x * 256 + threadIdx.x; col < n; col += gridDim.x * 256) {
      float sum = 0.0f;
      for (int s = 0; s < per; ++s) {
        const int64_t q = t * per + s;
        const int id = ids[q];
        if (id >= 0 && id < groups) sum += pairs[q * n + col];
      }
      d[t * ldd + col] = sum;
    }
  }
}

}  // namespace b200
