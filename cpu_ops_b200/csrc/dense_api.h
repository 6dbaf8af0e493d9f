// Entry points of the 16-bit products, their epilogue's gradient, layer norm and the balance loss.
// Included by api.cu only, after row_chosen_api.h, whose call plumbing they share.
#pragma once

#include "dense_kernels.h"
#include "row_chosen_api.h"

namespace {

static_assert(int{kF32} == CPUOPS_B200_TYPE_F32 && int{kF16} == CPUOPS_B200_TYPE_F16 && int{kBf16} == CPUOPS_B200_TYPE_BF16,
              "kernels and header agree on the types");
constexpr int kDenseMost = 1 << 30;  // of m, n, k: sums of an extent and a tile stay within 31 bits

bool activation_ok(int act) {
  return act == 0 || act == CPUOPS_B200_OP_RELU || act == CPUOPS_B200_OP_GELU || act == CPUOPS_B200_OP_SILU;
}
int kernel_activation(int act) {
  return act == CPUOPS_B200_OP_RELU ? kOpRelu : act == CPUOPS_B200_OP_GELU ? kOpGelu : act == CPUOPS_B200_OP_SILU ? kOpSilu : 0;
}
bool rows_aligned(const void* base, int64_t ld, int type) {
  return ((reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(ld * type_bytes(type))) & 15u) == 0;
}

// ---- 16-bit products -----------------------------------------------------------------------

// 2-D tensor of 16- or 32-bit elements; boxes of box0 x box1, swizzled by their row's 64 or 128 bytes.
int make_tensor_map_elements(CUtensorMap* tm, const void* base, int type, uint64_t inner, uint64_t outer, uint64_t pitch,
                             uint32_t box0, uint32_t box1) {
  const uint32_t size = static_cast<uint32_t>(type_bytes(type));
  if (outer <= 1) pitch = (inner * size + 15) / 16 * 16;
  const TensorMapKey key{reinterpret_cast<uint64_t>(base), inner, outer, pitch, box1, 16u + box0 * size * 2u + (size >> 2)};
  TensorMapSlot& slot = tensor_map_slot(key);
  if (slot.valid && slot.key == key) {
    *tm = slot.map;
    return 0;
  }
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {pitch};
  const cuuint32_t box[2] = {box0, box1};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_encode(tm, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
                              const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              box0 * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed with %d (base %p inner %llu outer %llu pitch %llu box %u x %u)",
              static_cast<int>(r), base, (unsigned long long)inner, (unsigned long long)outer, (unsigned long long)pitch, box0, box1);
    return CPUOPS_B200_STATUS_CUDA_ERROR;
  }
  slot.valid = true;
  slot.key = key;
  slot.map = *tm;
  return 0;
}

// Clusters of each form that fit the device at once, by form and cluster size (0: not asked yet, else one more).
int g_product_clusters[64][3][kProductMaxParts + 1];
int product_clusters(DeviceState& st, int form, int size) {
  int& known = g_product_clusters[st.device][form][size];
  if (known == 0) {
    cudaLaunchConfig_t probe = {};
    probe.gridDim = dim3(static_cast<unsigned>(st.sm_count / size * size));
    probe.blockDim = dim3(static_cast<unsigned>(product_threads(form, kProductEpiWarps)));
    probe.dynamicSmemBytes = static_cast<size_t>(st.smem_optin);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(size);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    probe.attrs = attr;
    probe.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, product_kernel_of(form, true, true), &probe) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    known = n + 1;
  }
  return known - 1;
}

struct ProductChoice {
  int form = kProductTiles, BN = 128, parts = 1, stages = 0, epi_warps = kProductEpiWarps, ring_bytes = 0, ring_depth = 1;
  int tile_rows = 128;
  bool swapped = false, pieces = false;
};

// Shared memory of a choice: stages, epilogue warps and their buffers.  `chunks`: bytes of one chunk each of C, D and
// Z (0: not by TMA); `rows`: an epilogue warp's otherwise.  False: it does not fit.
bool fit_product(ProductChoice& c, int smem_optin, int chunks, int rows, int k_blocks) {
  const int room = smem_optin - 1024 - kProductBarrierBytes - 4 * kProductBiasFloats;
  const int stage = (kTileM + c.BN / (c.form == kProductPairs ? 2 : 1)) * 128;
  if (c.form == kProductParts) {
    c.epi_warps = 4;  // (together: the sums of an owner's columns from all parts)
    c.ring_bytes = c.BN * kTileM;
    c.stages = (room - 4 * c.ring_bytes) / stage;
  } else {
    // Eight epilogue warps with two buffers for each matrix, unless that leaves the ring of stages short: then one
    // buffer, or four warps (which do not have the registers for the pieces' sums).
    for (int attempt = 0; attempt < 3; ++attempt) {
      c.epi_warps = attempt < 2 || c.pieces ? 8 : 4;
      c.ring_depth = attempt == 0 ? 2 : 1;
      c.ring_bytes = chunks ? c.ring_depth * chunks : rows;
      c.stages = (room - c.epi_warps * c.ring_bytes) / stage;
      if (c.stages >= 5) break;
    }
  }
  c.stages = std::min({c.stages, kProductMaxStages, std::max(2, (k_blocks + c.parts - 1) / c.parts)});
  return c.stages >= 2;
}

// Estimated time in us; the choice whose is least is taken.  Measured on B200 at K = 1024 .. 8192 (a k-block of one tile,
// rounds of tiles, and what does not shrink with k); us, estimated / measured:
//   512 x 2048 x 1024: tiles of 64 6.5 / 6.3, of 128 9.2 / 7.4, pairs of 128 9.2 / 7.3, of 256 14.5 / 11.2, two parts 11.7 / 11.4
//   256 x 4096 x 4096: tiles of 64 16.6 / 16.3, pairs of 128 20.7 / 18.1, two parts of 128 19.1 / 20.4
//   4096 x 4096 x 4096: pairs of 256 100 / 94, of 192 102 / 95, of 128 106 / 100, tiles of 128 125 / 115
// chunk_us: an epilogue warp's time for 32 x 32 elements; hbm_us: the bytes that the call cannot do without.
double product_us(const ProductChoice& c, const DeviceState& st, int Mk, int Nk, int k_blocks, int piece_blocks, double chunk_us, double hbm_us) {
  const bool pair = c.form == kProductPairs;
  const int tile_m = pair ? 256 : c.tile_rows;
  const int64_t tiles = static_cast<int64_t>((Mk + tile_m - 1) / tile_m) * ((Nk + c.BN - 1) / c.BN);
  const int64_t slots = std::max(1, c.form == kProductTiles ? st.sms() : st.sms() / (pair ? 2 : c.parts));
  const double rounds = static_cast<double>((tiles + slots - 1) / slots);
  double block = pair ? (c.BN == 128 ? 0.215 : c.BN == 192 ? 0.285 : 0.345)
                      : (c.BN <= 16 ? 0.13 : c.BN == 32 ? 0.145 : c.BN == 64 ? 0.185 : c.BN == 128 ? 0.26 : 0.45);
  if (c.pieces) block += 0.4 / piece_blocks;
  const double kb = static_cast<double>((k_blocks + c.parts - 1) / c.parts);
  // (a short loop does not reach the memory's rate from its first load on)
  auto together = [&](double us) { return std::max(hbm_us, us) + 0.25 * std::min(hbm_us, us); };
  if (c.form == kProductParts) {
    const int own = c.BN / c.parts, items = own >= 8 ? (4 * own / 8 + 6) / 7 : 1;
    const double tail = 0.6 * items + (c.parts > 1 ? 1.6 + 0.011 * c.BN : 0.0);
    return together(rounds * kb * block + (rounds - 1.0) * 3.0) + 3.3 + rounds * tail;
  }
  const double epilogue = 0.6 + (c.BN + 63) / 64 * chunk_us * (c.epi_warps == 8 ? 1.0 : 1.6) * (pair ? 1.0 : 1.1);
  return together(rounds * std::max(kb * block, epilogue)) + 1.2 + epilogue + (pair ? 1.0 : 0.0);
}

int dense_kernels_ready(DeviceState& st) {
  static bool ready[64] = {};
  if (ready[st.device]) return 0;
  for (int form : {kProductTiles, kProductPairs, kProductParts})
    for (bool pieces : {false, true})
      for (bool tma : {false, true})
        CUDA_TRY(cudaFuncSetAttribute(product_kernel_of(form, pieces, tma), cudaFuncAttributeMaxDynamicSharedMemorySize, st.smem_optin));
  for (int x : {kF32, kF16, kBf16})
    for (int y : {kF32, kF16, kBf16})
      for (bool gradient : {false, true}) {
        if (x != y && x != kF32) continue;
        for (int n : {1024, 2048, 4096, 8192}) {  // (those with shared memory)
          const NormChoice c = norm_choice(x, y, n, true, true, true, gradient);
          CUDA_TRY(cudaFuncSetAttribute(c.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormMostSmem));
        }
      }
  ready[st.device] = true;
  return 0;
}

int gemm16_call(const cpuops_b200_gemm16_desc* d) {
  if (int rc = check_desc(d)) return rc;
  if (!type_ok(d->type) || !type_ok(d->c_type) || !type_ok(d->d_type) || !activation_ok(d->activation)) {
    set_error("gemm16: unknown element type or activation");
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  if (d->type == kF32 || (d->d_type != kF32 && d->d_type != d->type) || (d->c_type != kF32 && d->c_type != d->type)) {
    set_error("gemm16: A and B are f16 or bf16, C and D f32 or of their type");
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  if (d->m < 0 || d->n < 0 || d->k < 0) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (d->m == 0 || d->n == 0) return CPUOPS_B200_STATUS_SUCCESS;
  if (d->m > kDenseMost || d->n > kDenseMost || d->k > kDenseMost) return refuse("gemm16: m, n and k are at most 2^30");
  const bool use_c = d->beta != 0.0f;  // (a NaN is used)
  if (!d->d || (use_c && !d->c) || (d->k > 0 && (!d->a || !d->b))) return refuse("gemm16: a buffer is missing");
  if (d->ldd < d->n || (use_c && d->ldc < d->n) || (d->z && d->ldz < d->n) ||
      (d->k > 0 && (d->lda < (d->a_row_major ? d->k : d->m) || d->ldb < (d->b_row_major ? d->n : d->k))))
    return refuse("gemm16: a leading dimension is too small");
  if (use_c && d->c == d->d && (d->ldc != d->ldd || d->c_type != d->d_type))
    return refuse("gemm16: in place, C and D have the same leading dimension and type");
  if (d->z && (d->z == d->d || (use_c && d->z == d->c))) return refuse("gemm16: Z is a buffer of its own");
  if (d->split_k_slices < 0 || d->split_k_slices > kProductMaxParts || (d->split_k_slices & (d->split_k_slices - 1)) != 0 ||
      d->tile_n < 0 || d->tile_n > 256 || d->tile_n % 16 != 0)
    return refuse("gemm16: split_k_slices is 0, 1, 2, 4 or 8, tile_n 0 or a multiple of 16 up to 256");
  // 2-byte (f32: 4-byte) elements, whole
  const auto off = [](const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) != 0; };
  if (off(d->a, d->type) || off(d->b, d->type) || (use_c && off(d->c, d->c_type)) || off(d->d, d->d_type) ||
      off(d->z, d->d_type) || off(d->bias, kF32))
    return refuse("gemm16: a buffer is not aligned to its elements");
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->a, d->b, d->bias, use_c ? d->c : nullptr, d->d, d->z})) return rc;
  DeviceState& st = *call.st;
  if (int rc = dense_kernels_ready(st)) return rc;

  ProductParams p;
  memset(&p, 0, sizeof(p));
  p.act = kernel_activation(d->activation);
  p.alpha = d->alpha;
  p.beta = d->beta;
  p.bias = d->bias;
  p.C = use_c ? d->c : nullptr;
  p.D = d->d;
  p.Z = d->z;
  p.ldc = d->ldc;
  p.ldd = d->ldd;
  p.ldz = d->ldz;
  p.type = d->type;
  p.c_type = d->c_type;
  p.d_type = d->d_type;
  p.error = st.error_dev;
  p.wait_budget_us = g_wait_budget_us.load();
  if (d->k == 0) {
    p.Mk = d->m;
    p.Nk = d->n;
    const int64_t blocks = (static_cast<int64_t>(d->m) * d->n + 255) / 256;
    if (int rc = launch_after(product_empty(), dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 16 * st.sms()))), 256, 0,
                              call.stream, p))
      return rc;
    return call.finish();
  }
  const int k_blocks = (d->k + 63) / 64;
  p.k_blocks = k_blocks;
  // Storage of the operands: rows of `inner` contiguous elements.
  struct Side {
    const void* base;
    int64_t ld;
    int inner, outer, mn;  // mn: the contiguous direction is m (n)
  };
  Side a{d->a, d->lda, d->a_row_major ? d->k : d->m, d->a_row_major ? d->m : d->k, d->a_row_major ? 0 : 1};
  Side b{d->b, d->ldb, d->b_row_major ? d->n : d->k, d->b_row_major ? d->k : d->n, d->b_row_major ? 1 : 0};
  const auto tma_rows = [](const void* base, int64_t ld, int type) { return rows_aligned(base, ld, type); };
  const bool by_tma = tma_rows(d->d, d->ldd, d->d_type) && (!use_c || tma_rows(d->c, d->ldc, d->c_type)) &&
                      (!d->z || tma_rows(d->z, d->ldz, d->d_type));
  const int chunks = by_tma ? chunk_bytes(d->d_type) * (d->z ? 2 : 1) + (use_c ? chunk_bytes(d->c_type) : 0) : 0;
  // Pieces of k: an f32 D shows what the tensor cores drop of a running sum from k = 512 on; a 16-bit one where it comes
  // near half of the rounding's half step (product_kernel.cuh), which sums of 16384 (f16) or 131072 elements (bf16) stay
  // below.  Their pieces are longer, so that they cost little: 256 x 256 x 65536 f16 by tiles of 128 in one running sum 205 us
  // (4.3e-4 of the result dropped), in pieces of 8192 215 (4.9e-5), an f32 D's of 512 240.
  const bool f32_d = d->d_type == kF32;
  const int piece_blocks = f32_d ? kProductPieceBlocks : kProductPieceBlocks16;
  const int running = d->type == kF16 ? kProductRunningBlocksF16 : kProductRunningBlocksBf16;

  // The choice of form and tile.
  const double c_size = use_c ? type_bytes(d->c_type) : 0, d_size = type_bytes(d->d_type) * (d->z ? 2 : 1);
  const double hbm_us = (2.0 * d->k * (static_cast<double>(d->m) + d->n) + static_cast<double>(d->m) * d->n * (c_size + d_size)) / 6.4e6;
  const double chunk_us = 1.15 + (d->activation > CPUOPS_B200_OP_RELU ? 0.5 : 0.0) + 0.1 * (d_size + c_size) * (by_tma ? 1.0 : 4.0);
  ProductChoice best;
  double least = 0.0;
  bool found = false;
  auto consider = [&](int form, int BN, int parts, bool swapped) {
    ProductChoice c;
    c.form = form;
    c.BN = BN;
    c.parts = parts;
    c.swapped = swapped;
    c.pieces = f32_d ? k_blocks > piece_blocks : (k_blocks + parts - 1) / parts > running;
    const int b_mn = swapped ? a.mn : b.mn, rows = BN / (form == kProductPairs ? 2 : 1);
    if (b_mn && rows % 64 != 0) return;  // (boxes of 64)
    if (parts > k_blocks) return;
    if (d->tile_n && d->tile_n != BN) return;
    if (d->split_k_slices && (d->split_k_slices > 1 || form == kProductParts) && !(form == kProductParts && parts == d->split_k_slices)) return;
    if ((d->flags & CPUOPS_B200_FLAG_PAIR_ON) && form != kProductPairs) return;
    if ((d->flags & CPUOPS_B200_FLAG_PAIR_OFF) && form == kProductPairs) return;
    if (form != kProductTiles && product_clusters(st, form, form == kProductPairs ? 2 : parts) < 1) return;
    if (!fit_product(c, st.smem_optin, chunks, use_c && d->c_type == kF32 ? 2 * 4096 : 4096, k_blocks)) return;
    const int Mk = swapped ? d->n : d->m, Nk = swapped ? d->m : d->n;
    if (form == kProductParts && !(swapped ? b.mn : a.mn)) {
      // Tiles of fewer rows where that gives every cluster one (a tile's other rows are neither loaded nor used):
      // 8 x 14336 x 4096 as 138 tiles of 104 rows instead of 112 of 128.
      const int64_t columns = (Nk + BN - 1) / BN, clusters = std::max<int64_t>(1, std::min(product_clusters(st, form, parts), st.sms() / parts));
      const int64_t tiles = (Mk + 127) / 128 * columns, rounds = (tiles + clusters - 1) / clusters;
      const int64_t along_m = std::max<int64_t>(1, rounds * clusters / columns);
      c.tile_rows = static_cast<int>(std::min<int64_t>(128, ((Mk + along_m - 1) / along_m + 7) / 8 * 8));
    }
    // (parts are launched all at once: a limit on the SMs is kept by the other forms)
    if (form == kProductParts && st.sms() < st.sm_count &&
        static_cast<int64_t>((Mk + c.tile_rows - 1) / c.tile_rows) * ((Nk + BN - 1) / BN) * parts > st.sms())
      return;
    const double us = product_us(c, st, Mk, Nk, k_blocks, piece_blocks, chunk_us, hbm_us);
    if (!found || us < least) {
      best = c;
      least = us;
      found = true;
    }
  };
  for (int BN : {32, 64, 128, 256}) consider(kProductTiles, BN, 1, false);
  for (int BN : {128, 192, 256}) consider(kProductPairs, BN, 1, false);
  for (int parts : {1, 2, 4, 8}) {
    for (int BN : {16, 32, 64, 128}) {
      if (BN < parts) continue;
      if (d->m <= 128) consider(kProductParts, BN, parts, true);
      if (parts > 1) consider(kProductParts, BN, parts, false);  // (one part of rows: kProductTiles)
    }
  }
  if (!found) return refuse("gemm16: no kernel has the tile, the slices and the pair form that this call forces");
  const ProductChoice& c = best;

  // Operands that TMA cannot address are copied into aligned rows first.
  Plan plan;
  size_t off_copy[2] = {0, 0};
  RepackJob jobs[2] = {};
  int n_jobs = 0;
  Side* sides[2] = {&a, &b};
  for (int i = 0; i < 2; ++i) {
    Side& s = *sides[i];
    if (tma_addressable(s.base, s.ld * 2, s.outer)) continue;
    if (s.inner > INT32_MAX / 2 - 16) return refuse("gemm16: rows longer than 2^30 bytes need 16-byte aligned operands");
    const int64_t pitch = (static_cast<int64_t>(s.inner) * 2 + 127) / 128 * 128;  // (a box's row is one line then)
    off_copy[n_jobs] = plan.take(static_cast<size_t>(pitch) * s.outer);
    RepackJob& j = jobs[n_jobs++];
    j.src = static_cast<const uint8_t*>(s.base);
    j.src_pitch = s.ld * 2;
    j.dst_pitch = pitch;
    j.rows = s.outer;
    j.row_bytes = s.inner * 2;
  }
  if (n_jobs > 0) {
    uint8_t* ws = nullptr;
    if (int rc = ensure_workspace(st, call.stream, plan.total, &ws)) return rc;
    for (int i = 0; i < n_jobs; ++i) jobs[i].dst = ws + off_copy[i];
    if (int rc = launch_repack(jobs[0], jobs[1], call.stream)) return rc;
    for (int i = 0, j = 0; i < 2; ++i) {
      Side& s = *sides[i];
      if (tma_addressable(s.base, s.ld * 2, s.outer)) continue;
      s.base = jobs[j].dst;
      s.ld = jobs[j].dst_pitch / 2;
      ++j;
    }
  }

  const Side& ka = c.swapped ? b : a;
  const Side& kb = c.swapped ? a : b;
  const int ctas = c.form == kProductPairs ? 2 : 1, b_rows = c.BN / ctas, tile_m = 128 * ctas;
  p.swapped = c.swapped ? 1 : 0;
  p.Mk = c.swapped ? d->n : d->m;
  p.Nk = c.swapped ? d->m : d->n;
  const int tile_rows = c.form == kProductParts ? c.tile_rows : tile_m;
  p.tile_rows = tile_rows;
  p.m_tiles = (p.Mk + tile_rows - 1) / tile_rows;
  p.n_tiles = (p.Nk + c.BN - 1) / c.BN;
  p.BN = c.BN;
  p.stages = c.stages;
  p.nacc = 2;
  p.parts = c.parts;
  p.piece_blocks = piece_blocks;
  p.a_mn = ka.mn;
  p.b_mn = kb.mn;
  p.epi_warps = c.epi_warps;
  p.ring_bytes = c.ring_bytes;
  p.ring_depth = c.ring_depth;
  const uint32_t fmt = d->type == kBf16 ? 1u : 0u;
  p.idesc = make_idesc(1 /*f32*/, fmt, fmt, static_cast<uint32_t>(ka.mn), static_cast<uint32_t>(kb.mn), tile_m, c.BN);
  const int64_t total_tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  if (total_tiles * c.parts > INT32_MAX) return refuse("gemm16: too many tiles");
  // (walked so that the tiles in flight share bands of both operands of about the same size)
  const int at_once = std::max(1, st.sms() / (ctas * c.parts));
  p.raster_m = std::max(1, std::min(p.m_tiles, static_cast<int>(std::lround(std::sqrt(static_cast<double>(at_once) * c.BN / tile_m)))));

  CUtensorMap tmA, tmB, tmC, tmD, tmZ;
  if (int rc = make_tensor_map_elements(&tmA, ka.base, d->type, ka.inner, ka.outer, ka.ld * 2, 64, ka.mn ? 64 : std::min(tile_rows, 128))) return rc;
  if (int rc = make_tensor_map_elements(&tmB, kb.base, d->type, kb.inner, kb.outer, kb.ld * 2, 64, kb.mn ? 64 : b_rows)) return rc;
  tmC = tmD = tmZ = tmA;
  if (by_tma && c.form != kProductParts) {
    if (int rc = make_tensor_map_elements(&tmD, d->d, d->d_type, d->n, d->m, static_cast<uint64_t>(d->ldd) * type_bytes(d->d_type), 32, 32)) return rc;
    if (use_c)
      if (int rc = make_tensor_map_elements(&tmC, d->c, d->c_type, d->n, d->m, static_cast<uint64_t>(d->ldc) * type_bytes(d->c_type), 32, 32)) return rc;
    if (d->z)
      if (int rc = make_tensor_map_elements(&tmZ, d->z, d->d_type, d->n, d->m, static_cast<uint64_t>(d->ldz) * type_bytes(d->d_type), 32, 32)) return rc;
  }
  const int stage_bytes = (kTileM + b_rows) * 128;
  // At least 120 KB so that two CTAs never share an SM: each allocates all of tensor memory.
  const int smem = std::max(1024 + c.stages * stage_bytes + c.epi_warps * c.ring_bytes + kProductBarrierBytes + 4 * kProductBiasFloats, 120 * 1024);
  cudaLaunchConfig_t cfg = {};
  int64_t grid = std::min<int64_t>(total_tiles, st.sms());
  if (c.form == kProductPairs)
    grid = 2 * std::min<int64_t>({total_tiles, product_clusters(st, c.form, 2), std::max(1, st.sms() / 2)});
  if (c.form == kProductParts) grid = total_tiles * c.parts;
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(product_threads(c.form, c.epi_warps)));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = call.stream;
  cudaLaunchAttribute attr[2];
  int n_attr = 0;
  attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n_attr++].val.programmaticStreamSerializationAllowed = 1;
  if (c.form != kProductTiles) {
    attr[n_attr].id = cudaLaunchAttributeClusterDimension;
    attr[n_attr].val.clusterDim.x = static_cast<unsigned>(c.form == kProductPairs ? 2 : c.parts);
    attr[n_attr].val.clusterDim.y = attr[n_attr].val.clusterDim.z = 1;
    ++n_attr;
  }
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(n_attr);
  g_last_plan = cpuops_b200_plan{};
  g_last_plan.swapped = p.swapped;
  g_last_plan.tile_n = c.BN;
  g_last_plan.pair = c.form == kProductPairs ? 1 : 0;
  g_last_plan.slices = c.parts;
  g_last_plan.stages = c.stages;
  g_last_plan.grid = static_cast<int32_t>(grid);
  g_last_plan.c_ring = by_tma && use_c && c.form != kProductParts ? 1 : 0;
  g_last_plan.epilogue_warps = c.epi_warps;
  CUDA_TRY(cudaLaunchKernelEx(&cfg, product_kernel_of(c.form, c.pieces, by_tma), tmA, tmB, tmC, tmD, tmZ, p));
  g_launches.fetch_add(1);
  return call.finish();
}

// ---- columns' sums -------------------------------------------------------------------------

int launch_column_sum(const float* in, float* out0, float* out1, int parts, int n, int count, cudaStream_t stream) {
  ColumnSumParams s{in, out0, out1, parts, n};
  return launch_after(column_sum(), dim3(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>(count)), 32 * std::min(32, parts), 0, stream, s);
}

// ---- gradient of bias and activation ----------------------------------------------------------

int epilogue_grad_call(const cpuops_b200_epilogue_grad_desc* d) {
  if (int rc = check_desc(d)) return rc;
  if (!type_ok(d->type) || !activation_ok(d->activation)) {
    set_error("epilogue_grad: unknown element type or activation");
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  if (d->m < 0 || d->n < 0) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (d->n == 0 || (d->m == 0 && !d->dbias)) return CPUOPS_B200_STATUS_SUCCESS;
  if (d->m > kDenseMost || d->n > kDenseMost) return refuse("epilogue_grad: m and n are at most 2^30");
  const bool act = d->activation != 0;
  if (d->m > 0) {
    if (!d->dy || (act && !d->z)) return refuse("epilogue_grad: a buffer is missing");
    if (!d->dz && (act || !d->dbias)) return refuse("epilogue_grad: dZ is missing (only without an activation dbias alone can be asked for)");
    if (d->lddy < d->n || (act && d->ldz < d->n) || (d->dz && d->lddz < d->n)) return refuse("epilogue_grad: a leading dimension is too small");
    if (d->dz && ((d->dz == d->dy && d->lddz != d->lddy) || (act && d->dz == d->z && d->lddz != d->ldz)))
      return refuse("epilogue_grad: in place, both have the same leading dimension");
  }
  const auto off = [](const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) != 0; };
  if (off(d->dy, d->type) || (act && off(d->z, d->type)) || off(d->dz, d->type) || off(d->dbias, kF32))
    return refuse("epilogue_grad: a buffer is not aligned to its elements");
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->dy, act ? d->z : nullptr, d->dz, d->dbias})) return rc;
  EpilogueGradParams p;
  memset(&p, 0, sizeof(p));
  p.dy = d->dy;
  p.z = act ? d->z : nullptr;
  p.dz = d->dz;
  p.lddy = d->lddy;
  p.ldz = d->ldz;
  p.lddz = d->lddz;
  p.m = d->m;
  p.n = d->n;
  const bool wide = rows_aligned(d->dy, d->lddy, d->type) && (!act || rows_aligned(d->z, d->ldz, d->type)) &&
                    (!d->dz || rows_aligned(d->dz, d->lddz, d->type));
  // 16-bit rows on odd elements: every second one begins in the middle of a word, and a block takes those or the others.
  p.every = !wide && d->type != kF32 && d->m > 1 && (d->dz ? d->lddz : d->lddy) % 2 != 0 ? 2 : 1;
  // Blocks of rows: enough CTAs for six on every SM, at least 32 rows each.
  const int strips = (d->n + (wide || d->type == kF32 ? 255 : 256)) / 256;
  const int want = std::max(1, 6 * call.st->sms() / strips);
  int block_rows = std::max(32, (d->m + want - 1) / want);
  block_rows = std::max(block_rows, (d->m + 32766) / 32767);
  const int blocks = p.every * std::max(1, (d->m + block_rows * p.every - 1) / (block_rows * p.every));
  p.block_rows = block_rows;
  float* parts = nullptr;
  if (d->dbias && blocks > 1) {
    uint8_t* ws = nullptr;
    if (int rc = ensure_workspace(*call.st, call.stream, static_cast<size_t>(blocks) * d->n * sizeof(float), &ws)) return rc;
    parts = reinterpret_cast<float*>(ws);
  }
  p.sums = d->dbias ? (parts ? parts : d->dbias) : nullptr;
  if (int rc = launch_after(epilogue_grad_of(d->type, kernel_activation(d->activation), wide), dim3(static_cast<unsigned>(strips), static_cast<unsigned>(blocks)), 256, 0,
                            call.stream, p))
    return rc;
  if (parts)
    if (int rc = launch_column_sum(parts, d->dbias, nullptr, blocks, d->n, 1, call.stream)) return rc;
  return call.finish();
}

// ---- layer norm ----------------------------------------------------------------------------

bool norm_types_ok(int x, int y) { return x == y || (x == kF32 && y != kF32); }

int layer_norm_call(const cpuops_b200_layer_norm_desc* d) {
  if (int rc = check_desc(d)) return rc;
  if (!type_ok(d->x_type) || !type_ok(d->y_type)) {
    set_error("layer_norm: unknown element type");
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  if (!norm_types_ok(d->x_type, d->y_type)) {
    set_error("layer_norm: Y is of X's type, or of any type where X is f32");
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  if (d->m < 0 || d->n < 0) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (d->m == 0 || d->n == 0) return CPUOPS_B200_STATUS_SUCCESS;
  if (d->m > kDenseMost || d->n > kDenseMost) return refuse("layer_norm: m and n are at most 2^30");
  if (!(d->eps >= 0.0f)) return refuse("layer_norm: eps is negative or NaN");
  if (!d->x || !d->y) return refuse("layer_norm: a buffer is missing");
  if (d->ldx < d->n || d->ldy < d->n) return refuse("layer_norm: a leading dimension is too small");
  if (d->x == d->y && (d->ldx != d->ldy || d->x_type != d->y_type)) return refuse("layer_norm: in place, X and Y have the same leading dimension and type");
  const auto off = [](const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) != 0; };
  if (off(d->x, d->x_type) || off(d->y, d->y_type) || off(d->gamma, kF32) || off(d->beta, kF32) || off(d->mean, kF32) || off(d->rstd, kF32))
    return refuse("layer_norm: a buffer is not aligned to its elements");
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->x, d->gamma, d->beta, d->y, d->mean, d->rstd})) return rc;
  if (int rc = dense_kernels_ready(*call.st)) return rc;
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = d->x;
  p.gamma = d->gamma;
  p.beta = d->beta;
  p.y = d->y;
  p.mean = d->mean;
  p.rstd = d->rstd;
  p.ldx = d->ldx;
  p.ldy = d->ldy;
  p.m = d->m;
  p.n = d->n;
  p.eps = d->eps;
  const bool wide = rows_aligned(d->x, d->ldx, d->x_type) && rows_aligned(d->y, d->ldy, d->y_type);
  const NormChoice c = norm_choice(d->x_type, d->y_type, d->n, wide, d->m >= 4 * call.st->sms(), false, false);
  const int rows = (d->m + c.rows_at_once - 1) / c.rows_at_once;
  const int grid = std::min(rows, call.st->sms() * (c.ring ? 1 : std::max(1, std::min(16, 1536 / c.threads))));
  p.ring = c.ring;
  p.error = call.st->error_dev;
  p.wait_budget_us = g_wait_budget_us.load();
  if (int rc = launch_after(c.kernel, dim3(static_cast<unsigned>(grid)), c.threads, static_cast<size_t>(c.smem), call.stream, p)) return rc;
  return call.finish();
}

int layer_norm_grad_call(const cpuops_b200_layer_norm_grad_desc* d) {
  if (int rc = check_desc(d)) return rc;
  if (!type_ok(d->x_type) || !type_ok(d->y_type)) {
    set_error("layer_norm_grad: unknown element type");
    return CPUOPS_B200_STATUS_BAD_DESCRIPTOR;
  }
  if (!norm_types_ok(d->x_type, d->y_type)) {
    set_error("layer_norm_grad: dY is of X's type, or of any type where X is f32");
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  if (d->m < 0 || d->n < 0) return CPUOPS_B200_STATUS_INVALID_PROBLEM;
  if (d->n == 0 || (d->m == 0 && !d->dgamma && !d->dbeta)) return CPUOPS_B200_STATUS_SUCCESS;
  if (d->m > kDenseMost || d->n > kDenseMost) return refuse("layer_norm_grad: m and n are at most 2^30");
  if (d->m > 0) {
    if (!d->x || !d->dy || !d->mean || !d->rstd || !d->dx) return refuse("layer_norm_grad: a buffer is missing");
    if (d->ldx < d->n || d->lddy < d->n || d->lddx < d->n || (d->dr && d->lddr < d->n)) return refuse("layer_norm_grad: a leading dimension is too small");
    if ((d->dx == d->x && d->lddx != d->ldx) || (d->dx == d->dy && (d->lddx != d->lddy || d->x_type != d->y_type)) ||
        (d->dr && d->dx == d->dr && d->lddx != d->lddr))
      return refuse("layer_norm_grad: in place, both have the same leading dimension and type");
  }
  const auto off = [](const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) != 0; };
  if (off(d->x, d->x_type) || off(d->dy, d->y_type) || off(d->dr, d->x_type) || off(d->dx, d->x_type) || off(d->gamma, kF32) ||
      off(d->mean, kF32) || off(d->rstd, kF32) || off(d->dgamma, kF32) || off(d->dbeta, kF32))
    return refuse("layer_norm_grad: a buffer is not aligned to its elements");
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->x, d->dy, d->dr, d->gamma, d->mean, d->rstd, d->dx, d->dgamma, d->dbeta})) return rc;
  if (int rc = dense_kernels_ready(*call.st)) return rc;
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = d->x;
  p.dy = d->dy;
  p.dr = d->dr;
  p.gamma = d->gamma;
  p.mean_in = d->mean;
  p.rstd_in = d->rstd;
  p.y = d->dx;
  p.ldx = d->ldx;
  p.lddy = d->lddy;
  p.lddr = d->lddr;
  p.ldy = d->lddx;
  p.m = d->m;
  p.n = d->n;
  const bool wide = rows_aligned(d->x, d->ldx, d->x_type) && rows_aligned(d->dy, d->lddy, d->y_type) &&
                    rows_aligned(d->dx, d->lddx, d->x_type) && (!d->dr || rows_aligned(d->dr, d->lddr, d->x_type));
  const NormChoice c = norm_choice(d->x_type, d->y_type, d->n, wide, d->m >= 4 * call.st->sms(), d->dr != nullptr, true);
  const int rows = std::max(1, (d->m + c.rows_at_once - 1) / c.rows_at_once);
  int grid = std::min(rows, call.st->sms() * std::max(1, std::min(4, 512 / c.threads)));  // (a row of sums each)
  if (c.even && grid > 1) grid &= ~1;
  p.ring = c.ring;
  p.error = call.st->error_dev;
  p.wait_budget_us = g_wait_budget_us.load();
  const bool sums = d->dgamma || d->dbeta, is_long = norm_is_long(d->n);
  int parts = grid, block_rows = 0;
  if (is_long) {
    block_rows = std::max(64, (d->m + 1023) / 1024);
    parts = std::max(1, (d->m + block_rows - 1) / block_rows);
  }
  if (sums) {
    uint8_t* ws = nullptr;
    if (int rc = ensure_workspace(*call.st, call.stream, static_cast<size_t>(2) * parts * d->n * sizeof(float), &ws)) return rc;
    p.sums = reinterpret_cast<float*>(ws);
  }
  // (long rows: the columns first, since dx may take the place of x or dy)
  if (is_long && sums)
    if (int rc = launch_after(norm_grad_columns(d->x_type, d->y_type), dim3(static_cast<unsigned>((d->n + 255) / 256), static_cast<unsigned>(parts)),
                              256, 0, call.stream, p, block_rows))
      return rc;
  if (int rc = launch_after(c.kernel, dim3(static_cast<unsigned>(grid)), c.threads, static_cast<size_t>(c.smem), call.stream, p)) return rc;
  if (sums)
    if (int rc = launch_column_sum(p.sums, d->dgamma, d->dbeta, parts, d->n, 2, call.stream)) return rc;
  return call.finish();
}

// ---- balance loss ------------------------------------------------------------------------------

int balance_loss_call(const cpuops_b200_balance_loss_desc* d) {
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
  if (d->experts > kMaxGroups || d->top_k > kMaxTopK) {
    set_error("balance_loss: %d experts, top_k %d; at most %d and %d are supported", d->experts, d->top_k, kMaxGroups, kMaxTopK);
    return CPUOPS_B200_STATUS_UNSUPPORTED;
  }
  if (static_cast<int64_t>(d->tokens) * d->top_k > INT32_MAX) return refuse("balance_loss: tokens * top_k must fit 31 bits");
  if (d->tokens > 0) {
    if (!d->logits || !d->ids) return refuse("balance_loss: logits or ids missing");
    if (d->ld_logits < d->experts || (d->dlogits && d->ld_dlogits < d->experts)) return refuse("balance_loss: a leading dimension is too small");
    if (d->dlogits == d->logits && d->ld_dlogits != d->ld_logits) return refuse("balance_loss: in place, both have the same leading dimension");
  }
  const auto off = [](const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) != 0; };
  if (off(d->logits, d->logits_type) || off(d->dlogits, d->logits_type) || off(d->ids, kF32) || off(d->counts, kF32) || off(d->loss, kF32) ||
      off(d->upstream, kF32))
    return refuse("balance_loss: a buffer is not aligned to its elements");
  if (!d->counts && !d->loss && !d->dlogits) return CPUOPS_B200_STATUS_SUCCESS;
  RowCall call;
  if (int rc = call.enter(*d)) return rc;
  if (int rc = call.check(d->memory_space, {d->logits, d->ids, d->counts, d->loss, d->dlogits, d->upstream})) return rc;
  BalanceParams p;
  memset(&p, 0, sizeof(p));
  p.logits = d->logits;
  p.ids = d->ids;
  p.dlogits = d->dlogits;
  p.counts = d->counts;
  p.loss = d->loss;
  p.upstream = d->upstream;
  p.ld = d->ld_logits;
  p.ldg = d->ld_dlogits;
  p.tokens = d->tokens;
  p.experts = d->experts;
  p.top_k = d->top_k;
  p.sigmoid = d->scoring == CPUOPS_B200_SCORE_SIGMOID ? 1 : 0;
  p.coefficient = d->coefficient;
  int grid = 1;
  const int warps = balance_warps_of(d->experts);
  if (d->tokens > 32) {
    grid = std::min((d->tokens + warps - 1) / warps, call.st->sms());
    p.count_blocks = std::min(64, (d->tokens + 255) / 256);
    Plan plan;
    const size_t off_ticket = plan.take(sizeof(int32_t));
    const size_t off_counts = plan.take(static_cast<size_t>(p.count_blocks) * (d->experts + 1) * sizeof(int32_t));
    const size_t off_scores = plan.take(static_cast<size_t>(grid) * d->experts * sizeof(float));
    uint8_t* ws = nullptr;
    if (int rc = ensure_workspace(*call.st, call.stream, plan.total, &ws)) return rc;
    p.ticket = reinterpret_cast<int32_t*>(ws + off_ticket);
    p.part_counts = reinterpret_cast<int32_t*>(ws + off_counts);
    p.part_scores = reinterpret_cast<float*>(ws + off_scores);
    if (int rc = launch_after(balance_count(), dim3(static_cast<unsigned>(p.count_blocks)), 256, 0, call.stream, p)) return rc;
  }
  if (int rc = launch_after(balance_of(d->logits_type, d->experts), dim3(static_cast<unsigned>(grid)), 32 * warps, 0, call.stream, p)) return rc;
  return call.finish();
}

}  // namespace

extern "C" {

CPUOPS_B200_API int cpuops_b200_gemm16(const cpuops_b200_gemm16_desc* d) { return gemm16_call(d); }
CPUOPS_B200_API int cpuops_b200_epilogue_grad(const cpuops_b200_epilogue_grad_desc* d) { return epilogue_grad_call(d); }
CPUOPS_B200_API int cpuops_b200_layer_norm(const cpuops_b200_layer_norm_desc* d) { return layer_norm_call(d); }
CPUOPS_B200_API int cpuops_b200_layer_norm_grad(const cpuops_b200_layer_norm_grad_desc* d) { return layer_norm_grad_call(d); }
CPUOPS_B200_API int cpuops_b200_balance_loss(const cpuops_b200_balance_loss_desc* d) { return balance_loss_call(d); }

}  // extern "C"
