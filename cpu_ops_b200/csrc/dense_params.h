// Parameter blocks of the 16-bit products, their epilogue's gradient, layer norm and the balance loss,
// shared by the launcher (dense_api.h, in api.cu) and the kernels (dense_kernels.cu).
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace b200 {

enum : int32_t { kF32 = 0, kF16 = 1, kBf16 = 2 };  // element types (CPUOPS_B200_TYPE_*)
__host__ __device__ inline int type_bytes(int type) { return type == kF32 ? 4 : 2; }

// ---- 16-bit products ------------------------------------------------------------------------

// Forms of the kernel: persistent with one CTA or a pair of them per tile; or one tile per cluster, whose CTAs
// take a part of k each.
enum : int32_t { kProductTiles = 0, kProductPairs = 1, kProductParts = 2 };

constexpr int kProductEpiWarps = 8;    // at most; 4 where shared memory is short of stages otherwise, and in kProductParts
constexpr int kProductMaxStages = 12;
constexpr int kProductMaxParts = 8;
constexpr int kProductBarrierBytes = 512;
constexpr int kProductBiasFloats = 1024;  // 128 for each of eight epilogue warps, 256 for each of four; behind the barriers
// kPieces: k-blocks of a piece of k where D is f32; where D has 16 bits, and the longest running sum of such a D, by type.
constexpr int kProductPieceBlocks = 8, kProductPieceBlocks16 = 128;
constexpr int kProductRunningBlocksF16 = 256, kProductRunningBlocksBf16 = 2048;

struct ProductParams {
  // Kernel view: Dk (Mk x Nk) = Ak Bk, Ak on the MMA's M side.  `swapped`: the caller's B is Ak, so that
  // kernel rows are the caller's columns.
  int32_t Mk, Nk;
  int32_t m_tiles, n_tiles, k_blocks;   // tiles of 128 (pairs: 256) x BN; k-blocks of 64
  int32_t BN, stages, nacc, raster_m, parts;
  int32_t piece_blocks;                 // kPieces: k-blocks of a piece of k
  int32_t tile_rows;                    // kProductParts: rows of Ak per tile, at most 128 (others: 128)
  int32_t a_mn, b_mn;                   // 1: the m (n) direction is contiguous in memory
  int32_t swapped;
  uint32_t idesc;
  int32_t epi_warps;
  int32_t act;                          // kOp* or 0
  float alpha, beta;
  const float* bias;                    // by the caller's column, or null
  const void* C;                        // null: beta == 0
  void* D;
  void* Z;                              // alpha A B + bias, or null
  int64_t ldc, ldd, ldz;
  int32_t type, c_type, d_type;         // of A and B, of C, of D and Z
  int32_t ring_bytes, ring_depth;       // epilogue buffers of one warp, and how many chunks of each matrix they hold
  int32_t* error;
  uint32_t wait_budget_us;
};

// Chunks of 32 x 32 elements, as rows of 64 or 128 bytes.
__host__ __device__ inline int chunk_bytes(int type) { return 1024 * type_bytes(type); }

// ---- gradient of bias and activation ----------------------------------------------------------

struct EpilogueGradParams {
  const void* dy;
  const void* z;      // null: no activation
  void* dz;           // may be null without an activation
  float* sums;        // one row of n per block of rows, or the result itself where there is one block; or null
  int64_t lddy, ldz, lddz;
  int32_t m, n;
  int32_t block_rows;
  int32_t every;      // rows that are not 16-byte aligned: a block takes every row, or every second one
};

// Sum of `parts` rows of n, `parts * count` floats apart from one result to the next.
struct ColumnSumParams {
  const float* in;
  float* out0;
  float* out1;
  int32_t parts, n;
};

// ---- layer norm ---------------------------------------------------------------------------------

struct NormParams {
  const void* x;
  const void* dy;        // gradient
  const void* dr;        // gradient: added to dx, or null
  const float* gamma;    // or null (1)
  const float* beta;     // or null (0)
  void* y;               // y, or dx
  float* mean;           // forward: or null
  float* rstd;
  const float* mean_in;  // gradient
  const float* rstd_in;
  float* sums;           // gradient: per CTA, n sums of dy xhat, then (from n * gridDim.x on) n of dy; or null
  int64_t ldx, lddy, lddr, ldy;
  int32_t m, n;
  int32_t ring;          // gradient by bulk copies: rows on their way
  float eps;
  int32_t* error;        // kernels that wait for bulk copies
  uint32_t wait_budget_us;
};

// ---- balance loss -------------------------------------------------------------------------------

struct BalanceParams {
  const void* logits;
  const int32_t* ids;
  void* dlogits;           // or null
  int32_t* counts;         // or null
  float* loss;             // or null
  const float* upstream;   // or null (1)
  int32_t* part_counts;    // per counting block: experts counts, then the number of tokens with an expert
  float* part_scores;      // per main block: experts sums of scores
  int32_t* ticket;
  int64_t ld, ldg;
  int32_t tokens, experts, top_k, sigmoid;
  int32_t count_blocks;
  float coefficient;
};

}  // namespace b200
