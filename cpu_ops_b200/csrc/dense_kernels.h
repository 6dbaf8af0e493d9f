// The kernels of dense_kernels.cu, as the launcher asks for them.
#pragma once

#include <cuda.h>

#include "dense_params.h"

namespace b200 {

using ProductKernel = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, ProductParams);
// tma: C, D and Z by TMA (kProductParts: either).
ProductKernel product_kernel_of(int form, bool pieces, bool tma);
using ProductEmptyKernel = void (*)(ProductParams);
ProductEmptyKernel product_empty();
int product_threads(int form, int epi_warps);

// Types (x, y) of the norms: equal, or f32 and a 16-bit type.
using NormKernel = void (*)(NormParams);
struct NormChoice {
  NormKernel kernel;
  int threads;
  int rows_at_once;  // of a CTA
  int smem;
  int ring;          // rows on their way by bulk copies (0: none)
  bool even;         // takes an even number of CTAs (of two rows or more)
};
// wide: 16-byte aligned rows.  `many`: rows enough for several on every SM; `dr`: the gradient adds one.
NormChoice norm_choice(int x_type, int y_type, int n, bool wide, bool many, bool dr, bool gradient);
constexpr int kNormMostSmem = 200 * 1024;  // of a choice
using NormColumnsKernel = void (*)(NormParams, int);
NormColumnsKernel norm_grad_columns(int x_type, int y_type);
bool norm_is_long(int n);

using EpilogueGradKernel = void (*)(EpilogueGradParams);
EpilogueGradKernel epilogue_grad_of(int type, int act, bool wide);
using ColumnSumKernel = void (*)(ColumnSumParams);
ColumnSumKernel column_sum();

using BalanceKernel = void (*)(BalanceParams);
BalanceKernel balance_count();
BalanceKernel balance_of(int type, int experts);
int balance_warps_of(int experts);  // of its CTAs

}  // namespace b200
