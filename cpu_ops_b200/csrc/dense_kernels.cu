// The 16-bit products, their epilogue's gradient, layer norm and the balance loss: a translation unit of its
// own, compiled beside api.cu.
#include "dense_kernels.h"

#include "balance_kernel.cuh"
#include "norm_kernel.cuh"
#include "product_kernel.cuh"

namespace b200 {

ProductKernel product_kernel_of(int form, bool pieces) {
  if (form == kProductPairs) return pieces ? product_kernel<kProductPairs, true> : product_kernel<kProductPairs, false>;
  if (form == kProductParts) return pieces ? product_kernel<kProductParts, true> : product_kernel<kProductParts, false>;
  return pieces ? product_kernel<kProductTiles, true> : product_kernel<kProductTiles, false>;
}
ProductEmptyKernel product_empty() { return product_empty_kernel; }
int product_threads(int form, int epi_warps) { return form == kProductParts ? 224 : 96 + 32 * epi_warps; }

namespace {

template <typename X, typename Y, bool kGradient>
NormChoice norm_choice_for(int n, bool wide) {
  NormChoice c{};
  c.rows_at_once = 1;
  if (n > kNormMaxHeld) {
    c.threads = kNormLongThreads;
    if constexpr (kGradient) {
      c.kernel = norm_grad_long_kernel<X, Y>;
    } else {
      c.kernel = norm_long_kernel<X, Y>;
    }
    return c;
  }
  if (n <= 256) {
    c.threads = 128;
    c.rows_at_once = 4;
    if constexpr (kGradient) {
      c.kernel = wide ? norm_grad_kernel<X, Y, true, true, 1> : norm_grad_kernel<X, Y, false, true, 1>;
    } else {
      c.kernel = wide ? norm_kernel<X, Y, true, true, 1> : norm_kernel<X, Y, false, true, 1>;
    }
    return c;
  }
  const bool one = n <= 8 * kNormMaxThreads;
  const int per = one ? 8 : 16;
  c.threads = ((n + per - 1) / per + 31) / 32 * 32;
  if constexpr (kGradient) {
    c.kernel = one ? (wide ? norm_grad_kernel<X, Y, true, false, 1> : norm_grad_kernel<X, Y, false, false, 1>)
                   : (wide ? norm_grad_kernel<X, Y, true, false, 2> : norm_grad_kernel<X, Y, false, false, 2>);
  } else {
    c.kernel = one ? (wide ? norm_kernel<X, Y, true, false, 1> : norm_kernel<X, Y, false, false, 1>)
                   : (wide ? norm_kernel<X, Y, true, false, 2> : norm_kernel<X, Y, false, false, 2>);
  }
  return c;
}

template <bool kGradient>
NormChoice norm_choice_of(int x_type, int y_type, int n, bool wide) {
  if (x_type == kF16) return norm_choice_for<__half, __half, kGradient>(n, wide);
  if (x_type == kBf16) return norm_choice_for<__nv_bfloat16, __nv_bfloat16, kGradient>(n, wide);
  if (y_type == kF16) return norm_choice_for<float, __half, kGradient>(n, wide);
  if (y_type == kBf16) return norm_choice_for<float, __nv_bfloat16, kGradient>(n, wide);
  return norm_choice_for<float, float, kGradient>(n, wide);
}

}  // namespace

bool norm_is_long(int n) { return n > kNormMaxHeld; }
NormChoice norm_choice(int x_type, int y_type, int n, bool wide, bool gradient) {
  return gradient ? norm_choice_of<true>(x_type, y_type, n, wide) : norm_choice_of<false>(x_type, y_type, n, wide);
}
NormColumnsKernel norm_grad_columns(int x_type, int y_type) {
  if (x_type == kF16) return norm_grad_columns_kernel<__half, __half>;
  if (x_type == kBf16) return norm_grad_columns_kernel<__nv_bfloat16, __nv_bfloat16>;
  if (y_type == kF16) return norm_grad_columns_kernel<float, __half>;
  if (y_type == kBf16) return norm_grad_columns_kernel<float, __nv_bfloat16>;
  return norm_grad_columns_kernel<float, float>;
}

EpilogueGradKernel epilogue_grad_of(int type, bool wide) {
  if (type == kF32) return wide ? epilogue_grad_kernel<float, true> : epilogue_grad_kernel<float, false>;
  if (type == kF16) return wide ? epilogue_grad_kernel<__half, true> : epilogue_grad_kernel<__half, false>;
  return wide ? epilogue_grad_kernel<__nv_bfloat16, true> : epilogue_grad_kernel<__nv_bfloat16, false>;
}
ColumnSumKernel column_sum() { return column_sum_kernel; }

BalanceKernel balance_count() { return balance_count_kernel; }
BalanceKernel balance_of(int experts) {
  const int per_lane = (experts + 31) / 32;
  return per_lane <= 1 ? balance_kernel<1> : per_lane <= 2 ? balance_kernel<2> : per_lane <= 4 ? balance_kernel<4>
       : per_lane <= 8 ? balance_kernel<8> : per_lane <= 16 ? balance_kernel<16> : balance_kernel<32>;
}

}  // namespace b200
