// The 16-bit products, their epilogue's gradient, layer norm and the balance loss: a translation unit of its
// own, compiled beside api.cu.
#include "dense_kernels.h"

#include <algorithm>

#include "balance_kernel.cuh"
#include "norm_kernel.cuh"
#include "product_kernel.cuh"

namespace b200 {

template <int kForm>
static ProductKernel product_kernel_for(bool pieces, bool tma) {
  if (tma) return pieces ? product_kernel<kForm, true, true> : product_kernel<kForm, false, true>;
  return pieces ? product_kernel<kForm, true, false> : product_kernel<kForm, false, false>;
}
ProductKernel product_kernel_of(int form, bool pieces, bool tma) {
  if (form == kProductParts) return pieces ? product_kernel<kProductParts, true, true> : product_kernel<kProductParts, false, true>;
  return form == kProductPairs ? product_kernel_for<kProductPairs>(pieces, tma) : product_kernel_for<kProductTiles>(pieces, tma);
}
ProductEmptyKernel product_empty() { return product_empty_kernel; }
int product_threads(int form, int epi_warps) { return form == kProductParts ? 224 : 96 + 32 * epi_warps; }

namespace {

template <typename X, typename Y, bool kGradient>
NormChoice norm_choice_for(int n, bool wide, bool many, bool dr) {
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
  if constexpr (kGradient) {
    if (n <= 256) {
      c.threads = 128;
      c.rows_at_once = 4;
      c.kernel = wide ? norm_grad_kernel<X, Y, true, true, 1> : norm_grad_kernel<X, Y, false, true, 1>;
      return c;
    }
    if constexpr (sizeof(X) == 2) {
      if (wide && many && n <= 1024) {  // (a row per warp: no barrier, and few rows of partial sums)
        c.threads = 128;
        c.rows_at_once = 4;
        c.kernel = norm_grad_kernel<X, Y, true, true, 4>;
        return c;
      }
    }
    const int row_bytes = n * static_cast<int>((dr ? 2 : 1) * sizeof(X) + sizeof(Y));
    if (wide && many && n % 8 == 0) {
      // sixteen elements per thread, so that few threads share in a row's two sums; two CTAs per SM and more, or one of
      // rows beyond 4096
      const bool one = n > 4096;
      c.threads = ((n + 15) / 16 + 31) / 32 * 32;
      c.ring = std::min(kNormMaxRing, (one ? kNormMostSmem : std::min(100 * 1024, c.threads * 400)) / row_bytes);
      c.smem = c.ring * row_bytes;
      c.kernel = one ? norm_grad_ring_kernel<X, Y, 2, 512> : norm_grad_ring_kernel<X, Y, 2, 256>;
      if (c.ring >= 2) return c;
      c.ring = c.smem = 0;
    }
    if (!wide) {
      c.threads = kNormGradPairThreads;
      c.even = true;
      c.kernel = n <= 2048 ? norm_grad_pairs_kernel<X, Y, 5> : n <= 4096 ? norm_grad_pairs_kernel<X, Y, 9> : norm_grad_pairs_kernel<X, Y, 17>;
      return c;
    }
    // (many rows: sixteen elements per thread, so that half as many threads share in a row's two sums)
    const bool two = n > 8 * kNormMaxThreads || (many && n > 1024 && sizeof(X) == 2);
    const int per = two ? 16 : 8;
    c.threads = ((n + per - 1) / per + 31) / 32 * 32;
    c.kernel = two ? norm_grad_kernel<X, Y, true, false, 2> : norm_grad_kernel<X, Y, true, false, 1>;
  } else {
    constexpr int kSlots = sizeof(X) == 2 ? 2 : 1;
    if (wide && many && n % 8 == 0 && n > 256 && n <= 2048) {
      c.threads = 32 * 2 * kNormWarps;
      c.rows_at_once = 2 * kNormWarps;
      c.ring = 1;
      c.smem = 2 * n * static_cast<int>(sizeof(float)) + kSlots * 2 * kNormWarps * n * static_cast<int>(sizeof(X));
      c.kernel = n <= 1024 ? norm_ring_kernel<X, Y, 4, 2 * kNormWarps, kSlots> : norm_ring_kernel<X, Y, 8, 2 * kNormWarps, kSlots>;
      return c;
    }
    if (wide && many && n % 8 == 0 && n > 1024 && n <= kNormWarpMost) {
      c.threads = 32 * kNormWarps;
      c.rows_at_once = kNormWarps;
      c.ring = 1;
      c.smem = 2 * n * static_cast<int>(sizeof(float)) + kSlots * kNormWarps * n * static_cast<int>(sizeof(X));
      c.kernel = norm_ring_kernel<X, Y, 16, kNormWarps, kSlots>;
      return c;
    }
    if (!wide && n > 256) {
      c.threads = kNormPairThreads;
      c.kernel = n <= 4096 ? norm_pairs_kernel<X, Y, 17> : norm_pairs_kernel<X, Y, 33>;
      return c;
    }
    if (n <= 256 || (many && n <= kNormWarpMost)) {
      c.threads = 32 * kNormWarps;
      c.rows_at_once = kNormWarps;
      c.smem = 2 * ((n + 7) / 8 * 8) * static_cast<int>(sizeof(float));
      // (beyond 256 columns rows of whole vectors took norm_ring_kernel)
      c.kernel = n <= 256    ? (wide ? norm_rows_kernel<X, Y, true, 1> : norm_rows_kernel<X, Y, false, 1>)
                 : n <= 1024 ? norm_rows_kernel<X, Y, true, 4>
                             : norm_rows_kernel<X, Y, true, 16>;
      return c;
    }
    const bool two = n > 8 * kNormMaxThreads;
    const int per = two ? 16 : 8;
    c.threads = ((n + per - 1) / per + 31) / 32 * 32;
    c.kernel = two ? norm_kernel<X, Y, 2> : norm_kernel<X, Y, 1>;
  }
  return c;
}

template <bool kGradient>
NormChoice norm_choice_of(int x_type, int y_type, int n, bool wide, bool many, bool dr) {
  if (x_type == kF16) return norm_choice_for<__half, __half, kGradient>(n, wide, many, dr);
  if (x_type == kBf16) return norm_choice_for<__nv_bfloat16, __nv_bfloat16, kGradient>(n, wide, many, dr);
  if (y_type == kF16) return norm_choice_for<float, __half, kGradient>(n, wide, many, dr);
  if (y_type == kBf16) return norm_choice_for<float, __nv_bfloat16, kGradient>(n, wide, many, dr);
  return norm_choice_for<float, float, kGradient>(n, wide, many, dr);
}

template <typename T, bool kWide>
EpilogueGradKernel epilogue_grad_for(int act) {
  return act == kOpRelu   ? epilogue_grad_kernel<T, kOpRelu, kWide>
         : act == kOpGelu ? epilogue_grad_kernel<T, kOpGelu, kWide>
         : act == kOpSilu ? epilogue_grad_kernel<T, kOpSilu, kWide>
                          : epilogue_grad_kernel<T, 0, kWide>;
}
template <typename T>
EpilogueGradKernel epilogue_grad_pairs_for(int act) {
  return act == kOpRelu   ? epilogue_grad_pairs_kernel<T, kOpRelu>
         : act == kOpGelu ? epilogue_grad_pairs_kernel<T, kOpGelu>
         : act == kOpSilu ? epilogue_grad_pairs_kernel<T, kOpSilu>
                          : epilogue_grad_pairs_kernel<T, 0>;
}

template <typename T>
BalanceKernel balance_for(int experts) {
  const int per_lane = (experts + 31) / 32;
  return per_lane <= 1   ? balance_kernel<T, 1>
         : per_lane <= 2 ? balance_kernel<T, 2>
         : per_lane <= 4 ? balance_kernel<T, 4>
         : per_lane <= 8 ? balance_kernel<T, 8>
         : per_lane <= 16 ? balance_kernel<T, 16>
                          : balance_kernel<T, 32>;
}

}  // namespace

bool norm_is_long(int n) { return n > kNormMaxHeld; }
NormChoice norm_choice(int x_type, int y_type, int n, bool wide, bool many, bool dr, bool gradient) {
  return gradient ? norm_choice_of<true>(x_type, y_type, n, wide, many, dr) : norm_choice_of<false>(x_type, y_type, n, wide, many, dr);
}
NormColumnsKernel norm_grad_columns(int x_type, int y_type) {
  if (x_type == kF16) return norm_grad_columns_kernel<__half, __half>;
  if (x_type == kBf16) return norm_grad_columns_kernel<__nv_bfloat16, __nv_bfloat16>;
  if (y_type == kF16) return norm_grad_columns_kernel<float, __half>;
  if (y_type == kBf16) return norm_grad_columns_kernel<float, __nv_bfloat16>;
  return norm_grad_columns_kernel<float, float>;
}

EpilogueGradKernel epilogue_grad_of(int type, int act, bool wide) {
  if (type == kF32) return wide ? epilogue_grad_for<float, true>(act) : epilogue_grad_for<float, false>(act);
  if (type == kF16) return wide ? epilogue_grad_for<__half, true>(act) : epilogue_grad_pairs_for<__half>(act);
  return wide ? epilogue_grad_for<__nv_bfloat16, true>(act) : epilogue_grad_pairs_for<__nv_bfloat16>(act);
}
ColumnSumKernel column_sum() { return column_sum_kernel; }

BalanceKernel balance_count() { return balance_count_kernel; }
int balance_warps_of(int experts) { return balance_warps((experts + 31) / 32); }
BalanceKernel balance_of(int type, int experts) {
  return type == kF32 ? balance_for<float>(experts) : type == kF16 ? balance_for<__half>(experts) : balance_for<__nv_bfloat16>(experts);
}

}  // namespace b200
