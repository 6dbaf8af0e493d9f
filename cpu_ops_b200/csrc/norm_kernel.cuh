// Layer norm and its gradient, the gradient of bias and activation, and sums of columns.
//
//   mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = 1 / sqrt(var + eps)
//   y = (x - mean) rstd gamma + beta
//   g = dy gamma, xhat = (x - mean) rstd:  dx = rstd (g - sum g / n - xhat sum(g xhat) / n) + dr,
//   dgamma = sum over rows of dy xhat, dbeta = sum over rows of dy
//
// All are bound by HBM: a row is read once and held in registers between its sums and its result; the
// variance is the sum of squared differences from the mean, not a difference of large sums.  CTAs
// stay for many rows, with gamma and beta (and the columns' sums) in registers too.
#pragma once

#include "dense_params.h"
#include "gemm_params.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace b200 {

constexpr int kNormMaxThreads = 512;
constexpr int kNormMaxHeld = 16 * kNormMaxThreads;  // longest row that is held in registers
constexpr int kNormLongThreads = 1024;
constexpr int kNormStrip = 256;      // columns of a CTA of the column kernels

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {  // (rounded to nearest even)
  if constexpr (sizeof(T) == 4) {
    return v;
  } else if constexpr (std::is_same<T, __half>::value) {
    return __float2half_rn(v);
  } else {
    return __float2bfloat16_rn(v);
  }
}

// Eight elements of a row in flight.  kWide: rows are 16-byte aligned; thread t of T holds the elements
// 8 (t + T j) .. + 7; otherwise t + T i.  `left`: elements of the row from `p` on.
template <typename T>
struct alignas(16) Eight {
  T v[8];
};
template <typename T, bool kWide>
__device__ __forceinline__ int element_of(int t, int threads, int j, int i) {
  return kWide ? 8 * (t + threads * j) + i : t + threads * (8 * j + i);
}
template <typename T, bool kWide>
__device__ __forceinline__ Eight<T> load_eight(const T* row, int n, int t, int threads, int j) {
  Eight<T> e;
  if constexpr (kWide) {
    const int c = 8 * (t + threads * j);
    if (c + 8 <= n) {
      const uint4* src = reinterpret_cast<const uint4*>(row + c);
      uint4* dst = reinterpret_cast<uint4*>(e.v);
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(T) / 2); ++w) dst[w] = src[w];
      return e;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = element_of<T, kWide>(t, threads, j, i);
    e.v[i] = c < n ? row[c] : from_f32<T>(0.0f);
  }
  return e;
}
template <typename T, bool kWide>
__device__ __forceinline__ void store_eight(T* row, int n, int t, int threads, int j, const float (&v)[8]) {
  if constexpr (kWide) {
    const int c = 8 * (t + threads * j);
    if (c + 8 <= n) {
      Eight<T> e;
#pragma unroll
      for (int i = 0; i < 8; ++i) e.v[i] = from_f32<T>(v[i]);
      uint4* dst = reinterpret_cast<uint4*>(row + c);
      const uint4* src = reinterpret_cast<const uint4*>(e.v);
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(T) / 2); ++w) dst[w] = src[w];
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = element_of<T, kWide>(t, threads, j, i);
    if (c < n) row[c] = from_f32<T>(v[i]);
  }
}
// Eight of gamma, beta or the like (f32, any alignment; `otherwise` for a null vector and beyond n).
template <bool kWide>
__device__ __forceinline__ void load_vector(const float* vec, int n, int t, int threads, int j, float otherwise, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = element_of<float, kWide>(t, threads, j, i);
    v[i] = vec != nullptr && c < n ? __ldg(vec + c) : otherwise;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The sum over a CTA's warps, the same in every thread.  `slot`: 32 floats of shared memory that no warp may
// still be reading from two calls before (callers take turns over several).
__device__ __forceinline__ float block_sum(float v, float* slot) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? slot[lane] : 0.0f);
}

// kWarp: every warp takes rows of its own (n <= 256 * kV); otherwise the CTA takes one row at a time.
template <typename X, typename Y, bool kWide, bool kWarp, int kV>
__global__ void __launch_bounds__(kWarp ? 128 : kNormMaxThreads) norm_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float slots[4][32];
  const int threads = kWarp ? 32 : static_cast<int>(blockDim.x);
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int first = kWarp ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int step = kWarp ? gridDim.x * 4 : gridDim.x;
  const float inverse = 1.0f / static_cast<float>(p.n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (first >= p.m) return;
  float gamma[kV][8], beta[kV][8];
  Eight<X> next[kV];
  const X* x = static_cast<const X*>(p.x);
#pragma unroll
  for (int j = 0; j < kV; ++j) next[j] = load_eight<X, kWide>(x + first * p.ldx, p.n, t, threads, j);
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    load_vector<kWide>(p.gamma, p.n, t, threads, j, 1.0f, gamma[j]);
    load_vector<kWide>(p.beta, p.n, t, threads, j, 0.0f, beta[j]);
  }
  int turn = 0;
  for (int64_t row = first; row < p.m; row += step, turn ^= 2) {
    float v[kV][8], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = to_f32(next[j].v[i]);
        sum += v[j][i];
      }
    if (row + step < p.m) {
#pragma unroll
      for (int j = 0; j < kV; ++j) next[j] = load_eight<X, kWide>(x + (row + step) * p.ldx, p.n, t, threads, j);
    }
    const float mean = (kWarp ? warp_sum(sum) : block_sum(sum, slots[turn])) * inverse;
    float square = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = element_of<X, kWide>(t, threads, j, i) < p.n ? v[j][i] - mean : 0.0f;
        square = __fmaf_rn(v[j][i], v[j][i], square);
      }
    const float var = (kWarp ? warp_sum(square) : block_sum(square, slots[turn + 1])) * inverse;
    const float rstd = 1.0f / sqrtf(var + p.eps);
    if (t == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
    Y* y = static_cast<Y*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __fmaf_rn(v[j][i] * rstd, gamma[j][i], beta[j][i]);
      store_eight<Y, kWide>(y, p.n, t, threads, j, r);
    }
  }
}

// Rows too long for registers: three passes, the second and third out of L2.
template <typename X, typename Y>
__global__ void __launch_bounds__(kNormLongThreads) norm_long_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float slots[4][32];
  const float inverse = 1.0f / static_cast<float>(p.n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x, turn ^= 2) {
    const X* x = static_cast<const X*>(p.x) + row * p.ldx;
    Y* y = static_cast<Y*>(p.y) + row * p.ldy;
    float sum = 0.0f, square = 0.0f;
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < p.n; c += kNormLongThreads) sum += to_f32(x[c]);
    const float mean = block_sum(sum, slots[turn]) * inverse;
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < p.n; c += kNormLongThreads) {
      const float d = to_f32(x[c]) - mean;
      square = __fmaf_rn(d, d, square);
    }
    const float rstd = 1.0f / sqrtf(block_sum(square, slots[turn + 1]) * inverse + p.eps);
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < p.n; c += kNormLongThreads)
      y[c] = from_f32<Y>(__fmaf_rn((to_f32(x[c]) - mean) * rstd, p.gamma ? __ldg(p.gamma + c) : 1.0f, p.beta ? __ldg(p.beta + c) : 0.0f));
  }
}

// X: the type of x, dx and dr; Y: of dy.  The columns' sums of a CTA's rows go to its row of p.sums.
template <typename X, typename Y, bool kWide, bool kWarp, int kV>
__global__ void __launch_bounds__(kWarp ? 128 : kNormMaxThreads) norm_grad_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float slots[4][32];
  __shared__ float join[kWarp ? 4 : 1][kWarp ? 256 : 1];
  const int threads = kWarp ? 32 : static_cast<int>(blockDim.x);
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int first = kWarp ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int step = kWarp ? gridDim.x * 4 : gridDim.x;
  const float inverse = 1.0f / static_cast<float>(p.n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float gamma[kV][8], dgamma[kV][8], dbeta[kV][8];
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    load_vector<kWide>(p.gamma, p.n, t, threads, j, 1.0f, gamma[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dgamma[j][i] = dbeta[j][i] = 0.0f;
  }
  const X* x = static_cast<const X*>(p.x);
  const Y* dy = static_cast<const Y*>(p.dy);
  Eight<X> next_x[kV];
  Eight<Y> next_dy[kV];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      next_x[j] = load_eight<X, kWide>(x + row * p.ldx, p.n, t, threads, j);
      next_dy[j] = load_eight<Y, kWide>(dy + row * p.lddy, p.n, t, threads, j);
    }
    next_mean = __ldg(p.mean_in + row);
    next_rstd = __ldg(p.rstd_in + row);
  };
  if (first < p.m) fetch(first);
  int turn = 0;
  for (int64_t row = first; row < p.m; row += step, turn ^= 2) {
    float xhat[kV][8], g[kV][8], sum = 0.0f, along = 0.0f;
    const float mean = next_mean, rstd = next_rstd;
    Eight<X> dr[kV];
    if (p.dr) {
#pragma unroll
      for (int j = 0; j < kV; ++j) dr[j] = load_eight<X, kWide>(static_cast<const X*>(p.dr) + row * p.lddr, p.n, t, threads, j);
    }
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = to_f32(next_dy[j].v[i]);
        xhat[j][i] = element_of<X, kWide>(t, threads, j, i) < p.n ? (to_f32(next_x[j].v[i]) - mean) * rstd : 0.0f;
        g[j][i] = d * gamma[j][i];
        dgamma[j][i] = __fmaf_rn(d, xhat[j][i], dgamma[j][i]);
        dbeta[j][i] += d;
        sum += g[j][i];
        along = __fmaf_rn(g[j][i], xhat[j][i], along);
      }
    if (row + step < p.m) fetch(row + step);
    if constexpr (kWarp) {
      sum = warp_sum(sum);
      along = warp_sum(along);
    } else {
      sum = warp_sum(sum);
      along = warp_sum(along);
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
      if (lane == 0) {
        slots[turn][warp] = sum;
        slots[turn + 1][warp] = along;
      }
      __syncthreads();
      sum = warp_sum(lane < warps ? slots[turn][lane] : 0.0f);
      along = warp_sum(lane < warps ? slots[turn + 1][lane] : 0.0f);
    }
    sum *= inverse;
    along *= inverse;
    X* dx = static_cast<X*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[i] = rstd * (g[j][i] - __fmaf_rn(xhat[j][i], along, sum));
        if (p.dr) r[i] += to_f32(dr[j].v[i]);
      }
      store_eight<X, kWide>(dx, p.n, t, threads, j, r);
    }
  }
  if (p.sums == nullptr) return;
  float* out = p.sums + static_cast<int64_t>(blockIdx.x) * p.n;
  const int64_t other = static_cast<int64_t>(gridDim.x) * p.n;
  if constexpr (kWarp) {
    // (columns 0 .. 255: the four warps' sums, added in turn)
    const int warp = threadIdx.x >> 5;
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) join[warp][element_of<X, kWide>(t, 32, 0, i)] = which ? dbeta[0][i] : dgamma[0][i];
      __syncthreads();
      for (int c = threadIdx.x; c < p.n; c += 128)
        out[c + which * other] = ((join[0][c] + join[1][c]) + join[2][c]) + join[3][c];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = element_of<X, kWide>(t, threads, j, i);
        if (c < p.n) {
          out[c] = dgamma[j][i];
          out[c + other] = dbeta[j][i];
        }
      }
  }
}

// Rows too long for registers: dx in two passes, the columns' sums in a kernel of their own.
template <typename X, typename Y>
__global__ void __launch_bounds__(kNormLongThreads) norm_grad_long_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float slots[4][32];
  const float inverse = 1.0f / static_cast<float>(p.n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x, turn ^= 2) {
    const X* x = static_cast<const X*>(p.x) + row * p.ldx;
    const Y* dy = static_cast<const Y*>(p.dy) + row * p.lddy;
    const X* dr = p.dr ? static_cast<const X*>(p.dr) + row * p.lddr : nullptr;
    X* dx = static_cast<X*>(p.y) + row * p.ldy;
    const float mean = __ldg(p.mean_in + row), rstd = __ldg(p.rstd_in + row);
    float sum = 0.0f, along = 0.0f;
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < p.n; c += kNormLongThreads) {
      const float g = to_f32(dy[c]) * (p.gamma ? __ldg(p.gamma + c) : 1.0f);
      sum += g;
      along = __fmaf_rn(g, (to_f32(x[c]) - mean) * rstd, along);
    }
    sum = block_sum(sum, slots[turn]) * inverse;
    along = block_sum(along, slots[turn + 1]) * inverse;
    for (int64_t c = threadIdx.x; c < p.n; c += kNormLongThreads) {
      const float g = to_f32(dy[c]) * (p.gamma ? __ldg(p.gamma + c) : 1.0f), xhat = (to_f32(x[c]) - mean) * rstd;
      float r = rstd * (g - __fmaf_rn(xhat, along, sum));
      if (dr) r += to_f32(dr[c]);
      dx[c] = from_f32<X>(r);
    }
  }
}
// One thread per column; block (x, y) takes 256 columns of the rows y * rows_per_block and on.
template <typename X, typename Y>
__global__ void __launch_bounds__(kNormStrip) norm_grad_columns_kernel(const NormParams p, int rows_per_block) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormStrip + threadIdx.x;
  if (c >= p.n) return;
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * rows_per_block, end = min(begin + rows_per_block, static_cast<int64_t>(p.m));
  const X* x = static_cast<const X*>(p.x) + c;
  const Y* dy = static_cast<const Y*>(p.dy) + c;
  float dgamma = 0.0f, dbeta = 0.0f;
#pragma unroll 4
  for (int64_t row = begin; row < end; ++row) {
    const float d = to_f32(dy[row * p.lddy]);
    dgamma = __fmaf_rn(d, (to_f32(x[row * p.ldx]) - __ldg(p.mean_in + row)) * __ldg(p.rstd_in + row), dgamma);
    dbeta += d;
  }
  float* out = p.sums + static_cast<int64_t>(blockIdx.y) * p.n + c;
  out[0] = dgamma;
  out[static_cast<int64_t>(gridDim.y) * p.n] = dbeta;
}

// ---- gradient of bias and activation --------------------------------------------------------

// act'(z).  Beyond the clamps the slopes are 0 or 1 to the last bit of f32, and the products of an infinity
// and a zero that the formulas have there are not formed.  t = exp(-|v|) gives both the logistic and one
// minus it without a cancellation.
__device__ __forceinline__ float activation_slope(float z, int act) {
  if (act == kOpRelu) return z <= 0.0f ? 0.0f : 1.0f;
  const bool gelu = act == kOpGelu;
  const float most = gelu ? 12.0f : 100.0f;
  z = z > most ? most : (z < -most ? -most : z);  // (NaN stays)
  float v = z, slope = 1.0f;
  if (gelu) {
    const float c = 2.0f * 0.7978845608028654f, zz = z * z;
    v = c * z * __fmaf_rn(0.044715f, zz, 1.0f);
    slope = c * __fmaf_rn(3.0f * 0.044715f, zz, 1.0f);
  }
  const float t = expf(-fabsf(v)), big = __fdividef(1.0f, 1.0f + t), small = t * big;
  const float s = v >= 0.0f ? big : small, rest = v >= 0.0f ? small : big;
  return s * __fmaf_rn(z * slope, rest, 1.0f);
}

// A warp takes rows of the CTA's strip of 256 columns in turn, eight columns per lane: loads and stores of whole
// rows' pieces, the columns' sums in registers until the CTA's rows are done.
template <typename T, bool kWide>
__global__ void __launch_bounds__(256) epilogue_grad_kernel(const EpilogueGradParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float join[8][kNormStrip];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kNormStrip;
  const int n = static_cast<int>(min(static_cast<int64_t>(kNormStrip), p.n - c0));  // columns of this strip
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * p.block_rows;
  const int64_t end = min(begin + p.block_rows, static_cast<int64_t>(p.m));
  const T* dy = static_cast<const T*>(p.dy) + c0;
  const T* z = static_cast<const T*>(p.z) + c0;
  T* dz = static_cast<T*>(p.dz) + c0;
  float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kRows = 4;  // in flight per warp
  for (int64_t r0 = begin + warp; r0 < end; r0 += 8 * kRows) {
    Eight<T> a[kRows], b[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int64_t row = r0 + 8 * k;
      if (row >= end) break;
      a[k] = load_eight<T, kWide>(dy + row * p.lddy, n, lane, 32, 0);
      if (p.z) b[k] = load_eight<T, kWide>(z + row * p.ldz, n, lane, 32, 0);
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int64_t row = r0 + 8 * k;
      if (row >= end) break;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = to_f32(a[k].v[i]);
        if (p.z) {
          const float s = activation_slope(to_f32(b[k].v[i]), p.act);
          v[i] = p.act == kOpRelu && s == 0.0f ? 0.0f : v[i] * s;
        }
        sums[i] += v[i];
      }
      if (p.dz) store_eight<T, kWide>(dz + row * p.lddz, n, lane, 32, 0, v);
    }
  }
  if (p.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) join[warp][element_of<T, kWide>(lane, 32, 0, i)] = sums[i];
  __syncthreads();
  const int c = threadIdx.x;
  if (c < n) {
    float s = join[0][c];
#pragma unroll
    for (int w = 1; w < 8; ++w) s += join[w][c];
    p.sums[static_cast<int64_t>(blockIdx.y) * p.n + c0 + c] = s;
  }
}

// Block (x, y): 32 columns of result y; its warps take the parts in turn.
__global__ void __launch_bounds__(1024) column_sum_kernel(const ColumnSumParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float join[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float* out = p.out[blockIdx.y];
  if (out == nullptr) return;
  float sum = 0.0f;
  if (c < p.n) {
    const float* in = p.in + static_cast<int64_t>(blockIdx.y) * p.parts * p.n + c;
#pragma unroll 4
    for (int i = warp; i < p.parts; i += 32) sum += __ldcg(in + static_cast<int64_t>(i) * p.n);
  }
  join[warp][lane] = sum;
  __syncthreads();
  sum = warp_sum(join[lane][warp]);  // warp w: column w
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + warp;
  if (lane == 0 && column < p.n) out[column] = sum;
}

}  // namespace b200
