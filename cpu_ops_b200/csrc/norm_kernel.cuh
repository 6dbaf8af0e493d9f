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
#include "dense_types.cuh"
#include "gemm_params.h"
#include "ptx_sm100.cuh"

namespace b200 {

constexpr int kNormMaxThreads = 512;
constexpr int kNormMaxHeld = 16 * kNormMaxThreads;  // longest row that a CTA holds in registers
constexpr int kNormWarpMost = 4096;                 // ... that a warp does
constexpr int kNormWarps = 8;                       // rows that a CTA of norm_rows_kernel has in flight
constexpr int kNormMaxRing = 4;                     // rows on their way of norm_grad_ring_kernel
constexpr int kNormLongThreads = 1024;
constexpr int kNormStrip = 256;      // columns of a CTA of the column kernels

// Eight elements of a row in flight.  kWide: rows are 16-byte aligned; thread t of T holds the elements
// 8 (t + T j) .. + 7; otherwise t + T i.  `left`: elements of the row from `p` on.
// (held as the words they came in: an element takes a register of its own only while it is worked on)
template <typename T>
struct Eight {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[i / 2]);
      return i % 2 ? __high2float(h) : __low2float(h);
    } else {
      return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {  // elements 2 i and 2 i + 1
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    return make_float2((*this)[2 * i], (*this)[2 * i + 1]);
  }
};
// Two f32 operations per instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 a, b, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 r, a, b; mov.b64 {%0, %1}, r; }"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 a, b, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 r, a, b; mov.b64 {%0, %1}, r; }"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{ .reg .b64 a, b, c, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 r, a, b, c; mov.b64 {%0, %1}, r; }"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <bool kWide>
__device__ __forceinline__ int element_of(int t, int threads, int j, int i) {
  return kWide ? 8 * (t + threads * j) + i : t + threads * (8 * j + i);
}
template <typename T, bool kWide>
__device__ __forceinline__ Eight<T> load_eight(const T* row, int n, int t, int threads, int j) {
  using Word = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
  Eight<T> e;
  if constexpr (kWide) {
    const int c = 8 * (t + threads * j);
    if (c + 8 <= n) {
      const uint4* src = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h) {
        const uint4 v = src[h];
        e.w[4 * h] = v.x;
        e.w[4 * h + 1] = v.y;
        e.w[4 * h + 2] = v.z;
        e.w[4 * h + 3] = v.w;
      }
      return e;
    }
  }
  const Word* words = reinterpret_cast<const Word*>(row);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = element_of<kWide>(t, threads, j, i);
    const uint32_t v = c < n ? static_cast<uint32_t>(words[c]) : 0u;
    if constexpr (sizeof(T) == 4) {
      e.w[i] = v;
    } else {
      e.w[i / 2] = i % 2 ? e.w[i / 2] | (v << 16) : v;
    }
  }
  return e;
}
template <typename T, bool kWide>
__device__ __forceinline__ void store_eight(T* row, int n, int t, int threads, int j, const float (&v)[8]) {
  if constexpr (kWide) {
    const int c = 8 * (t + threads * j);
    if (c + 8 <= n) {
      uint32_t w[2 * sizeof(T)];
#pragma unroll
      for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) {
        if constexpr (sizeof(T) == 4) {
          w[i] = __float_as_uint(v[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      uint4* dst = reinterpret_cast<uint4*>(row + c);
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h) dst[h] = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = element_of<kWide>(t, threads, j, i);
    if (c < n) row[c] = from_f32<T>(v[i]);
  }
}
// Eight of gamma, beta or the like (f32, any alignment; `otherwise` for a null vector and beyond n).
template <bool kWide>
__device__ __forceinline__ void load_vector(const float* vec, int n, int t, int threads, int j, float otherwise, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = element_of<kWide>(t, threads, j, i);
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

// Subtracts the mean from eight elements (those beyond the row stay zero) and adds their squares up.
template <bool kWide>
__device__ __forceinline__ float centred_squares(float (&v)[8], float mean, int n, int t, int threads, int j, float square) {
  if (kWide && 8 * (t + threads * j) + 8 <= n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] -= mean;
      square = __fmaf_rn(v[i], v[i], square);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = element_of<kWide>(t, threads, j, i) < n ? v[i] - mean : 0.0f;
      square = __fmaf_rn(v[i], v[i], square);
    }
  }
  return square;
}

// One row per CTA at a time (of 16-byte aligned rows): few rows, or rows longer than a warp holds.
template <typename X, typename Y, int kV>
__global__ void __launch_bounds__(kNormMaxThreads) norm_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float slots[4][32];
  const int threads = blockDim.x, t = threadIdx.x;
  const float inverse = 1.0f / static_cast<float>(p.n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float gamma[kV][8], beta[kV][8];
  Eight<X> next[kV];
  const X* x = static_cast<const X*>(p.x);
#pragma unroll
  for (int j = 0; j < kV; ++j) next[j] = load_eight<X, true>(x + blockIdx.x * p.ldx, p.n, t, threads, j);
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    load_vector<true>(p.gamma, p.n, t, threads, j, 1.0f, gamma[j]);
    load_vector<true>(p.beta, p.n, t, threads, j, 0.0f, beta[j]);
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x, turn ^= 2) {
    float v[kV][8], sum = 0.0f, square = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = next[j][i];
        sum += v[j][i];
      }
    if (row + gridDim.x < p.m) {
#pragma unroll
      for (int j = 0; j < kV; ++j) next[j] = load_eight<X, true>(x + (row + gridDim.x) * p.ldx, p.n, t, threads, j);
    }
    const float mean = block_sum(sum, slots[turn]) * inverse;
#pragma unroll
    for (int j = 0; j < kV; ++j) square = centred_squares<true>(v[j], mean, p.n, t, threads, j, square);
    const float rstd = 1.0f / sqrtf(block_sum(square, slots[turn + 1]) * inverse + p.eps);
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
      store_eight<Y, true>(y, p.n, t, threads, j, r);
    }
  }
}

// Where element c of gamma (or beta) lies in a vector of n in shared memory whose eights are read by neighbouring lanes: the
// fours of all eights' first halves, then those of the second, so that a warp reads whole lines without conflicts.
__device__ __forceinline__ int weight_at(int c, int n) { return ((c >> 2) & 1) * (n >> 1) + (c >> 3) * 4 + (c & 3); }

// One row per warp at a time, n <= 256 * kV: sums need no barrier, and each of the SM's warps has a whole row on its
// way.  gamma and beta lie in shared memory (2 n floats).
template <typename X, typename Y, bool kWide, int kV>
__global__ void __launch_bounds__(32 * kNormWarps, sizeof(X) == 2 || kV < 16 ? 2 : 1) norm_rows_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) float weights[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float inverse = 1.0f / static_cast<float>(p.n);
  const int room = (p.n + 7) / 8 * 8;  // (whole vectors of eight)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int c = threadIdx.x; c < room; c += 32 * kNormWarps) {
    const int at = kWide ? weight_at(c, room) : c;
    weights[at] = p.gamma != nullptr && c < p.n ? __ldg(p.gamma + c) : 1.0f;
    weights[room + at] = p.beta != nullptr && c < p.n ? __ldg(p.beta + c) : 0.0f;
  }
  __syncthreads();
  const int64_t step = static_cast<int64_t>(gridDim.x) * kNormWarps;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kNormWarps + warp; row < p.m; row += step) {
    const X* x = static_cast<const X*>(p.x) + row * p.ldx;
    Eight<X> raw[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j)
      if (256 * j < p.n) raw[j] = load_eight<X, kWide>(x, p.n, lane, 32, j);
    float sum = 0.0f, square = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      if (256 * j >= p.n) continue;
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) part += raw[j][i];
      sum += part;
    }
    const float mean = warp_sum(sum) * inverse;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      if (256 * j >= p.n) continue;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = raw[j][i];
      square += centred_squares<kWide>(v, mean, p.n, lane, 32, j, 0.0f);
    }
    const float rstd = 1.0f / sqrtf(warp_sum(square) * inverse + p.eps);
    if (lane == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
    Y* y = static_cast<Y*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      if (256 * j >= p.n) continue;
      float r[8];
      if constexpr (kWide) {
        const int c = 8 * (lane + 32 * j);
        if (c < p.n) {
          const float4* g = reinterpret_cast<const float4*>(weights + (c >> 1));
          const float4* b = reinterpret_cast<const float4*>(weights + room + (c >> 1));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 gg = g[h * (room >> 3)], bb = b[h * (room >> 3)];
            r[4 * h] = __fmaf_rn((raw[j][4 * h] - mean) * rstd, gg.x, bb.x);
            r[4 * h + 1] = __fmaf_rn((raw[j][4 * h + 1] - mean) * rstd, gg.y, bb.y);
            r[4 * h + 2] = __fmaf_rn((raw[j][4 * h + 2] - mean) * rstd, gg.z, bb.z);
            r[4 * h + 3] = __fmaf_rn((raw[j][4 * h + 3] - mean) * rstd, gg.w, bb.w);
          }
          store_eight<Y, kWide>(y, p.n, lane, 32, j, r);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = min(element_of<kWide>(lane, 32, j, i), p.n - 1);
          r[i] = __fmaf_rn((raw[j][i] - mean) * rstd, weights[c], weights[room + c]);
        }
        store_eight<Y, kWide>(y, p.n, lane, 32, j, r);
      }
    }
  }
}

// Waits for the bulk copies of rows that are on their way, `row` the first of up to `ring` of them, before the CTA or warp that
// gave up ends.  (Not inlined: its loop beside the rows' cost the gradient's registers, 8192 x 4096 with dr 55 us, 51 in this form.)
__device__ __noinline__ void drain_rows(uint32_t bar, int ring, uint32_t slot, uint32_t phase, int64_t row, int64_t step, int64_t m) {
  for (int i = 0; i < ring && row < m; ++i, row += step) {
    mbar_drain(bar + 8u * slot, phase);
    if (++slot == static_cast<uint32_t>(ring)) {
      slot = 0;
      phase ^= 1u;
    }
  }
}

// The same with a warp's next kSlots rows (two of a 16-bit type, one of f32) on their way by bulk copies: the loads do not wait
// for the arithmetic (8192 x 4096 bf16 44 us without, 25 in this form; 31 before gamma and beta lay without bank conflicts, when
// 12 warps with two rows each, or 16 with one, took 31 and 36).  Rows are whole vectors of eight, 16-byte aligned.  Shared
// memory: gamma and beta, kSlots rows per warp.
template <typename X, typename Y, int kV, int kWarps, int kSlots>
__global__ void __launch_bounds__(32 * kWarps, 1) norm_ring_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) float weights[];
  __shared__ __align__(8) uint64_t barriers[kWarps][kSlots];
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = p.n;
  const float inverse = 1.0f / static_cast<float>(n);
  const uint32_t row_bytes = static_cast<uint32_t>(n) * sizeof(X);
  const uint32_t ring = smem_u32(weights + 2 * n) + static_cast<uint32_t>(kSlots * warp) * row_bytes, bar = smem_u32(&barriers[warp][0]);
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane < kSlots) mbar_init(bar + 8u * lane, 1);
  fence_mbar_init();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  auto request = [&](int64_t r, uint32_t slot) {
    if (lane == 0 && r < p.m) {
      mbar_expect_tx(bar + 8u * slot, row_bytes);
      bulk_load(ring + slot * row_bytes, static_cast<const X*>(p.x) + r * p.ldx, row_bytes, bar + 8u * slot);
    }
  };
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kSlots; ++i) request(row + i * step, static_cast<uint32_t>(i));
  for (int c = threadIdx.x; c < n; c += 32 * kWarps) {
    weights[weight_at(c, n)] = p.gamma != nullptr ? __ldg(p.gamma + c) : 1.0f;
    weights[n + weight_at(c, n)] = p.beta != nullptr ? __ldg(p.beta + c) : 0.0f;
  }
  __syncthreads();
  const uint64_t budget_ns = static_cast<uint64_t>(p.wait_budget_us) * 1000ull;
  uint32_t slot = 0, phase = 0;
  for (; row < p.m; row += step) {
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar + 8u * slot, phase, &abort_flag, budget_ns))) {
      if (lane == 0) {
        leave_error(p.error, kErrProducerWait);
        drain_rows(bar, kSlots, slot, phase, row, step, p.m);
      }
      break;
    }
    Eight<X> raw[kV];
    const uint32_t from = ring + slot * row_bytes;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const int c = 8 * (lane + 32 * j);
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(X) / 2); ++h) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (c < n)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(from + static_cast<uint32_t>(c * static_cast<int>(sizeof(X)) + 16 * h)));
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[j].w[4 * h + i] = w[i];
      }
    }
    __syncwarp();  // every lane has read the slot
    fence_proxy_async_shared_cta();
    request(row + kSlots * step, slot);
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1u;
    }
    float2 sum = both(0.0f), square = both(0.0f);
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = add2(sum, raw[j].pair(i));  // (zeros beyond the row)
    const float mean = warp_sum(sum.x + sum.y) * inverse;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      if (8 * (lane + 32 * j) < n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 d = add2(raw[j].pair(i), both(-mean));
          square = fma2(d, d, square);
        }
      }
    }
    const float rstd = 1.0f / sqrtf(warp_sum(square.x + square.y) * inverse + p.eps);
    if (lane == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
    Y* y = static_cast<Y*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const int c = 8 * (lane + 32 * j);
      if (c < n) {
        const float4* g = reinterpret_cast<const float4*>(weights + (c >> 1));
        const float4* b = reinterpret_cast<const float4*>(weights + n + (c >> 1));
        float r[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 gg = g[h * (n >> 3)], bb = b[h * (n >> 3)];
          const float2 lo = fma2(mul2(add2(raw[j].pair(2 * h), both(-mean)), both(rstd)), make_float2(gg.x, gg.y), make_float2(bb.x, bb.y));
          const float2 hi = fma2(mul2(add2(raw[j].pair(2 * h + 1), both(-mean)), both(rstd)), make_float2(gg.z, gg.w), make_float2(bb.z, bb.w));
          r[4 * h] = lo.x;
          r[4 * h + 1] = lo.y;
          r[4 * h + 2] = hi.x;
          r[4 * h + 3] = hi.y;
        }
        store_eight<Y, true>(y, n, lane, 32, j, r);
      }
    }
  }
}

// ---- rows that are not 16-byte aligned --------------------------------------------------------
//
// Elements are taken in pairs that lie in aligned words where the types have 16 bits: where a row begins in the middle of
// a word (every second row of an odd leading dimension), the pairs are (-1, 0), (1, 2), ... .  `s`, the row's
// shift, is 0 or 1.  (Element by element these kernels took 170 us for 8192 x 4096, 214 for the gradient.)

template <typename T>
__device__ __forceinline__ int row_shift(const T* row) {
  return sizeof(T) == 2 ? static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 1) & 1u) : 0;
}
template <typename T>
struct Pair {
  uint32_t w[sizeof(T) / 2];
  __device__ __forceinline__ float2 get() const {
    if constexpr (sizeof(T) == 4) {
      return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    } else if constexpr (std::is_same<T, __half>::value) {
      return __half22float2(*reinterpret_cast<const __half2*>(&w[0]));
    } else {
      return make_float2(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xFFFF0000u));
    }
  }
};
// Elements e and e + 1 of a row of n (zeros outside); `word`: they lie in one aligned word.
template <typename T>
__device__ __forceinline__ Pair<T> load_pair(const T* row, int e, int n, bool word) {
  Pair<T> p;
  if constexpr (sizeof(T) == 4) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(row);
    p.w[0] = e >= 0 && e < n ? u[e] : 0u;
    p.w[1] = e + 1 < n ? u[e + 1] : 0u;
  } else {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(row);
    if (word && e >= 0 && e + 1 < n) {
      p.w[0] = *reinterpret_cast<const uint32_t*>(u + e);
    } else {
      p.w[0] = e >= 0 && e < n ? u[e] : 0u;
      if (e + 1 < n) p.w[0] |= static_cast<uint32_t>(u[e + 1]) << 16;
    }
  }
  return p;
}
template <typename T>
__device__ __forceinline__ void store_pair(T* row, int e, int n, bool word, float2 v) {
  if constexpr (sizeof(T) == 2) {
    if (word && e >= 0 && e + 1 < n) {
      uint32_t w;
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v.x, v.y);
        w = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        w = *reinterpret_cast<const uint32_t*>(&h);
      }
      *reinterpret_cast<uint32_t*>(row + e) = w;
      return;
    }
  }
  if (e >= 0 && e < n) row[e] = from_f32<T>(v.x);
  if (e + 1 < n) row[e + 1] = from_f32<T>(v.y);
}
__device__ __forceinline__ float2 vector_pair(const float* vec, int e, int n, float otherwise) {
  return make_float2(vec != nullptr && e >= 0 && e < n ? __ldg(vec + e) : otherwise, vec != nullptr && e + 1 < n ? __ldg(vec + e + 1) : otherwise);
}

constexpr int kNormPairThreads = 128, kNormGradPairThreads = 256;

// One row per CTA at a time; gamma and beta stay in the first cache.
template <typename X, typename Y, int kP>
__global__ void __launch_bounds__(kNormPairThreads) norm_pairs_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float slots[4][32];
  const int t = threadIdx.x, n = p.n;
  const float inverse = 1.0f / static_cast<float>(n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x, turn ^= 2) {
    const X* x = static_cast<const X*>(p.x) + row * p.ldx;
    Y* y = static_cast<Y*>(p.y) + row * p.ldy;
    const int s = sizeof(Y) == 2 ? row_shift(y) : row_shift(x);
    const bool word = row_shift(x) == s;
    Pair<X> raw[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i)
      if (2 * kNormPairThreads * i < n + s) raw[i] = load_pair(x, 2 * (t + kNormPairThreads * i) - s, n, word);
    float2 sum = both(0.0f), square = both(0.0f);
#pragma unroll
    for (int i = 0; i < kP; ++i)
      if (2 * kNormPairThreads * i < n + s) sum = add2(sum, raw[i].get());
    const float mean = block_sum(sum.x + sum.y, slots[turn]) * inverse;
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      if (2 * kNormPairThreads * i >= n + s) continue;
      const int e = 2 * (t + kNormPairThreads * i) - s;
      float2 d = add2(raw[i].get(), both(-mean));
      if (e < 0 || e >= n) d.x = 0.0f;
      if (e + 1 >= n) d.y = 0.0f;
      square = fma2(d, d, square);
    }
    const float rstd = 1.0f / sqrtf(block_sum(square.x + square.y, slots[turn + 1]) * inverse + p.eps);
    if (t == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      if (2 * kNormPairThreads * i >= n + s) continue;
      const int e = 2 * (t + kNormPairThreads * i) - s;
      const float2 v = fma2(mul2(add2(raw[i].get(), both(-mean)), both(rstd)), vector_pair(p.gamma, e, n, 1.0f), vector_pair(p.beta, e, n, 0.0f));
      store_pair(y, e, n, true, v);
    }
  }
}

// A CTA's rows have the same shift, so that a thread's columns stay the same: there is an even number of CTAs, or one row.
template <typename X, typename Y, int kP>
__global__ void __launch_bounds__(kNormGradPairThreads, kP <= 5 || (kP <= 9 && sizeof(X) == 2) ? 2 : 1) norm_grad_pairs_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float2 slots[2][32];
  const int t = threadIdx.x, n = p.n, lane = t & 31, warp = t >> 5;
  constexpr int kWarps = kNormGradPairThreads / 32;
  const float inverse = 1.0f / static_cast<float>(n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const X* x0 = static_cast<const X*>(p.x);
  const Y* dy0 = static_cast<const Y*>(p.dy);
  const int64_t first = blockIdx.x, step = gridDim.x;
  const int s = first < p.m ? (sizeof(Y) == 2 ? row_shift(dy0 + first * p.lddy) : row_shift(x0 + first * p.ldx)) : 0;
  auto inside = [&](int i) { return 2 * kNormGradPairThreads * i < n + s; };
  auto element = [&](int i) { return 2 * (t + kNormGradPairThreads * i) - s; };
  Pair<X> next_x[kP], next_dr[kP];
  Pair<Y> next_dy[kP];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t row) {
    const X* x = x0 + row * p.ldx;
    const Y* dy = dy0 + row * p.lddy;
    const X* dr = p.dr ? static_cast<const X*>(p.dr) + row * p.lddr : nullptr;
    const bool word_x = row_shift(x) == s, word_dy = row_shift(dy) == s, word_dr = dr && row_shift(dr) == s;
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      if (!inside(i)) continue;
      next_x[i] = load_pair(x, element(i), n, word_x);
      next_dy[i] = load_pair(dy, element(i), n, word_dy);
      if (dr) next_dr[i] = load_pair(dr, element(i), n, word_dr);
    }
    next_mean = __ldg(p.mean_in + row);
    next_rstd = __ldg(p.rstd_in + row);
  };
  if (first < p.m) fetch(first);
  float2 dgamma[kP], dbeta[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) dgamma[i] = dbeta[i] = both(0.0f);
  int turn = 0;
  for (int64_t row = first; row < p.m; row += step, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    Pair<X> xs[kP], drs[kP];
    Pair<Y> dys[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      xs[i] = next_x[i];
      dys[i] = next_dy[i];
      if (p.dr) drs[i] = next_dr[i];
    }
    if (kP <= 9 && row + step < p.m) fetch(row + step);
    float2 sum = both(0.0f), along = both(0.0f);
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      if (!inside(i)) continue;
      // (elements outside the row: dy is zero, and with it all that is added up)
      const float2 d = dys[i].get(), xhat = mul2(add2(xs[i].get(), both(-mean)), both(rstd));
      const float2 g = mul2(d, vector_pair(p.gamma, element(i), n, 1.0f));
      dgamma[i] = fma2(d, xhat, dgamma[i]);
      dbeta[i] = add2(dbeta[i], d);
      sum = add2(sum, g);
      along = fma2(g, xhat, along);
    }
    float s1 = warp_sum(sum.x + sum.y), s2 = warp_sum(along.x + along.y);
    if (lane == 0) slots[turn][warp] = make_float2(s1, s2);
    __syncthreads();
    const float2 v = lane < kWarps ? slots[turn][lane] : make_float2(0.0f, 0.0f);
    s1 = warp_sum(v.x) * inverse;
    s2 = warp_sum(v.y) * inverse;
    X* dx = static_cast<X*>(p.y) + row * p.ldy;
    const bool word = row_shift(dx) == s;
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      if (!inside(i)) continue;
      const float2 xhat = mul2(add2(xs[i].get(), both(-mean)), both(rstd)), even = fma2(xhat, both(s2), both(s1));
      const float2 g = mul2(dys[i].get(), vector_pair(p.gamma, element(i), n, 1.0f));
      float2 r = mul2(both(rstd), add2(g, make_float2(-even.x, -even.y)));
      if (p.dr) r = add2(r, drs[i].get());
      store_pair(dx, element(i), n, word, r);
    }
    if (kP > 9 && row + step < p.m) fetch(row + step);  // (no registers for two rows)
  }
  if (p.sums == nullptr) return;
  float* out = p.sums + static_cast<int64_t>(blockIdx.x) * n;
  const int64_t other = static_cast<int64_t>(gridDim.x) * n;
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    if (!inside(i)) continue;
    store_pair(out, element(i), n, false, dgamma[i]);
    store_pair(out + other, element(i), n, false, dbeta[i]);
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

// X: the type of x, dx and dr; Y: of dy.  The columns' sums of a CTA's rows go to its row of p.sums.  A row's elements
// stay as they were loaded between its sums and its result, and the next row is on its way meanwhile.
// kWarp: every warp takes rows of its own (n <= 256 * kV).
template <typename X, typename Y, bool kWide, bool kWarp, int kV>
__global__ void __launch_bounds__(kWarp ? 128 : kNormMaxThreads) norm_grad_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float2 slots[2][32];
  __shared__ float join[kWarp ? 4 : 1][kWarp ? 256 * kV : 1];
  const int threads = kWarp ? 32 : static_cast<int>(blockDim.x);
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int first = kWarp ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int step = kWarp ? gridDim.x * 4 : gridDim.x;
  const float inverse = 1.0f / static_cast<float>(p.n);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const X* x = static_cast<const X*>(p.x);
  const Y* dy = static_cast<const Y*>(p.dy);
  Eight<X> next_x[kV], next_dr[kV];
  Eight<Y> next_dy[kV];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      next_x[j] = load_eight<X, kWide>(x + row * p.ldx, p.n, t, threads, j);
      next_dy[j] = load_eight<Y, kWide>(dy + row * p.lddy, p.n, t, threads, j);
      if (p.dr) next_dr[j] = load_eight<X, kWide>(static_cast<const X*>(p.dr) + row * p.lddr, p.n, t, threads, j);
    }
    next_mean = __ldg(p.mean_in + row);
    next_rstd = __ldg(p.rstd_in + row);
  };
  if (first < p.m) fetch(first);
  float gamma[kV][8], dgamma[kV][8], dbeta[kV][8];
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    load_vector<kWide>(p.gamma, p.n, t, threads, j, 1.0f, gamma[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dgamma[j][i] = dbeta[j][i] = 0.0f;
  }
  int turn = 0;
  for (int64_t row = first; row < p.m; row += step, turn ^= 1) {
    float sum = 0.0f, along = 0.0f;
    const float mean = next_mean, rstd = next_rstd;
    Eight<X> this_x[kV], this_dr[kV];
    Eight<Y> this_dy[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      this_x[j] = next_x[j];
      this_dy[j] = next_dy[j];
      if (p.dr) this_dr[j] = next_dr[j];
    }
    if (row + step < p.m) fetch(row + step);
    // (elements beyond the row: dy is zero, and with it all that is added up)
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = this_dy[j][i], xhat = (this_x[j][i] - mean) * rstd, g = d * gamma[j][i];
        dgamma[j][i] = __fmaf_rn(d, xhat, dgamma[j][i]);
        dbeta[j][i] += d;
        sum += g;
        along = __fmaf_rn(g, xhat, along);
      }
    sum = warp_sum(sum);
    along = warp_sum(along);
    if constexpr (!kWarp) {
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
      if (lane == 0) slots[turn][warp] = make_float2(sum, along);
      __syncthreads();
      const float2 v = lane < warps ? slots[turn][lane] : make_float2(0.0f, 0.0f);
      sum = warp_sum(v.x);
      along = warp_sum(v.y);
    }
    sum *= inverse;
    along *= inverse;
    X* dx = static_cast<X*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xhat = (this_x[j][i] - mean) * rstd;
        r[i] = rstd * (this_dy[j][i] * gamma[j][i] - __fmaf_rn(xhat, along, sum));
        if (p.dr) r[i] += this_dr[j][i];
      }
      store_eight<X, kWide>(dx, p.n, t, threads, j, r);
    }
  }
  if (p.sums == nullptr) return;
  float* out = p.sums + static_cast<int64_t>(blockIdx.x) * p.n;
  const int64_t other = static_cast<int64_t>(gridDim.x) * p.n;
  if constexpr (kWarp) {
    // (the four warps' sums, added in turn)
    const int warp = threadIdx.x >> 5;
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) join[warp][element_of<kWide>(t, 32, j, i)] = which ? dbeta[j][i] : dgamma[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < p.n; c += 128)
        out[c + which * other] = ((join[0][c] + join[1][c]) + join[2][c]) + join[3][c];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kV; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = element_of<kWide>(t, threads, j, i);
        if (c < p.n) {
          out[c] = dgamma[j][i];
          out[c + other] = dbeta[j][i];
        }
      }
    }
  }
}

// The same with rows on their way by bulk copies, p.ring rows ahead (rows of whole vectors of eight, 16-byte aligned):
// a thread holds no row but the one it works on (8192 x 4096 bf16 with dr 76 us with the next row in registers, 51 in this
// form: 5.2 TB/s).  Shared memory: p.ring times the rows of x, dy and dr.
template <typename X, typename Y, int kV, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads, kMaxThreads == 256 && sizeof(X) == 2 ? 2 : 1) norm_grad_ring_kernel(const NormParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) uint8_t rows[];
  __shared__ float2 slots[2][32];
  __shared__ __align__(8) uint64_t barriers[kNormMaxRing];
  __shared__ int abort_flag;
  const int t = threadIdx.x, threads = blockDim.x, n = p.n, lane = t & 31, warp = t >> 5, warps = threads >> 5;
  const float inverse = 1.0f / static_cast<float>(n);
  const uint32_t x_bytes = static_cast<uint32_t>(n) * sizeof(X), dy_bytes = static_cast<uint32_t>(n) * sizeof(Y);
  const uint32_t slot_bytes = (p.dr ? 2u : 1u) * x_bytes + dy_bytes, bar = smem_u32(barriers), ring0 = smem_u32(rows);
  if (t == 0) {
    abort_flag = 0;
    for (int i = 0; i < p.ring; ++i) mbar_init(bar + 8u * i, 1);
    fence_mbar_init();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t step = gridDim.x;
  auto request = [&](int64_t r, uint32_t slot) {  // thread 0
    if (r >= p.m) return;
    const uint32_t to = ring0 + slot * slot_bytes, b = bar + 8u * slot;
    mbar_expect_tx(b, slot_bytes);
    bulk_load(to, static_cast<const X*>(p.x) + r * p.ldx, x_bytes, b);
    bulk_load(to + x_bytes, static_cast<const Y*>(p.dy) + r * p.lddy, dy_bytes, b);
    if (p.dr) bulk_load(to + x_bytes + dy_bytes, static_cast<const X*>(p.dr) + r * p.lddr, x_bytes, b);
  };
  int64_t row = blockIdx.x;
  if (t == 0)
    for (int i = 0; i < p.ring; ++i) request(row + i * step, static_cast<uint32_t>(i));
  float2 gamma[kV][4], dgamma[kV][4], dbeta[kV][4];
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    float g[8];
    load_vector<true>(p.gamma, n, t, threads, j, 1.0f, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      gamma[j][i] = make_float2(g[2 * i], g[2 * i + 1]);
      dgamma[j][i] = dbeta[j][i] = both(0.0f);
    }
  }
  float next_mean = row < p.m ? __ldg(p.mean_in + row) : 0.0f, next_rstd = row < p.m ? __ldg(p.rstd_in + row) : 0.0f;
  __syncthreads();
  const uint64_t budget_ns = static_cast<uint64_t>(p.wait_budget_us) * 1000ull;
  uint32_t slot = 0, phase = 0, turn = 0;
  for (; row < p.m; row += step, turn ^= 1u) {
    const float mean = next_mean, rstd = next_rstd;
    if (row + step < p.m) {
      next_mean = __ldg(p.mean_in + row + step);
      next_rstd = __ldg(p.rstd_in + row + step);
    }
    const bool ran_out = !mbar_wait_bounded(bar + 8u * slot, phase, &abort_flag, budget_ns);
    const uint32_t from = ring0 + slot * slot_bytes;
    Eight<X> xs[kV], drs[kV];
    Eight<Y> dys[kV];
    auto take = [&](auto& e, uint32_t base, int c) {
      constexpr int kWords = sizeof(e.w) / 4;
#pragma unroll
      for (int h = 0; h < kWords / 4; ++h) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (c < n)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(base + static_cast<uint32_t>(c * (kWords / 2) + 16 * h)));
#pragma unroll
        for (int i = 0; i < 4; ++i) e.w[4 * h + i] = w[i];
      }
    };
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const int c = 8 * (t + threads * j);
      take(xs[j], from, c);
      take(dys[j], from + x_bytes, c);
      if (p.dr) take(drs[j], from + x_bytes + dy_bytes, c);
    }
    // (elements beyond the row: dy is zero, and with it all that is added up)
    float2 sum = both(0.0f), along = both(0.0f);
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 d = dys[j].pair(i), xhat = mul2(add2(xs[j].pair(i), both(-mean)), both(rstd)), g = mul2(d, gamma[j][i]);
        dgamma[j][i] = fma2(d, xhat, dgamma[j][i]);
        dbeta[j][i] = add2(dbeta[j][i], d);
        sum = add2(sum, g);
        along = fma2(g, xhat, along);
      }
    float s1 = warp_sum(sum.x + sum.y), s2 = warp_sum(along.x + along.y);
    if (lane == 0) slots[turn][warp] = make_float2(s1, s2);
    fence_proxy_async_shared_cta();  // the slot has been read: before it is filled again
    if (__syncthreads_or(ran_out)) break;
    if (t == 0) request(row + p.ring * step, slot);
    if (++slot == static_cast<uint32_t>(p.ring)) {
      slot = 0;
      phase ^= 1u;
    }
    const float2 v = lane < warps ? slots[turn][lane] : make_float2(0.0f, 0.0f);
    s1 = warp_sum(v.x) * inverse;
    s2 = warp_sum(v.y) * inverse;
    X* dx = static_cast<X*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      float r[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 xhat = mul2(add2(xs[j].pair(i), both(-mean)), both(rstd));
        const float2 even = fma2(xhat, both(s2), both(s1));
        float2 v2 = mul2(both(rstd), add2(mul2(dys[j].pair(i), gamma[j][i]), make_float2(-even.x, -even.y)));
        if (p.dr) v2 = add2(v2, drs[j].pair(i));
        r[2 * i] = v2.x;
        r[2 * i + 1] = v2.y;
      }
      store_eight<X, true>(dx, n, t, threads, j, r);
    }
  }
  if (row < p.m) {  // (a wait ran out)
    if (t == 0) {
      leave_error(p.error, kErrProducerWait);
      drain_rows(bar, p.ring, slot, phase, row, step, p.m);
    }
    __syncthreads();
    return;
  }
  if (p.sums == nullptr) return;
  float* out = p.sums + static_cast<int64_t>(blockIdx.x) * n;
  const int64_t other = static_cast<int64_t>(gridDim.x) * n;
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const int c = 8 * (t + threads * j);
    if (c < n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *reinterpret_cast<float2*>(out + c + 2 * i) = dgamma[j][i];
        *reinterpret_cast<float2*>(out + other + c + 2 * i) = dbeta[j][i];
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

// min and max that keep a NaN.
__device__ __forceinline__ float clamp_nan(float v, float most) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(most));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(-most));
  return v;
}
// dy act'(z) of two elements.  gelu and silu are z s with s = 1 / (1 + t), t = exp(-v): their slope is
// s (1 + z v' (1 - s)) with 1 - s = t s, which does not cancel.  z is clamped where the slope is 0 or 1 to the last
// bit of f32 and t still a number (exp(88.5)): beyond, the products of an infinity and a zero that the formulas have there
// are not formed.  exp2 of a rounded product is exact enough: with u = 2^-24 t is off by e = (4 |v| + 4) u (silu 1.25 |v|), s
// by (1 - s) e + 3 u, t s by s e + 4 u, and the whole by 7.6e-7 of dy at most (silu 5.7e-7).
template <int kAct>
__device__ __forceinline__ float2 slope_times(float2 dy, float2 z) {
  if constexpr (kAct == 0) return dy;
  if constexpr (kAct == kOpRelu) return make_float2(z.x <= 0.0f ? 0.0f : dy.x, z.y <= 0.0f ? 0.0f : dy.y);
  constexpr bool kGelu = kAct == kOpGelu;
  constexpr float most = kGelu ? 10.05f : 88.4f, log2e = 1.4426950408889634f;
  z = make_float2(clamp_nan(z.x, most), clamp_nan(z.y, most));
  float2 v, w;  // -v log2(e), and z v'
  if constexpr (kGelu) {
    constexpr float c = 2.0f * 0.7978845608028654f;
    const float2 zz = mul2(z, z);
    v = mul2(z, fma2(both(-c * 0.044715f * log2e), zz, both(-c * log2e)));
    w = mul2(z, fma2(both(c * 3.0f * 0.044715f), zz, both(c)));
  } else {
    v = mul2(z, both(-log2e));
    w = z;
  }
  float2 t, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(v.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(v.y));
  const float2 d = add2(t, both(1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(d.y));
  return mul2(mul2(dy, s), fma2(w, mul2(t, s), both(1.0f)));
}

// A warp takes rows of the CTA's strip of 256 columns in turn, eight columns per lane: loads and stores of whole
// rows' pieces, the columns' sums in registers until the CTA's rows are done.  Bound by HBM and, with gelu or silu, nearly by
// the instructions of the slope: 8192 x 14336 bf16 116 us with relu, 126 with silu, 132 with gelu (705 MB, 107 us at the
// measured copy rate; element by element 150).
template <typename T, int kAct, bool kWide>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && kWide ? 4 : 3) epilogue_grad_kernel(const EpilogueGradParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float join[8][kNormStrip];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kNormStrip;
  const int n = static_cast<int>(min(static_cast<int64_t>(kNormStrip), p.n - c0));  // columns of this strip
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * p.block_rows;
  const int64_t end = min(begin + p.block_rows, static_cast<int64_t>(p.m));
  const T* dy = static_cast<const T*>(p.dy) + c0;
  const T* z = kAct ? static_cast<const T*>(p.z) + c0 : nullptr;
  T* dz = p.dz ? static_cast<T*>(p.dz) + c0 : nullptr;
  float2 sums[4] = {both(0.0f), both(0.0f), both(0.0f), both(0.0f)};
  auto finish = [&](int64_t row, const Eight<T>& a, const Eight<T>& b) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 r = slope_times<kAct>(a.pair(i), kAct ? b.pair(i) : both(0.0f));
      sums[i] = add2(sums[i], r);
      v[2 * i] = r.x;
      v[2 * i + 1] = r.y;
    }
    if (kAct || dz) store_eight<T, kWide>(dz + row * p.lddz, n, lane, 32, 0, v);
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int64_t row = begin + warp;
  for (; row + 8 < end; row += 16) {  // two rows in flight
    Eight<T> a[2], b[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      a[k] = load_eight<T, kWide>(dy + (row + 8 * k) * p.lddy, n, lane, 32, 0);
      if (kAct) b[k] = load_eight<T, kWide>(z + (row + 8 * k) * p.ldz, n, lane, 32, 0);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) finish(row + 8 * k, a[k], b[k]);
  }
  if (row < end) {
    const Eight<T> a = load_eight<T, kWide>(dy + row * p.lddy, n, lane, 32, 0);
    Eight<T> b = a;
    if (kAct) b = load_eight<T, kWide>(z + row * p.ldz, n, lane, 32, 0);
    finish(row, a, b);
  }
  if (p.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) join[warp][element_of<kWide>(lane, 32, 0, i)] = i % 2 ? sums[i / 2].y : sums[i / 2].x;
  __syncthreads();
  const int c = threadIdx.x;
  if (c < n) {
    float s = join[0][c];
#pragma unroll
    for (int w = 1; w < 8; ++w) s += join[w][c];
    p.sums[static_cast<int64_t>(blockIdx.y) * p.n + c0 + c] = s;
  }
}

// A word or a 16-bit element if `valid`, else zero.
__device__ __forceinline__ uint32_t load_word_if(const void* p, bool valid) {
  uint32_t v;
  asm volatile("{ .reg .pred q; setp.ne.b32 q, %2, 0; mov.b32 %0, 0; @q ld.global.b32 %0, [%1]; }"
               : "=r"(v) : "l"(p), "r"(valid ? 1 : 0) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_half_if(const void* p, bool valid) {
  uint16_t v;
  asm volatile("{ .reg .pred q; setp.ne.b32 q, %2, 0; mov.b16 %0, 0; @q ld.global.b16 %0, [%1]; }"
               : "=h"(v) : "l"(p), "r"(valid ? 1 : 0) : "memory");
  return v;
}
// load_pair of a 16-bit type by predicated loads: behind load_pair's branches each load waits for the one before it
// (8192 x 14336, gelu's gradient with a leading dimension of 14339: 258 us, 193 in this form and with two rows in flight).
// Where a row is asked for ahead of its use it is the slower one, since it puts the halves together at once
// (layer norm's gradient of 8192 x 4096 146 -> 308 us).
template <typename T>
__device__ __forceinline__ Pair<T> load_pair_at_once(const T* row, int e, int n, bool word) {
  const bool lo = e >= 0 && e < n, hi = e + 1 < n, whole = word && lo && hi;
  Pair<T> p;
  p.w[0] = load_word_if(row + e, whole) | load_half_if(row + e, lo && !whole) | load_half_if(row + e + 1, hi && !whole) << 16;
  return p;
}

// The same for 16-bit rows that are not 16-byte aligned.  A CTA's rows have the same shift s (with odd leading dimensions it
// takes every second one), and its strip begins s columns earlier.
template <typename T, int kAct>
__global__ void __launch_bounds__(256, 3) epilogue_grad_pairs_kernel(const EpilogueGradParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float join[8][kNormStrip];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = p.n;
  const int64_t block = static_cast<int64_t>(blockIdx.y) / p.every, begin = block * p.block_rows * p.every + blockIdx.y % p.every;
  const int64_t end = min(begin + static_cast<int64_t>(p.block_rows) * p.every, static_cast<int64_t>(p.m));
  const T* dy0 = static_cast<const T*>(p.dy);
  const T* z0 = static_cast<const T*>(p.z);
  T* dz0 = static_cast<T*>(p.dz);
  float2 sums[4] = {both(0.0f), both(0.0f), both(0.0f), both(0.0f)};
  const int s = begin < p.m ? row_shift(dz0 ? dz0 + begin * p.lddz : dy0 + begin * p.lddy) : 0;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kNormStrip - s;  // (-1 in the first strip: outside the row)
  if (c0 >= n) return;
  auto element = [&](int i) { return static_cast<int>(c0) + 2 * (lane + 32 * i); };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  struct Row {
    Pair<T> a[4], b[4];
  };
  auto load = [&](Row& r, int64_t row) {
    const T* dy = dy0 + row * p.lddy;
    const T* z = kAct ? z0 + row * p.ldz : nullptr;
    const bool word_dy = row_shift(dy) == s, word_z = kAct && row_shift(z) == s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.a[i] = load_pair_at_once(dy, element(i), n, word_dy);
      if (kAct) r.b[i] = load_pair_at_once(z, element(i), n, word_z);
    }
  };
  auto finish = [&](const Row& r, int64_t row) {
    T* dz = dz0 + row * p.lddz;
    const bool word = row_shift(dz) == s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = slope_times<kAct>(r.a[i].get(), kAct ? r.b[i].get() : both(0.0f));
      sums[i] = add2(sums[i], v);
      if (kAct || dz0) store_pair(dz, element(i), n, word, v);
    }
  };
  const int64_t step = 8 * p.every;
  int64_t row = begin + static_cast<int64_t>(warp) * p.every;
  for (; row + step < end; row += 2 * step) {  // two rows in flight
    Row r0, r1;
    load(r0, row);
    load(r1, row + step);
    finish(r0, row);
    finish(r1, row + step);
  }
  if (row < end) {
    Row r;
    load(r, row);
    finish(r, row);
  }
  if (p.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    join[warp][2 * (lane + 32 * i)] = sums[i].x;
    join[warp][2 * (lane + 32 * i) + 1] = sums[i].y;
  }
  __syncthreads();
  const int64_t c = c0 + threadIdx.x;
  if (c >= 0 && c < n) {
    float sum = join[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < 8; ++w) sum += join[w][threadIdx.x];
    p.sums[static_cast<int64_t>(blockIdx.y) * n + c] = sum;
  }
}

// Block (x, y): 64 columns of result y, two to a lane; its warps take the parts in turn, all of a warp's loads in flight.
// Bound by a launch and one latency: 4 to 5 us for the 296 parts of 2 x 4096 columns.
__global__ void __launch_bounds__(1024) column_sum_kernel(const ColumnSumParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float2 join[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + 2 * lane;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float* out = blockIdx.y == 0 ? p.out0 : p.out1;
  if (out == nullptr) return;
  float2 sum = both(0.0f);
  const float* in = p.in + static_cast<int64_t>(blockIdx.y) * p.parts * p.n + c;
  if (p.n % 2 == 0) {
    if (c < p.n) {
#pragma unroll 10
      for (int i = warp; i < p.parts; i += warps) sum = add2(sum, __ldcg(reinterpret_cast<const float2*>(in + static_cast<int64_t>(i) * p.n)));
    }
  } else if (c < p.n) {
    const bool two = c + 1 < p.n;
#pragma unroll 5
    for (int i = warp; i < p.parts; i += warps) {
      const float* at = in + static_cast<int64_t>(i) * p.n;
      sum = add2(sum, make_float2(__ldcg(at), two ? __ldcg(at + 1) : 0.0f));
    }
  }
  join[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < p.n) {
    for (int w = 1; w < warps; ++w) sum = add2(sum, join[w][lane]);
    out[c] = sum.x;
    if (c + 1 < p.n) out[c + 1] = sum.y;
  }
}

}  // namespace b200
