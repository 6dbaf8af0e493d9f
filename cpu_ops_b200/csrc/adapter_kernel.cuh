// Low-rank adapters beside a shared projection: D[t] = C[t] + scale_g * (x[t] A_g^T) B_g^T, every
// row t with its own adapter g = ids[t], or with none.
//
// adapter_rows_kernel: a cluster of eight CTAs per row, one launch.  The row's k is cut over the
// CTAs for u = x A^T; the eight partial sums meet in distributed shared memory, where every CTA
// adds them in ascending order of k (a fixed order: results do not depend on timing); then the
// CTAs cut n among them for D = C + scale * u B^T.  Nothing passes through global memory between
// the two products, so a call needs no workspace.
#pragma once

#include "ptx_sm100_pair.cuh"
#include "route_kernel.cuh"

namespace b200 {

constexpr int kMaxRank = 256;
constexpr int kAdapterCluster = 8;
constexpr int kAdapterThreads = 256;

struct AdapterParams {
  const void* x;
  const void* a;
  const void* b;
  const int32_t* ids;
  const float* scales;  // or null
  const float* c;
  float* d;
  int64_t ldx, lda, ldb, a_stride, b_stride, ldc, ldd;
  int32_t m, n, k, rank, adapters;
  int32_t wide_k, wide_r;  // 1: rows of x and A (of B) start on 16-byte boundaries
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Elements i .. i + 7 of a row of `len` (zeros behind it); `wide`: the row is 16-byte aligned, i a
// multiple of 8.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int i, int len, bool wide, float (&v)[8]) {
  if (wide && i + 8 <= len) {
    if constexpr (sizeof(T) == 4) {
      const float4 lo = *reinterpret_cast<const float4*>(row + i), hi = *reinterpret_cast<const float4*>(row + i + 4);
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
      v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(row + i);
      const T* h = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(h[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < len ? to_f32<T>(row[i + j]) : 0.0f;
  }
}

template <typename X, typename W>
__global__ void __launch_bounds__(kAdapterThreads) __cluster_dims__(kAdapterCluster, 1, 1)
    adapter_rows_kernel(const AdapterParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // Shared memory of another CTA exists once that CTA has started: the waits below, before the first
  // store to it, are for every CTA's arrival here.
  cluster_arrive();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float part[kAdapterCluster][kMaxRank];  // [CTA the sum comes from][rank]
  __shared__ float u[kMaxRank];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = static_cast<int>(cluster_cta_rank());
  const int row = static_cast<int>(blockIdx.x) / kAdapterCluster;
  const int g = p.ids[row];
  const bool has = g >= 0 && g < p.adapters;  // (the same in the whole cluster)

  if (has) {
    // u, this CTA's part of k (whole groups of eight elements)
    const int per = ((p.k + kAdapterCluster - 1) / kAdapterCluster + 7) / 8 * 8;
    const int k0 = min(cta * per, p.k), k1 = min(k0 + per, p.k);
    const X* x = static_cast<const X*>(p.x) + row * p.ldx;
    const W* a = static_cast<const W*>(p.a) + g * p.a_stride;
    for (int j = warp; j < p.rank; j += kAdapterThreads / 32) {
      const W* aj = a + j * p.lda;
      float sum = 0.0f;
      for (int i = k0 + lane * 8; i < k1; i += 256) {
        float xv[8], av[8];
        load8<X>(x, i, k1, p.wide_k, xv);
        load8<W>(aj, i, k1, p.wide_k, av);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __fmaf_rn(xv[e], av[e], sum);
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      if (lane == 0) part[cta][j] = sum;
    }
  }
  __syncwarp();
  cluster_wait();
  __syncthreads();
  if (has) {
    // this CTA's sums to the seven others
    for (int i = threadIdx.x; i < p.rank * kAdapterCluster; i += kAdapterThreads) {
      const int j = i / kAdapterCluster, to_cta = i % kAdapterCluster;
      if (to_cta == cta) continue;
      const uint32_t to = map_to_cta(smem_u32(&part[cta][j]), static_cast<uint32_t>(to_cta));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(part[cta][j]) : "memory");
    }
  }
  // all partial sums are in place; and no CTA has left while another still writes to it
  __syncwarp();
  cluster_sync_all();
  if (has) {
    const float scale = p.scales != nullptr ? p.scales[g] : 1.0f;
    for (int j = threadIdx.x; j < p.rank; j += kAdapterThreads) {
      float sum = part[0][j];
#pragma unroll
      for (int c = 1; c < kAdapterCluster; ++c) sum += part[c][j];
      u[j] = sum * scale;
    }
    __syncthreads();
  } else if (p.c == p.d) {
    return;
  }
  const int per_n = (p.n + kAdapterCluster - 1) / kAdapterCluster;
  const int n0 = cta * per_n, n1 = min(n0 + per_n, p.n);
  const W* b = static_cast<const W*>(p.b) + (has ? g * p.b_stride : 0);
  for (int col = n0 + threadIdx.x; col < n1; col += kAdapterThreads) {
    float sum = 0.0f;
    if (has) {
      const W* bj = b + col * p.ldb;
      for (int i = 0; i < p.rank; i += 8) {
        float bv[8];
        load8<W>(bj, i, p.rank, p.wide_r, bv);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < p.rank) sum = __fmaf_rn(u[i + e], bv[e], sum);
      }
      p.d[row * p.ldd + col] = p.c[row * p.ldc + col] + sum;
    } else {
      p.d[row * p.ldd + col] = p.c[row * p.ldc + col];
    }
  }
}

}  // namespace b200
