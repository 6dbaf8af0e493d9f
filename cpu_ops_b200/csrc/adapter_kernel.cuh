// Low-rank adapters beside a shared projection: D[t] = C[t] + scale_g * (x[t] A_g^T) B_g^T, every
// row t with its own adapter g = ids[t], or with none.
//
// adapter_rows_kernel: a cluster of eight CTAs per row, one launch.  The row's k is cut over the
// CTAs for u = x A^T; the eight partial sums meet in distributed shared memory, where every CTA
// adds them in ascending order of k (a fixed order: results do not depend on timing); then the
// CTAs cut n among them for D = C + scale * u B^T.  Nothing passes through global memory between
// the two products, so a call needs no workspace.
//
// adapter_down_kernel, adapter_up_kernel: many rows.  Rows are sorted by adapter (the row plan of
// route_kernel.cuh, with a table of tiles of 64 rows), so that one read of an adapter serves
// 64 rows, and both products run on the tensor cores (mma.sync: the arithmetic is a fraction of
// what the memory traffic takes, 2 rank operations per byte of x, C or D):
//   down: u = x A^T for a tile and a part of k, f32 partial sums to the workspace.  16-bit x and A
//         are multiplied as they are.
//   up:   D = C + scale * (the parts' sum, ascending) B^T for a tile and 128 columns.
// A factor in f32 (x where it is f32, and always u, which is not rounded to 16 bits) is cut into two
// tf32 numbers, 22 bits together; 16-bit factors are tf32 numbers as they are.
#pragma once

#include <type_traits>

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

// ---- many rows ---------------------------------------------------------------------------------

constexpr int kAdapterTileCols = 128;  // columns of D per CTA of the up kernel
constexpr int kDownStages = 4;
constexpr int kDownDepth = 64;         // elements of k per stage

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// v = hi + lo, both tf32 (11 bits each; what is left is below 2^-22 of v).  Of an infinity or NaN hi keeps it.
__device__ __forceinline__ void split_tf32(float v, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(v));
  const float rest = v - __uint_as_float(hi);
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
  if (!(fabsf(rest) < INFINITY)) lo = 0u;
}
// Two 16-bit numbers of a word as f32 bits.
template <typename W>
__device__ __forceinline__ void widen(uint32_t pair, uint32_t& first, uint32_t& second) {
  if constexpr (sizeof(W) == 2 && std::is_same<W, __nv_bfloat16>::value) {
    first = pair << 16;
    second = pair & 0xffff0000u;
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    first = __float_as_uint(f.x);
    second = __float_as_uint(f.y);
  }
}

// One 16-byte piece of a row into shared memory: elements i .. of `row`, `left` of which exist (the
// others become zero).  wide: the piece is 16-byte aligned in global memory (asynchronous copy).
template <typename T>
__device__ __forceinline__ void fill_piece(uint32_t dst, const T* row, int i, int left, bool wide) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  const int valid = min(max(left, 0), kPer);
  if (wide) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(valid > 0 ? row + i : row),
                 "r"(valid * static_cast<int>(sizeof(T)))
                 : "memory");
  } else {
    __align__(16) T v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = j < valid ? row[i + j] : T(0.0f);
    const uint4 w = *reinterpret_cast<const uint4*>(v);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
  }
}

struct AdapterTileParams {
  AdapterParams a;
  const int4* tiles;      // {adapter, first place, rows, -}
  const int32_t* order;   // rows sorted by adapter
  float* u;               // [splits][m][rank_pad]
  int32_t rank_pad;       // a multiple of 8
  int32_t splits, depth;  // parts of k and their length (a multiple of kDownDepth)
};

template <typename X>
__host__ __device__ constexpr int down_x_bytes() { return kPlanTileRows * kDownDepth * static_cast<int>(sizeof(X)); }
template <typename X, int kRanks>
__host__ __device__ constexpr int down_smem_bytes() { return kDownStages * (down_x_bytes<X>() + kRanks * kDownDepth * 2); }

// Ranks blockIdx.z * kRanks .. of u for tile blockIdx.x and part blockIdx.y of k.  128 threads, a warp for
// every 16 rows.
template <typename X, typename W, int kRanks>
__global__ void __launch_bounds__(128) adapter_down_kernel(const AdapterTileParams t) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ __align__(128) uint8_t down_smem[];
  const AdapterParams& p = t.a;
  const int4 tile = t.tiles[blockIdx.x];
  if (tile.z == 0 || tile.x >= p.adapters) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank0 = static_cast<int>(blockIdx.z) * kRanks;
  const int k0 = static_cast<int>(blockIdx.y) * t.depth, k1 = min(k0 + t.depth, p.k);
  const uint32_t base = smem_u32(down_smem);
  constexpr int kXBytes = down_x_bytes<X>(), kStage = kXBytes + kRanks * kDownDepth * 2;
  constexpr int kXPieces = kDownDepth * static_cast<int>(sizeof(X)) / 16;  // per row: 8 or 16
  constexpr int kXTurns = kPlanTileRows * kXPieces / 128, kATurns = kRanks * 8 / 128;

  // This thread copies the same piece of a few rows in every stage.
  const X* xrow[kXTurns];
  const W* arow[kATurns];
#pragma unroll
  for (int i = 0; i < kXTurns; ++i) {
    const int r = (tid + 128 * i) / kXPieces;
    xrow[i] = r < tile.z ? static_cast<const X*>(p.x) + t.order[tile.y + r] * p.ldx : nullptr;
  }
#pragma unroll
  for (int i = 0; i < kATurns; ++i) {
    const int j = rank0 + (tid + 128 * i) / 8;
    arow[i] = j < p.rank ? static_cast<const W*>(p.a) + tile.x * p.a_stride + j * p.lda : nullptr;
  }
  auto fill = [&](int stage, int k) {
    const uint32_t xs = base + stage * kStage, as = xs + kXBytes;
#pragma unroll
    for (int i = 0; i < kXTurns; ++i) {
      const int piece = tid + 128 * i, r = piece / kXPieces, c = piece % kXPieces;
      const int at = k + c * (16 / static_cast<int>(sizeof(X)));
      fill_piece<X>(xs + r * (kXPieces * 16) + ((c ^ (r & 7)) << 4), xrow[i] ? xrow[i] : static_cast<const X*>(p.x), at,
                    xrow[i] ? k1 - at : 0, p.wide_k);
    }
#pragma unroll
    for (int i = 0; i < kATurns; ++i) {
      const int piece = tid + 128 * i, j = piece >> 3, c = piece & 7;
      const int at = k + c * 8;
      fill_piece<W>(as + j * 128 + ((c ^ (j & 7)) << 4), arow[i] ? arow[i] : static_cast<const W*>(p.a), at,
                    arow[i] ? k1 - at : 0, p.wide_k);
    }
  };
  const int steps = (k1 - k0 + kDownDepth - 1) / kDownDepth;
#pragma unroll
  for (int s = 0; s < kDownStages - 1; ++s) {
    if (s < steps) fill(s, k0 + s * kDownDepth);
    cp_async_commit();
  }
  float acc[kRanks / 8][4];
#pragma unroll
  for (int j = 0; j < kRanks / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;

  for (int s = 0; s < steps; ++s) {
    cp_async_wait<kDownStages - 2>();
    __syncthreads();  // stage s is complete; everyone is done with the one that is filled next
    if (s + kDownStages - 1 < steps) fill((s + kDownStages - 1) % kDownStages, k0 + (s + kDownStages - 1) * kDownDepth);
    cp_async_commit();
    const uint32_t xs = base + (s % kDownStages) * kStage, as = xs + kXBytes;
    if constexpr (sizeof(X) == 2) {
#pragma unroll
      for (int kk = 0; kk < kDownDepth / 16; ++kk) {
        uint32_t a[4];
        const int r = warp * 16 + (lane & 15), c = 2 * kk + (lane >> 4);
        ldmatrix_x4(a, xs + r * 128 + ((c ^ (r & 7)) << 4));
#pragma unroll
        for (int j = 0; j < kRanks / 16; ++j) {
          uint32_t b[4];  // 16 ranks x 16 elements
          const int n = j * 16 + (lane & 7) + ((lane >> 4) << 3), d = 2 * kk + ((lane >> 3) & 1);
          ldmatrix_x4(b, as + n * 128 + ((d ^ (n & 7)) << 4));
          mma_f16(acc[2 * j], a, b[0], b[1], W());
          mma_f16(acc[2 * j + 1], a, b[2], b[3], W());
        }
      }
    } else {
      // eight elements of k at a time; elements 2 i and 2 i + 1 take the places i and i + 4 of the
      // instruction's k in both factors, so that every thread reads neighbours
      const int g = lane >> 2, i = lane & 3;
#pragma unroll
      for (int kk = 0; kk < kDownDepth / 8; ++kk) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = warp * 16 + g + 8 * h, c = 2 * kk + (i >> 1);
          float2 v;
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                       : "=f"(v.x), "=f"(v.y)
                       : "r"(xs + r * 256 + ((c ^ (r & 7)) << 4) + (i & 1) * 8));
          split_tf32(v.x, hi[h], lo[h]);
          split_tf32(v.y, hi[h + 2], lo[h + 2]);
        }
#pragma unroll
        for (int j = 0; j < kRanks / 8; ++j) {
          const int n = j * 8 + g;
          uint32_t pair, b0, b1;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pair) : "r"(as + n * 128 + ((kk ^ (n & 7)) << 4) + i * 4));
          widen<W>(pair, b0, b1);
          mma_tf32(acc[j], lo, b0, b1);
          mma_tf32(acc[j], hi, b0, b1);
        }
      }
    }
  }
  cp_async_wait<0>();
  // (row g or g + 8, ranks 2 i and 2 i + 1 of eight)
  float* u = t.u + (static_cast<int64_t>(blockIdx.y) * p.m + tile.y) * t.rank_pad;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + (lane >> 2) + 8 * h;
    if (r >= tile.z) continue;
#pragma unroll
    for (int j = 0; j < kRanks / 8; ++j) {
      const int at = rank0 + j * 8 + 2 * (lane & 3);
      if (at < t.rank_pad)
        *reinterpret_cast<float2*>(u + static_cast<int64_t>(r) * t.rank_pad + at) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
    }
  }
}

// Shared memory of the up kernel: u (rows rank_pad + 4 floats apart), then B's 128 rows (rank_pad + 8
// elements apart): a warp's fragment reads meet every bank once.
__host__ __device__ inline int up_smem_bytes(int rank_pad) {
  return kPlanTileRows * (rank_pad + 4) * 4 + kAdapterTileCols * (rank_pad + 8) * 2;
}

// D = C + u B^T for tile blockIdx.y and columns blockIdx.x * 128 ..; 256 threads, a warp for 16 rows x 64
// columns.  Rows without an adapter make up tiles of their own, of which D is C.
template <typename W>
__global__ void __launch_bounds__(256) adapter_up_kernel(const AdapterTileParams t) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ __align__(128) uint8_t up_smem[];
  const AdapterParams& p = t.a;
  const int4 tile = t.tiles[blockIdx.y];
  if (tile.z == 0) return;
  const bool has = tile.x < p.adapters;
  if (!has && p.c == p.d) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, i = lane & 3;
  const int row0 = (warp >> 1) * 16, col0 = static_cast<int>(blockIdx.x) * kAdapterTileCols + (warp & 1) * 64;

  // C first: its loads are in flight during all that follows.  A thread has rows g and g + 8 of its 16
  // and columns 2 i, 2 i + 1 of every eight.
  const bool pairs = (p.ldc & 1) == 0 && (p.ldd & 1) == 0 && (reinterpret_cast<uintptr_t>(p.c) & 7) == 0 &&
                     (reinterpret_cast<uintptr_t>(p.d) & 7) == 0;
  int64_t row[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = row0 + g + 8 * h;
    row[h] = r < tile.z ? t.order[tile.y + r] : -1;
  }
  float2 c[8][2];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int col = col0 + j * 8 + 2 * i;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      c[j][h] = make_float2(0.0f, 0.0f);
      if (row[h] >= 0) {
        const float* src = p.c + row[h] * p.ldc + col;
        if (pairs && col + 1 < p.n) {
          c[j][h] = *reinterpret_cast<const float2*>(src);
        } else {
          if (col < p.n) c[j][h].x = src[0];
          if (col + 1 < p.n) c[j][h].y = src[1];
        }
      }
    }
  }
  float acc[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
  if (has) {
    float* us = reinterpret_cast<float*>(up_smem);
    const int u_ld = t.rank_pad + 4, b_ld = t.rank_pad + 8;
    const uint32_t bs = smem_u32(up_smem) + kPlanTileRows * u_ld * 4;
    const W* b = static_cast<const W*>(p.b) + tile.x * p.b_stride;
    const int pieces = t.rank_pad / 8;
    for (int q = tid; q < kAdapterTileCols * pieces; q += 256) {
      const int n = q / pieces, piece = q - n * pieces;
      const int col = static_cast<int>(blockIdx.x) * kAdapterTileCols + n;
      const bool in = col < p.n;
      fill_piece<W>(bs + (n * b_ld + piece * 8) * 2, in ? b + col * p.ldb : b, piece * 8, in ? p.rank - piece * 8 : 0, p.wide_r);
    }
    cp_async_commit();
    const float scale = p.scales != nullptr ? p.scales[tile.x] : 1.0f;
    for (int q = tid; q < kPlanTileRows * (t.rank_pad / 4); q += 256) {
      const int r = q / (t.rank_pad / 4), e = (q - r * (t.rank_pad / 4)) * 4;
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < tile.z) {
        const float* from = t.u + static_cast<int64_t>(tile.y + r) * t.rank_pad + e;
        for (int s = 0; s < t.splits; ++s) {
          const float4 v = *reinterpret_cast<const float4*>(from + static_cast<int64_t>(s) * p.m * t.rank_pad);
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
        }
      }
      *reinterpret_cast<float4*>(us + r * u_ld + e) = make_float4(sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale);
    }
    cp_async_wait<0>();
    __syncthreads();
    const int nb = (warp & 1) * 64;
    for (int kk = 0; kk < pieces; ++kk) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 v = *reinterpret_cast<const float2*>(us + (row0 + g + 8 * h) * u_ld + kk * 8 + 2 * i);
        split_tf32(v.x, hi[h], lo[h]);
        split_tf32(v.y, hi[h + 2], lo[h + 2]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t pair, b0, b1;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pair) : "r"(bs + ((nb + j * 8 + g) * b_ld + kk * 8 + 2 * i) * 2));
        widen<W>(pair, b0, b1);
        mma_tf32(acc[j], lo, b0, b1);
        mma_tf32(acc[j], hi, b0, b1);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int col = col0 + j * 8 + 2 * i;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (row[h] < 0) continue;
      float* dst = p.d + row[h] * p.ldd + col;
      // (a row without an adapter is C itself: no zero is added to it)
      const float2 y = has ? make_float2(c[j][h].x + acc[j][2 * h], c[j][h].y + acc[j][2 * h + 1]) : c[j][h];
      if (pairs && col + 1 < p.n) {
        *reinterpret_cast<float2*>(dst) = y;
      } else {
        if (col < p.n) dst[0] = y.x;
        if (col + 1 < p.n) dst[1] = y.y;
      }
    }
  }
}

}  // namespace b200
