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
//   up:   D = C + scale * (the parts' sum, ascending) B^T for a tile and some columns.
// A factor in f32 is not rounded to 16 bits: x (where it is f32) is cut into two tf32 numbers, 22 bits
// together (16-bit factors are tf32 numbers as they are), u into two or three of B's type.
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
  int32_t align_k, align_r, align_c, align_d;  // what rows of x and A (of B, C, D) start on: 16, 8, 4 or 2 bytes
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

// Sixteen elements of a row of B as they are stored, `left` of which exist.
template <typename W>
struct Sixteen {
  uint4 lo, hi;
  __device__ __forceinline__ void load(const W* row, int left, bool wide) {
    lo = hi = make_uint4(0, 0, 0, 0);
    if (wide && left >= 16) {
      lo = reinterpret_cast<const uint4*>(row)[0];
      hi = reinterpret_cast<const uint4*>(row)[1];
    } else {
      __align__(16) W v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = j < left ? row[j] : W(0.0f);
      lo = reinterpret_cast<const uint4*>(v)[0];
      hi = reinterpret_cast<const uint4*>(v)[1];
    }
  }
  // sum + the product with 16 floats (shared memory, 16-byte aligned); what does not exist on either side is zero
  __device__ __forceinline__ float dot(const float* u, float sum) const {
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 f = reinterpret_cast<const float4*>(u)[j];
      const W* h = reinterpret_cast<const W*>(&w[2 * j]);
      sum = __fmaf_rn(f.x, to_f32<W>(h[0]), sum);
      sum = __fmaf_rn(f.y, to_f32<W>(h[1]), sum);
      sum = __fmaf_rn(f.z, to_f32<W>(h[2]), sum);
      sum = __fmaf_rn(f.w, to_f32<W>(h[3]), sum);
    }
    return sum;
  }
};

// What bounds it is latency (one row: two reads from memory after one another, the exchange between them),
// with many rows the traffic; so a thread has the B of two columns, and their C, on their way before u is known.
constexpr int kRowCols = 2;  // columns a thread works on at a time
template <typename X, typename W>
__global__ void __launch_bounds__(kAdapterThreads, 4) __cluster_dims__(kAdapterCluster, 1, 1)
    adapter_rows_kernel(const AdapterParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // Shared memory of another CTA exists once that CTA has started: the wait below, before the first
  // store to it, is for every CTA's arrival here.
  cluster_arrive();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float part[kAdapterCluster][kMaxRank];  // [CTA the sum comes from][rank]
  __shared__ __align__(16) float u[kMaxRank];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = static_cast<int>(cluster_cta_rank());
  const int row = static_cast<int>(blockIdx.x) / kAdapterCluster;
  const int g = p.ids[row];
  const bool has = g >= 0 && g < p.adapters;  // (the same in the whole cluster)
  cluster_wait();

  // This CTA's columns; of a thread: n0 + tid, + 256, ...
  const int per_n = (p.n + kAdapterCluster - 1) / kAdapterCluster;
  const int n0 = cta * per_n, n1 = min(n0 + per_n, p.n);
  const W* b = static_cast<const W*>(p.b) + (has ? g * p.b_stride : 0);
  const float* c_row = p.c + row * p.ldc;
  float* d_row = p.d + row * p.ldd;
  const bool wide_r = p.align_r == 16;
  Sixteen<W> bv[kRowCols];
  float cv[kRowCols];
  auto load = [&](int col0) {
#pragma unroll
    for (int j = 0; j < kRowCols; ++j) {
      const int col = col0 + j * kAdapterThreads;
      cv[j] = col < n1 ? c_row[col] : 0.0f;
      bv[j].lo = bv[j].hi = make_uint4(0, 0, 0, 0);
      if (has && col < n1) bv[j].load(b + col * p.ldb, p.rank, wide_r);
    }
  };
  if (has || p.c != p.d) load(n0 + tid);

  if (has) {
    // u, this CTA's part of k (whole groups of eight elements), two ranks of a warp at a time
    const int per = ((p.k + kAdapterCluster - 1) / kAdapterCluster + 7) / 8 * 8;
    const int k0 = min(cta * per, p.k), k1 = min(k0 + per, p.k);
    const X* x = static_cast<const X*>(p.x) + row * p.ldx;
    const W* a = static_cast<const W*>(p.a) + g * p.a_stride;
    const bool wide_k = p.align_k == 16;
    for (int j = 2 * warp; j < p.rank; j += 2 * kAdapterThreads / 32) {
      const bool two = j + 1 < p.rank;
      const W *a0 = a + j * p.lda, *a1 = two ? a0 + p.lda : a0;
      float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll 2
      for (int i = k0 + lane * 8; i < k1; i += 256) {
        float xv[8], v0[8], v1[8];
        load8<X>(x, i, k1, wide_k, xv);
        load8<W>(a0, i, k1, wide_k, v0);
        load8<W>(a1, i, k1, wide_k, v1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum0 = __fmaf_rn(xv[e], v0[e], sum0);
          sum1 = __fmaf_rn(xv[e], v1[e], sum1);
        }
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) {
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, s);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, s);
      }
      // to all eight CTAs: lane l to CTA l % 8, lanes 8-15 the second rank
      if (lane < kAdapterCluster || (two && lane < 2 * kAdapterCluster)) {
        const int rank = j + lane / kAdapterCluster;
        const uint32_t to = map_to_cta(smem_u32(&part[cta][rank]), static_cast<uint32_t>(lane % kAdapterCluster));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(lane < kAdapterCluster ? sum0 : sum1) : "memory");
      }
    }
  }
  // all partial sums are in place; and no CTA has left while another still writes to it
  __syncwarp();
  cluster_sync_all();
  if (!has && p.c == p.d) return;
  const int rank_pad = (p.rank + 15) / 16 * 16;
  if (has) {
    const float scale = p.scales != nullptr ? p.scales[g] : 1.0f;
    for (int j = tid; j < rank_pad; j += kAdapterThreads) {
      float sum = 0.0f;
      if (j < p.rank) {
        sum = part[0][j];
#pragma unroll
        for (int c = 1; c < kAdapterCluster; ++c) sum += part[c][j];
      }
      u[j] = sum * scale;
    }
    __syncthreads();
  }
  for (int col0 = n0 + tid; col0 < n1; col0 += kRowCols * kAdapterThreads) {
    if (col0 != n0 + tid) load(col0);
    float sum[kRowCols];
#pragma unroll
    for (int j = 0; j < kRowCols; ++j) sum[j] = 0.0f;
    if (has) {
      for (int r0 = 0; r0 < p.rank; r0 += 16) {
        if (r0 > 0) {
#pragma unroll
          for (int j = 0; j < kRowCols; ++j) {
            const int col = col0 + j * kAdapterThreads;
            if (col < n1) bv[j].load(b + col * p.ldb + r0, p.rank - r0, wide_r);
          }
        }
#pragma unroll
        for (int j = 0; j < kRowCols; ++j) sum[j] = bv[j].dot(u + r0, sum[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kRowCols; ++j) {
      const int col = col0 + j * kAdapterThreads;
      // (a row without an adapter is C itself: no zero is added to it)
      if (col < n1) d_row[col] = has ? cv[j] + sum[j] : cv[j];
    }
  }
}

// ---- many rows ---------------------------------------------------------------------------------

constexpr int kUpCols = 64;            // columns of D per step of the up kernel
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
// v = hi + lo, both tf32 (11 bits each; what is left is below 2^-22 of v).  hi is cut, lo rounded, by
// masks: the conversion instruction has a sixteenth of their rate and bound the up kernel (127 us of
// 8192 rows, rank 64, n 4096).  Of an infinity or NaN hi keeps it.
__device__ __forceinline__ void split_tf32(float v, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(v) & 0xffffe000u;
  const float rest = v - __uint_as_float(hi);
  lo = fabsf(rest) < INFINITY ? (__float_as_uint(rest) + 0x1000u) & 0xffffe000u : 0u;
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
// others become zero).  `align`: the boundary that pieces start on in global memory; from four bytes
// on the copies are asynchronous (synchronous ones of a D of 777 x 1999, eight-byte aligned, took
// 15.6 us where these take 12.6).
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int bytes) {
  if constexpr (kBytes == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(kBytes) : "memory");
  }
}
// Such a piece by plain loads, and its way into shared memory.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* row, int i, int left) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  __align__(16) T v[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) v[j] = j < left ? row[i + j] : T(0.0f);
  return *reinterpret_cast<const uint4*>(v);
}
__device__ __forceinline__ void store_piece(uint32_t dst, const uint4& w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}
template <typename T>
__device__ __forceinline__ void fill_piece(uint32_t dst, const T* row, int i, int left, int align) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  const int valid = min(max(left, 0), kPer);
  const int bytes = valid * static_cast<int>(sizeof(T));
  const char* from = reinterpret_cast<const char*>(valid > 0 ? row + i : row);
  if (align == 16) {
    copy_async<16>(dst, from, bytes);
  } else if (align == 8) {
#pragma unroll
    for (int j = 0; j < 16; j += 8) copy_async<8>(dst + j, from + (bytes > j ? j : 0), min(8, max(0, bytes - j)));
  } else if (align == 4) {
#pragma unroll
    for (int j = 0; j < 16; j += 4) copy_async<4>(dst + j, from + (bytes > j ? j : 0), min(4, max(0, bytes - j)));
  } else {
    store_piece(dst, load_piece<T>(row, i, valid));
  }
}

struct AdapterTileParams {
  AdapterParams a;
  const int4* tiles;      // {adapter, first place, rows, -}
  const int32_t* order;   // rows sorted by adapter
  float* u;               // [splits][m][rank_pad]
  int32_t rank_pad;       // a multiple of 16
  int32_t splits, depth;  // parts of k and their length (a multiple of kDownDepth)
  int32_t up_cols;        // columns of D per CTA of the up kernel (a multiple of kUpCols)
};

// What the tiles' products make NaN is made anew from the whole factors: with an infinity in the 16-bit factor the
// products of the other one's terms may be of either sign or, of a term of zero, NaN, and so may those of a
// term that is an infinity and others that are beyond f16's range.  (The check costs 1 us of 98, 8192 rows,
// rank 64, n 4096; beside the products, in their loops, it cost f32 rows 7 of 146.)
//
// Element j of this CTA's part of u for row r of its tile, of f32 rows (which alone are cut there).
template <typename W>
__device__ __forceinline__ void whole_part(const AdapterTileParams& t, int r, int j) {
  const AdapterParams& p = t.a;
  const int4 tile = t.tiles[blockIdx.x];
  const int k0 = static_cast<int>(blockIdx.y) * t.depth, k1 = min(k0 + t.depth, p.k);
  const float* x = static_cast<const float*>(p.x) + t.order[tile.y + r] * p.ldx;
  const W* a = static_cast<const W*>(p.a) + tile.x * p.a_stride + j * p.lda;
  float u = 0.0f;
#pragma unroll 1
  for (int i = k0; i < k1 && u == u; ++i) u = __fmaf_rn(x[i], to_f32<W>(a[i]), u);
  t.u[(static_cast<int64_t>(blockIdx.y) * p.m + tile.y + r) * t.rank_pad + j] = u;
}

template <typename X>
__host__ __device__ constexpr int down_x_bytes() { return kPlanTileRows * kDownDepth * static_cast<int>(sizeof(X)); }
template <typename X, int kRanks>
__host__ __device__ constexpr int down_smem_bytes() { return kDownStages * (down_x_bytes<X>() + kRanks * kDownDepth * 2); }

// Ranks blockIdx.z * kRanks .. of u for tile blockIdx.x and part blockIdx.y of k.  128 threads, a warp for
// every 16 rows.  kWide: rows of x and A start on 16-byte boundaries (the other kinds of copy in the
// same loop cost 2 us of 28).
template <typename X, typename W, int kRanks, bool kWide>
__global__ void __launch_bounds__(128) adapter_down_kernel(const __grid_constant__ AdapterTileParams t) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ __align__(128) uint8_t down_smem[];
  const AdapterParams& p = t.a;
  const int4 tile = t.tiles[blockIdx.x];
  if (tile.z == 0 || tile.x >= p.adapters) return;
  const int align = kWide ? 16 : p.align_k;
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
    if (!kWide && align == 2) {
      // rows on odd elements: all of this thread's pieces are loaded before the first is stored (piece by piece
      // a stage took eight memory latencies: 8192 rows, rank 64, 2000 x 2000, bf16 157 us, 138 so, f32 267, 184)
      uint4 vx[kXTurns], va[kATurns];
#pragma unroll
      for (int i = 0; i < kXTurns; ++i) {
        const int at = k + (tid + 128 * i) % kXPieces * (16 / static_cast<int>(sizeof(X)));
        vx[i] = load_piece<X>(xrow[i], at, xrow[i] ? k1 - at : 0);
      }
#pragma unroll
      for (int i = 0; i < kATurns; ++i) {
        const int at = k + ((tid + 128 * i) & 7) * 8;
        va[i] = load_piece<W>(arow[i], at, arow[i] ? k1 - at : 0);
      }
#pragma unroll
      for (int i = 0; i < kXTurns; ++i) {
        const int piece = tid + 128 * i, r = piece / kXPieces, c = piece % kXPieces;
        store_piece(xs + r * (kXPieces * 16) + ((c ^ (r & 7)) << 4), vx[i]);
      }
#pragma unroll
      for (int i = 0; i < kATurns; ++i) {
        const int piece = tid + 128 * i, j = piece >> 3, c = piece & 7;
        store_piece(as + j * 128 + ((c ^ (j & 7)) << 4), va[i]);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kXTurns; ++i) {
      const int piece = tid + 128 * i, r = piece / kXPieces, c = piece % kXPieces;
      const int at = k + c * (16 / static_cast<int>(sizeof(X)));
      fill_piece<X>(xs + r * (kXPieces * 16) + ((c ^ (r & 7)) << 4), xrow[i] ? xrow[i] : static_cast<const X*>(p.x), at,
                    xrow[i] ? k1 - at : 0, align);
    }
#pragma unroll
    for (int i = 0; i < kATurns; ++i) {
      const int piece = tid + 128 * i, j = piece >> 3, c = piece & 7;
      const int at = k + c * 8;
      fill_piece<W>(as + j * 128 + ((c ^ (j & 7)) << 4), arow[i] ? arow[i] : static_cast<const W*>(p.a), at,
                    arow[i] ? k1 - at : 0, align);
    }
  };
  const int steps = (k1 - k0 + kDownDepth - 1) / kDownDepth;
#pragma unroll
  for (int s = 0; s < kDownStages - 1; ++s) {
    if (s < steps) fill(s, k0 + s * kDownDepth);
    cp_async_commit();
  }
  // The tensor cores drop the low bits of a running sum, so it is handed over after every kDownPiece stages (16
  // instructions that add to it) to one in f32.  8192 rows of bf16, k 4096 in three parts: 1e-6 off
  // float64 in one sum, 2.9e-7 so; 777 rows of f32, k 1501: 7.9e-7 handed over every four stages, 2.3e-7 every one.
  constexpr int kDownPiece = sizeof(X) == 4 ? 1 : 4;
  float acc[kRanks / 8][4], sum[kRanks / 8][4];
#pragma unroll
  for (int j = 0; j < kRanks / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = sum[j][e] = 0.0f;

  for (int s = 0; s < steps; ++s) {
    if (s > 0 && s % kDownPiece == 0) {
#pragma unroll
      for (int j = 0; j < kRanks / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum[j][e] += acc[j][e];
          acc[j][e] = 0.0f;
        }
    }
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
  float any = 0.0f;  // NaN where one of this thread's is
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + (lane >> 2) + 8 * h;
    if (r >= tile.z) continue;
#pragma unroll
    for (int j = 0; j < kRanks / 8; ++j) {
      const int at = rank0 + j * 8 + 2 * (lane & 3);
      const float2 v = make_float2(sum[j][2 * h] + acc[j][2 * h], sum[j][2 * h + 1] + acc[j][2 * h + 1]);
      if (at < t.rank_pad) *reinterpret_cast<float2*>(u + static_cast<int64_t>(r) * t.rank_pad + at) = v;
      any += v.x + v.y;
    }
  }
  if constexpr (sizeof(X) == 4) {
    if (any != any) {
      // (this thread's own stores, read back)
#pragma unroll 1
      for (int at = 0; at < kRanks / 2; ++at) {
        const int r = warp * 16 + (lane >> 2) + 8 * (at & 1), e = rank0 + (at >> 2) * 8 + 2 * (lane & 3) + (at >> 1 & 1);
        if (r >= tile.z || e >= p.rank) continue;
        const float v = u[static_cast<int64_t>(r) * t.rank_pad + e];
        if (v != v) whole_part<W>(t, r, e);
      }
    }
  }
}

// u in the up kernel, as 16-bit numbers that the tensor cores multiply with B as it is: three bf16 terms
// (24 bits), or two f16 terms (22 bits) of a row scaled by a power of two that brings its largest
// element to [2^14, 2^15) (f16's range would be too small for the row as it is; what is lost below its
// smallest number is 2^-40 of the largest).
template <typename W>
struct UpTerms;
template <>
struct UpTerms<__nv_bfloat16> {
  static constexpr int kCount = 3;
};
template <>
struct UpTerms<__half> {
  static constexpr int kCount = 2;
};
// The next term of v, which is left with the rest.
__device__ __forceinline__ __nv_bfloat16 take_term(float& v, __nv_bfloat16) {
  const __nv_bfloat16 h = __float2bfloat16(v);
  v -= __bfloat162float(h);
  if (!(fabsf(v) < INFINITY)) v = 0.0f;  // (of an infinity or NaN the first term keeps it)
  return h;
}
__device__ __forceinline__ __half take_term(float& v, __half) {
  const __half h = __float2half(v);
  v -= __half2float(h);
  if (!(fabsf(v) < INFINITY)) v = 0.0f;
  return h;
}

// Steps in the ring: three, two where u's terms leave no room for three.
__host__ __device__ inline int up_stages(int rank_pad) { return rank_pad <= 128 ? 3 : 2; }
constexpr int kUpCWords = kUpCols + 8;  // words from one row of C to the next in shared memory (8 modulo 32)
// Shared memory of the up kernel: u's terms, 64 rows each; per stage 64 rows of B and 64 rows of C; the
// rows' scales.  Rows of u and B are rank_pad + 8 elements of 16 bits apart: ldmatrix, and the
// reads of C by fragment, meet every bank once.
__host__ __device__ inline int up_stage_bytes(int rank_pad) { return kUpCols * (rank_pad + 8) * 2 + kPlanTileRows * kUpCWords * 4; }
__host__ __device__ inline int up_smem_bytes(int rank_pad, int terms) {
  return terms * kPlanTileRows * (rank_pad + 8) * 2 + up_stages(rank_pad) * up_stage_bytes(rank_pad) + kPlanTileRows * 4;
}

// As whole_part, of the second product: column col of scale * u B^T for row r of this CTA's tile.
template <typename W>
__device__ __forceinline__ float whole_product(const AdapterTileParams& t, int r, int col) {
  const AdapterParams& p = t.a;
  const int4 tile = t.tiles[blockIdx.y];
  const float scale = p.scales != nullptr ? p.scales[tile.x] : 1.0f;
  const W* b = static_cast<const W*>(p.b) + tile.x * p.b_stride + col * p.ldb;
  float y = 0.0f;
#pragma unroll 1
  for (int j = 0; j < p.rank && y == y; ++j) {
    float u = 0.0f;
#pragma unroll 1
    for (int s = 0; s < t.splits; ++s) u += t.u[(static_cast<int64_t>(s) * p.m + tile.y + r) * t.rank_pad + j];
    y = __fmaf_rn(u * scale, to_f32<W>(b[j]), y);
  }
  return y;
}

// D = C + u B^T for tile blockIdx.y and t.up_cols columns from blockIdx.x * t.up_cols on, 64 at a time;
// 256 threads, a warp for 16 rows x 32 columns of a step.  The time is that of the traffic, C in and D
// out, so B and C come through a ring in shared memory, a step or two ahead.  (C one step ahead in
// registers, with three CTAs per SM: 8192 rows, rank 64, n 4096 97 us.)
// Rows without an adapter make up tiles of their own, of which D is C.
// kWhole: 16-byte aligned rows of B, C and D, whole steps of 64 columns and ranks in eights, so nothing
// needs a check: a step is 400 instructions of a warp with them, 200 without (85 / 70 us of the above).
template <typename W, int kUpStages, bool kWhole>
__global__ void __launch_bounds__(256, 2) adapter_up_kernel(const __grid_constant__ AdapterTileParams t) {
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
  const int row0 = (warp >> 1) * 16, half = (warp & 1) * 32;
  const int first = static_cast<int>(blockIdx.x) * t.up_cols, last = min(first + t.up_cols, p.n);

  // The rows whose C this thread copies in and whose D it copies out, four columns of 64 each (rows that
  // do not exist are read as the tile's last).
  const bool wide_d = kWhole || p.align_d == 16;
  const float* c_from[4];
  float* d_to[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = t.order[tile.y + min((tid >> 4) + 16 * j, tile.z - 1)];
    c_from[j] = p.c + row * p.ldc + first + (tid & 15) * 4;
    d_to[j] = p.d + row * p.ldd + first + (tid & 15) * 4;
  }
  constexpr int kTerms = UpTerms<W>::kCount;
  const int ld = t.rank_pad + 8, pieces = t.rank_pad / 8;
  W* us = reinterpret_cast<W*>(up_smem);
  const uint32_t us0 = smem_u32(up_smem), ring0 = us0 + kTerms * kPlanTileRows * ld * 2;
  const uint32_t stage_bytes = static_cast<uint32_t>(up_stage_bytes(t.rank_pad)), c_off = static_cast<uint32_t>(kUpCols * ld * 2);
  float* row_scale = reinterpret_cast<float*>(up_smem + kTerms * kPlanTileRows * ld * 2 + kUpStages * stage_bytes);
  // B: four threads to a row
  const W* b_from = static_cast<const W*>(p.b) + (has ? tile.x * p.b_stride : 0) + (first + (tid >> 2)) * p.ldb;
  const uint32_t c_to = c_off + ((tid >> 4) * kUpCWords + (tid & 15) * 4) * 4, b_to = (tid >> 2) * ld * 2;
  // (called for one step after another: the pointers move on)
  auto fill = [&](int col0, int stage) {
    const uint32_t to = ring0 + stage * stage_bytes;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t dst = to + c_to + 16 * j * kUpCWords * 4;
      if constexpr (kWhole) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(c_from[j]) : "memory");
      } else {
        fill_piece<float>(dst, c_from[j], 0, p.n - col0 - (tid & 15) * 4, p.align_c);
      }
      c_from[j] += kUpCols;
    }
    if (has) {
      if constexpr (kWhole) {
        for (int piece = tid & 3; piece < pieces; piece += 4)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + b_to + piece * 16),
                       "l"(b_from + (piece * 8 < p.rank ? piece * 8 : 0)), "r"(piece * 8 < p.rank ? 16 : 0)
                       : "memory");
      } else {
        const bool in = col0 + (tid >> 2) < p.n;
        for (int piece = tid & 3; piece < pieces; piece += 4)
          fill_piece<W>(to + b_to + piece * 16, in ? b_from : static_cast<const W*>(p.b), piece * 8,
                        in ? p.rank - piece * 8 : 0, p.align_r);
      }
      b_from += kUpCols * p.ldb;
    }
  };
#pragma unroll
  for (int s = 0; s < kUpStages - 1; ++s) {
    if (first + s * kUpCols < last) fill(first + s * kUpCols, s);
    cp_async_commit();
  }
  if (has) {
    const float scale = p.scales != nullptr ? p.scales[tile.x] : 1.0f;
    const int r = tid >> 2;  // four threads to a row
    // elements e .. e + 3 of this thread's row: the parts of k in ascending order, four of them on their
    // way at a time (one after another they took a third of a CTA's time)
    auto sum_at = [&](int e) {
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < tile.z) {
        const float* from = t.u + static_cast<int64_t>(tile.y + r) * t.rank_pad + e;
        const int64_t step = static_cast<int64_t>(p.m) * t.rank_pad;
        for (int s0 = 0; s0 < t.splits; s0 += 4) {
          float4 v[4];
#pragma unroll
          for (int s = 0; s < 4; ++s)
            v[s] = s0 + s < t.splits ? *reinterpret_cast<const float4*>(from + (s0 + s) * step) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            if (s0 + s >= t.splits) break;
            sum.x += v[s].x;
            sum.y += v[s].y;
            sum.z += v[s].z;
            sum.w += v[s].w;
          }
        }
      }
      return make_float4(sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale);
    };
    float grow = 1.0f;
    if constexpr (std::is_same<W, __half>::value) {
      float top = 0.0f;
      for (int e = (tid & 3) * 4; e < t.rank_pad; e += 16) {
        const float4 v = sum_at(e);
        top = fmaxf(fmaxf(fmaxf(top, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // top's exponent field, kept where both powers of two are normal numbers (127 for an infinity)
      const int field = static_cast<int>(__float_as_uint(top) >> 23);
      const int at = field == 255 ? 141 : max(field, 15);
      grow = __uint_as_float(static_cast<uint32_t>(268 - at) << 23);             // 2^(141 - at)
      if ((tid & 3) == 0) row_scale[r] = __uint_as_float(static_cast<uint32_t>(at - 14) << 23);  // 2^(at - 141)
    }
#pragma unroll 4
    for (int e = (tid & 3) * 4; e < t.rank_pad; e += 16) {
      const float4 sum = sum_at(e);
      float v[4] = {sum.x * grow, sum.y * grow, sum.z * grow, sum.w * grow};
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
        __align__(8) W w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = take_term(v[j], W());
        *reinterpret_cast<uint2*>(us + (term * kPlanTileRows + r) * ld + e) = *reinterpret_cast<const uint2*>(w);
      }
    }
  }
  const uint32_t a_at = us0 + ((row0 + (lane & 15)) * ld + (lane >> 4) * 8) * 2;
  const uint32_t b_at = ((half + (lane & 7) + ((lane >> 4) << 3)) * ld + ((lane >> 3) & 1) * 8) * 2;
  const uint32_t c_at = c_off + ((row0 + g) * kUpCWords + half + 2 * i) * 4;
  int stage = 0;
  for (int col0 = first; col0 < last; col0 += kUpCols) {
    cp_async_wait<kUpStages - 2>();
    __syncthreads();  // this step's B and C (and u) are in place; everyone is done with the stage filled next
    if (const int ahead = col0 + (kUpStages - 1) * kUpCols; ahead < last)
      fill(ahead, stage == 0 ? kUpStages - 1 : stage - 1);
    cp_async_commit();
    const uint32_t at = ring0 + stage * stage_bytes;
    float acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
    if (has) {
      for (int kk = 0; kk < pieces / 2; ++kk) {
        uint32_t b[2][4];  // 16 elements of k x 32 columns
        ldmatrix_x4(b[0], at + b_at + kk * 32);
        ldmatrix_x4(b[1], at + b_at + 16 * ld * 2 + kk * 32);
#pragma unroll
        for (int term = kTerms - 1; term >= 0; --term) {
          uint32_t a[4];
          ldmatrix_x4(a, a_at + term * kPlanTileRows * ld * 2 + kk * 32);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_f16(acc[j], a, b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1], W());
        }
      }
      if constexpr (std::is_same<W, __half>::value) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] *= row_scale[row0 + g + 8 * (e >> 1)];
      }
    }
    // D takes C's place in the stage (a row without an adapter is C itself: no zero is added to it) ...
    if (has) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t place = at + c_at + (8 * h * kUpCWords + j * 8) * 4;
          float2 y;
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(y.x), "=f"(y.y) : "r"(place));
          y.x += acc[j][2 * h];
          y.y += acc[j][2 * h + 1];
          asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(place), "f"(y.x), "f"(y.y) : "memory");
        }
      }
    }
    __syncthreads();
    // ... and leaves it row by row, 256 bytes at a time
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float4 y;
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w)
                   : "r"(at + c_to + 16 * j * kUpCWords * 4));
      if ((tid >> 4) + 16 * j < tile.z) {
        const float any = y.x + y.y + y.z + y.w;  // (NaN where one of them is)
        if (any != any && has) {
#pragma unroll 1
          for (int e = 0; e < 4; ++e) {
            const float v = e == 0 ? y.x : e == 1 ? y.y : e == 2 ? y.z : y.w;
            const int r = (tid >> 4) + 16 * j, col = col0 + (tid & 15) * 4 + e;
            if (v == v || col >= p.n) continue;
            // (of a D that is C this thread alone writes the element, below)
            const float made = p.c[t.order[tile.y + r] * p.ldc + col] + whole_product<W>(t, r, col);
            y = make_float4(e == 0 ? made : y.x, e == 1 ? made : y.y, e == 2 ? made : y.z, e == 3 ? made : y.w);
          }
        }
        const int left = kWhole ? 4 : p.n - col0 - (tid & 15) * 4;  // columns from here on
        if (wide_d && left >= 4) {
          *reinterpret_cast<float4*>(d_to[j]) = y;
        } else {
          if (left > 0) d_to[j][0] = y.x;
          if (left > 1) d_to[j][1] = y.y;
          if (left > 2) d_to[j][2] = y.z;
          if (left > 3) d_to[j][3] = y.w;
        }
      }
      d_to[j] += kUpCols;
    }
    if (++stage == kUpStages) stage = 0;
  }
  cp_async_wait<0>();
}

}  // namespace b200
