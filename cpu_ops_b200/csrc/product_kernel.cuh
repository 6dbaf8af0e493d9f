// Products of 16-bit matrices with bias, activation and residual in the epilogue:
//     z = alpha A B + bias,   D = act(z) + beta C,   Z = z if asked for
// f16 or bf16 operands, each by rows or by columns, f32 accumulators in tensor memory
// (tcgen05.mma kind::f16), D and C f32 or of the operands' type.
//
// Roles are those of gemm_tcgen05_kernel: two TMA producer warps that take alternate k-blocks of 64
// elements (128-byte swizzled rows), one MMA issuer, the other warps drain the accumulators.
//   K-major operand: rows of 64 k; 8-row groups 1024 bytes apart.
//   MN-major operand: boxes of 64 m (n) x 64 k, whose 128-byte rows run along m (n): 8 k are 1024
//   bytes, the next 64 of m (n) 8192 bytes further on.
// Every wait is bounded, as there.
#pragma once

#include "dense_params.h"
#include "dense_types.cuh"
#include "exchange.h"
#include "gemm_params.h"
#include "ptx_sm100.cuh"
#include "ptx_sm100_pair.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200 {

constexpr int kProductThreads = 96 + 32 * kProductEpiWarps;
constexpr uint32_t kTmemCols512 = 512;

__device__ __forceinline__ void product_error(const ProductParams& p, volatile int* abort_flag, int code) {
  leave_error(p.error, code);
  *abort_flag = 1;
  __threadfence_block();
}

// Hands an accumulator back to the pair's leader.  Its reads are complete (tcgen05.wait::ld), nothing else is published:
// with release semantics the arrival waits for the thread's stores, which took 1000 to 2500 cycles (8192 x 4096 x 1024
// 53 us, 49 in this form; with gelu, Z and C 91 and 80).
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <bool kPair>
__device__ __forceinline__ void mma_f16_g(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                          uint32_t idesc, uint32_t accumulate, uint32_t issue) {
  if constexpr (kPair) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t"
        "}\n"
        :
        : "r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
  } else {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
        "}\n"
        :
        : "r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
  }
}

struct ProductTile {
  int m_tile, n_tile, kb0, nkb;
};

// Tiles are walked in groups of raster_m m-tiles (m fastest), as decode_tile does.  kProductParts: part
// `part` of balanced contiguous ranges of k-blocks.
__device__ __forceinline__ ProductTile product_tile(const ProductParams& p, int t, int part) {
  ProductTile c;
  const int per_group = p.raster_m * p.n_tiles, g = t / per_group, first_m = g * p.raster_m;
  const int gsize = min(p.raster_m, p.m_tiles - first_m), in = t - g * per_group;
  c.m_tile = first_m + in % gsize;
  c.n_tile = in / gsize;
  const int base = p.k_blocks / p.parts, rem = p.k_blocks % p.parts;
  c.kb0 = part * base + min(part, rem);
  c.nkb = base + (part < rem ? 1 : 0);
  return c;
}

__device__ __forceinline__ float load_as_f32(const void* base, int64_t i, int type) {
  if (type == kF32) return static_cast<const float*>(base)[i];
  if (type == kF16) return __half2float(static_cast<const __half*>(base)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
}
// (one rounding, to nearest even; a value beyond f16's range becomes an infinity)
__device__ __forceinline__ void store_from_f32(void* base, int64_t i, int type, float v) {
  if (type == kF32) {
    static_cast<float*>(base)[i] = v;
  } else if (type == kF16) {
    static_cast<__half*>(base)[i] = __float2half_rn(v);
  } else {
    static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  }
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, int type) {
  if (type == kF16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, int type) {
  if (type == kF16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// A lane's row of a 32 x 32 chunk in shared memory as TMA lays it out: rows of 128 bytes (f32), 16-byte
// pieces XOR-swizzled by row & 7; or of 64 bytes, by (row >> 1) & 3.
__device__ __forceinline__ void put_chunk_row(uint32_t buf, int lane, const uint32_t (&r)[32], int type) {
  if (type == kF32) {
    const uint32_t row = buf + static_cast<uint32_t>(lane) * 128u;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + (static_cast<uint32_t>(j ^ (lane & 7)) << 4)),
                   "r"(r[4 * j]), "r"(r[4 * j + 1]), "r"(r[4 * j + 2]), "r"(r[4 * j + 3])
                   : "memory");
  } else {
    const uint32_t row = buf + static_cast<uint32_t>(lane) * 64u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2(__uint_as_float(r[8 * j + 2 * i]), __uint_as_float(r[8 * j + 2 * i + 1]), type);
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + (static_cast<uint32_t>(j ^ ((lane >> 1) & 3)) << 4)),
                   "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                   : "memory");
    }
  }
}
// r += beta * the lane's row of C.
__device__ __forceinline__ void add_chunk_row(uint32_t buf, int lane, uint32_t (&r)[32], float beta, int type) {
  if (type == kF32) {
    const uint32_t row = buf + static_cast<uint32_t>(lane) * 128u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float c[4];
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                   : "r"(row + (static_cast<uint32_t>(j ^ (lane & 7)) << 4)));
#pragma unroll
      for (int i = 0; i < 4; ++i) r[4 * j + i] = __float_as_uint(__fmaf_rn(beta, c[i], __uint_as_float(r[4 * j + i])));
    }
  } else {
    const uint32_t row = buf + static_cast<uint32_t>(lane) * 64u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "r"(row + (static_cast<uint32_t>(j ^ ((lane >> 1) & 3)) << 4)));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 c = unpack2(w[i], type);
        r[8 * j + 2 * i] = __float_as_uint(__fmaf_rn(beta, c.x, __uint_as_float(r[8 * j + 2 * i])));
        r[8 * j + 2 * i + 1] = __float_as_uint(__fmaf_rn(beta, c.y, __uint_as_float(r[8 * j + 2 * i + 1])));
      }
    }
  }
}

// z / (1 + exp(-v)) from one exp2 and one reciprocal, both within 2 ulp: 3e-7 of z.  (silu_f32 and gelu_f32, to the last
// bit, take some 90 instructions an element: 8192 x 4096 x 1024 with gelu and Z 88 us, 49 in this form.)  Where
// exp(-v) overflows the quotient is 0 (of -inf: NaN).
__device__ __forceinline__ float times_logistic(float z, float v) {
  float t, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + t));
  return z * r;
}
// The tanh form: 0.5 z (1 + tanh(u)) = z / (1 + exp(-2 u)).
__device__ __forceinline__ float gelu_fast(float z) {
  constexpr float c = 2.0f * 0.7978845608028654f;
  return times_logistic(z, z * __fmaf_rn(c * 0.044715f, z * z, c));
}
__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case kOpRelu: return z < 0.0f ? 0.0f : z;
    case kOpGelu: return gelu_fast(z);
    case kOpSilu: return times_logistic(z, z);
    default: return z;
  }
}

// z of a chunk: alpha acc + bias by column (`bias`: 32 floats of shared memory, or null).
__device__ __forceinline__ void product_z(float alpha, const float* bias, uint32_t (&r)[32]) {
  if (bias == nullptr) {
    if (alpha != 1.0f) {
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(alpha * __uint_as_float(r[i]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(bias + i);
    r[i] = __float_as_uint(__fmaf_rn(alpha, __uint_as_float(r[i]), v.x));
    r[i + 1] = __float_as_uint(__fmaf_rn(alpha, __uint_as_float(r[i + 1]), v.y));
    r[i + 2] = __float_as_uint(__fmaf_rn(alpha, __uint_as_float(r[i + 2]), v.z));
    r[i + 3] = __float_as_uint(__fmaf_rn(alpha, __uint_as_float(r[i + 3]), v.w));
  }
}
__device__ __forceinline__ void activate_chunk(uint32_t (&r)[32], int act) {
  if (act == kOpRelu) {
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __uint_as_float(r[i]) < 0.0f ? 0u : r[i];
  } else if (act == kOpGelu) {
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(gelu_fast(__uint_as_float(r[i])));
  } else if (act == kOpSilu) {
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(times_logistic(__uint_as_float(r[i]), __uint_as_float(r[i])));
  }
}

// Where C, D or Z cannot be addressed by TMA: a chunk's f32 values (in shared memory, put there by
// put_chunk_row) leave row by row, lane = column, and C is read the same way, all of a chunk's rows at once.
// Asks for a chunk's C ahead of its use, a row per lane.
__device__ __forceinline__ void prefetch_c_rows(const ProductParams& p, int row0, int col0, int lane) {
  if (row0 + lane >= p.Mk || col0 >= p.Nk) return;
  const char* at = static_cast<const char*>(p.C) + (static_cast<int64_t>(row0 + lane) * p.ldc + col0) * type_bytes(p.c_type);
  asm volatile("prefetch.global.L1 [%0];" ::"l"(at));
}
template <int kRows>
__device__ __forceinline__ void load_c_rows(const ProductParams& p, int row0, int col0, int lane, float (&c)[kRows]) {
  const int nrows = lane < p.Nk - col0 ? p.Mk - row0 : 0;
  const int64_t at = static_cast<int64_t>(row0) * p.ldc + col0 + lane;
  auto rows = [&](auto* base) {
    base += at;
#pragma unroll
    for (int r = 0; r < kRows; ++r, base += p.ldc) c[r] = r < nrows ? to_f32(*base) : 0.0f;
  };
  if (p.c_type == kF32) {
    rows(static_cast<const float*>(p.C));
  } else if (p.c_type == kF16) {
    rows(static_cast<const __half*>(p.C));
  } else {
    rows(static_cast<const __nv_bfloat16*>(p.C));
  }
}
// An f32 C's chunk into shared memory, rows of 128 bytes, without registers in between; one group of copies.
__device__ __forceinline__ void fetch_c_rows(const ProductParams& p, uint32_t buf, int row0, int col0, int lane) {
  const int nrows = lane < p.Nk - col0 ? p.Mk - row0 : 0;
  const float* src = static_cast<const float*>(p.C) + (static_cast<int64_t>(row0) * p.ldc + col0 + lane);
#pragma unroll 8
  for (int r = 0; r < 32; ++r, src += p.ldc) {
    const bool valid = r < nrows;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(buf + static_cast<uint32_t>(r * 128 + lane * 4)),
                 "l"(valid ? src : static_cast<const float*>(p.C)), "r"(valid ? 4 : 0)
                 : "memory");
  }
  cp_async_commit();
}
// Rows r0 .. r0 + kRows of the chunk whose first row and column are row0 and col0; C (add_c) from c, or from shared memory
// (c_buf: fetch_c_rows').
template <int kRows>
__device__ __forceinline__ void write_chunk_rows(const ProductParams& p, uint32_t buf, void* dst, int64_t ld, bool add_c,
                                                 const float (&c)[kRows], uint32_t c_buf, int r0, int row0, int col0, int lane) {
  const int nrows = lane < p.Nk - col0 ? p.Mk - row0 - r0 : 0;
  const int64_t at = static_cast<int64_t>(row0 + r0) * ld + col0 + lane;
  auto rows = [&](auto* base) {
    using T = std::remove_pointer_t<decltype(base)>;
    base += at;
    constexpr int kAtOnce = kRows < 8 ? kRows : 8;
#pragma unroll
    for (int i0 = 0; i0 < kRows; i0 += kAtOnce) {
      float v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int r = r0 + i0 + i;
        asm volatile("ld.shared.f32 %0, [%1];"
                     : "=f"(v[i])
                     : "r"(buf + static_cast<uint32_t>(r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4)));
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i, base += ld) {
        if (add_c) {
          float x = c[i0 + i];
          if (c_buf) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(c_buf + static_cast<uint32_t>((r0 + i0 + i) * 128 + lane * 4)));
          v[i] = __fmaf_rn(p.beta, x, v[i]);
        }
        if (i0 + i < nrows) *base = from_f32<T>(v[i]);
      }
    }
  };
  if (p.d_type == kF32) {
    rows(static_cast<float*>(dst));
  } else if (p.d_type == kF16) {
    rows(static_cast<__half*>(dst));
  } else {
    rows(static_cast<__nv_bfloat16*>(dst));
  }
}

// A lane's row of a chunk, straight to global memory.
__device__ __forceinline__ void store_lane_row(void* dst, int64_t ld, int row, int col0, int ncols, const uint32_t (&r)[32], int type) {
  const int64_t at = static_cast<int64_t>(row) * ld + col0;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < ncols) store_from_f32(dst, at + i, type, __uint_as_float(r[i]));
}

// The owner's part of kProductParts' epilogue: its columns' sums, [part][column][row] from `base`, `slab` bytes a
// part.  A warp takes 32 rows and kCols columns at a time, a lane a row, so that shared memory is read without
// conflicts; where rows are contiguous in D (swapped) a warp's stores are whole lines, otherwise a lane's eight
// columns leave as one or two 16-byte stores where D's rows allow it.
template <typename T, typename TC, int kCols>
__device__ __forceinline__ void finish_columns(const ProductParams& p, uint32_t base, uint32_t slab, const float* bias, int row, int col,
                                               int kr, int kc, int ncols) {
  float v[kCols], c[kCols];
  const int64_t i = p.swapped ? kc : kr, j = p.swapped ? kr : kc;  // the caller's row and column of the first element
  if (p.C) {
    const TC* from = static_cast<const TC*>(p.C) + (i * p.ldc + j);
    const int64_t step = p.swapped ? p.ldc : 1;
#pragma unroll
    for (int u = 0; u < kCols; ++u) c[u] = u < ncols ? to_f32(from[u * step]) : 0.0f;
  }
  const uint32_t at = base + static_cast<uint32_t>((col * kTileM + row) * 4);
#pragma unroll
  for (int u = 0; u < kCols; ++u) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[u]) : "r"(at + 512u * u));
  for (int s = 1; s < p.parts; ++s) {
    float x[kCols];
#pragma unroll
    for (int u = 0; u < kCols; ++u) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x[u]) : "r"(at + static_cast<uint32_t>(s) * slab + 512u * u));
#pragma unroll
    for (int u = 0; u < kCols; ++u) v[u] += x[u];
  }
  if (p.bias) {
#pragma unroll
    for (int u = 0; u < kCols; ++u) v[u] = __fmaf_rn(p.alpha, v[u], bias[p.swapped ? row : col + u]);
  } else {
#pragma unroll
    for (int u = 0; u < kCols; ++u) v[u] *= p.alpha;
  }
  auto store = [&](void* matrix, int64_t ld) {
    T* to = static_cast<T*>(matrix) + (i * ld + j);
    if constexpr (kCols == 8) {
      if (!p.swapped && ncols >= 8 && (reinterpret_cast<uintptr_t>(to) & 15u) == 0) {
        uint4* out = reinterpret_cast<uint4*>(to);
        if constexpr (std::is_same<T, float>::value) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            out[h] = make_uint4(__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3]));
        } else {
          constexpr int type = std::is_same<T, __half>::value ? kF16 : kBf16;
          *out = make_uint4(pack2(v[0], v[1], type), pack2(v[2], v[3], type), pack2(v[4], v[5], type), pack2(v[6], v[7], type));
        }
        return;
      }
    }
    const int64_t step = p.swapped ? ld : 1;
#pragma unroll
    for (int u = 0; u < kCols; ++u)
      if (u < ncols) to[u * step] = from_f32<T>(v[u]);
  };
  if (p.Z) store(p.Z, p.ldz);
  if (p.act == kOpRelu) {
#pragma unroll
    for (int u = 0; u < kCols; ++u) v[u] = v[u] < 0.0f ? 0.0f : v[u];
  } else if (p.act == kOpGelu) {
#pragma unroll
    for (int u = 0; u < kCols; ++u) v[u] = gelu_fast(v[u]);
  } else if (p.act == kOpSilu) {
#pragma unroll
    for (int u = 0; u < kCols; ++u) v[u] = times_logistic(v[u], v[u]);
  }
  if (p.C) {
#pragma unroll
    for (int u = 0; u < kCols; ++u) v[u] = __fmaf_rn(p.beta, c[u], v[u]);
  }
  store(p.D, p.ldd);
}
// leave_exchange's view of a cluster: a warp of one of its `parts` CTAs.
struct PartsCluster {
  volatile int* late;  // this CTA's word, which any CTA sets
  uint32_t received;   // its barrier
  int parts, lane;
  __device__ __forceinline__ void tell_late() {
    if (lane < parts)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_cta(smem_u32(const_cast<int*>(late)), static_cast<uint32_t>(lane))), "r"(1)
                   : "memory");
  }
  __device__ __forceinline__ void barrier() {
    __syncwarp();
    cluster_sync_all();
  }
  __device__ __forceinline__ bool any_late() { return *late != 0; }
  __device__ __forceinline__ void wait_for_copies() { mbar_drain(received, 0); }
};

// By warp `warp` of `warps`, all of them on one CTA's columns.
__device__ __forceinline__ void finish_parts(const ProductParams& p, uint32_t base, uint32_t slab, const float* bias, int warp, int warps,
                                             int lane, int tile, int part) {
  const int own = p.BN / p.parts;
  const ProductTile tc = product_tile(p, tile, part);
  const int row0 = tc.m_tile * p.tile_rows, col0 = tc.n_tile * p.BN + part * own;
  const int nrows = min(p.tile_rows, p.Mk - row0), ncols = min(own, p.Nk - col0);  // (ncols may be negative)
  auto finish = [&](auto type, auto c_type, auto cols) {
    constexpr int kCols = decltype(cols)::value;
    for (int item = warp; item < 4 * (own / kCols); item += warps) {
      const int row = (item & 3) * 32 + lane, col = (item >> 2) * kCols;
      if (row < nrows && col < ncols)
        finish_columns<decltype(type), decltype(c_type), kCols>(p, base, slab, bias, row, col, row0 + row, col0 + col, ncols - col);
    }
  };
  auto with_cols = [&](auto type, auto c_type) {
    if (own >= 8) {
      finish(type, c_type, std::integral_constant<int, 8>{});
    } else {
      finish(type, c_type, std::integral_constant<int, 2>{});
    }
  };
  // (C is f32 or of the operands' type, as D is)
  const bool c_f32 = p.c_type == kF32;
  if (p.type == kF16) {
    if (p.d_type == kF32) {
      if (c_f32) with_cols(0.0f, 0.0f); else with_cols(0.0f, __half{});
    } else {
      if (c_f32) with_cols(__half{}, 0.0f); else with_cols(__half{}, __half{});
    }
  } else {
    if (p.d_type == kF32) {
      if (c_f32) with_cols(0.0f, 0.0f); else with_cols(0.0f, __nv_bfloat16{});
    } else {
      if (c_f32) with_cols(__nv_bfloat16{}, 0.0f); else with_cols(__nv_bfloat16{}, __nv_bfloat16{});
    }
  }
}

// kProductPairs: clusters of two CTAs compute 256-row tiles with the cta_group::2 instructions; each CTA
// stages its own 128 rows of A and its half of B's BN rows, and drains its own 128 rows of the accumulator.
//
// kProductParts: few tiles.  The CTAs of a cluster take a part of k each; then each of them owns an equal
// share of the tile's columns, of which all CTAs send it their sums by bulk copies between shared memories, and adds
// them in the order of k.  No workspace, no second launch, and the same result on every run.  (Stored element by element
// into the owner's memory, a warp's store took some 65 cycles: 256 x 4096 x 4096 in two parts 35 us.)
//
// kPieces: the accumulator is taken down every p.piece_blocks k-blocks and the pieces added in f32 registers.  The tensor cores
// drop the low bits of a running sum, towards zero.  Against float64, with operands of both signs, it is off by 1e-9 of the
// result's norm per element of k (2.1e-6 at k = 2048); where all products have one sign by 6.5e-9 of the result (5.4e-5 at 8192,
// 4.3e-4 at 65536: what an instruction drops, of 16 elements, goes with the sum so far, at most 2^-22 of it).  An f32 D is
// summed in pieces of 512: 7e-7 of the norm up to k = 65536 and 1.0e-6 at 2^20, 2.8e-6 of one sign.  A 16-bit D's running sums end
// where the loss reaches half of the least half step of its rounding (2^-12 of the value for f16, 2^-9 for bf16): after 16384
// elements, 131072 of bf16; longer ones are summed in pieces of 8192, which drop 6e-5 at most.
//
// kTma: C, D and Z pass through shared memory by TMA.  Instances of their own, because next to the pieces' 128 sums either
// path's registers are at the other's expense (bytes of spill stores of a thread: 680 with both, 204 with TMA alone, 556 without
// TMA).  (kProductParts: true.)
template <int kForm, bool kPieces, bool kTma>
__global__ void __launch_bounds__(kForm == kProductParts ? 224 : kProductThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmD,
                   const __grid_constant__ CUtensorMap tmZ, const ProductParams p) {
  constexpr bool kPair = kForm == kProductPairs, kParts = kForm == kProductParts;
  constexpr int kCtas = kPair ? 2 : 1;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t cta_rank = kForm == kProductTiles ? 0u : cluster_cta_rank();
  const bool leader = !kPair || cta_rank == 0;
  const int part = kParts ? static_cast<int>(cta_rank) : 0;
  const int work0 = static_cast<int>(blockIdx.x) / (kParts ? p.parts : kCtas);
  const int total_tiles = p.m_tiles * p.n_tiles;
  const int work_step = kParts ? total_tiles : static_cast<int>(gridDim.x) / kCtas;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = ((raw_addr + 1023u) & ~1023u) - raw_addr;
  uint8_t* smem = smem_raw + pad;
  const uint32_t smem_base = raw_addr + pad;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t budget_ns = static_cast<uint64_t>(p.wait_budget_us) * 1000ull;
  const int stages = p.stages, b_rows = p.BN / kCtas;
  const int stage_bytes = (kTileM + b_rows) * 128, tile_rows = kParts ? p.tile_rows : kTileM;
  const uint32_t ring_base = smem_base + static_cast<uint32_t>(stages * stage_bytes);
  const int n_epi = p.epi_warps, warp_producer2 = 2 + n_epi;
  const uint32_t bar_base = ring_base + static_cast<uint32_t>(n_epi * p.ring_bytes);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kProductMaxStages + s); };
  auto acc_full_bar = [&](int b) { return bar_base + 8u * (2 * kProductMaxStages + b); };
  auto acc_empty_bar = [&](int b) { return bar_base + 8u * (2 * kProductMaxStages + 2 + b); };
  const uint32_t drain_bar = bar_base + 8u * (2 * kProductMaxStages + 4);
  auto c_full_bar = [&](int w, int b) { return bar_base + 8u * (2 * kProductMaxStages + 5 + 2 * w + b); };
  constexpr int kRecvBar = 2 * kProductMaxStages + 5 + 2 * kProductEpiWarps, kBarriers = kRecvBar + 1;
  const uint32_t recv_bar = bar_base + 8u * kRecvBar;
  static_assert(8 * kBarriers + 12 <= kProductBarrierBytes, "barriers, tensor memory slot, abort and late flags");
  float* bias_smem = reinterpret_cast<float*>(smem + (bar_base - smem_base) + kProductBarrierBytes);  // a warp's chunks' bias
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (bar_base - smem_base) + 8 * kBarriers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* late_flag = abort_flag + 1;  // kProductParts: some CTA's wait for the parts' sums ran out

  if (warp == 2) {
    for (int i = lane; i < kBarriers; i += 32) {
      const bool acc_empty = i == 2 * kProductMaxStages + 2 || i == 2 * kProductMaxStages + 3;
      mbar_init(bar_base + 8u * static_cast<uint32_t>(i), acc_empty ? static_cast<uint32_t>(n_epi) * kCtas : 1u);
    }
    if (lane == 0) *abort_flag = *late_flag = 0;
    fence_mbar_init_cluster();
    __syncwarp();
    if (kParts && lane == 0) mbar_expect_tx(recv_bar, static_cast<uint32_t>(p.BN * kTileM * 4));  // its columns' sums from all parts
  }
  if (warp == 1) {
    tmem_alloc_g<kPair>(smem_u32(tmem_slot), kTmemCols512);
    tmem_relinquish_g<kPair>();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
    if (!kParts && kTma) {
      prefetch_tensormap(&tmD);
      if (p.C) prefetch_tensormap(&tmC);
      if (p.Z) prefetch_tensormap(&tmZ);
    }
  }
  tc_fence_before_sync();
  if constexpr (kForm != kProductTiles) {
    cluster_sync_all();  // the other CTAs run and their barriers are initialised before anything reaches them
  } else {
    __syncthreads();
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int nacc = p.nacc;

  if (warp == 0 || warp == warp_producer2) {
    // ------------------------------ TMA producers -----------------------------
    const int np = stages >= 4 ? 2 : 1, me = warp == 0 ? 0 : 1;
    if (me < np) {
      const uint32_t el = elect_one() ? 1u : 0u;
      int s = me, g_par = 0;
      uint32_t ph = 0, armed = 0, armed_parity = 0, peek = 0;
      bool ok = true;
      const uint32_t tx_bytes = static_cast<uint32_t>(tile_rows + b_rows) * 128u * kCtas;
      // pair: every load of both CTAs credits the leader's barrier, which the leader arms with the bytes of both
      const uint32_t full0 = kPair ? map_to_cta(full_bar(0), 0) : full_bar(0), empty0 = empty_bar(0);
      const int a_mn = p.a_mn, b_mn = p.b_mn, b_chunks = b_rows / 64;
      asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int t = work0; t < total_tiles && ok; t += work_step) {
        const ProductTile tc = product_tile(p, t, part);
        const int m0 = (tc.m_tile * kCtas + (kPair ? static_cast<int>(cta_rank) : 0)) * tile_rows;
        const int n0 = tc.n_tile * p.BN + (kPair ? static_cast<int>(cta_rank) * b_rows : 0);
        const int i0 = np == 1 ? 0 : ((me ^ g_par) & 1);
        int kx = (tc.kb0 + i0) * 64;
        for (int i = i0; i < tc.nkb; i += np, kx += 64 * np) {
          const uint32_t full_addr = full0 + 8u * s;
          if (!peek && !__all_sync(0xffffffffu, mbar_wait_bounded(empty0 + 8u * s, ph ^ 1u, abort_flag, budget_ns))) {
            if (el) product_error(p, abort_flag, kErrProducerWait);
            ok = false;
            break;
          }
          int sn = s + np;
          uint32_t phn = ph;
          if (sn >= stages) {
            sn -= stages;
            phn ^= 1u;
          }
          const uint32_t probe = mbar_test_wait(empty0 + 8u * sn, phn ^ 1u);
          if (leader) {
            mbar_expect_tx_p(full_bar(s), tx_bytes, el);
            armed |= 1u << s;
            armed_parity = (armed_parity & ~(1u << s)) | (ph << s);
          }
          const uint32_t a_dst = smem_base + static_cast<uint32_t>(s * stage_bytes), b_dst = a_dst + kTileM * 128;
          if (!a_mn) {
            tma_load_2d_g<kPair>(a_dst, &tmA, full_addr, kx, m0, el);
          } else {
            tma_load_2d_g<kPair>(a_dst, &tmA, full_addr, m0, kx, el);
            tma_load_2d_g<kPair>(a_dst + 8192, &tmA, full_addr, m0 + 64, kx, el);
          }
          if (!b_mn) {
            tma_load_2d_g<kPair>(b_dst, &tmB, full_addr, kx, n0, el);
          } else {
            for (int c = 0; c < b_chunks; ++c) tma_load_2d_g<kPair>(b_dst + c * 8192, &tmB, full_addr, n0 + c * 64, kx, el);
          }
          peek = __all_sync(0xffffffffu, probe != 0) ? 1u : 0u;
          s = sn;
          ph = phn;
        }
        g_par = (g_par + tc.nkb) & 1;
      }
      if (*abort_flag != 0 && el) {
        // copies that were already issued land before the CTA exits
        for (int st = 0; st < stages; ++st)
          if (armed & (1u << st)) mbar_drain(full_bar(st), (armed_parity >> st) & 1u);
        if (kPair && !leader) {  // (the peer cannot watch the leader's barriers: time for its copies)
          const uint64_t t_end = global_timer_ns() + 100000;
          while (global_timer_ns() < t_end) __nanosleep(1000);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------- MMA issuer -------------------------------
    if (leader) {
      const uint32_t el = elect_one() ? 1u : 0u;
      constexpr uint32_t kAll = 0xffffffffu;
      bool ok = true;
      const uint64_t a_hi64 = p.a_mn ? make_smem_desc_hi(8192, 1024, 2) : make_smem_desc_hi(16, 1024, 2);
      const uint64_t b_hi64 = p.b_mn ? make_smem_desc_hi(8192, 1024, 2) : make_smem_desc_hi(16, 1024, 2);
      const uint32_t a_hi = static_cast<uint32_t>(a_hi64 >> 32), b_hi = static_cast<uint32_t>(b_hi64 >> 32);
      // (14 address bits: in a cluster the CTA's rank stands above them)
      const uint32_t a_lo0 = static_cast<uint32_t>(a_hi64) | ((smem_base >> 4) & 0x3FFFu);
      const uint32_t b_lo0 = static_cast<uint32_t>(b_hi64) | (((smem_base + kTileM * 128) >> 4) & 0x3FFFu);
      const uint32_t stage_step = static_cast<uint32_t>(stage_bytes) >> 4;
      // descriptor step of 16 k: 32 bytes along a row, or 16 rows of 128 bytes
      const uint32_t a_k = p.a_mn ? 128u : 2u, b_k = p.b_mn ? 128u : 2u;
      const uint32_t idesc = p.idesc, full0 = full_bar(0), empty0 = empty_bar(0);
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0, peek = 0;
      uint32_t a_lo = a_lo0, b_lo = b_lo0, full_addr = full0, empty_addr = empty0;
      asm volatile("griddepcontrol.wait;" ::: "memory");  // (operands come no earlier: the kernel before is not charged to the wait)
      for (int t = work0; t < total_tiles && ok; t += work_step) {
        const ProductTile tc = product_tile(p, t, part);
        int i = 0;
        do {  // one piece of k, or all of it
          if (!__all_sync(kAll, mbar_wait_bounded(acc_empty_bar(buf), acc_ph ^ 1u, abort_flag, budget_ns))) {
            if (el) product_error(p, abort_flag, kErrMmaWaitAcc);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(buf * p.BN);
          uint32_t accumulate = 0;
          const int piece_end = kPieces ? min(i + p.piece_blocks, tc.nkb) : tc.nkb;
          for (; i < piece_end; ++i) {
            if (!peek && !__all_sync(kAll, mbar_wait_bounded(full_addr, ph, abort_flag, budget_ns))) {
              if (el) product_error(p, abort_flag, kErrMmaWaitFull);
              ok = false;
              break;
            }
            const uint32_t nfull = (s + 1 == stages) ? full0 : full_addr + 8;
            const uint32_t nph = (s + 1 == stages) ? (ph ^ 1u) : ph;
            const uint32_t probe = mbar_test_wait(nfull, nph);
            tc_fence_after_sync();
            mma_f16_g<kPair>(d_tmem, a_lo, a_hi, b_lo, b_hi, idesc, accumulate, el);
            mma_f16_g<kPair>(d_tmem, a_lo + a_k, a_hi, b_lo + b_k, b_hi, idesc, 1u, el);
            mma_f16_g<kPair>(d_tmem, a_lo + 2 * a_k, a_hi, b_lo + 2 * b_k, b_hi, idesc, 1u, el);
            mma_f16_g<kPair>(d_tmem, a_lo + 3 * a_k, a_hi, b_lo + 3 * b_k, b_hi, idesc, 1u, el);
            accumulate = 1u;
            tc_commit_both<kPair>(empty_addr, el);
            peek = __all_sync(kAll, probe != 0) ? 1u : 0u;
            if (++s == stages) {
              s = 0;
              ph ^= 1u;
              a_lo = a_lo0;
              b_lo = b_lo0;
              full_addr = full0;
              empty_addr = empty0;
            } else {
              a_lo += stage_step;
              b_lo += stage_step;
              full_addr += 8;
              empty_addr += 8;
            }
          }
          if (ok) tc_commit_both<kPair>(acc_full_bar(buf), el);
          if (++buf == nacc) {
            buf = 0;
            acc_ph ^= 1u;
          }
        } while (kPieces && ok && i < tc.nkb);
      }
      // nothing may still be executing when tensor memory is released
      tc_commit_g<kPair>(drain_bar, el);
      if (!__all_sync(kAll, mbar_drain(drain_bar, 0)) && el)
        product_error(p, abort_flag, kErrDrainWait);
    }
    __syncwarp();
  } else if constexpr (!kParts) {
    // -------------------------------- epilogue --------------------------------
    const int q = warp & 3, ew = warp - 2;
    const int cstep = n_epi >> 2, c0 = ew >> 2;
    // This warp's buffers, p.ring_depth each, for chunks of C, of D and of Z.
    const uint32_t ring = ring_base + static_cast<uint32_t>(ew * p.ring_bytes), depth = static_cast<uint32_t>(p.ring_depth);
    const uint32_t d_chunk = static_cast<uint32_t>(chunk_bytes(p.d_type)), c_chunk = p.C ? static_cast<uint32_t>(chunk_bytes(p.c_type)) : 0u;
    const uint32_t c_buf0 = ring, d_buf0 = ring + depth * c_chunk, z_buf0 = d_buf0 + depth * d_chunk;
    constexpr bool by_tma = kTma;
    const bool has_c = p.C != nullptr, has_z = p.Z != nullptr;
    const bool c_copied = has_c && !by_tma && p.c_type == kF32;  // by cp.async, before the chunk's turn
    // (a TMA store writes whole 16-byte pieces: the last chunk of rows that end within one is stored lane by lane)
    const int whole_cols = p.Nk % (16 / type_bytes(p.d_type)) == 0 ? p.Nk : p.Nk / 32 * 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // before C is read, D or Z written
    const uint32_t acc_empty0 = kPair ? map_to_cta(acc_empty_bar(0), 0) : acc_empty_bar(0);
    uint32_t c_b = 0, c_ph = 0, c_want = 0, asked = 0, taken = 0, d_b = 0;
    bool alive = true;
    int it = 0;
    auto request_c = [&](int col, int row) {  // lane 0 only
      mbar_expect_tx(c_full_bar(ew, c_want), c_chunk);
      tma_load_2d(c_buf0 + c_want * c_chunk, &tmC, c_full_bar(ew, c_want), col, row);
      ++asked;
      if (++c_want == depth) c_want = 0;
    };
    // (every lane counts; lane 0 asks)
    auto next_c = [&]() {
      ++taken;
      if (++c_b == depth) {
        c_b = 0;
        c_ph ^= 1u;
      }
    };
    float* my_bias = bias_smem + ew * (kProductBiasFloats / n_epi);
    // Sums of one chunk -> D (and Z).  False: C did not arrive.
    auto finish_chunk = [&](uint32_t (&r)[32], int row0, int n0, int c, int nchunks) -> bool {
      const int col0 = n0 + c * 32, ncols = min(32, p.Nk - col0);
      const bool inside = row0 < p.Mk && ncols > 0;
      product_z(p.alpha, p.bias ? my_bias + (c - c0) / cstep * 32 : nullptr, r);
      if constexpr (by_tma) {
        const bool ragged = col0 >= whole_cols, mine = inside && row0 + lane < p.Mk;
        if (!ragged || has_c) {
          // the stores that last read these buffers are done with them
          if (lane == 0) {
            if (depth == 2) bulk_wait_group_read<1>(); else bulk_wait_group_read<0>();
          }
          __syncwarp();
        }
        if (has_z) {
          if (!ragged) {
            put_chunk_row(z_buf0 + d_b * d_chunk, lane, r, p.d_type);
          } else if (mine) {
            store_lane_row(p.Z, p.ldz, row0 + lane, col0, ncols, r, p.d_type);
          }
        }
        activate_chunk(r, p.act);
        if (has_c) {
          const bool got = mbar_wait_bounded(c_full_bar(ew, c_b), c_ph, abort_flag, budget_ns);
          if (!__all_sync(0xffffffffu, got)) return false;
          add_chunk_row(c_buf0 + c_b * c_chunk, lane, r, p.beta, p.c_type);
          next_c();
        }
        if (!ragged) {
          put_chunk_row(d_buf0 + d_b * d_chunk, lane, r, p.d_type);
        } else if (mine) {
          store_lane_row(p.D, p.ldd, row0 + lane, col0, ncols, r, p.d_type);
        }
        fence_proxy_async_shared_cta();  // this lane's rows -> visible to the TMA stores (and C's are read)
        __syncwarp();
        if (lane == 0) {
          if (inside && !ragged) {
            if (has_z) tma_store_2d(&tmZ, z_buf0 + d_b * d_chunk, col0, row0);
            tma_store_2d(&tmD, d_buf0 + d_b * d_chunk, col0, row0);
          }
          bulk_commit_group();
          const int ahead = c + static_cast<int>(depth) * cstep;
          if (has_c && ahead < nchunks) request_c(n0 + ahead * 32, row0);
        }
        if (++d_b == depth) d_b = 0;
      } else if (inside) {
        // (the pieces' sums leave registers for a few rows of C at a time only)
        constexpr int kRows = kPieces ? 8 : 32;
        float cc[kRows];
        if (!kPieces && has_c && !c_copied) load_c_rows(p, row0, col0, lane, cc);
        __syncwarp();  // every lane has read the chunk before
        if (has_z) {
          put_chunk_row(ring, lane, r, kF32);
          __syncwarp();
#pragma unroll 1
          for (int r0 = 0; r0 < 32; r0 += kRows) write_chunk_rows(p, ring, p.Z, p.ldz, false, cc, 0u, r0, row0, col0, lane);
          __syncwarp();
        }
        activate_chunk(r, p.act);
        put_chunk_row(ring, lane, r, kF32);
        if (c_copied) cp_async_wait<0>();
        __syncwarp();
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += kRows) {
          if (kPieces && has_c && !c_copied) load_c_rows(p, row0 + r0, col0, lane, cc);
          write_chunk_rows(p, ring, p.D, p.ldd, has_c, cc, c_copied ? ring + 4096u : 0u, r0, row0, col0, lane);
        }
      }
      if (c_copied && c + cstep < nchunks) {
        // the next chunk's C, as soon as this one's is used (a second buffer would cost stages of operands: 4096 x 4097 x 8192
        // 296 us, 378 with it)
        cp_async_wait<0>();
        __syncwarp();
        fetch_c_rows(p, ring + 4096u, row0, col0 + cstep * 32, lane);
      }
      return true;
    };
    auto accumulator = [&](uint32_t& taddr, int& buf) -> bool {  // the next one, when it is ready
      buf = it % nacc;
      const bool ready = mbar_wait_bounded(acc_full_bar(buf), static_cast<uint32_t>(it / nacc) & 1u, abort_flag, budget_ns);
      if (!__all_sync(0xffffffffu, ready)) return false;
      tc_fence_after_sync();
      taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(buf * p.BN);
      ++it;
      return true;
    };
    auto hand_back = [&](int buf) {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair) {
          mbar_arrive_cluster_relaxed(acc_empty0 + 8u * buf);
        } else {
          mbar_arrive(acc_empty_bar(buf));
        }
      }
    };
    for (int t = work0; t < total_tiles && alive; t += work_step) {
      const ProductTile tc = product_tile(p, t, 0);
      const int row0 = (tc.m_tile * kCtas + (kPair ? static_cast<int>(cta_rank) : 0)) * kTileM + q * 32;
      const int n0 = tc.n_tile * p.BN, nchunks = p.BN / 32;
      if (has_c && by_tma && lane == 0) {
        // the tile's first chunks of C, before the accumulator is ready
        for (int c = c0; c < min(nchunks, c0 + static_cast<int>(depth) * cstep); c += cstep) request_c(n0 + c * 32, row0);
      }
      if (c_copied) {
        if (c0 < nchunks) {
          cp_async_wait<0>();
          __syncwarp();
          fetch_c_rows(p, ring + 4096u, row0, n0 + c0 * 32, lane);
        }
      } else if (has_c && !by_tma) {
        for (int c = c0; c < nchunks; c += cstep) prefetch_c_rows(p, row0, n0 + c * 32, lane);
      }
      if (p.bias) {  // the tile's bias, likewise (as loads of a chunk their latency followed every accumulator)
        __syncwarp();
        for (int c = c0, j = 0; c < nchunks; c += cstep, ++j) {
          const int col = n0 + c * 32 + lane;
          my_bias[32 * j + lane] = col < p.Nk ? __ldg(p.bias + col) : 0.0f;
        }
        __syncwarp();
      }
      uint32_t taddr = 0;
      int buf = 0;
      if constexpr (kPieces) {
        constexpr int kMine = 4;  // chunks of a warp, of eight warps' 256 columns
        uint32_t sum[kMine][32];
        for (int i = 0; i < tc.nkb && alive; i += p.piece_blocks) {
          if (!accumulator(taddr, buf)) {
            alive = false;
            break;
          }
#pragma unroll
          for (int j = 0; j < kMine; ++j) {
            const int c = c0 + 2 * j;
            if (c >= nchunks) continue;
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              uint32_t v[16];
              tmem_ld_32x16(taddr + static_cast<uint32_t>(c * 32 + h), v);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e)
                sum[j][h + e] = i == 0 ? v[e] : __float_as_uint(__fadd_rn(__uint_as_float(sum[j][h + e]), __uint_as_float(v[e])));
            }
          }
          hand_back(buf);
        }
#pragma unroll
        for (int j = 0; j < kMine; ++j)
          if (alive && c0 + 2 * j < nchunks) alive = finish_chunk(sum[j], row0, n0, c0 + 2 * j, nchunks);
      } else {
        if (!accumulator(taddr, buf)) {
          alive = false;
          break;
        }
        if (c0 >= nchunks) hand_back(buf);  // a tile narrower than this warp's first chunk
        for (int c = c0; c < nchunks && alive; c += cstep) {
          uint32_t r[32];
          tmem_ld_32x32(taddr + static_cast<uint32_t>(c * 32), r);
          tmem_ld_wait();
          if (c + cstep >= nchunks) hand_back(buf);
          alive = finish_chunk(r, row0, n0, c, nchunks);
        }
      }
    }
    if (!alive && lane == 0) product_error(p, abort_flag, kErrEpilogueWait);
    if (by_tma && lane == 0) {
      bulk_wait_group_all();  // D and Z are complete before the kernel ends
      while (taken < asked) {  // (after a failed wait: chunks of C that are on their way)
        mbar_drain(c_full_bar(ew, c_b), c_ph);
        next_c();
      }
    }
  } else {
    // ------------------- sums of a part of k, to the columns' owners ------------------
    const int q = warp & 3;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // before bias and C are read, D or Z written
    if (p.bias) {  // of this tile's rows (swapped), or of the columns that this CTA will own
      const ProductTile tc = product_tile(p, work0, part);
      const int i = static_cast<int>(threadIdx.x) - 64, own = p.BN / p.parts;
      const int at = p.swapped ? tc.m_tile * tile_rows + i : tc.n_tile * p.BN + part * own + i;
      bias_smem[i] = (p.swapped || i < own) && at < (p.swapped ? p.Mk : p.Nk) ? __ldg(p.bias + at) : 0.0f;
    }
    // The sums as [column][row] where the stages were: every load has landed and every MMA has read it
    // once the last accumulator is there (two stages hold BN <= 128 columns).
    const uint32_t mine = smem_base + static_cast<uint32_t>((q * 32 + lane) * 4);
    auto put = [&](const uint32_t (&r)[16], int c) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(mine + static_cast<uint32_t>((c + i) * kTileM * 4)), "r"(r[i]) : "memory");
    };
    constexpr int kGroups = kPieces ? 8 : 1;  // of 16 columns
    [[maybe_unused]] uint32_t sum[kGroups][16];
    const int nkb = product_tile(p, work0, part).nkb;
    bool alive = true;
    for (int i = 0, it = 0; i < nkb && alive; i += kPieces ? p.piece_blocks : nkb, ++it) {
      const int buf = it % nacc;
      const bool ready = mbar_wait_bounded(acc_full_bar(buf), static_cast<uint32_t>(it / nacc) & 1u, abort_flag, budget_ns);
      if (!__all_sync(0xffffffffu, ready)) {
        if (lane == 0) product_error(p, abort_flag, kErrEpilogueWait);
        alive = false;
        break;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(buf * p.BN);
      if constexpr (kPieces) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          if (16 * g >= p.BN) continue;
          uint32_t v[16];
          tmem_ld_32x16(taddr + static_cast<uint32_t>(16 * g), v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sum[g][e] = i == 0 ? v[e] : __float_as_uint(__fadd_rn(__uint_as_float(sum[g][e]), __uint_as_float(v[e])));
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty_bar(buf));
      } else {
        for (int c = 0; c < p.BN; c += 16) {
          uint32_t r[16];
          tmem_ld_32x16(taddr + static_cast<uint32_t>(c), r);
          tmem_ld_wait();
          put(r, c);
        }
        tc_fence_before_sync();
      }
    }
    if constexpr (kPieces) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        if (alive && 16 * g < p.BN) put(sum[g], 16 * g);
    }
    // (a CTA that gave up sends as well: the others do not wait for it)
    fence_proxy_async_shared_cta();
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the four epilogue warps
    const uint32_t slab = static_cast<uint32_t>(p.BN / p.parts * kTileM * 4);
    if (warp == 2 && lane < p.parts) {
      const uint32_t to = ring_base + static_cast<uint32_t>(part) * slab;
      asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       map_to_cta(to, static_cast<uint32_t>(lane))),
                   "r"(smem_base + static_cast<uint32_t>(lane) * slab), "r"(slab), "r"(map_to_cta(recv_bar, static_cast<uint32_t>(lane)))
                   : "memory");
    }
  }

  if constexpr (kParts) {
    // This CTA's columns, by all warps: the parts' sums added in the order of k, and the epilogue.
    __syncthreads();  // (the bias is there)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool got = __all_sync(0xffffffffu, mbar_wait_bounded(recv_bar, 0, abort_flag, budget_ns));
    if (!got) {
      if (lane == 0) product_error(p, abort_flag, kErrEpilogueWait);
    } else if (*abort_flag == 0) {
      finish_parts(p, ring_base, static_cast<uint32_t>(p.BN / p.parts * kTileM * 4), bias_smem, warp, 7, lane, work0, part);
    }
    tc_fence_before_sync();
    PartsCluster cluster{late_flag, recv_bar, p.parts, lane};
    leave_exchange(cluster, got);
  } else if constexpr (kPair) {
    tc_fence_before_sync();
    // no CTA may leave while another can still touch its shared memory, barriers or accumulator
    __syncwarp();
    cluster_sync_all();
  } else {
    tc_fence_before_sync();
    __syncthreads();
  }
  if (warp == 1) tmem_dealloc_g<kPair>(tmem_base, kTmemCols512);
}

// k == 0: the sums are zero.
__global__ void __launch_bounds__(256) product_empty_kernel(ProductParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t total = static_cast<int64_t>(p.Mk) * p.Nk, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < total; e += step) {
    const int64_t i = e / p.Nk, j = e - i * p.Nk;
    float v = p.bias ? __ldg(p.bias + j) : 0.0f;
    if (p.Z) store_from_f32(p.Z, i * p.ldz + j, p.d_type, v);
    v = activate(v, p.act);
    if (p.C) v = __fmaf_rn(p.beta, load_as_f32(p.C, i * p.ldc + j, p.c_type), v);
    store_from_f32(p.D, i * p.ldd + j, p.d_type, v);
  }
}

}  // namespace b200
