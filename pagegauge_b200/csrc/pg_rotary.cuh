// Rotary positions of query and key rows: pairs of dims (a, b) of the first
// 2 * pairs dims of a row turn by the angle of the row's position,
//   a' = a cos - b sin,  b' = b cos + a sin     (adjoint: sin negated)
// computed in FP32 from FP32 tables and rounded once.  Half layout pairs
// (j, j + pairs), interleaved (2j, 2j + 1); the other dims are copied.
#pragma once

#include "pg_int4.cuh"

namespace pg {

struct RotaryParams {
  const void* x[2];  // query rows, key rows (or null)
  void* y[2];
  int64_t x_stride_t[2], y_stride_t[2];
  int32_t x_stride_h[2], y_stride_h[2];  // heads times these stay below 2^31
  int32_t heads[2];
  int64_t tokens;
  int32_t head_dim, pairs, interleaved;
  float sign;  // -1: adjoint
  const float* cos;
  const float* sin;
  int64_t table_stride, table_rows;
  const int32_t* positions;
  int* error_flag;
  int32_t in_place[2];  // the dims past the pairs are there already
  // pg_rotary_kernel: turning 16-byte chunks of a row, one per thread, and
  // threads that share a chunk over a token's rows.
  int32_t chunks, row_groups;
  // pg_rotary_rows_kernel: tokens of a block, rows of a token's tile and the
  // elements from row to row in it; over_n() of a row's chunks and pairs (at
  // most a token's threads).
  int32_t block_tokens, tile_rows, pitch, over_cols, over_pairs;
};

// Rows that are 16-byte aligned and whose parts are whole 16-byte chunks, where
// little data, or much of whole heads, makes the way through shared memory the
// slower one.  A thread takes one turning chunk (half layout: of both halves)
// of every row_groups-th row of one token, so it reads its table entries once,
// and the rows' copied chunks with it, two rows requested before the first is
// used.
// Bound by latency where there is little data, by HBM where there is much (each
// row is read and written once: 49,152 tokens of 40 FP16 rows, 1.03 GB, 174
// us, 5.9 TB/s), so bytes in flight count against registers: interleaved rows
// hold half as much per thread and run six blocks per SM, half-layout rows
// four.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(256, INTERLEAVED ? 6 : 4)
    pg_rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int V = 16 / sizeof(T), U = 2;
  constexpr int E = INTERLEAVED ? V / 2 : V;  // table entries of a chunk
  pdl_launch_dependents();
  pdl_wait_primary();
  const int per_token = p.chunks * p.row_groups;
  const int rows = p.heads[0] + p.heads[1];
  const int64_t u = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  // A 32-bit division where the index allows it.
  const int64_t token = u < (int64_t(1) << 31)
                            ? static_cast<int64_t>(static_cast<uint32_t>(u) / per_token)
                            : u / per_token;
  if (token >= p.tokens) return;
  const int rest = static_cast<int>(u - token * per_token);
  const int group = rest / p.chunks;
  const int chunk = rest - group * p.chunks;
  const int pos = p.positions[token];
  const T* xq = static_cast<const T*>(p.x[0]) + token * p.x_stride_t[0] + chunk * V;
  const T* xk = static_cast<const T*>(p.x[1]) + token * p.x_stride_t[1] + chunk * V;
  uint4 a[U], b[U];
  auto load_rows = [&](int r0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int row = r0 + i * p.row_groups;
      if (row >= rows) continue;
      const T* x = row < p.heads[0] ? xq + row * p.x_stride_h[0]
                                    : xk + (row - p.heads[0]) * p.x_stride_h[1];
      a[i] = *reinterpret_cast<const uint4*>(x);
      if constexpr (!INTERLEAVED) b[i] = *reinterpret_cast<const uint4*>(x + p.pairs);
    }
  };
  // The first rows are asked for along with the position.
  load_rows(group);
  if (pos < 0 || pos >= p.table_rows) {
    record_error(p.error_flag, kDevBadPosition);
    return;
  }
  float c[E], s[E];
  {
    const float* cr = p.cos + pos * p.table_stride + chunk * E;
    const float* sr = p.sin + pos * p.table_stride + chunk * E;
    constexpr int W = E >= 4 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < E; i += W) {
      if constexpr (W == 4) {
        const float4 u4 = __ldg(reinterpret_cast<const float4*>(cr + i));
        const float4 v4 = __ldg(reinterpret_cast<const float4*>(sr + i));
        c[i] = u4.x; c[i + 1] = u4.y; c[i + 2] = u4.z; c[i + 3] = u4.w;
        s[i] = v4.x; s[i + 1] = v4.y; s[i + 2] = v4.z; s[i + 3] = v4.w;
      } else {
        const float2 u2 = __ldg(reinterpret_cast<const float2*>(cr + i));
        const float2 v2 = __ldg(reinterpret_cast<const float2*>(sr + i));
        c[i] = u2.x; c[i + 1] = u2.y;
        s[i] = v2.x; s[i + 1] = v2.y;
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) s[i] *= p.sign;
  }
  T* yq = static_cast<T*>(p.y[0]) + token * p.y_stride_t[0] + chunk * V;
  T* yk = static_cast<T*>(p.y[1]) + token * p.y_stride_t[1] + chunk * V;
  // The copied chunks d = chunk, chunk + chunks, ... of a row start here,
  // relative to its turning chunk.
  const int tail = 2 * p.pairs;
  const int copied = (p.head_dim - 2 * p.pairs) / V;
  for (int r0 = group; r0 < rows; r0 += U * p.row_groups) {
    if (r0 != group) load_rows(r0);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (r0 + i * p.row_groups >= rows) break;
      T* ea = reinterpret_cast<T*>(&a[i]);
      T* eb = reinterpret_cast<T*>(&b[i]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        T& ta = INTERLEAVED ? ea[2 * e] : ea[e];
        T& tb = INTERLEAVED ? ea[2 * e + 1] : eb[e];
        const float xa = to_float<T>(ta), xb = to_float<T>(tb);
        ta = from_float<T>(__fsub_rn(__fmul_rn(xa, c[e]), __fmul_rn(xb, s[e])));
        tb = from_float<T>(__fadd_rn(__fmul_rn(xb, c[e]), __fmul_rn(xa, s[e])));
      }
      T* y = r0 + i * p.row_groups < p.heads[0]
                 ? yq + (r0 + i * p.row_groups) * p.y_stride_h[0]
                 : yk + (r0 + i * p.row_groups - p.heads[0]) * p.y_stride_h[1];
      *reinterpret_cast<uint4*>(y) = a[i];
      if constexpr (!INTERLEAVED) *reinterpret_cast<uint4*>(y + p.pairs) = b[i];
    }
    for (int d = chunk; d < copied; d += p.chunks) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int row = r0 + i * p.row_groups;
        if (row >= rows) continue;
        const T* x = row < p.heads[0] ? xq + row * p.x_stride_h[0]
                                      : xk + (row - p.heads[0]) * p.x_stride_h[1];
        a[i] = *reinterpret_cast<const uint4*>(x + tail + (d - chunk) * V);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int row = r0 + i * p.row_groups;
        const bool is_q = row < p.heads[0];
        if (row >= rows || (is_q ? p.in_place[0] : p.in_place[1])) continue;
        T* y = is_q ? yq + row * p.y_stride_h[0] : yk + (row - p.heads[0]) * p.y_stride_h[1];
        *reinterpret_cast<uint4*>(y + tail + (d - chunk) * V) = a[i];
      }
    }
  }
}

// 16 bytes into shared memory.
__device__ __forceinline__ void cp_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// t / n for t and n up to 256, times = over_n(n).
__host__ __device__ constexpr int32_t over_n(int32_t n) { return (1 << 20) / n + 1; }
__device__ __forceinline__ int small_div(int t, int32_t times) { return (t * times) >> 20; }

// Any pairs, head sizes and alignments.  Rows pass through shared memory, so
// that the copies in and out are 16-byte ones (VEC; else single elements) and
// many are in flight without registers, while the pairs, which start anywhere,
// are turned element by element: thread j of a token's threads takes pair j (W
// pairs from W j on) of every few rows.  block_tokens tokens (or tile_rows rows
// of one) share a block, of 256 / block_tokens threads each.  A row is whole in
// its block, so rows may be turned in place.  8,000 tokens of 40 FP16 rows with
// 58 of 128 dims turning (165 MB): 30.9 us in half layout, 29.7 us interleaved
// (5.6 TB/s; FP32 51 us, 6.4 TB/s); with a thread per pair and no tiles 162 us.
template <typename T, bool INTERLEAVED, bool VEC, int W>
__global__ void __launch_bounds__(256)
    pg_rotary_rows_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int N = INTERLEAVED ? 2 * W : W;  // elements of one access
  struct __align__(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Elements { T e[N]; };
  extern __shared__ __align__(16) uint8_t smem_rotary[];
  pdl_launch_dependents();
  const int threads = 256 / p.block_tokens;  // a power of two tokens
  const int sub = threadIdx.x / static_cast<unsigned>(threads);
  const int t = threadIdx.x - sub * threads;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * p.block_tokens + sub;
  const int row0 = blockIdx.y * p.tile_rows;
  const int rows = min(p.tile_rows, p.heads[0] + p.heads[1] - row0);
  T* tile = reinterpret_cast<T*>(smem_rotary) + sub * p.tile_rows * p.pitch;
  // Column c0, c0 + cols, ... of rows ry, ry + row_step, ...
  const int chunks = p.head_dim / V;
  const int cols = min(chunks, threads), ry = small_div(t, p.over_cols), c0 = t - ry * cols;
  const int row_step = small_div(threads, p.over_cols);
  bool live = token < p.tokens;
  // Chunks of a query or key row that are read and written.
  const int turning = (2 * p.pairs + V - 1) / V;
  const int chunks_q = p.in_place[0] ? turning : chunks;
  const int chunks_k = p.in_place[1] ? turning : chunks;
  pdl_wait_primary();
  if (live && ry < row_step) {
    const T* xq = static_cast<const T*>(p.x[0]) + token * p.x_stride_t[0];
    const T* xk = static_cast<const T*>(p.x[1]) + token * p.x_stride_t[1];
    for (int r = ry; r < rows; r += row_step) {
      const int h = row0 + r;
      const bool is_q = h < p.heads[0];
      const T* from = is_q ? xq + h * p.x_stride_h[0] : xk + (h - p.heads[0]) * p.x_stride_h[1];
      T* to = tile + r * p.pitch;
      for (int c = c0; c < (is_q ? chunks_q : chunks_k); c += cols) {
        if constexpr (VEC)
          cp_async16(to + c * V, from + c * V);
        else
          to[c] = from[c];
      }
    }
  }
  const int groups = p.pairs / W, lanes = min(groups, threads);
  const int rg = small_div(t, p.over_pairs), group_step = small_div(threads, p.over_pairs);
  int j = t - rg * lanes;
  float c[W], s[W];
  const float* cos_row = p.cos;
  const float* sin_row = p.sin;
  auto entries = [&] {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      c[i] = __ldg(cos_row + W * j + i);
      s[i] = p.sign * __ldg(sin_row + W * j + i);
    }
  };
  if (live) {
    const int pos = p.positions[token];
    if (pos < 0 || pos >= p.table_rows) {
      record_error(p.error_flag, kDevBadPosition);
      live = false;
    } else {
      cos_row += pos * p.table_stride;
      sin_row += pos * p.table_stride;
      entries();
    }
  }
  if constexpr (VEC) cp_async_wait_all();
  __syncthreads();
  if (live && rg < group_step) {
    while (true) {
      T* a = tile + (INTERLEAVED ? 2 : 1) * W * j;
#pragma unroll 4
      for (int r = rg; r < rows; r += group_step) {
        T* x = a + r * p.pitch;
        Elements v = *reinterpret_cast<const Elements*>(x), w = v;
        if constexpr (!INTERLEAVED) w = *reinterpret_cast<const Elements*>(x + p.pairs);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          T& ta = INTERLEAVED ? v.e[2 * i] : v.e[i];
          T& tb = INTERLEAVED ? v.e[2 * i + 1] : w.e[i];
          const float xa = to_float<T>(ta), xb = to_float<T>(tb);
          ta = from_float<T>(__fsub_rn(__fmul_rn(xa, c[i]), __fmul_rn(xb, s[i])));
          tb = from_float<T>(__fadd_rn(__fmul_rn(xb, c[i]), __fmul_rn(xa, s[i])));
        }
        *reinterpret_cast<Elements*>(x) = v;
        if constexpr (!INTERLEAVED) *reinterpret_cast<Elements*>(x + p.pairs) = w;
      }
      j += lanes;
      if (j >= groups) break;
      entries();
    }
  }
  __syncthreads();
  if (live && ry < row_step) {
    T* yq = static_cast<T*>(p.y[0]) + token * p.y_stride_t[0];
    T* yk = static_cast<T*>(p.y[1]) + token * p.y_stride_t[1];
    for (int r = ry; r < rows; r += row_step) {
      const int h = row0 + r;
      const bool is_q = h < p.heads[0];
      T* to = is_q ? yq + h * p.y_stride_h[0] : yk + (h - p.heads[0]) * p.y_stride_h[1];
      const T* from = tile + r * p.pitch;
      for (int c = c0; c < (is_q ? chunks_q : chunks_k); c += cols) {
        if constexpr (VEC)
          reinterpret_cast<uint4*>(to)[c] = reinterpret_cast<const uint4*>(from)[c];
        else
          to[c] = from[c];
      }
    }
  }
}

}  // namespace pg
