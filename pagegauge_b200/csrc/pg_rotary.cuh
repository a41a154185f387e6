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
  // pg_rotary_kernel only:
  int32_t chunks;       // turning 16-byte chunks of a row, one per thread
  int32_t row_groups;   // threads that share a chunk over a token's rows
  int32_t in_place[2];  // the dims past the pairs are there already
};

// Rows that are 16-byte aligned and whose parts are whole 16-byte chunks.  A
// thread takes one turning chunk (half layout: of both halves) of every
// row_groups-th row of one token, so it reads its table entries once, and the
// rows' copied chunks with it, two rows requested before the first is used.
// Bound by HBM (each row is read and written once), so what counts is bytes in
// flight against registers: interleaved rows hold half as much per thread and
// run six blocks per SM (8,191 tokens: 32.9 us, 38.4 us with four rows in
// flight on four blocks), half-layout rows four.
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

// Any other rows: one thread per (token, row, pair) or copied dim.
template <typename T>
__global__ void __launch_bounds__(256)
    pg_rotary_any_kernel(const __grid_constant__ RotaryParams p) {
  pdl_launch_dependents();
  pdl_wait_primary();
  const int units = p.head_dim - p.pairs;
  const int rows = p.heads[0] + p.heads[1];
  const int64_t total = p.tokens * rows * units;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int unit = static_cast<int>(i % units);
    const int64_t tr = i / units;
    const int row = static_cast<int>(tr % rows);
    const int64_t token = tr / rows;
    const int which = row < p.heads[0] ? 0 : 1;
    const int h = which == 0 ? row : row - p.heads[0];
    const int pos = p.positions[token];
    if (pos < 0 || pos >= p.table_rows) {
      record_error(p.error_flag, kDevBadPosition);
      continue;
    }
    const T* x = static_cast<const T*>(p.x[which]) + token * p.x_stride_t[which] +
                 h * p.x_stride_h[which];
    T* y = static_cast<T*>(p.y[which]) + token * p.y_stride_t[which] + h * p.y_stride_h[which];
    if (unit >= p.pairs) {
      y[unit + p.pairs] = x[unit + p.pairs];
      continue;
    }
    const int da = p.interleaved ? 2 * unit : unit;
    const int db = p.interleaved ? 2 * unit + 1 : unit + p.pairs;
    const float c = p.cos[pos * p.table_stride + unit];
    const float s = p.sign * p.sin[pos * p.table_stride + unit];
    const float a = to_float<T>(x[da]), b = to_float<T>(x[db]);
    y[da] = from_float<T>(__fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)));
    y[db] = from_float<T>(__fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)));
  }
}

}  // namespace pg
