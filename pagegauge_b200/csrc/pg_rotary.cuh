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
  int64_t x_stride_t[2], x_stride_h[2], y_stride_t[2], y_stride_h[2];
  int32_t heads[2];
  int64_t tokens;
  int32_t head_dim, pairs, interleaved;
  float sign;  // -1: adjoint
  const float* cos;
  const float* sin;
  int64_t table_stride, table_rows;
  const int32_t* positions;
  int* error_flag;
};

// One thread per (token, row, pair) or copied dim.
template <typename T>
__global__ void __launch_bounds__(256)
    pg_rotary_kernel(const __grid_constant__ RotaryParams p) {
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
