// The 4-bit paged cache: record layout, the fused rotation + append of any
// number of tokens, and the read-back of stored tokens.
//
// One record of 2560 bytes per (page of 16 tokens, KV head), [pages, Hkv,
// 2560] bytes in all, so a page of one head is one contiguous copy:
//   [0, 1024)     key codes, 64 bytes per token
//   [1024, 2048)  value codes, 64 bytes per token
//   [2048, 2304)  key scales and midpoints, 16 bytes per token
//   [2304, 2560)  value scales and midpoints
// A token's key (or value) x of 128 dims is held in four groups of 32 dims:
//   s = f16((max x - min x) / 15),  m = f16(min x + 8 s)
//   z = clamp(rint((x - m) / s), -8, 7) + 8,   x ~ (z - 8) s + m
// with all arithmetic in FP32 (the division by s is a product with the
// rounded reciprocal, which differs only at exact ties of a code).  16 bytes
// of scales per 64 bytes of codes: a group of 32 halves the error's power of
// one scale per head row for 8 bytes more.
//
// Every byte of a record belongs to one token, so tokens of one page may be
// written by different warps or launches in any order.  The order of the
// codes within a token's 64 bytes is the decode kernel's tensor-core operand
// order: see key_code_byte / value_code_byte.
#pragma once

#include <cuda_bf16.h>

#include "pg_common.cuh"

namespace pg {

constexpr int kInt4Record = 2560;
constexpr int kInt4Value = 1024;    // value codes
constexpr int kInt4KeyMeta = 2048;  // key scales and midpoints
constexpr int kInt4ValueMeta = 2304;
constexpr int kInt4Group = 32;  // dims that share a scale and a midpoint

// Element types of q/k/v rows (the C ABI's PG_DTYPE_*).
constexpr int kDtypeF16 = 0;
constexpr int kDtypeBf16 = 1;
constexpr int kDtypeF32 = 2;

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }

// 8 consecutive 16-bit elements at p: one 16-byte access, or one by one
// when rows are not 16-byte aligned.
template <typename T, bool FAST>
__device__ __forceinline__ uint4 load8(const T* p) {
  if constexpr (FAST) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
    return w;
  }
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float* x) {
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
}

template <typename T, bool FAST>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (FAST) {
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_float<T>(x[i]);
  }
}

// Two FP32 operations in one instruction.  A sum of products in this form may
// be contracted, so no product of it feeds a sum of it.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Minimum and maximum that keep a NaN, so that one shows in what is read.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Token tok's row of value codes: tokens 8p + 2u + e lie at row 8p + 4e + u,
// so that the decode's reads of tokens {0, 2, 4, 6} (and {1, 3, 5, 7}) of a
// half page are contiguous in shared memory.
__host__ __device__ constexpr int value_code_row(int tok) {
  return (tok & 8) + 4 * (tok & 1) + ((tok >> 1) & 3);
}

// Quantise lane m's 8 dims 8m .. 8m+7 of one row (16 lanes per row; lanes
// 4j .. 4j+3 hold group j).  Returns the 8 codes, dim 8m + i in nibble i.
// Bound by the ALU pipe (minima, selections, logic run at half rate), so the
// clamps are taken only by warps that need them, and rounding and packing are
// FP32 additions: r + 1.5 2^23 has rint(r) in its low bits, and four codes
// c0 + 16 c1 + 256 c2 + 4096 c3 are exact.  (57,304 tokens of 32 + 16 rows:
// 321 us with a clamp, a conversion and a shift per element, 222 us so.)
__device__ __forceinline__ uint32_t int4_quantize8(float* x, __half& scale, __half& mid) {
  float lo = min3_nan(x[0], x[1], x[2]), hi = max3_nan(x[0], x[1], x[2]);
  lo = min3_nan(min3_nan(lo, x[3], x[4]), x[5], min_nan(x[6], x[7]));
  hi = max3_nan(max3_nan(hi, x[3], x[4]), x[5], max_nan(x[6], x[7]));
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (__any_sync(0xffffffffu, !(hi <= 65504.f && lo >= -65504.f))) {
    lo = min_nan(max_nan(lo, -65504.f), 65504.f);
    hi = min_nan(max_nan(hi, -65504.f), 65504.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = min_nan(max_nan(x[i], -65504.f), 65504.f);
  }
  scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const float s = __half2float(scale);
  mid = __float2half_rn(__fadd_rn(lo, 8.f * s));
  const float m = __half2float(mid);
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 r = mul2(add2(make_float2(x[i], x[i + 1]), make_float2(-m, -m)),
                          make_float2(inv, inv));
    x[i] = r.x;
    x[i + 1] = r.y;
  }
  // The map is monotonic, so its extremes say whether any code needs a clamp
  // (where the midpoint's rounding is a large part of a step, or for a NaN,
  // which keeps code 0: its group's scale and midpoint are NaN).
  const bool inside = __fmul_rn(__fsub_rn(lo, m), inv) >= -8.5f &&
                      __fmul_rn(__fsub_rn(hi, m), inv) < 7.5f;
  if (__any_sync(0xffffffffu, !inside)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -8.f), 7.f);
  }
  uint32_t half[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float c[4];
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float2 r = add2(make_float2(__fadd_rn(x[4 * i + j], 12582920.f),
                                        __fadd_rn(x[4 * i + j + 1], 12582920.f)),
                            make_float2(-12582912.f, -12582912.f));
      c[j] = r.x;
      c[j + 1] = r.y;
    }
    const float sum = fmaf(c[3], 4096.f, fmaf(c[2], 256.f, fmaf(c[1], 16.f, c[0])));
    half[i] = __float_as_uint(__fadd_rn(sum, 8388608.f));
  }
  return prmt(half[0], half[1], 0x5410u);
}

struct Int4AppendParams {
  const void* q;
  const void* k;
  const void* v;
  int64_t q_stride_t, k_stride_t, v_stride_t;
  void* rotated_q;  // [T, Hq, 128]
  void* rotated_k;  // [T, Hkv, 128] or null
  int64_t rq_stride_t, rk_stride_t;
  // Heads times these stay below 2^31.
  int32_t q_stride_h, k_stride_h, v_stride_h, rq_stride_h, rk_stride_h;
  const float* cos;  // [table_rows, pairs]
  const float* sin;
  int64_t table_stride, table_rows;
  const int32_t* positions;  // [T]
  const int32_t* slots;      // [T]: page * 16 + token, negative: skipped
  uint8_t* records;
  int64_t num_pages;
  const void* key_center;  // [centers, Hkv, 128] or null
  const void* value_center;
  const int32_t* center_rows;  // [T] or null (row 0)
  int64_t num_centers;
  int64_t tokens;
  int32_t hq, hkv, pairs, interleaved;
  int32_t split;  // warps that share one token's rows
  int* error_flag;
};

// Lane m's 8 dims of a row, rotated (raw: the row's elements 8m .. 8m + 7,
// base: its element 0).  Half layout: dims (d, d + pairs) turn together;
// interleaved: (2j, 2j + 1).  c, s: this lane's table entries, or read from
// the rows here if !FAST.
template <typename T, bool FAST>
__device__ __forceinline__ void rotate8(float* x, const uint4& raw, const T* base, int m,
                                        int pairs, bool interleaved, const float* c,
                                        const float* s, const float* cos_row,
                                        const float* sin_row) {
  unpack8<T>(raw, x);
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const int j = 4 * m + (i >> 1);
      if (j >= pairs) continue;
      const float cj = FAST ? c[i >> 1] : cos_row[j], sj = FAST ? s[i >> 1] : sin_row[j];
      const float a = x[i], b = x[i + 1];
      x[i] = __fsub_rn(__fmul_rn(a, cj), __fmul_rn(b, sj));
      x[i + 1] = __fadd_rn(__fmul_rn(b, cj), __fmul_rn(a, sj));
    }
    return;
  }
  if constexpr (FAST) {
    // pairs is a multiple of 8: a lane's partner dims are one lane's.  The
    // first half's lanes hold -s, so both halves add.
    const int step = pairs >> 3;
    const bool turns = m < 2 * step;
    const int peer = !turns ? m : m < step ? m + step : m - step;
    uint4 other;
    other.x = __shfl_sync(0xffffffffu, raw.x, peer, 16);
    other.y = __shfl_sync(0xffffffffu, raw.y, peer, 16);
    other.z = __shfl_sync(0xffffffffu, raw.z, peer, 16);
    other.w = __shfl_sync(0xffffffffu, raw.w, peer, 16);
    float o[8];
    unpack8<T>(other, o);
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 r = add2(
            make_float2(__fmul_rn(x[i], c[i]), __fmul_rn(x[i + 1], c[i + 1])),
            make_float2(__fmul_rn(o[i], s[i]), __fmul_rn(o[i + 1], s[i + 1])));
        x[i] = r.x;
        x[i + 1] = r.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = 8 * m + i;
      if (d >= 2 * pairs) continue;
      const int j = d < pairs ? d : d - pairs;
      const float o = to_float<T>(base[d < pairs ? d + pairs : j]);
      const float a = __fmul_rn(x[i], cos_row[j]), b = __fmul_rn(o, sin_row[j]);
      x[i] = d < pairs ? __fsub_rn(a, b) : __fadd_rn(a, b);
    }
  }
}

// What an append warp knows of its token.
struct Int4Token {
  int64_t token, page, center;
  int tok;
  const float* cos_row;
  const float* sin_row;
};

// Quantise and store lane m's 8 dims of one row of KV head h (the two halves
// of a warp hold two rows; a row past the last stores nothing).
__device__ __forceinline__ void store_int4_row(const Int4AppendParams& p, const Int4Token& k,
                                               bool is_key, int h, int m, float* x) {
  __half scale, mid;
  const uint32_t codes = int4_quantize8(x, scale, mid);
  uint8_t* rec = p.records + (k.page * p.hkv + (h < p.hkv ? h : 0)) * kInt4Record;
  const int grp = m >> 2;
  if (is_key) {
    if (h < p.hkv)
      *reinterpret_cast<uint32_t*>(rec + k.tok * 64 + (m & 3) * 16 + grp * 4) = codes;
  } else {
    // Dims 4a .. 4a+3 of groups 2i and 2i+1 are one word: lanes of an even
    // group take their first four dims' word, of an odd one the other.
    const uint32_t other = __shfl_xor_sync(0xffffffffu, codes, 4);
    const uint32_t word = (grp & 1) ? prmt(other, codes, 0x7632u) : prmt(codes, other, 0x5410u);
    if (h < p.hkv)
      *reinterpret_cast<uint32_t*>(rec + kInt4Value + value_code_row(k.tok) * 64 + (m & 3) * 16 +
                                   (grp & 1) * 8 + (grp >> 1) * 4) = word;
  }
  // The token's four scales and midpoints as one 16-byte store.
  const uint32_t sm = static_cast<uint32_t>(__half_as_ushort(scale)) |
                      (static_cast<uint32_t>(__half_as_ushort(mid)) << 16);
  const uint32_t s1 = __shfl_down_sync(0xffffffffu, sm, 4, 16);
  const uint32_t s2 = __shfl_down_sync(0xffffffffu, sm, 8, 16);
  const uint32_t s3 = __shfl_down_sync(0xffffffffu, sm, 12, 16);
  if (m == 0 && h < p.hkv)
    *reinterpret_cast<uint4*>(rec + (is_key ? kInt4KeyMeta : kInt4ValueMeta) + k.tok * 16) =
        make_uint4(prmt(sm, s1, 0x5410u), prmt(s2, s3, 0x5410u), prmt(sm, s1, 0x7632u),
                   prmt(s2, s3, 0x7632u));
}

template <typename T>
__device__ __forceinline__ void subtract_center(const Int4AppendParams& p, const Int4Token& k,
                                                const void* centers, int h, int m, float* x) {
  if (centers == nullptr) return;
  float y[8];
  unpack8<T>(load8<T, true>(static_cast<const T*>(centers) +
                            (k.center * p.hkv + h) * kHeadDim + 8 * m), y);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 r = add2(make_float2(x[i], x[i + 1]), make_float2(-y[i], -y[i + 1]));
    x[i] = r.x;
    x[i + 1] = r.y;
  }
}

// `split` warps share one token.  A warp takes two rows at a time (16 lanes of
// 8 dims each) and requests U query row pairs, or a key and a value row pair,
// before it uses the first.  U = 4 where tokens alone fill the GPU: the
// table entries, slot and position are then read once per token; U = 1 with
// a warp per row pair for few tokens, where latency is all.
template <typename T, bool FAST, int U>
__global__ void __launch_bounds__(256, 4)
    pg_rope_append_int4_kernel(const __grid_constant__ Int4AppendParams p) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, half = lane >> 4, m = lane & 15;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  Int4Token k;
  k.token = p.split == 1 ? w : static_cast<uint32_t>(w) / p.split;  // w is small if split
  const int part = static_cast<int>(w - k.token * p.split);
  if (k.token >= p.tokens) return;
  pdl_wait_primary();
  const int slot = p.slots[k.token];
  const int pos = p.positions[k.token];
  k.center = p.center_rows != nullptr ? p.center_rows[k.token] : 0;
  // The first query rows are asked for along with the token's indices.
  const T* q = static_cast<const T*>(p.q) + k.token * p.q_stride_t + 8 * m;
  const int nq = (p.hq + 2 * U - 1) / (2 * U), nk = (p.hkv + 1) >> 1;
  uint4 raw[U];
  auto load_queries = [&](int u) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = 2 * (u * U + i) + half;
      raw[i] = load8<T, FAST>(q + (h < p.hq ? h : p.hq - 1) * p.q_stride_h);
    }
  };
  if (part < nq) load_queries(part);
  if (slot < 0) return;
  k.page = slot >> 4;
  k.tok = slot & 15;
  if (k.page >= p.num_pages ||
      (p.key_center != nullptr && (k.center < 0 || k.center >= p.num_centers))) {
    record_error(p.error_flag, kDevBadPageId);
    return;
  }
  if (pos < 0 || pos >= p.table_rows) {
    record_error(p.error_flag, kDevBadPosition);
    return;
  }
  k.cos_row = p.cos + pos * p.table_stride;
  k.sin_row = p.sin + pos * p.table_stride;
  float c[8], s[8];
  if constexpr (FAST) {
    // The lane's entries: half layout 8 of them, interleaved 4.
    const int step = p.pairs >> 3;
    const int j = p.interleaved ? 4 * m : 8 * (m < step ? m : m - step);
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const bool in = (p.interleaved ? i == 0 : m < 2 * step) && j + i < p.pairs;
      const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 a = in ? __ldg(reinterpret_cast<const float4*>(k.cos_row + j + i)) : z;
      const float4 b = in ? __ldg(reinterpret_cast<const float4*>(k.sin_row + j + i)) : z;
      c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
      const float sign = !p.interleaved && m < step ? -1.f : 1.f;
      s[i] = sign * b.x; s[i + 1] = sign * b.y; s[i + 2] = sign * b.z; s[i + 3] = sign * b.w;
    }
  }
  const T* kr = static_cast<const T*>(p.k) + k.token * p.k_stride_t;
  const T* vr = static_cast<const T*>(p.v) + k.token * p.v_stride_t;
  T* rq = static_cast<T*>(p.rotated_q) + k.token * p.rq_stride_t;
  // Row h of two halves; an odd last row is loaded by both, stored by one.
  auto turn_and_store = [&](float* x, const uint4& raw, const T* row, T* out, bool store) {
    rotate8<T, FAST>(x, raw, row, m, p.pairs, p.interleaved, c, s, k.cos_row, k.sin_row);
    // In place, other lanes' partner dims are this lane's.
    if constexpr (!FAST) __syncwarp();
    if (store) store8<T, FAST>(out + 8 * m, x);
  };
  auto append_row = [&](const uint4& raw, bool is_key, int h, const T* row) {
    const int hc = h < p.hkv ? h : p.hkv - 1;
    float x[8];
    if (is_key)
      turn_and_store(x, raw, row,
                     static_cast<T*>(p.rotated_k) + k.token * p.rk_stride_t + hc * p.rk_stride_h,
                     p.rotated_k != nullptr && h < p.hkv);
    else
      unpack8<T>(raw, x);
    subtract_center<T>(p, k, is_key ? p.key_center : p.value_center, hc, m, x);
    store_int4_row(p, k, is_key, h, m, x);
  };
  for (int u = part; u < nq; u += p.split) {
    if (u != part) load_queries(u);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = 2 * (u * U + i) + half;
      if (2 * (u * U + i) >= p.hq) break;
      const int hc = h < p.hq ? h : p.hq - 1;
      float x[8];
      turn_and_store(x, raw[i], q - 8 * m + hc * p.q_stride_h, rq + hc * p.rq_stride_h, h < p.hq);
    }
  }
  // This warp's first unit past the query rows.
  const int first = part >= nq ? part - nq : (p.split - (nq - part) % p.split) % p.split;
  if constexpr (U > 1) {
    for (int u = first; u < nk; u += p.split) {
      const int h = 2 * u + half;
      const int hc = h < p.hkv ? h : p.hkv - 1;
      const uint4 x = load8<T, FAST>(kr + hc * p.k_stride_h + 8 * m);
      const uint4 y = load8<T, FAST>(vr + hc * p.v_stride_h + 8 * m);
      append_row(x, true, h, kr + hc * p.k_stride_h);
      append_row(y, false, h, nullptr);
    }
  } else {
    for (int u = first; u < 2 * nk; u += p.split) {
      const bool is_key = u < nk;
      const int h = 2 * (u - (is_key ? 0 : nk)) + half;
      const int hc = h < p.hkv ? h : p.hkv - 1;
      const T* row = is_key ? kr + hc * p.k_stride_h : vr + hc * p.v_stride_h;
      append_row(load8<T, FAST>(row + 8 * m), is_key, h, row);
    }
  }
}

struct Int4ReadParams {
  const uint8_t* records;
  int64_t num_pages;
  const int32_t* slots;
  int64_t tokens;
  int32_t hkv;
  int32_t split;  // warps that share one token's heads
  void* key;      // [T, Hkv, 128]
  void* value;    // [T, Hkv, 128]
  int* error_flag;
};

// One warp per token and 2 U KV heads (16 lanes per head's key and value row),
// with everything requested before it is used; skipped slots read as zeros.
// U = 4 where tokens alone fill the GPU, as in the append.
template <typename T, int U>
__global__ void __launch_bounds__(256)
    pg_int4_read_kernel(const __grid_constant__ Int4ReadParams p) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, half = lane >> 4, m = lane & 15, grp = m >> 2;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  // A 32-bit division where the index allows it.
  const int64_t token = w < (int64_t(1) << 31)
                            ? static_cast<int64_t>(static_cast<uint32_t>(w) / p.split)
                            : w / p.split;
  if (token >= p.tokens) return;
  const int h0 = 2 * U * static_cast<int>(w - token * p.split) + half;
  pdl_wait_primary();
  const int slot = p.slots[token];
  const bool held = slot >= 0 && (slot >> 4) < p.num_pages;
  if (slot >= 0 && !held) record_error(p.error_flag, kDevBadPageId);
  uint32_t codes[U][2];
  __half s[U][2], mid[U][2];
#pragma unroll
  for (int i = 0; i < U; ++i) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[i][kv] = 0u;
      s[i][kv] = mid[i][kv] = __ushort_as_half(0);
    }
    const int h = h0 + 2 * i;
    if (held && h < p.hkv) {
      const int tok = slot & 15;
      const uint8_t* rec =
          p.records + (static_cast<int64_t>(slot >> 4) * p.hkv + h) * kInt4Record;
      const __half* km = reinterpret_cast<const __half*>(rec + kInt4KeyMeta + tok * 16) + grp;
      const __half* vm = reinterpret_cast<const __half*>(rec + kInt4ValueMeta + tok * 16) + grp;
      codes[i][0] = *reinterpret_cast<const uint32_t*>(rec + tok * 64 + (m & 3) * 16 + grp * 4);
      // The word of store_int4_row; its other lane's makes the two halves.
      codes[i][1] = *reinterpret_cast<const uint32_t*>(
          rec + kInt4Value + value_code_row(tok) * 64 + (m & 3) * 16 + (grp & 1) * 8 +
          (grp >> 1) * 4);
      s[i][0] = km[0];
      mid[i][0] = km[4];
      s[i][1] = vm[0];
      mid[i][1] = vm[4];
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, codes[i][1], 4);
    codes[i][1] = (grp & 1) ? prmt(other, codes[i][1], 0x7632u) : prmt(codes[i][1], other, 0x5410u);
    const int h = h0 + 2 * i;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      T* out = static_cast<T*>(kv == 0 ? p.key : p.value) +
               (token * p.hkv + (h < p.hkv ? h : 0)) * kHeadDim + 8 * m;
      const float sc = __half2float(s[i][kv]), md = __half2float(mid[i][kv]);
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // Nibbles j and j + 4 as the halves 1024 + z, less 1032 (exact).
        const uint32_t c = ((codes[i][kv] >> (4 * j)) & 0x000f000fu) | 0x64006400u;
        const uint32_t z = hsub2_u32(c, 0x64086408u);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&z));
        x[j] = __fadd_rn(__fmul_rn(f.x, sc), md);
        x[j + 4] = __fadd_rn(__fmul_rn(f.y, sc), md);
      }
      if (h >= p.hkv) continue;
      if constexpr (sizeof(T) == 2) {
        store8<T, true>(out, x);
      } else {
        reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
  }
}

}  // namespace pg
