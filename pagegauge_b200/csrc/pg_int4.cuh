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

// Scale, midpoint and codes of one lane's 8 dims of a group, four lanes (l & 3)
// to a group.  Returns the 8 codes, the first dim in nibble 0; meta: the
// scale's bits and, in the upper half, the midpoint's.  lo, hi: the group's
// extremes, which the caller has clamped with x.
__device__ __forceinline__ uint32_t int4_codes8(float* x, float lo, float hi, bool& clamped,
                                                uint32_t& meta) {
  const __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const float s = __half2float(scale);
  const __half mid = __float2half_rn(__fadd_rn(lo, 8.f * s));
  const float m = __half2float(mid);
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
  meta = static_cast<uint32_t>(__half_as_ushort(scale)) |
         (static_cast<uint32_t>(__half_as_ushort(mid)) << 16);
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
  clamped = !(__fmul_rn(__fsub_rn(lo, m), inv) >= -8.5f &&
              __fmul_rn(__fsub_rn(hi, m), inv) < 7.5f);
  if (__any_sync(0xffffffffu, clamped)) {
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

// Quantise one row of 8 lanes: lane l holds dims 8l .. 8l+7 (a) and
// 64 + 8l .. (b), so lanes 0-3 and 4-7 hold groups 0, 1 (a) and 2, 3 (b).
// Bound by the ALU pipe (minima, selections, logic run at half rate), so the
// clamps are taken only by warps that need them, and rounding and packing are
// FP32 additions: r + 1.5 2^23 has rint(r) in its low bits, and four codes
// c0 + 16 c1 + 256 c2 + 4096 c3 are exact.
__device__ __forceinline__ void int4_quantize16(float* a, float* b, uint32_t* codes,
                                                uint32_t* meta) {
  float lo[2], hi[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float* x = k == 0 ? a : b;
    lo[k] = min3_nan(min3_nan(x[0], x[1], x[2]), min3_nan(x[3], x[4], x[5]), min_nan(x[6], x[7]));
    hi[k] = max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max_nan(x[6], x[7]));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo[k] = min_nan(lo[k], __shfl_xor_sync(0xffffffffu, lo[k], o));
      hi[k] = max_nan(hi[k], __shfl_xor_sync(0xffffffffu, hi[k], o));
    }
  }
  const bool fits = max_nan(hi[0], hi[1]) <= 65504.f && min_nan(lo[0], lo[1]) >= -65504.f;
  if (__any_sync(0xffffffffu, !fits)) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      lo[k] = min_nan(max_nan(lo[k], -65504.f), 65504.f);
      hi[k] = min_nan(max_nan(hi[k], -65504.f), 65504.f);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = min_nan(max_nan(a[i], -65504.f), 65504.f);
      b[i] = min_nan(max_nan(b[i], -65504.f), 65504.f);
    }
  }
  bool clamped;
  codes[0] = int4_codes8(a, lo[0], hi[0], clamped, meta[0]);
  codes[1] = int4_codes8(b, lo[1], hi[1], clamped, meta[1]);
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
  int32_t split;      // warps that share one token's rows
  int32_t row_shift;  // a warp's four rows are of 4 >> row_shift tokens (FEW)
  int* error_flag;
};

// How an append rotates: the whole head in half layout, whose partner dims lie
// in one lane (kTurnHalf); up to half of the head in half layout (kTurnPart);
// neighbouring pairs (kTurnInterleaved); parts that are not whole 16-byte
// chunks, or tables that are not aligned, in half layout, through shared
// memory (kTurnOdd), and interleaved (kTurnOddInterleaved); and rows that are
// not 16-byte aligned (kTurnAny).  8,000 tokens of 32 + 16 FP16 rows with 58
// turning dims, append and read: 56.4 us in half layout, 46.3 us
// interleaved (128 dims: 45.2 / 46.2 us); with the partners read one by one
// from the rows 138.8 / 118.7 us.
constexpr int kTurnAny = 0, kTurnHalf = 1, kTurnInterleaved = 2, kTurnPart = 3, kTurnOdd = 4,
              kTurnOddInterleaved = 5;

// A token's table rows and lane l's entries of them: kTurnHalf 8l .. 8l+7,
// kTurnPart those of its first chunk, interleaved 4l .. 4l+3 and 32 + 4l ..,
// others l, l + 8, ...
struct Int4Turn {
  const float* cos_row;
  const float* sin_row;
  float c[8], s[8];
  int pairs, l;
  bool interleaved;
};

// 8 dims d .. d + 7 (a chunk) of a row with partner dims o.
template <bool FIRST>
__device__ __forceinline__ void turn_half(float* x, const float* o, const float* c,
                                          const float* s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = __fmul_rn(x[i], c[i]), b = __fmul_rn(o[i], s[i]);
    x[i] = FIRST ? __fsub_rn(a, b) : __fadd_rn(a, b);
  }
}

// The first n pairs.
__device__ __forceinline__ void turn_interleaved(float* x, const float* c, const float* s,
                                                 int n = 4) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= n) break;
    const float a = x[2 * i], b = x[2 * i + 1];
    x[2 * i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    x[2 * i + 1] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
  }
}

// A row in shared memory: rows of a warp start eight banks apart.
constexpr int kTurnPitch = kHeadDim + 8;

// Lane l's two chunks of a row (ra, rb as loaded), rotated into a and b.
// tile: the row's floats in shared memory (kTurnOdd, kTurnAny).
template <typename T, int TURN>
__device__ __forceinline__ void rotate16(float* a, float* b, const uint4& ra, const uint4& rb,
                                         const Int4Turn& t, float* tile) {
  unpack8<T>(ra, a);
  unpack8<T>(rb, b);
  const int l = t.l, pairs = t.pairs;
  if constexpr (TURN == kTurnHalf) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = a[i];
    turn_half<true>(a, b, t.c, t.s);
    turn_half<false>(b, o, t.c, t.s);
  } else if constexpr (TURN == kTurnInterleaved) {
    if (4 * l < pairs) turn_interleaved(a, t.c, t.s);
    if (32 + 4 * l < pairs) turn_interleaved(b, t.c + 4, t.s + 4);
  } else if constexpr (TURN == kTurnPart) {
    // Chunks c < n = pairs / 8 turn with c + n, n <= 4: all of them in a.
    const int n = pairs >> 3;
    const int peer = l < n ? l + n : l - n;
    uint4 oa;
    const uint32_t* wa = reinterpret_cast<const uint32_t*>(&ra);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint32_t*>(&oa)[i] = __shfl_sync(0xffffffffu, wa[i], peer & 7, 8);
    if (l < 2 * n) {
      float o[8];
      unpack8<T>(oa, o);
      if (l < n)
        turn_half<true>(a, o, t.c, t.s);
      else
        turn_half<false>(a, o, t.c, t.s);
    }
  } else if (TURN == kTurnOddInterleaved || (TURN == kTurnAny && t.interleaved)) {
    turn_interleaved(a, t.c, t.s, pairs - 4 * l);
    turn_interleaved(b, t.c + 4, t.s + 4, pairs - 32 - 4 * l);
  } else {
    static_assert(TURN == kTurnAny || TURN == kTurnOdd || TURN == kTurnOddInterleaved,
                  "the others have no tile");
    // Lane l turns pairs l, l + 8, ... of its row.
    float4* mine = reinterpret_cast<float4*>(tile + 8 * l);
    mine[0] = make_float4(a[0], a[1], a[2], a[3]);
    mine[1] = make_float4(a[4], a[5], a[6], a[7]);
    mine[16] = make_float4(b[0], b[1], b[2], b[3]);
    mine[17] = make_float4(b[4], b[5], b[6], b[7]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = l + 8 * i;
      if (8 * i >= pairs) break;
      if (j < pairs) {
        const float x = tile[j], y = tile[j + pairs];
        tile[j] = __fsub_rn(__fmul_rn(x, t.c[i]), __fmul_rn(y, t.s[i]));
        tile[j + pairs] = __fadd_rn(__fmul_rn(y, t.c[i]), __fmul_rn(x, t.s[i]));
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 x = mine[i], y = mine[16 + i];
      a[4 * i] = x.x; a[4 * i + 1] = x.y; a[4 * i + 2] = x.z; a[4 * i + 3] = x.w;
      b[4 * i] = y.x; b[4 * i + 1] = y.y; b[4 * i + 2] = y.z; b[4 * i + 3] = y.w;
    }
  }
}

// What an append warp knows of its token.
struct Int4Token {
  int64_t token, page, center;
  int tok;
};

// Quantise and store lane l's two chunks of one row of KV head h (a warp
// holds four rows; a row past the last stores nothing).
__device__ __forceinline__ void store_int4_row(const Int4AppendParams& p, const Int4Token& k,
                                               bool is_key, int h, int l, float* a, float* b) {
  uint32_t codes[2], meta[2];
  int4_quantize16(a, b, codes, meta);
  uint8_t* rec = p.records + (k.page * p.hkv + (h < p.hkv ? h : 0)) * kInt4Record;
  const bool store = h < p.hkv;
  if (is_key) {
    uint8_t* at = rec + k.tok * 64 + (l & 3) * 16 + (l >> 2) * 4;
    if (store) {
      *reinterpret_cast<uint32_t*>(at) = codes[0];
      *reinterpret_cast<uint32_t*>(at + 8) = codes[1];
    }
  } else {
    // Dims 4e .. 4e+3 of the four groups are 8 bytes: lanes 0-3 take those of
    // their chunks' first four dims, lanes 4-7 the other four.
    const uint32_t x = __shfl_xor_sync(0xffffffffu, codes[0], 4);
    const uint32_t y = __shfl_xor_sync(0xffffffffu, codes[1], 4);
    const uint2 w = l < 4 ? make_uint2(prmt(codes[0], x, 0x5410u), prmt(codes[1], y, 0x5410u))
                          : make_uint2(prmt(x, codes[0], 0x7632u), prmt(y, codes[1], 0x7632u));
    if (store)
      *reinterpret_cast<uint2*>(rec + kInt4Value + value_code_row(k.tok) * 64 + (l & 3) * 16 +
                                (l >> 2) * 8) = w;
  }
  // The token's four scales and midpoints as one 16-byte store.
  const uint32_t m1 = __shfl_down_sync(0xffffffffu, meta[0], 4, 8);
  const uint32_t m3 = __shfl_down_sync(0xffffffffu, meta[1], 4, 8);
  if (l == 0 && store)
    *reinterpret_cast<uint4*>(rec + (is_key ? kInt4KeyMeta : kInt4ValueMeta) + k.tok * 16) =
        make_uint4(prmt(meta[0], m1, 0x5410u), prmt(meta[1], m3, 0x5410u),
                   prmt(meta[0], m1, 0x7632u), prmt(meta[1], m3, 0x7632u));
}

template <typename T>
__device__ __forceinline__ void subtract_center(const Int4AppendParams& p, const Int4Token& k,
                                                const void* centers, int h, int l, float* a,
                                                float* b) {
  if (centers == nullptr) return;
  const T* row = static_cast<const T*>(centers) + (k.center * p.hkv + h) * kHeadDim + 8 * l;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float* x = j == 0 ? a : b;
    float y[8];
    unpack8<T>(load8<T, true>(row + 64 * j), y);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 r = add2(make_float2(x[i], x[i + 1]), make_float2(-y[i], -y[i + 1]));
      x[i] = r.x;
      x[i + 1] = r.y;
    }
  }
}

// `split` warps share one token.  A warp takes four rows at a time (8 lanes
// of two 8-dim chunks each: the partners of the half layout in one lane, so
// nothing is computed twice) and requests U times four query rows, or four
// key and four value rows, before it uses the first.  U = 2 where tokens
// alone fill the GPU: the table entries, slot and position are then read once
// per token, and with one or two KV heads (FEW) the four rows are of four or two
// tokens (42,000 tokens of 1 + 2 rows with the read: 65.8 -> 24.4 us); U = 1
// with a warp per four rows for few tokens, where latency is all.  Bound by
// HBM: 57,304 tokens of 32 + 16 FP16 rows (1.277 GB) take 206 us, 6.2 TB/s;
// with 16 lanes of one chunk per row, partners by shuffles, 241 us; with a
// clamp, a conversion and a shift per code, 321 us.
template <typename T, int TURN, int U, bool FEW>
__global__ void __launch_bounds__(256, 4)
    pg_rope_append_int4_kernel(const __grid_constant__ Int4AppendParams p) {
  constexpr bool FAST = TURN != kTurnAny;
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, sub = lane >> 3, l = lane & 7;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int shift = FEW ? p.row_shift : 2, step = 1 << shift, hs = sub & (step - 1);
  const int64_t tokens = p.split == 1 ? w : static_cast<uint32_t>(w) / p.split;  // w is small then
  const int part = static_cast<int>(w - tokens * p.split);
  Int4Token k;
  k.token = tokens << (2 - shift);
  if (k.token >= p.tokens) return;
  k.token += sub >> shift;
  bool live = true;
  if (FEW && k.token >= p.tokens) {
    k.token = p.tokens - 1;
    live = false;
  }
  pdl_wait_primary();
  const int slot = p.slots[k.token];
  int pos = p.positions[k.token];
  k.center = p.center_rows != nullptr ? p.center_rows[k.token] : 0;
  // The first query rows are asked for along with the token's indices.
  const T* q = static_cast<const T*>(p.q) + k.token * p.q_stride_t;
  const int nq = (p.hq + U * step - 1) / (U * step), nk = (p.hkv + step - 1) >> shift;
  uint4 ra[U], rb[U];
  auto load_rows = [&](const T* base, int stride, int heads, int unit, uint4& x, uint4& y) {
    const int h = step * unit + hs;
    const T* row = base + (h < heads ? h : heads - 1) * stride + 8 * l;
    x = load8<T, FAST>(row);
    y = load8<T, FAST>(row + 64);
  };
  auto load_queries = [&](int u) {
#pragma unroll
    for (int i = 0; i < U; ++i) load_rows(q, p.q_stride_h, p.hq, u * U + i, ra[i], rb[i]);
  };
  if (part < nq) load_queries(part);
  // Skipped tokens, and those that are reported, store nothing.
  live = live && slot >= 0;
  k.page = slot >> 4;
  k.tok = slot & 15;
  if (live && (k.page >= p.num_pages ||
               (p.key_center != nullptr && (k.center < 0 || k.center >= p.num_centers)))) {
    record_error(p.error_flag, kDevBadPageId);
    live = false;
  }
  if (live && (pos < 0 || pos >= p.table_rows)) {
    record_error(p.error_flag, kDevBadPosition);
    live = false;
  }
  if (FEW ? !__any_sync(0xffffffffu, live) : !live) return;
  if (FEW && !live) {
    pos = 0;
    k.page = k.center = 0;
  }
  Int4Turn t;
  t.cos_row = p.cos + pos * p.table_stride;
  t.sin_row = p.sin + pos * p.table_stride;
  t.pairs = p.pairs;
  t.l = l;
  t.interleaved = p.interleaved != 0;
  if constexpr (TURN == kTurnHalf || TURN == kTurnInterleaved || TURN == kTurnPart) {
    const int first = TURN == kTurnPart && 8 * l >= p.pairs ? 8 * l - p.pairs : 8 * l;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const int j = TURN == kTurnInterleaved ? 4 * l + 8 * i : first + i;
      const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 c = j < p.pairs ? __ldg(reinterpret_cast<const float4*>(t.cos_row + j)) : z;
      const float4 s = j < p.pairs ? __ldg(reinterpret_cast<const float4*>(t.sin_row + j)) : z;
      t.c[i] = c.x; t.c[i + 1] = c.y; t.c[i + 2] = c.z; t.c[i + 3] = c.w;
      t.s[i] = s.x; t.s[i + 1] = s.y; t.s[i + 2] = s.z; t.s[i + 3] = s.w;
    }
  }
  if constexpr (TURN == kTurnAny || TURN == kTurnOdd || TURN == kTurnOddInterleaved) {
    const bool quads = TURN == kTurnOddInterleaved || (TURN == kTurnAny && t.interleaved);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = quads ? 4 * l + 8 * (i & 4) + (i & 3) : l + 8 * i;
      t.c[i] = j < p.pairs ? __ldg(t.cos_row + j) : 0.f;
      t.s[i] = j < p.pairs ? __ldg(t.sin_row + j) : 0.f;
    }
  }
  constexpr bool kTile = TURN == kTurnAny || TURN == kTurnOdd;
  __shared__ __align__(16) float s_rows[kTile ? 8 : 1][kTile ? 4 * kTurnPitch : 4];
  float* tile = kTile ? &s_rows[threadIdx.x >> 5][sub * kTurnPitch] : nullptr;
  const T* kr = static_cast<const T*>(p.k) + k.token * p.k_stride_t;
  const T* vr = static_cast<const T*>(p.v) + k.token * p.v_stride_t;
  // A last unit's missing rows repeat the last row and store nothing.
  auto turn_and_store = [&](float* a, float* b, const uint4& x, const uint4& y, T* out,
                            bool store) {
    rotate16<T, TURN>(a, b, x, y, t, tile);
    if (store) {
      store8<T, FAST>(out + 8 * l, a);
      store8<T, FAST>(out + 64 + 8 * l, b);
    }
  };
  auto append_rows = [&](const uint4& x, const uint4& y, bool is_key, int unit) {
    const int h = step * unit + hs, hc = h < p.hkv ? h : p.hkv - 1;
    float a[8], b[8];
    if (is_key) {
      turn_and_store(a, b, x, y,
                     static_cast<T*>(p.rotated_k) + k.token * p.rk_stride_t + hc * p.rk_stride_h,
                     p.rotated_k != nullptr && (!FEW || live) && h < p.hkv);
    } else {
      unpack8<T>(x, a);
      unpack8<T>(y, b);
    }
    subtract_center<T>(p, k, is_key ? p.key_center : p.value_center, hc, l, a, b);
    store_int4_row(p, k, is_key, !FEW || live ? h : p.hkv, l, a, b);
  };
  T* rq = static_cast<T*>(p.rotated_q) + k.token * p.rq_stride_t;
  for (int u = part; u < nq; u += p.split) {
    if (u != part) load_queries(u);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = step * (u * U + i) + hs;
      if (step * (u * U + i) >= p.hq) break;
      const int hc = h < p.hq ? h : p.hq - 1;
      float a[8], b[8];
      turn_and_store(a, b, ra[i], rb[i], rq + hc * p.rq_stride_h,
                     (!FEW || live) && h < p.hq);
    }
  }
  // This warp's first unit past the query rows.
  const int first = part >= nq ? part - nq : (p.split - (nq - part) % p.split) % p.split;
  if constexpr (U > 1) {
    for (int u = first; u < nk; u += p.split) {
      load_rows(kr, p.k_stride_h, p.hkv, u, ra[0], rb[0]);
      load_rows(vr, p.v_stride_h, p.hkv, u, ra[1], rb[1]);
      append_rows(ra[0], rb[0], true, u);
      append_rows(ra[1], rb[1], false, u);
    }
  } else {
    for (int u = first; u < 2 * nk; u += p.split) {
      const bool is_key = u < nk;
      const int unit = u - (is_key ? 0 : nk);
      load_rows(is_key ? kr : vr, is_key ? p.k_stride_h : p.v_stride_h, p.hkv, unit, ra[0],
                rb[0]);
      append_rows(ra[0], rb[0], is_key, unit);
    }
  }
}

struct Int4ReadParams {
  const uint8_t* records;
  int64_t num_pages;
  const int32_t* slots;
  int64_t tokens;
  int32_t hkv;
  void* key;      // [T, Hkv, 128]
  void* value;    // [T, Hkv, 128]
  int* error_flag;
};

// A warp reads 2 U rows (KV heads of consecutive tokens), 16 lanes per row's
// key and value, with everything requested before it is used; skipped slots
// read as zeros.  U = 4 where the rows alone fill the GPU, as in the append.
// SAME: the KV heads are a multiple of 2 U, so a warp's rows are one token's
// (57,304 tokens of 8 heads: 57 us, 63 us with the tokens followed).
template <typename T, int U, bool SAME>
__global__ void __launch_bounds__(256)
    pg_int4_read_kernel(const __grid_constant__ Int4ReadParams p) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, half = lane >> 4, m = lane & 15, grp = m >> 2;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int64_t end = p.tokens * p.hkv;
  if (2 * U * w >= end) return;
  const int64_t first = 2 * U * w + half;  // of this half warp
  // A 32-bit division where the index allows it.
  int64_t token = first < (int64_t(1) << 31)
                      ? static_cast<int64_t>(static_cast<uint32_t>(first) / p.hkv)
                      : first / p.hkv;
  int h = static_cast<int>(first - token * p.hkv);
  pdl_wait_primary();
  int slot = -1;
  auto load_slot = [&](bool held) {
    slot = held ? p.slots[token] : -1;
    if (slot >= 0 && (slot >> 4) >= p.num_pages) {
      record_error(p.error_flag, kDevBadPageId);
      slot = -1;
    }
  };
  if constexpr (SAME) load_slot(true);
  uint32_t codes[U][2];
  __half s[U][2], mid[U][2];
#pragma unroll
  for (int i = 0; i < U; ++i) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[i][kv] = 0u;
      s[i][kv] = mid[i][kv] = __ushort_as_half(0);
    }
    if constexpr (!SAME) load_slot(first + 2 * i < end);
    if (slot >= 0) {
      const int tok = slot & 15;
      const uint8_t* rec =
          p.records + (static_cast<int64_t>(slot >> 4) * p.hkv + h) * kInt4Record;
      const __half* km = reinterpret_cast<const __half*>(rec + kInt4KeyMeta + tok * 16) + grp;
      const __half* vm = reinterpret_cast<const __half*>(rec + kInt4ValueMeta + tok * 16) + grp;
      codes[i][0] = *reinterpret_cast<const uint32_t*>(rec + tok * 64 + (m & 3) * 16 + grp * 4);
      // One word of two groups' four dims; another lane's makes both halves.
      codes[i][1] = *reinterpret_cast<const uint32_t*>(
          rec + kInt4Value + value_code_row(tok) * 64 + (m & 3) * 16 + (grp & 1) * 8 +
          (grp >> 1) * 4);
      s[i][0] = km[0];
      mid[i][0] = km[4];
      s[i][1] = vm[0];
      mid[i][1] = vm[4];
    }
    h += 2;
    if constexpr (!SAME)
      for (; h >= p.hkv; h -= p.hkv) ++token;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, codes[i][1], 4);
    codes[i][1] = (grp & 1) ? prmt(other, codes[i][1], 0x7632u) : prmt(codes[i][1], other, 0x5410u);
    const int64_t row = first + 2 * i;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      T* out = static_cast<T*>(kv == 0 ? p.key : p.value) + row * kHeadDim + 8 * m;
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
      if (!SAME && row >= end) continue;
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
