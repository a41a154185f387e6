// Decode attention over the 4-bit paged cache (record layout: pg_int4.cuh):
// one query token per request, a GQA group of up to 8 query heads per KV
// head, split over the planner's work items (request, KV head, run of pages).
//
// Every warp owns a ring of records in shared memory (one 2560-byte bulk copy
// per page) and computes, per page of 16 tokens,
//   S^T = K (16 tok x 128) . Q^T (128 x 8 rows)
//   O^T += V^T (128 x 16 tok) . P^T (16 tok x 8 rows)
// on the FP16 tensor path with FP32 accumulators.  The codes need no
// conversion: a code z in the low bits of a half is the subnormal z 2^-24
// (z 2^-20 one nibble higher), exact in the product, so one AND makes two
// operands.  A word of key codes holds 8 dims of one token and its nibble i
// and i + 4 are one operand register; the query's odd dims are divided by 16
// to match.  The rows are first scaled by a power of two that brings their
// largest element to [512, 1024), so that this division loses nothing.
//
// The scales and midpoints come after the products.  With qs_g = the sum of
// q over group g's 32 dims,
//   score = sum_g s_g (sum_d q_d z_d - 8 qs_g) + m_g qs_g
// -8 qs_g is the initial accumulator of group g's products, and the last
// term one TF32 product with qs split in two.  For the values
//   O_d = sum_t (P_t s_tg) z_td - 8 sum_t (P_t s_tg) + sum_t P_t m_tg
// where P s is formed in FP32 and rounded once to FP16, and the sum times 8
// comes from tensor-core products of the same rounded operands, so that a
// rounding of P s weighs (z - 8) s and not z s; the last sum is FP32.  P =
// 2^(score - ref), all sums relative to a row's reference: not its largest score,
// which left small scales beside a dominant token of the warp in subnormal halves
// (700 tokens, one of zero values 10 nats above the rest: 3.7 % off, now 0.2 %, which
// is the FP16 output's step; values of deviation 0.001: 4.7e-4, now 2.3e-4), but that
// and the largest value scale, so that P s fills the half's range.  What is left is
// half a subnormal step, 2^-37 of (largest weight) x (largest scale), per token.  It
// costs 1-2 %.
//
// Bound by the compute of a page, not by its bytes: eight ragged requests of
// 300,000 tokens in all (384 MB) take 76.3 us in a captured loop (82-87 us per
// call, sustained, at the power cap's clocks), the copies alone 60.1 us.  A
// tensor instruction costs about 6 issue cycles here whatever else runs (its
// pipe is 30 % busy), an AND 2, so the layouts above save instructions first.
// 49,152 tokens of one request take 17.7 us (9.7 us of bytes): 24,576 pages and
// heads at the same rate are 12.5 us, the rest is the first pages' latency and the
// join's launch.
#pragma once

#include "pg_decode_core.cuh"
#include "pg_int4.cuh"

namespace pg {

struct Int4DecodeParams {
  const void* q;
  int64_t q_stride_b, q_stride_h;
  const uint8_t* records;
  int32_t num_pages;
  const int32_t* indices;
  const int32_t* last_len;
  const DecodeItem* items;
  const int32_t* item_slots;  // where an item's partial state goes (null: its index)
  const int32_t* item_off;
  int32_t num_items, batch, hkv, group;
  float sm_scale_log2;
  float* part_o;    // [num_items, group, 128]
  float* part_lse;  // [num_items, group]
  int32_t* counter; // items handed out past the grid; zero between launches
  int32_t final_mode;
  void* out;
  int64_t out_stride_b, out_stride_h;
  float* lse_out;
  const void* value_center;  // [B, Hkv, 128] or null
  int64_t vc_stride_b;
  int* error_flag;
};

constexpr int kInt4Warps = 4;
constexpr int kInt4Slots = 2;  // pairs of pages in a warp's ring
constexpr int kInt4CtasPerSm = 3;
constexpr int kInt4RingBytes = kInt4Slots * 2 * kInt4Record;
// The warps' rings, then their barriers, then the combine buffer (its own, so
// that the next item's pages can arrive while it is in use).
constexpr int kInt4CombineFloats = kInt4Warps * (16 + 8 * kCoStride);
constexpr int kInt4CombineAt = kInt4Warps * (kInt4RingBytes + kInt4Slots * 8);
constexpr int kInt4SmemBytes = kInt4CombineAt + kInt4CombineFloats * 4;
static_assert(kInt4CombineAt % 16 == 0, "the combine buffer is read in 16-byte rows");
// Pages per warp asked of the L2 ahead of the dependency wait: 49,152 tokens
// 18.2 -> 17.6 us (16 pages would cost 0.5 us).
constexpr int kInt4Prefetch = 4;
// A row's reference before its first token: finite, so that masked scores of -inf
// give weights of 0.
constexpr float kInt4NoRef = -3e38f;
// Where a reference is raised the largest P s is 2^12 to 2^13, 2^26 above the least
// normal half, and later ones may pass it by the slack: P s < 2^15.
constexpr float kInt4Headroom = 12.f, kInt4Slack = 2.f;
// Scores past this are taken without their scale (P <= 1): their own steps are what
// counts.
constexpr float kInt4FarScore = 0x1p22f;

// Largest of a token's four value scales, as the half's bits.
__device__ __forceinline__ uint32_t int4_largest_scale(const uint8_t* scales) {
  const uint2 x = *reinterpret_cast<const uint2*>(scales);
  const __half2 pair = __hmax2(*reinterpret_cast<const __half2*>(&x.x),
                               *reinterpret_cast<const __half2*>(&x.y));
  return __half_as_ushort(__hmax(__low2half(pair), __high2half(pair)));
}

// D = A(16x16 f16) * B(16x8 f16) + C.
__device__ __forceinline__ void mma_16816_c(float* d, uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                            float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
        "f"(c3));
}
__device__ __forceinline__ void mma_16816_acc(float* d, uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  mma_16816_c(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}
// D = A(16x8 tf32) * B(8x8 tf32).
__device__ __forceinline__ void mma_1688_tf32(float* d, float a0, float a1, float a2, float a3,
                                              float b0, float b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)),
        "r"(__float_as_uint(a3)), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)), "f"(0.f));
}
// Rounded to TF32's 11 bits (the product itself would cut the rest off): two
// such parts leave 2^-24 of a value.
__device__ __forceinline__ float round_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return __uint_as_float(r);
}
// The 8x8 matrix of halves whose row g lane (g, t) holds columns 2t, 2t+1
// of, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ int load_volatile(const int32_t* p) {
  int v;
  asm volatile("ld.volatile.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Bring `bytes` (a multiple of 16, 16-byte aligned) into the L2.
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                   reinterpret_cast<uint64_t>(p)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ float2 half2_float2(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

constexpr uint32_t kNibble0 = 0x000f000fu;  // z 2^-24 as a subnormal half
constexpr uint32_t kNibble1 = 0x00f000f0u;  // z 2^-20
constexpr uint32_t kNibbles = 0x00ff00ffu;  // (z0 + 16 z1) 2^-24

// One warp's query operands (row g) and constants.
struct Int4Query {
  uint32_t b[16];     // B operands of the 8 key steps
  float c0[4][2];     // -8 qs_g 2^-24 of rows 2t, 2t+1
  float qs_hi, qs_lo; // qs_t 2^-24 of row g in two TF32 parts
  float cr[2];        // score factor of rows 2t, 2t+1 (log2 units)
};

struct Int4State {
  float ref[2], l[2];  // reference and sum of rows 2t, 2t+1's weights (this lane's tokens)
  // Tile 2j + e, rows g: dims d = 32j + 4g + 2e; rows g + 8: d and d + 1 as
  // z_d + 16 z_(d+1) (one AND less than the two nibbles apart).
  float o[8][4];
  float sums[4];     // row k: sum of part k's rounded P s
  float mid[4][2];   // sum P m of part k (this lane's tokens); NARROW: k < 2
};

// NARROW (GQA group <= 4): columns 4-7 of the products repeat the query rows
// 0-3, so that one B operand of the value products holds two dim groups'
// weights (columns 0-3 with group 2i's scale, 4-7 with group 2i + 1's): half
// the multiplies, conversions and transposes, and each value product still
// reads its own columns.
template <typename T, bool NARROW>
__device__ __forceinline__ void load_query_int4(const Int4DecodeParams& p, int r, int h, int g,
                                                int t, Int4Query& iq) {
  float x[4][8];
  float big = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
    const int q = NARROW ? g & 3 : g;
    if (q < p.group) {
      const T* row = static_cast<const T*>(p.q) + r * p.q_stride_b +
                     static_cast<int64_t>(h * p.group + q) * p.q_stride_h + 32 * j + 8 * t;
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *(reinterpret_cast<const uint32_t*>(row) + i);
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[j][i] = to_float<T>(e[i]);
        big = fmaxf(big, fabsf(x[j][i]));
      }
    }
  }
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
  // big = a 2^e with a in [1, 2): scale by 2^(9 - e).  Rows of zeros and
  // rows with an infinity (whose results are NaN) keep their scale; below
  // 2^-90 a row's scores are nothing.
  int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
  e = (big == 0.f || e > 127) ? 9 : max(e, -90);
  const float up = __uint_as_float(static_cast<uint32_t>(127 + 9 - e) << 23);
  float qs[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[j][i] *= up;
      sum += x[j][i];
    }
    iq.b[4 * j + 0] = pack_half2(x[j][0], x[j][4]);
    iq.b[4 * j + 1] = pack_half2(x[j][1] * 0.0625f, x[j][5] * 0.0625f);
    iq.b[4 * j + 2] = pack_half2(x[j][2], x[j][6]);
    iq.b[4 * j + 3] = pack_half2(x[j][3] * 0.0625f, x[j][7] * 0.0625f);
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    qs[j] = sum * 0x1p-24f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      iq.c0[j][i] = -8.f * __shfl_sync(0xffffffffu, qs[j], 4 * (2 * t + i));
  }
  const float mine = t == 0 ? qs[0] : t == 1 ? qs[1] : t == 2 ? qs[2] : qs[3];
  iq.qs_hi = round_tf32(mine);
  iq.qs_lo = round_tf32(mine - iq.qs_hi);
  // 2^24 undoes the subnormal codes.
  const float down = p.sm_scale_log2 * 0x1p24f / up;
#pragma unroll
  for (int i = 0; i < 2; ++i) iq.cr[i] = __shfl_sync(0xffffffffu, down, 4 * (2 * t + i));
}

// Two pages at rec and rec + kInt4Record in shared memory.  MASKED: only the
// first valid[i] tokens count (the others' scales may hold anything).
template <bool NARROW, bool MASKED>
__device__ __forceinline__ void pages_int4(const uint8_t* rec, const Int4Query& iq, Int4State& st,
                                           const int* valid, int g, int t) {
  const int lane = 4 * g + t;
  // Scores of tokens g (s[i][0], s[i][1]: rows 2t, 2t+1) and g + 8.
  float s[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* page = rec + i * kInt4Record;
    {
      const __half* mid = reinterpret_cast<const __half*>(page + kInt4KeyMeta + 8) + t;
      const float m0 = __half2float(mid[8 * g]), m1 = __half2float(mid[8 * g + 64]);
      mma_1688_tf32(s[i], m0, m1, m0, m1, iq.qs_hi, iq.qs_lo);
    }
    const uint4 ka = lds128(page, 16 * lane), kb = lds128(page, 512 + 16 * lane);
    const uint2 sa = *reinterpret_cast<const uint2*>(page + kInt4KeyMeta + 16 * g);
    const uint2 sb = *reinterpret_cast<const uint2*>(page + kInt4KeyMeta + 128 + 16 * g);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = j == 0 ? ka.x : j == 1 ? ka.y : j == 2 ? ka.z : ka.w;
      const uint32_t b = j == 0 ? kb.x : j == 1 ? kb.y : j == 2 ? kb.z : kb.w;
      float acc[4];
      mma_16816_c(acc, a & kNibble0, b & kNibble0, a & kNibble1, b & kNibble1, iq.b[4 * j],
                  iq.b[4 * j + 1], iq.c0[j][0], iq.c0[j][1], iq.c0[j][0], iq.c0[j][1]);
      mma_16816_acc(acc, (a >> 8) & kNibble0, (b >> 8) & kNibble0, (a >> 8) & kNibble1,
                    (b >> 8) & kNibble1, iq.b[4 * j + 2], iq.b[4 * j + 3]);
      const float2 fa = half2_float2(j < 2 ? sa.x : sa.y);
      const float2 fb = half2_float2(j < 2 ? sb.x : sb.y);
      const float wa = (j & 1) ? fa.y : fa.x, wb = (j & 1) ? fb.y : fb.x;
      s[i][0] = fmaf(wa, acc[0], s[i][0]);
      s[i][1] = fmaf(wa, acc[1], s[i][1]);
      s[i][2] = fmaf(wb, acc[2], s[i][2]);
      s[i][3] = fmaf(wb, acc[3], s[i][3]);
    }
  }
  // In log2 units, rounded here: the maximum below and the differences from it
  // are of the same numbers, so that however large they are (FP32 steps of many
  // units) the largest gives a weight of 1.
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = __fmul_rn(s[i][j], iq.cr[j & 1]);
  if constexpr (MASKED) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (g >= valid[i]) s[i][0] = s[i][1] = kNegInf;
      if (g + 8 >= valid[i]) s[i][2] = s[i][3] = kNegInf;
    }
  }
  // Lane 16 i + tok looks at the value scales of page i's token tok.  The exponent of
  // the pages' largest (of 2^-24 where all are zero; finite), less the headroom: a
  // whole number, so that the weight of a largest score is a power of two and adds
  // no rounding to its scale.
  uint32_t scale = int4_largest_scale(rec + (lane >> 4) * kInt4Record + kInt4ValueMeta +
                                      16 * (lane & 15));
  if constexpr (MASKED)
    if ((lane & 15) >= (lane < 16 ? valid[0] : valid[1])) scale = 0u;
  scale = min(max(__reduce_max_sync(0xffffffffu, scale), 1u), 0x7bffu);
  scale = __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(scale))));
  const float ls =
      __uint_as_float(0x4b000000u | (scale >> 23)) - (8388608.f + 127.f + kInt4Headroom);
  const float lm0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
  const float lm1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
  if (__any_sync(0xffffffffu, lm0 + (ls - kInt4Slack) > st.ref[0] ||
                                  lm1 + (ls - kInt4Slack) > st.ref[1] ||
                                  !(fmaxf(fabsf(lm0), fabsf(lm1)) <= kInt4FarScore))) {
    const float top[2] = {warp_max_xor_g(lm0), warp_max_xor_g(lm1)};
    float a[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float ref =
          fmaxf(st.ref[i], fabsf(top[i]) <= kInt4FarScore ? top[i] + ls : top[i]);
      a[i] = st.ref[i] == kInt4NoRef ? 1.f : fast_exp2(st.ref[i] - ref);
      st.ref[i] = ref;
      st.l[i] *= a[i];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[j][i] *= a[i & 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) st.sums[i] *= a[i & 1];
#pragma unroll
    for (int k = 0; k < (NARROW ? 2 : 4); ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) st.mid[k][i] *= a[i];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* page = rec + i * kInt4Record;
    const float p0 = fast_exp2(s[i][0] - st.ref[0]);
    const float p1 = fast_exp2(s[i][1] - st.ref[1]);
    const float p2 = fast_exp2(s[i][2] - st.ref[0]);
    const float p3 = fast_exp2(s[i][3] - st.ref[1]);
    st.l[0] += p0 + p2;
    st.l[1] += p1 + p3;
    // Value scales and midpoints of tokens g and g + 8: four groups', or
    // (NARROW) the two of this lane's columns.
    constexpr int kParts = NARROW ? 2 : 4;
    float wa[kParts], wb[kParts];
    {
      float ma[kParts], mb[kParts];
      const uint8_t* at = page + kInt4ValueMeta + 16 * g;
      if constexpr (NARROW) {
        const __half* sa = reinterpret_cast<const __half*>(at) + (t >> 1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          wa[k] = __half2float(sa[2 * k]);
          ma[k] = __half2float(sa[4 + 2 * k]);
          wb[k] = __half2float(sa[64 + 2 * k]);
          mb[k] = __half2float(sa[68 + 2 * k]);
        }
      } else {
        const uint4 x = lds128(at, 0), y = lds128(at, 128);
        const float2 a0 = half2_float2(x.x), a1 = half2_float2(x.y);
        const float2 a2 = half2_float2(x.z), a3 = half2_float2(x.w);
        const float2 b0 = half2_float2(y.x), b1 = half2_float2(y.y);
        const float2 b2 = half2_float2(y.z), b3 = half2_float2(y.w);
        wa[0] = a0.x; wa[1] = a0.y; wa[kParts - 2] = a1.x; wa[kParts - 1] = a1.y;
        ma[0] = a2.x; ma[1] = a2.y; ma[kParts - 2] = a3.x; ma[kParts - 1] = a3.y;
        wb[0] = b0.x; wb[1] = b0.y; wb[kParts - 2] = b1.x; wb[kParts - 1] = b1.y;
        mb[0] = b2.x; mb[1] = b2.y; mb[kParts - 2] = b3.x; mb[kParts - 1] = b3.y;
      }
      if constexpr (MASKED) {
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
          if (g >= valid[i]) wa[k] = ma[k] = 0.f;
          if (g + 8 >= valid[i]) wb[k] = mb[k] = 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        st.mid[k][0] = fmaf(p0, ma[k], fmaf(p2, mb[k], st.mid[k][0]));
        st.mid[k][1] = fmaf(p1, ma[k], fmaf(p3, mb[k], st.mid[k][1]));
      }
    }
    // Codes of tokens 2t, 2t+1 and 2t+8, 2t+9.
    const uint8_t* codes = page + kInt4Value + 64 * t + 8 * g;
    const uint2 c00 = *reinterpret_cast<const uint2*>(codes);
    const uint2 c01 = *reinterpret_cast<const uint2*>(codes + 256);
    const uint2 c10 = *reinterpret_cast<const uint2*>(codes + 512);
    const uint2 c11 = *reinterpret_cast<const uint2*>(codes + 768);
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const uint32_t b0 = transpose_8x8(pack_half2(p0 * wa[k], p1 * wa[k]));
      const uint32_t b1 = transpose_8x8(pack_half2(p2 * wb[k], p3 * wb[k]));
      const uint32_t one = g == k ? 0x3c003c00u : 0u;
      mma_16816_acc(st.sums, one, 0u, one, 0u, b0, b1);
#pragma unroll
      for (int e = 0; e < 4 / kParts; ++e) {
        const int j = k * (4 / kParts) + e;
        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
        const uint32_t x = j < 2 ? prmt(c00.x, c01.x, sel) : prmt(c00.y, c01.y, sel);
        const uint32_t y = j < 2 ? prmt(c10.x, c11.x, sel) : prmt(c10.y, c11.y, sel);
        mma_16816_acc(st.o[2 * j], x & kNibble0, x & kNibbles, y & kNibble0, y & kNibbles, b0,
                      b1);
        const uint32_t xh = prmt(x, 0u, 0x4341u), yh = prmt(y, 0u, 0x4341u);
        mma_16816_acc(st.o[2 * j + 1], xh & kNibble0, xh, yh & kNibble0, yh, b0, b1);
      }
    }
  }
}

// m + log2(sum) of a positive sum.  Its power of two goes to m, which is coarser
// for it, so that the logarithm is of a number in [1, 2).
__device__ __forceinline__ float int4_lse(float m, float sum) {
  const int e = min(static_cast<int>(__float_as_uint(sum) >> 23) - 127, 126);
  const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  return (m + static_cast<float>(e)) + fast_log2(sum * down);
}

// Output row element (v, base-2 lse): the value centre is added where the
// row attended to anything.
template <typename T>
__device__ __forceinline__ void int4_store_out(const Int4DecodeParams& p, int r, int h, int q,
                                               int d, float v, float lse) {
  if (p.value_center != nullptr && lse != kNegInf)
    v += to_float<T>(static_cast<const T*>(p.value_center)[r * p.vc_stride_b + h * kHeadDim + d]);
  const int qh = h * p.group + q;
  static_cast<T*>(p.out)[r * p.out_stride_b + qh * p.out_stride_h + d] = from_float<T>(v);
  if (d == 0 && p.lse_out != nullptr)
    p.lse_out[static_cast<int64_t>(r) * (p.hkv * p.group) + qh] = lse;
}

// A warp's share of a work item: every kInt4Warps-th page from its own, one
// per lane at most (the planner's limit for four warps).
__device__ __forceinline__ int int4_warp_pages(int count, int warp) {
  const int n = count & 0x7fffffff;
  const int mine = n > warp ? (n - warp + kInt4Warps - 1) / kInt4Warps : 0;
  return mine < 32 ? mine : 32;
}

// Persistent: of G blocks, block b takes items b, 2 G - 1 - b and 2 G + b, then
// the next item that no block has (a counter, which the last block to ask sets
// back to zero).  An item's page ids are read, and its first pages requested,
// before the item ahead of it is finished, so only the first item of a block
// waits for them; a block must therefore know an item two ahead.  Handing out
// the second and third items that early gave some blocks three before others
// had two: 16 x 3,923 pages in 880 items 45.4 us, 36.4 us so; and asking later,
// halfway through an item, cost 5 % wherever blocks have many.  Which block
// takes an item changes no result: partial states are stored by item.  The
// plan lists the largest items first, so that the last ones are short and the
// blocks of one SM get items of all sizes.
template <typename T, bool NARROW>
__global__ void __launch_bounds__(kInt4Warps * 32, kInt4CtasPerSm)
    pg_decode_int4_kernel(const __grid_constant__ Int4DecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem_int4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem_int4 + warp * kInt4RingBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_int4 + kInt4Warps * kInt4RingBytes) +
                   warp * kInt4Slots;
  if (lane == 0) {
    for (int i = 0; i < kInt4Slots; ++i) mbar_init(bars + i, 1);
    fence_barrier_init();
  }
  __syncwarp();
  pdl_launch_dependents();
  __shared__ int s_next[2];  // the item after the next one, by parity
  const int grid = gridDim.x;
  auto take = [&] {  // one thread, for each item but the first that another one follows
    const int taken = atomicAdd(p.counter, 1);
    if (taken == p.num_items - 2 * grid - 1) *p.counter = 0;
    return taken + 3 * grid;
  };
  int index = blockIdx.x;
  DecodeItem item = p.items[index];  // plan data
  int n_w = int4_warp_pages(item.count, warp);
  // Pages and page ids may be written by the kernel just before: what counts
  // is read after the wait.  Ahead of it the warp only asks the L2 for its
  // first pages, under ids that may be stale.
  if (lane < n_w && lane < kInt4Prefetch) {
    const int guess = load_volatile(p.indices + item.idx_begin + warp + kInt4Warps * lane);
    if (guess >= 0 && guess < p.num_pages)
      prefetch_l2(p.records + (static_cast<int64_t>(guess) * p.hkv + (item.head_seg & 0xffff)) *
                                  kInt4Record,
                  kInt4Record);
  }
  pdl_wait_primary();
  // Lane u holds the record of the warp's page u (at most 32 per warp) and
  // copies it itself; ids outside the pool leave their page out.
  const uint8_t* mine = nullptr;
  uint32_t bad_pages = 0;
  auto resolve = [&](int id, const DecodeItem& it, int pages) {
    const bool bad = lane < pages && (id < 0 || id >= p.num_pages);
    if (bad) {
      record_error(p.error_flag, kDevBadPageId);
      id = 0;
    }
    bad_pages = __ballot_sync(0xffffffffu, bad);
    mine = lane < pages ? p.records + (static_cast<int64_t>(id) * p.hkv +
                                       (it.head_seg & 0xffff)) * kInt4Record
                        : nullptr;
  };
  // Pair u's copies into slot `at`: its first lane announces the bytes.
  auto issue = [&](int u, int at) {
    if (lane == 2 * u)
      mbar_arrive_expect_tx(bars + at, 2 * u + 1 < n_w ? 2 * kInt4Record : kInt4Record);
    __syncwarp();
    if ((lane >> 1) == u && mine != nullptr)
      bulk_load_hint(ring + (2 * at + (lane & 1)) * kInt4Record, mine, kInt4Record, bars + at,
                     l2_evict_first_policy());
  };
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;  // no wait of this warp has run out
  // The item's first pairs go to the slots from `slot` on.
  auto issue_first = [&] {
    int at = slot;
    for (int u = 0; u < kInt4Slots && 2 * u < n_w; ++u) {
      issue(u, at);
      if (++at == kInt4Slots) at = 0;
    }
  };
  resolve(lane < n_w ? load_volatile(p.indices + item.idx_begin + warp + kInt4Warps * lane) : 0,
          item, n_w);
  issue_first();
  int next_index = 2 * grid - 1 - index;
  bool first = true;
  for (int parity = 1;; parity ^= 1) {
    const int r = item.request, h = item.head_seg & 0xffff;
    const int n_pages = item.count & 0x7fffffff, n_pairs = (n_w + 1) >> 1;
    if (n_pages > 32 * kInt4Warps) record_error(p.error_flag, kDevBadPageId);
    const bool more = next_index < p.num_items;
    if (more && !first && threadIdx.x == 0) s_next[parity] = take();
    // Tokens that count in the warp's last page, if it is the request's last.
    int tail = kPage;
    if (item.count < 0 && n_w > 0 && warp + kInt4Warps * (n_w - 1) == n_pages - 1) {
      const int lv = __ldg(p.last_len + r);
      tail = lv < 0 ? 0 : (lv > kPage ? kPage : lv);
    }
    Int4Query iq;
    load_query_int4<T, NARROW>(p, r, h, g, t, iq);
    int next_id = 0;
    if (more) {
      const DecodeItem next = p.items[next_index];
      if (lane < int4_warp_pages(next.count, warp))
        next_id = load_volatile(p.indices + next.idx_begin + warp + kInt4Warps * lane);
    }
    Int4State st;
    st.l[0] = st.l[1] = 0.f;
    st.ref[0] = st.ref[1] = kInt4NoRef;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[j][i] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) st.sums[i] = st.mid[i][0] = st.mid[i][1] = 0.f;

    // Pairs of whole pages; the others (the last pair at most, unless ids were
    // bad) are masked.
    const int n_whole = bad_pages != 0u ? 0 : (n_w - (tail != kPage)) >> 1;
    for (int u = 0; u < n_pairs && ok; ++u) {
      const bool waited = mbar_wait_bounded(bars + slot, phase);
      if (!__all_sync(0xffffffffu, waited)) {
        // Let the copies in flight land; this warp copies nothing more.
        record_error(p.error_flag, kDevWaitTimeout);
        int at = slot;
        uint32_t ph = phase;
        for (int v = u; v < n_pairs && v < u + kInt4Slots; ++v) {
          mbar_wait_bounded(bars + at, ph);
          if (++at == kInt4Slots) {
            at = 0;
            ph ^= 1u;
          }
        }
        ok = false;
        break;
      }
      const uint8_t* pages = ring + 2 * slot * kInt4Record;
      if (u < n_whole) {
        pages_int4<NARROW, false>(pages, iq, st, nullptr, g, t);
      } else {
        int valid[2] = {kPage, kPage};
        if (u == n_pairs - 1) valid[n_w & 1 ? 0 : 1] = tail;
        if (u == n_pairs - 1 && (n_w & 1)) valid[1] = 0;
        if ((bad_pages >> (2 * u)) & 1u) valid[0] = 0;
        if ((bad_pages >> (2 * u)) & 2u) valid[1] = 0;
        pages_int4<NARROW, true>(pages, iq, st, valid, g, t);
      }
      __syncwarp();
      if (u + kInt4Slots < n_pairs) issue(u + kInt4Slots, slot);
      if (++slot == kInt4Slots) {
        slot = 0;
        phase ^= 1u;
      }
    }
    if (more) {
      item = p.items[next_index];
      n_w = ok ? int4_warp_pages(item.count, warp) : 0;
      resolve(next_id, item, n_w);
      issue_first();
    }

    // Warp totals over the 8 token lanes, then the output rows.
    const float l0 = warp_sum_xor_g(st.l[0]), l1 = warp_sum_xor_g(st.l[1]);
#pragma unroll
    for (int k = 0; k < (NARROW ? 2 : 4); ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) st.mid[k][i] = warp_sum_xor_g(st.mid[k][i]);
    __syncthreads();  // the combine buffer is free
    float* cm = reinterpret_cast<float*>(smem_int4 + kInt4CombineAt);  // [W][8]
    float* cl = cm + kInt4Warps * 8;                                   // [W][8]
    float* co = cl + kInt4Warps * 8;                                   // [W][8][kCoStride]
    if (g == 0) {
      cm[warp * 8 + 2 * t] = ok ? st.ref[0] : kInt4NoRef;
      cm[warp * 8 + 2 * t + 1] = ok ? st.ref[1] : kInt4NoRef;
      cl[warp * 8 + 2 * t] = ok ? l0 : 0.f;
      cl[warp * 8 + 2 * t + 1] = ok ? l1 : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // The row of this lane's column, and its sums (shuffled by every lane).
      const int q = NARROW ? (2 * t + i) & 3 : 2 * t + i;
      float* row = co + (warp * 8 + q) * kCoStride;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = NARROW ? j >> 1 : j;
        const float add = st.mid[k][i] - 8.f * __shfl_sync(0xffffffffu, st.sums[i], 4 * k + t);
        if (q < p.group && (!NARROW || (t >> 1) == (j & 1))) {
          const float* a = st.o[2 * j];
          const float* b = st.o[2 * j + 1];
          *reinterpret_cast<float4*>(row + 32 * j + 4 * g) =
              make_float4(fmaf(a[i], 0x1p24f, add), fmaf(a[2 + i] - a[i], 0x1p20f, add),
                          fmaf(b[i], 0x1p24f, add), fmaf(b[2 + i] - b[i], 0x1p20f, add));
        }
      }
    }
    __syncthreads();
    // Thread -> four dims of one row.
    for (int idx = threadIdx.x; idx < p.group * 32; idx += blockDim.x) {
      const int q = idx >> 5, d = 4 * (idx & 31);
      float M = kNegInf, L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kInt4Warps; ++w) M = fmaxf(M, cm[w * 8 + q]);
#pragma unroll
      for (int w = 0; w < kInt4Warps; ++w) {
        if (cl[w * 8 + q] == 0.f) continue;
        const float e = fast_exp2(cm[w * 8 + q] - M);
        const float4 o = *reinterpret_cast<const float4*>(co + (w * 8 + q) * kCoStride + d);
        L += cl[w * 8 + q] * e;
        O.x += o.x * e;
        O.y += o.y * e;
        O.z += o.z * e;
        O.w += o.w * e;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const float lse = L == 0.f ? kNegInf : int4_lse(M, L);
      O = make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
      if (p.final_mode) {
        int4_store_out<T>(p, r, h, q, d + 0, O.x, lse);
        int4_store_out<T>(p, r, h, q, d + 1, O.y, lse);
        int4_store_out<T>(p, r, h, q, d + 2, O.z, lse);
        int4_store_out<T>(p, r, h, q, d + 3, O.w, lse);
      } else {
        const int64_t base =
            static_cast<int64_t>(p.item_slots != nullptr ? p.item_slots[index] : index) * p.group +
            q;
        *reinterpret_cast<float4*>(p.part_o + base * kHeadDim + d) = O;
        if (d == 0) p.part_lse[base] = lse;
      }
    }
    if (!more) break;
    index = next_index;
    // Stored ahead of the two barriers above.
    next_index = first ? 2 * grid + static_cast<int>(blockIdx.x) : s_next[parity];
    first = false;
  }
}

// Joins the work items of each (request, query head): R warps per row fold
// partials w, w + R, ... with four dims per lane and up to eight loads in
// flight, then a row's warps are combined.  R = 8 (a block per row) where some
// row has many partials for the number of rows, else 1 (eight rows per block).
template <typename T, int R>
__global__ void __launch_bounds__(256)
    pg_int4_merge_kernel(const __grid_constant__ Int4DecodeParams p) {
  constexpr int W = 8, U = 8;
  __shared__ float s_m[W], s_l[W];
  __shared__ float4 s_o[W][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hq = p.hkv * p.group;
  const int row = blockIdx.x * (W / R) + warp / R;
  const bool live = row < p.batch * hq;
  const int r = live ? row / hq : 0, qh = live ? row % hq : 0;
  const int h = qh / p.group, q = qh % p.group;
  const int begin = p.item_off[r * p.hkv + h];
  const int end = live ? p.item_off[r * p.hkv + h + 1] : begin;
  pdl_launch_dependents();
  pdl_wait_primary();
  float m = kNegInf, den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = begin + warp % R; i0 < end; i0 += R * U) {
    float l[U];
    float4 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + R * k;
      l[k] = kNegInf;
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < end) {
        const int64_t b = static_cast<int64_t>(i) * p.group + q;
        l[k] = __ldcg(p.part_lse + b);
        v[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + b * kHeadDim) + lane);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (l[k] == kNegInf) continue;
      const float mn = fmaxf(m, l[k]);
      const float a = fast_exp2(m - mn), e = fast_exp2(l[k] - mn);
      acc.x = acc.x * a + e * v[k].x;
      acc.y = acc.y * a + e * v[k].y;
      acc.z = acc.z * a + e * v[k].z;
      acc.w = acc.w * a + e * v[k].w;
      den = den * a + e;
      m = mn;
    }
  }
  if constexpr (R > 1) {
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = den;
    }
    s_o[warp][lane] = acc;
    __syncthreads();
    if (warp % R != 0) return;
    float M = kNegInf;
#pragma unroll
    for (int w = 0; w < R; ++w) M = fmaxf(M, s_m[warp + w]);
    den = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < R; ++w) {
      if (s_l[warp + w] == 0.f) continue;
      const float e = fast_exp2(s_m[warp + w] - M);
      const float4 o = s_o[warp + w][lane];
      den += s_l[warp + w] * e;
      acc.x += o.x * e;
      acc.y += o.y * e;
      acc.z += o.z * e;
      acc.w += o.w * e;
    }
    m = M;
  }
  if (!live) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const float lse = den == 0.f ? kNegInf : m + fast_log2(den);
  int4_store_out<T>(p, r, h, q, 4 * lane + 0, acc.x * inv, lse);
  int4_store_out<T>(p, r, h, q, 4 * lane + 1, acc.y * inv, lse);
  int4_store_out<T>(p, r, h, q, 4 * lane + 2, acc.z * inv, lse);
  int4_store_out<T>(p, r, h, q, 4 * lane + 3, acc.w * inv, lse);
}

}  // namespace pg
