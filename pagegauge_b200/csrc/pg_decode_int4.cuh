// Decode attention over the 4-bit paged cache (record layout: pg_int4.cuh):
// one query token per request, GQA group of up to 8 query heads per KV head,
// split over the planner's work items (request, KV head, run of pages).
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
  const int32_t* item_off;
  int32_t num_items, batch, hkv, group;
  float sm_scale_log2;
  float* part_o;    // [num_items, group, 128]
  float* part_lse;  // [num_items, group]
  int32_t final_mode;
  void* out;
  int64_t out_stride_b, out_stride_h;
  float* lse_out;
  const void* value_center;  // [B, Hkv, 128] or null
  int64_t vc_stride_b;
  int* error_flag;
};

constexpr int kInt4Warps = 4;

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

// One CTA per work item; warps take every fourth page, lane l holds dims
// 4l .. 4l+3 of every row.
template <typename T>
__global__ void __launch_bounds__(kInt4Warps * 32)
    pg_decode_int4_kernel(const __grid_constant__ Int4DecodeParams p) {
  __shared__ float sm_m[kInt4Warps][8], sm_l[kInt4Warps][8], sm_o[kInt4Warps][8][kHeadDim];
  pdl_launch_dependents();
  const DecodeItem item = p.items[blockIdx.x];
  const int r = item.request, h = item.head_seg & 0xffff;
  const int n_pages = item.count & 0x7fffffff;
  pdl_wait_primary();
  int last = kPage;
  if (item.count < 0) {
    const int lv = p.last_len[r];
    last = lv < 1 ? 1 : (lv > kPage ? kPage : lv);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float q[8][4], o[8][4], m[8], l[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    m[g] = kNegInf;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[g][i] = 0.f;
      q[g][i] = g < p.group ? to_float<T>(static_cast<const T*>(
                                  p.q)[r * p.q_stride_b + (h * p.group + g) * p.q_stride_h +
                                       4 * lane + i]) * p.sm_scale_log2
                            : 0.f;
    }
  }
  for (int u = warp; u < n_pages; u += kInt4Warps) {
    int id = p.indices[item.idx_begin + u];
    if (id < 0 || id >= p.num_pages) {
      record_error(p.error_flag, kDevBadPageId);
      continue;
    }
    const uint8_t* rec = p.records + (static_cast<int64_t>(id) * p.hkv + h) * kInt4Record;
    const int valid = u == n_pages - 1 ? last : kPage;
    for (int t = 0; t < valid; ++t) {
      const int grp = lane >> 3;
      const uint32_t kw = *reinterpret_cast<const uint16_t*>(
          rec + t * 64 + ((lane >> 1) & 3) * 16 + grp * 4 + (lane & 1) * 2);
      const uint32_t vw = *reinterpret_cast<const uint16_t*>(
          rec + kInt4Value + value_code_row(t) * 64 + (lane & 7) * 8 + grp * 2);
      const __half* km = reinterpret_cast<const __half*>(rec + kInt4KeyMeta + t * 16);
      const __half* vm = reinterpret_cast<const __half*>(rec + kInt4ValueMeta + t * 16);
      const float ks = __half2float(km[grp]), kmid = __half2float(km[4 + grp]);
      const float vs = __half2float(vm[grp]), vmid = __half2float(vm[4 + grp]);
      float k[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k[i] = fmaf(static_cast<float>(static_cast<int>((kw >> (4 * i)) & 15u) - 8), ks, kmid);
        v[i] = fmaf(static_cast<float>(static_cast<int>((vw >> (4 * i)) & 15u) - 8), vs, vmid);
      }
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        if (g >= p.group) break;
        float s = q[g][0] * k[0] + q[g][1] * k[1] + q[g][2] * k[2] + q[g][3] * k[3];
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float mn = fmaxf(m[g], s);
        const float a = fast_exp2(m[g] - mn), e = fast_exp2(s - mn);
        m[g] = mn;
        l[g] = l[g] * a + e;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[g][i] = o[g][i] * a + e * v[i];
      }
    }
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    if (g >= p.group) break;
    if (lane == 0) {
      sm_m[warp][g] = m[g];
      sm_l[warp][g] = l[g];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sm_o[warp][g][4 * lane + i] = o[g][i];
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < p.group * kHeadDim; idx += blockDim.x) {
    const int g = idx >> 7, d = idx & 127;
    float M = kNegInf, L = 0.f, O = 0.f;
    for (int w = 0; w < kInt4Warps; ++w) M = fmaxf(M, sm_m[w][g]);
    for (int w = 0; w < kInt4Warps; ++w) {
      const float e = sm_l[w][g] == 0.f ? 0.f : fast_exp2(sm_m[w][g] - M);
      L += sm_l[w][g] * e;
      O += sm_o[w][g][d] * e;
    }
    const float v = L == 0.f ? 0.f : O / L, lse = L == 0.f ? kNegInf : M + fast_log2(L);
    if (p.final_mode) {
      int4_store_out<T>(p, r, h, g, d, v, lse);
    } else {
      const int64_t base = static_cast<int64_t>(blockIdx.x) * p.group + g;
      p.part_o[base * kHeadDim + d] = v;
      if (d == 0) p.part_lse[base] = lse;
    }
  }
}

// Joins the work items of each (request, query head): one CTA of 128 threads
// per row, thread = dim.
template <typename T>
__global__ void __launch_bounds__(kHeadDim)
    pg_int4_merge_kernel(const __grid_constant__ Int4DecodeParams p) {
  const int hq = p.hkv * p.group;
  const int r = blockIdx.x / hq, qh = blockIdx.x % hq;
  const int h = qh / p.group, q = qh % p.group, d = threadIdx.x;
  const int begin = p.item_off[r * p.hkv + h], end = p.item_off[r * p.hkv + h + 1];
  pdl_launch_dependents();
  pdl_wait_primary();
  float M = kNegInf, L = 0.f, O = 0.f;
  for (int i = begin; i < end; ++i) {
    const int64_t b = static_cast<int64_t>(i) * p.group + q;
    const float lse = __ldcg(p.part_lse + b);
    if (lse == kNegInf) continue;
    const float mn = fmaxf(M, lse);
    const float a = fast_exp2(M - mn), e = fast_exp2(lse - mn);
    M = mn;
    L = L * a + e;
    O = O * a + e * __ldcg(p.part_o + b * kHeadDim + d);
  }
  int4_store_out<T>(p, r, h, q, d, L == 0.f ? 0.f : O / L, L == 0.f ? kNegInf : M + fast_log2(L));
}

}  // namespace pg
