// What the kernels of attention over pages share.
#pragma once
#include <cuda.h>

#include "paged.cuh"

constexpr int kHeadParts = 8;  // elements of a head per lane: heads of up to 256
constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights reach the values in the values' type.  In f16 what lies below 2^-14 loses bits and below 2^-25 everything, so f16 weights are
// 2^(s - m) for an m that lies under the row's maximum: by 15, so that the largest is 2^15, or (attn_paged_tc.cu) by 7, where a maximum
// may still grow by 2^8.  Sums and joins go by that m, whatever it is.  A key with nearly all weight and no value, 24 powers of two above 600
// others: 7 % off without, 0.3 % with 7 (at 20 powers 0.4 and 0.06 %), 0.05 % with 15, which is the outputs' rounding.
template <typename T> constexpr float weights_up(float by) { return 0.0f; }
template <> constexpr float weights_up<__half>(float by) { return by; }

// What a CTA does with one item: keys of tiles [tile0, tile1) for rows [row0, row0 + rows) of (request r, key head g).
struct Segment {
  PagedRequest rq;
  uint32_t r, g, row0, rows, tile0, tile1;
};

// One row over keys [k0, k1) by a warp, a key at a time; m and scores in powers of two, o not divided by l.
template <typename T>
__device__ void row_again(const PagedAttn& a, const Segment& s, uint32_t rep, uint32_t row, uint32_t k0, uint32_t k1, float* o_out, float& m_out, float& l_out) {
  const uint32_t lane = threadIdx.x & 31u, hd = a.pool.hd, i = row / rep, pos = s.rq.cached + i;
  const T* qs = static_cast<const T*>(a.q) + (size_t)(s.rq.t0 + i) * a.q_ld + (size_t)(s.g * rep + row % rep) * hd;
  float q[kHeadParts], o[kHeadParts], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int j = 0; j < kHeadParts; ++j) {
    const uint32_t e = lane + 32u * j;
    q[j] = e < hd ? to_f32<T>(qs[e]) : 0.0f;
    o[j] = 0.0f;
  }
  for (uint32_t k = max(k0, paged_low(pos, a.window)); k < min(k1, pos + 1); ++k) {
    const int32_t pg = paged_page(a, s.r, k);
    if (pg < 0) continue;
    const size_t at = ((((size_t)pg * a.pool.KV + s.g) << a.pool.page_log2) + (k & ((1u << a.pool.page_log2) - 1u))) * hd;
    float d = 0.0f;
#pragma unroll
    for (int j = 0; j < kHeadParts; ++j) {
      const uint32_t e = lane + 32u * j;
      if (e < hd) d = fmaf(q[j], to_f32<T>(static_cast<const T*>(a.pool.k)[at + e]), d);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, off);
    d *= a.scale * kLog2e;
    if (d == -INFINITY) continue;
    const float m_new = fmaxf(m, d), corr = m == -INFINITY ? 0.0f : exp2_of(m - m_new), pr = exp2_of(d - m_new);
    l = fmaf(l, corr, pr);
    m = m_new;
#pragma unroll
    for (int j = 0; j < kHeadParts; ++j) {
      const uint32_t e = lane + 32u * j;
      if (e < hd) o[j] = fmaf(pr, to_f32<T>(static_cast<const T*>(a.pool.v)[at + e]), o[j] * corr);
    }
  }
#pragma unroll
  for (int j = 0; j < kHeadParts; ++j) {
    const uint32_t e = lane + 32u * j;
    if (e < hd) o_out[e] = o[j];
  }
  m_out = m;
  l_out = l;
}

// attn_paged_tc.cu: the requests with more than `rows_over` rows (tokens x query heads of a key head) on the tensor cores, 256 rows at a
// time.  1: launched; 0: this shape is not taken; < 0: error.
int ruai_paged_attention_tc(ruai_ctx* c, const PagedAttn& a, uint32_t rows_over);
// The same in f32, with operands as two fp16 pieces (attn_prefill_tc.cu).
int ruai_paged_attention_pieces(ruai_ctx* c, const PagedAttn& a, uint32_t rows_over);

typedef CUresult (*ruai_tensor_map_encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                           const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// cuTensorMapEncodeTiled, or NULL where the driver has none.
ruai_tensor_map_encode ruai_tensor_map_fn();
