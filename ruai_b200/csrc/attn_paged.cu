// Causal attention of every request's new tokens over its pages: softmax(scale q k^T + mask) v, where the token at position p sees
// keys p - window + 1 .. p (window 0: all of 0 .. p).
//
// One warp per (token, query head), a key at a time: the running maximum m, sum l and weighted values o of a softmax in f32,
// o <- o e^(m - m') + e^(s - m') v.
#include "paged.cuh"

namespace {

constexpr int kHeadParts = 8;  // elements of a head per lane: heads of up to 256

template <typename T>
__global__ void __launch_bounds__(256) one_row_kernel(const PagedAttn a) {
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t lane = threadIdx.x & 31u, row = blockIdx.x * 8 + (threadIdx.x >> 5), hd = a.pool.hd;
  if (row >= a.tokens * a.H) return;
  const uint32_t t = row / a.H, head = row % a.H, g = head / (a.H / a.pool.KV);
  uint32_t lo = 0, hi = a.R;  // the last request that starts at or before t
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (a.starts[mid] <= (int32_t)t) lo = mid;
    else hi = mid;
  }
  PagedRequest rq;
  if (!paged_request(a, lo, rq) || t < rq.t0 || t - rq.t0 >= rq.fresh) return;
  const uint32_t pos = rq.cached + t - rq.t0;
  float q[kHeadParts], o[kHeadParts], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int j = 0; j < kHeadParts; ++j) {
    const uint32_t e = lane + 32u * j;
    q[j] = e < hd ? to_f32<T>(static_cast<const T*>(a.q)[(size_t)t * a.q_ld + head * hd + e]) : 0.0f;
    o[j] = 0.0f;
  }
  for (uint32_t k = paged_low(pos, a.window); k <= pos; ++k) {
    const int32_t pg = paged_page(a, lo, k);
    if (pg < 0) continue;
    const size_t at = ((((size_t)pg * a.pool.KV + g) << a.pool.page_log2) + (k & ((1u << a.pool.page_log2) - 1u))) * hd;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kHeadParts; ++j) {
      const uint32_t e = lane + 32u * j;
      if (e < hd) s = fmaf(q[j], to_f32<T>(static_cast<const T*>(a.pool.k)[at + e]), s);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, off);
    s *= a.scale;
    if (s == -INFINITY) continue;
    const float m_new = fmaxf(m, s), corr = m == -INFINITY ? 0.0f : expf(m - m_new), pr = expf(s - m_new);
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
    if (e < hd) static_cast<T*>(a.out)[(size_t)t * a.out_ld + head * hd + e] = from_f32<T>(l == 0.0f ? 0.0f : o[j] / l);
  }
}

}  // namespace

int ruai_paged_attention_launch(ruai_ctx* c, const PagedAttn& a) {
  const dim3 grid((a.tokens * a.H + 7) / 8), block(256);
  RUAI_CUDA(c, a.pool.dtype == RUAI_F32   ? ruai_launch(c, one_row_kernel<float>, grid, block, 0, true, a)
               : a.pool.dtype == RUAI_F16 ? ruai_launch(c, one_row_kernel<__half>, grid, block, 0, true, a)
                                          : ruai_launch(c, one_row_kernel<__nv_bfloat16>, grid, block, 0, true, a));
  return RUAI_OK;
}
