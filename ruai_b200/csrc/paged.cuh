// A cache in pages: requests of different lengths hold pages of one pool, listed in a block table.
#pragma once
#include "common.cuh"

// Keys and values lie in [pages][KV][page][hd]; the pages of request r, in order, in table[r * table_ld ..].
struct PagedPool {
  void *k, *v;
  uint32_t pages, page_log2, KV, hd;
  int dtype;
};

struct PagedAttn {
  PagedPool pool;
  const void* q;  // [tokens, q_ld], the query heads side by side, in the pool's type
  void* out;      // [tokens, out_ld]
  uint32_t q_ld, out_ld;
  const int32_t *table, *cached, *starts;
  uint32_t table_ld, R, tokens, H;
  float scale;
  uint32_t window, most_fresh, most_len;  // bounds that hold for every request
  int* status;
};

struct PagedAppend {
  PagedPool pool;
  const void* x;  // [tokens, ld] of x_dtype: query heads, key heads at k_off, value heads at v_off
  int x_dtype;
  uint32_t ld, k_off, v_off, tokens, H, rot, max_pos;
  const float2* rope;  // [max_pos][rot / 2] (cos, sin), or NULL: no rotation
  const int32_t *positions, *slots;
  void* q_out;  // [tokens, q_ld] in the pool's type, or NULL
  uint32_t q_ld;
  int* status;
};

// What the status word says: kept apart from the codes of waits (common.cuh).
constexpr int kStatusPlan = 6;   // lengths that do not fit the table or the buffers, or too few free pages: nothing was planned
constexpr int kStatusPaged = 7;  // a page, slot, position or length out of range: what it belongs to was left out

constexpr uint32_t kPlanRowsMax = 8192, kPlanTokensMax = 1u << 18;

// Checked arguments (the C ABI's checks are these).
int ruai_paged_check_pool(ruai_ctx* c, const PagedPool& p, const char* who);
int ruai_paged_append_launch(ruai_ctx* c, const PagedAppend& a);
int ruai_paged_attention_launch(ruai_ctx* c, const PagedAttn& a);

#ifdef __CUDACC__
// Request r as a kernel may use it: its new tokens and lengths, false (and the status) where they are out of range.
struct PagedRequest { uint32_t t0, fresh, cached, len; };
__device__ __forceinline__ bool paged_request(const PagedAttn& a, uint32_t r, PagedRequest& q) {
  const int32_t s0 = a.starts[r], s1 = a.starts[r + 1], past = a.cached[r];
  q.t0 = (uint32_t)s0; q.fresh = 0; q.cached = 0; q.len = 0;
  if (s0 == s1) return true;  // no new tokens: its lengths are nothing to this call
  const unsigned long long len = (unsigned long long)(uint32_t)past + (uint32_t)(s1 - s0);
  if (s0 < 0 || s1 < s0 || (uint32_t)s1 > a.tokens || past < 0 || (uint32_t)(s1 - s0) > a.most_fresh || len > a.most_len ||
      len > ((unsigned long long)a.table_ld << a.pool.page_log2)) {
    if (a.status) atomicCAS(a.status, 0, kStatusPaged);
    return false;
  }
  q.fresh = (uint32_t)(s1 - s0);
  q.cached = (uint32_t)past;
  q.len = (uint32_t)len;
  return true;
}
// The first key that a token at `pos` sees.
__device__ __forceinline__ uint32_t paged_low(uint32_t pos, uint32_t window) { return window && pos >= window ? pos + 1 - window : 0; }
// The page that holds key j of request r, or a negative number (and the status).
__device__ __forceinline__ int32_t paged_page(const PagedAttn& a, uint32_t r, uint32_t j) {
  const int32_t pg = a.table[(size_t)r * a.table_ld + (j >> a.pool.page_log2)];
  if ((uint32_t)pg < a.pool.pages) return pg;
  if (a.status) atomicCAS(a.status, 0, kStatusPaged);
  return -1;
}
#endif
