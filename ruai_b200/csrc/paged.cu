// The cache in pages: block tables and slots from request lengths, and the writing of keys and values at those slots.
//
// plan_kernel.  Request r has cached[r] tokens in the cache and brings fresh[r] new ones, or has ended (-1).  Three exclusive
// sums over the requests (new tokens, pages they need beyond those they hold, pages given back) say where everything lies: token t
// belongs to the request whose range of the first sum holds it, the k-th page that is needed is the ring's (first + k)-th, and the
// j-th that is given back goes behind the free ones.  Latency bounds it (two dependent loads, a scan, a search in shared memory), not
// bytes: every CTA works the sums out for itself, so that nothing is exchanged, and they share the tokens and pages, a token per thread.
// 64 requests of one token: 5.7 us a call, of 2000 requests with 33000 tokens 6.9.  Where the pool's words are written in place all CTAs must have read them before: they are one cluster then, of eight, and meet.
//
// append_kernel.  A CTA per token; a thread takes eight elements of a head, the two fours that rotate into each other where there is a
// rotation: y_i = x_i cos - x_(i+h) sin, y_(i+h) = x_(i+h) cos + x_i sin, in f32, rounded once to the cache's type.  Bound by HBM: every
// element is read and written once (8000 tokens of 48 heads of 128 in bf16, 299 MB: 47 us, 6.4 TB/s).
#include <algorithm>

#include "attn_paged.cuh"
#include "pipeline.cuh"

namespace {

struct PlanArgs {
  const int32_t *cached, *fresh;
  int32_t *table, *ring;
  const int32_t* words_in;
  int32_t *words_out, *starts, *positions, *slots;
  uint32_t R, tokens, page_log2, table_ld, pages, in_place;
  int* status;
};

// The last i in [0, n) with sums[i] <= v, for sums[0] = 0: whose range holds v (ranges may be empty).
__device__ __forceinline__ uint32_t owner_of(const uint32_t* sums, uint32_t n, uint32_t v) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (sums[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

constexpr uint32_t kPlanCluster = 8;

__global__ void __launch_bounds__(1024) plan_kernel(const PlanArgs a) {
  extern __shared__ uint32_t sums[];  // three exclusive sums over the requests, R + 1 each, and their lengths
  __shared__ uint32_t part[3][32];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ld = a.R + 1, page = 1u << a.page_log2;
  uint32_t *s_n = sums, *s_need = sums + ld, *s_back = sums + 2 * ld, *s_cached = sums + 3 * ld;
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t first = (uint32_t)a.words_in[0], free = (uint32_t)a.words_in[1];
  const uint32_t per = (a.R + blockDim.x - 1) / blockDim.x, r0 = min(tid * per, a.R), r1 = min(r0 + per, a.R);
  uint32_t sum[3] = {0, 0, 0};
  bool bad = false;
#pragma unroll 4
  for (uint32_t r = r0; r < r1; ++r) {
    const int32_t past = a.cached[r], f = a.fresh[r];
    uint32_t n = 0, need = 0, back = 0;
    const uint32_t held = past < 0 ? 0u : ((uint32_t)past + page - 1) >> a.page_log2;
    if (past < 0 || held > a.table_ld || (f > 0 && (uint32_t)f > a.tokens)) bad = true;
    else if (f < 0) back = held;
    else {
      n = (uint32_t)f;
      const uint32_t all = ((uint32_t)past + n + page - 1) >> a.page_log2;
      if (all > a.table_ld) bad = true;
      else need = all - held;
    }
    s_n[r] = n; s_need[r] = need; s_back[r] = back; s_cached[r] = (uint32_t)past;
    sum[0] += n; sum[1] += need; sum[2] += back;
  }
  uint32_t inc[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    inc[i] = sum[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc[i], o);
      if (lane >= (uint32_t)o) inc[i] += v;
    }
    if (lane == 31) part[i][warp] = inc[i];
  }
  bad = __syncthreads_or(bad);
  uint32_t at[3], total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint32_t v = lane < blockDim.x / 32 ? part[i][lane] : 0u, before = lane < warp ? v : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
      before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    }
    total[i] = v;
    at[i] = before + inc[i] - sum[i];
  }
  for (uint32_t r = r0; r < r1; ++r) {
    const uint32_t n = s_n[r], need = s_need[r], back = s_back[r];
    s_n[r] = at[0]; s_need[r] = at[1]; s_back[r] = at[2];
    at[0] += n; at[1] += need; at[2] += back;
  }
  if (tid == 0) { s_n[a.R] = total[0]; s_need[a.R] = total[1]; s_back[a.R] = total[2]; }
  const uint32_t missing = total[1] > free ? total[1] - free : 0u;
  bad = bad || first >= a.pages || free > a.pages || total[0] > a.tokens || (free <= a.pages && total[2] > a.pages - free);  // pages go back behind all that are free, given out in this step or not
  const bool ok = !bad && !missing;
  __syncthreads();
  const uint32_t step = gridDim.x * blockDim.x, me = blockIdx.x * blockDim.x + tid;
  auto ring_at = [&](uint32_t i) { return (uint32_t)(((unsigned long long)first + i) % a.pages); };
  for (uint32_t r = me; r <= a.R; r += step) a.starts[r] = ok ? (int32_t)s_n[r] : 0;
  for (uint32_t t = me; t < a.tokens; t += step) {
    int32_t pos = -1, slot = -1;
    if (ok && t < total[0]) {
      const uint32_t r = owner_of(s_n, a.R, t), past = s_cached[r], held = (past + page - 1) >> a.page_log2;
      const uint32_t p = past + t - s_n[r], i = p >> a.page_log2;
      const int32_t pg = i < held ? a.table[(size_t)r * a.table_ld + i] : a.ring[ring_at(s_need[r] + i - held)];
      pos = (int32_t)p;
      if ((uint32_t)pg < a.pages) slot = (int32_t)(((uint32_t)pg << a.page_log2) + (p & (page - 1)));
      else atomicCAS(a.status, 0, kStatusPaged);
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  if (ok) {
    for (uint32_t k = me; k < total[1]; k += step) {
      const uint32_t r = owner_of(s_need, a.R, k), held = (s_cached[r] + page - 1) >> a.page_log2;
      a.table[(size_t)r * a.table_ld + held + k - s_need[r]] = a.ring[ring_at(k)];
    }
    for (uint32_t k = me; k < total[2]; k += step) {
      const uint32_t r = owner_of(s_back, a.R, k);
      a.ring[ring_at(free + k)] = a.table[(size_t)r * a.table_ld + k - s_back[r]];
    }
  }
  if (a.in_place && gridDim.x > 1) pipe::cluster_sync_all();  // every CTA has read the words
  else __syncthreads();
  if (me == 0) {
    a.words_out[0] = (int32_t)(ok ? ring_at(total[1]) : first);
    a.words_out[1] = (int32_t)(ok ? free - total[1] + total[2] : free);
    a.words_out[2] = (int32_t)(bad ? 0u : missing);
    if (!ok) atomicCAS(a.status, 0, kStatusPlan);
  }
}

template <typename T> struct Four;
template <> struct Four<float> { using V = float4; };
template <> struct Four<__half> { using V = uint2; };
template <> struct Four<__nv_bfloat16> { using V = uint2; };

template <typename T> __device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  typename Four<T>::V raw = *reinterpret_cast<const typename Four<T>::V*>(p);
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(e[i]);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  typename Four<T>::V raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<typename Four<T>::V*>(p) = raw;
}

constexpr int kAppendThreads = 256;

template <typename X, typename T>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const PagedAppend a) {
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t t = blockIdx.x, hd = a.pool.hd, KV = a.pool.KV, half = a.rot / 2, per = hd / 8;
  const int32_t slot = a.slots[t], pos = a.rope ? a.positions[t] : 0;
  if (slot < 0) return;  // a row behind the last token
  const uint32_t pg = (uint32_t)slot >> a.pool.page_log2, off = (uint32_t)slot & ((1u << a.pool.page_log2) - 1u);
  if (pg >= a.pool.pages || (a.rope && (uint32_t)pos >= a.max_pos)) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, kStatusPaged);
    return;
  }
  const X* row = static_cast<const X*>(a.x) + (size_t)t * a.ld;
  T* q = static_cast<T*>(a.q_out);
  for (uint32_t u = threadIdx.x + (q ? 0u : a.H * per); u < (a.H + 2 * KV) * per; u += kAppendThreads) {
    const uint32_t head = u / per, i = u % per;
    const bool value = head >= a.H + KV, query = head < a.H;
    const bool turned = !value && a.rope && 4 * i < half;
    const uint32_t e0 = turned ? 4 * i : 8 * i, e1 = turned ? e0 + half : e0 + 4;
    const uint32_t kv = value ? head - a.H - KV : head - a.H;
    const X* src = row + (query ? head * hd : (value ? a.v_off : a.k_off) + kv * hd);
    float x0[4], x1[4];
    load4<X>(src + e0, x0);
    load4<X>(src + e1, x1);
    if (turned) {
      const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * half + e0);  // (cos, sin) of two pairs
      const float4 c01 = cs[0], c23 = cs[1];
      const float co[4] = {c01.x, c01.z, c23.x, c23.z}, si[4] = {c01.y, c01.w, c23.y, c23.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y0 = x0[j] * co[j] - x1[j] * si[j], y1 = x1[j] * co[j] + x0[j] * si[j];
        x0[j] = y0;
        x1[j] = y1;
      }
    }
    T* dst = query ? q + (size_t)t * a.q_ld + head * hd : static_cast<T*>(value ? a.pool.v : a.pool.k) + ((((size_t)pg * KV + kv) << a.pool.page_log2) + off) * hd;
    store4<T>(dst + e0, x0);
    store4<T>(dst + e1, x1);
  }
}

template <typename X>
cudaError_t launch_append(ruai_ctx* c, const PagedAppend& a) {
  const dim3 grid(a.tokens), block(kAppendThreads);
  if (a.pool.dtype == RUAI_F32) return ruai_launch(c, append_kernel<X, float>, grid, block, 0, true, a);
  if (a.pool.dtype == RUAI_F16) return ruai_launch(c, append_kernel<X, __half>, grid, block, 0, true, a);
  return ruai_launch(c, append_kernel<X, __nv_bfloat16>, grid, block, 0, true, a);
}

bool known(int dtype) { return dtype == RUAI_F32 || dtype == RUAI_F16 || dtype == RUAI_BF16; }
uint32_t bytes_of(int dtype) { return dtype == RUAI_F32 ? 4u : 2u; }
bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
bool page_log2(uint32_t page, uint32_t* out) {
  if (page < 16 || page > 256 || (page & (page - 1))) return false;
  *out = (uint32_t)__builtin_ctz(page);
  return true;
}

}  // namespace

int ruai_paged_check_pool(ruai_ctx* c, const PagedPool& p, const char* who) {
  if (!known(p.dtype)) return ruai_fail(c, RUAI_ERR_ARG, "%s: unknown type %d of the pages", who, p.dtype);
  if (!p.pages || !p.KV) return ruai_fail(c, RUAI_ERR_SHAPE, "%s: a pool of %u pages of %u key heads", who, p.pages, p.KV);
  if (!p.hd || p.hd % 8 || p.hd > 256) return ruai_fail(c, RUAI_ERR_SHAPE, "%s: heads of %u: a multiple of 8 up to 256", who, p.hd);
  if (((unsigned long long)p.pages * p.KV << p.page_log2) >= (1ull << 31))
    return ruai_fail(c, RUAI_ERR_SHAPE, "%s: %u pages of %u x %u rows are 2^31 rows or more", who, p.pages, p.KV, 1u << p.page_log2);
  if (!aligned(p.k, 16) || !aligned(p.v, 16)) return ruai_fail(c, RUAI_ERR_ARG, "%s: pages must start on 16-byte boundaries", who);
  return RUAI_OK;
}

ruai_tensor_map_encode ruai_tensor_map_fn() {
  static const ruai_tensor_map_encode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult st;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &st) != cudaSuccess || st != cudaDriverEntryPointSuccess) p = nullptr;
    return (ruai_tensor_map_encode)p;
  }();
  return fn;
}

int ruai_paged_append_launch(ruai_ctx* c, const PagedAppend& a) {
  if (!a.tokens) return RUAI_OK;
  RUAI_CUDA(c, a.x_dtype == RUAI_F32 ? launch_append<float>(c, a) : a.x_dtype == RUAI_F16 ? launch_append<__half>(c, a) : launch_append<__nv_bfloat16>(c, a));
  return RUAI_OK;
}

RUAI_API int ruai_page_plan(ruai_ctx* c, const int32_t* cached, const int32_t* fresh, uint32_t R, uint32_t tokens, uint32_t page, int32_t* table,
                            uint32_t table_ld, int32_t* ring, uint32_t pages, const int32_t* words_in, int32_t* words_out, int32_t* starts,
                            int32_t* positions, int32_t* slots) {
  if (!c || !cached || !fresh || !table || !ring || !words_in || !words_out || !starts || (tokens && (!positions || !slots)))
    return ruai_fail(c, RUAI_ERR_ARG, "ruai_page_plan: NULL argument");
  PlanArgs a = {cached, fresh, table, ring, words_in, words_out, starts, positions, slots, R, tokens, 0, table_ld, pages, words_in == words_out ? 1u : 0u, c->status};
  if (!page_log2(page, &a.page_log2)) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_page_plan: pages of %u: a power of two from 16 to 256", page);
  if (words_in != words_out && (const char*)words_in < (const char*)(words_out + 3) && (const char*)words_out < (const char*)(words_in + 3))
    return ruai_fail(c, RUAI_ERR_ARG, "ruai_page_plan: words_out is words_in or lies apart from it");
  if (!R || R > kPlanRowsMax || tokens > kPlanTokensMax)
    return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_page_plan: %u requests and %u tokens: 1 to %u and up to %u", R, tokens, kPlanRowsMax, kPlanTokensMax);
  if (!table_ld || table_ld > (1u << 18)) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_page_plan: rows of %u pages: 1 to %u", table_ld, 1u << 18);
  if (!pages || ((unsigned long long)pages << a.page_log2) >= (1ull << 31)) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_page_plan: a pool of %u pages of %u", pages, page);
  DeviceGuard g(c->ordinal);
  const uint32_t most = R > tokens ? R : tokens;
  const dim3 block(most <= 256 ? 256 : 1024), grid(most <= 1024 ? 1 : a.in_place ? kPlanCluster : std::min((most + 1023) / 1024, (uint32_t)c->sm_count));
  const size_t smem = 4 * (size_t)(R + 1) * sizeof(uint32_t);
  if (smem > 48 * 1024) {
    static bool done[64] = {};
    if (!done[c->ordinal & 63]) {
      RUAI_CUDA(c, cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(4 * (kPlanRowsMax + 1) * sizeof(uint32_t))));
      done[c->ordinal & 63] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = c->stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (c->use_pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.in_place && grid.x > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = kPlanCluster; attr[n].val.clusterDim.y = 1; attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr; cfg.numAttrs = n;
  c->launches++;
  RUAI_CUDA(c, cudaLaunchKernelEx(&cfg, plan_kernel, a));
  return RUAI_OK;
}

RUAI_API int ruai_paged_append(ruai_ctx* c, int x_dtype, const void* x, uint32_t ld, uint32_t k_off, uint32_t v_off, uint32_t tokens, uint32_t H,
                               uint32_t rot, const float* rope, uint32_t max_pos, const int32_t* positions, const int32_t* slots, int dtype,
                               void* k_pages, void* v_pages, uint32_t pages, uint32_t KV, uint32_t page, uint32_t hd, void* q_out, uint32_t q_ld) {
  if (!c || !x || !slots || !k_pages || !v_pages || (rope && !positions)) return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_append: NULL argument");
  PagedAppend a = {{k_pages, v_pages, pages, 0, KV, hd, dtype}, x, x_dtype, ld, k_off, v_off, tokens, H, rope ? rot : 0u, max_pos,
                   reinterpret_cast<const float2*>(rope), positions, slots, q_out, q_ld, c->status};
  if (!page_log2(page, &a.pool.page_log2)) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_append: pages of %u: a power of two from 16 to 256", page);
  RUAI_TRY(ruai_paged_check_pool(c, a.pool, "ruai_paged_append"));
  if (!known(x_dtype)) return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_append: unknown type %d of x", x_dtype);
  if (rope && (!rot || rot % 8 || rot > hd || !max_pos))
    return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_append: rotation of %u of %u over %u positions: a multiple of 8", rot, hd, max_pos);
  if (tokens && q_out == x && (x_dtype != dtype || q_ld != ld)) return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_append: queries may take the place of x's only in its own type and rows");
  if (ld % 4 || k_off % 4 || v_off % 4 || (q_out && q_ld % 4) || !aligned(x, 4 * bytes_of(x_dtype)) || (q_out && !aligned(q_out, 4 * bytes_of(dtype))) || !aligned(rope, 16))
    return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_append: rows and heads must start on boundaries of four elements, the rotations on one of 16 bytes");
  const unsigned long long wide = (unsigned long long)H * hd, kv = (unsigned long long)KV * hd;
  if (wide >= (1ull << 31) || kv >= (1ull << 30)) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_append: %u and twice %u heads of %u", H, KV, hd);
  if (ld < k_off + kv || ld < v_off + kv || (q_out && (ld < wide || q_ld < wide)))
    return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_append: rows of %u (queries %u) do not hold %u and twice %u heads of %u", ld, q_ld, H, KV, hd);
  if (tokens > 0x7FFFFFFFu) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_append: %u tokens", tokens);
  DeviceGuard g(c->ordinal);
  return ruai_paged_append_launch(c, a);
}

RUAI_API int ruai_paged_attention(ruai_ctx* c, int dtype, const void* q, uint32_t q_ld, const void* k_pages, const void* v_pages, uint32_t pages,
                                  uint32_t KV, uint32_t page, uint32_t hd, const int32_t* table, uint32_t table_ld, const int32_t* cached,
                                  const int32_t* starts, uint32_t R, uint32_t tokens, uint32_t H, float scale, uint32_t window, uint32_t most_fresh,
                                  uint32_t most_len, void* out, uint32_t out_ld) {
  if (!c || !k_pages || !v_pages || !table || !cached || !starts || (tokens && (!q || !out))) return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_attention: NULL argument");
  PagedAttn a = {{const_cast<void*>(k_pages), const_cast<void*>(v_pages), pages, 0, KV, hd, dtype}, q, out, q_ld, out_ld, table, cached, starts,
                 table_ld, R, tokens, H, scale, window, most_fresh, most_len, c->status};
  if (!page_log2(page, &a.pool.page_log2)) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_attention: pages of %u: a power of two from 16 to 256", page);
  RUAI_TRY(ruai_paged_check_pool(c, a.pool, "ruai_paged_attention"));
  if (!H || H % KV || H / KV > 256 || (unsigned long long)H * kPlanTokensMax >= (1ull << 31)) return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_attention: heads %u must be a multiple of kv_heads %u, 256 times them and 8191 at most", H, KV);
  const uint32_t four = 16 / bytes_of(dtype);
  if (q_ld % four || out_ld % four || !aligned(q, 16) || !aligned(out, 16))
    return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_attention: rows of q and out must start on 16-byte boundaries");
  if (R && tokens && most_fresh && q == out) return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_attention: out must lie apart from q");
  if ((unsigned long long)H * hd > q_ld || (unsigned long long)H * hd > out_ld)
    return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_attention: rows of %u and %u do not hold %u heads of %u", q_ld, out_ld, H, hd);
  if (!table_ld || R > kPlanRowsMax || tokens > kPlanTokensMax)
    return ruai_fail(c, RUAI_ERR_SHAPE, "ruai_paged_attention: %u requests of up to %u pages, %u tokens: up to %u and %u", R, table_ld, tokens, kPlanRowsMax, kPlanTokensMax);
  if (most_len >= (1u << 30) || !(scale == scale)) return ruai_fail(c, RUAI_ERR_ARG, "ruai_paged_attention: lengths of up to %u, scale %f", most_len, (double)scale);
  if (!R || !tokens || !most_fresh) return RUAI_OK;
  if (a.most_fresh > tokens) a.most_fresh = tokens;  // no request has more
  DeviceGuard g(c->ordinal);
  return ruai_paged_attention_launch(c, a);
}
