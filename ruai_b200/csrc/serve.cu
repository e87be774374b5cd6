// Serving: requests of different lengths that come and go, over one pool of pages per layer and one block table for all layers.
//
// A step takes the new tokens of any requests side by side (prompts, parts of prompts, single tokens): plan (paged.cu), embedding, then per
// layer the Linears over all tokens, rotation and append to the pages, attention over them (attn_paged.cu, attn_paged_tc.cu), and the
// head over the last token of every request.  The host keeps the lengths too, so that it refuses a step that does not fit before anything
// runs; the device's words are taken over from the plan only when the step has ended well.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "decode_ops.cuh"
#include "model.cuh"
#include "paged.cuh"

struct Serve {
  uint32_t pages = 0, page_log2 = 4, requests = 0, row_pages = 0, free = 0;
  int dtype = RUAI_F32;
  std::vector<DevBuf> k, v;           // per layer
  DevBuf table, ring, words[2];       // the words before and after a step
  DevBuf up, plan, q, att;            // what the host sends; starts, positions, slots; queries and attention's output in the pages' type
  uint32_t tokens = 0;                // that the buffers hold
  std::vector<uint32_t> len;
  std::vector<int32_t> sent;
};

namespace {

// The embedding of every token, plus that of its position where there is a table of positions.
__global__ void embed_at_kernel(const int32_t* __restrict__ ids, const int32_t* __restrict__ positions, const float* __restrict__ embed,
                                const float* __restrict__ wpe, uint32_t d, uint32_t vocab, uint32_t max_pos, float* __restrict__ x, int* __restrict__ err) {
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t r = blockIdx.x;
  int32_t id = ids[r];
  if (id < 0 || (uint32_t)id >= vocab) {
    if (threadIdx.x == 0) atomicExch(err, 1);
    id = 0;
  }
  const float* e = embed + (size_t)id * d;
  const uint32_t pos = min((uint32_t)max(positions[r], 0), max_pos - 1);  // -1 where the plan was refused
  const float* p = wpe ? wpe + (size_t)pos * d : nullptr;
  for (uint32_t i = threadIdx.x; i < d; i += blockDim.x) x[(size_t)r * d + i] = p ? e[i] + p[i] : e[i];
}

void release(Serve* s) {
  for (DevBuf& b : s->k) b.release();
  for (DevBuf& b : s->v) b.release();
  for (DevBuf* b : {&s->table, &s->ring, &s->words[0], &s->words[1], &s->up, &s->plan, &s->q, &s->att}) b->release();
}

uint32_t bytes_of(const Serve* s) { return s->dtype == RUAI_F32 ? 4u : 2u; }

int start(ruai_model* m, Serve* s) {
  ruai_ctx* c = m->ctx;
  const size_t pool = ((size_t)s->pages * m->KVl << s->page_log2) * m->hd * bytes_of(s);
  s->k.resize(m->L);
  s->v.resize(m->L);
  for (uint32_t l = 0; l < m->L; ++l) {
    RUAI_TRY(s->k[l].alloc(c, pool));
    RUAI_TRY(s->v[l].alloc(c, pool));
  }
  RUAI_TRY(s->table.alloc(c, (size_t)s->requests * s->row_pages * sizeof(int32_t)));
  RUAI_TRY(s->ring.alloc(c, (size_t)s->pages * sizeof(int32_t)));
  for (DevBuf& w : s->words) RUAI_TRY(w.alloc(c, 3 * sizeof(int32_t)));
  RUAI_CUDA(c, cudaMemsetAsync(s->table.p, 0xFF, s->table.bytes, c->stream));
  std::vector<int32_t> ring(s->pages);
  for (uint32_t i = 0; i < s->pages; ++i) ring[i] = (int32_t)i;
  const int32_t words[3] = {0, (int32_t)s->pages, 0};
  RUAI_CUDA(c, cudaMemcpyAsync(s->ring.p, ring.data(), s->ring.bytes, cudaMemcpyHostToDevice, c->stream));
  RUAI_CUDA(c, cudaMemcpyAsync(s->words[0].p, words, sizeof words, cudaMemcpyHostToDevice, c->stream));
  RUAI_CUDA(c, cudaStreamSynchronize(c->stream));
  s->len.assign(s->requests, 0);
  s->free = s->pages;
  return RUAI_OK;
}

int reserve(ruai_model* m, Serve* s, uint32_t tokens) {
  if (tokens <= s->tokens) return RUAI_OK;
  ruai_ctx* c = m->ctx;
  RUAI_CUDA(c, cudaStreamSynchronize(c->stream));
  s->tokens = 0;
  RUAI_TRY(s->plan.alloc(c, ((size_t)s->requests + 1 + 2 * (size_t)tokens) * sizeof(int32_t)));
  RUAI_TRY(s->up.alloc(c, (3 * (size_t)s->requests + tokens) * sizeof(int32_t)));
  const size_t rows = (size_t)tokens * m->Hl * m->hd * 2;
  if (s->dtype != RUAI_F32) {
    RUAI_TRY(s->q.alloc(c, rows));
    RUAI_TRY(s->att.alloc(c, rows));
  }
  s->tokens = tokens;
  return RUAI_OK;
}

// Issues the step: T tokens, the last of n_out requests with logits.  most_fresh, most_len: over the requests.
int issue(ruai_model* m, Serve* s, uint32_t T, uint32_t n_out, uint32_t most_fresh, uint32_t most_len) {
  ruai_ctx* c = m->ctx;
  const uint32_t R = s->requests, d = m->d, hd = m->hd, nql = m->Hl * hd, nkvl = m->KVl * hd, nqkv = nql + 2 * nkvl;
  const int32_t *cached = s->up.as<int32_t>(), *fresh = cached + R, *rows = fresh + R, *ids = rows + R;
  int32_t *starts = s->plan.as<int32_t>(), *positions = starts + R + 1, *slots = positions + T;
  RUAI_TRY(ruai_page_plan(c, cached, fresh, R, T, 1u << s->page_log2, s->table.as<int32_t>(), s->row_pages, s->ring.as<int32_t>(), s->pages, s->words[0].as<int32_t>(),
                          s->words[1].as<int32_t>(), starts, positions, slots));
  if (!T) return RUAI_OK;
  float *x = m->x.as<float>(), *qkv = m->qkv.as<float>(), *hb = m->hbuf.as<float>();
  RUAI_CUDA(c, ruai_launch(c, embed_at_kernel, dim3(T), dim3(256), 0, true, ids, (const int32_t*)positions, m->embed.as<float>(), m->llama ? nullptr : m->wpe.as<float>(), d, m->V,
                           m->max_pos, x, m->d_err.as<int>()));
  const bool f32 = s->dtype == RUAI_F32;
  for (uint32_t l = 0; l < m->L; ++l) {
    Layer& Ly = m->layers[l];
    GemvEpilogue e;
    e.bias = Ly.qkv.bias.as<float>();
    RUAI_TRY(model_normed_linear(m, Ly.qkv.w, x, Ly.n1w.as<float>(), Ly.n1b.as<float>(), T, qkv, e));
    const PagedPool pool = {s->k[l].p, s->v[l].p, s->pages, s->page_log2, m->KVl, hd, s->dtype};
    PagedAppend ap = {pool, qkv, RUAI_F32, nqkv, nql, nql + nkvl, T, m->Hl, m->llama ? hd : 0u, m->max_pos, m->llama ? m->rope_table.as<float2>() : nullptr,
                      positions, slots, f32 ? (void*)qkv : s->q.p, f32 ? nqkv : nql, c->status};
    if (f32 && !m->llama) ap.q_out = nullptr;  // queries are where they belong already
    RUAI_TRY(ruai_paged_append_launch(c, ap));
    void* att = f32 ? m->att.p : s->att.p;
    PagedAttn pa = {pool, f32 ? (const void*)qkv : s->q.p, att, f32 ? nqkv : nql, nql, s->table.as<int32_t>(), cached, starts, s->row_pages, R, T, m->Hl,
                    1.0f / sqrtf((float)hd), 0, most_fresh, most_len, c->status};
    RUAI_TRY(ruai_paged_attention_launch(c, pa));
    GemvEpilogue eo;
    eo.bias = Ly.o.bias.as<float>();
    eo.resid = x;
    RUAI_TRY(ruai_gemv_launch(c, Ly.o.w, att, s->dtype, nql, T, x, eo));
    GemvEpilogue eu;
    eu.bias = Ly.up.bias.as<float>();
    eu.act = m->llama ? ACT_SWIGLU : ACT_GELU;
    RUAI_TRY(model_normed_linear(m, Ly.up.w, x, Ly.n2w.as<float>(), Ly.n2b.as<float>(), T, hb, eu));
    GemvEpilogue ed;
    ed.bias = Ly.down.bias.as<float>();
    ed.resid = x;
    RUAI_TRY(ruai_gemv_launch(c, Ly.down.w, hb, RUAI_F32, m->fl, T, x, ed));
  }
  RUAI_TRY(ruai_take_rows(c, x, rows, n_out, d, m->xl.as<float>()));
  RUAI_TRY(model_normed_linear(m, m->head.w, m->xl.as<float>(), m->final_w.as<float>(), m->final_b.as<float>(), n_out, m->logits.as<float>(), GemvEpilogue()));
  return ruai_argmax(c, m->logits.as<float>(), m->Vl, n_out, m->Vl, m->d_ids.as<int32_t>(), 0);
}

}  // namespace

void serve_destroy(ruai_model* m) {
  if (!m->serve) return;
  release(m->serve);
  delete m->serve;
  m->serve = nullptr;
}

RUAI_API int ruai_model_serve_start(ruai_model* m, uint32_t pages, uint32_t page, uint32_t requests, uint32_t request_pages, int dtype) {
  if (!m) return ruai_fail(nullptr, RUAI_ERR_ARG, "model is NULL");
  ruai_ctx* c = m->ctx;
  if (!m->quantized || m->hy || m->world > 1) return model_fail(m, RUAI_ERR_UNSUPPORTED, "serving over pages needs a quantized Llama or GPT-2 on one GPU");
  if (page < 16 || page > 256 || (page & (page - 1))) return model_fail(m, RUAI_ERR_SHAPE, "pages of %u: a power of two from 16 to 256", page);
  if (!requests || requests > kPlanRowsMax || !request_pages || request_pages > (1u << 18))
    return model_fail(m, RUAI_ERR_SHAPE, "%u requests of up to %u pages: 1 to %u, 1 to %u", requests, request_pages, kPlanRowsMax, 1u << 18);
  DeviceGuard g(c->ordinal);
  const PagedPool pool = {nullptr, nullptr, pages, (uint32_t)__builtin_ctz(page), m->KVl, m->hd, dtype};
  RUAI_TRY(ruai_paged_check_pool(c, pool, "ruai_model_serve_start"));
  if ((unsigned long long)m->Hl * kPlanTokensMax >= (1ull << 31) || m->Hl / m->KVl > 256) return model_fail(m, RUAI_ERR_UNSUPPORTED, "%u heads over %u", m->Hl, m->KVl);
  RUAI_CUDA(c, cudaStreamSynchronize(c->stream));
  serve_destroy(m);
  Serve* s = new (std::nothrow) Serve();
  if (!s) return model_fail(m, RUAI_ERR_CUDA, "no host memory to serve with");
  s->pages = pages; s->page_log2 = pool.page_log2; s->requests = requests; s->row_pages = request_pages; s->dtype = dtype;
  int rc;
  try {
    rc = start(m, s);
  } catch (const std::bad_alloc&) {
    rc = model_fail(m, RUAI_ERR_CUDA, "no host memory for %u requests over %u pages", requests, pages);
  }
  if (rc != RUAI_OK) {
    (void)cudaGetLastError();
    release(s);
    delete s;
    return rc;
  }
  m->serve = s;
  return RUAI_OK;
}

RUAI_API int ruai_model_serve_stop(ruai_model* m) {
  if (!m) return ruai_fail(nullptr, RUAI_ERR_ARG, "model is NULL");
  DeviceGuard g(m->ctx->ordinal);
  RUAI_CUDA(m->ctx, cudaStreamSynchronize(m->ctx->stream));
  serve_destroy(m);
  return RUAI_OK;
}

RUAI_API int ruai_model_serve_free(const ruai_model* m, uint32_t* free_pages) {
  if (!m || !free_pages) return ruai_fail(m ? m->ctx : nullptr, RUAI_ERR_ARG, "ruai_model_serve_free: NULL argument");
  if (!m->serve) return ruai_fail(m->ctx, RUAI_ERR_UNSUPPORTED, "the model does not serve: call ruai_model_serve_start first");
  *free_pages = m->serve->free;
  return RUAI_OK;
}

RUAI_API int ruai_model_serve_step(ruai_model* m, const int32_t* fresh, const int32_t* ids, float* logits, int32_t* next) {
  if (!m || !fresh) return ruai_fail(m ? m->ctx : nullptr, RUAI_ERR_ARG, "ruai_model_serve_step: NULL argument");
  Serve* s = m->serve;
  if (!s) return model_fail(m, RUAI_ERR_UNSUPPORTED, "the model does not serve: call ruai_model_serve_start first");
  ruai_ctx* c = m->ctx;
  DeviceGuard g(c->ordinal);
  const uint32_t R = s->requests, page = 1u << s->page_log2;
  unsigned long long T = 0;
  uint32_t n_out = 0, need = 0, back = 0, most_fresh = 0, most_len = 0;
  bool any = false;
  auto held = [&](uint32_t n) { return (n + page - 1) >> s->page_log2; };
  for (uint32_t r = 0; r < R; ++r) {
    const uint32_t len = s->len[r];
    any = any || fresh[r] != 0;
    if (fresh[r] < 0) { back += held(len); continue; }
    if (!fresh[r]) continue;
    const unsigned long long now = (unsigned long long)len + (uint32_t)fresh[r];
    if (now > m->max_pos) return model_fail(m, RUAI_ERR_SHAPE, "context %llu of request %u exceeds %s %u", now, r, m->llama ? "max_position_embeddings" : "n_positions", m->max_pos);
    if (now > (unsigned long long)s->row_pages * page) return model_fail(m, RUAI_ERR_SHAPE, "request %u of %llu positions exceeds its %u pages of %u", r, now, s->row_pages, page);
    need += held((uint32_t)now) - held(len);
    T += (uint32_t)fresh[r];
    ++n_out;
    most_fresh = std::max(most_fresh, (uint32_t)fresh[r]);
    most_len = std::max(most_len, (uint32_t)now);
  }
  if (!any) return RUAI_OK;
  if (T > kPlanTokensMax) return model_fail(m, RUAI_ERR_SHAPE, "a step of %llu tokens: up to %u", T, kPlanTokensMax);
  if (T && !ids) return model_fail(m, RUAI_ERR_ARG, "ruai_model_serve_step: ids is NULL");
  // pages given back in this step are given out from the next one on
  if (need > s->free) return model_fail(m, RUAI_ERR_SHAPE, "the step needs %u more pages, %u are free", need, s->free);
  RUAI_TRY(reserve(m, s, std::max((uint32_t)T, 1u)));
  if (T) RUAI_TRY(model_activations(m, (uint32_t)T, n_out, 1, 2));
  try {
    s->sent.assign(3 * (size_t)R + T, 0);
  } catch (const std::bad_alloc&) {
    return model_fail(m, RUAI_ERR_CUDA, "no host memory for a step of %llu tokens", T);
  }
  uint32_t t = 0, o = 0;
  for (uint32_t r = 0; r < R; ++r) {
    s->sent[r] = (int32_t)s->len[r];
    s->sent[R + r] = fresh[r];
    if (fresh[r] > 0) {
      t += (uint32_t)fresh[r];
      s->sent[2 * R + o++] = (int32_t)t - 1;
    }
  }
  std::copy(ids, ids + T, s->sent.begin() + 3 * (size_t)R);
  RUAI_CUDA(c, cudaMemcpyAsync(s->up.p, s->sent.data(), s->sent.size() * sizeof(int32_t), cudaMemcpyHostToDevice, c->stream));
  RUAI_TRY(issue(m, s, (uint32_t)T, n_out, most_fresh, most_len));
  if (logits && n_out) RUAI_CUDA(c, cudaMemcpyAsync(logits, m->logits.p, (size_t)n_out * m->Vl * sizeof(float), cudaMemcpyDeviceToHost, c->stream));
  RUAI_TRY(model_read_back(m, next, next ? n_out : 0));
  // the step has ended well: its plan is the state now
  std::swap(s->words[0], s->words[1]);
  s->free = s->free + back - need;
  for (uint32_t r = 0; r < R; ++r) s->len[r] = fresh[r] < 0 ? 0 : s->len[r] + (uint32_t)fresh[r];
  return RUAI_OK;
}
