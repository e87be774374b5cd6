// Causal attention of every request's new tokens over its pages: softmax(scale q k^T + mask) v, where the token at position p sees
// keys p - window + 1 .. p (window 0: all of 0 .. p).
//
// rows_kernel: single tokens, drafts of a few, and whatever the kernels for chunks do not take.  The rows of an item are the (token,
// query head) pairs of one request and key head, 16 WR of them, so that a cached row is read once for all query heads of its key
// head.  HBM bounds it; an item's keys pass through once, in tiles of TK, with a running maximum m, sum l and weighted values o per row:
// o <- o 2^(m - m') + 2^(s - m') v, in f32 registers.
// 64 requests of 64 to 4096 positions (32 heads of 128, 8 of keys, bf16; 610 MB): 104 us, 5.8 TB/s; one of 32000: 37 us, 3.5 TB/s (the parts' way through
// scratch and its join are latency); 24 drafts of five tokens in f32 (124 MB): 40 us, the splitting of operands.  (Here and below: inputs
// that change from call to call.)
//   Split: the tiles of all items, in a row, are cut into equal runs, one per CTA, whatever the requests' lengths are (they are known to the
// device only).  An item cut by a run's end leaves (m, l, o) of its part in scratch, and the CTA that arrives last joins the parts, in
// their order: the same bits every time.
//   Tile: four warps; WK = 4 / WR of them share an item's rows and take a part of the tile's keys each.  A fifth walks the run and copies
// tiles ahead, across items, page by page (TMA boxes with the 128-byte swizzle, so that eight rows of a column lie in eight banks of 16 bytes).  Products are mma.sync: the tensor pipe waits for HBM here, and 16 rows
// by 8 keys fit few query heads where a tcgen05 tile would be a sixteenth full.  f32 operands are split in two tf32 numbers, x = hi + lo
// (22 bits), three of the four products; the
// tensor core's sums truncate, so it adds up 32 elements of a score and a tile's keys only, f32 registers the rest.  In 16 bits the weights are rounded once, to the values' type; l sums them unrounded.
// (bf16: 1.7e-3 of the outputs' norm off from 64 bits for single tokens, as with unrounded weights, whose outputs round to 1.7e-3; f16 2.2e-4 for 2.1e-4.
// Two pieces of each weight would double the products of weights and values.)  f16: under a power of two (weights_up).
//   A row that is not finite at the end is worked out again key by key (row_again): a key that it does not see, or that weighs
// nothing, must not reach it through 0 x inf.
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "attn_paged.cuh"
#include "pipeline.cuh"

namespace {

using pipe::smem_u32;

// ---- products ---------------------------------------------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, each of 11 bits (lo's last ones are cut by the tensor core)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"((uint64_t)map), "r"(x), "r"(y),
               "r"(smem_u32(bar))
               : "memory");
}

// ---- the kernel ---------------------------------------------------------------------------------------------------------------

constexpr int kSoftWarps = 4, kThreads = 32 * (kSoftWarps + 1);
constexpr int kSegments = 3;   // segments that the copying warp is ahead
constexpr int kItemCost = 1;   // tiles that an item's queries and results take as long as
constexpr int kTilesLeast = 3; // of a run, that cost included (three for one warp's rows, more for more: parts are as large as the rows are many)

// HP: the head's width, up to 64, 128 or 256.  WR: warps that have rows of their own, 16 each; 0: eight rows in all (f32).
template <typename T, int HP, int WR>
struct Shape {
  static constexpr bool F32 = sizeof(T) == 4, NARROW = WR == 0;
  static constexpr int WK = NARROW ? 4 : 4 / (NARROW ? 1 : WR), RW = NARROW ? 8 : 16, RB = RW * 4 / WK, TK = !F32 || NARROW ? 64 : HP == 256 && WR == 2 ? 16 : 32, KW = TK / WK;
  static_assert(!NARROW || (F32 && HP <= 128), "eight rows: f32, heads of up to 128");
  static constexpr int PANEL_ELEMS = 128 / (int)sizeof(T), PANELS = HP / PANEL_ELEMS, PANEL = TK * 128;  // 128 bytes of every key of a tile
  static constexpr int HALF = PANELS * PANEL, STAGE = 2 * HALF;                                          // keys, values
  static constexpr bool QSMEM = (F32 && !NARROW) || HP == 256;  // queries in shared memory, not in registers
  static constexpr int QPITCH = HP * (int)sizeof(T) + 16, QBYTES = QSMEM ? RB * QPITCH : 0;
  static constexpr int MERGE = kSoftWarps * RW * (HP + 4) * 4;  // the warps' results at the end, in the queries' place
  static constexpr int KEPT = MERGE > QBYTES ? MERGE : QBYTES;
  static constexpr bool ONE = HP == 256 || (HP == 128 && (WR == 4 || NARROW));  // one CTA per SM: two have too few registers (eight rows: too little shared memory)
  static constexpr int ROOM = (ONE ? 216 : 108) * 1024 - KEPT, STAGES = ROOM / STAGE < 6 ? ROOM / STAGE : 6;
  static constexpr int SMEM = STAGES * STAGE + KEPT + 1024;
  static_assert(STAGES >= 2 && PANELS >= 1, "two stages at least");
  static constexpr size_t PART = (size_t)RB * (HP + 2) * sizeof(float);  // one part of an item in scratch
};

struct alignas(64) Maps { CUtensorMap k, v; };

struct RowsPlan {
  float* parts;        // [CTAs][2]: the part that ends the item a CTA begins with, the part that begins the one it ends with
  unsigned* arrived;   // per CTA in which a cut item begins; zero between launches
  uint32_t rows_most;  // requests with more rows are another kernel's
  uint32_t box_rows;
};

// What the copying warp tells the others of a segment.
struct Work {
  Segment s;
  uint32_t ta, n;         // its tiles that a row sees
  uint32_t whole0, whole1;  // keys that all rows see: [whole0, whole1)
  uint32_t cut, first, last;  // 0: the whole item, 1: a part of it, 2: the part that begins it; the CTAs in which it begins and ends
  uint32_t more;
};

template <typename T, int HP, int WR>
__global__ void __launch_bounds__(kThreads, Shape<T, HP, WR>::ONE ? 1 : 2) rows_kernel(const PagedAttn a, const RowsPlan plan, const __grid_constant__ Maps maps) {
  using S = Shape<T, HP, WR>;
  constexpr int WK = S::WK, RB = S::RB, RW = S::RW, TK = S::TK, KW = S::KW, ST = S::STAGES, WRN = S::NARROW ? 1 : WR;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[ST], empty[ST], work_full[kSegments], work_empty[kSegments], meet;
  __shared__ Work s_work[kSegments];
  __shared__ unsigned long long s_part[kSoftWarps + 1], s_base;
  __shared__ uint32_t s_r, s_last;
  __shared__ volatile int s_abort;
  __shared__ float s_m[kSoftWarps][16], s_l[kSoftWarps][16];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t hd = a.pool.hd, KV = a.pool.KV, rep = a.H / KV, plog = a.pool.page_log2;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* res = reinterpret_cast<float*>(smem + ST * S::STAGE);  // [warp][16][HP + 4]
  unsigned char* qsm = smem + ST * S::STAGE;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) { pipe::mbar_init(&full[i], 1); pipe::mbar_init(&empty[i], kSoftWarps); }
    for (int i = 0; i < kSegments; ++i) { pipe::mbar_init(&work_full[i], 1); pipe::mbar_init(&work_empty[i], kSoftWarps); }
    pipe::mbar_init(&meet, kSoftWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
  }
  if (warp == 0 && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)(&maps.k + lane)) : "memory");
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- which tiles of which items
  auto tiles_of = [&](const PagedRequest& q) { return (q.len + TK - 1) / TK - paged_low(q.cached, a.window) / TK; };
  auto units_of = [&](const PagedRequest& q) -> unsigned long long {
    const uint32_t rows = q.fresh * rep;
    return rows == 0 || rows > plan.rows_most ? 0ull : (unsigned long long)(KV * ((rows + RB - 1) / RB)) * (tiles_of(q) + kItemCost);
  };
  const uint32_t per_thread = (a.R + kThreads - 1) / kThreads, ra = min(tid * per_thread, a.R), rb = min(ra + per_thread, a.R);
  unsigned long long mine = 0;
  for (uint32_t r = ra; r < rb; ++r) {
    PagedRequest q;
    paged_request(a, r, q);
    mine += units_of(q);
  }
  unsigned long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= (uint32_t)o) inc += v;
  }
  if (lane == 31) s_part[warp] = inc;
  __syncthreads();
  unsigned long long before = inc - mine, total = 0;
  for (uint32_t w = 0; w <= (uint32_t)kSoftWarps; ++w) {
    if (w < warp) before += s_part[w];
    total += s_part[w];
  }
  const unsigned long long per = max((total + gridDim.x - 1) / gridDim.x, (unsigned long long)(kTilesLeast + 2 * (WRN - 1)));
  const unsigned long long u0 = per * blockIdx.x, u1 = min(u0 + per, total);
  if (u0 >= u1) return;
  if (before <= u0 && u0 < before + mine) {
    unsigned long long base = before;
    for (uint32_t r = ra; r < rb; ++r) {
      PagedRequest q;
      paged_request(a, r, q);
      const unsigned long long n = units_of(q);
      if (u0 < base + n) { s_r = r; s_base = base; break; }
      base += n;
    }
  }
  __syncthreads();

  bool ok = true;
  // A warp whose wait ran out walks on without waiting, so that the others meet it; the results are void, and the host is told.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok) ok = __all_sync(0xFFFFFFFFu, !s_abort && pipe::mbar_wait(bar, parity));
    if (!ok) s_abort = 1;
    return ok;
  };

  if (warp == kSoftWarps) {
    // ===== segments, their keys and values: a lane per box
    uint32_t r = s_r, segs = 0, st = 0;  // stages asked for
    unsigned long long base = s_base, u = u0;
    const uint32_t boxes = TK / plan.box_rows, box = lane % boxes, panel = lane / boxes;
    const uint32_t dst = smem_u32(smem) + panel * S::PANEL + box * plan.box_rows * 128;
    auto page_at = [&](uint32_t tile, uint32_t len) {
      const uint32_t key = tile * TK + box * plan.box_rows;
      return key < len ? a.table[(size_t)r * a.table_ld + (key >> plog)] : -1;
    };
    while (u < u1 && ok) {
      Work w;
      w.s.r = r;
      paged_request(a, r, w.s.rq);
      const unsigned long long units = units_of(w.s.rq);
      if (u >= base + units) { base += units; ++r; continue; }
      const uint32_t tiles = tiles_of(w.s.rq), all_rows = w.s.rq.fresh * rep, blocks = (all_rows + RB - 1) / RB;
      const uint32_t item = (uint32_t)((u - base) / (tiles + kItemCost));
      const unsigned long long item_u = base + (unsigned long long)item * (tiles + kItemCost) + kItemCost;
      if (u < item_u) { u = item_u; continue; }
      const unsigned long long end = min(u1, item_u + tiles);
      const uint32_t skip = paged_low(w.s.rq.cached, a.window) / TK;
      w.s.g = item / blocks;
      w.s.row0 = (item % blocks) * RB;
      w.s.rows = min((uint32_t)RB, all_rows - w.s.row0);
      w.s.tile0 = skip + (uint32_t)(u - item_u);
      w.s.tile1 = skip + (uint32_t)(end - item_u);
      w.first = (uint32_t)(item_u / per);
      w.last = (uint32_t)((item_u + tiles - 1) / per);
      w.cut = w.first == w.last ? 0u : u == item_u ? 2u : 1u;
      // of these tiles, the ones that the rows see
      const uint32_t pos0 = w.s.rq.cached + w.s.row0 / rep, pos1 = w.s.rq.cached + (w.s.row0 + w.s.rows - 1) / rep;  // first and last row's positions
      w.whole0 = paged_low(pos1, a.window);
      w.whole1 = pos0 + 1;
      w.ta = max(w.s.tile0, paged_low(pos0, a.window) / TK);
      const uint32_t tb = min(w.s.tile1, pos1 / TK + 1);
      w.n = tb > w.ta ? tb - w.ta : 0;
      w.more = 1;
      int32_t pg = w.n ? page_at(w.ta, w.s.rq.len) : -1;
      if (segs >= kSegments && !wait(&work_empty[segs % kSegments], (segs / kSegments - 1) & 1u)) break;
      if (lane == 0) {
        s_work[segs % kSegments] = w;
        pipe::mbar_arrive(&work_full[segs % kSegments]);
      }
      ++segs;
      for (uint32_t i = 0; i < w.n; ++i, ++st) {
        const uint32_t key = (w.ta + i) * TK + box * plan.box_rows, slot = st % ST;
        if (pg < -1 || pg >= (int32_t)a.pool.pages || (pg < 0 && key < w.s.rq.len)) {
          if (a.status) atomicCAS(a.status, 0, kStatusPaged);
          pg = -1;
        }
        const int y = pg >= 0 ? (int)((((uint32_t)pg * KV + w.s.g) << plog) + (key & ((1u << plog) - 1u))) : 0;
        const bool take = pg >= 0 && panel * S::PANEL_ELEMS < hd;
        const uint32_t bytes = 2 * __popc(__ballot_sync(0xFFFFFFFFu, take && panel < (uint32_t)S::PANELS)) * plan.box_rows * 128;
        pg = i + 1 < w.n ? page_at(w.ta + i + 1, w.s.rq.len) : -1;
        if (st >= ST && !wait(&empty[slot], (st / ST - 1) & 1u)) break;
        if (lane == 0) pipe::mbar_expect_tx(&full[slot], bytes);
        __syncwarp();
        if (take && panel < (uint32_t)S::PANELS) {
          tma_2d(dst + slot * S::STAGE, &maps.k, (int)panel * S::PANEL_ELEMS, y, &full[slot]);
          tma_2d(dst + slot * S::STAGE + S::HALF, &maps.v, (int)panel * S::PANEL_ELEMS, y, &full[slot]);
        }
      }
      u = end;
    }
    if (ok && (segs < kSegments || wait(&work_empty[segs % kSegments], (segs / kSegments - 1) & 1u)) && lane == 0) {
      s_work[segs % kSegments].more = 0;
      pipe::mbar_arrive(&work_full[segs % kSegments]);
    }
    // leave no copy in flight into shared memory that another CTA may get
    for (uint32_t i = st > ST ? st - ST : 0; i < st; ++i) (void)pipe::mbar_wait(&full[i % ST], (i / ST) & 1u);
    if (s_abort && lane == 0 && a.status) atomicCAS(a.status, 0, 3);
    return;
  }

  // ===== products and softmax
  const uint32_t g4 = lane >> 2, t4 = lane & 3, wr = WRN == 1 ? 0 : warp % WRN, wk = warp / WRN;
  const float c = a.scale * kLog2e;
  uint32_t st = 0, meets = 0;
  auto gather = [&]() {  // the four warps meet
    __syncwarp();
    if (lane == 0) pipe::mbar_arrive(&meet);
    wait(&meet, meets++ & 1u);
  };
  for (uint32_t segs = 0;; ++segs) {
    if (!wait(&work_full[segs % kSegments], (segs / kSegments) & 1u)) return;  // the copying warp has given up: nobody meets again
    const Work& w = s_work[segs % kSegments];
    if (!w.more) return;
    const Segment& s = w.s;
    const uint32_t t0 = s.rq.t0, cached = s.rq.cached, len = s.rq.len, row_end = s.row0 + s.rows, n = w.n, ta = w.ta;

    // ---- queries
    const uint32_t row_lo = s.row0 + wr * 16 + g4, row_hi = row_lo + 8;
    auto q_at = [&](uint32_t row) { return static_cast<const T*>(a.q) + (size_t)(t0 + row / rep) * a.q_ld + (size_t)(s.g * rep + row % rep) * hd; };
    uint32_t qf[S::QSMEM ? 1 : S::NARROW ? HP / 8 : HP / 16][4];
    if constexpr (S::NARROW) {  // row g4: (hi, hi, lo, lo) of elements t4 and t4 + 4 of every eight
      const float* q = g4 < s.rows ? reinterpret_cast<const float*>(q_at(s.row0 + g4)) + t4 : nullptr;
#pragma unroll
      for (int e = 0; e < HP / 8; ++e) {
        const bool in = q && e * 8 < (int)hd;
        split_tf32(in ? q[e * 8] : 0.0f, qf[e][0], qf[e][2]);
        split_tf32(in ? q[e * 8 + 4] : 0.0f, qf[e][1], qf[e][3]);
      }
    } else if constexpr (S::QSMEM) {
      constexpr uint32_t kChunks = HP * sizeof(T) / 16;
      for (uint32_t x = tid; x < RB * kChunks; x += 32 * kSoftWarps) {
        const uint32_t row = x / kChunks, col = x % kChunks;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < s.rows && col * (16 / sizeof(T)) < hd) v = *reinterpret_cast<const uint4*>(q_at(s.row0 + row) + col * (16 / sizeof(T)));
        *reinterpret_cast<uint4*>(qsm + row * S::QPITCH + col * 16) = v;
      }
      gather();
    } else {
      const T* q0 = row_lo < row_end ? q_at(row_lo) : nullptr;
      const T* q1 = row_hi < row_end ? q_at(row_hi) : nullptr;
#pragma unroll
      for (int e = 0; e < HP / 16; ++e)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t col = e * 16 + h * 8 + 2 * t4;
          qf[e][2 * h] = q0 && col < hd ? *reinterpret_cast<const uint32_t*>(q0 + col) : 0u;
          qf[e][2 * h + 1] = q1 && col < hd ? *reinterpret_cast<const uint32_t*>(q1 + col) : 0u;
        }
    }
    // the positions of this thread's two rows: g4 and g4 + 8 of its warp's, or 2 t4 and 2 t4 + 1 of eight
    const uint32_t p_lo = cached + min(S::NARROW ? s.row0 + 2 * t4 : row_lo, row_end - 1) / rep, p_hi = cached + min(S::NARROW ? s.row0 + 2 * t4 + 1 : row_hi, row_end - 1) / rep;
    const uint32_t l_lo = paged_low(p_lo, a.window), l_hi = paged_low(p_hi, a.window), whole0 = w.whole0, whole1 = w.whole1;

    constexpr int OT = S::NARROW ? HP / 16 : HP / 8;  // tiles of the output: 16 rows x 8 columns, or 16 columns x 8 rows
    float o[OT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;

    for (uint32_t i = 0; i < n; ++i, ++st) {
      const uint32_t slot = st % ST;
      wait(&full[slot], (st / ST) & 1u);
      unsigned char* ks = smem + slot * S::STAGE + wk * KW * 128;
      unsigned char* vs = ks + S::HALF;
      const uint32_t key0 = (ta + i) * TK + wk * KW;
      if (key0 + KW > len) {  // positions behind the request's end: their values weigh nothing, and must be numbers for that
        for (uint32_t x = lane; x < KW * 8 * S::PANELS; x += 32) {
          const uint32_t row = x / 8 % KW;
          if (key0 + row >= len) *reinterpret_cast<uint4*>(vs + x / (8 * KW) * S::PANEL + row * 128 + (x & 7u) * 16) = make_uint4(0, 0, 0, 0);
        }
        pipe::fence_proxy_async_smem();
        __syncwarp();
      }
      if constexpr (S::NARROW) {
        // S^T = K Q^T, 16 keys x 8 rows: key g4 (and g4 + 8) of rows 2 t4 and 2 t4 + 1; half the products of 16 rows with 8 of them empty
        float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const unsigned char* kf = ks + g4 * 128 + t4 * 4;
#pragma unroll
        for (int p0 = 0; p0 < S::PANELS; p0 += 2) {
          if (p0 * 32 >= (int)hd) break;
          float part[2][2][4];
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) part[y][0][x] = part[y][1][x] = 0.0f;
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            uint32_t ah[2][4], al[2][4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const unsigned char* kj = kf + (p0 + y) * S::PANEL;
              const uint32_t c0 = ((2 * f) ^ g4) << 4, c1 = ((2 * f + 1) ^ g4) << 4;
              split_tf32(*reinterpret_cast<const float*>(kj + c0), ah[y][0], al[y][0]);
              split_tf32(*reinterpret_cast<const float*>(kj + 8 * 128 + c0), ah[y][1], al[y][1]);
              split_tf32(*reinterpret_cast<const float*>(kj + c1), ah[y][2], al[y][2]);
              split_tf32(*reinterpret_cast<const float*>(kj + 8 * 128 + c1), ah[y][3], al[y][3]);
            }
#pragma unroll
            for (int z = 0; z < 3; ++z)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t* q = qf[(p0 + y) * 4 + f];
                mma8(part[y][z == 2], z == 0 ? al[y] : ah[y], z == 1 ? q[2] : q[0], z == 1 ? q[3] : q[1]);
              }
          }
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if ((p0 + y) * 32 < (int)hd) {  // a panel behind the head's end may hold anything
#pragma unroll
              for (int x = 0; x < 4; ++x) sc[x] += part[y][0][x] + part[y][1][x];
            }
        }
        const bool whole = key0 >= whole0 && key0 + KW <= whole1;
        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t key = key0 + g4 + (x & 2) * 4;
          sc[x] = whole || (key <= (x & 1 ? p_hi : p_lo) && key >= (x & 1 ? l_hi : l_lo)) ? sc[x] * c : -INFINITY;
          if (x & 1) x1 = fmaxf(x1, sc[x]);
          else x0 = fmaxf(x0, sc[x]);
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, off));
          x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, off));
        }
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        if (__any_sync(0xFFFFFFFFu, n0 > m0 || n1 > m1)) {
          const float c0 = m0 == -INFINITY ? 0.0f : exp2_of(m0 - n0), c1 = m1 == -INFINITY ? 0.0f : exp2_of(m1 - n1);
          l0 *= c0;
          l1 *= c1;
#pragma unroll
          for (int d = 0; d < OT; ++d) { o[d][0] *= c0; o[d][1] *= c1; o[d][2] *= c0; o[d][3] *= c1; }
          m0 = n0;
          m1 = n1;
        }
        const float b0 = m0 == -INFINITY ? 0.0f : m0, b1 = m1 == -INFINITY ? 0.0f : m1;
        sc[0] = exp2_of(sc[0] - b0); sc[1] = exp2_of(sc[1] - b1);
        sc[2] = exp2_of(sc[2] - b0); sc[3] = exp2_of(sc[3] - b1);
        l0 += sc[0] + sc[2];
        l1 += sc[1] + sc[3];
        // O^T += V^T P^T, 16 columns x 8 rows; the product's k is key 2 t4 for t4, 2 t4 + 1 for t4 + 4
        uint32_t ph[2][2], pl[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int from = (int)((2 * t4 + y) * 4 + (g4 >> 1));
            const float even = __shfl_sync(0xFFFFFFFFu, sc[2 * h], from), odd = __shfl_sync(0xFFFFFFFFu, sc[2 * h + 1], from);
            split_tf32(g4 & 1 ? odd : even, ph[h][y], pl[h][y]);
          }
        const unsigned char* v0 = vs + 2 * t4 * 128 + (g4 & 3) * 4;
#pragma unroll
        for (int d0 = 0; d0 < OT; d0 += 2) {
          if (d0 * 16 >= (int)hd) break;
          float part[2][2][4];
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) part[y][0][x] = part[y][1][x] = 0.0f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned char* vj = v0 + (d0 / 2) * S::PANEL + h * 8 * 128;
            uint32_t ah[2][4], al[2][4];
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int x = 0; x < 4; ++x) {  // columns g4 and g4 + 8, keys 2 t4 and 2 t4 + 1
                const uint32_t ch = 4 * y + (g4 >> 2) + (x & 1) * 2, key = 2 * t4 + (x >> 1);
                split_tf32(*reinterpret_cast<const float*>(vj + (x >> 1) * 128 + ((ch ^ key) << 4)), ah[y][x], al[y][x]);
              }
#pragma unroll
            for (int z = 0; z < 3; ++z)
#pragma unroll
              for (int y = 0; y < 2; ++y) mma8(part[y][z == 2], z == 0 ? al[y] : ah[y], z == 1 ? pl[h][0] : ph[h][0], z == 1 ? pl[h][1] : ph[h][1]);
          }
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[d0 + y][x] += part[y][0][x] + part[y][1][x];
        }
      } else {
      float sc[KW / 8][4];
#pragma unroll
      for (int j = 0; j < KW / 8; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
      if constexpr (!S::F32) {
        const uint32_t kaddr = smem_u32(ks) + ((lane & 7) + ((lane >> 4) << 3)) * 128, hi = (lane >> 3) & 1, sw = lane & 7;
        const uint32_t qaddr = smem_u32(qsm) + (wr * 16 + (lane & 15)) * S::QPITCH + (lane >> 4) * 16;
#pragma unroll
        for (int e = 0; e < HP / 16; ++e) {
          if (HP != 64 && e * 16 >= (int)hd) break;
          uint32_t qa[4];
          if constexpr (S::QSMEM) ldmatrix4(qa, qaddr + e * 32);
          else { qa[0] = qf[e][0]; qa[1] = qf[e][1]; qa[2] = qf[e][2]; qa[3] = qf[e][3]; }
#pragma unroll
          for (int j = 0; j < KW / 16; ++j) {
            uint32_t b[4];
            ldmatrix4(b, kaddr + (e / 4) * S::PANEL + j * 16 * 128 + ((((e & 3) * 2 + hi) ^ sw) << 4));
            mma16<T>(sc[2 * j], qa, b[0], b[1]);
            mma16<T>(sc[2 * j + 1], qa, b[2], b[3]);
          }
        }
      } else {
        const unsigned char* kf = ks + g4 * 128 + t4 * 4;
        const float* qs = reinterpret_cast<const float*>(qsm) + (wr * 16 + g4) * (S::QPITCH / 4) + t4;
        constexpr int G = KW >= 32 ? 1 : HP == 64 ? 2 : 32 / KW;  // panels at a time: four sums that do not wait for one another, where there are
#pragma unroll 1
        for (uint32_t p0 = 0; 32 * p0 < hd; p0 += G) {
          float part[G][KW / 8][4];
#pragma unroll
          for (int y = 0; y < G; ++y)
#pragma unroll
            for (int j = 0; j < KW / 8; ++j) part[y][j][0] = part[y][j][1] = part[y][j][2] = part[y][j][3] = 0.0f;
#pragma unroll
          for (uint32_t f = 0; f < 4; ++f) {  // eight elements of each of the panels; zeros behind the head's end
            uint32_t ah[G][4], al[G][4], bh[G][KW / 8][2], bl[G][KW / 8][2];
#pragma unroll
            for (int y = 0; y < G; ++y) {
              const float* q = qs + (p0 + y) * 32 + f * 8;
              split_tf32(q[0], ah[y][0], al[y][0]);
              split_tf32(q[8 * (S::QPITCH / 4)], ah[y][1], al[y][1]);
              split_tf32(q[4], ah[y][2], al[y][2]);
              split_tf32(q[8 * (S::QPITCH / 4) + 4], ah[y][3], al[y][3]);
#pragma unroll
              for (int j = 0; j < KW / 8; ++j) {
                const unsigned char* kj = kf + (p0 + y) * S::PANEL + j * 8 * 128;
                split_tf32(*reinterpret_cast<const float*>(kj + (((2 * f) ^ g4) << 4)), bh[y][j][0], bl[y][j][0]);
                split_tf32(*reinterpret_cast<const float*>(kj + (((2 * f + 1) ^ g4) << 4)), bh[y][j][1], bl[y][j][1]);
              }
            }
#pragma unroll
            for (int z = 0; z < 3; ++z)  // the small products first
#pragma unroll
              for (int y = 0; y < G; ++y)
#pragma unroll
                for (int j = 0; j < KW / 8; ++j)
                  mma8(part[y][j], z == 0 ? al[y] : ah[y], z == 1 ? bl[y][j][0] : bh[y][j][0], z == 1 ? bl[y][j][1] : bh[y][j][1]);
          }
#pragma unroll
          for (int y = 0; y < G; ++y)
            if (32 * (p0 + y) < hd) {
#pragma unroll
              for (int j = 0; j < KW / 8; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[j][x] += part[y][j][x];
            }
        }
      }
      // ---- softmax; row g4 in elements 0 and 1, row g4 + 8 in 2 and 3
      const bool whole = key0 >= whole0 && key0 + KW <= whole1;
#pragma unroll
      for (int j = 0; j < KW / 8; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t key = key0 + j * 8 + 2 * t4 + (x & 1);
          const float v = sc[j][x] * c;
          sc[j][x] = whole || (key <= (x < 2 ? p_lo : p_hi) && key >= (x < 2 ? l_lo : l_hi)) ? v : -INFINITY;
        }
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int j = 0; j < KW / 8; ++j) {
        x0 = fmaxf(x0, fmaxf(sc[j][0], sc[j][1]));
        x1 = fmaxf(x1, fmaxf(sc[j][2], sc[j][3]));
      }
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, off));
        x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, off));
      }
      const float n0 = fmaxf(m0, x0 - weights_up<T>(15.0f)), n1 = fmaxf(m1, x1 - weights_up<T>(15.0f));
      if (__any_sync(0xFFFFFFFFu, n0 > m0 || n1 > m1)) {
        const float c0 = m0 == -INFINITY ? 0.0f : exp2_of(m0 - n0), c1 = m1 == -INFINITY ? 0.0f : exp2_of(m1 - n1);
        l0 *= c0;
        l1 *= c1;
#pragma unroll
        for (int d = 0; d < HP / 8; ++d) { o[d][0] *= c0; o[d][1] *= c0; o[d][2] *= c1; o[d][3] *= c1; }
        m0 = n0;
        m1 = n1;
      }
      const float b0 = m0 == -INFINITY ? 0.0f : m0, b1 = m1 == -INFINITY ? 0.0f : m1;
#pragma unroll
      for (int j = 0; j < KW / 8; ++j) {
        sc[j][0] = exp2_of(sc[j][0] - b0); sc[j][1] = exp2_of(sc[j][1] - b0);
        sc[j][2] = exp2_of(sc[j][2] - b1); sc[j][3] = exp2_of(sc[j][3] - b1);
        l0 += sc[j][0] + sc[j][1];
        l1 += sc[j][2] + sc[j][3];
      }
      // ---- weighted values
      if constexpr (!S::F32) {
        const uint32_t vaddr = smem_u32(vs) + ((lane & 7) + ((lane >> 3) & 1) * 8) * 128, hi = lane >> 4, sw = lane & 7;
#pragma unroll
        for (int j = 0; j < KW / 16; ++j) {
          const uint32_t pa[4] = {pack2<T>(sc[2 * j][0], sc[2 * j][1]), pack2<T>(sc[2 * j][2], sc[2 * j][3]), pack2<T>(sc[2 * j + 1][0], sc[2 * j + 1][1]),
                                  pack2<T>(sc[2 * j + 1][2], sc[2 * j + 1][3])};
#pragma unroll
          for (int d = 0; d < HP / 16; ++d) {
            if (HP != 64 && d * 16 >= (int)hd) break;
            uint32_t b[4];
            ldmatrix4t(b, vaddr + (d / 4) * S::PANEL + j * 16 * 128 + ((((d & 3) * 2 + hi) ^ sw) << 4));
            mma16<T>(o[2 * d], pa, b[0], b[1]);
            mma16<T>(o[2 * d + 1], pa, b[2], b[3]);
          }
        }
      } else {
        const unsigned char* v0 = vs + 2 * t4 * 128 + (g4 & 3) * 4;
        uint32_t ph[KW / 8][4], pl[KW / 8][4];  // the product's k is key 2 t4 for t4, 2 t4 + 1 for t4 + 4
#pragma unroll
        for (int j = 0; j < KW / 8; ++j) {
          split_tf32(sc[j][0], ph[j][0], pl[j][0]);
          split_tf32(sc[j][2], ph[j][1], pl[j][1]);
          split_tf32(sc[j][1], ph[j][2], pl[j][2]);
          split_tf32(sc[j][3], ph[j][3], pl[j][3]);
        }
#pragma unroll
        for (int d0 = 0; d0 < HP / 8; d0 += 4) {  // a panel of 32 columns: four sums that do not wait for one another
          if (d0 * 8 >= (int)hd) break;
          float part[4][4];
#pragma unroll
          for (int y = 0; y < 4; ++y) part[y][0] = part[y][1] = part[y][2] = part[y][3] = 0.0f;
#pragma unroll
          for (int j = 0; j < KW / 8; ++j) {
            const unsigned char* vj = v0 + (d0 / 4) * S::PANEL + j * 8 * 128;
            uint32_t bh[4][2], bl[4][2];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t ch = 2 * y + (g4 >> 2);
              split_tf32(*reinterpret_cast<const float*>(vj + ((ch ^ (2 * t4)) << 4)), bh[y][0], bl[y][0]);
              split_tf32(*reinterpret_cast<const float*>(vj + 128 + ((ch ^ (2 * t4 + 1)) << 4)), bh[y][1], bl[y][1]);
            }
#pragma unroll
            for (int z = 0; z < 3; ++z)
#pragma unroll
              for (int y = 0; y < 4; ++y) mma8(part[y], z == 0 ? pl[j] : ph[j], z == 1 ? bl[y][0] : bh[y][0], z == 1 ? bl[y][1] : bh[y][1]);
          }
#pragma unroll
          for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[d0 + y][x] += part[y][x];
        }
      }
      }
      __syncwarp();
      if (lane == 0) pipe::mbar_arrive(&empty[slot]);
    }

    // ---- the warps' results meet
#pragma unroll
    for (int off = S::NARROW ? 4 : 1; off < (S::NARROW ? 32 : 4); off <<= 1) {
      l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, off);
      l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, off);
    }
    if constexpr (S::QSMEM) gather();  // the queries have been read
    if constexpr (S::NARROW) {
      float* d0 = res + (warp * 8 + 2 * t4) * (HP + 4) + g4;
#pragma unroll
      for (int d = 0; d < OT; ++d) {
        if (d * 16 >= (int)hd) break;
        d0[d * 16] = o[d][0]; d0[HP + 4 + d * 16] = o[d][1];
        d0[d * 16 + 8] = o[d][2]; d0[HP + 4 + d * 16 + 8] = o[d][3];
      }
      if (g4 == 0) { s_m[warp][2 * t4] = m0; s_l[warp][2 * t4] = l0; s_m[warp][2 * t4 + 1] = m1; s_l[warp][2 * t4 + 1] = l1; }
    } else {
      float* d0 = res + (warp * 16 + g4) * (HP + 4) + 2 * t4;
      float* d1 = d0 + 8 * (HP + 4);
#pragma unroll
      for (int d = 0; d < HP / 8; ++d) {
        if (d * 8 >= (int)hd) break;
        *reinterpret_cast<float2*>(d0 + d * 8) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(d1 + d * 8) = make_float2(o[d][2], o[d][3]);
      }
      if (t4 == 0) { s_m[warp][g4] = m0; s_l[warp][g4] = l0; s_m[warp][g4 + 8] = m1; s_l[warp][g4 + 8] = l1; }
    }
    gather();
    const uint32_t cut = w.cut, first = w.first, last = w.last;
    float* part = plan.parts + ((size_t)blockIdx.x * 2 + (cut == 2 ? 1 : 0)) * (RB * (HP + 2));
    auto out_at = [&](uint32_t row) { return static_cast<T*>(a.out) + (size_t)(t0 + row / rep) * a.out_ld + (size_t)(s.g * rep + row % rep) * hd; };
    // a warp per row
    for (uint32_t row = warp; row < s.rows; row += kSoftWarps) {
      const uint32_t w0 = row / RW, rr = row % RW;  // the row's warps are w0, w0 + WR, ...
      float m = -INFINITY, l = 0.0f, f[WK], v[HP / 32];
#pragma unroll
      for (int x = 0; x < WK; ++x) m = fmaxf(m, s_m[w0 + x * WRN][rr]);
#pragma unroll
      for (int x = 0; x < WK; ++x) {
        const float mw = s_m[w0 + x * WRN][rr];
        f[x] = mw == -INFINITY ? 0.0f : exp2_of(mw - m);
        l = fmaf(s_l[w0 + x * WRN][rr], f[x], l);
      }
      bool fine = isfinite(l);
#pragma unroll
      for (int j = 0; j < HP / 32; ++j) {
        const uint32_t e = lane + 32 * j;
        v[j] = 0.0f;
        if (e < hd) {
#pragma unroll
          for (int x = 0; x < WK; ++x) v[j] = fmaf(res[((w0 + x * WRN) * RW + rr) * (HP + 4) + e], f[x], v[j]);
          fine = fine && isfinite(v[j]);
        }
      }
      if (!__all_sync(0xFFFFFFFFu, fine)) {
        float* again = res + (w0 * RW + rr) * (HP + 4);
        row_again<T>(a, s, rep, s.row0 + row, s.tile0 * TK, s.tile1 * TK, again, m, l);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < HP / 32; ++j) v[j] = lane + 32 * j < hd ? again[lane + 32 * j] : 0.0f;
      }
      if (!cut) {
        T* dst = out_at(s.row0 + row);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int j = 0; j < HP / 32; ++j)
          if (lane + 32 * j < hd) dst[lane + 32 * j] = from_f32<T>(l == 0.0f ? 0.0f : v[j] * inv);
      } else {
        float* dst = part + row * HP;
#pragma unroll
        for (int j = 0; j < HP / 32; ++j) dst[lane + 32 * j] = v[j];
        if (lane == 0) { part[RB * HP + row] = m; part[RB * HP + RB + row] = l; }
      }
    }
    if (cut) {
      // ---- the item's parts, joined by the CTA that comes last
      __threadfence();
      gather();
      if (tid == 0) s_last = atomicAdd(&plan.arrived[first], 1u) == last - first ? 1u : 0u;
      gather();
      if (s_last) {
        __threadfence();
        auto part_of = [&](uint32_t p) { return plan.parts + ((size_t)p * 2 + (p == first ? 1 : 0)) * (RB * (HP + 2)); };
        constexpr int C = HP / 32 < 4 ? HP / 32 : 4, VECS = HP / 32 / C;  // columns of a load, loads of a row, per lane
        for (uint32_t row = warp; row < s.rows; row += kSoftWarps) {
          float m = -INFINITY, l = 0.0f, v[VECS][C];
#pragma unroll
          for (int x = 0; x < VECS; ++x)
#pragma unroll
            for (int y = 0; y < C; ++y) v[x][y] = 0.0f;
          for (uint32_t p0 = first; p0 <= last; p0 += 32) {  // 32 parts' maxima and sums at a time, a lane each
            const uint32_t np = min(32u, last + 1 - p0);
            const float mp = lane < np ? __ldcg(part_of(p0 + lane) + RB * HP + row) : -INFINITY, lp = lane < np ? __ldcg(part_of(p0 + lane) + RB * HP + RB + row) : 0.0f;
            float top = mp;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
            const float m_new = fmaxf(m, top), corr = m == -INFINITY ? 0.0f : exp2_of(m - m_new), f = mp == -INFINITY ? 0.0f : exp2_of(mp - m_new);
            float add = lp * f;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) add += __shfl_xor_sync(0xFFFFFFFFu, add, off);
            l = fmaf(l, corr, add);
            m = m_new;
#pragma unroll
            for (int x = 0; x < VECS; ++x)
#pragma unroll
              for (int y = 0; y < C; ++y) v[x][y] *= corr;
#pragma unroll 8
            for (uint32_t i = 0; i < np; ++i) {
              const float fi = __shfl_sync(0xFFFFFFFFu, f, (int)i);
              const float* src = part_of(p0 + i) + row * HP + lane * C;
#pragma unroll
              for (int x = 0; x < VECS; ++x) {
                float w[C];
                if constexpr (C == 4) *reinterpret_cast<float4*>(w) = __ldcg(reinterpret_cast<const float4*>(src + x * 128));
                else *reinterpret_cast<float2*>(w) = __ldcg(reinterpret_cast<const float2*>(src));
#pragma unroll
                for (int y = 0; y < C; ++y) v[x][y] = fmaf(w[y], fi, v[x][y]);
              }
            }
          }
          T* dst = out_at(s.row0 + row);
#pragma unroll
          for (int x = 0; x < VECS; ++x)
#pragma unroll
            for (int y = 0; y < C; ++y) {
              const uint32_t e = x * 128 + lane * C + y;
              if (e < hd) dst[e] = from_f32<T>(l == 0.0f ? 0.0f : v[x][y] / l);
            }
        }
        if (tid == 0) plan.arrived[first] = 0;
      }
    }
    gather();  // the results have been read
    if (lane == 0) pipe::mbar_arrive(&work_empty[segs % kSegments]);
  }
}

// A pool's rows (page, key head, position in the page) of hd elements, in boxes of box_rows x 128 bytes; elements past hd read as zero.
CUresult encode(CUtensorMap* map, const PagedPool& p, void* base, uint32_t box_rows) {
  const bool f32 = p.dtype == RUAI_F32;
  const cuuint64_t dims[2] = {p.hd, ((cuuint64_t)p.pages * p.KV) << p.page_log2}, strides[1] = {(cuuint64_t)p.hd * (f32 ? 4 : 2)};
  const cuuint32_t box[2] = {f32 ? 32u : 64u, box_rows}, one[2] = {1, 1};
  return ruai_tensor_map_fn()(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : p.dtype == RUAI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims,
                              strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <typename T, int HP, int WR>
int launch_rows(ruai_ctx* c, const PagedAttn& a, uint32_t rows_most) {
  using S = Shape<T, HP, WR>;
  static int per_sm[64] = {};
  int& n = per_sm[c->ordinal & 63];
  if (!n) {
    RUAI_CUDA(c, cudaFuncSetAttribute(rows_kernel<T, HP, WR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    RUAI_CUDA(c, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, rows_kernel<T, HP, WR>, kThreads, S::SMEM));
    n = std::max(n, 1);
  }
  RowsPlan p = {nullptr, nullptr, rows_most, std::min(1u << a.pool.page_log2, (uint32_t)S::TK)};
  Maps maps;
  if (!ruai_tensor_map_fn()) return ruai_fail(c, RUAI_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const CUresult rk = encode(&maps.k, a.pool, a.pool.k, p.box_rows), rv = encode(&maps.v, a.pool, a.pool.v, p.box_rows);
  if (rk != CUDA_SUCCESS || rv != CUDA_SUCCESS)
    return ruai_fail(c, RUAI_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d, %d) for %u pages of %u heads of %u", (int)rk, (int)rv, a.pool.pages, a.pool.KV, a.pool.hd);
  // a run per resident CTA, as far as the context's first scratch holds their parts: it never grows for them
  const uint32_t grid = (uint32_t)std::min<size_t>((size_t)c->sm_count * n, kScratchBytes / (2 * S::PART));
  RUAI_TRY(ruai_ctx_reserve(c, grid * 2 * S::PART, grid));  // it is there, unless an earlier call has run out of memory
  p.parts = c->partial;
  p.arrived = c->counters;
  RUAI_CUDA(c, ruai_launch(c, rows_kernel<T, HP, WR>, dim3(grid), dim3(kThreads), S::SMEM, true, a, p, maps));
  return RUAI_OK;
}

template <typename T, int HP>
int launch_width(ruai_ctx* c, const PagedAttn& a, uint32_t rows, uint32_t rows_most) {
  if constexpr (sizeof(T) == 4 && HP <= 128) {
    if (rows <= 8) return launch_rows<T, HP, 0>(c, a, rows_most);
  }
  if (rows <= 16) return launch_rows<T, HP, 1>(c, a, rows_most);
  if (rows <= 32 || HP == 256) return launch_rows<T, HP, 2>(c, a, rows_most);
  return launch_rows<T, HP == 256 ? 128 : HP, 4>(c, a, rows_most);
}

template <typename T>
int launch_type(ruai_ctx* c, const PagedAttn& a, uint32_t rows, uint32_t rows_most) {
  return a.pool.hd <= 64    ? launch_width<T, 64>(c, a, rows, rows_most)
         : a.pool.hd <= 128 ? launch_width<T, 128>(c, a, rows, rows_most)
                            : launch_width<T, 256>(c, a, rows, rows_most);
}

// A step whose requests all have few rows stays on the kernel here; else it keeps those of up to kRowsBeside rows.
constexpr uint32_t kRowsBeside = 16;
// f16 and bf16: up to 24 rows.  us, here | attn_paged_tc.cu, heads of 128, 8 of keys: 20 rows of 4 requests of 1000 28 | 24 (a rule by rows alone leaves
// these 4 us), of 32 47 | 47, 24 rows (heads of 64) of 64 requests of 200 11 | 19; 32 rows of 8 requests of 4000 60 | 44, of 64 of 200 46 | 33, of one of 8000
// 49 | 27; 64 rows of 8 of 4000 110 | 44.
constexpr uint32_t kRowsAlone = 24;
// f32: from 33 rows on whichever is the shorter by the times of both, which go by the pairs of a row and a key here, and there by the splitting
// of all keys and the longest row of key tiles, which one CTA walks.  us, here | attn_prefill_tc.cu (the same heads): 64 rows of 8 requests of 4000 270 |
// 246, of 64 of 200 187 | 138, of one of 8000 118 | 265; 48 rows of 32 requests of 1000 272 | 263; 32 rows of 32 requests of 1000 (heads of 64) 60 | 75.
bool in_pieces(const ruai_ctx* c, const PagedAttn& a, uint32_t rows) {
  if (rows <= 32) return false;
  const double len = a.most_len, rep = a.H / a.pool.KV, items = a.pool.KV * ceil(a.tokens * rep / 128.0);
  const double many = ceil((double)(a.tokens > a.R ? a.tokens - a.R : 0) / (a.most_fresh > 1 ? a.most_fresh - 1 : 1));  // requests with as many rows as the most
  const double here = 10.0 + a.tokens * (double)a.H * len / 36e3, split = std::min(many, (double)a.R) * len * a.pool.KV * a.pool.hd * 16.0 / 3e6, there = split + 15.0 + 2.0 * ceil(len / 64.0) * ceil(items / c->sm_count);
  return there < here;
}

}  // namespace

int ruai_paged_attention_launch(ruai_ctx* c, const PagedAttn& a) {
  const ScratchLock held(c->scratch_lock);
  if (!c->partial_in_graph || !c->counters_in_graph) {  // parts and counters lie in the context's scratch, whose address a graph keeps
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    RUAI_CUDA(c, cudaStreamIsCapturing(c->stream, &capture));
    if (capture != cudaStreamCaptureStatusNone) c->partial_in_graph = c->counters_in_graph = true;
  }
  uint32_t rows = a.most_fresh * (a.H / a.pool.KV), rows_most = 0xFFFFFFFFu;  // below 2^31: most_fresh is checked against the tokens
  if (a.pool.dtype == RUAI_F32 ? in_pieces(c, a, rows) : rows > kRowsAlone) {
    const uint32_t rep = a.H / a.pool.KV, over = a.R > 1 && rep <= kRowsBeside ? kRowsBeside : 0u;
    const int took = a.pool.dtype == RUAI_F32 ? ruai_paged_attention_pieces(c, a, over) : ruai_paged_attention_tc(c, a, over);
    if (took < 0) return RUAI_ERR_CUDA;
    if (took && !over) return RUAI_OK;
    if (took) rows = rows_most = over;
  }
  return a.pool.dtype == RUAI_F32   ? launch_type<float>(c, a, rows, rows_most)
         : a.pool.dtype == RUAI_F16 ? launch_type<__half>(c, a, rows, rows_most)
                                    : launch_type<__nv_bfloat16>(c, a, rows, rows_most);
}
