// Attention of chunks over pages on the tensor cores (tcgen05), f16 and bf16: what attn_paged.cu computes, for the requests with many rows.
//
// An item is two tiles of up to 128 rows (token, query head; whole tokens) of one request and key head, over the keys that any of them
// sees, 128 at a time.  One warp copies a tile's keys and values page by page (TMA boxes of a page's rows, so that pages lie in shared
// memory as one tile, 128-byte swizzle); one issues the MMAs, S_t = Q_t K^T and O_t += P_t V in turn for both row tiles, so that one
// tile's products run beside the other's softmax; one finds the items
// for the others; two warpgroups are the softmax, a thread per row.  Scores,
// probabilities (written over the scores, rounded once to the values' type) and outputs stay in tensor memory: 2 x (128 + 128)
// columns.  Outputs are rescaled only where a row's maximum has grown by more than 2^8 since the last time: weights of up to 256 are as exact
// as those of up to 1, and nearly every tile leaves the outputs where they are (f16: of up to 2^15, the largest of 2^7 at least: attn_paged.cuh).
//   Split: the key tiles of all items, in a row, in equal runs, one per CTA, their ends moved to an item's edge where one is near (us: four
// prompts of 2000 177 -> 172, one of 2000 64.3 -> 63.6; 500 tokens after 8192 83.5 -> 84.3, 64 after 8192 32.1 -> 33.3).  An item cut by a run's end leaves (m, l, o) of its parts in
// scratch, and join_kernel adds them up, many CTAs to an item (the last CTA to arrive alone took 90 us for 17 parts).
//   Bound by the softmax warps (an exponential per pair, scores and weights through tensor memory) beside the MMAs.  32 heads of 128, 8 of keys, bf16:
// one prompt of 8000 530 us, 990 TFLOP/s; 2048 tokens after 8192 311 us, 994 TFLOP/s; four prompts of 2000 172 us, 761 TFLOP/s (short items).  All times:
// inputs that change from call to call (the same ones again and again: 465, 269 and 157).
//   Weights in bf16 leave outputs 2.1e-3 to 2.3e-3 of their norm off from 64 bits, unrounded ones 1.7e-3 (f16 2.8e-4 and 2.1e-4): two pieces of each
// would take half as many products again, and as much packing once more on the softmax warps, which are the bound.
//   Values of the positions behind a request's end are cleared in shared memory (0 x NaN), and a row that is not finite at the end is worked
// out again key by key.  Every mbarrier wait is bounded.
#include <algorithm>
#include <type_traits>

#include "attn_paged.cuh"
#include "pipeline.cuh"

namespace {

using namespace pipe;

constexpr int kKeys = 128, kRows = 128, kItemRows = 2 * kRows;
constexpr int kPanel = 128 * 128;  // bytes of 128 rows of 64 elements
constexpr int kThreads = 384;
constexpr uint32_t kOutCol = 256;  // tensor memory: scores of both tiles, then their outputs
constexpr float kGrowth = 8.0f;
constexpr int kItemCost = 2;    // units of a run that an item takes beside its tiles: its queries' and outputs' way, 5500 clocks where a tile takes 3100
constexpr int kTilesLeast = 6;  // units of a run
constexpr int kSnap = 1, kSnapShare = 32;  // units, or a share of a run, that a run's end may move to an item's edge (up to 4 units: 500 after 8192 85 -> 88 us)

struct alignas(64) Maps { CUtensorMap q, k, v, o; };

// A cut item, left by the CTA in which it begins for the CTAs that join it.
struct Cut { uint32_t last, token, tokens, g; };  // the CTA in which it ends (0: nothing was cut), its tokens' rows of the step, the key head
struct TcPlan {
  float* parts;  // [CTAs][2]: the part that ends the item a CTA begins with, the part that begins the one it ends with; [columns / 4][256 rows][4], maxima, sums
  Cut* cuts;     // [CTAs], or NULL: items stay whole
  uint32_t rows_over, box_rows, part_floats;
  uint32_t tile_tokens;  // tokens of a row tile
  uint32_t whole;        // no item is long enough to be cut
  uint32_t boxed;        // 32 rows of a tile are a box of the output's map
};

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"((uint64_t)map), "r"(x), "r"(y),
               "r"(z), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"((uint64_t)map), "r"(x), "r"(y),
               "r"(smem_u32(bar))
               : "memory");
}
// 32 columns of this thread's lane; the registers may be used once tmem_ld32_end has returned.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32_end(uint32_t (&r)[32]) {  // nothing that uses them can be placed ahead of it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld32_start(taddr, r);
  tmem_ld32_end(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// An operand whose rows are the sum's index (values [key][element]): panels of 64 elements kPanel apart, eight keys 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(kPanel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Two f32 operations in one instruction.
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
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

// A part of an item: what every role of the CTA walks through in the same order.
struct Piece {
  Segment s;                 // row0: the item's first row; tiles of keys [tile0, tile1)
  unsigned long long item_u;
  uint32_t tiles, last;      // of the whole item; the CTA that has its end, where that is cut off here
  uint32_t token, tokens;    // of the request
  uint32_t n[2], n_all;      // how many tiles from tile0 on each row tile sees
  bool cut_begin, cut_end;
};
struct Walk {
  unsigned long long u, base;  // the next unit; the first unit of the requests' row block b
  uint32_t r, b;
  bool begun;
};

// Runs of `per` units, whose boundaries move to an item's edge where that is within `snap` units: a part costs as much as a few tiles.
struct Runs {
  unsigned long long u1, per, snap;
  uint32_t rep, rows_over, tokens;  // tokens of an item
  __device__ __forceinline__ uint32_t tiles(const PagedAttn& a, const PagedRequest& q, uint32_t b, uint32_t& skip) const {
    skip = paged_low(q.cached + b * tokens, a.window) / kKeys;
    return (q.cached + min((b + 1) * tokens, q.fresh) - 1) / kKeys + 1 - skip;
  }
  // Where a boundary at u of runs lies that falls on an item's units, slot .. stop - 1.
  __device__ __forceinline__ unsigned long long edge(unsigned long long u, unsigned long long slot, unsigned long long stop) const {
    return u - slot <= kItemCost + snap ? slot : stop - u <= snap ? stop : u;
  }
  __device__ unsigned long long units(const PagedAttn& a, const PagedRequest& q) const {
    if (q.fresh * rep <= rows_over) return 0;
    unsigned long long n = 0;
    uint32_t skip;
    for (uint32_t b = 0; b * tokens < q.fresh; ++b) n += tiles(a, q, b, skip) + kItemCost;
    return n * a.pool.KV;
  }
  __device__ bool next(const PagedAttn& a, const TcPlan& plan, Walk& w, Piece& p) const {
    while (w.u < u1) {
      PagedRequest q;
      paged_request(a, w.r, q);
      if (q.fresh * rep <= rows_over || w.b * tokens >= q.fresh) { ++w.r; w.b = 0; continue; }
      uint32_t skip;
      const uint32_t n = tiles(a, q, w.b, skip);
      const unsigned long long all = (unsigned long long)(n + kItemCost) * a.pool.KV;
      if (w.u >= w.base + all) { w.base += all; ++w.b; continue; }
      const uint32_t g = (uint32_t)(w.u - w.base) / (n + kItemCost);  // fewer than 2^32 units in a block of rows: keys / 128 x key heads
      const unsigned long long slot = w.base + (unsigned long long)g * (n + kItemCost), stop = slot + kItemCost + n;
      p.item_u = slot + kItemCost;
      if (!w.begun) {  // where the run's own beginning lies
        w.begun = true;
        w.u = edge(w.u, slot, stop);
        if (w.u >= stop) continue;
      }
      const unsigned long long from = max(w.u, p.item_u), to = u1 >= stop ? stop : edge(u1, slot, stop);
      if (to <= from) return false;  // the rest is the next CTA's
      p.tiles = n;
      p.s.rq = q; p.s.r = w.r; p.s.g = g;
      p.token = w.b * tokens;
      p.tokens = min(tokens, q.fresh - p.token);
      p.s.row0 = p.token * rep;
      p.s.rows = p.tokens * rep;
      p.s.tile0 = skip + (uint32_t)(from - p.item_u);
      p.s.tile1 = skip + (uint32_t)(to - p.item_u);
      p.cut_begin = from != p.item_u;
      p.cut_end = to != stop;
      if (p.cut_end) {  // the CTA that has the item's end: the last boundary inside it that is not moved to its end
        const unsigned long long k = (stop - 1) / per, moved = (stop - snap + per - 1) / per;  // boundaries before the end; the first within `snap` of it
        p.last = (uint32_t)(min(k + 1, moved) - 1);
      }
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t) {
        p.n[t] = 0;
        if (p.tokens > t * plan.tile_tokens) {
          const uint32_t last = (q.cached + p.token + min(p.tokens, (t + 1) * plan.tile_tokens) - 1) / kKeys + 1, stop = min(p.s.tile1, last);
          p.n[t] = stop > p.s.tile0 ? stop - p.s.tile0 : 0u;
        }
      }
      p.n_all = max(p.n[0], p.n[1]);
      w.u = to;
      return true;
    }
    return false;
  }
};

constexpr int kPieces = 3;  // pieces that the scheduling warp is ahead
constexpr int kSoftWarps = 8, kControlWarps = 4;
constexpr int kStage = 32 * 128;  // bytes in which a softmax warp leaves 32 rows of 64 columns for their copy to the output

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const PagedAttn a, const TcPlan plan, const __grid_constant__ Maps maps) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t piece_full[kPieces], piece_empty[kPieces], q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2][2], o_full[2], v_last, v_cleared, fin;
  __shared__ Piece s_piece[kPieces];
  __shared__ uint32_t s_tmem, s_r;
  __shared__ volatile int s_abort;
  __shared__ unsigned long long s_part[kThreads / 32], s_base;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = a.pool.hd, panels = (hd + 63) / 64, plog = a.pool.page_log2;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t q_tile = panels * kPanel, slot_bytes = panels * kPanel;
  const uint32_t sq = smem_u32(smem), sk = sq + 2 * q_tile, sv = sk + 2 * slot_bytes;

  if (tid == 0) {
    mbar_init(&q_full, 1); mbar_init(&q_empty, 1); mbar_init(&v_last, 1); mbar_init(&v_cleared, 1); mbar_init(&fin, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_ready[i][0], 4); mbar_init(&p_ready[i][1], 4); mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kPieces; ++i) { mbar_init(&piece_full[i], 1); mbar_init(&piece_empty[i], kSoftWarps + 2); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(&s_tmem, 512);
  if (warp == 0 && lane < 4) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)(&maps.q + lane)) : "memory");
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- this CTA's run of units (a unit: a tile of keys of an item)
  Runs runs = {0, 0, 0, a.H / a.pool.KV, plan.rows_over, 2 * plan.tile_tokens};
  Walk walk = {0, 0, 0, 0, false};
  {
    const uint32_t each = (a.R + kThreads - 1) / kThreads, ra = min(tid * each, a.R), rb = min(ra + each, a.R);
    unsigned long long mine = 0;
    for (uint32_t r = ra; r < rb; ++r) {
      PagedRequest q;
      paged_request(a, r, q);
      mine += runs.units(a, q);
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
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += s_part[w];
      total += s_part[w];
    }
    runs.per = max((total + gridDim.x - 1) / gridDim.x, (unsigned long long)kTilesLeast);
    runs.snap = !plan.cuts ? 1ull << 40 : plan.whole ? kSnap : max((unsigned long long)kSnap, runs.per / kSnapShare);  // without scratch for parts: every item whole
    walk.u = runs.per * blockIdx.x;
    runs.u1 = min(walk.u + runs.per, total);
    if (walk.u < runs.u1 && before <= walk.u && walk.u < before + mine) {
      unsigned long long base = before;
      for (uint32_t r = ra; r < rb; ++r) {
        PagedRequest q;
        paged_request(a, r, q);
        const unsigned long long n = runs.units(a, q);
        if (walk.u < base + n) { s_r = r; s_base = base; break; }
        base += n;
      }
    }
    __syncthreads();
    walk.r = s_r;
    walk.base = s_base;
  }

  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // the same answer for the whole warp
    if (ok) ok = __all_sync(0xFFFFFFFFu, !s_abort && mbar_wait(bar, parity));
    if (!ok) s_abort = 1;
    return ok;
  };
  uint32_t pieces = 0;
  auto next = [&](Piece& p) {  // the next piece that the scheduling warp has found; false behind the last one
    const uint32_t slot = pieces % kPieces;
    if (!wait(&piece_full[slot], (pieces / kPieces) & 1u)) return false;
    p = s_piece[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&piece_empty[slot]);
    ++pieces;
    return p.tiles != 0;
  };

  // registers: the launch's 384 x 168 hold 128 x 72 and 256 x 216
  if (warp < (uint32_t)kControlWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ===== an item's queries, then its keys and values, a lane per box; rows behind the item's tokens hold whatever follows there
      const uint32_t boxes = kKeys / plan.box_rows, box = lane % boxes, panel = lane / boxes;
      const uint32_t dst = panel * kPanel + box * plan.box_rows * 128;
      uint32_t kt = 0, vt = 0, items = 0, lasts = 0;  // asked for
      Piece p;
      while (ok && next(p)) {
        if (!p.n_all) continue;
        if (items && !wait(&q_empty, (items - 1) & 1u)) break;
        {
          const uint32_t tiles = p.tokens > plan.tile_tokens ? 2u : 1u, t = lane / panels, pn = lane % panels;
          if (lane == 0) mbar_expect_tx(&q_full, tiles * panels * plan.tile_tokens * runs.rep * 128);
          __syncwarp();
          if (t < tiles) tma_3d(sq + t * q_tile + pn * kPanel, &maps.q, (int)pn * 64, (int)(p.s.g * runs.rep), (int)(p.s.rq.t0 + p.token + t * plan.tile_tokens), &q_full);
          ++items;
        }
        for (uint32_t j = 0; j < p.n_all; ++j) {
          const uint32_t key = (p.s.tile0 + j) * kKeys + box * plan.box_rows, slot = kt & 1u;
          int32_t pg = -1;
          if (key < p.s.rq.len) pg = paged_page(a, p.s.r, key);
          const uint32_t bytes = __popc(__ballot_sync(0xFFFFFFFFu, lane < boxes && pg >= 0)) * panels * plan.box_rows * 128;
          const int y = pg >= 0 ? (int)((((uint32_t)pg * a.pool.KV + p.s.g) << plog) + (key & ((1u << plog) - 1u))) : 0;
          const bool mine = panel < panels && pg >= 0;
          if (kt >= 2 && !wait(&k_empty[slot], (kt / 2 - 1) & 1u)) break;
          if (lane == 0) mbar_expect_tx(&k_full[slot], bytes);
          __syncwarp();
          if (mine) tma_2d(sk + slot * slot_bytes + dst, &maps.k, (int)panel * 64, y, &k_full[slot]);
          ++kt;
          if (vt >= 2 && !wait(&v_empty[slot], (vt / 2 - 1) & 1u)) break;
          if (lane == 0) mbar_expect_tx(&v_full[slot], bytes);
          __syncwarp();
          if (mine) tma_2d(sv + slot * slot_bytes + dst, &maps.v, (int)panel * 64, y, &v_full[slot]);
          ++vt;
        }
        const uint32_t end = (p.s.tile0 + p.n_all) * kKeys;
        if (ok && end > p.s.rq.len) {  // positions behind the request's end: their values weigh nothing, and must be numbers for that
          if (!wait(&v_last, lasts++ & 1u)) break;  // they have come
          for (uint32_t r = p.s.rq.len - (end - kKeys) + (lane >> 3); r < (uint32_t)kKeys; r += 4)
            for (uint32_t pn = 0; pn < panels; ++pn)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + ((vt - 1) & 1u) * slot_bytes + pn * kPanel + r * 128 + (lane & 7u) * 16), "r"(0) : "memory");
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_cleared);
        }
      }
      if (items) (void)mbar_wait(&q_full, (items - 1) & 1u);
      // leave no copy in flight into shared memory that another CTA may get, whoever gives up
      for (uint32_t i = kt > 2 ? kt - 2 : 0; i < kt; ++i) (void)mbar_wait(&k_full[i & 1u], (i / 2) & 1u);
      for (uint32_t i = vt > 2 ? vt - 2 : 0; i < vt; ++i) (void)mbar_wait(&v_full[i & 1u], (i / 2) & 1u);
    } else if (warp == 1) {
      // ===== MMAs
      constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc_s = (1u << 4) | (kType << 7) | (kType << 10) | ((kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
      const uint32_t vcols = (hd + 15) / 16 * 16;
      const uint32_t idesc_o = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | ((vcols >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
      // One thread for all of it: a warp that votes and elects between the products takes 100 clocks an MMA, the tensor core 64.
      if (elect_one()) {
        const uint64_t qd[2] = {umma_desc_sw128(sq), umma_desc_sw128(sq + q_tile)}, kd[2] = {umma_desc_sw128(sk), umma_desc_sw128(sk + slot_bytes)},
                       vd[2] = {umma_desc_mn128(sv), umma_desc_mn128(sv + slot_bytes)};
        const uint32_t steps = (hd + 15) / 16;
        uint32_t kt = 0, items = 0, pc[2] = {0, 0}, cleared = 0;
        auto wait1 = [&](uint64_t* bar, uint32_t parity) {
          if (ok && !mbar_wait(bar, parity)) { s_abort = 1; ok = false; }
          return ok;
        };
        auto scores = [&](uint32_t t, uint32_t slot) {
          const uint64_t q = qd[t], k = slot ? kd[1] : kd[0];
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e) {
            if (e >= steps) break;
            umma_f16_ss(tmem + t * kKeys, umma_desc_advance(q, (e >> 2) * kPanel + (e & 3u) * 32u), umma_desc_advance(k, (e >> 2) * kPanel + (e & 3u) * 32u), idesc_s, e != 0 ? 1u : 0u);
          }
          umma_commit(&s_full[t]);
        };
        for (; ok; ++pieces) {
          const uint32_t ps = pieces % kPieces;
          if (!wait1(&piece_full[ps], (pieces / kPieces) & 1u)) break;
          const uint32_t n0 = s_piece[ps].n[0], n1 = s_piece[ps].n[1], n = max(n0, n1), stop = s_piece[ps].tiles == 0;
          const bool tail = (s_piece[ps].s.tile0 + n) * kKeys > s_piece[ps].s.rq.len;
          mbar_arrive(&piece_empty[ps]);
          if (stop) break;
          if (!n) continue;
          if (!wait1(&q_full, items & 1u) || !wait1(&k_full[kt & 1u], (kt / 2) & 1u)) break;
          tc_fence_after_sync();
          if (n0) scores(0, kt & 1u);
          if (n1) scores(1, kt & 1u);
          umma_commit(&k_empty[kt & 1u]);
          if (n == 1) umma_commit(&q_empty);
          for (uint32_t j = 0; j < n; ++j, ++kt) {
            const uint32_t slot = kt & 1u, nslot = slot ^ 1u;
            if (!wait1(&v_full[slot], (kt / 2) & 1u)) break;
            if (tail && j + 1 == n) {
              mbar_arrive(&v_last);
              if (!wait1(&v_cleared, cleared++ & 1u)) break;
            }
            bool have_k = false;
#pragma unroll
            for (uint32_t t = 0; t < 2; ++t) {
              const uint32_t nt = t ? n1 : n0;
              if (ok && j < nt) {
                const uint64_t v = slot ? vd[1] : vd[0];
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {  // the first half of the weights is there while the softmax is at the other one
                  if (!wait1(&p_ready[t][h], pc[t] & 1u)) break;
                  tc_fence_after_sync();
#pragma unroll
                  for (uint32_t e = 4 * h; e < 4 * h + 4; ++e)
                    umma_f16_ts(tmem + kOutCol + t * 128, tmem + t * kKeys + e * 8, umma_desc_advance(v, e * 2048u), idesc_o, (j | e) != 0 ? 1u : 0u);
                  if (h == 1 && j + 1 == nt) umma_commit(&o_full[t]);
                }
                ++pc[t];
              }
              if (ok && j + 1 < nt) {
                if (!have_k) {
                  if (!wait1(&k_full[nslot], ((kt + 1) / 2) & 1u)) break;
                  tc_fence_after_sync();
                  have_k = true;
                }
                scores(t, nslot);
              }
            }
            if (!ok) break;
            if (j + 1 < n) umma_commit(&k_empty[nslot]);
            if (j + 2 == n) umma_commit(&q_empty);
            umma_commit(&v_empty[slot]);
          }
          ++items;
        }
        umma_commit(&fin);  // nothing is left running when tensor memory is freed
        if (!mbar_wait(&fin, 0)) s_abort = 1;
      }
      __syncwarp();
    } else if (warp == 2) {
      // ===== the run's pieces, and what is cut
      if (lane == 0) {
        Cut cut = {0, 0, 0, 0};
        bool more = true;
        for (uint32_t i = 0; more; ++i) {
          Piece p;
          p.tiles = 0;
          more = runs.next(a, plan, walk, p);
          if (more && p.cut_end && !p.cut_begin) cut = {p.last, p.s.rq.t0 + p.token, p.tokens, p.s.g};
          if (i >= kPieces && (s_abort || !mbar_wait(&piece_empty[i % kPieces], (i / kPieces - 1) & 1u))) { s_abort = 1; break; }
          s_piece[i % kPieces] = p;
          mbar_arrive(&piece_full[i % kPieces]);
        }
        if (plan.cuts) plan.cuts[blockIdx.x] = cut;
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ===== softmax: thread = row
    const uint32_t t = (warp - kControlWarps) >> 2, quarter = warp & 3u, rep = runs.rep, row = quarter * 32 + lane, mine = row / rep;
    const uint32_t lanes = (quarter * 32u) << 16, s_at = tmem + lanes + t * kKeys, o_at = tmem + lanes + kOutCol + t * 128;
    unsigned char* stage = smem + 2 * q_tile + 4 * slot_bytes + (warp - kControlWarps) * kStage;
    const uint32_t box_head = quarter * 32 % rep, box_token = t * plan.tile_tokens + quarter * 32 / rep;
    const float c = a.scale * kLog2e;
    const unsigned long long c2 = pair_of(c, c);
    uint32_t sc = 0, oc = 0;
    for (;; ++pieces) {
      // the piece stays where it is until the rows are done: its numbers are read when they are needed
      const uint32_t slot = pieces % kPieces;
      if (!wait(&piece_full[slot], (pieces / kPieces) & 1u)) break;
      const Piece& p = s_piece[slot];
      if (p.tiles == 0) break;
      const uint32_t n = t ? p.n[1] : p.n[0], token = t * plan.tile_tokens + mine;  // of the item
      const bool live = mine < plan.tile_tokens && token < p.tokens;
      const uint32_t pos = p.s.rq.cached + p.token + min(token, p.tokens - 1), low = paged_low(pos, a.window);
      float m = -INFINITY, l = 0.0f;
      for (uint32_t j = 0; j < n; ++j, ++sc) {
        if (!wait(&s_full[t], sc & 1u)) break;
        tc_fence_after_sync();
        const uint32_t key0 = (p.s.tile0 + j) * kKeys;
        const uint32_t hi = pos + 1 > key0 ? pos + 1 - key0 : 0u, lo = low > key0 ? low - key0 : 0u;  // keys key0 + lo .. key0 + hi - 1 are seen
        // which of the 32 keys from i on: all of them for nearly every tile
        auto seen = [&](uint32_t i) {
          const uint32_t up = hi <= i ? 0u : hi - i >= 32 ? 0xFFFFFFFFu : (1u << (hi - i)) - 1u;
          return lo <= i ? up : lo - i >= 32 ? 0u : up & ~((1u << (lo - i)) - 1u);
        };
        float s[kKeys];
        {
          uint32_t r[4][32];
#pragma unroll
          for (int x = 0; x < 4; ++x) tmem_ld32_start(s_at + 32 * x, r[x]);
#pragma unroll
          for (int x = 0; x < 4; ++x) tmem_ld32_end(r[x]);
#pragma unroll
          for (int y = 0; y < kKeys; ++y) s[y] = __uint_as_float(r[y / 32][y % 32]);
        }
        if (!__all_sync(0xFFFFFFFFu, lo == 0 && hi >= (uint32_t)kKeys)) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t bits = seen(32 * x);
            if (!__all_sync(0xFFFFFFFFu, bits == 0xFFFFFFFFu)) {
#pragma unroll
              for (int y = 0; y < 32; ++y) s[32 * x + y] = (bits >> y) & 1u ? s[32 * x + y] : -INFINITY;
            }
          }
        }
        float top[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) top[y] = fmaxf(s[y], s[y + 4]);
#pragma unroll
        for (int y = 8; y < kKeys; y += 8) {
#pragma unroll
          for (int z = 0; z < 4; ++z) top[z] = max3(top[z], s[y + z], s[y + z + 4]);
        }
        float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        mx = fmaf(mx, c, -weights_up<T>(7.0f));  // c > 0
        if (__any_sync(0xFFFFFFFFu, mx > m + kGrowth)) {
          const float m_new = fmaxf(m, mx), f = m == -INFINITY ? 0.0f : exp2_of(m - m_new);
          m = m_new;
          l *= f;
          if (j > 0) {  // the products before have finished: this tile's scores came after them
#pragma unroll 1
            for (uint32_t i = 0; i < hd; i += 32) {
              float o[32];
              tmem_ld32(o_at + i, o);
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] *= f;
              tmem_st32(o_at + i, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : -m;
        const unsigned long long base2 = pair_of(base, base);
        unsigned long long add0 = 0, add1 = 0;
#pragma unroll
        for (int i = 0; i < kKeys; i += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int y = 0; y < 32; y += 2) {
            const unsigned long long v = fma2(pair_of(s[i + y], s[i + y + 1]), c2, base2);
            const float e0 = exp2_of(__uint_as_float((uint32_t)v)), e1 = exp2_of(__uint_as_float((uint32_t)(v >> 32)));
            if (y & 2) add1 = add2(add1, pair_of(e0, e1));
            else add0 = add2(add0, pair_of(e0, e1));
            pk[y / 2] = pack2<T>(e0, e1);
          }
          tmem_st16(s_at + i / 2, pk);
          if (i & 32) {  // half of the weights
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[t][i >> 6]);
          }
        }
        add0 = add2(add0, add1);
        l += __uint_as_float((uint32_t)add0) + __uint_as_float((uint32_t)(add0 >> 32));
      }
      if (n) { wait(&o_full[t], oc & 1u); ++oc; tc_fence_after_sync(); }
      if (!ok) break;
      // ---- the rows' results: out, or a part of an item
      const bool cut = p.cut_begin || p.cut_end;
      float* part = plan.parts + ((size_t)blockIdx.x * 2 + (p.cut_begin ? 0 : 1)) * plan.part_floats;
      T* out = static_cast<T*>(a.out) + (size_t)(p.s.rq.t0 + p.token + t * plan.tile_tokens) * a.out_ld + (size_t)(p.s.g * rep) * hd;
      const uint32_t row_end = (p.tokens > t * plan.tile_tokens ? min(p.tokens - t * plan.tile_tokens, plan.tile_tokens) : 0u) * rep;  // of the tile
      const bool boxed = plan.boxed && quarter * 32 + 32 <= row_end;  // a box of the output's map: all of the warp's rows
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      unsigned long long odd[2] = {pair_of(l * 0.0f, 0.0f), 0};  // NaN where anything is not finite
#pragma unroll 1
      for (uint32_t i = 0; i < hd; i += 64) {
        if (!cut) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the staged rows before have been read
          __syncwarp();
        }
#pragma unroll 1
        for (uint32_t x = i; x < i + 64 && x < hd; x += 32) {
          float o[32];
          if (n) tmem_ld32(o_at + x, o);
          else {
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = 0.0f;
          }
          if (x + 32 > hd) {  // columns that no product wrote
#pragma unroll
            for (int y = 0; y < 32; y += 8)
              if (x + y >= hd) {
#pragma unroll
                for (int z = 0; z < 8; ++z) o[y + z] = 0.0f;
              }
          }
#pragma unroll
          for (int y = 0; y < 32; y += 2) odd[(y / 2) & 1] = fma2(pair_of(o[y], o[y + 1]), 0ull, odd[(y / 2) & 1]);
          if (cut) {
#pragma unroll
            for (int y = 0; y < 32; y += 4)
              if (live && x + y < hd) *reinterpret_cast<float4*>(part + ((size_t)((x + y) / 4) * kItemRows + t * kRows + row) * 4) = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
          } else {
#pragma unroll
            for (int y = 0; y < 32; y += 8)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((((x & 32u) / 8 + y / 8) ^ lane) & 7u) * 16) =
                  make_uint4(pack2<T>(o[y] * inv, o[y + 1] * inv), pack2<T>(o[y + 2] * inv, o[y + 3] * inv), pack2<T>(o[y + 4] * inv, o[y + 5] * inv), pack2<T>(o[y + 6] * inv, o[y + 7] * inv));
          }
        }
        if (!cut) {
          if (boxed) fence_proxy_async_smem();
          __syncwarp();
          if (boxed) {
            if (lane == 0) {
              tma_store_3d(&maps.o, smem_u32(stage), (int)i, (int)(p.s.g * rep + box_head), (int)(p.s.rq.t0 + p.token + box_token));
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
#pragma unroll 1
            for (uint32_t x = 0; x < 32; x += 4) {  // four rows of 128 bytes at a time
              const uint32_t rr = x + (lane >> 3), at = quarter * 32 + rr, col = i + (lane & 7u) * 8;
              const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((lane ^ rr) & 7u) * 16);
              if (at < row_end && col < hd) *reinterpret_cast<uint4*>(out + (size_t)(at / rep) * a.out_ld + (size_t)(at % rep) * hd + col) = v;
            }
            __syncwarp();
          }
        }
      }
      // rows that are not finite, key by key
      odd[0] = add2(odd[0], odd[1]);
      const bool fine = __uint_as_float((uint32_t)odd[0]) + __uint_as_float((uint32_t)(odd[0] >> 32)) == 0.0f;
      uint32_t bad = __ballot_sync(0xFFFFFFFFu, live && !fine);
      if (bad) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // what they replace has been written
        __syncwarp();
      }
      for (; bad; bad &= bad - 1) {
        const uint32_t who = (uint32_t)__ffs((int)bad) - 1, which = quarter * 32 + who;
        float* tmp = reinterpret_cast<float*>(stage);
        float m2, l2;
        row_again<T>(a, p.s, rep, p.s.row0 + t * plan.tile_tokens * rep + which, p.s.tile0 * kKeys, p.s.tile1 * kKeys, tmp, m2, l2);
        __syncwarp();
        for (uint32_t e = lane; e < hd; e += 32) {
          if (cut) part[((size_t)(e / 4) * kItemRows + t * kRows + which) * 4 + (e & 3u)] = tmp[e];
          else out[(size_t)(which / rep) * a.out_ld + (size_t)(which % rep) * hd + e] = from_f32<T>(l2 == 0.0f ? 0.0f : tmp[e] / l2);
        }
        __syncwarp();
        if (lane == who) { m = m2; l = l2; }
      }
      if (cut && live) {
        part[hd * kItemRows + t * kRows + row] = m;
        part[(hd + 1) * kItemRows + t * kRows + row] = l;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[slot]);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  if (s_abort && tid == 0 && a.status) atomicCAS(a.status, 0, 3);
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// grid (CTAs of chunk_kernel, groups of 32 rows): the parts of an item, in their order.
constexpr int kJoinThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const PagedAttn a, const TcPlan plan) {
  grid_dependency_wait();
  grid_launch_dependents();
  const Cut cut = plan.cuts[blockIdx.x];
  if (!cut.last) return;
  const uint32_t hd = a.pool.hd, rep = a.H / a.pool.KV, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y * 32 + lane;
  const uint32_t tile = row / kRows, mine = row % kRows / rep, token = tile * plan.tile_tokens + mine;
  if (mine >= plan.tile_tokens || token >= cut.tokens) return;
  auto part_of = [&](uint32_t i) { return plan.parts + ((size_t)i * 2 + (i == blockIdx.x ? 1 : 0)) * plan.part_floats; };
  constexpr int kAhead = 4;  // parts whose loads are under way together
  T* dst = static_cast<T*>(a.out) + (size_t)(cut.token + token) * a.out_ld + (size_t)(cut.g * rep + row % kRows % rep) * hd;
  for (uint32_t e = 4 * warp; e < hd; e += kJoinThreads / 8) {
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i0 = blockIdx.x; i0 <= cut.last; i0 += kAhead) {
      float mp[kAhead], lp[kAhead], top = m;
      float4 v[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        mp[x] = -INFINITY; lp[x] = 0.0f; v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i0 + x > cut.last) continue;
        const float* part = part_of(i0 + x);
        mp[x] = part[hd * kItemRows + row];
        lp[x] = part[(hd + 1) * kItemRows + row];
        v[x] = *reinterpret_cast<const float4*>(part + ((size_t)(e / 4) * kItemRows + row) * 4);
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) top = fmaxf(top, mp[x]);
      const float corr = m == -INFINITY ? 0.0f : exp2_of(m - top);
      l *= corr;
#pragma unroll
      for (int y = 0; y < 4; ++y) o[y] *= corr;
      m = top;
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const float f = mp[x] == -INFINITY ? 0.0f : exp2_of(mp[x] - m);  // a part whose every score is NaN has no maximum; its sums are NaN
        l = fmaf(lp[x], f, l);
        o[0] = fmaf(v[x].x, f, o[0]); o[1] = fmaf(v[x].y, f, o[1]); o[2] = fmaf(v[x].z, f, o[2]); o[3] = fmaf(v[x].w, f, o[3]);
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2*>(dst + e) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  }
}

// Queries or outputs [tokens][heads][hd], in boxes of 64 elements, some heads and some tokens; what lies outside reads as zero and is not written.
CUresult encode_rows(ruai_tensor_map_encode fn, CUtensorMap* map, const PagedAttn& a, void* base, uint32_t ld, uint32_t heads, uint32_t tokens) {
  const cuuint64_t dims[3] = {a.pool.hd, a.H, a.tokens}, strides[2] = {(cuuint64_t)a.pool.hd * 2, (cuuint64_t)ld * 2};
  const cuuint32_t box[3] = {64, heads, tokens}, one[3] = {1, 1, 1};
  return fn(map, a.pool.dtype == RUAI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}
// A pool's rows (page, key head, position in the page) of hd elements, in boxes of box_rows x 64; elements past hd read as zero.
CUresult encode(ruai_tensor_map_encode fn, CUtensorMap* map, const PagedPool& p, void* base, uint32_t box_rows) {
  const cuuint64_t dims[2] = {p.hd, ((cuuint64_t)p.pages * p.KV) << p.page_log2}, strides[1] = {(cuuint64_t)p.hd * 2};
  const cuuint32_t box[2] = {64, box_rows}, one[2] = {1, 1};
  return fn(map, p.dtype == RUAI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <typename T>
cudaError_t launch_chunk(ruai_ctx* c, const PagedAttn& a, const TcPlan& plan, const Maps& maps) {
  const uint32_t panels = (a.pool.hd + 63) / 64;
  const int extra = kSoftWarps * kStage + 1024, smem = 6 * (int)panels * kPanel + extra, most = 12 * kPanel + extra;
  static bool done[64] = {};
  if (!done[c->ordinal & 63]) {
    cudaError_t e = cudaFuncSetAttribute(chunk_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    done[c->ordinal & 63] = true;
  }
  // one CTA per SM: each takes all of tensor memory
  const cudaError_t e = ruai_launch(c, chunk_kernel<T>, dim3(c->sm_count), dim3(kThreads), (size_t)std::max(smem, 120 * 1024), true, a, plan, maps);
  if (e != cudaSuccess || !plan.cuts || plan.whole) return e;
  return ruai_launch(c, join_kernel<T>, dim3(c->sm_count, kItemRows / 32), dim3(kJoinThreads), 0, true, a, plan);
}

}  // namespace

int ruai_paged_attention_tc(ruai_ctx* c, const PagedAttn& a, uint32_t rows_over) {
  const PagedPool& p = a.pool;
  // heads narrower than a copied box, and scores that shrink with their product, stay on attn_paged.cu
  const uint32_t rep = a.H / p.KV;
  if (!c->use_tc || p.dtype == RUAI_F32 || p.hd < 64 || p.hd > 128 || rep > (uint32_t)kRows || !(a.scale > 0.0f)) return 0;
  const ruai_tensor_map_encode fn = ruai_tensor_map_fn();
  if (!fn) { ruai_fail(c, RUAI_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver"); return -1; }
  TcPlan plan = {};
  plan.rows_over = rows_over;
  plan.box_rows = std::min(1u << p.page_log2, (uint32_t)kKeys);
  plan.part_floats = (p.hd + 2) * kItemRows;
  plan.tile_tokens = kRows / rep;
  Maps maps;
  plan.boxed = 32 % rep == 0 || rep % 32 == 0;
  const uint32_t heads = std::min(rep, 32u);
  const CUresult rq = encode_rows(fn, &maps.q, a, const_cast<void*>(a.q), a.q_ld, rep, plan.tile_tokens), ro = encode_rows(fn, &maps.o, a, a.out, a.out_ld, heads, 32 / heads), rk = encode(fn, &maps.k, p, p.k, plan.box_rows), rv = encode(fn, &maps.v, p, p.v, plan.box_rows);
  if (rq != CUDA_SUCCESS || ro != CUDA_SUCCESS || rk != CUDA_SUCCESS || rv != CUDA_SUCCESS) {
    ruai_fail(c, RUAI_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d, %d, %d, %d) for %u pages of %u heads of %u", (int)rq, (int)ro, (int)rk, (int)rv, p.pages, p.KV, p.hd);
    return -1;
  }
  // parts of cut items: two per CTA.  Nothing may be allocated while the stream is captured; items then stay whole
  const size_t parts = 2 * (size_t)c->sm_count * plan.part_floats * sizeof(float), need = parts + c->sm_count * sizeof(Cut);
  bool cuts = true;
  if (need > c->partial_bytes) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(c->stream, &capture) != cudaSuccess || capture != cudaStreamCaptureStatusNone) cuts = false;
    else cuts = ruai_ctx_reserve(c, need, 0) == RUAI_OK;  // no memory for the parts: the scratch as it was
  }
  plan.parts = c->partial;
  // items of so few tiles are never cut, whatever the runs are (one end or the other is within kSnap): nothing to join
  plan.whole = (a.most_len + kKeys - 1) / kKeys <= 2 * kSnap + 1;
  plan.cuts = cuts ? reinterpret_cast<Cut*>(reinterpret_cast<unsigned char*>(c->partial) + parts) : nullptr;
  const cudaError_t e = p.dtype == RUAI_F16 ? launch_chunk<__half>(c, a, plan, maps) : launch_chunk<__nv_bfloat16>(c, a, plan, maps);
  if (e != cudaSuccess) { ruai_fail(c, RUAI_ERR_CUDA, "attention over pages: %s", cudaGetErrorString(e)); return -1; }
  return 1;
}
