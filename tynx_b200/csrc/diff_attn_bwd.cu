// Differential attention backward on tcgen05: one launch, three kinds of blocks.
//
// Every block keeps 128 rows in shared memory and streams the other side in
// steps of 64 rows.  K blocks (rows: keys) and V blocks (rows: keys) run over
// the queries of every head that shares them and sum dK and dV; Q blocks (rows:
// queries) run over the keys and sum dQ.  With R the resident side, X the
// streamed one, per step
//   S_m = R_m X_m^T                  (128 x 64 each, three fp16 products)
//   A_m = 2^(S_m - lse_m)
//   K, Q: dP = R_v X_v^T, ds_m = A_m (dP - D_m), acc_m += ds_m X_m
//   V:    w = A_1 - lam A_2,         acc += w dO
// ds and w go back over S in TMEM as pairs of fp16, scaled by powers of two:
// |w| <= 1 + |lam|, and |dP - D| <= 2 max |dO_i| max |V_j| (2-norms of rows, found
// by the split), so nothing overflows and the largest stay near 2^13.  The
// steps' products are added in registers (the tensor core's own addition
// truncates); they carry the step's factors: f of X's tile, the scale of ds or w,
// -lam of the head for map 2.
// Scores are computed three times over.  In return there are no atomic additions
// and no partial results, so sums have one order; TMEM holds two steps' S, so that
// a step's S and sums run under the elementwise part (a block that summed dK and
// dV together would have room for one); and the three kinds' blocks, longest
// first, fill the SMs together.
// An instruction of 128 rows takes 64 cycles whether it makes 64 or 128 columns.
// So dP multiplies R_hi with X_hi and X_lo side by side (their halves are added
// elementwise): a step takes 24 instructions for S, 16 for dP and 24 for the sums
// in K and Q blocks, 4096 cycles, and 24 + 12 in V blocks, 2304.  2 x 2048 causal
// tokens of 8 heads over 4 take 252 us (with dP as three products 260; with a
// step's S alone in TMEM 421): these instructions are 309 of the 427 thousand
// cycles an SM is busy, and where a step's elementwise chain (about 500
// instructions a warp, four warps a scheduler) is behind, the tensor core waits.
// 256 sequences of 128 tokens of 2 heads, where a block has two steps and its
// start and stores count as much, take 142 us; so the first scores wait for what
// they need alone (with all resident tiles 145 us).
#include "diff_attn.cuh"

namespace tx_diff {
namespace {

constexpr int kThreads = 640, kStep = 64;  // producer, MMA, two spare warps, 16 elementwise warps
enum { kModeK = 0, kModeQ = 1, kModeV = 2 };

// PACK: rows of queries are those of a group's heads in turn (Shape::P = G)
template <int DV, bool PACK>
struct Cfg {
  static constexpr int RQ = 2 * 128 * 64 * 2;  // one map's resident tile, heads and tails
  static constexpr int RV = 2 * 128 * DV * 2;
  static constexpr int XBLK = kStep * 64 * 2;  // [64 rows x 64] fp16
  static constexpr int XQ = 2 * XBLK;          // one map's step
  static constexpr int XV = 2 * (DV / 64) * XBLK;
  static constexpr int STATS = PACK ? 5 : 4;   // lse1, lse2, D1, D2 of 64 queries, and lam / 2^E
  static constexpr int STAT = STATS * kStep * 4;
  // resident | two steps of both maps | V's or dO's step (V blocks: two, no resident value tile)
  static constexpr int TILES = 2 * RQ + RV + 2 * (2 * XQ) + XV;
  static constexpr int SMEM = TILES + 2 * STAT + 512;
  static_assert(SMEM <= 232448, "shared memory of an SM");
  static_assert(XV <= RV, "a V block's second dO step takes the resident value tile's place");
};

struct Grads {
  const float *stats, *sums;  // [b][h][steps of queries][4 or 5][64], [b][h][qt][P]
  float *dq, *dk, *dv, *dlam;
  // blocks of one tile level: K, Q and V; in turn level by level, or kind after kind
  unsigned nk, nq, levels, by_level, kt, qt;
  int each_head;  // K and V blocks of one query head each, dk and dv for every query head
};
// the block's kind and its index within it
__device__ __forceinline__ int block_kind(const Grads &o, unsigned i, unsigned &block) {
  if (o.by_level) {
    const unsigned per = 2 * o.nk + o.nq;
    unsigned level = i / per, at = i - level * per;
    if (level >= o.levels) {  // the side with more tiles goes on alone
      const unsigned rest = i - o.levels * per, each = o.kt > o.levels ? 2 * o.nk : o.nq;
      level = o.levels + rest / each;
      at = rest % each + (o.kt > o.levels ? 0 : o.nk);
      if (o.kt > o.levels && at >= o.nk) at += o.nq;
    }
    const int kind = at < o.nk ? kModeK : at < o.nk + o.nq ? kModeQ : kModeV;
    const unsigned before = kind == kModeK ? 0 : kind == kModeQ ? o.nk : o.nk + o.nq;
    block = level * (kind == kModeQ ? o.nq : o.nk) + (at - before);
    return kind;
  }
  const unsigned k = o.nk * o.kt, q = o.nq * o.qt;
  block = i < k ? i : i < k + q ? i - k : i - k - q;
  return i < k ? kModeK : i < k + q ? kModeQ : kModeV;
}

template <int DV, int MODE, bool PACK>
__device__ __forceinline__ void body(const Shape &s, const Split &x, const CUtensorMap &mq, const CUtensorMap &mk,
                                     const CUtensorMap &mv, const CUtensorMap &mg, const Grads &o, uint8_t *sm,
                                     unsigned block) {
  using C = Cfg<DV, PACK>;
  constexpr bool KEYS = MODE != kModeQ;  // the rows are keys
  const int P = PACK ? s.P : 1, Hq = PACK ? s.row_heads() : s.H;
  // TMEM: two steps' S_1 and S_2 (64 columns each), dP in two halves, acc_1 and acc_2 (64 each) or acc
  constexpr uint32_t kDp = 256, ACC = 384;
  const uint32_t srq = su32(sm), sx = srq + 2 * C::RQ;
  const uint32_t srv = sx, sxq = sx + C::RV, sxv = sxq + 4 * C::XQ;
  // where block p of [heads | tails] goes
  auto xv_block = [](int p) { return DV == 64 ? p : (p & 1) * 2 + (p >> 1); };
  auto xv_at = [&](int i) { return MODE == kModeV && (i & 1) ? srv : sxv; };
  const float *stat = reinterpret_cast<const float *>(sm + C::TILES);
  uint64_t *bars = reinterpret_cast<uint64_t *>(sm + C::TILES + 2 * C::STAT);
  uint64_t *r_full = bars, *x_full = bars + 1, *x_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 6,
           *s_full = bars + 7, *p_full = bars + 9, *a_full = bars + 11, *all_done = bars + 12, *rv_full = bars + 13;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 16);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
  uint32_t *vmax = tmem_holder + 2;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  // keys: the first tiles are seen by most queries; queries: the last tiles see most keys
  const bool each = KEYS && !PACK && o.each_head;
  const int heads = KEYS && !each ? s.Hk : Hq;
  const int rheads = (int)s.B * heads, rtiles = (int)(KEYS ? x.kt : x.qt), T = (int)s.T * P;  // T: rows of queries
  const int level = block / rheads, bh = block - level * rheads, b = bh / heads;
  const int rt = KEYS ? level : rtiles - 1 - level, rh = bh - b * heads, hk = PACK || (KEYS && !each) ? rh : rh / s.G;
  const int r0 = rt * 128, n = (int)s.length(b), q_steps = (T + kStep - 1) / kStep;
  int first = 0, per_head;  // steps of each head, keys: from step `first` on
  if (KEYS) {
    int64_t q_first = s.causal ? r0 - s.start : 0;  // the first query that sees the first key
    if (q_first < 0) q_first = 0;
    first = q_first < s.T ? (int)q_first * P / kStep : q_steps;
    per_head = first < q_steps && r0 < n ? q_steps - first : 0;
  } else {
    const int last = r0 + 127 < T ? r0 + 127 : T - 1;
    per_head = ((int)s.seen(PACK ? last / P : last, n) + kStep - 1) / kStep;
  }
  const int steps = __shfl_sync(0xffffffffu, KEYS && !each && !PACK ? per_head * s.G : per_head, 0);

  if (threadIdx.x == 0) {
    bar_init(r_full, 1);
    bar_init(rv_full, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(x_full + i, 1);
      bar_init(x_empty + i, 1);
      bar_init(s_full + i, 1);
      bar_init(p_full + i, 512);
    }
    bar_init(v_full, 1);
    bar_init(v_empty, 1);
    bar_init(a_full, 1);
    bar_init(all_done, 1);
    *abort_flag = 0;
    *vmax = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_holder)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  wait_for_previous();  // the split operands and statistics
  next_may_start();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_holder;

  // step i: head, first streamed row
  auto head_of = [&](int i) { return KEYS && !each && !PACK ? hk * s.G + i / per_head : rh; };
  auto step_of = [&](int i) { return KEYS ? first + i % per_head : i; };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0 && lane == 0 && steps) {
      bar_expect(r_full, 2 * C::RQ);
      for (int p = 0; p < 8; ++p)  // (map, head or tail, 64-row half)
        tma_3d(srq + p * C::XBLK, KEYS ? &mk : &mq, r_full, (p >> 1 & 1) * 64, r0 + (p & 1) * 64,
               (KEYS ? b * 2 * s.Hk + 2 * hk : b * 2 * Hq + 2 * rh) + (p >> 2));
      bool ok = true;
      int lx = 0, lv = 0;
      for (int i = 0; i < steps && ok; ++i) {
        const int st = i & 1, h = head_of(i), step = step_of(i);
        if (i > 1) ok = bar_wait(x_empty + st, ((i >> 1) - 1) & 1, abort_flag, s.err, 11);
        if (!ok) break;
        bar_expect(x_full + st, 2 * C::XQ + (KEYS ? C::STAT : 0) + (MODE == kModeV ? C::XV : 0));
        for (int p = 0; p < 4; ++p)
          tma_3d(sxq + st * 2 * C::XQ + p * C::XBLK, KEYS ? &mq : &mk, x_full + st, (p & 1) * 64, step * kStep,
                 (KEYS ? b * 2 * Hq + 2 * h : b * 2 * s.Hk + 2 * hk) + (p >> 1));
        if (KEYS)
          bulk_load(su32(stat) + st * C::STAT, o.stats + ((int64_t)(b * Hq + h) * q_steps + step) * (C::STATS * kStep), C::STAT,
                    x_full + st);
        if (MODE == kModeV)
          for (int p = 0; p < 2 * (DV / 64); ++p)
            tma_3d(xv_at(i) + xv_block(p) * C::XBLK, &mg, x_full + st, p * 64, step * kStep, b * Hq + h);
        ++lx;
        if (MODE != kModeV) {
          if (i == 0) {  // behind what the first scores need
            bar_expect(rv_full, C::RV);
            for (int p = 0; p < 4 * (DV / 64); ++p)
              tma_3d(srv + p * C::XBLK, KEYS ? &mv : &mg, rv_full, (p >> 1) * 64, r0 + (p & 1) * 64,
                     KEYS ? b * s.Hk + hk : b * Hq + rh);
          }
          if (i) ok = bar_wait(v_empty, (i - 1) & 1, abort_flag, s.err, 12);
          if (!ok) break;
          bar_expect(v_full, C::XV);
          for (int p = 0; p < 2 * (DV / 64); ++p)  // heads and tails of a column block side by side
            tma_3d(sxv + xv_block(p) * C::XBLK, KEYS ? &mg : &mv, v_full, p * 64, step * kStep,
                   KEYS ? b * Hq + h : b * s.Hk + hk);
          ++lv;
        }
      }
      // every copy has landed before the CTA's memory is released
      bar_drain(r_full, 0);
      if (lv) bar_drain(rv_full, 0);
      for (int i = lx - 1; i >= 0 && i > lx - 3; --i) bar_drain(x_full + (i & 1), (i >> 1) & 1);
      if (lv) bar_drain(v_full, (lv - 1) & 1);
    } else if (warp == 1 && steps) {
      const uint32_t one = elect_one();
      constexpr uint32_t id_s = idesc(kStep, false), id_p = idesc(2 * kStep, false), id_a = idesc(64, true), id_v = idesc(DV, true);
      bool ok = mma_wait(r_full, 0, abort_flag, s.err, 13);
      auto scores = [&](int i) {  // S_1 and S_2 of step i
        const int st = i & 1;
        const uint32_t ts = tmem + st * 128;
        ok = ok && mma_wait(x_full + st, (i >> 1) & 1, abort_flag, s.err, 14);
        if (!ok) return;
        fence_after();
        for (int m = 0; m < 2; ++m) {
          const uint32_t rh_ = srq + m * C::RQ, rl = rh_ + C::RQ / 2, xh = sxq + st * 2 * C::XQ + m * C::XQ, xl = xh + C::XBLK;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_ss(ts + m * 64, kdesc(rh_, k), kdesc(xl, k), id_s, k ? 1u : 0u, one);
            mma_ss(ts + m * 64, kdesc(rl, k), kdesc(xh, k), id_s, 1u, one);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ss(ts + m * 64, kdesc(rh_, k), kdesc(xh, k), id_s, 1u, one);
        }
      };
      auto values = [&](int i) {  // dP of step i, in two halves: R_hi X_hi, and the small products (their truncations cost nothing there)
        if (MODE != kModeV && ok) {
          if (i == 0) ok = mma_wait(rv_full, 0, abort_flag, s.err, 13);
          ok = ok && mma_wait(v_full, i & 1, abort_flag, s.err, 15);
          if (!ok) return;
          fence_after();
#pragma unroll
          for (int c = 0; c < DV / 64; ++c) {
            const uint32_t rh_ = srv + c * 16384, rl = rh_ + (DV / 64) * 16384, xh = sxv + c * 2 * C::XBLK;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              mma_ss(tmem + kDp, kdesc(rh_, k), kdesc(xh, k), id_p, (c || k) ? 1u : 0u, one);
              mma_ss(tmem + kDp + 64, kdesc(rl, k), kdesc(xh, k), id_s, 1u, one);
            }
          }
          mma_commit(v_empty, one);
        }
        if (ok) mma_commit(s_full + (i & 1), one);
      };
      scores(0);
      values(0);
      if (steps > 1) scores(1);
      for (int i = 0; i < steps && ok; ++i) {
        const int st = i & 1;
        const uint32_t ts = tmem + st * 128;
        ok = ok && mma_wait(p_full + st, (i >> 1) & 1, abort_flag, s.err, 16);
        if (!ok) break;
        fence_after();
        if (i + 1 < steps) values(i + 1);  // its dP's place is free: the elementwise part has read the last one
        if (!ok) break;
        if (MODE == kModeV) {
          const uint32_t xh = xv_at(i), xl = xh + C::XBLK, ta = tmem + ACC;
          constexpr uint32_t next = 2 * C::XBLK;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_ts(ta, ts + k * 16, ndesc(xl, k, next), id_v, k ? 1u : 0u, one);
            mma_ts(ta, ts + k * 16 + 8, ndesc(xh, k, next), id_v, 1u, one);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ts(ta, ts + k * 16, ndesc(xh, k, next), id_v, 1u, one);
        } else {
          for (int m = 0; m < 2; ++m) {
            const uint32_t xh = sxq + st * 2 * C::XQ + m * C::XQ, xl = xh + C::XBLK, ta = tmem + ACC + m * 64;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              mma_ts(ta, ts + m * 64 + k * 16, ndesc(xl, k, C::XBLK), id_a, k ? 1u : 0u, one);
              mma_ts(ta, ts + m * 64 + k * 16 + 8, ndesc(xh, k, C::XBLK), id_a, 1u, one);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_ts(ta, ts + m * 64 + k * 16, ndesc(xh, k, C::XBLK), id_a, 1u, one);
          }
        }
        mma_commit(x_empty + st, one);
        mma_commit(a_full, one);
        if (i + 2 < steps) scores(i + 2);
      }
      mma_commit(all_done, one);
      bar_drain(all_done, 0);
    } else if (warp == 2 && o.dlam) {
      for (int h = blockIdx.x; h < s.H; h += gridDim.x) sum_dlam(s, o.sums, x.qt, o.dlam, h);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // warpgroup `part` takes streamed rows 16 part .. of every step, and of the results half of map
    // part / 2's columns (K, Q) or a quarter of the columns (V)
    const int part = (warp - 4) >> 2, half = part >> 1, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_row = (uint32_t)(quad * 32) << 16;
    const int row = r0 + r;
    constexpr int AC = MODE == kModeV ? DV / 4 : 32;  // columns of the result a thread sums
    uint64_t acc[AC / 2];
#pragma unroll
    for (int j = 0; j < AC / 2; ++j) acc[j] = two(0.f, 0.f);
    if (MODE != kModeV) {
      // the largest row norm of this head's values (all tiles: D runs over all keys)
      for (int64_t i = threadIdx.x - 128; i < x.kt; i += 512)
        atomicMax(vmax, __float_as_uint(x.nv[(int64_t)(b * s.Hk + hk) * x.kt + i]));
      asm volatile("bar.sync 1, 512;" ::: "memory");
    }
    const float vn = __uint_as_float(*vmax);
    // resident factors: of both maps, and of V (keys) or dO (queries)
    const int64_t rq = (int64_t)(KEYS ? b * 2 * s.Hk + 2 * hk : b * 2 * Hq + 2 * rh) * rtiles + rt;
    const float fr0 = (KEYS ? x.fk : x.fq)[rq], fr1 = (KEYS ? x.fk : x.fq)[rq + rtiles];
    const float frv = (KEYS ? x.fv : x.fg)[(int64_t)(KEYS ? b * s.Hk + hk : b * Hq + rh) * rtiles + rt];
    float mine[4] = {INFINITY, INFINITY, 0.f, 0.f};  // Q: this row's statistics
    if (!KEYS && row < T) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mine[k] = o.stats[((int64_t)(b * Hq + rh) * q_steps + row / kStep) * (C::STATS * kStep) + k * kStep + row % kStep];
    }
    const int seen = KEYS ? 0 : row < T ? (int)s.seen(PACK ? row / P : row, n) : 0;
    const int64_t from64 = s.causal ? row - s.start : 0;  // keys: the first query that sees this one
    const int from0 = from64 < 0 ? 0 : from64 >= s.T ? T : (int)from64 * P;
    // PACK: lam is its column's (keys: all but 2^E, which the largest in the group gives) or this row's
    float lam_most = 0.f, lam_own = 0.f;
    if (PACK && KEYS) {
      const int e = lam_exponent(s, rh * P, lam_most);
      lam_own = __uint_as_float((uint32_t)(127 + e) << 23);
    }
    if (PACK && !KEYS) lam_own = row < T ? __ldg(s.lam + rh * P + row % P) : 0.f;
    bool ok = true;
    float ga = 0.f;  // factor of the last step's products
    // What a step needs besides its scores; read a step ahead, or its latency adds to every step's chain
    // (1700 cycles of 4700).
    struct StepData {
      float fx0, fx1, fxv, lam, gn;
      int x0;
    } next;
    int step_head = KEYS && !each && !PACK ? hk * s.G : rh, step = first;  // of the step to be read next
    const int xtiles = (int)(KEYS ? x.qt : x.kt);
    auto read_step = [&]() {
      const int xt = step >> 1;  // tiles have two steps
      const int64_t xq = (int64_t)(KEYS ? b * 2 * Hq + 2 * step_head : b * 2 * s.Hk + 2 * hk) * xtiles + xt;
      next.fx0 = (KEYS ? x.fq : x.fk)[xq];
      next.fx1 = (KEYS ? x.fq : x.fk)[xq + xtiles];
      next.lam = PACK ? lam_own : __ldg(s.lam + step_head);
      next.fxv = (KEYS ? x.fg : x.fv)[(int64_t)(KEYS ? b * Hq + step_head : b * s.Hk + hk) * xtiles + xt];
      if (MODE != kModeV) next.gn = x.ng[(int64_t)(b * Hq + step_head) * x.qt + (KEYS ? xt : rt)];
      next.x0 = step * kStep;
      if (++step == first + per_head) step = first, ++step_head;
    };
    if (steps) read_step();
    auto add_products = [&]() {
      const uint64_t g2 = two(ga, ga);
#pragma unroll
      for (int c = 0; c < AC / 16; ++c) {
        uint32_t y[16];
        tld16_issue(tmem + lane_row + ACC + part * AC + 16 * c, y);
        tld_wait();
        after_wait(y);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[8 * c + j] = fma2(two(y[2 * j], y[2 * j + 1]), g2, acc[8 * c + j]);
      }
    };
    for (int i = 0; i < steps; ++i) {
      const int st = i & 1, x0 = next.x0;
      const float f0 = factor2(fr0, next.fx0), f1 = factor2(fr1, next.fx1), lam = next.lam;
      float next_ga, beta = 0.f, fp = 0.f, sw = 0.f;
      if (MODE == kModeV) {  // w scale: 1 + |lam| -> [2^13, 2^14)
        int e = (int)(__float_as_uint(1.f + (PACK ? lam_most : fabsf(lam))) >> 23) - 127;
        e = e > 113 ? 113 : e;
        sw = __uint_as_float((uint32_t)(140 - e) << 23);
        next_ga = next.fxv * __uint_as_float((uint32_t)(114 + e) << 23);
      } else {  // ds scale: 2 |dO| |V| below 2^14
        // (sums of exponents: the products themselves may leave fp32's range)
        int e = (int)(__float_as_uint(next.gn) >> 23) + (int)(__float_as_uint(vn) >> 23) - 2 * 127 + 2;
        e = e < -113 ? -113 : e > 113 ? 113 : e;
        beta = __uint_as_float((uint32_t)(140 - e) << 23);
        const int ep = (int)(__float_as_uint(frv) >> 23) + (int)(__float_as_uint(next.fxv) >> 23) - 127 + 13 - e;
        fp = ep < 1 ? 0.f : __uint_as_float((uint32_t)(ep > 254 ? 254 : ep) << 23);
        next_ga = (half ? -lam * next.fx1 : next.fx0) * (KEYS ? kLn2 : s.scale) * __uint_as_float((uint32_t)(114 + e) << 23);
        next_ga = fminf(fmaxf(next_ga, -1.7014118e38f), 1.7014118e38f);
      }
      const uint64_t f02 = two(f0, f0), f12 = two(f1, f1), fp2 = two(fp, fp), nb2 = two(-beta, -beta),
                     sw2 = two(sw, sw), lw2 = two(-lam * sw, -lam * sw);
      ok = __all_sync(0xffffffffu, bar_wait(s_full + st, (i >> 1) & 1, abort_flag, s.err, 17));
      // keys: the statistics came with the step's copies; waiting here orders their reads
      if (KEYS) ok = ok && __all_sync(0xffffffffu, bar_wait(x_full + st, (i >> 1) & 1, abort_flag, s.err, 18));
      if (!ok) break;
      fence_after();
      if (i + 1 < steps) read_step();
      // columns of these 16 that are seen: [lo_c, hi_c); queries behind the last have lse = +inf
      int lo_c = 0, hi_c = 16;
      if (KEYS) {
        const int from = from0 - x0 - 16 * part;
        lo_c = from < 0 ? 0 : from > 16 ? 16 : from;
        if (row >= n) hi_c = 0;
      } else {
        const int end = seen - x0 - 16 * part;
        hi_c = end < 0 ? 0 : end > 16 ? 16 : end;
      }
      const bool whole = __all_sync(0xffffffffu, lo_c == 0 && hi_c == 16);
      const uint32_t ts = tmem + lane_row + st * 128 + 16 * part, tp = tmem + lane_row + kDp + 16 * part;
      const float *col = stat + st * (C::STATS * kStep) + 16 * part;
      {
        uint32_t y0[16], y1[16], yp[16], yq[16];
        tld16_issue(ts, y0);
        tld16_issue(ts + 64, y1);
        if (MODE != kModeV) {
          tld16_issue(tp, yp);
          tld16_issue(tp + 64, yq);
        }
        tld_wait();
        after_wait(y0);
        after_wait(y1);
        if (MODE != kModeV) {
          after_wait(yp);
          after_wait(yq);
        }
        uint32_t h0[8], l0[8], h1[8], l1[8];
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4) {  // four columns
          float q[C::STATS][4];
          if (KEYS) {
#pragma unroll
            for (int k = 0; k < C::STATS; ++k) {
              if (MODE == kModeV && (k == 2 || k == 3)) continue;
              const float4 v = *reinterpret_cast<const float4 *>(col + k * kStep + 4 * j4);
              q[k][0] = v.x, q[k][1] = v.y, q[k][2] = v.z, q[k][3] = v.w;
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int j = 2 * j4 + u, e0 = 2 * j, e1 = e0 + 1;
            auto st2 = [&](int k) { return KEYS ? two(q[k][2 * u], q[k][2 * u + 1]) : two(mine[k], mine[k]); };
            float a, d, a1, d1;
            untwo(sub2(mul2(two(y0[e0], y0[e1]), f02), st2(0)), a, d);
            untwo(sub2(mul2(two(y1[e0], y1[e1]), f12), st2(1)), a1, d1);
            a = ex2(a), d = ex2(d), a1 = ex2(a1), d1 = ex2(d1);
            if (!whole) {
              if (e0 < lo_c || e0 >= hi_c) a = a1 = 0.f;
              if (e1 < lo_c || e1 >= hi_c) d = d1 = 0.f;
            }
            const uint64_t p0 = two(a, d);
            uint64_t p1 = two(a1, d1);
            if (PACK && KEYS) p1 = mul2(p1, two(q[C::STATS - 1][2 * u], q[C::STATS - 1][2 * u + 1]));
            if (MODE == kModeV) {
              cut2(fma2(p1, lw2, mul2(p0, sw2)), h0[j], l0[j]);
            } else {
              const uint64_t dp = add2(two(yp[e0], yp[e1]), two(yq[e0], yq[e1]));
              cut2(mul2(p0, fma2(dp, fp2, mul2(st2(2), nb2))), h0[j], l0[j]);
              cut2(mul2(p1, fma2(dp, fp2, mul2(st2(3), nb2))), h1[j], l1[j]);
            }
          }
        }
        tst_pairs(ts, h0, l0);
        if (MODE != kModeV) tst_pairs(ts + 64, h1, l1);
      }
      if (i) {  // ran under this step's scores
        ok = __all_sync(0xffffffffu, bar_wait(a_full, (i - 1) & 1, abort_flag, s.err, 19));
        if (!ok) break;
        fence_after();
        add_products();
      }
      tst_wait();
      fence_before();
      bar_arrive(p_full + st);
      ga = next_ga;
    }
    if (steps) {
      ok = __all_sync(0xffffffffu, ok && bar_wait(all_done, 0, abort_flag, s.err, 20));
      fence_after();
      if (ok) add_products();
    }
    // through shared memory, so that a warp stores whole rows
    constexpr int W = 4 * AC, CH = W / 4;  // columns of the block's result: both maps, or V's
    float4 *stage = reinterpret_cast<float4 *>(sm);
#pragma unroll
    for (int c = 0; c < AC / 4; ++c) {
      float4 v;
      untwo(acc[2 * c], v.x, v.y);
      untwo(acc[2 * c + 1], v.z, v.w);
      stage[r * CH + ((part * (AC / 4) + c) ^ (r & 7))] = v;
    }
    asm volatile("bar.sync 1, 512;" ::: "memory");
    const int rows = KEYS ? (int)s.S : T;
    if (ok) {
      const int w = MODE == kModeV ? s.dv : s.d;  // a result row: one of w, or two maps' of w
      float *dst = MODE == kModeV ? o.dv : MODE == kModeK ? o.dk : o.dq;
      const bool four = (w & 3) == 0 && ((uintptr_t)dst & 15) == 0;
      const int c = lane % CH, sub = lane / CH;
      const int m = MODE == kModeV ? 0 : c / 16, e = 4 * (MODE == kModeV ? c : c % 16);
      for (int k = (warp - 4) * (32 / CH) + sub; k < 128; k += 16 * (32 / CH)) {
        if (r0 + k >= rows) break;
        const float4 v = stage[k * CH + (c ^ (k & 7))];
        int64_t to = ((int64_t)b * rows + r0 + k) * heads + rh;
        if (PACK && !KEYS) to = (int64_t)b * rows * heads + (int64_t)((r0 + k) / P) * s.H + rh * P + (r0 + k) % P;
        float *p = dst + to * (MODE == kModeV ? w : 2 * w) + m * w + e;
        if (four) {
          if (e < w) *reinterpret_cast<float4 *>(p) = v;
        } else {
          if (e < w) p[0] = v.x;
          if (e + 1 < w) p[1] = v.y;
          if (e + 2 < w) p[2] = v.z;
          if (e + 3 < w) p[3] = v.w;
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

template <int DV, bool PACK>
__global__ void __launch_bounds__(kThreads, 1)
    k_diff_bwd(const __grid_constant__ Shape s, const __grid_constant__ Split x, const __grid_constant__ CUtensorMap mq,
               const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
               const __grid_constant__ CUtensorMap mg, const __grid_constant__ Grads o) {
  extern __shared__ __align__(1024) uint8_t sm[];
  if (su32(sm) & 1023) {  // the swizzled tiles need it; there is no room to align by hand
    if (threadIdx.x == 0) atomicCAS(s.err, 0, DEVERR_LAYOUT);
    return;
  }
  unsigned block;
  const int kind = block_kind(o, blockIdx.x, block);
  if (kind == kModeK)
    body<DV, kModeK, PACK>(s, x, mq, mk, mv, mg, o, sm, block);
  else if (kind == kModeQ)
    body<DV, kModeQ, PACK>(s, x, mq, mk, mv, mg, o, sm, block);
  else
    body<DV, kModeV, PACK>(s, x, mq, mk, mv, mg, o, sm, block);
}

// dst[row][hk][w] = sum over the heads g of a group of src[row][hk G + g][w], for dk and dv in turn
struct GroupSum {
  const float *src[2];
  float *dst[2];
  int w[2];
};
__global__ void __launch_bounds__(256) k_diff_group_sum(const __grid_constant__ GroupSum j, int64_t heads, int G) {
  wait_for_previous();
  const int which = blockIdx.y, w = j.w[which];
  const int64_t n = heads * w;
  const bool four = (w & 3) == 0 && ((uintptr_t)j.dst[which] & 15) == 0;
  const int64_t step = (int64_t)gridDim.x * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (four) {
    const int w4 = w >> 2;
    for (int64_t i = first; i < n >> 2; i += step) {
      const int64_t head = i / w4;
      const float4 *p = reinterpret_cast<const float4 *>(j.src[which]) + head * G * w4 + (i - head * w4);
      float4 v = *p;
      for (int g = 1; g < G; ++g) {
        const float4 y = p[(int64_t)g * w4];
        v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
      }
      reinterpret_cast<float4 *>(j.dst[which])[i] = v;
    }
  } else {
    for (int64_t i = first; i < n; i += step) {
      const int64_t head = i / w;
      const float *p = j.src[which] + head * G * w + (i - head * w);
      float v = *p;
      for (int g = 1; g < G; ++g) v += p[(int64_t)g * w];
      j.dst[which][i] = v;
    }
  }
}

template <int DV, bool PACK>
int launch(tx_ctx *ctx, const Shape &s, const Split &x, const float *stats, const float *sums, float *dq, float *dk,
           float *dv, float *dlam) {
  CUtensorMap mq, mk, mv, mg;
  if (!split_map(&mq, x.q, 64, s.rows(), s.B * 2 * s.row_heads()) || !split_map(&mk, x.k, 64, s.S, s.B * 2 * s.Hk) ||
      !split_map(&mv, x.v, DV, s.S, s.B * s.Hk) || !split_map(&mg, x.g, DV, s.rows(), s.B * s.row_heads()))
    return tx_fail(ctx, TX_ERR_UNSUPPORTED, "differential attention: tensor map");
  // A key block that runs over all heads of a group may outlast everything else: then each head has
  // blocks and sums of its own, added up afterwards (5 x 413, 3 heads over 1: 27 + 2.5 us for 64).  Where
  // the whole fills the SMs longer anyway it would cost: 2 x 2048 causal, 8 heads over 4: 276 + 10 us for
  // 263.  Lengths in steps; a V block's step counts half.
  const double q_steps = (double)((s.T + kStep - 1) / kStep), k_steps = (double)((s.S + kStep - 1) / kStep);
  const double work = (s.causal ? 0.5 : 1.0) * (double)(s.B * s.H) *
                      ((dk ? 1.5 * (double)x.kt * q_steps : 0.0) + (dq ? (double)x.qt * k_steps : 0.0));
  const bool each = !PACK && dk && s.G > 1 && (double)s.G * q_steps > work / ctx->num_sms;
  const size_t rows = (size_t)(s.B * s.S * s.H);
  Scratch part(ctx, each ? rows * (size_t)(2 * s.d + s.dv) * 4 : 0);
  if (each && !part.ptr) return TX_ERR_OOM;
  // dv's part first, whole 16-byte groups either way
  float *pv = part.as<float>(), *pk = each ? pv + rows * s.dv : nullptr;
  if (each && ((rows * s.dv) & 3)) pk = pv, pv = pk + rows * 2 * s.d;
  const unsigned nk = dk ? (unsigned)(s.B * (each ? s.H : s.Hk)) : 0, nq = dq ? (unsigned)(s.B * s.row_heads()) : 0;
  // Blocks start in order, so the longest come first.  Causal tiles get shorter from level to level:
  // the kinds take turns, and the last blocks are the shortest of each.  Otherwise K and Q blocks are
  // alike and V blocks half as long, so V comes last.
  const unsigned kt = (unsigned)x.kt, qt = (unsigned)x.qt;
  const Grads o{stats, sums, dq, each ? pk : dk, each ? pv : dv, dlam, nk, nq, kt < qt ? kt : qt,
                (unsigned)(s.causal && nk && nq), kt, qt, each};
  static SmemGrant granted;
  TX_TRY(granted.take(ctx, (const void *)k_diff_bwd<DV, PACK>, Cfg<DV, PACK>::SMEM));
  TX_TRY(launch_behind(ctx, "k_diff_bwd", k_diff_bwd<DV, PACK>, 2 * nk * kt + nq * qt, kThreads, Cfg<DV, PACK>::SMEM, s,
                       x, mq, mk, mv, mg, o));
  if (each) {
    const GroupSum j{{pk, pv}, {dk, dv}, {2 * s.d, s.dv}};
    const int64_t n = s.B * s.S * s.Hk * (2 * s.d > s.dv ? 2 * s.d : s.dv);
    TX_TRY(launch_behind(ctx, "k_diff_group_sum", k_diff_group_sum, dim3(grid_for(n / 4, 256), 2), 256, 0, j,
                         s.B * s.S * s.Hk, s.G));
  }
  return TX_OK;
}

}  // namespace

int tc_backward(tx_ctx *ctx, const Shape &s, const Split &x, const float *stats, const float *sums, float *dq,
                float *dk, float *dv, float *dlam) {
  if (s.P > 1)
    return x.vw == 64 ? launch<64, true>(ctx, s, x, stats, sums, dq, dk, dv, dlam)
                      : launch<128, true>(ctx, s, x, stats, sums, dq, dk, dv, dlam);
  return x.vw == 64 ? launch<64, false>(ctx, s, x, stats, sums, dq, dk, dv, dlam)
                    : launch<128, false>(ctx, s, x, stats, sums, dq, dk, dv, dlam);
}

}  // namespace tx_diff
