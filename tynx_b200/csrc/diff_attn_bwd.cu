// Differential attention backward on tcgen05: two kernels of one form.
//
// Both keep 128 rows in shared memory and stream the other side in steps of
// 64 rows.  KV: the rows are keys (K of both maps, V) and the steps run over the
// queries (Q, dO) of every head that shares them; it accumulates dK and dV.  Q:
// the rows are queries (Q, dO), the steps run over the keys; it accumulates dQ.
// Computing the scores in both costs 6 of 14 products, and needs neither atomic
// additions nor a buffer of partial sums: the results do not depend on any order.
// With R the resident side and X the streamed one, per step
//   S_m = R_m X_m^T, dP = R_v X_v^T        (R rows x 64, three fp16 products each)
//   A_m = 2^(S_m - lse_m),  ds_m = A_m (dP - D_m),  w = A_1 - lam A_2
//   acc_m += ds_m X_m,  KV: acc_v += w X_v
// ds and w go back over S and dP in TMEM as pairs of fp16, scaled by powers of
// two: |w| <= 1 + |lam|, and |dP - D| <= 2 max |dO_i| max |V_j| (2-norms of rows,
// found by the split), so nothing overflows and the largest stay near 2^13.
// The steps' products are added in registers (the tensor core's own addition
// truncates); they carry the step's factors: f of X's tile, 1 / scale of ds,
// -lam of the head for map 2.
// Tensor time a step: KV 2 x 384 + 768 + 2 x 384 + 768 = 3072 cycles, Q 2304;
// its elementwise part is about 22 issue slots for each of the 8192 pairs over
// eight warps, 1400 cycles.  Q keeps two steps' scores in TMEM, so that the next
// step's products run under it; KV's accumulators leave room for one.
#include "diff_attn.cuh"

namespace tx_diff {
namespace {

constexpr int kThreads = 384, kStep = 64;

template <int DV>
struct Cfg {
  static constexpr int RQ = 2 * 128 * 64 * 2;              // one map's resident tile, heads and tails
  static constexpr int RV = 2 * 128 * DV * 2;
  static constexpr int XBLK = kStep * 64 * 2;              // [64 rows x 64] fp16
  static constexpr int XQ = 2 * XBLK;                      // one map's step
  static constexpr int XV = 2 * (DV / 64) * XBLK;
  static constexpr int STAT = kStep * 16;                  // float4 a streamed query
  static constexpr int TILES = 2 * RQ + RV + 2 * (2 * XQ) + XV;
  static constexpr int SMEM = TILES + 2 * STAT + 512;
  static_assert(SMEM <= 232448, "shared memory of an SM");
};

struct Grads {
  const float4 *stats;
  float *d1, *dv;  // dq, or dk and dv
};

template <int DV, bool KV>
__global__ void __launch_bounds__(kThreads, 1)
    k_diff_bwd(const __grid_constant__ Shape s, const __grid_constant__ Split x, const __grid_constant__ CUtensorMap mrq,
               const __grid_constant__ CUtensorMap mrv, const __grid_constant__ CUtensorMap mxq,
               const __grid_constant__ CUtensorMap mxv, Grads o) {
  using C = Cfg<DV>;
  constexpr int NB = KV ? 1 : 2;                        // steps whose scores TMEM holds
  constexpr uint32_t ACC = KV ? 256 : 384;              // acc_1, acc_2 (64 columns each), acc_v
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t srq = su32(sm), srv = srq + 2 * C::RQ, sxq = srv + C::RV, sxv = sxq + 4 * C::XQ;
  const float4 *stat = reinterpret_cast<const float4 *>(sm + C::TILES);
  uint64_t *bars = reinterpret_cast<uint64_t *>(sm + C::TILES + 2 * C::STAT);
  uint64_t *r_full = bars, *x_full = bars + 1, *x_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 6,
           *s_full = bars + 7, *p_full = bars + 9, *a_full = bars + 11, *all_done = bars + 12;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 16);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
  uint32_t *vmax = tmem_holder + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (srq & 1023) {  // the swizzled tiles need it; there is no room to align by hand
    if (threadIdx.x == 0) atomicCAS(s.err, 0, DEVERR_LAYOUT);
    return;
  }

  // KV: block = (tile of keys, b, key head), the first tiles see most queries;
  // Q: (tile of queries, b, head), the last tiles see most keys
  const int64_t rheads = s.B * (KV ? s.Hk : s.H), rtiles = KV ? x.kt : x.qt;
  const int64_t rt = KV ? (int64_t)blockIdx.x / rheads : rtiles - 1 - (int64_t)blockIdx.x / rheads;
  const int64_t bh = (int64_t)blockIdx.x % rheads, b = bh / (KV ? s.Hk : s.H);
  const int rh = (int)(bh - b * (KV ? s.Hk : s.H)), hk = KV ? rh : rh / s.G;
  const int64_t r0 = rt * 128, n = s.length(b);
  int first = 0, per_head;  // steps of each head, KV: from step `first` on
  if (KV) {
    const int64_t all = (s.T + kStep - 1) / kStep;
    int64_t q_first = s.causal ? r0 - s.start : 0;  // the first query that sees the first key
    if (q_first < 0) q_first = 0;
    first = (int)(q_first / kStep);
    per_head = first < all && r0 < n ? (int)all - first : 0;
  } else {
    const int64_t last = r0 + 127 < s.T ? r0 + 127 : s.T - 1;
    per_head = (int)((s.seen(last, n) + kStep - 1) / kStep);
  }
  const int steps = KV ? per_head * s.G : per_head;

  if (threadIdx.x == 0) {
    bar_init(r_full, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(x_full + i, 1);
      bar_init(x_empty + i, 1);
      bar_init(s_full + i, 1);
      bar_init(p_full + i, 256);
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
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_holder;
  // the largest row norm of this head's values (all tiles: D runs over all keys)
  for (int64_t i = threadIdx.x; i < x.kt; i += kThreads)
    atomicMax(vmax, __float_as_uint(__ldg(x.nv + (b * s.Hk + hk) * x.kt + i)));
  __syncthreads();

  // step i: head, first streamed row
  auto head_of = [&](int i) { return KV ? hk * s.G + i / per_head : rh; };
  auto row_of = [&](int i) { return (int64_t)(KV ? first + i % per_head : i) * kStep; };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0 && lane == 0 && steps) {
      bar_expect(r_full, 2 * C::RQ + C::RV);
      for (int m = 0; m < 2; ++m)
        for (int p = 0; p < 2; ++p)
          tma_3d(srq + m * C::RQ + p * (C::RQ / 2), &mrq, r_full, p * 64, (int)r0,
                 (int)(KV ? b * 2 * s.Hk + 2 * hk + m : b * 2 * s.H + 2 * rh + m));
      for (int p = 0; p < 2 * (DV / 64); ++p)
        tma_3d(srv + p * (128 * 128), &mrv, r_full, p * 64, (int)r0, (int)(KV ? b * s.Hk + hk : b * s.H + rh));
      bool ok = true;
      int lx = 0, lv = 0;
      for (int i = 0; i < steps && ok; ++i) {
        const int st = i & 1, h = head_of(i);
        const int64_t x0 = row_of(i);
        if (i > 1) ok = bar_wait(x_empty + st, ((i >> 1) - 1) & 1, abort_flag, s.err, 11);
        if (!ok) break;
        const int64_t live = s.T - x0 < kStep ? s.T - x0 : kStep;
        bar_expect(x_full + st, 2 * C::XQ + (KV ? (uint32_t)live * 16u : 0u));
        for (int m = 0; m < 2; ++m)
          for (int p = 0; p < 2; ++p)
            tma_3d(sxq + st * 2 * C::XQ + m * C::XQ + p * C::XBLK, &mxq, x_full + st, p * 64, (int)x0,
                   (int)(KV ? b * 2 * s.H + 2 * h + m : b * 2 * s.Hk + 2 * hk + m));
        if (KV)
          bulk_load(su32(stat + st * kStep), o.stats + (b * s.H + h) * s.T + x0, (uint32_t)live * 16u, x_full + st);
        ++lx;
        if (i) ok = bar_wait(v_empty, (i - 1) & 1, abort_flag, s.err, 12);
        if (!ok) break;
        bar_expect(v_full, C::XV);
        for (int p = 0; p < 2 * (DV / 64); ++p)
          tma_3d(sxv + p * C::XBLK, &mxv, v_full, p * 64, (int)x0, (int)(KV ? b * s.H + h : b * s.Hk + hk));
        ++lv;
      }
      // every copy has landed before the CTA's memory is released
      bar_drain(r_full, 0);
      for (int i = lx - 1; i >= 0 && i > lx - 3; --i) bar_drain(x_full + (i & 1), (i >> 1) & 1);
      if (lv) bar_drain(v_full, (lv - 1) & 1);
    } else if (warp == 1 && lane == 0 && steps) {
      constexpr uint32_t id_s = idesc(kStep, false), id_a = idesc(64, true), id_v = idesc(DV, true);
      bool ok = bar_wait(r_full, 0, abort_flag, s.err, 13);
      auto scores = [&](int i) {  // S_1, S_2, dP of step i
        const uint32_t ts = tmem + (i % NB) * 192;
        const int st = i & 1;
        ok = ok && bar_wait(x_full + st, (i >> 1) & 1, abort_flag, s.err, 14);
        if (!ok) return;
        fence_after();
        for (int m = 0; m < 2; ++m) {
          const uint32_t rh_ = srq + m * C::RQ, rl = rh_ + C::RQ / 2, xh = sxq + st * 2 * C::XQ + m * C::XQ, xl = xh + C::XBLK;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_ss(ts + m * 64, kdesc(rh_, k), kdesc(xl, k), id_s, k ? 1u : 0u);
            mma_ss(ts + m * 64, kdesc(rl, k), kdesc(xh, k), id_s, 1u);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ss(ts + m * 64, kdesc(rh_, k), kdesc(xh, k), id_s, 1u);
        }
        ok = bar_wait(v_full, i & 1, abort_flag, s.err, 15);
        if (!ok) return;
        fence_after();
#pragma unroll
        for (int c = 0; c < DV / 64; ++c) {
          const uint32_t rh_ = srv + c * 16384, rl = rh_ + (DV / 64) * 16384, xh = sxv + c * C::XBLK,
                         xl = xh + (DV / 64) * C::XBLK;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_ss(ts + 128, kdesc(rh_, k), kdesc(xl, k), id_s, (c || k) ? 1u : 0u);
            mma_ss(ts + 128, kdesc(rl, k), kdesc(xh, k), id_s, 1u);
          }
        }
#pragma unroll
        for (int c = 0; c < DV / 64; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ss(ts + 128, kdesc(srv + c * 16384, k), kdesc(sxv + c * C::XBLK, k), id_s, 1u);
        if (!KV) mma_commit(v_empty);
        mma_commit(s_full + i % NB);
      };
      scores(0);
      for (int i = 0; i < steps && ok; ++i) {
        if (NB == 2 && i + 1 < steps) scores(i + 1);
        const uint32_t ts = tmem + (i % NB) * 192;
        const int st = i & 1;
        ok = ok && bar_wait(p_full + i % NB, (i / NB) & 1, abort_flag, s.err, 16);
        if (!ok) break;
        fence_after();
        if (KV) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_ts(tmem + ACC + 128, ts + 128 + k * 16, ndesc(sxv + (DV / 64) * C::XBLK, k, C::XBLK), id_v, k ? 1u : 0u);
            mma_ts(tmem + ACC + 128, ts + 128 + k * 16 + 8, ndesc(sxv, k, C::XBLK), id_v, 1u);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ts(tmem + ACC + 128, ts + 128 + k * 16, ndesc(sxv, k, C::XBLK), id_v, 1u);
          mma_commit(v_empty);
        }
        for (int m = 0; m < 2; ++m) {
          const uint32_t xh = sxq + st * 2 * C::XQ + m * C::XQ, xl = xh + C::XBLK, ta = tmem + ACC + m * 64;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_ts(ta, ts + m * 64 + k * 16, ndesc(xl, k, C::XBLK), id_a, k ? 1u : 0u);
            mma_ts(ta, ts + m * 64 + k * 16 + 8, ndesc(xh, k, C::XBLK), id_a, 1u);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ts(ta, ts + m * 64 + k * 16, ndesc(xh, k, C::XBLK), id_a, 1u);
        }
        mma_commit(x_empty + st);
        mma_commit(a_full);
        if (NB == 1 && i + 1 < steps) scores(i + 1);
      }
      mma_commit(all_done);
      bar_drain(all_done, 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // warpgroup `half` takes streamed rows 32 half .. of every step, and of the
    // results acc_half (64 columns) and its half of acc_v's
    const int half = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_row = (uint32_t)(quad * 32) << 16;
    const int64_t row = r0 + r;
    constexpr int VC = KV ? DV / 2 : 0;  // columns of acc_v
    float acc[64], acv[KV ? VC : 1];
#pragma unroll
    for (int j = 0; j < 64; ++j) acc[j] = 0.f;
    if (KV) {
#pragma unroll
      for (int j = 0; j < VC; ++j) acv[j] = 0.f;
    }
    const float vn = __uint_as_float(*vmax);
    // resident factors: fr of both maps and of V (KV) or dO (Q)
    const int64_t rq = KV ? (b * 2 * s.Hk + 2 * hk) * x.kt + rt : (b * 2 * s.H + 2 * rh) * x.qt + rt;
    const float fr0 = __ldg((KV ? x.fk : x.fq) + rq), fr1 = __ldg((KV ? x.fk : x.fq) + rq + rtiles);
    const float frv = __ldg((KV ? x.fv : x.fg) + (KV ? (b * s.Hk + hk) : (b * s.H + rh)) * rtiles + rt);
    float4 mine = make_float4(INFINITY, INFINITY, 0.f, 0.f);  // Q: this row's statistics
    if (!KV && row < s.T) mine = __ldg(o.stats + (b * s.H + rh) * s.T + row);
    const int64_t seen = KV ? 0 : row < s.T ? s.seen(row, n) : 0;
    bool ok = true;
    float ga = 0.f, gv = 0.f;  // factors of the last step's products
    auto add_products = [&]() {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t y[32];
        tld32_issue(tmem + lane_row + ACC + half * 64 + 32 * c, y);
        tld_wait();
        after_wait(y);
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[32 * c + j] = fmaf(__uint_as_float(y[j]), ga, acc[32 * c + j]);
      }
      if (KV) {
#pragma unroll
        for (int c = 0; c < VC / 32; ++c) {
          uint32_t y[32];
          tld32_issue(tmem + lane_row + ACC + 128 + half * VC + 32 * c, y);
          tld_wait();
          after_wait(y);
#pragma unroll
          for (int j = 0; j < 32; ++j) acv[32 * c + j] = fmaf(__uint_as_float(y[j]), gv, acv[32 * c + j]);
        }
      }
    };
    for (int i = 0; i < steps; ++i) {
      const int h = head_of(i);
      const int64_t x0 = row_of(i), xt = x0 >> 7;
      const int64_t xq = KV ? (b * 2 * s.H + 2 * h) * x.qt + xt : (b * 2 * s.Hk + 2 * hk) * x.kt + xt;
      const int64_t xtiles = KV ? x.qt : x.kt;
      const float fx0 = __ldg((KV ? x.fq : x.fk) + xq), fx1 = __ldg((KV ? x.fq : x.fk) + xq + xtiles);
      const float fxv = __ldg((KV ? x.fg : x.fv) + (KV ? (b * s.H + h) * x.qt : (b * s.Hk + hk) * x.kt) + xt);
      const float gn = __ldg(x.ng + (b * s.H + h) * x.qt + (KV ? xt : rt)), lam = __ldg(s.lam + h);
      // ds scale: 2 gn vn -> [2^13, 2^14); w scale: 1 + |lam| likewise
      int e = (int)(__float_as_uint(2.f * gn * vn) >> 23) - 127;
      e = e < -113 ? -113 : e > 113 ? 113 : e;
      const float beta = __uint_as_float((uint32_t)(140 - e) << 23), ibeta = __uint_as_float((uint32_t)(114 + e) << 23);
      int el = (int)(__float_as_uint(1.f + fabsf(lam)) >> 23) - 127;
      el = el > 100 ? 100 : el;
      const float sw = __uint_as_float((uint32_t)(140 - el) << 23), isw = __uint_as_float((uint32_t)(114 + el) << 23);
      const float f0 = factor2(fr0, fx0), f1 = factor2(fr1, fx1), fp = factor2(frv, fxv) * beta, lw = -lam * sw;
      const int st = i & 1;
      ok = __all_sync(0xffffffffu, bar_wait(s_full + i % NB, (i / NB) & 1, abort_flag, s.err, 17));
      if (!ok) break;
      // KV: the statistics came by the step's copies; their barrier is complete, this read orders them
      if (KV) ok = __all_sync(0xffffffffu, bar_wait(x_full + st, (i >> 1) & 1, abort_flag, s.err, 18));
      if (!ok) break;
      fence_after();
      if (NB == 1 && i) add_products();  // behind the scores of this step the last step's products are done
      // columns 0 .. of this half's 32 that exist and are seen: [lo, hi)
      int lo_c = 0, hi_c;
      if (KV) {
        const int64_t end = s.T - x0 - 32 * half;
        hi_c = end < 0 ? 0 : end > 32 ? 32 : (int)end;
        const int64_t from = s.causal ? row - s.start - x0 - 32 * half : 0;  // the first query that sees this key
        lo_c = from < 0 ? 0 : from > 32 ? 32 : (int)from;
        if (row >= n) hi_c = 0;
      } else {
        const int64_t end = seen - x0 - 32 * half;
        hi_c = end < 0 ? 0 : end > 32 ? 32 : (int)end;
      }
      const bool whole = __all_sync(0xffffffffu, lo_c == 0 && hi_c == 32);
      const uint32_t ts = tmem + lane_row + (i % NB) * 192 + 32 * half;
      const float4 *col = stat + st * kStep + 32 * half;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t y0[16], y1[16], yp[16];
        tld16_issue(ts + 16 * c, y0);
        tld16_issue(ts + 64 + 16 * c, y1);
        tld16_issue(ts + 128 + 16 * c, yp);
        tld_wait();
        after_wait(y0);
        after_wait(y1);
        after_wait(yp);
        uint32_t h0[8], l0[8], h1[8], l1[8], hw[8], lw_[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float a0[2], a1[2], w[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int k = 2 * j + u;
            const float4 q = KV ? col[16 * c + k] : mine;
            float p0 = ex2(fmaf(__uint_as_float(y0[k]), f0, -q.x)), p1 = ex2(fmaf(__uint_as_float(y1[k]), f1, -q.y));
            if (!whole && (16 * c + k < lo_c || 16 * c + k >= hi_c)) p0 = p1 = 0.f;
            const float dp = __uint_as_float(yp[k]);
            float g0 = fmaf(dp, fp, -q.z * beta), g1 = fmaf(dp, fp, -q.w * beta);
            if (!whole && (16 * c + k < lo_c || 16 * c + k >= hi_c)) g0 = g1 = 0.f;
            a0[u] = p0 * g0;
            a1[u] = p1 * g1;
            w[u] = fmaf(p1, lw, p0 * sw);
          }
          split2(a0[0], a0[1], h0[j], l0[j]);
          split2(a1[0], a1[1], h1[j], l1[j]);
          if (KV) split2(w[0], w[1], hw[j], lw_[j]);
        }
        tst_pairs(ts + 16 * c, h0, l0);
        tst_pairs(ts + 64 + 16 * c, h1, l1);
        if (KV) tst_pairs(ts + 128 + 16 * c, hw, lw_);
      }
      if (NB == 2 && i) {  // ran under this step's scores
        ok = __all_sync(0xffffffffu, bar_wait(a_full, (i - 1) & 1, abort_flag, s.err, 19));
        if (!ok) break;
        fence_after();
        add_products();
      }
      tst_wait();
      fence_before();
      bar_arrive(p_full + i % NB);
      ga = KV ? (half ? -lam * fx1 : fx0) * kLn2 * ibeta : (half ? -lam * fx1 : fx0) * s.scale * ibeta;
      gv = fxv * isw;
    }
    if (steps) {
      ok = __all_sync(0xffffffffu, ok && bar_wait(all_done, 0, abort_flag, s.err, 20));
      fence_after();
      if (ok) add_products();
    }
    const int64_t rows = KV ? s.S : s.T;
    if (row < rows && ok) {
      const int maps = 2 * (KV ? s.Hk : s.H);
      float *d1 = o.d1 + ((b * rows + row) * maps + 2 * rh + half) * s.d;
      const bool four = (s.d & 3) == 0 && ((uintptr_t)o.d1 & 15) == 0;
#pragma unroll
      for (int j = 0; j < 64; j += 4) {
        if (four) {
          if (j < s.d) *reinterpret_cast<float4 *>(d1 + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (j + u < s.d) d1[j + u] = acc[j + u];
        }
      }
      if (KV) {
        float *dv = o.dv + ((b * rows + row) * s.Hk + rh) * s.dv + half * VC;
        const bool vfour = (s.dv & 3) == 0 && ((uintptr_t)o.dv & 15) == 0;
        const int left = s.dv - half * VC;
#pragma unroll
        for (int j = 0; j < VC; j += 4) {
          if (vfour) {
            if (j < left) *reinterpret_cast<float4 *>(dv + j) = make_float4(acv[j], acv[j + 1], acv[j + 2], acv[j + 3]);
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (j + u < left) dv[j + u] = acv[j + u];
          }
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

template <int DV>
int launch(tx_ctx *ctx, const Shape &s, const Split &x, const float4 *stats, float *dq, float *dk, float *dv) {
  CUtensorMap q128, q64, k128, k64, v128, v64, g128, g64;
  if (!split_map(&q128, x.q, 64, s.T, s.B * 2 * s.H, 128) || !split_map(&q64, x.q, 64, s.T, s.B * 2 * s.H, kStep) ||
      !split_map(&k128, x.k, 64, s.S, s.B * 2 * s.Hk, 128) || !split_map(&k64, x.k, 64, s.S, s.B * 2 * s.Hk, kStep) ||
      !split_map(&v128, x.v, DV, s.S, s.B * s.Hk, 128) || !split_map(&v64, x.v, DV, s.S, s.B * s.Hk, kStep) ||
      !split_map(&g128, x.g, DV, s.T, s.B * s.H, 128) || !split_map(&g64, x.g, DV, s.T, s.B * s.H, kStep))
    return tx_fail(ctx, TX_ERR_UNSUPPORTED, "differential attention: tensor map");
  constexpr int smem = Cfg<DV>::SMEM;
  if (dk) {
    TX_CUDA(ctx, cudaFuncSetAttribute(k_diff_bwd<DV, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    k_diff_bwd<DV, true><<<(unsigned)(x.kt * s.B * s.Hk), kThreads, smem, ctx->stream>>>(s, x, k128, v128, q64, g64,
                                                                                       Grads{stats, dk, dv});
    TX_LAUNCHED(ctx, "k_diff_bwd (keys)");
  }
  if (dq) {
    TX_CUDA(ctx, cudaFuncSetAttribute(k_diff_bwd<DV, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    k_diff_bwd<DV, false><<<(unsigned)(x.qt * s.B * s.H), kThreads, smem, ctx->stream>>>(s, x, q128, g128, k64, v64,
                                                                                      Grads{stats, dq, nullptr});
    TX_LAUNCHED(ctx, "k_diff_bwd (queries)");
  }
  return TX_OK;
}

}  // namespace

int tc_backward(tx_ctx *ctx, const Shape &s, const Split &x, const float4 *stats, float *dq, float *dk, float *dv) {
  return x.vw == 64 ? launch<64>(ctx, s, x, stats, dq, dk, dv) : launch<128>(ctx, s, x, stats, dq, dk, dv);
}

}  // namespace tx_diff
