// Differential attention forward on tcgen05.
//
// A CTA owns 128 queries of one head and streams its keys in tiles of 128,
// both maps side by side: eight warps keep map 1's rows (running maximum, sum
// and output; two threads a row, half of the keys and of the output columns
// each), eight map 2's, and both maps multiply the same value tile.  Per tile and map
//   S = Q K^T               three fp16 products of 128 x 128 x 64   (768 cycles)
//   P = 2^(S - maximum)     registers, split into fp16 pairs, back over S in TMEM
//   O = P V                 three fp16 products of 128 x 128 x 128 (1536 cycles)
// so while one map's warps work on their softmax (about 450 instructions a
// warp, two warps a scheduler; with one warp of all 128 columns the chain of
// dependent instructions took 5400 cycles a tile) the tensor core runs the
// other map's 2304 cycles: it is what bounds the kernel.  TMEM holds S1 | S2 | O1 | O2, all 512
// columns; P lies over S (16 keys' heads and tails take the 16 columns of their
// scores).  O is one tile's product and is added to the running output in
// registers, rescaled there: the tensor core adds into its accumulator with
// truncation, which over thousands of keys loses 1e-5 of the result, and over
// the 24 products of one tile 1e-7.  Shared memory: Q of both maps (64 KB), one
// key tile of both (64 KB, each map's half refilled as soon as its S is done),
// and a ring of three half value tiles (96 KB).
// One CTA an SM takes (query tile, head) after (query tile, head): while its
// warps store one's rows (through the value ring, so that whole lines go out),
// the next one's Q and K arrive and its first scores are multiplied.  Where few
// queries would leave tiles half empty, a tile holds the queries of all heads
// that share a key head (PACK).
// 8192 causal tokens of 8 heads: 428 to 446 us, 628 GFLOP of fp16 products, the
// tensor cores' sustained rate under the power limit; 4 x 64 queries of 8 heads
// over 4 against 4096 keys: 27 us, four tiles a block.
#include "diff_attn.cuh"

namespace tx_diff {
namespace {

constexpr int kThreads = 640;  // producer, MMA, two spare warps, 2 x 8 softmax warps

template <int DV>
struct Cfg {
  static constexpr int HALF = 128 * 64 * 2;           // [128 x 64] fp16
  static constexpr int QK = 2 * HALF;                 // heads and tails of one map's tile
  static constexpr int VBLK = 64 * 64 * 2;            // [64 keys x 64] fp16
  static constexpr int VSLOT = 2 * (DV / 64) * VBLK;  // 64 keys: heads, tails
  static constexpr int RING = 3;
  static constexpr int SMEM = 4 * QK + RING * VSLOT + 512 /*barriers*/ + 2048 /*row exchange*/;
  static_assert(SMEM <= 232448, "shared memory of an SM");
  // output rows pass through the value ring: 32 rows x CW columns a warp at a time
  static constexpr int CW = DV == 128 ? 32 : 16;
  static_assert(16 * 32 * CW * 4 <= RING * VSLOT, "output staging");
};

struct Out {
  float *out, *out2, *lse;
  Parts parts;
  int per;  // tiles of a range of keys
};

__device__ __forceinline__ void store4(float *dst, int c, float4 v, int dv, bool four) {
  if (four) {
    if (c < dv) *reinterpret_cast<float4 *>(dst + c) = v;
  } else {
    if (c < dv) dst[c] = v.x;
    if (c + 1 < dv) dst[c + 1] = v.y;
    if (c + 2 < dv) dst[c + 2] = v.z;
    if (c + 3 < dv) dst[c + 3] = v.w;
  }
}

// One unit of work: a query tile of a head (of a group's heads, Shape::P), and a range of its keys.
struct Item {
  int b, r0, n;  // sequence, first row, valid keys
  int h, hk, qt, split, tile0, tiles;
};
// Item `at` in the order of work: causal, the queries with most keys first.
template <bool PACK>
__device__ __forceinline__ Item item_at(const Shape &s, const Split &x, const Out &o, unsigned at) {
  const int P = PACK ? s.P : 1, row_heads = PACK ? s.row_heads() : s.H;
  const unsigned heads = (unsigned)s.B * row_heads, blocks = (unsigned)x.qt * heads;
  Item w;
  w.split = at / blocks;
  at -= w.split * blocks;
  const unsigned level = at / heads, bh = at - level * heads;
  w.qt = (int)x.qt - 1 - (int)level;
  w.b = bh / row_heads;
  w.h = bh - w.b * row_heads;
  w.hk = PACK ? w.h : w.h / s.G;
  w.r0 = w.qt * 128;
  const int rows = (int)s.T * P, last = w.r0 + 127 < rows ? w.r0 + 127 : rows - 1, tl = PACK ? last / P : last;
  w.n = (int)s.length(w.b);
  w.tile0 = w.split * o.per;
  const int all = ((int)s.seen(tl, w.n) + 127) / 128;
  w.tiles = all <= w.tile0 ? 0 : all - w.tile0 < o.per ? all - w.tile0 : o.per;
  return w;
}
// The item of this CTA's round r: rounds run forth and back, so that a CTA's share of a falling order is
// even.  False: none, in the last round.
__device__ __forceinline__ bool item_of_round(unsigned items, int r, unsigned &at) {
  at = r * gridDim.x + (r & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  return at < items;
}

// PACK: rows are queries of a group's heads (Shape::P = G), otherwise one head's
template <int DV, bool PACK>
__global__ void __launch_bounds__(kThreads, 1)
    k_diff_fwd(const __grid_constant__ Shape s, const __grid_constant__ Split x, const __grid_constant__ CUtensorMap mq,
               const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, Out o) {
  using C = Cfg<DV>;
  extern __shared__ __align__(1024) uint8_t sm[];
  if (su32(sm) & 1023) {  // the swizzled tiles need it
    if (threadIdx.x == 0) atomicCAS(s.err, 0, DEVERR_LAYOUT);
    return;
  }
  const uint32_t sq = su32(sm), sk = sq + 2 * C::QK, sv = sk + 2 * C::QK;
  uint64_t *bars = reinterpret_cast<uint64_t *>(sm + 4 * C::QK + C::RING * C::VSLOT);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 8,
           *s_full = bars + 11, *p_full = bars + 13, *o_full = bars + 15, *q_empty = bars + 17, *staged = bars + 18,
           *all_done = bars + 19;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 20);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
  float *swap = reinterpret_cast<float *>(bars + 64);  // [map][half][row]
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int P = PACK ? s.P : 1, row_heads = PACK ? s.row_heads() : s.H;
  const unsigned items = (unsigned)(x.qt * s.B * row_heads * o.parts.splits);
  const int rounds = (int)((items + gridDim.x - 1) / gridDim.x);

  if (threadIdx.x == 0) {
    bar_init(q_full, 1);
    bar_init(q_empty, 1);
    for (int m = 0; m < 2; ++m) {
      bar_init(k_full + m, 1);
      bar_init(k_empty + m, 1);
      bar_init(s_full + m, 1);
      bar_init(p_full + m, 256);
      bar_init(o_full + m, 1);
    }
    for (int i = 0; i < C::RING; ++i) {
      bar_init(v_full + i, 1);
      bar_init(v_empty + i, 1);
    }
    bar_init(staged, 512);
    bar_init(all_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_holder)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  wait_for_previous();  // the split operands
  next_may_start();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0 && lane == 0) {
      bool ok = true;
      int nq = 0, ni = 0;                // items with keys so far, items so far
      int nk = 0, loaded_k = 0, nv = 0;  // tiles of a map so far, loads of both maps, half value tiles
      for (int r = 0; r < rounds && ok; ++r) {
        unsigned at;
        if (!item_of_round(items, r, at)) continue;
        const Item w = item_at<PACK>(s, x, o, at);
        if (w.tiles) {
          if (nq) ok = bar_wait(q_empty, (nq - 1) & 1, abort_flag, s.err, 1);
          if (!ok) break;
          bar_expect(q_full, 2 * C::QK);
          for (int p = 0; p < 8; ++p)  // (map, head or tail, 64-row half)
            tma_3d(sq + p * C::VBLK, &mq, q_full, (p >> 1 & 1) * 64, w.r0 + (p & 1) * 64,
                   w.b * 2 * row_heads + 2 * w.h + (p >> 2));
          ++nq;
        } else if (ni) {  // no phase is passed over: parities would repeat
          ok = bar_wait(staged, (ni - 1) & 1, abort_flag, s.err, 3);
        }
        for (int i = 0; i < w.tiles && ok; ++i, ++nk) {
          for (int m = 0; m < 2 && ok; ++m) {
            if (nk) ok = bar_wait(k_empty + m, (nk - 1) & 1, abort_flag, s.err, 2);
            if (!ok) break;
            bar_expect(k_full + m, C::QK);
            for (int p = 0; p < 4; ++p)
              tma_3d(sk + m * C::QK + p * C::VBLK, &mk, k_full + m, (p >> 1) * 64, (w.tile0 + i) * 128 + (p & 1) * 64,
                     w.b * 2 * s.Hk + 2 * w.hk + m);
            ++loaded_k;
          }
          // the ring carried the last item's output rows until its warps say so
          if (ok && i == 0 && ni) ok = bar_wait(staged, (ni - 1) & 1, abort_flag, s.err, 3);
          for (int hf = 0; hf < 2 && ok; ++hf, ++nv) {
            const int slot = nv % C::RING, use = nv / C::RING;
            if (use) ok = bar_wait(v_empty + slot, (use - 1) & 1, abort_flag, s.err, 4);
            if (!ok) break;
            bar_expect(v_full + slot, C::VSLOT);
            for (int p = 0; p < 2 * (DV / 64); ++p)
              tma_3d(sv + slot * C::VSLOT + p * C::VBLK, &mv, v_full + slot, p * 64, (w.tile0 + i) * 128 + hf * 64,
                     w.b * s.Hk + w.hk);
          }
        }
        ++ni;
      }
      // every copy has landed before the CTA's memory is released
      if (nq) bar_drain(q_full, (nq - 1) & 1);
      for (int m = 0; m < 2; ++m) {
        const int c = (loaded_k + 1 - m) / 2;  // loads of this map
        if (c) bar_drain(k_full + m, (c - 1) & 1);
      }
      for (int u = nv - 1; u >= 0 && u > nv - 1 - C::RING; --u) bar_drain(v_full + u % C::RING, (u / C::RING) & 1);
    } else if (warp == 1) {
      const uint32_t one = elect_one();
      constexpr uint32_t id_s = idesc(128, false), id_o = idesc(DV, true);
      const int slices = (s.d + 15) / 16;  // of queries and keys; zeros behind them
      bool ok = true, any = false;
      int nq = 0, nt = 0, nv = 0;  // items with keys, tiles and half value tiles so far
      for (int r = 0; r < rounds && ok; ++r) {
        unsigned at;
        if (!item_of_round(items, r, at)) continue;
        const int tiles = __shfl_sync(0xffffffffu, item_at<PACK>(s, x, o, at).tiles, 0);
        if (!tiles) continue;
        any = true;
        ok = mma_wait(q_full, nq & 1, abort_flag, s.err, 5);
        ++nq;
        for (int i = 0; i <= tiles && ok; ++i) {
          for (int m = 0; m < 2 && ok; ++m) {
            const uint32_t ts = tmem + m * 128, to = tmem + 256 + m * DV;
            if (i) {  // O = P V of the tile before
              ok = mma_wait(p_full + m, (nt + i - 1) & 1, abort_flag, s.err, 6);
              // the small products of both halves first: truncation then takes from small sums
              const int u = nv + 2 * (i - 1), slots[2] = {u % C::RING, (u + 1) % C::RING};
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                ok = ok && mma_wait(v_full + slots[hf], ((u + hf) / C::RING) & 1, abort_flag, s.err, 7);
                if (!ok) break;
                fence_after();
                const uint32_t vh = sv + slots[hf] * C::VSLOT, vl = vh + (DV / 64) * C::VBLK;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const uint32_t ph = ts + (hf * 4 + k) * 16;
                  mma_ts(to, ph, ndesc(vl, k, C::VBLK), id_o, (hf || k) ? 1u : 0u, one);
                  mma_ts(to, ph + 8, ndesc(vh, k, C::VBLK), id_o, 1u, one);
                }
              }
              if (!ok) break;
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const uint32_t vh = sv + slots[hf] * C::VSLOT;
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_ts(to, ts + (hf * 4 + k) * 16, ndesc(vh, k, C::VBLK), id_o, 1u, one);
                if (m) mma_commit(v_empty + slots[hf], one);
              }
              mma_commit(o_full + m, one);
            }
            if (i < tiles && ok) {
              ok = mma_wait(k_full + m, (nt + i) & 1, abort_flag, s.err, 8);
              if (!ok) break;
              fence_after();
              const uint32_t qh = sq + m * C::QK, ql = qh + C::HALF, kh = sk + m * C::QK, kl = kh + C::HALF;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < slices) {
                  mma_ss(ts, kdesc(qh, k), kdesc(kl, k), id_s, k ? 1u : 0u, one);
                  mma_ss(ts, kdesc(ql, k), kdesc(kh, k), id_s, 1u, one);
                }
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < slices) mma_ss(ts, kdesc(qh, k), kdesc(kh, k), id_s, 1u, one);
              mma_commit(k_empty + m, one);
              mma_commit(s_full + m, one);
              if (m && i == tiles - 1) mma_commit(q_empty, one);
            }
          }
        }
        nt += tiles;
        nv += 2 * tiles;
      }
      if (any) {
        mma_commit(all_done, one);  // all products of this CTA
        bar_drain(all_done, 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int m = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, quad = warp & 3, r = quad * 32 + lane;
    constexpr int DH = DV / 2;  // output columns of this thread
    const uint32_t lane_row = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + m * 128 + 64 * half + lane_row, to = tmem + 256 + m * DV + half * DH + lane_row;
    float *mine = swap + (2 * m + half) * 128 + r, *other = swap + (2 * m + (half ^ 1)) * 128 + r;
    // the two warps of a map's rows; the four warps of both maps' rows
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * m + quad) : "memory"); };
    auto quad_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(9 + quad) : "memory"); };
    // P = 2^(S - ref): the reference is kCarry below the row's maximum when it is set, so that fp16
    // tails hold, and follows only when the maximum has outgrown it by kSlack more (fp16 ends at 2^16)
    constexpr float kCarry = 8.f, kSlack = 6.f;
    constexpr uint32_t kGone = 0x7fc0dead;  // in a maximum's place: this warp gave up (no product has these bits)
    uint64_t acc[DH / 2];
    auto add_tile = [&](float g) {  // acc += g O
      const uint64_t g2 = two(g, g);
#pragma unroll
      for (int c = 0; c < DH / 16; ++c) {
        uint32_t y[16];
        tld16_issue(to + 16 * c, y);
        tld_wait();
        after_wait(y);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[8 * c + j] = fma2(two(y[2 * j], y[2 * j + 1]), g2, acc[8 * c + j]);
      }
    };
    // The loops over a tile's columns stay rolled: the warps of a scheduler run them at different
    // places, and unrolled they wait for instructions more than for anything else.
    auto mask = [&](uint32_t (&y)[16], int left) {  // columns from `left` on are not seen
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j >= left) y[j] = 0xff800000u;  // -inf
    };
    int nt = 0;  // tiles so far
    // Named barriers have no limit: every warp passes the same ones for every item, whatever its waits
    // said (after a wait has run out they all return at once).
    for (int round = 0; round < rounds; ++round) {
      unsigned index;
      if (!item_of_round(items, round, index)) continue;
      const Item w = item_at<PACK>(s, x, o, index);
      const int tiles = w.tiles;
      if (threadIdx.x == 128 && w.h == 0 && w.qt == 0 && w.split == 0) report_length(s, w.b);
      // this thread's row is query row / P of the head w.h * P + row % P
      const int rows = (int)s.T * P, row = w.r0 + r;
      const int at_row = row < rows ? row : rows - 1;
      const int seen = (int)s.seen(PACK ? at_row / P : at_row, w.n) - w.tile0 * 128 - 64 * half;
      const float fq = x.fq[(int64_t)(w.b * 2 * row_heads + 2 * w.h + m) * x.qt + w.qt];
      const float *fk = x.fk + (int64_t)(w.b * 2 * s.Hk + 2 * w.hk + m) * x.kt + w.tile0;
      const float *fv = x.fv + (int64_t)(w.b * s.Hk + w.hk) * x.kt + w.tile0;
      float ref = -INFINITY, top = -INFINITY;  // top: the maximum that ref was set by
      uint64_t sum2[2] = {two(0.f, 0.f), two(0.f, 0.f)};
#pragma unroll
      for (int j = 0; j < DH / 2; ++j) acc[j] = two(0.f, 0.f);
      bool ok = true;
      float gv = 0.f;
      for (int i = 0; i < tiles; ++i) {
        const float f = factor2(fq, fk[i]), next_gv = fv[i];
        if (i) {  // the last tile's product, while the tensor core works on this tile's scores
          ok = __all_sync(0xffffffffu, bar_wait(o_full + m, (nt + i - 1) & 1, abort_flag, s.err, 9));
          fence_after();
          if (ok) add_tile(gv);
        }
        ok = ok && __all_sync(0xffffffffu, bar_wait(s_full + m, (nt + i) & 1, abort_flag, s.err, 10));
        const int left = seen - i * 128;
        const int lim = left < 0 ? 0 : left > 64 ? 64 : left;
        const bool whole = __all_sync(0xffffffffu, lim == 64);
        float mx = -INFINITY;
        fence_after();
        if (ok) {
          float mx2[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t y[16];
            tld16_issue(ts + 16 * c, y);
            tld_wait();
            after_wait(y);
            if (!whole) mask(y, lim - 16 * c);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              mx2[j & 1] = max3(mx2[j & 1], __uint_as_float(y[2 * j]), __uint_as_float(y[2 * j + 1]));
          }
          mx = fmaxf(mx2[0], mx2[1]) * f;
        }
        // a pair leaves the loop together, or one of them would wait for the other without a limit
        *mine = ok ? mx : __uint_as_float(kGone);
        pair_sync();
        const float theirs = *other;
        ok = ok && !__any_sync(0xffffffffu, __float_as_uint(theirs) == kGone);
        if (!ok) break;
        mx = fmaxf(mx, theirs);
        gv = next_gv;
        if (__any_sync(0xffffffffu, mx > top + kSlack || (top == -INFINITY && mx > top))) {
          const float now = fmaxf(top, mx);
          const float shrink = top == -INFINITY ? 0.f : ex2(top - now);
          const uint64_t s2 = two(shrink, shrink);
          top = now;
          ref = now - kCarry;
          sum2[0] = mul2(sum2[0], s2);
          sum2[1] = mul2(sum2[1], s2);
#pragma unroll
          for (int j = 0; j < DH / 2; ++j) acc[j] = mul2(acc[j], s2);
        }
        const float at = top == -INFINITY ? 0.f : ref;  // no key yet: all weights are 2^-inf
        const uint64_t f2 = two(f, f), at2 = two(-at, -at);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t y[16], hi[8], lo[8];
          tld16_issue(ts + 16 * c, y);
          tld_wait();
          after_wait(y);
          if (!whole) mask(y, lim - 16 * c);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float a, d;
            untwo(fma2(two(y[2 * j], y[2 * j + 1]), f2, at2), a, d);
            const uint64_t p = two(ex2(a), ex2(d));
            sum2[j & 1] = add2(sum2[j & 1], p);
            cut2(p, hi[j], lo[j]);
          }
          tst_pairs(ts + 16 * c, hi, lo);
        }
        tst_wait();
        fence_before();
        bar_arrive(p_full + m);
      }
      nt += tiles;
      if (tiles) ok = __all_sync(0xffffffffu, ok && bar_wait(o_full + m, (nt - 1) & 1, abort_flag, s.err, 11));
      fence_after();
      if (tiles && ok) add_tile(gv);
      float s0, s1, s2, s3;
      untwo(sum2[0], s0, s1);
      untwo(sum2[1], s2, s3);
      const float part = (s0 + s1) + (s2 + s3);
      const int t = PACK ? row / P : row, h = PACK ? w.h * P + (row - t * P) : w.h;
      pair_sync();  // both have read the last maxima
      *mine = part;
      pair_sync();
      const float sum = half ? *other + part : part + *other;
      const bool none = top == -INFINITY, live = row < rows && ok;
      const bool parts = o.parts.splits > 1;
      const float inv = parts ? 1.f : none ? 0.f : 1.0f / sum;
      const int64_t at0 = (int64_t)(w.b * s.Hk + w.hk) * s.T * s.G + (PACK ? 0 : h - w.hk * s.G);  // row 0
      const int next = PACK ? 1 : s.G;
      if (live && parts && half == 0)
        o.parts.ml[((at0 + (int64_t)row * next) * 2 + m) * o.parts.splits + w.split] = make_float2(none ? -INFINITY : ref, sum);
      if (live && !parts && o.lse && half == 0)
        o.lse[(int64_t)(w.b * 2 * s.H + 2 * h + m) * s.T + t] = none ? INFINITY : ref + log2f(sum);
      const uint64_t inv2 = two(inv, inv);
#pragma unroll
      for (int j = 0; j < DH / 2; ++j) acc[j] = mul2(acc[j], inv2);
      // map 2's rows to map 1's warps, over its own products in TMEM
      if (m && !parts) {
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
          uint32_t y[2][8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float a, d;
            untwo(acc[8 * c + j], a, d);
            y[j >> 2][2 * (j & 3)] = __float_as_uint(a);
            y[j >> 2][2 * (j & 3) + 1] = __float_as_uint(d);
          }
          tst_pairs(to + 16 * c, y[0], y[1]);
        }
        tst_wait();
        fence_before();
      }
      quad_sync();
      if (!m && !parts) {
        const float lam = __ldg(s.lam + h);
        const uint64_t nl2 = two(-lam, -lam);
        fence_after();
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
          uint32_t y[16];
          tld16_issue(to + DV + 16 * c, y);
          tld_wait();
          after_wait(y);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[8 * c + j] = fma2(two(y[2 * j], y[2 * j + 1]), nl2, acc[8 * c + j]);
        }
      }
      // the value ring is free once the other map's last product is done too
      if (tiles) ok = __all_sync(0xffffffffu, ok && bar_wait(o_full + (m ^ 1), (nt - 1) & 1, abort_flag, s.err, 12));
      float *dst = parts ? o.parts.o : m ? o.out2 : o.out;
      if (ok && dst) {
        constexpr int CW = C::CW, CH = CW / 4;  // columns and 16-byte chunks of a staged row
        float4 *box = reinterpret_cast<float4 *>(sm + 4 * C::QK + (warp - 4) * (32 * CW * 4));
        auto place = [&](int i, int c) { return box + i * CH + (c ^ (CH == 8 ? i & 7 : i >> 1 & 3)); };
        const bool four = (s.dv & 3) == 0 && ((uintptr_t)dst & 15) == 0;
        // partial rows follow one another, a packed tile's output rows go P heads a token
        const int64_t stride = parts ? (int64_t)2 * next * o.parts.splits * s.dv : (int64_t)s.H * s.dv;
        const bool turns = PACK && !parts;
        float *base = parts ? dst + ((at0 * 2 + m) * o.parts.splits + w.split) * s.dv
                            : dst + ((int64_t)w.b * s.T * s.H + w.h * P) * s.dv;
        const int row0 = w.r0 + quad * 32;
        if (!turns) base += row0 * stride;
        auto row_at = [&](int i) {
          return turns ? base + (row0 + i) / P * stride + (row0 + i) % P * s.dv : base + i * stride;
        };
#pragma unroll
        for (int c0 = 0; c0 < DH / CW; ++c0) {
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            float4 v;
            untwo(acc[c0 * (CW / 2) + 2 * c], v.x, v.y);
            untwo(acc[c0 * (CW / 2) + 2 * c + 1], v.z, v.w);
            *place(lane, c) = v;
          }
          __syncwarp();
          const int c = lane % CH;
#pragma unroll
          for (int k = 0; k < CH; ++k) {
            const int i = k * (32 / CH) + lane / CH;
            if (row0 + i < rows) store4(row_at(i), half * DH + c0 * CW + 4 * c, *place(i, c), s.dv, four);
          }
          __syncwarp();
        }
      }
      // copies write the ring next, and behind them products what was read of TMEM
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      fence_before();
      bar_arrive(staged);
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
int launch(tx_ctx *ctx, const Shape &s, const Split &x, const Out &o) {
  CUtensorMap mq, mk, mv;
  if (!split_map(&mq, x.q, 64, s.rows(), s.B * 2 * s.row_heads()) || !split_map(&mk, x.k, 64, s.S, s.B * 2 * s.Hk) ||
      !split_map(&mv, x.v, DV, s.S, s.B * s.Hk))
    return tx_fail(ctx, TX_ERR_UNSUPPORTED, "differential attention: tensor map");
  static SmemGrant granted;
  TX_TRY(granted.take(ctx, (const void *)k_diff_fwd<DV, PACK>, Cfg<DV>::SMEM));
  const int64_t items = x.qt * s.B * s.row_heads() * o.parts.splits;
  const unsigned blocks = (unsigned)(items < ctx->num_sms ? items : ctx->num_sms);
  return launch_behind(ctx, "k_diff_fwd", k_diff_fwd<DV, PACK>, blocks, kThreads, Cfg<DV>::SMEM, s, x, mq, mk, mv, o);
}

}  // namespace

int tc_forward_splits(tx_ctx *ctx, const Shape &s) {
  // Too few query tiles for the SMs: the keys are shared out too, one range a block, where the tiles of keys
  // that a block is spared (3.4 us each) are worth the join (4 us and 1 us for 1600 rows and heads).
  const int64_t blocks = (s.rows() + kRows - 1) / kRows * s.B * s.row_heads(), tiles = (s.S + kRows - 1) / kRows;
  int64_t splits = blocks ? ctx->num_sms / blocks : 1;
  if (splits < 2) return 1;
  const int64_t per = (tiles + splits - 1) / splits;
  splits = (tiles + per - 1) / per;
  const double spared = 3.4 * (double)(tiles - per), join = 4.0 + (double)(s.B * s.T * s.H) / 1600.0;
  return spared > join ? (int)splits : 1;
}

int tc_forward(tx_ctx *ctx, const Shape &s, const Split &x, float *out, float *out2, float *lse, const Parts &parts) {
  const int64_t tiles = (s.S + kRows - 1) / kRows;
  const Out o{out, out2, lse, parts, (int)((tiles + parts.splits - 1) / parts.splits)};
  if (s.P > 1) return x.vw == 64 ? launch<64, true>(ctx, s, x, o) : launch<128, true>(ctx, s, x, o);
  return x.vw == 64 ? launch<64, false>(ctx, s, x, o) : launch<128, false>(ctx, s, x, o);
}

}  // namespace tx_diff
