// Differential attention: out = A1 v - lam A2 v with A_m = softmax(scale q_m k_m^T).
//
// With D_m = rowsum(dO * O_m) (O_m = A_m v) and dP = dO v^T the gradients are
//   dS1 = A1 (dP - D1) scale,  dS2 = -lam A2 (dP - D2) scale,
//   dq_m = dS_m k_m,  dk_m = dS_m^T q_m,  dv = (A1 - lam A2)^T dO,  dlam = -sum D2,
// and A_m comes back from the saved log-sum-exp without a second softmax pass.
// Statistics, sums and accumulators are fp32.
#include <cmath>
#include <mutex>

#include "diff_attn.cuh"

namespace tx_diff {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A block splits one tile of 128 rows of one head; blockIdx.z picks the tensor.
struct SplitJob {
  const float *src;
  __half *dst;
  float *f, *norm;  // norm: nullptr where it is not needed
  int64_t N, tiles;  // rows and tiles of a head
  int heads, w;
  float factor;
  int masked;  // rows behind the sequence's length become zeros
};
struct SplitJobs {
  SplitJob j[4];
  // with the output's gradient (job 3) its rows' D1 = dO . (out + lam out2) and D2 = dO . out2 go to
  // stats, beside lse, and each tile's sum of D2 to sums
  const float *out, *out2, *lse;
  float *stats, *sums;
};
constexpr int kSplitThreads = 512, kSplitWarps = kSplitThreads / 32;
template <int W, bool STATS>
__device__ __forceinline__ void split_tile(const Shape &s, const SplitJobs &jobs, const SplitJob &J, uint32_t *red) {
  constexpr int PARTS = W / 8, ROWS = kSplitThreads / PARTS, UNITS = kRows / ROWS;  // 8 elements a thread and unit
  const int64_t head = (int64_t)blockIdx.x / J.tiles, tile = (int64_t)blockIdx.x - head * J.tiles;
  const int64_t b = head / J.heads, n0 = tile * kRows;
  const int hh = (int)(head - b * J.heads), c = threadIdx.x % PARTS * 8, r0 = threadIdx.x / PARTS;
  const int64_t n_end = J.masked ? s.length(b) : J.N;
  const bool four = (J.w & 3) == 0 && ((uintptr_t)J.src & 15) == 0;
  float x[UNITS][8];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t n = n0 + r0 + u * ROWS;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
    if (n < n_end) {
      const float *src = J.src + ((b * J.N + n) * J.heads + hh) * J.w + c;
      if (four) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (c + 4 * i < J.w) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(src) + i);
            x[u][4 * i] = v.x, x[u][4 * i + 1] = v.y, x[u][4 * i + 2] = v.z, x[u][4 * i + 3] = v.w;
          }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < J.w) x[u][i] = __ldg(src + i);
      }
    }
  }
  if (STATS) {
    const float lam = __ldg(s.lam + hh);
    const int64_t steps = (J.N + 63) / 64;
    float total = 0.f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t n = n0 + r0 + u * ROWS, at = ((b * J.N + n) * J.heads + hh) * J.w + c;
      float d1 = 0.f, d2 = 0.f;
      if (n < J.N) {
        auto add = [&](float g, float y, float y2) {
          d1 += g * (y + lam * y2);
          d2 += g * y2;
        };
        if (four && ((uintptr_t)jobs.out & 15) == 0 && ((uintptr_t)jobs.out2 & 15) == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (c + 4 * i < J.w) {
              const float4 y = __ldg(reinterpret_cast<const float4 *>(jobs.out + at) + i);
              const float4 z = __ldg(reinterpret_cast<const float4 *>(jobs.out2 + at) + i);
              add(x[u][4 * i], y.x, z.x), add(x[u][4 * i + 1], y.y, z.y);
              add(x[u][4 * i + 2], y.z, z.z), add(x[u][4 * i + 3], y.w, z.w);
            }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < J.w) add(x[u][i], __ldg(jobs.out + at + i), __ldg(jobs.out2 + at + i));
        }
      }
#pragma unroll
      for (int o = PARTS / 2; o; o >>= 1) {
        d1 += __shfl_xor_sync(0xffffffffu, d1, o);
        d2 += __shfl_xor_sync(0xffffffffu, d2, o);
      }
      if (c == 0 && n / 64 < steps) {  // rows behind the last up to a step's end too
        float *to = jobs.stats + (head * steps + n / 64) * 256 + n % 64;
        const bool live = n < J.N;
        to[0] = live ? __ldg(jobs.lse + (b * 2 * s.H + 2 * hh) * J.N + n) : INFINITY;
        to[64] = live ? __ldg(jobs.lse + (b * 2 * s.H + 2 * hh + 1) * J.N + n) : INFINITY;
        to[128] = d1;
        to[192] = d2;
        total += d2;
      }
    }
    total = warp_sum(total);
    if ((threadIdx.x & 31) == 0) red[2 * kSplitWarps + (threadIdx.x >> 5)] = __float_as_uint(total);
  }
  // the tile's largest finite magnitude (and row norm)
  uint32_t top = 0;
  float norm = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[u][i] *= J.factor;
      const uint32_t a = __float_as_uint(x[u][i]) & 0x7fffffffu;
      if (a < 0x7f800000u && a > top) top = a;
      ss += x[u][i] * x[u][i];
    }
    if (J.norm) {
#pragma unroll
      for (int o = PARTS / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      norm = fmaxf(norm, ss);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const uint32_t nb = __reduce_max_sync(0xffffffffu, __float_as_uint(norm));
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = top;
    red[kSplitWarps + (threadIdx.x >> 5)] = nb;
  }
  __syncthreads();
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kSplitWarps; ++i) {
    top = red[i] > top ? red[i] : top;
    most = red[kSplitWarps + i] > most ? red[kSplitWarps + i] : most;
  }
  int e = (int)(top >> 23) - 127 - 13;
  e = e < -113 ? -113 : e > 114 ? 114 : e;
  if (threadIdx.x == 0) {
    J.f[blockIdx.x] = __uint_as_float((uint32_t)(127 + e) << 23);
    if (J.norm) J.norm[blockIdx.x] = fminf(sqrtf(__uint_as_float(most)), 1e16f);
    if (STATS) {
      float total = 0.f;
      for (int i = 0; i < kSplitWarps; ++i) total += __uint_as_float(red[2 * kSplitWarps + i]);
      jobs.sums[blockIdx.x] = total;
    }
  }
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t n = n0 + r0 + u * ROWS;
    if (n >= J.N) break;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split2(x[u][2 * i] * inv, x[u][2 * i + 1] * inv, hi[i], lo[i]);
    __half *dst = J.dst + (head * J.N + n) * (2 * W) + c;
    *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4 *>(dst + W) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}
// W: the values' width (queries and keys have 64); GRAD: the output's gradient alone
template <int W, bool GRAD>
__global__ void __launch_bounds__(kSplitThreads, 2)
    k_diff_split(const __grid_constant__ Shape s, const __grid_constant__ SplitJobs jobs) {
  __shared__ uint32_t red[3 * kSplitWarps];
  const SplitJob &J = jobs.j[GRAD ? 3 : blockIdx.z];
  if ((int64_t)blockIdx.x >= s.B * J.heads * J.tiles) return;
  if (GRAD)
    split_tile<W, true>(s, jobs, J, red);
  else if (blockIdx.z < 2)
    split_tile<64, false>(s, jobs, J, red);
  else
    split_tile<W, false>(s, jobs, J, red);
}

// ---- few query rows against many keys ----------------------------------------------------
// A block takes RP queries (token, head of the group) of one key head, both maps, and a range
// of keys, in tiles of 64: a thread works out a key's dots with all its map's rows, a warp the
// running maximum and sum of a row, a thread one column of all the rows' outputs.
constexpr int kTile = 64, kRowThreads = 128, kKeyLd = 132;

template <int RP>
__global__ void __launch_bounds__(kRowThreads)
    k_diff_rows(const __grid_constant__ Shape s, int splits, int64_t keys_per_split, float *part_o, float2 *part_ml) {
  extern __shared__ float4 smem4[];
  float *ks = reinterpret_cast<float *>(smem4);       // [64][132]: map 0, map 1
  float *vs = ks + kTile * kKeyLd;                    // [64][128]
  float *qs = vs + kTile * kMaxVdim;                  // [2 RP][64]
  float *ps = qs + 2 * RP * kMaxDim;                  // [64][2 RP]
  float *al = ps + kTile * 2 * RP;                    // [2 RP]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t b = blockIdx.y / s.Hk;
  const int hk = (int)(blockIdx.y - b * s.Hk);
  const int64_t n_items = s.T * s.G, item0 = (int64_t)blockIdx.z * RP;
  const int64_t n = s.length(b);
  if (tid == 0 && hk == 0 && blockIdx.x == 0 && blockIdx.z == 0) report_length(s, b);
  const int64_t last = item0 + RP <= n_items ? item0 + RP - 1 : n_items - 1;
  const int64_t k0 = (int64_t)blockIdx.x * keys_per_split;
  int64_t k1 = s.seen(last / s.G, n);
  if (k1 > k0 + keys_per_split) k1 = k0 + keys_per_split;

  for (int i = tid; i < 2 * RP * kMaxDim; i += kRowThreads) {
    const int c = i % kMaxDim, row = i / kMaxDim, m = row % 2;
    const int64_t item = item0 + row / 2;
    float x = 0.f;
    if (item < n_items && c < s.d) {
      const int64_t t = item / s.G;
      const int h = hk * s.G + (int)(item - t * s.G);
      x = s.q[((b * s.T + t) * (2 * s.H) + 2 * h + m) * s.d + c] * (s.scale * kLog2e);
    }
    qs[i] = x;
  }
  float acc[2 * RP], mx[(2 * RP + 3) / 4], sum[(2 * RP + 3) / 4];
#pragma unroll
  for (int r = 0; r < 2 * RP; ++r) acc[r] = 0.f;
#pragma unroll
  for (int i = 0; i < (2 * RP + 3) / 4; ++i) mx[i] = -INFINITY, sum[i] = 0.f;

  for (int64_t j0 = k0; j0 < k1; j0 += kTile) {
    __syncthreads();
    for (int i = tid; i < kTile * 2 * kMaxDim; i += kRowThreads) {
      const int c = i % kMaxDim, m = (i / kMaxDim) % 2, j = i / (2 * kMaxDim);
      ks[j * kKeyLd + m * kMaxDim + c] =
          (j0 + j < k1 && c < s.d) ? s.k[((b * s.S + j0 + j) * (2 * s.Hk) + 2 * hk + m) * s.d + c] : 0.f;
    }
    for (int i = tid; i < kTile * kMaxVdim; i += kRowThreads) {
      const int c = i % kMaxVdim, j = i / kMaxVdim;
      vs[i] = (j0 + j < k1 && c < s.dv) ? s.v[((b * s.S + j0 + j) * s.Hk + hk) * s.dv + c] : 0.f;
    }
    __syncthreads();
    {
      const int j = tid & 63, m = tid >> 6;
      float dot[RP];
#pragma unroll
      for (int r = 0; r < RP; ++r) dot[r] = 0.f;
      for (int c = 0; c < kMaxDim; c += 4) {
        const float4 kk = *reinterpret_cast<const float4 *>(ks + j * kKeyLd + m * kMaxDim + c);
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float4 qq = *reinterpret_cast<const float4 *>(qs + (2 * r + m) * kMaxDim + c);
          dot[r] += kk.x * qq.x + kk.y * qq.y + kk.z * qq.z + kk.w * qq.w;
        }
      }
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        const int64_t item = item0 + r;
        const bool ok = item < n_items && j0 + j < k1 && j0 + j < s.seen(item / s.G, n);
        ps[j * 2 * RP + 2 * r + m] = ok ? dot[r] : -INFINITY;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (2 * RP + 3) / 4; ++i) {
      const int r = i * 4 + warp;
      if (r < 2 * RP) {
        const float a = ps[lane * 2 * RP + r], c = ps[(lane + 32) * 2 * RP + r];
        const float m = fmaxf(mx[i], warp_max(fmaxf(a, c)));
        const float at = m == -INFINITY ? 0.f : m;  // no key yet: all weights are exp2(-inf) = 0
        const float pa = exp2f(a - at), pc = exp2f(c - at), f = exp2f(mx[i] - at);
        ps[lane * 2 * RP + r] = pa;
        ps[(lane + 32) * 2 * RP + r] = pc;
        sum[i] = sum[i] * f + warp_sum(pa + pc);
        mx[i] = m;
        if (lane == 0) al[r] = f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2 * RP; ++r) acc[r] *= al[r];
    for (int j = 0; j < kTile; ++j) {
      const float x = vs[j * kMaxVdim + tid];
#pragma unroll
      for (int r = 0; r < 2 * RP; ++r) acc[r] += ps[j * 2 * RP + r] * x;
    }
  }
  // partial rows: [b][hk][item][map] x [split]
#pragma unroll
  for (int i = 0; i < (2 * RP + 3) / 4; ++i) {
    const int r = i * 4 + warp;
    const int64_t item = item0 + r / 2;
    if (r < 2 * RP && lane == 0 && item < n_items)
      part_ml[(((b * s.Hk + hk) * n_items + item) * 2 + (r & 1)) * splits + blockIdx.x] = make_float2(mx[i], sum[i]);
  }
#pragma unroll
  for (int r = 0; r < 2 * RP; ++r) {
    const int64_t item = item0 + r / 2;
    if (item < n_items && tid < s.dv)
      part_o[((((b * s.Hk + hk) * n_items + item) * 2 + (r & 1)) * splits + blockIdx.x) * s.dv + tid] = acc[r];
  }
}

// out, out2 and lse from the splits' partial rows: a block per query and head.
__global__ void __launch_bounds__(kMaxVdim)
    k_diff_join(const __grid_constant__ Shape s, int splits, const float *part_o, const float2 *part_ml, float *out,
                float *out2, float *lse) {
  const int64_t n_items = s.T * s.G;
  const int64_t at = blockIdx.x;  // (b, hk, item)
  const int64_t item = at % n_items, bh = at / n_items;
  const int64_t b = bh / s.Hk, t = item / s.G;
  const int hk = (int)(bh - b * s.Hk), h = hk * s.G + (int)(item - t * s.G);
  const int c = threadIdx.x;
  float o[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float2 *ml = part_ml + (at * 2 + m) * splits;
    float top = -INFINITY;
    for (int i = 0; i < splits; ++i) top = fmaxf(top, ml[i].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f;
    for (int i = 0; i < splits; ++i) {
      const float2 p = ml[i];
      const float w = exp2f(p.x - ref);
      sum += p.y * w;
      if (c < s.dv && w != 0.f) x += part_o[((at * 2 + m) * splits + i) * s.dv + c] * w;
    }
    const bool none = top == -INFINITY;
    o[m] = none ? 0.f : x / sum;
    if (lse && c == 0) lse[(b * 2 * s.H + 2 * h + m) * s.T + t] = none ? INFINITY : ref + log2f(sum);
  }
  if (c < s.dv) {
    const int64_t i = ((b * s.T + t) * s.H + h) * s.dv + c;
    out[i] = o[0] - __ldg(s.lam + h) * o[1];
    if (out2) out2[i] = o[1];
  }
}

// dlam = -sum of D2, from the tiles' sums
__global__ void __launch_bounds__(256) k_diff_dlam(const __grid_constant__ Shape s, const float *sums, int64_t tiles,
                                                   float *dlam) {
  __shared__ float part[8];
  const int h = blockIdx.x;
  float v = 0.f;
  for (int64_t i = threadIdx.x; i < s.B * tiles; i += 256) {
    const int64_t b = i / tiles;
    v += sums[(b * s.H + h) * tiles + (i - b * tiles)];
  }
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) v += part[i];
    dlam[h] = -v;
  }
}

// ---- host ----------------------------------------------------------------------------------
// The split operands of one call and their memory.
struct Operands {
  Split x;
  Scratch data;
  int64_t tq = 0, tk = 0, tv = 0, tg = 0;  // tiles
  static int width(const Shape &s) { return s.dv <= 64 ? 64 : 128; }
  static size_t total(const Shape &s, bool gradient) {
    const int64_t w = width(s), qt = (s.T + kRows - 1) / kRows, kt = (s.S + kRows - 1) / kRows;
    const int64_t halves = 2 * (s.B * 2 * s.H * s.T * 64 + s.B * 2 * s.Hk * s.S * 64 + s.B * s.Hk * s.S * w +
                                (gradient ? s.B * s.H * s.T * w : 0));
    return (size_t)halves * 2 + (size_t)(s.B * (2 * s.H * qt + 2 * s.Hk * kt + 2 * s.Hk * kt + 2 * s.H * qt)) * 4;
  }
  Operands(tx_ctx *ctx, const Shape &s, bool gradient) : data(ctx, total(s, gradient)) {
    if (!data.ptr) return;
    const int64_t w = width(s), qt = (s.T + kRows - 1) / kRows, kt = (s.S + kRows - 1) / kRows;
    x.vw = (int)w;
    x.qt = qt;
    x.kt = kt;
    tq = s.B * 2 * s.H * qt, tk = s.B * 2 * s.Hk * kt, tv = s.B * s.Hk * kt, tg = s.B * s.H * qt;
    __half *p = data.as<__half>();
    x.q = p, p += s.B * 2 * s.H * s.T * 128;
    x.k = p, p += s.B * 2 * s.Hk * s.S * 128;
    x.v = p, p += s.B * s.Hk * s.S * 2 * w;
    x.g = p, p += gradient ? s.B * s.H * s.T * 2 * w : 0;
    float *f = reinterpret_cast<float *>(p);
    x.fq = f, f += tq;
    x.fk = f, f += tk;
    x.fv = f, f += tv;
    x.nv = f, f += tv;
    x.fg = f, f += tg;
    x.ng = f;
  }
  // p: the backward's description, or null
  int fill(tx_ctx *ctx, const Shape &s, const tx_diff_attention *p, float *stats, float *sums) {
    if (!data.ptr) return TX_ERR_OOM;
    const float *dout = p ? p->dout : nullptr;
    auto w = [](const float *p) { return const_cast<float *>(p); };
    SplitJobs jobs{};
    jobs.j[0] = SplitJob{s.q, x.q, w(x.fq), nullptr, s.T, x.qt, 2 * s.H, s.d, s.scale * kLog2e, 0};
    jobs.j[1] = SplitJob{s.k, x.k, w(x.fk), nullptr, s.S, x.kt, 2 * s.Hk, s.d, 1.0f, 1};
    jobs.j[2] = SplitJob{s.v, x.v, w(x.fv), w(x.nv), s.S, x.kt, s.Hk, s.dv, 1.0f, 1};
    jobs.j[3] = SplitJob{dout, x.g, w(x.fg), w(x.ng), s.T, x.qt, s.H, s.dv, 1.0f, 0};
    if (p) jobs.out = p->out, jobs.out2 = p->out2, jobs.lse = p->lse, jobs.stats = stats, jobs.sums = sums;
    const int64_t blocks = tq > tk ? tq : tk;
    const dim3 grid((unsigned)blocks, 1, 3);
    if (x.vw == 64)
      k_diff_split<64, false><<<grid, kSplitThreads, 0, ctx->stream>>>(s, jobs);
    else
      k_diff_split<128, false><<<grid, kSplitThreads, 0, ctx->stream>>>(s, jobs);
    TX_LAUNCHED(ctx, "k_diff_split");
    if (!p) return TX_OK;
    if (x.vw == 64)
      k_diff_split<64, true><<<(unsigned)tg, kSplitThreads, 0, ctx->stream>>>(s, jobs);
    else
      k_diff_split<128, true><<<(unsigned)tg, kSplitThreads, 0, ctx->stream>>>(s, jobs);
    TX_LAUNCHED(ctx, "k_diff_split (gradient)");
    return TX_OK;
  }
};

int check_desc(tx_ctx *ctx, const tx_diff_attention *p, Shape &s) {
  if (!p) return tx_fail(ctx, TX_ERR_INVALID, "differential attention: no description");
  if (p->dim < 1 || p->dim > kMaxDim || p->vdim < 1 || p->vdim > kMaxVdim)
    return tx_fail(ctx, TX_ERR_UNSUPPORTED, "differential attention: head dimension 1..64, value dimension 1..128");
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->heads > 32767)
    return tx_fail(ctx, TX_ERR_SHAPE, "differential attention: the query heads must be a multiple of the key heads");
  const int64_t most = (int64_t)1 << 30;
  if (p->batch < 0 || p->queries < 0 || p->keys < 0 || p->batch > most || p->queries > most || p->keys > most ||
      p->query_start > most || p->query_start < -most || (p->batch && p->heads > 65535 / p->batch) ||
      (p->batch && (p->queries > most / p->batch || p->keys > most / p->batch)))
    return tx_fail(ctx, TX_ERR_SHAPE, "differential attention: batch * heads up to 65535, lengths below 2^30 in all");
  if (!std::isfinite(p->scale)) return tx_fail(ctx, TX_ERR_INVALID, "differential attention: scale");
  s = Shape{p->batch, p->queries, p->keys, (int)p->heads, (int)p->kv_heads, (int)(p->heads / p->kv_heads), (int)p->dim,
            (int)p->vdim, p->q, p->k, p->v, p->lam, p->key_lengths, p->causal ? 1 : 0, p->query_start, p->scale,
            ctx->d_err};
  return TX_OK;
}

int join(tx_ctx *ctx, const Shape &s, const Parts &parts, float *out, float *out2, float *lse) {
  k_diff_join<<<(unsigned)(s.B * s.T * s.H), kMaxVdim, 0, ctx->stream>>>(s, parts.splits, parts.o, parts.ml, out, out2,
                                                                       lse);
  TX_LAUNCHED(ctx, "k_diff_join");
  return TX_OK;
}

template <int RP>
int launch_rows(tx_ctx *ctx, const Shape &s, float *out, float *out2, float *lse) {
  const int64_t items = s.T * s.G, chunks = (items + RP - 1) / RP;
  if (chunks > 65535) return tx_fail(ctx, TX_ERR_SHAPE, "differential attention: too many queries");
  const int64_t blocks = chunks * s.B * s.Hk;
  int64_t splits = (2 * ctx->num_sms + blocks - 1) / blocks, tiles = (s.S + kTile - 1) / kTile;
  if (splits > tiles) splits = tiles;
  if (splits < 1) splits = 1;
  int64_t per = ((tiles + splits - 1) / splits) * kTile;
  if (per < kTile) per = kTile;
  const int64_t rows = s.B * s.Hk * items * 2;
  Scratch po(ctx, (size_t)(rows * splits * s.dv) * 4), pm(ctx, (size_t)(rows * splits) * 8);
  if (!po.ptr || !pm.ptr) return TX_ERR_OOM;
  const int smem = (kTile * kKeyLd + kTile * kMaxVdim + 2 * RP * kMaxDim + kTile * 2 * RP + 2 * RP) * 4;
  TX_CUDA(ctx, cudaFuncSetAttribute(k_diff_rows<RP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  k_diff_rows<RP><<<dim3((unsigned)splits, (unsigned)(s.B * s.Hk), (unsigned)chunks), kRowThreads, smem, ctx->stream>>>(
      s, (int)splits, per, po.as<float>(), pm.as<float2>());
  TX_LAUNCHED(ctx, "k_diff_rows");
  return join(ctx, s, Parts{po.as<float>(), pm.as<float2>(), (int)splits}, out, out2, lse);
}

}  // namespace

bool split_map(CUtensorMap *m, const __half *base, int w, int64_t rows, int64_t heads) {
  std::call_once(g_encode_once, [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
  });
  if (!g_encode) return false;
  cuuint64_t dims[3] = {(cuuint64_t)(2 * w), (cuuint64_t)rows, (cuuint64_t)heads};
  cuuint64_t strides[2] = {(cuuint64_t)(4 * w), (cuuint64_t)(4 * w) * (cuuint64_t)rows};
  cuuint32_t bx[3] = {64u, 64u, 1u};
  cuuint32_t es[3] = {1u, 1u, 1u};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void *)base, dims, strides, bx, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tx_diff

using namespace tx_diff;

extern "C" int tx_diff_attention_fwd(tx_ctx *ctx, const tx_diff_attention *p) {
  if (!ctx) return TX_ERR_INVALID;
  Shape s;
  TX_TRY(check_desc(ctx, p, s));
  if ((p->out2 == nullptr) != (p->lse == nullptr))
    return tx_fail(ctx, TX_ERR_INVALID, "differential attention: out2 and lse come together");
  if (s.B * s.T == 0) return TX_OK;
  if (!p->q || !p->lam || !p->out || (s.S && (!p->k || !p->v)))
    return tx_fail(ctx, TX_ERR_INVALID, "differential attention: null buffer");
  DeviceScope device(ctx);
  if (s.T * s.G <= 1) return launch_rows<1>(ctx, s, p->out, p->out2, p->lse);
  if (s.T * s.G <= 2) return launch_rows<2>(ctx, s, p->out, p->out2, p->lse);
  if (s.T * s.G <= 4) return launch_rows<4>(ctx, s, p->out, p->out2, p->lse);
  if (s.T * s.G <= 8 || s.S == 0) return launch_rows<8>(ctx, s, p->out, p->out2, p->lse);
  Operands x(ctx, s, false);
  TX_TRY(x.fill(ctx, s, nullptr, nullptr, nullptr));
  const int splits = tc_forward_splits(ctx, s);
  if (splits == 1) return tc_forward(ctx, s, x.x, p->out, p->out2, p->lse, Parts{nullptr, nullptr, 1});
  const int64_t rows = s.B * s.H * s.T * 2;
  Scratch po(ctx, (size_t)(rows * splits * s.dv) * 4), pm(ctx, (size_t)(rows * splits) * 8);
  if (!po.ptr || !pm.ptr) return TX_ERR_OOM;
  const Parts parts{po.as<float>(), pm.as<float2>(), splits};
  TX_TRY(tc_forward(ctx, s, x.x, p->out, p->out2, p->lse, parts));
  return join(ctx, s, parts, p->out, p->out2, p->lse);
}

extern "C" int tx_diff_attention_bwd(tx_ctx *ctx, const tx_diff_attention *p) {
  if (!ctx) return TX_ERR_INVALID;
  Shape s;
  TX_TRY(check_desc(ctx, p, s));
  if ((p->dk == nullptr) != (p->dv == nullptr))
    return tx_fail(ctx, TX_ERR_INVALID, "differential attention: dk and dv come together");
  const int64_t rows = s.B * s.T * s.H;
  if (rows && (!p->q || !p->lam || !p->out || !p->out2 || !p->lse || !p->dout || (s.S && (!p->k || !p->v))))
    return tx_fail(ctx, TX_ERR_INVALID, "differential attention: null buffer");
  DeviceScope device(ctx);
  if (!rows || !s.S) {  // nothing to multiply: no query or no key
    if (p->dq) TX_CUDA(ctx, cudaMemsetAsync(p->dq, 0, (size_t)rows * 2 * s.d * 4, ctx->stream));
    if (p->dk) {
      const size_t keys = (size_t)(s.B * s.S * s.Hk);
      TX_CUDA(ctx, cudaMemsetAsync(p->dk, 0, keys * 2 * s.d * 4, ctx->stream));
      TX_CUDA(ctx, cudaMemsetAsync(p->dv, 0, keys * s.dv * 4, ctx->stream));
    }
    if (p->dlam) TX_CUDA(ctx, cudaMemsetAsync(p->dlam, 0, (size_t)s.H * 4, ctx->stream));
    return TX_OK;
  }
  Scratch stats(ctx, (size_t)(s.B * s.H * ((s.T + 63) / 64)) * 256 * 4);
  Operands x(ctx, s, true);
  Scratch sums(ctx, (size_t)x.tg * 4);
  if (!stats.ptr || !sums.ptr) return TX_ERR_OOM;
  TX_TRY(x.fill(ctx, s, p, stats.as<float>(), sums.as<float>()));
  if (p->dlam) {
    k_diff_dlam<<<(unsigned)s.H, 256, 0, ctx->stream>>>(s, sums.as<float>(), x.x.qt, p->dlam);
    TX_LAUNCHED(ctx, "k_diff_dlam");
  }
  if (!p->dq && !p->dk) return TX_OK;
  return tc_backward(ctx, s, x.x, stats.as<float>(), p->dq, p->dk, p->dv);
}
