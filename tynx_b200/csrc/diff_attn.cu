// Differential attention: out = A1 v - lam A2 v with A_m = softmax(scale q_m k_m^T).
//
// With D_m = rowsum(dO * O_m) (O_m = A_m v) and dP = dO v^T the gradients are
//   dS1 = A1 (dP - D1) scale,  dS2 = -lam A2 (dP - D2) scale,
//   dq_m = dS_m k_m,  dk_m = dS_m^T q_m,  dv = (A1 - lam A2)^T dO,  dlam = -sum D2,
// and A_m comes back from the saved log-sum-exp without a second softmax pass.
// Statistics, sums and accumulators are fp32.
#include <cmath>

#include "common.h"

namespace {

constexpr int kMaxDim = 64, kMaxVdim = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Shape {
  int64_t B, T, S;
  int H, Hk, G, d, dv;  // G = H / Hk
  const float *q, *k, *v, *lam;
  const int64_t *len;
  int causal;
  int64_t start;
  float scale;
  int *err;

  __device__ __forceinline__ int64_t length(int64_t b) const {
    if (!len) return S;
    const int64_t n = __ldg(len + b);
    return n < 0 ? 0 : n > S ? S : n;
  }
  // keys that query t of sequence b (valid keys n) sees: [0, seen)
  __device__ __forceinline__ int64_t seen(int64_t t, int64_t n) const {
    if (!causal) return n;
    const int64_t c = t + start + 1;
    return c < 0 ? 0 : c < n ? c : n;
  }
};

// A key length outside [0, S] raises the context's error flag.
__device__ __forceinline__ void report_length(const Shape &s, int64_t b) {
  if (!s.len) return;
  const int64_t n = __ldg(s.len + b);
  if (n < 0 || n > s.S)
    if (atomicCAS(s.err, 0, DEVERR_INDEX) == 0) {
      s.err[1] = (int)(n < -2147483647 ? -2147483647 : n > 2147483647 ? 2147483647 : n);
      s.err[2] = (int)(s.S + 1);
    }
}

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

// ---- backward ------------------------------------------------------------------------------
// delta[0], delta[1]: D1 and D2 of each (b, h, t); a warp per row.
__global__ void __launch_bounds__(256)
    k_diff_delta(const __grid_constant__ Shape s, const float *out, const float *out2, const float *dout, float *delta) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = s.B * s.T * s.H;
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int h = (int)(row % s.H);
  const int64_t bt = row / s.H, b = bt / s.T, t = bt - b * s.T;
  const float lam = __ldg(s.lam + h);
  float d1 = 0.f, d2 = 0.f;
  for (int c = lane; c < s.dv; c += 32) {
    const float g = dout[row * s.dv + c], o2 = out2[row * s.dv + c];
    d1 += g * (out[row * s.dv + c] + lam * o2);
    d2 += g * o2;
  }
  d1 = warp_sum(d1);
  d2 = warp_sum(d2);
  if (lane == 0) {
    const int64_t i = (b * s.H + h) * s.T + t;
    delta[i] = d1;
    delta[rows + i] = d2;
  }
}

__global__ void __launch_bounds__(256) k_diff_dlam(const __grid_constant__ Shape s, const float *delta2, float *dlam) {
  __shared__ float sums[8];
  const int h = blockIdx.x;
  float v = 0.f;
  for (int64_t i = threadIdx.x; i < s.B * s.T; i += 256) {
    const int64_t b = i / s.T, t = i - b * s.T;
    v += delta2[(b * s.H + h) * s.T + t];
  }
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) v += sums[i];
    dlam[h] = -v;
  }
}

// both maps' weights and score gradients of one (query, key) pair
struct Pair {
  float w, ds1, ds2;
};
__device__ __forceinline__ Pair pair_grad(const Shape &s, const float *q, const float *k, const float *g, const float *v,
                                          float lse1, float lse2, float d1, float d2, float lam) {
  float s1 = 0.f, s2 = 0.f, dp = 0.f;
  for (int c = 0; c < s.d; ++c) s1 += q[c] * k[c], s2 += q[s.d + c] * k[s.d + c];
  for (int c = 0; c < s.dv; ++c) dp += g[c] * v[c];
  const float f = s.scale * kLog2e;
  const float a1 = exp2f(s1 * f - lse1), a2 = exp2f(s2 * f - lse2);
  return {a1 - lam * a2, a1 * (dp - d1) * s.scale, -lam * a2 * (dp - d2) * s.scale};
}

__global__ void __launch_bounds__(128)
    k_diff_dq(const __grid_constant__ Shape s, const float *lse, const float *delta, const float *dout, float *dq) {
  __shared__ float g1[128], g2[128];
  const int64_t bt = blockIdx.x, b = bt / s.T, t = bt - b * s.T;
  const int h = blockIdx.y, hk = h / s.G, tid = threadIdx.x;
  const int64_t rows = s.B * s.T * s.H, n = s.seen(t, s.length(b));
  const float *q = s.q + (bt * 2 * s.H + 2 * h) * s.d, *g = dout + (bt * s.H + h) * s.dv;
  const float lse1 = lse[(b * 2 * s.H + 2 * h) * s.T + t], lse2 = lse[(b * 2 * s.H + 2 * h + 1) * s.T + t];
  const float d1 = delta[(b * s.H + h) * s.T + t], d2 = delta[rows + (b * s.H + h) * s.T + t], lam = s.lam[h];
  float acc = 0.f;
  for (int64_t j0 = 0; j0 < n; j0 += 128) {
    const int64_t j = j0 + tid;
    Pair p{0.f, 0.f, 0.f};
    if (j < n)
      p = pair_grad(s, q, s.k + ((b * s.S + j) * 2 * s.Hk + 2 * hk) * s.d, g, s.v + ((b * s.S + j) * s.Hk + hk) * s.dv,
                    lse1, lse2, d1, d2, lam);
    g1[tid] = p.ds1;
    g2[tid] = p.ds2;
    __syncthreads();
    if (tid < 2 * s.d)
      for (int i = 0; i < 128 && j0 + i < n; ++i)
        acc += (tid < s.d ? g1 : g2)[i] * s.k[((b * s.S + j0 + i) * 2 * s.Hk + 2 * hk) * s.d + tid];
    __syncthreads();
  }
  if (tid < 2 * s.d) dq[(bt * 2 * s.H + 2 * h) * s.d + tid] = acc;
}

__global__ void __launch_bounds__(128)
    k_diff_dkv(const __grid_constant__ Shape s, const float *lse, const float *delta, const float *dout, float *dk,
               float *dv) {
  __shared__ float w[128], g1[128], g2[128];
  const int64_t bj = blockIdx.x, b = bj / s.S, j = bj - b * s.S;
  const int hk = blockIdx.y, tid = threadIdx.x;
  const int64_t rows = s.B * s.T * s.H, n = s.length(b);
  const float *k = s.k + (bj * 2 * s.Hk + 2 * hk) * s.d, *v = s.v + (bj * s.Hk + hk) * s.dv;
  float ak = 0.f, av = 0.f;
  int64_t t0 = 0;
  if (s.causal && j - s.start > 0) t0 = j - s.start;
  if (j < n)
    for (int h = hk * s.G; h < (hk + 1) * s.G; ++h) {
      const float lam = s.lam[h];
      for (int64_t i0 = t0; i0 < s.T; i0 += 128) {
        const int64_t t = i0 + tid, i = (b * s.H + h) * s.T + t;
        Pair p{0.f, 0.f, 0.f};
        if (t < s.T)
          p = pair_grad(s, s.q + ((b * s.T + t) * 2 * s.H + 2 * h) * s.d, k, dout + ((b * s.T + t) * s.H + h) * s.dv, v,
                        lse[(b * 2 * s.H + 2 * h) * s.T + t], lse[(b * 2 * s.H + 2 * h + 1) * s.T + t], delta[i],
                        delta[rows + i], lam);
        w[tid] = p.w;
        g1[tid] = p.ds1;
        g2[tid] = p.ds2;
        __syncthreads();
        for (int u = 0; u < 128 && i0 + u < s.T; ++u) {
          const int64_t bt = b * s.T + i0 + u;
          if (tid < 2 * s.d) ak += (tid < s.d ? g1 : g2)[u] * s.q[(bt * 2 * s.H + 2 * h) * s.d + tid];
          if (tid < s.dv) av += w[u] * dout[(bt * s.H + h) * s.dv + tid];
        }
        __syncthreads();
      }
    }
  if (tid < 2 * s.d) dk[(bj * 2 * s.Hk + 2 * hk) * s.d + tid] = ak;
  if (tid < s.dv) dv[(bj * s.Hk + hk) * s.dv + tid] = av;
}

// ---- host ----------------------------------------------------------------------------------
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
  k_diff_join<<<(unsigned)(s.B * s.Hk * items), kMaxVdim, 0, ctx->stream>>>(s, (int)splits, po.as<float>(),
                                                                           pm.as<float2>(), out, out2, lse);
  TX_LAUNCHED(ctx, "k_diff_join");
  return TX_OK;
}

}  // namespace

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
  return launch_rows<8>(ctx, s, p->out, p->out2, p->lse);
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
  Scratch delta(ctx, rows ? (size_t)rows * 8 : 8);
  if (!delta.ptr) return TX_ERR_OOM;
  if (rows) {
    k_diff_delta<<<(unsigned)((rows + 7) / 8), 256, 0, ctx->stream>>>(s, p->out, p->out2, p->dout, delta.as<float>());
    TX_LAUNCHED(ctx, "k_diff_delta");
  }
  if (p->dlam) {
    k_diff_dlam<<<(unsigned)s.H, 256, 0, ctx->stream>>>(s, delta.as<float>() + rows, p->dlam);
    TX_LAUNCHED(ctx, "k_diff_dlam");
  }
  if (p->dq && rows) {
    k_diff_dq<<<dim3((unsigned)(s.B * s.T), (unsigned)s.H), 128, 0, ctx->stream>>>(s, p->lse, delta.as<float>(), p->dout,
                                                                                  p->dq);
    TX_LAUNCHED(ctx, "k_diff_dq");
  }
  if (p->dk && s.B * s.S) {
    k_diff_dkv<<<dim3((unsigned)(s.B * s.S), (unsigned)s.Hk), 128, 0, ctx->stream>>>(s, p->lse, delta.as<float>(),
                                                                                    p->dout, p->dk, p->dv);
    TX_LAUNCHED(ctx, "k_diff_dkv");
  }
  return TX_OK;
}
