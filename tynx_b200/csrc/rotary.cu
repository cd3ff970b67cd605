// Rotary positions, alone and behind a per-head norm of queries and keys.
//
// A head's first `dim` elements form dim / 2 pairs; pair i of a token at
// position p turns by the angle p * w_i (factor f on both outputs):
//   y_lo = f (x_lo cos - x_hi sin),   y_hi = f (x_lo sin + x_hi cos),
// with pairs (i, i + dim/2) or, interleaved, (2i, 2i + 1); the other elements
// pass through.  The gradient is the same map with the sine negated.  With the
// norm, x is first u * w, u = x * rsqrt(mean(x^2) + eps) over the head, and the
// backward with g = (transposed rotation of dy) is
//   dx = r (g w - u mean(g w u)),   dw = sum over tokens and heads of g u.
//
// Angles: w_i arrives as turns a position in 64 bits; p * turns is reduced to
// its fraction there and nothing has to be tabulated.  To what the turns
// themselves are off by this adds 2^-53 of the angle (the product) and 2^-26
// of a turn (the fraction in fp32): the angles of positions up to some 2^25
// turns are as exact as those of near ones.  Positions beyond 2^53 are rounded
// to 53 bits on their way to fp64.
//
// All of it is bound by memory: one pass reads x (and dy) and writes y (or dx)
// once.  A block takes a few tokens with all their heads, works out the
// tokens' cosines and sines once (shared memory; one sincospi a pair instead
// of one a pair and head), and walks the (token, head) rows with 8 elements a
// lane, so a row of 128 takes half a warp and both elements of every pair sit
// in one lane: the rotation needs no exchange, the norm a shuffle sum over the
// row's lanes.  Rows whose elements cannot be taken four at a time (head_dim, or
// in halves also dim, no multiple of 8, unaligned) run the same code with single
// elements: 6 x 3770 tokens of 24 heads of 40 with norms take 52 us forward and 99
// backward, twice the floor (with a warp a row 197 and 348).
#include "launch.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 1024;  // (token, pair) angles a block holds: 8 KB

// 8 elements of a row in a lane as four pairs (lo, hi).
struct Eight {
  float lo[4], hi[4];
};

struct RowShape {
  int dim;   // head_dim
  int half;  // rotating pairs
};

// VEC: the lane holds two float4 of unit u: pairs 4 u .. 4 u + 3 as elements 4 u
// and half + 4 u (behind the rotating part 8 consecutive elements); interleaved,
// elements 4 u and dim / 2 + 4 u, two pairs each, so that a warp's accesses are
// whole lines either way.  Otherwise pairs lane + LANES i one by one.
template <bool VEC, bool INTER, int LANES>
struct Lane {
  static __device__ __forceinline__ int pair(const RowShape s, int lane, int i) {
    if (!VEC) return lane + LANES * i;
    if (INTER) return (i < 2 ? 0 : s.dim >> 2) + 2 * lane + (i & 1);
    return 4 * lane + i;
  }
  // elements of pair p's lo and hi
  static __device__ __forceinline__ void place(const RowShape s, int p, int &a, int &b) {
    if (INTER || p >= s.half) {
      a = 2 * p;
      b = a + 1;
    } else {
      a = p;
      b = p + s.half;
    }
  }
  // VEC: first elements of the two float4
  static __device__ __forceinline__ void place4(const RowShape s, int lane, int &a, int &b) {
    a = 4 * lane;
    if (INTER) {
      b = a + (s.dim >> 1);
    } else if (a >= s.half) {
      a *= 2;
      b = a + 4;
    } else {
      b = a + s.half;
    }
  }
  static __device__ __forceinline__ void load(const float *row, const RowShape s, int lane, Eight &e) {
    if (VEC) {
      int a, b;
      place4(s, lane, a, b);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (8 * lane < s.dim) {
        x = __ldg(reinterpret_cast<const float4 *>(row + a));
        y = __ldg(reinterpret_cast<const float4 *>(row + b));
      }
      if (INTER) {
        e = Eight{{x.x, x.z, y.x, y.z}, {x.y, x.w, y.y, y.w}};
      } else {
        e = Eight{{x.x, x.y, x.z, x.w}, {y.x, y.y, y.z, y.w}};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int a, b;
        place(s, pair(s, lane, i), a, b);
        e.lo[i] = a < s.dim ? __ldg(row + a) : 0.f;
        e.hi[i] = b < s.dim ? __ldg(row + b) : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void store(float *row, const RowShape s, int lane, const Eight &e) {
    if (VEC) {
      int a, b;
      place4(s, lane, a, b);
      if (8 * lane >= s.dim) return;
      float4 x, y;
      if (INTER) {
        x = make_float4(e.lo[0], e.hi[0], e.lo[1], e.hi[1]);
        y = make_float4(e.lo[2], e.hi[2], e.lo[3], e.hi[3]);
      } else {
        x = make_float4(e.lo[0], e.lo[1], e.lo[2], e.lo[3]);
        y = make_float4(e.hi[0], e.hi[1], e.hi[2], e.hi[3]);
      }
      *reinterpret_cast<float4 *>(row + a) = x;
      *reinterpret_cast<float4 *>(row + b) = y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int a, b;
        place(s, pair(s, lane, i), a, b);
        if (a < s.dim) row[a] = e.lo[i];
        if (b < s.dim) row[b] = e.hi[i];
      }
    }
  }
};

// The angles of `tokens` tokens from token t0 on: (cos, sin) * factor of pair i
// of token j at cs[j * half + i].
__device__ __forceinline__ void fill_angles(float2 *cs, const tx_rotary &rot, const int64_t *pos, int64_t pos_stride,
                                            int64_t t0, int tokens, int64_t seq) {
  const int half = rot.dim >> 1;
  for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
    const int j = i / half, p = i - j * half;
    const int64_t t = t0 + j, b = t / seq, n = t - b * seq;
    const double at = pos ? (double)__ldg(pos + b * pos_stride + n) : (double)n;
    const double turn = at * rot.turns[p];
    float sn, c;
    sincospif(2.0f * (float)(turn - rint(turn)), &sn, &c);
    cs[i] = make_float2(c * rot.factor, sn * rot.factor);
  }
}

template <bool VEC, bool INTER, int LANES, bool BACK>
__device__ __forceinline__ void turn(Eight &e, const float2 *cs, const RowShape s, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = Lane<VEC, INTER, LANES>::pair(s, lane, i);
    if (p < s.half) {
      const float2 a = cs[p];
      const float s = BACK ? -a.y : a.y, lo = e.lo[i], hi = e.hi[i];
      e.lo[i] = lo * a.x - hi * s;
      e.hi[i] = lo * s + hi * a.x;
    }
  }
}

template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Args {
  const float *x[2], *dy[2], *w[2];
  float *y[2];
  float *part;  // backward: [gridDim.x][2][256] weight gradients
  const int64_t *pos;
  int64_t pos_stride, seq, tokens;  // tokens = batch * seq
  int heads[2], dim, group;         // group: tokens a block takes at a time
  float eps;
};

// NORM: rows are normalised (q and k in turn), else rotated only (x[0]).
// BACK (without NORM): the gradient's rotation.
template <bool VEC, bool INTER, int LANES, bool NORM, bool BACK>
__global__ void __launch_bounds__(kThreads, VEC ? (NORM ? 3 : 4) : 2)
    k_rotary(const __grid_constant__ Args A, const __grid_constant__ tx_rotary rot) {
  using L = Lane<VEC, INTER, LANES>;
  __shared__ float2 cs[kAngles];
  constexpr int SLOTS = kThreads / LANES, UN = 2;
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  const RowShape s{A.dim, rot.dim >> 1};
  const int64_t t0 = (int64_t)blockIdx.x * A.group;
  const int nt = (int)(A.tokens - t0 < A.group ? A.tokens - t0 : A.group);
  Eight w[NORM ? 2 : 1];
  if (NORM) {
    L::load(A.w[0], s, lane, w[0]);
    L::load(A.w[1], s, lane, w[1]);
  }
  // rows of q, then of k, UN a time; the next ones come while these are worked on, the first ones
  // while the angles are
  const int rows0 = nt * A.heads[0], rows = rows0 + (NORM ? nt * A.heads[1] : 0);
  Eight e[UN], next[UN];
  auto row_of = [&](float *const *base, int r) {
    return NORM && r >= rows0 ? base[1] + (t0 * A.heads[1] + r - rows0) * s.dim : base[0] + (t0 * A.heads[0] + r) * s.dim;
  };
  auto fetch = [&](int r0) {
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (r0 + u * SLOTS < rows) L::load(row_of(const_cast<float *const *>(A.x), r0 + u * SLOTS), s, lane, next[u]);
  };
  fetch(slot);
  fill_angles(cs, rot, A.pos, A.pos_stride, t0, nt, A.seq);
  __syncthreads();
  const float inv = 1.0f / (float)A.dim;
  for (int r0 = slot; r0 < rows + slot; r0 += SLOTS * UN) {  // uniform within a warp: shuffles below
#pragma unroll
    for (int u = 0; u < UN; ++u) e[u] = next[u];
    fetch(r0 + SLOTS * UN);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int r = r0 + u * SLOTS;
      const bool second = NORM && r >= rows0;
      if (NORM) {
        float ss = 0.f;
        if (r < rows) {
#pragma unroll
          for (int i = 0; i < 4; ++i) ss += e[u].lo[i] * e[u].lo[i] + e[u].hi[i] * e[u].hi[i];
        }
        const float n = rsqrtf(row_sum<LANES>(ss) * inv + A.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[u].lo[i] *= n * (second ? w[NORM].lo[i] : w[0].lo[i]);
          e[u].hi[i] *= n * (second ? w[NORM].hi[i] : w[0].hi[i]);
        }
      }
      if (r < rows) {
        const int token = second ? (r - rows0) / A.heads[1] : r / A.heads[0];
        turn<VEC, INTER, LANES, BACK>(e[u], cs + token * s.half, s, lane);
        L::store(row_of(A.y, r), s, lane, e[u]);
      }
    }
  }
}

constexpr int kBackBlocks = 3;  // resident blocks an SM

// The norm's backward: dx, and this block's share of both weight gradients.
template <bool VEC, bool INTER, int LANES>
__global__ void __launch_bounds__(kThreads, kBackBlocks)
    k_qk_norm_bwd(const __grid_constant__ Args A, const __grid_constant__ tx_rotary rot) {
  using L = Lane<VEC, INTER, LANES>;
  next_may_start();
  __shared__ float2 cs[kAngles];
  __shared__ __align__(16) float sums[kThreads / 32][256];
  constexpr int SLOTS = kThreads / LANES, UN = 2;
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  const RowShape s{A.dim, rot.dim >> 1};
  const float inv = 1.0f / (float)A.dim;
  Eight dw[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) dw[0].lo[i] = dw[0].hi[i] = dw[1].lo[i] = dw[1].hi[i] = 0.f;
  for (int64_t t0 = (int64_t)blockIdx.x * A.group; t0 < A.tokens; t0 += (int64_t)gridDim.x * A.group) {
    const int nt = (int)(A.tokens - t0 < A.group ? A.tokens - t0 : A.group);
    __syncthreads();
    fill_angles(cs, rot, A.pos, A.pos_stride, t0, nt, A.seq);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int H = A.heads[which], rows = nt * H;
      const int64_t base = t0 * H;
      Eight w;
      L::load(A.w[which], s, lane, w);
      for (int r0 = slot; r0 < rows + slot; r0 += SLOTS * UN) {
        Eight x[UN], g[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int r = r0 + u * SLOTS;
          if (r < rows) {
            L::load(A.x[which] + (base + r) * s.dim, s, lane, x[u]);
            L::load(A.dy[which] + (base + r) * s.dim, s, lane, g[u]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u].lo[i] = x[u].hi[i] = g[u].lo[i] = g[u].hi[i] = 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int r = r0 + u * SLOTS;
          if (r < rows) turn<VEC, INTER, LANES, true>(g[u], cs + (r / H) * s.half, s, lane);
          float ss = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            ss += x[u].lo[i] * x[u].lo[i] + x[u].hi[i] * x[u].hi[i];
            dot += g[u].lo[i] * w.lo[i] * x[u].lo[i] + g[u].hi[i] * w.hi[i] * x[u].hi[i];
          }
          // behind the last row 0, not rsqrt(0 + eps): infinite without eps, and NaN in the weight gradients
          const float all = row_sum<LANES>(ss), n = r < rows ? rsqrtf(all * inv + A.eps) : 0.f;
          const float c = row_sum<LANES>(dot) * inv * n * n;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dw[which].lo[i] += g[u].lo[i] * x[u].lo[i] * n;
            dw[which].hi[i] += g[u].hi[i] * x[u].hi[i] * n;
            x[u].lo[i] = n * (g[u].lo[i] * w.lo[i] - x[u].lo[i] * c);
            x[u].hi[i] = n * (g[u].hi[i] * w.hi[i] - x[u].hi[i] * c);
          }
          if (r < rows) L::store(A.y[which] + (base + r) * s.dim, s, lane, x[u]);
        }
      }
    }
  }
  // rows of a warp's slots, then the block's warps, in a fixed order
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) {
        dw[which].lo[i] += __shfl_xor_sync(0xffffffffu, dw[which].lo[i], o);
        dw[which].hi[i] += __shfl_xor_sync(0xffffffffu, dw[which].hi[i], o);
      }
    }
    __syncthreads();
    if ((threadIdx.x & 31) < LANES) L::store(sums[warp], s, lane, dw[which]);
    __syncthreads();
    if (threadIdx.x < s.dim) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) v += sums[i][threadIdx.x];
      A.part[((int64_t)blockIdx.x * 2 + which) * 256 + threadIdx.x] = v;
    }
  }
}

// dw[which][c] = sum over the blocks' shares, 32 columns a block.
__global__ void __launch_bounds__(1024) k_qk_norm_dw(const float *part, int blocks, int dim, float *dqw, float *dkw) {
  __shared__ float sums[32][33];
  const int which = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), row = threadIdx.x >> 5;
  float v = 0.f;
  wait_for_previous();
  if (c < dim) {
#pragma unroll 4
    for (int b = row; b < blocks; b += 32) v += part[((int64_t)b * 2 + which) * 256 + c];
  }
  sums[row][threadIdx.x & 31] = v;
  __syncthreads();
  v = sums[threadIdx.x & 31][row];  // a warp a column
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0 && blockIdx.x * 32 + row < dim) (which ? dkw : dqw)[blockIdx.x * 32 + row] = v;
}

bool four(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Tokens a block takes at a time, within the angle table.  Long inputs: with the norm, eight rows a
// slot, so that weights, angles and the block's start are shared by more (4 x 4096 tokens of 20 heads of
// 128: forward 61.5 us, backward 92 us; with four 65 and 104), without it four (8 x 2048 tokens of 16
// heads of 64: 21.9 us, with eight 23.6).  Short ones four, so that all SMs have blocks.
int group_of(int lanes, int heads, int half, int64_t tokens, int sms, bool norm) {
  const int slots = kThreads / lanes;
  int64_t g = 8 * slots / heads;
  if (!norm || tokens < 6 * sms * g) g = 4 * slots / heads;
  const int64_t share = (tokens + sms - 1) / sms;  // few tokens: one wave of smaller blocks
  if (g > share) g = share;
  if (half && g > kAngles / half) g = kAngles / half;
  return g < 1 ? 1 : (int)g;  // half <= 128: the table holds one token's angles at least
}

int check_rotary(tx_ctx *ctx, int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads, int64_t head_dim,
                 const int64_t *pos, int64_t pos_stride, const tx_rotary *rot) {
  if (!rot) return tx_fail(ctx, TX_ERR_INVALID, "rotary: no frequencies");
  if (batch < 0 || seq < 0 || heads < 1 || kv_heads < 0 || heads > 65535 || kv_heads > 65535)
    return tx_fail(ctx, TX_ERR_SHAPE, "rotary: batch, sequence or head count");
  if (head_dim < 1 || head_dim > 256) return tx_fail(ctx, TX_ERR_UNSUPPORTED, "rotary: head dimension 1..256");
  if (rot->dim < 0 || (rot->dim & 1) || rot->dim > head_dim)
    return tx_fail(ctx, TX_ERR_SHAPE, "rotary: an even number of rotating elements within the head is needed");
  if (batch && seq > ((int64_t)1 << 31) / batch) return tx_fail(ctx, TX_ERR_SHAPE, "rotary: at most 2^31 tokens");
  if (pos && pos_stride != 0 && pos_stride != seq) return tx_fail(ctx, TX_ERR_SHAPE, "rotary: position stride");
  return TX_OK;
}

template <bool VEC, bool INTER, int LANES>
int launch_rows(tx_ctx *ctx, Args &A, const tx_rotary &rot, int mode, float *dqw, float *dkw) {
  const int heads = A.heads[0] + A.heads[1];
  A.group = group_of(LANES, heads, rot.dim >> 1, A.tokens, ctx->num_sms, mode >= 2);
  const int64_t groups = (A.tokens + A.group - 1) / A.group;
  if (mode == 0) k_rotary<VEC, INTER, LANES, false, false><<<(unsigned)groups, kThreads, 0, ctx->stream>>>(A, rot);
  if (mode == 1) k_rotary<VEC, INTER, LANES, false, true><<<(unsigned)groups, kThreads, 0, ctx->stream>>>(A, rot);
  if (mode == 2) k_rotary<VEC, INTER, LANES, true, false><<<(unsigned)groups, kThreads, 0, ctx->stream>>>(A, rot);
  if (mode == 3) {
    // one wave; the blocks' shares are summed in their order
    const int64_t wave = (int64_t)kBackBlocks * ctx->num_sms;
    const unsigned blocks = (unsigned)(groups < wave ? groups : wave);
    Scratch part(ctx, (size_t)blocks * 512 * sizeof(float));
    if (!part.ptr) return TX_ERR_OOM;
    A.part = part.as<float>();
    k_qk_norm_bwd<VEC, INTER, LANES><<<blocks, kThreads, 0, ctx->stream>>>(A, rot);
    TX_LAUNCHED(ctx, "k_qk_norm_bwd");
    return launch_behind(ctx, "k_qk_norm_dw", k_qk_norm_dw, dim3((unsigned)((A.dim + 31) / 32), 2), 1024, 0,
                         part.as<float>(), (int)blocks, A.dim, dqw, dkw);
  }
  TX_LAUNCHED(ctx, "k_rotary");
  return TX_OK;
}

// Lanes a row: two to thirty-two, so that four pairs a lane just hold it (heads of 16 with eight lanes take 46
// and 69 us where two take 16 and 31).
template <bool VEC, bool INTER>
int launch_width(tx_ctx *ctx, Args &A, const tx_rotary &rot, int mode, float *dqw, float *dkw) {
  if (A.dim <= 16) return launch_rows<VEC, INTER, 2>(ctx, A, rot, mode, dqw, dkw);
  if (A.dim <= 32) return launch_rows<VEC, INTER, 4>(ctx, A, rot, mode, dqw, dkw);
  if (A.dim <= 64) return launch_rows<VEC, INTER, 8>(ctx, A, rot, mode, dqw, dkw);
  if (A.dim <= 128) return launch_rows<VEC, INTER, 16>(ctx, A, rot, mode, dqw, dkw);
  return launch_rows<VEC, INTER, 32>(ctx, A, rot, mode, dqw, dkw);
}

template <bool INTER>
int launch_layout(tx_ctx *ctx, Args &A, const tx_rotary &rot, int mode, bool vec, float *dqw, float *dkw) {
  return vec ? launch_width<true, INTER>(ctx, A, rot, mode, dqw, dkw)
             : launch_width<false, INTER>(ctx, A, rot, mode, dqw, dkw);
}

int launch(tx_ctx *ctx, Args &A, const tx_rotary &rot, int mode, float *dqw = nullptr, float *dkw = nullptr) {
  bool vec = A.dim % 8 == 0 && (rot.interleaved || rot.dim % 8 == 0);
  for (int i = 0; i < 2; ++i) vec = vec && four(A.x[i]) && four(A.y[i]) && four(A.w[i]) && four(A.dy[i]);
  return rot.interleaved ? launch_layout<true>(ctx, A, rot, mode, vec, dqw, dkw)
                         : launch_layout<false>(ctx, A, rot, mode, vec, dqw, dkw);
}

}  // namespace

extern "C" int tx_rotary_apply(tx_ctx *ctx, const float *x, float *y, int64_t batch, int64_t seq, int64_t heads,
                               int64_t head_dim, const int64_t *pos, int64_t pos_stride, const tx_rotary *rot,
                               int inverse) {
  if (!ctx) return TX_ERR_INVALID;
  TX_TRY(check_rotary(ctx, batch, seq, heads, 0, head_dim, pos, pos_stride, rot));
  if (batch * seq == 0) return TX_OK;
  if (!x || !y) return tx_fail(ctx, TX_ERR_INVALID, "rotary: null buffer");
  DeviceScope device(ctx);
  Args A{};
  A.x[0] = x;
  A.y[0] = y;
  A.pos = pos;
  A.pos_stride = pos_stride;
  A.seq = seq;
  A.tokens = batch * seq;
  A.heads[0] = (int)heads;
  A.dim = (int)head_dim;
  return launch(ctx, A, *rot, inverse ? 1 : 0);
}

extern "C" int tx_qk_norm_rotary_fwd(tx_ctx *ctx, const float *q, const float *k, const float *qw, const float *kw,
                                     float *yq, float *yk, int64_t batch, int64_t seq, int64_t heads,
                                     int64_t kv_heads, int64_t head_dim, const int64_t *pos, int64_t pos_stride,
                                     const tx_rotary *rot, float eps) {
  if (!ctx) return TX_ERR_INVALID;
  TX_TRY(check_rotary(ctx, batch, seq, heads, kv_heads, head_dim, pos, pos_stride, rot));
  if (kv_heads < 1) return tx_fail(ctx, TX_ERR_SHAPE, "qk norm: key heads");
  if (batch * seq == 0) return TX_OK;
  if (!q || !k || !qw || !kw || !yq || !yk) return tx_fail(ctx, TX_ERR_INVALID, "qk norm: null buffer");
  DeviceScope device(ctx);
  Args A{};
  A.x[0] = q, A.x[1] = k;
  A.w[0] = qw, A.w[1] = kw;
  A.y[0] = yq, A.y[1] = yk;
  A.pos = pos;
  A.pos_stride = pos_stride;
  A.seq = seq;
  A.tokens = batch * seq;
  A.heads[0] = (int)heads, A.heads[1] = (int)kv_heads;
  A.dim = (int)head_dim;
  A.eps = eps;
  return launch(ctx, A, *rot, 2);
}

extern "C" int tx_qk_norm_rotary_bwd(tx_ctx *ctx, const float *q, const float *k, const float *qw, const float *kw,
                                     const float *dyq, const float *dyk, float *dq, float *dk, float *dqw, float *dkw,
                                     int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                     const int64_t *pos, int64_t pos_stride, const tx_rotary *rot, float eps) {
  if (!ctx) return TX_ERR_INVALID;
  TX_TRY(check_rotary(ctx, batch, seq, heads, kv_heads, head_dim, pos, pos_stride, rot));
  if (kv_heads < 1) return tx_fail(ctx, TX_ERR_SHAPE, "qk norm: key heads");
  if (!q || !k || !qw || !kw || !dyq || !dyk || !dq || !dk || !dqw || !dkw)
    return tx_fail(ctx, TX_ERR_INVALID, "qk norm: null buffer");
  DeviceScope device(ctx);
  if (batch * seq == 0) {
    TX_CUDA(ctx, cudaMemsetAsync(dqw, 0, head_dim * sizeof(float), ctx->stream));
    TX_CUDA(ctx, cudaMemsetAsync(dkw, 0, head_dim * sizeof(float), ctx->stream));
    return TX_OK;
  }
  Args A{};
  A.x[0] = q, A.x[1] = k;
  A.w[0] = qw, A.w[1] = kw;
  A.dy[0] = dyq, A.dy[1] = dyk;
  A.y[0] = dq, A.y[1] = dk;
  A.pos = pos;
  A.pos_stride = pos_stride;
  A.seq = seq;
  A.tokens = batch * seq;
  A.heads[0] = (int)heads, A.heads[1] = (int)kv_heads;
  A.dim = (int)head_dim;
  A.eps = eps;
  return launch(ctx, A, *rot, 3, dqw, dkw);
}
