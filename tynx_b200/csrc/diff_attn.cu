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

// A block splits one tile of 128 rows of one head; blockIdx.z picks the tensor.  Bound by memory: 100 MB
// of q, k and v of 8192 tokens become as many bytes of pairs in 39 us, 5.2 TB/s (three blocks an SM, with
// the registers that leaves, 44 us where the statistics are made too, for 34).
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
  // stats, beside lse, and each tile's sum of D2 (P > 1: each head's in the tile) to sums
  const float *out, *out2, *lse;
  float *stats, *sums;
  int first;  // the first job to do
};
constexpr int kSplitThreads = 512, kSplitWarps = kSplitThreads / 32;
// PACK: Shape::P heads' queries are the rows of one
template <int W, bool STATS, bool PACK>
__device__ __forceinline__ void split_tile(const Shape &s, const SplitJobs &jobs, const SplitJob &J, uint32_t *red,
                                           float *d2_of) {
  const int P = PACK ? s.P : 1;
  constexpr int PARTS = W / 8, ROWS = kSplitThreads / PARTS, UNITS = kRows / ROWS;  // 8 elements a thread and unit
  const int64_t head = (int64_t)blockIdx.x / J.tiles, tile = (int64_t)blockIdx.x - head * J.tiles;
  const int64_t b = head / J.heads, n0 = tile * kRows;
  const int hh = (int)(head - b * J.heads), c = threadIdx.x % PARTS * 8, r0 = threadIdx.x / PARTS;
  const int64_t n_end = J.masked ? s.length(b) : J.N;
  // the row of src (for P > 1: token, head of the P heads' maps or of the P heads)
  auto row_of = [&](int64_t n) {
    if (P == 1) return (b * J.N + n) * J.heads + hh;
    const int t = (int)n / P, g = (int)n - t * P;
    return (b * J.N + (int64_t)t * P) * J.heads + (STATS ? hh * P + g : (hh & ~1) * P + 2 * g + (hh & 1));
  };
  const bool four = (J.w & 3) == 0 && ((uintptr_t)J.src & 15) == 0;
  float x[UNITS][8];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t n = n0 + r0 + u * ROWS;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
    if (n < n_end) {
      const float *src = J.src + row_of(n) * J.w + c;
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
    const float lam_one = P == 1 ? __ldg(s.lam + hh) : 0.f;
    float most;
    const int shrink = P == 1 ? 0 : lam_exponent(s, hh * P, most);
    const int64_t steps = (J.N + 63) / 64;
    float total = 0.f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t n = n0 + r0 + u * ROWS;
      const int t = P == 1 ? (int)n : (int)n / P, h = P == 1 ? hh : hh * P + (int)n - t * P;
      const float lam = P == 1 ? lam_one : n < J.N ? __ldg(s.lam + h) : 0.f;
      float d1 = 0.f, d2 = 0.f;
      if (n < J.N) {
        const int64_t at = row_of(n) * J.w + c;
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
        float *to = jobs.stats + (head * steps + n / 64) * (P == 1 ? 256 : 320) + n % 64;
        const bool live = n < J.N;
        to[0] = live ? __ldg(jobs.lse + (b * 2 * s.H + 2 * h) * s.T + t) : INFINITY;
        to[64] = live ? __ldg(jobs.lse + (b * 2 * s.H + 2 * h + 1) * s.T + t) : INFINITY;
        to[128] = d1;
        to[192] = d2;
        if (P > 1) to[256] = lam * __uint_as_float((uint32_t)(127 - shrink) << 23);
        total += d2;
      }
      if (P > 1 && c == 0) d2_of[r0 + u * ROWS] = d2;
    }
    total = warp_sum(total);
    if ((threadIdx.x & 31) == 0) red[2 * kSplitWarps + (threadIdx.x >> 5)] = __float_as_uint(total);
  }
  // the tile's largest finite magnitude
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < UNITS; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[u][i] *= J.factor;
      const uint32_t a = __float_as_uint(x[u][i]) & 0x7fffffffu;
      if (a < 0x7f800000u && a > top) top = a;
    }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSplitWarps; ++i) top = red[i] > top ? red[i] : top;
  int e = (int)(top >> 23) - 127 - 13;
  e = e < -113 ? -113 : e > 114 ? 114 : e;
  const float f = __uint_as_float((uint32_t)(127 + e) << 23), inv = __uint_as_float((uint32_t)(127 - e) << 23);
  if (threadIdx.x == 0) {
    J.f[blockIdx.x] = f;
    if (STATS && P == 1) {
      float total = 0.f;
      for (int i = 0; i < kSplitWarps; ++i) total += __uint_as_float(red[2 * kSplitWarps + i]);
      jobs.sums[blockIdx.x] = total;
    }
  }
  if (STATS && P > 1 && threadIdx.x < P) {  // rows of head threadIdx.x, in their order
    float total = 0.f;
    for (int i = (int)((threadIdx.x + P - n0 % P) % P); i < kRows && n0 + i < J.N; i += P) total += d2_of[i];
    jobs.sums[(int64_t)blockIdx.x * P + threadIdx.x] = total;
  }
  if (J.norm) {  // the largest row norm, from the scaled elements: their squares neither overflow nor vanish
    float norm = 0.f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += (x[u][i] * inv) * (x[u][i] * inv);
#pragma unroll
      for (int o = PARTS / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      norm = fmaxf(norm, ss);
    }
    const uint32_t nb = __reduce_max_sync(0xffffffffu, __float_as_uint(norm));
    if ((threadIdx.x & 31) == 0) red[kSplitWarps + (threadIdx.x >> 5)] = nb;
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t most = 0;
      for (int i = 0; i < kSplitWarps; ++i) most = red[kSplitWarps + i] > most ? red[kSplitWarps + i] : most;
      J.norm[blockIdx.x] = fminf(sqrtf(__uint_as_float(most)) * f, 3e38f);
    }
  }
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
// W: the values' width (queries and keys have 64)
template <int W, bool PACK>
__global__ void __launch_bounds__(kSplitThreads, 2)
    k_diff_split(const __grid_constant__ Shape s, const __grid_constant__ SplitJobs jobs) {
  __shared__ uint32_t red[3 * kSplitWarps];
  __shared__ float d2_of[PACK ? kRows : 1];
  next_may_start();
  const int job = jobs.first + blockIdx.z;
  const SplitJob &J = jobs.j[job];
  if ((int64_t)blockIdx.x >= s.B * J.heads * J.tiles) return;
  if (job == 3)
    split_tile<W, true, PACK>(s, jobs, J, red, d2_of);
  else if (PACK && job == 0)
    split_tile<64, false, PACK>(s, jobs, J, red, d2_of);
  else if (job < 2)
    split_tile<64, false, false>(s, jobs, J, red, d2_of);
  else
    split_tile<W, false, false>(s, jobs, J, red, d2_of);
}

// ---- few query rows against many keys ----------------------------------------------------
// Bound by reading the keys and values once: 105 MB (8 sequences of 4607 to 8190 keys of 2 heads) in
// 25.6 us, 4.1 TB/s (537 MB of 8 heads in 79, the copy rate).  A block takes RP queries (token, head of the
// group) of one key head, both maps, and a range of keys; its warps take four keys at a time in turn and meet
// only at the end.  A lane holds four of a key's 64 elements (half a warp a map) and four of a value's 128.
// The 4 RP dot products of a map are added over its 16 lanes by halving: each exchange passes on the half that
// the partner keeps, so the sum costs about one shuffle a product and leaves one (key, query) score a lane,
// where its exponential is taken.  The weights go through shared memory back to all lanes.
// The running maximum is followed only when it has grown by 2^16 (fp32 sums lose nothing below).
constexpr int kRowWarps = 8, kRowThreads = 32 * kRowWarps;
// keys of a group: a lane holds 4 RP products before they are added, 2 RP for eight queries
template <int RP>
constexpr int kGroupOf = RP == 8 ? 2 : 4;

template <int RP>
struct RowSmem {
  float2 p[kRowWarps][kGroupOf<RP>][2 * RP];  // weights, each twice (a pair's factor); then factors of a new maximum
  float2 ml[kRowWarps][2 * RP];
  float acc[kRowWarps][2 * RP][kMaxVdim];
};

// four elements of which `have` exist, as two pairs; VEC: all or none, 16-byte aligned
template <bool VEC>
__device__ __forceinline__ void load4(const float *p, int have, uint64_t (&x)[2]) {
  x[0] = x[1] = two(0.f, 0.f);
  if (VEC) {
    if (have > 0) {
      const ulonglong2 v = __ldg(reinterpret_cast<const ulonglong2 *>(p));
      x[0] = v.x, x[1] = v.y;
    }
  } else {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (have > i) v[i] = __ldg(p + i);
    x[0] = two(v[0], v[1]), x[1] = two(v[2], v[3]);
  }
}

// VEC: key and value rows can be read four elements at a time
template <int RP, bool VEC>
__global__ void __launch_bounds__(kRowThreads, 2)
    k_diff_rows(const __grid_constant__ Shape s, const Parts parts, int64_t keys_per_split) {
  next_may_start();
  extern __shared__ __align__(16) uint8_t raw[];
  RowSmem<RP> &sh = *reinterpret_cast<RowSmem<RP> *>(raw);
  constexpr int kGroup = kGroupOf<RP>;
  constexpr int NV = kGroup * RP;                // scores of a map's group, v = query * kGroup + key
  static_assert(NV <= 16, "one score a lane at the end");
  constexpr int COPY = 16 / NV;                  // lanes that hold the same one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, m = lane >> 4, l16 = lane & 15;
  const int bh = blockIdx.x / parts.splits, split = blockIdx.x - bh * parts.splits, b = bh / s.Hk, hk = bh - b * s.Hk;
  const int n_items = (int)(s.T * s.G), item0 = blockIdx.y * RP;  // few_queries()
  const int64_t n = s.length(b);
  if (threadIdx.x == 0 && hk == 0 && split == 0 && blockIdx.y == 0) report_length(s, b);
  const int last = item0 + RP <= n_items ? item0 + RP - 1 : n_items - 1;
  const int64_t k0 = (int64_t)split * keys_per_split;
  const int64_t end = s.seen(last / s.G, n) - k0;
  const int keys = end < 0 ? 0 : end > keys_per_split ? (int)keys_per_split : (int)end;  // of this block

  // this lane's elements of its map's queries, and the query whose scores it holds
  uint64_t q[RP][2];
  const int have_d = s.d - 4 * l16, have_v = s.dv - 4 * lane;
#pragma unroll
  for (int r = 0; r < RP; ++r) {
    const int item = item0 + r < n_items ? item0 + r : last, t = item / s.G, h = hk * s.G + item - t * s.G;
    load4<false>(s.q + ((b * s.T + t) * (2 * s.H) + 2 * h + m) * s.d + 4 * l16, have_d, q[r]);
    const float f = s.scale * kLog2e;
    q[r][0] = mul2(q[r][0], two(f, f)), q[r][1] = mul2(q[r][1], two(f, f));
  }
  const int mine = l16 / COPY / kGroup, key = l16 / COPY % kGroup;
  const int my_item = item0 + mine < n_items ? item0 + mine : last;
  const int64_t my_end = s.seen(my_item / s.G, n) - k0;
  const int seen = my_end < 0 ? 0 : my_end > keys ? keys : (int)my_end;

  uint64_t acc[2 * RP][2];
#pragma unroll
  for (int r = 0; r < 2 * RP; ++r) acc[r][0] = acc[r][1] = two(0.f, 0.f);
  float ref = -INFINITY, sum = 0.f;
  const int64_t k_stride = (int64_t)2 * s.Hk * s.d, v_stride = (int64_t)s.Hk * s.dv;
  int j0 = kGroup * warp;
  const float *kp = s.k + (b * s.S + k0 + j0) * k_stride + (2 * hk + m) * s.d + 4 * l16;
  const float *vp = s.v + (b * s.S + k0 + j0) * v_stride + hk * s.dv + 4 * lane;
  uint64_t kk[kGroup][2], vv[kGroup][2];
#pragma unroll
  for (int g = 0; g < kGroup; ++g) load4<VEC>(kp + g * k_stride, j0 + g < keys ? have_d : 0, kk[g]);
  for (; j0 < keys; j0 += kGroup * kRowWarps) {  // uniform in a warp
#pragma unroll
    for (int g = 0; g < kGroup; ++g) load4<VEC>(vp + g * v_stride, j0 + g < keys ? have_v : 0, vv[g]);
    vp += kGroup * kRowWarps * v_stride;
    float v[NV];
#pragma unroll
    for (int r = 0; r < RP; ++r)
#pragma unroll
      for (int g = 0; g < kGroup; ++g) {
        float x, y;
        untwo(fma2(kk[g][0], q[r][0], mul2(kk[g][1], q[r][1])), x, y);
        v[r * kGroup + g] = x + y;
      }
    kp += kGroup * kRowWarps * k_stride;
#pragma unroll
    for (int g = 0; g < kGroup; ++g)
      load4<VEC>(kp + g * k_stride, j0 + kGroup * kRowWarps + g < keys ? have_d : 0, kk[g]);
    int left = NV;
#pragma unroll
    for (int o = 8; o; o >>= 1) {
      if (left > 1) {  // pass on the half that the partner keeps
        const bool up = l16 & o;
        left >>= 1;
#pragma unroll
        for (int i = 0; i < NV / 2; ++i)
          if (i < left) {
            const float keep = up ? v[i + left] : v[i], give = up ? v[i] : v[i + left];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      }
    }
    // v[0]: the score of query `mine` and key `key`
    if (j0 + key >= seen) v[0] = -INFINITY;
    float top = v[0];
#pragma unroll
    for (int o = COPY; o < COPY * kGroup; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (__any_sync(0xffffffffu, top > ref + 16.f || (ref == -INFINITY && top > ref))) {
      const float now = fmaxf(ref, top), f = ref == -INFINITY ? 0.f : ex2(ref - now);
      sum *= f;
      ref = now;
      if (l16 % (16 / RP) == 0) sh.p[warp][0][m * RP + mine] = make_float2(f, f);
      __syncwarp();
#pragma unroll
      for (int r = 0; r < 2 * RP; ++r) {
        const uint64_t g = *reinterpret_cast<const uint64_t *>(&sh.p[warp][0][r]);
        acc[r][0] = mul2(acc[r][0], g), acc[r][1] = mul2(acc[r][1], g);
      }
      __syncwarp();
    }
    const float at = ref == -INFINITY ? 0.f : ref;  // no key yet: all weights are 2^-inf
    const float w = ex2(v[0] - at);
    sum += w;
    if (l16 % COPY == 0) sh.p[warp][key][m * RP + mine] = make_float2(w, w);
    __syncwarp();
#pragma unroll
    for (int g = 0; g < kGroup; ++g)
#pragma unroll
      for (int r = 0; r < 2 * RP; r += 2) {
        const ulonglong2 p = *reinterpret_cast<const ulonglong2 *>(&sh.p[warp][g][r]);
        acc[r][0] = fma2(vv[g][0], p.x, acc[r][0]), acc[r][1] = fma2(vv[g][1], p.x, acc[r][1]);
        acc[r + 1][0] = fma2(vv[g][0], p.y, acc[r + 1][0]), acc[r + 1][1] = fma2(vv[g][1], p.y, acc[r + 1][1]);
      }
    __syncwarp();
  }
#pragma unroll
  for (int o = COPY; o < COPY * kGroup; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (l16 % (16 / RP) == 0) sh.ml[warp][m * RP + mine] = make_float2(ref, sum);
#pragma unroll
  for (int r = 0; r < 2 * RP; ++r)
    *reinterpret_cast<ulonglong2 *>(&sh.acc[warp][r][4 * lane]) = make_ulonglong2(acc[r][0], acc[r][1]);
  __syncthreads();
  // the warps' shares, in their order
  for (int i = threadIdx.x; i < 2 * RP * kMaxVdim; i += kRowThreads) {
    const int row = i / kMaxVdim, c = i % kMaxVdim, mm = row / RP;
    const int item = item0 + row % RP;
    if (item >= n_items) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, sh.ml[w][row].x);
    const float at = top == -INFINITY ? 0.f : top;
    float x = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float2 ml = sh.ml[w][row];
      const float f = ex2(ml.x - at);
      l += ml.y * f;
      x += sh.acc[w][row][c] * f;
    }
    const int64_t to = (((int64_t)bh * n_items + item) * 2 + mm) * parts.splits + split;
    if (c == 0) parts.ml[to] = make_float2(top, l);
    if (c < s.dv) parts.o[to * s.dv + c] = x;
  }
}

// out, out2 and lse from the ranges' partial rows: W warps per query, head and map, each a share of the
// ranges, four columns a lane.  Latency alone: 32 ranges' references at a time, one a lane, then U loads that
// do not depend on one another.
constexpr int kJoinRows = 4;  // a block at most, with W = 1
template <int U, int W>
__global__ void __launch_bounds__(64 * (W > 1 ? W : kJoinRows), W > 1 ? 2 : 3)
    k_diff_join(const __grid_constant__ Shape s, const Parts parts, float *out, float *out2, float *lse) {
  __shared__ float4 second[W > 1 ? 1 : kJoinRows][32], shares[W][2][32];
  __shared__ float sums[W][2];
  const int lane = threadIdx.x & 31, m = (threadIdx.x >> 5) & 1, splits = parts.splits;
  const int row = W > 1 ? 0 : threadIdx.x >> 6, share = W > 1 ? threadIdx.x >> 6 : 0;
  const int64_t n_items = s.T * s.G, rows = s.B * s.Hk * n_items;
  const int64_t at = W > 1 ? blockIdx.x : (int64_t)blockIdx.x * (blockDim.x >> 6) + row;  // (b, hk, item)
  const bool live = at < rows;
  const float2 *ml = parts.ml + (live ? at * 2 + m : 0) * splits;
  wait_for_previous();
  // the first 32 ranges' references stay in registers
  const float2 mine = lane < splits ? ml[lane] : make_float2(-INFINITY, 0.f);
  float top = mine.x;
  for (int i = lane + 32; i < splits; i += 32) top = fmaxf(top, ml[i].x);
  top = warp_max(top);
  const bool none = top == -INFINITY;
  const float ref = none ? 0.f : top;
  const int c = 4 * lane;
  const bool four = (s.dv & 3) == 0;  // the partial rows are aligned
  const float *p = parts.o + (live ? at * 2 + m : 0) * splits * s.dv + c;
  float sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  const int each = (splits + W - 1) / W, first = share * each, end = first + each < splits ? first + each : splits;
  for (int i0 = first; i0 < end; i0 += 32) {
    const float2 v = i0 == 0 ? mine : i0 + lane < splits ? ml[i0 + lane] : make_float2(-INFINITY, 0.f);
    const int n = end - i0 < 32 ? end - i0 : 32;
    const float w = lane < n ? ex2(v.x - ref) : 0.f;
    sum += v.y * w;
    for (int j = 0; j < n; j += U) {
      float4 y[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j + i < n) {
          const float *q = p + (int64_t)(i0 + j + i) * s.dv;
          if (four) {
            if (c < s.dv) y[i] = *reinterpret_cast<const float4 *>(q);
          } else {
            if (c < s.dv) y[i].x = q[0];
            if (c + 1 < s.dv) y[i].y = q[1];
            if (c + 2 < s.dv) y[i].z = q[2];
            if (c + 3 < s.dv) y[i].w = q[3];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float f = __shfl_sync(0xffffffffu, w, (j + i) & 31);
        if (j + i < n) x = make_float4(x.x + y[i].x * f, x.y + y[i].y * f, x.z + y[i].z * f, x.w + y[i].w * f);
      }
    }
  }
  sum = warp_sum(sum);
  if (W > 1) {  // the warps' shares, in their order
    shares[share][m][lane] = x;
    if (lane == 0) sums[share][m] = sum;
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int i = 1; i < W; ++i) {
      const float4 y = shares[i][m][lane];
      x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
      sum += sums[i][m];
    }
  }
  const float inv = none ? 0.f : 1.f / sum;
  x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  if (m) second[row][lane] = x;
  if (W > 1)
    asm volatile("bar.sync 1, 64;" ::: "memory");  // the two warps that are left
  else
    __syncthreads();
  if (!live) return;
  const int64_t bh = at / n_items, item = at - bh * n_items;
  const int64_t b = bh / s.Hk, t = item / s.G;
  const int hk = (int)(bh - b * s.Hk), h = hk * s.G + (int)(item - t * s.G);
  if (lse && lane == 0) lse[(b * 2 * s.H + 2 * h + m) * s.T + t] = none ? INFINITY : top + log2f(sum);
  float *dst = m ? out2 : out;
  if (!dst) return;
  if (!m) {
    const float lam = __ldg(s.lam + h);
    const float4 y = second[row][lane];
    x = make_float4(x.x - lam * y.x, x.y - lam * y.y, x.z - lam * y.z, x.w - lam * y.w);
  }
  dst += ((b * s.T + t) * s.H + h) * s.dv + c;
  if (c < s.dv) dst[0] = x.x;
  if (c + 1 < s.dv) dst[1] = x.y;
  if (c + 2 < s.dv) dst[2] = x.z;
  if (c + 3 < s.dv) dst[3] = x.w;
}

// dlam where it is the only gradient wanted (otherwise the backward's blocks sum it)
__global__ void __launch_bounds__(32) k_diff_dlam(const __grid_constant__ Shape s, const float *sums, int64_t tiles,
                                                  float *dlam) {
  sum_dlam(s, sums, tiles, dlam, blockIdx.x);
}

// ---- host ----------------------------------------------------------------------------------
// The split operands of one call: q, k and v in `saved` or in memory of the call, the output's gradient
// in memory of the call.
struct Operands {
  Split x{};
  Scratch own, grad;
  int64_t tq, tk, tv, tg;  // tiles
  bool ok;
  static int64_t width(const Shape &s) { return s.dv <= 64 ? 64 : 128; }
  static int64_t tiles(int64_t rows) { return (rows + kRows - 1) / kRows; }
  static size_t bytes(const Shape &s) {
    const int64_t halves = 2 * (s.B * 2 * s.H * s.T * 64 + s.B * 2 * s.Hk * s.S * 64 + s.B * s.Hk * s.S * width(s));
    return (size_t)halves * 2 + (size_t)(s.B * (2 * s.row_heads() * tiles(s.rows()) + 4 * s.Hk * tiles(s.S))) * 4;
  }
  static size_t grad_bytes(const Shape &s) {
    return (size_t)(s.B * s.H * s.T * 2 * width(s)) * 2 + (size_t)(2 * s.B * s.row_heads() * tiles(s.rows())) * 4;
  }
  Operands(tx_ctx *ctx, const Shape &s, void *saved, bool gradient)
      : own(ctx, saved ? 0 : bytes(s)), grad(ctx, gradient ? grad_bytes(s) : 0) {
    const int64_t w = width(s);
    x.vw = (int)w;
    x.qt = tiles(s.rows());
    x.kt = tiles(s.S);
    tq = s.B * 2 * s.row_heads() * x.qt, tk = s.B * 2 * s.Hk * x.kt, tv = s.B * s.Hk * x.kt, tg = s.B * s.row_heads() * x.qt;
    ok = (saved || own.ptr) && (!gradient || grad.ptr);
    if (!ok) return;
    __half *p = reinterpret_cast<__half *>(saved ? saved : own.ptr);
    x.q = p, p += s.B * 2 * s.H * s.T * 128;
    x.k = p, p += s.B * 2 * s.Hk * s.S * 128;
    x.v = p, p += s.B * s.Hk * s.S * 2 * w;
    float *f = reinterpret_cast<float *>(p);
    x.fq = f, f += tq;
    x.fk = f, f += tk;
    x.fv = f, f += tv;
    x.nv = f;
    if (!gradient) return;
    x.g = grad.as<__half>();
    x.fg = reinterpret_cast<float *>(x.g + s.B * s.H * s.T * 2 * w);
    x.ng = x.fg + tg;
  }
  // made: q, k and v are there.  p: the backward's description, or null
  int fill(tx_ctx *ctx, const Shape &s, bool made, const tx_diff_attention *p, float *stats, float *sums) {
    if (!ok) return TX_ERR_OOM;
    SplitJobs jobs{};
    jobs.j[0] = SplitJob{s.q, x.q, x.fq, nullptr, s.rows(), x.qt, 2 * s.row_heads(), s.d, s.scale * kLog2e, 0};
    jobs.j[1] = SplitJob{s.k, x.k, x.fk, nullptr, s.S, x.kt, 2 * s.Hk, s.d, 1.0f, 1};
    jobs.j[2] = SplitJob{s.v, x.v, x.fv, x.nv, s.S, x.kt, s.Hk, s.dv, 1.0f, 1};
    jobs.j[3] = SplitJob{p ? p->dout : nullptr, x.g, x.fg, x.ng, s.rows(), x.qt, s.row_heads(), s.dv, 1.0f, 0};
    jobs.first = made ? 3 : 0;
    if (p) jobs.out = p->out, jobs.out2 = p->out2, jobs.lse = p->lse, jobs.stats = stats, jobs.sums = sums;
    const int64_t blocks = made ? tg : tq > tk ? tq : tk;
    const dim3 grid((unsigned)blocks, 1, made ? 1 : p ? 4 : 3);
    auto kernel = s.P > 1 ? (x.vw == 64 ? k_diff_split<64, true> : k_diff_split<128, true>)
                          : (x.vw == 64 ? k_diff_split<64, false> : k_diff_split<128, false>);
    kernel<<<grid, kSplitThreads, 0, ctx->stream>>>(s, jobs);
    TX_LAUNCHED(ctx, "k_diff_split");
    return TX_OK;
  }
};

// Few queries take k_diff_rows, which reads keys and values once for every eight of them and needs no split
// operands: eight (token, head of a group), or up to 24 against so few keys that the tensor cores' longer
// way counts.  8 x 8192 keys of 4 heads: 8 queries 110 us, on the tensor cores 173; 16 queries 210 and 174.
// 1 x 8192: 16 queries 36 and 37, 24 queries 47 and 38; 4 x 512: 24 queries 20 and 23.
bool few_queries(const Shape &s) {
  const int64_t rows = s.T * s.G, reads = (rows + 7) / 8;
  return rows <= 8 || (rows <= 24 && reads * s.B * s.Hk * s.S <= 1 << 16);
}

// Shape::P: a group's heads share query tiles where that makes fewer tiles (4 x 64 queries of 8 heads over 4
// against 4096 keys: forward 27 us for 38; as many tiles cost more than one head's: 4 x 256 queries against
// 512 keys 25 us for 23).  keep: for a backward, whose blocks of keys then have one run over all of a group's
// queries: up to half a tile of tokens, if a head's blocks alone would fill the SMs (63 x 26 queries of 24 heads
// over 8 against 285 keys: 61 and 276 us for 135 and 431; 8 x 64 queries of 4 heads over 2: 15 and 12 for 13 and 10).
int pack_of(const tx_ctx *ctx, const Shape &s, bool keep) {
  if (s.G == 1) return 1;
  if (keep) return s.T <= kRows / 2 && s.G <= 32 && s.B * s.H > ctx->num_sms ? s.G : 1;
  return s.T * s.G <= (int64_t)1 << 30 && Operands::tiles(s.T * s.G) < s.G * Operands::tiles(s.T) ? s.G : 1;
}

int check_desc(tx_ctx *ctx, const tx_diff_attention *p, Shape &s) {
  if (!p) return tx_fail(ctx, TX_ERR_INVALID, "differential attention: no description");
  if (p->dim < 1 || p->dim > kMaxDim || p->vdim < 1 || p->vdim > kMaxVdim)
    return tx_fail(ctx, TX_ERR_UNSUPPORTED, "differential attention: head dimension 1..64, value dimension 1..128");
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->heads > 32767)
    return tx_fail(ctx, TX_ERR_SHAPE, "differential attention: the query heads must be a multiple of the key heads");
  const int64_t most = (int64_t)1 << 30;
  if (p->batch < 0 || p->queries < 0 || p->keys < 0 || p->batch > most || p->queries > most || p->keys > most ||
      p->query_start > most || p->query_start < -most || (p->batch && p->heads > (1 << 22) / p->batch) ||
      (p->batch && (p->queries > most / p->batch || p->keys > most / p->batch)))
    return tx_fail(ctx, TX_ERR_SHAPE, "differential attention: batch * heads up to 2^22, batch * length up to 2^30");
  // blocks of a launch: queries of a head, and key tiles twice
  if (p->batch * p->heads * ((p->queries + 127) / 128 + 2 * ((p->keys + 127) / 128)) >= ((int64_t)1 << 31))
    return tx_fail(ctx, TX_ERR_SHAPE, "differential attention: too many heads and tiles for one call");
  if (!std::isfinite(p->scale)) return tx_fail(ctx, TX_ERR_INVALID, "differential attention: scale");
  s = Shape{p->batch, p->queries, p->keys, (int)p->heads, (int)p->kv_heads, (int)(p->heads / p->kv_heads), (int)p->dim,
            (int)p->vdim, p->q, p->k, p->v, p->lam, p->key_lengths, p->causal ? 1 : 0, p->query_start, p->scale,
            ctx->d_err, 1};
  return TX_OK;
}

int join(tx_ctx *ctx, const Shape &s, const Parts &parts, float *out, float *out2, float *lse) {
  const int64_t rows = s.B * s.T * s.H;
  if (parts.splits > 12 && rows < 8 * ctx->num_sms) {  // many ranges of few rows (74 of 32 rows: 5.1 us for 9.2)
    return launch_behind(ctx, "k_diff_join", k_diff_join<12, 4>, (unsigned)rows, 256, 0, s, parts, out, out2, lse);
  }
  const int each = rows < 8 * ctx->num_sms ? 1 : kJoinRows;  // few rows: an SM each
  const unsigned blocks = (unsigned)((rows + each - 1) / each);
  if (parts.splits <= 4)  // (3 ranges of 8192 rows: 8.9 us, with twelve loads in flight 13.7)
    return launch_behind(ctx, "k_diff_join", k_diff_join<4, 1>, blocks, 64 * each, 0, s, parts, out, out2, lse);
  return launch_behind(ctx, "k_diff_join", k_diff_join<12, 1>, blocks, 64 * each, 0, s, parts, out, out2, lse);
}

// Partial results' memory.
struct PartMemory {
  Scratch o, ml;
  Parts parts;
  PartMemory(tx_ctx *ctx, const Shape &s, int splits)
      : o(ctx, (size_t)(s.B * s.H * s.T * 2 * splits * s.dv) * 4), ml(ctx, (size_t)(s.B * s.H * s.T * 2 * splits) * 8) {
    parts = Parts{o.as<float>(), ml.as<float2>(), splits};
  }
  bool ok() const { return o.ptr && ml.ptr; }
};

template <int RP>
int launch_rows(tx_ctx *ctx, const Shape &s, float *out, float *out2, float *lse) {
  const int64_t chunks = (s.T * s.G + RP - 1) / RP, blocks = chunks * s.B * s.Hk;
  // two blocks an SM, each with four rounds of its warps at least
  constexpr int64_t round = kGroupOf<RP> * kRowWarps;
  int64_t splits = 2 * ctx->num_sms / blocks, most = (s.S + 4 * round - 1) / (4 * round);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  const int64_t per = ((s.S + splits - 1) / splits + round - 1) / round * round;
  PartMemory mem(ctx, s, (int)splits);
  if (!mem.ok()) return TX_ERR_OOM;
  const int smem = (int)sizeof(RowSmem<RP>);
  const bool vec = (s.d & 3) == 0 && (s.dv & 3) == 0 && ((uintptr_t)s.k & 15) == 0 && ((uintptr_t)s.v & 15) == 0;
  auto kernel = vec ? k_diff_rows<RP, true> : k_diff_rows<RP, false>;
  static SmemGrant granted[2];
  TX_TRY(granted[vec].take(ctx, (const void *)kernel, smem));
  kernel<<<dim3((unsigned)(splits * s.B * s.Hk), (unsigned)chunks), kRowThreads, smem, ctx->stream>>>(
      s, mem.parts, per);
  TX_LAUNCHED(ctx, "k_diff_rows");
  return join(ctx, s, mem.parts, out, out2, lse);
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

extern "C" int tx_diff_attention_saved_bytes(tx_ctx *ctx, const tx_diff_attention *p, int64_t *bytes) {
  if (!ctx || !bytes) return TX_ERR_INVALID;
  Shape s;
  TX_TRY(check_desc(ctx, p, s));
  s.P = pack_of(ctx, s, true);
  *bytes = few_queries(s) || s.B * s.T * s.S == 0 ? 0 : (int64_t)Operands::bytes(s);
  return TX_OK;
}

extern "C" int tx_diff_attention_fwd(tx_ctx *ctx, const tx_diff_attention *p) {
  if (!ctx) return TX_ERR_INVALID;
  Shape s;
  TX_TRY(check_desc(ctx, p, s));
  if ((uintptr_t)p->saved & 15) return tx_fail(ctx, TX_ERR_INVALID, "differential attention: saved is not aligned");
  if ((p->out2 == nullptr) != (p->lse == nullptr))
    return tx_fail(ctx, TX_ERR_INVALID, "differential attention: out2 and lse come together");
  if (s.B * s.T == 0) return TX_OK;
  if (!p->q || !p->lam || !p->out || (s.S && (!p->k || !p->v)))
    return tx_fail(ctx, TX_ERR_INVALID, "differential attention: null buffer");
  DeviceScope device(ctx);
  if (s.S == 0) {
    const size_t rows = (size_t)(s.B * s.T * s.H);
    TX_CUDA(ctx, cudaMemsetAsync(p->out, 0, rows * s.dv * 4, ctx->stream));
    if (!p->out2) return TX_OK;
    TX_CUDA(ctx, cudaMemsetAsync(p->out2, 0, rows * s.dv * 4, ctx->stream));
    return tx_fill_f32(ctx, p->lse, (int64_t)(2 * rows), INFINITY);
  }
  if (s.T * s.G <= 1) return launch_rows<1>(ctx, s, p->out, p->out2, p->lse);
  if (s.T * s.G <= 2) return launch_rows<2>(ctx, s, p->out, p->out2, p->lse);
  if (s.T * s.G <= 4) return launch_rows<4>(ctx, s, p->out, p->out2, p->lse);
  if (few_queries(s)) return launch_rows<8>(ctx, s, p->out, p->out2, p->lse);
  s.P = pack_of(ctx, s, p->saved);
  Operands x(ctx, s, p->saved, false);
  TX_TRY(x.fill(ctx, s, false, nullptr, nullptr, nullptr));
  const int splits = tc_forward_splits(ctx, s);
  if (splits == 1) return tc_forward(ctx, s, x.x, p->out, p->out2, p->lse, Parts{nullptr, nullptr, 1});
  PartMemory mem(ctx, s, splits);
  if (!mem.ok()) return TX_ERR_OOM;
  TX_TRY(tc_forward(ctx, s, x.x, p->out, p->out2, p->lse, mem.parts));
  return join(ctx, s, mem.parts, p->out, p->out2, p->lse);
}

extern "C" int tx_diff_attention_bwd(tx_ctx *ctx, const tx_diff_attention *p) {
  if (!ctx) return TX_ERR_INVALID;
  Shape s;
  TX_TRY(check_desc(ctx, p, s));
  if ((uintptr_t)p->saved & 15) return tx_fail(ctx, TX_ERR_INVALID, "differential attention: saved is not aligned");
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
  s.P = pack_of(ctx, s, true);
  Scratch stats(ctx, (size_t)(s.B * s.row_heads() * ((s.rows() + 63) / 64)) * (s.P > 1 ? 320 : 256) * 4);
  const bool made = p->saved && !few_queries(s);
  Operands x(ctx, s, made ? p->saved : nullptr, true);
  Scratch sums(ctx, (size_t)(x.tg * s.P) * 4);
  if (!stats.ptr || !sums.ptr) return TX_ERR_OOM;
  TX_TRY(x.fill(ctx, s, made, p, stats.as<float>(), sums.as<float>()));
  if (p->dq || p->dk) return tc_backward(ctx, s, x.x, stats.as<float>(), sums.as<float>(), p->dq, p->dk, p->dv, p->dlam);
  if (p->dlam) {
    k_diff_dlam<<<(unsigned)s.H, 32, 0, ctx->stream>>>(s, sums.as<float>(), x.x.qt, p->dlam);
    TX_LAUNCHED(ctx, "k_diff_dlam");
  }
  return TX_OK;
}
