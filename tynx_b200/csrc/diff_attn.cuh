// Shared declarations of differential attention: the problem's shape, the
// split operands of the tensor-core kernels, and their tcgen05 / TMA / mbarrier
// wrappers.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "launch.cuh"

namespace tx_diff {

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
  // Query rows of the tensor-core kernels: P heads' queries in turn, row i is token i / P of the head i % P
  // of its P; G or 1 (pack_of)
  int P;

  __host__ __device__ __forceinline__ int64_t rows() const { return T * P; }
  __host__ __device__ __forceinline__ int row_heads() const { return H / P; }
  __device__ __forceinline__ int64_t length(int64_t b) const {
    if (!len) return S;
    const int64_t n = __ldg(len + b);
    return n < 0 ? 0 : n > S ? S : n;
  }
  // keys that query t of a sequence with n valid keys sees: [0, seen)
  __device__ __forceinline__ int64_t seen(int64_t t, int64_t n) const {
    if (!causal) return n;
    const int64_t c = t + start + 1;
    return c < 0 ? 0 : c < n ? c : n;
  }
};

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

// dlam[h] = -sum of D2 over the tiles' sums [b][h / P][tiles][P], in a fixed order, by one warp
__device__ __forceinline__ void sum_dlam(const Shape &s, const float *sums, int64_t tiles, float *dlam, int h) {
  const int lane = threadIdx.x & 31, hq = h / s.P;
  float v = 0.f;
  for (int64_t i = lane; i < s.B * tiles; i += 32) {
    const int64_t b = i / tiles;
    v += sums[((b * s.row_heads() + hq) * tiles + (i - b * tiles)) * s.P + (h - hq * s.P)];
  }
  v = warp_sum(v);
  if (lane == 0) dlam[h] = -v;
}

// With P > 1 the backward's columns belong to several heads: their lam / 2^E, below 2, is a column's factor
// and 2^E the tile's.
__device__ __forceinline__ int lam_exponent(const Shape &s, int head0, float &most) {
  most = 0.f;
  for (int i = 0; i < s.P; ++i) most = fmaxf(most, fabsf(__ldg(s.lam + head0 + i)));
  const int e = (int)(__float_as_uint(most) >> 23) - 127;
  return e < -100 ? -100 : e > 113 ? 113 : e;
}

// Grants a kernel its dynamic shared memory once a device.
struct SmemGrant {
  std::atomic<uint64_t> devices{0};  // contexts may live on threads of their own
  int take(tx_ctx *ctx, const void *kernel, int bytes) {
    const uint64_t bit = ctx->device < 64 ? uint64_t(1) << ctx->device : 0;
    if (devices & bit) return TX_OK;
    TX_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    devices |= bit;
    return TX_OK;
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

// ---- split operands ------------------------------------------------------------------------
// The tensor-core kernels multiply pairs of fp16: x = f (hi + lo) with f a
// power of two for each tile of 128 rows that brings the tile's largest
// element into [2^13, 2^14), hi = fp16(x / f), lo = fp16(x / f - hi), and
// a b = hi hi + hi lo + lo hi.  That keeps 22 bits of every element down to 2^-17
// of its tile's largest (below, 2^-39 of the largest), at the cost of three fp16
// products: half the tensor time of three TF32 products of the same accuracy,
// in the memory of the fp32 value.  (Pairs of bf16 need no f but keep 16 bits:
// 6e-6 of an attention output's norm instead of 2e-7.)  A row is [W hi | W lo],
// zero beyond its width, with W = 64 for queries and keys (queries carry scale *
// log2 e, so scores come out in powers of two) and 64 or 128 for values.
constexpr int kRows = 128;  // rows of a tile
struct Split {
  __half *q, *k, *v, *g;         // [b][map or head][row][2 W] (q, g: Shape::rows()); g: the output's gradient
  float *fq, *fk, *fv, *fg;      // f of each [b][map or head][tile]
  float *nv, *ng;                // the largest 2-norm of a tile's rows
  int vw;                        // W of v and g
  int64_t qt, kt;                // tiles of a head's queries and keys
};
// 3-D map {2 W, rows, heads} with boxes of 64 columns x 64 rows (128-byte swizzle)
bool split_map(CUtensorMap *m, const __half *base, int w, int64_t rows, int64_t heads);

// Partial results of ranges of keys, joined afterwards: part_ml[(at * 2 + map) *
// splits + split] holds the reference and the sum of the range's exponentials
// (reference -inf: no key), part_o the same times dv the unnormalised output; at
// counts (b, key head, query, head of its group).
struct Parts {
  float *o;
  float2 *ml;
  int splits;
};
// how many ranges of keys the tensor-core forward should take
int tc_forward_splits(tx_ctx *ctx, const Shape &s);
// out, out2 and lse, or with parts.splits > 1 the partial results
int tc_forward(tx_ctx *ctx, const Shape &s, const Split &x, float *out, float *out2, float *lse, const Parts &parts);
// stats [b][h / P][ceil(rows / 64)][4][64]: the log-sum-exp of both maps (+inf behind the last query), D1, D2;
// with P > 1 [5]: lam / 2^E too (lam_exponent)
// sums [b][h / P][tiles of queries][P]: the tiles' sums of D2; dq, dk and dv, dlam are optional
int tc_backward(tx_ctx *ctx, const Shape &s, const Split &x, const float *stats, const float *sums, float *dq,
                float *dk, float *dv, float *dlam);

// ---- device wrappers -------------------------------------------------------------------------
constexpr uint64_t kWaitNs = 2000000000ull;  // 2 s

__device__ __forceinline__ uint32_t su32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t gtime() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void bar_init(uint64_t *b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(n));
}
__device__ __forceinline__ void bar_expect(uint64_t *b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(su32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait.  On expiry (or when another role gave up) false: the role
// leaves its loop, so every role reaches the CTA's last barrier.
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity, volatile int *abort_flag, int *err, int site) {
  if (bar_try(b, parity)) return true;
  const uint64_t t0 = gtime();
  while (true) {
    if (bar_try(b, parity)) return true;
    if (*abort_flag) return false;
    if (gtime() - t0 > kWaitNs) {
      *abort_flag = 1;
      if (atomicCAS(err, 0, DEVERR_TIMEOUT) == 0) err[1] = 200 + site;
      return false;
    }
  }
}
// the same for a whole warp: one answer
__device__ __forceinline__ bool mma_wait(uint64_t *b, uint32_t parity, volatile int *abort_flag, int *err, int site) {
  return __all_sync(0xffffffffu, bar_wait(b, parity, abort_flag, err, site));
}
// whatever the abort flag says: copies and MMAs in flight end before their memory is released
__device__ __forceinline__ void bar_drain(uint64_t *b, uint32_t parity) {
  const uint64_t t0 = gtime();
  while (!bar_try(b, parity) && gtime() - t0 < kWaitNs) {
  }
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, uint64_t *b, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(su32(b)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// plain bulk copy: both addresses and the size multiples of 16 bytes
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *b) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(su32(b))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The MMA warp runs its loop with all lanes, and these instructions under the
// predicate of one: the descriptors then stay in uniform registers (issued from
// a branch of one lane an instruction took 80 to 100 cycles, not the tensor
// core's 64).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one;
}
__device__ __forceinline__ void mma_commit(uint64_t *b, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(su32(b)),
      "r"(one)
      : "memory");
}
// Shared-memory descriptors, 128-byte swizzle, 8-row groups 1024 bytes apart: the low word carries the
// address and the distance of 64-column blocks, the high word is one constant.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// 16-deep slice k of a [rows x 64] fp16 tile read along its columns (K-major)
__device__ __forceinline__ uint32_t kdesc(uint32_t tile, int k) { return ((tile + k * 32) >> 4) | (1u << 16); }
// 16-deep slice k of [K rows x 64 columns] tiles read along their rows (MN-major);
// `next` is the distance between the tiles of neighbouring 64-column blocks
__device__ __forceinline__ uint32_t ndesc(uint32_t tile, int k, uint32_t next) {
  return ((tile + k * 2048) >> 4) | ((next >> 4) << 16);
}
// D[tmem] (+)= A B^T, A in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 da, {%1, %6};\n\t"
      "mov.b64 db, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(one), "r"(kDescHigh)
      : "memory");
}
// the same with A in TMEM (two fp16 a column)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 db, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(one), "r"(kDescHigh)
      : "memory");
}
// fp16 operands, fp32 accumulators, M = 128
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void tld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// keeps every use of loaded registers behind the wait
__device__ __forceinline__ void after_wait(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                 "+r"(r[31]));
}
__device__ __forceinline__ void tst_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 2^x, good to 2^-22
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 values in a register pair, and arithmetic on both at once
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t two(uint32_t a, uint32_t b) { return two(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ void untwo(uint64_t r, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// a pair of fp32 as fp16 heads (the first in the low half) and tails.  The head
// is cut off, not rounded: it needs no conversion back, and the tail keeps the
// cut part to 2^-21 of the value (an operand that meets rounded pairs, so the
// cut's sign does not add up).
__device__ __forceinline__ void cut2(uint64_t v, uint32_t &hi, uint32_t &lo) {
  float a, b, ra, rb;
  untwo(v, a, b);
  const float ha = __uint_as_float(__float_as_uint(a) & 0xffffe000u), hb = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
  untwo(sub2(v, two(ha, hb)), ra, rb);
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(hb), "f"(ha));
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(rb), "f"(ra));
}
// the same with a rounded head: within 2^-22 of the value
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ void tld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void after_wait(uint32_t (&r)[16]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
// 16 keys (rows) of an A operand: heads in columns 0 .. 7, tails in 8 .. 15
__device__ __forceinline__ void tst_pairs(uint32_t taddr, const uint32_t (&hi)[8], const uint32_t (&lo)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16};" ::"r"(taddr),
      "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]), "r"(hi[4]), "r"(hi[5]), "r"(hi[6]), "r"(hi[7]),
      "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]), "r"(lo[4]), "r"(lo[5]), "r"(lo[6]), "r"(lo[7])
      : "memory");
}
// a factor of scores or gradients; neither infinite nor 0, so that nothing times it is NaN
__device__ __forceinline__ float factor2(float a, float b) {
  return fminf(fmaxf(a * b, 1.1754944e-38f), 1.7014118e38f);
}

}  // namespace tx_diff
