// Key/value cache in 8 bits (layout and rules in q8.h): append, read back,
// and attention over it.
//
// Quantisation of a closed block x[16][head_dim] of one head, every step in
// fp32, round to nearest even:
//   a = max |x| over the finite values;  s = a / Q  (Q = 127 or 448; 0 when
//   a < 2^-117, so that 1 / s is finite);  r = 1 / s;
//   code = round(clamp(x * r, -Q, Q)), to an integer or to e4m3.
// NaN is stored as 0 and an infinity as +-Q: an 8-bit code holds neither.
// The product with r instead of a division keeps the writer at one
// multiplication an element; it moves a value across a rounding border only
// within 2^-23 of it.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "common.h"
#include "q8.cuh"
#include "smem.h"

namespace defer {
namespace {

constexpr float kQ8Tiny = 6.018531076210112e-36f;  // 2^-117

// Codes of four values times r. `odd`: the block holds a NaN (stored as 0) or
// an infinity (stored as +-Q); else |x * r| rounds to Q at most. int8: adding
// 3 * 2^22 leaves the rounded number in the low byte.
template <int KIND>
__device__ __forceinline__ uint32_t encode4(float x0, float x1, float x2, float x3, float r, bool odd) {
  float t[4] = {__fmul_rn(x0, r), __fmul_rn(x1, r), __fmul_rn(x2, r), __fmul_rn(x3, r)};
  if (odd) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      t[e] = t[e] == t[e] ? t[e] : 0.0f;
      if (KIND == kQ8Int8) t[e] = fminf(fmaxf(t[e], -127.0f), 127.0f);
    }
  }
  if constexpr (KIND == kQ8Int8) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = __float_as_uint(__fadd_rn(t[e], 12582912.0f));
    return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(t[0], t[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(t[2], t[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
}
// The value of a code byte.
template <int KIND>
__device__ __forceinline__ float decode(uint32_t byte) {
  if constexpr (KIND == kQ8Int8) {
    return (float)(int8_t)byte;
  } else {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
  }
}

// Unit of this warp: block `blk0` (of per_seq), head and K or V `h2`, sequence
// `i`; 4 warps a CTA, and fewer than 2^31 units (grid_of).
__device__ __forceinline__ bool unit_of(int n, int heads2, int per_seq, int& blk0, int& h2, int& i) {
  const unsigned w = blockIdx.x * 4u + (threadIdx.x >> 5);
  const unsigned a = w / (unsigned)per_seq;
  blk0 = (int)(w - a * (unsigned)per_seq);
  i = (int)(a / (unsigned)heads2);
  h2 = (int)(a - (unsigned)i * (unsigned)heads2);
  return i < n;
}

// ------------------------------------------------------------------ append
// Bound by the latency of its loads: 512 tokens, one a sequence, take 8.5 us
// with cold caches; 8 prompts of 666 to 1999 tokens (8B heads, bf16 to e4m3) 33
// us, where the bytes alone would take 10. One warp per (sequence, head, K or
// V, block). It holds the block in registers: 16 bytes of input a lane and
// step, so a step reads 512 contiguous bytes, then the block's largest value by
// shuffles, then the codes. The warp of a sequence's first block also stores
// the open block (the tail): it is the only one that reads the old tail, and it
// does so before it writes.
template <int TYPE, int KIND, int HDMAX, bool EXACT>
__global__ void __launch_bounds__(128, HDMAX <= 64 ? 10 : HDMAX <= 128 ? 7 : 4)
    k_q8_append(Q8View c, Q8Batch b, const int* __restrict__ pos, Q8Rows rk, Q8Rows rv, int aligned, int per_seq) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int VEC = 16 / (int)sizeof(T);             // elements of one step and lane
  constexpr int STEPS = kQ8Block * HDMAX / VEC / 32;  // at the widest head
  const int lane = threadIdx.x & 31;
  int blk0, h2, i;
  if (!unit_of(b.n, 2 * c.kvh, per_seq, blk0, h2, i)) return;
  const Seq s = seq_of(b, c.slots, i);
  if (s.slot < 0) return;
  const int p0 = __ldg(pos + i);
  if (p0 < 0 || p0 > c.cap || s.nrow > c.cap - p0) {
    if (b.status && lane == 0) atomicOr(b.status, (int)kQ8BadRange);
    return;
  }
  if (b.slots) {  // a slot is written by the first sequence that names it
    bool twice = false;
    for (int j = lane; j < i; j += 32) twice |= __ldg(b.slots + j) == s.slot;
    if (__any_sync(0xffffffffu, twice)) {
      if (b.status && lane == 0) atomicOr(b.status, (int)kQ8SlotTwice);
      return;
    }
  }
  const int h = h2 >> 1, hd = EXACT ? HDMAX : c.hd;
  const bool is_v = h2 & 1;
  const T* src = static_cast<const T*>(is_v ? rv.p : rk.p) + (size_t)h * (is_v ? rv.head : rk.head);
  const int64_t ts = is_v ? rv.token : rk.token;
  const size_t sh = (size_t)s.slot * c.kvh + h;
  T* tail = static_cast<T*>(is_v ? c.vt : c.kt) + sh * kQ8Block * hd;
  unsigned char* codes = (is_v ? c.vc : c.kc) + sh * c.cap * hd;
  float* scales = (is_v ? c.vs : c.ks) + sh * (c.cap / kQ8Block);
  const int end = p0 + s.nrow, first = p0 / kQ8Block, open = end / kQ8Block;
  const int vrow = hd / VEC, vblk = kQ8Block * vrow;  // vectors of a row, of a block
  auto load = [&](T(&x)[VEC], const T* p, bool vec) {
    if (vec) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) x[e] = p[e];
    }
  };
  for (int blk = first + blk0; blk < open; blk += per_seq) {  // blocks that close
    __align__(16) T x[STEPS][VEC];
    float a = 0.0f;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
      const int u = j * 32 + lane;
      if (u < vblk) {
        const int r = u / vrow, d = (u - r * vrow) * VEC, p = blk * kQ8Block + r;
        if (p < p0) load(x[j], tail + r * hd + d, true);
        else load(x[j], src + (int64_t)(s.row0 + p - p0) * ts + d, aligned);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float f = fabsf(E::to(x[j][e]));
          const bool fine = f <= FLT_MAX;
          odd |= !fine;
          a = fmaxf(a, fine ? f : 0.0f);
        }
      }
    }
    a = warp_max_all(a);
    odd = __any_sync(0xffffffffu, odd);
    const float sc = a < kQ8Tiny ? 0.0f : __fdiv_rn(a, KIND == kQ8Int8 ? 127.0f : 448.0f);
    const float rc = sc > 0.0f ? __fdiv_rn(1.0f, sc) : 0.0f;
    if (lane == 0) scales[blk] = sc;
    unsigned char* cb = codes + (size_t)blk * kQ8Block * hd;
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
      const int u = j * 32 + lane;
      if (u < vblk) {
        uint32_t o[VEC / 4];
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
          o[e / 4] = encode4<KIND>(E::to(x[j][e]), E::to(x[j][e + 1]), E::to(x[j][e + 2]), E::to(x[j][e + 3]), rc, odd);
        if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(cb + (size_t)u * VEC) = o[0];
        else *reinterpret_cast<uint2*>(cb + (size_t)u * VEC) = make_uint2(o[0], o[1]);
      }
    }
  }
  if (blk0 == 0) {  // the new tokens of the open block
    __syncwarp();   // every lane has read the old tail
    const int from = max(p0, open * kQ8Block);
    for (int u = lane; u < (end - from) * vrow; u += 32) {
      const int r = u / vrow, d = (u - r * vrow) * VEC;
      __align__(16) T x[VEC];
      load(x, src + (int64_t)(s.row0 + from - p0 + r) * ts + d, aligned);
      *reinterpret_cast<uint4*>(tail + (size_t)(from - open * kQ8Block + r) * hd + d) = *reinterpret_cast<uint4*>(x);
    }
  }
}

// -------------------------------------------------------------------- read
// Bound by the bytes: 8 sessions of 3001 to 4096 positions (8B heads, e4m3 to
// bf16) in 32 us, 5.4 TB/s. One warp per (sequence, head, K or V, block); 16
// bytes of output a lane and step, the block's loads sent off together, loads
// and stores past L1.
template <int TYPE, int KIND, int HD>
__global__ void __launch_bounds__(128) k_q8_read(Q8View c, int n, const int* __restrict__ lens,
                                                 const int* __restrict__ start, const int* __restrict__ slots,
                                                 int* status, int rows, Q8Out ok, Q8Out ov, int aligned,
                                                 int per_seq) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int VEC = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  int blk0, h2, i;
  if (!unit_of(n, 2 * c.kvh, per_seq, blk0, h2, i)) return;
  const int slot = slots ? __ldg(slots + i) : i;
  if (slot < 0) return;
  const int len = __ldg(lens + i), p0 = start ? __ldg(start + i) : 0;
  if (slot >= c.slots || len < 0 || len > c.cap || p0 < 0) {
    if (status && lane == 0) atomicOr(status, (int)kQ8BadRange);
    return;
  }
  const int p1 = (int)min((int64_t)len, (int64_t)p0 + rows);
  const int blk = p0 / kQ8Block + blk0;
  if ((int64_t)blk * kQ8Block >= p1) return;
  const int h = h2 >> 1, hd = HD ? HD : c.hd;
  const bool is_v = h2 & 1;
  const Q8Out& o = is_v ? ov : ok;
  T* dst = static_cast<T*>(o.p) + (int64_t)i * o.seq + (int64_t)h * o.head;
  const size_t sh = (size_t)slot * c.kvh + h;
  const T* tail = static_cast<const T*>(is_v ? c.vt : c.kt) + sh * kQ8Block * hd;
  const unsigned char* cb = (is_v ? c.vc : c.kc) + (sh * c.cap + (size_t)blk * kQ8Block) * hd;
  const bool open = blk == len / kQ8Block;
  const float sc = open ? 0.0f : (is_v ? c.vs : c.ks)[sh * (c.cap / kQ8Block) + blk];
  const int vrow = hd / VEC, vblk = kQ8Block * vrow;
  constexpr int PART = HD ? kQ8Block * HD / VEC / 32 : 1;  // steps whose loads are sent off together
#pragma unroll 1
  for (int u0 = lane; u0 < vblk; u0 += 32 * PART) {
    uint32_t q[PART][VEC / 4];
#pragma unroll
    for (int j = 0; j < PART; j++) {
      const size_t at = (size_t)(u0 + 32 * j) * VEC;
      if (open) continue;
      if constexpr (VEC == 4) {
        q[j][0] = __ldcs(reinterpret_cast<const uint32_t*>(cb + at));
      } else {
        const uint2 q2 = __ldcs(reinterpret_cast<const uint2*>(cb + at));
        q[j][0] = q2.x;
        q[j][1] = q2.y;
      }
    }
#pragma unroll
    for (int j = 0; j < PART; j++) {
      const int u = u0 + 32 * j, r = u / vrow, d = (u - r * vrow) * VEC, p = blk * kQ8Block + r;
      if (p < p0 || p >= p1) continue;
      __align__(16) T x[VEC];
      if (open) {
        *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(tail + r * hd + d);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++)
          x[e] = E::from(__fmul_rn(decode<KIND>(q[j][e / 4] >> (8 * (e & 3)) & 0xFFu), sc));
      }
      T* y = dst + (int64_t)(p - p0) * o.token + d;
      if (aligned) {
        __stcs(reinterpret_cast<uint4*>(y), *reinterpret_cast<uint4*>(x));
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) y[e] = x[e];
      }
    }
  }
}

// ------------------------------------------------------------------ attend
// Attention of a few rows of a sequence and key head (all of them where the
// tiles of q8_tile.cu do not serve): 8 or 16 rows read the cache once, and
// everything else is arranged around that stream.
//
// Mathematics. A code is a whole number (or an e4m3 number): exact in fp16,
// so the scores of a block are (codes . q) * s_K and its share of the output
// is (P . codes) * s_V with the scales outside the products, which run on the
// tensor cores (mma m16n8k16, fp32 sums). The other operand is made as exact
// as the cache's type asks: a q row is scaled by a power of two so that its
// largest element is in [2^14, 2^15) and held as one fp16 term (a bf16 or fp16
// row: its own bits, down to elements 2^31 below the row's largest) or two
// (fp32: 22 bits; a third term changes no error that was measured). The weights
// of a block are taken relative to the block's own largest score, P = 2^(x -
// max_block x) (x: score in base 2), times 2^14 in two fp16 terms: 22 bits, with
// one term (11 bits) the errors of 16-bit results are more than their own
// rounding; a weight 2^39 below the block's largest ends. The block's products P . codes come out of the tensor core by themselves and are added to
// fp32 registers times 2^(max_block x - m) s_V, m the running maximum of the
// scores: no block's values, however large, cost the others bits, and nothing
// is summed in a long chain inside the tensor core. The sum of the weights is
// relative to m too. Softmax: running maximum and sum per warp; warps, then
// splits, are merged in order. Values near fp32's largest number would make the
// sum of weights times values infinite where their quotient is not: scales from
// 2^73 on raise a power of two that the warp's output is held in units of.
//
// Work. The positions of the closed blocks are cut into units of 4 warp
// steps, the units into splits, one CTA each, 8 splits of a (sequence, key
// head, row tile) forming a cluster: partial results travel through
// distributed shared memory, and up to 8 splits need no workspace and no
// second launch. The clusters of longer sequences leave theirs in the
// workspace, for k_q8_merge. The number of splits follows from the sequence's
// length and rows alone, so its result does not depend on the batch it runs
// in. A warp loads its steps (4 KB of K and V) straight into the registers of
// the matrix instruction: the order of the dims inside the score product, and
// of the dims of the output, is free, so a thread takes 16 neighbouring bytes
// of a position wherever it can, and nothing of the stream passes through
// shared memory. K is loaded again as soon as its scores are done and V as soon
// as its products are, and every lane asks for one 128-byte line of a step
// further on to be brought into L2, which keeps enough bytes on their way. The
// open block (fp32 or 16-bit tokens) is added at the end by the last split, in
// fp32.
//
// What bounds it: waiting. Of 64 sequences (bf16) an SM issues 1.3 of 4
// instructions a cycle with 20 % of its warps active; the largest stalls are
// the loads (2.5 cycles an instruction) and the cluster's last CTA (2.3). A
// CTA's start, merges and open block take about 5 us beside its steps of 16
// positions and 128 dims. 8 sessions of 4096 positions (8B heads, fp32): 27 us,
// 2.5 TB/s; one sequence of 131077 (bf16): 68 us, 4.0 TB/s; 64 sequences of 129
// to 8191 (bf16): 159 us, 3.5 TB/s; 512 sessions of 16 to 767 (135M heads): 39
// us, 2.2 TB/s. CTAs of 4 warps let 4 of them overlap on an SM: with 8 warps
// (both with cold caches) the 64 sequences take 213 us instead of 164, 127
// sequences of 128 positions 88 instead of 59.
constexpr int kQsWarps = 4;
constexpr int kQsCluster = 8;     // splits of a cluster
constexpr int kQsMaxSplits = 64;  // of a sequence
// Value scales (in the open block: values) from 2^(kQsRoom + 1) on raise the
// unit that the output is summed in: 2^14 weights of 2^30 positions times 448
// scales of less stay below 2^127.
constexpr int kQsRoom = 72;

template <int HDP>
struct QsShape {
  static constexpr int TS = HDP >= 128 ? 16 : 2048 / HDP;  // positions of a warp step
  static constexpr int NG = TS / kQ8Block;                 // blocks of a step
  static constexpr int KS = HDP / 16;                      // k steps of the score product
  static constexpr int UNIT = kQsWarps * TS;               // positions of one step of the CTA
  static constexpr int ORow = HDP + 4;                     // floats of a result row
  static constexpr int KW = HDP / 16, VW = HDP / 32;       // words of K (V) a thread holds of one position
  static constexpr int AHEAD = 4;                          // steps that L2 is asked to bring in advance
};
template <int HDP, int NT, int QT>
constexpr size_t qs_smem() {
  using S = QsShape<HDP>;
  return (size_t)(kQsWarps + 1) * 8 * NT * S::ORow * 4     // results of the warps and of the CTA
         + (size_t)S::KS * NT * QT * 32 * 8                // q
         + (size_t)(8 * NT) * (6 + 3 * kQsWarps) * 4;      // row factors; m, l and unit of the CTA and of the warps
}

// Splits of a sequence of `rows` rows a key head with `closed` positions in
// closed blocks. Up to 16 rows: of 4 units or more (a single short sequence is
// a matter of latency: with cold caches 16 us, 18 with 8 units, for 1041
// positions of the 135M heads), up to the 8 that one cluster merges; of 16 units
// or more when that makes more of them (a CTA's start and its merges cost about
// 5 units: 64 sequences of up to 8191 positions take 164 us, 187 with 8 units).
// More rows are many CTAs anyway: of 8 units or more (512 rows over 2048
// positions of the 135M heads: 60 us, 68 with 4 units).
template <int HDP>
__host__ __device__ __forceinline__ int qs_splits(int closed, int64_t rows) {
  const int units = (closed + QsShape<HDP>::UNIT - 1) / QsShape<HDP>::UNIT;
  const int least = rows > 16 ? 8 : 4;
  const int n = units >= 16 * kQsCluster ? units / 16 : units / least < kQsCluster ? units / least : kQsCluster;
  return n < 1 ? 1 : n > kQsMaxSplits ? kQsMaxSplits : n;
}

// Position (of 8) that row r of the score product stands for: the positions of
// threads c = 0..3 in the value product, rows 2c and 2c + 1, are then
// neighbours.
__device__ __forceinline__ int qs_row(int r) { return (r >> 1) + (r & 1) * 4; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_join() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}
// W = 1, 2 or 4 words, past L1; where `on` is 0 the words stay as they are.
template <int W>
__device__ __forceinline__ void ld_words(uint32_t* w, const unsigned char* p, int on) {
  if constexpr (W == 4)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %5, 0;\n\t"
        "@p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
        : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3])
        : "l"(p), "r"(on));
  else if constexpr (W == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %3, 0;\n\t@p ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n\t}"
        : "+r"(w[0]), "+r"(w[1])
        : "l"(p), "r"(on));
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t@p ld.global.nc.L1::no_allocate.u32 %0, [%1];\n\t}"
                 : "+r"(w[0])
                 : "l"(p), "r"(on));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // 8 x 8 of 16 bits across the warp
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cluster_arrive_wait() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// This CTA's shared address `a` in the CTA of cluster rank `r`.
__device__ __forceinline__ uint32_t peer_addr(uint32_t a, uint32_t r) {
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(r));
  return d;
}
__device__ __forceinline__ float ld_peer(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_peer4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// Weight of a partial result with maximum m under the total's maximum M.
__device__ __forceinline__ float part_weight(float m, float M) { return m == -INFINITY ? 0.0f : ex2(m - M); }
// The output of a row: O in units of 2^(X - 14), L the weights' sum; 0 where nothing is seen.
__device__ __forceinline__ float row_result(float O, float L, int X) {
  return L == 0.0f ? 0.0f : O / (L * 16384.0f) * pow2(X);
}

// EXACT: head_dim is HDP; else HDP is the next instantiated size and the
// dims behind head_dim are zeros that are not read.
template <int TYPE, int KIND, int HDP, int NT, bool EXACT>
__global__ void __launch_bounds__(kQsWarps * 32, HDP == 256 || NT == 2 ? 2 : 4)
    k_q8_attend(const __grid_constant__ Q8View c, const __grid_constant__ Q8Batch b, const __grid_constant__ Q8Attend a,
                int tiles, int groups) {
  using S = QsShape<HDP>;
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int QT = TYPE == kQ8F32 ? 2 : 1;  // terms of q; the weights have two
  constexpr int ROWS = 8 * NT, MT = HDP / 16;
  constexpr int WO = ROWS * S::ORow;  // floats of a warp's result; before that, its tokens of the open block
  constexpr int KL = S::KW < 4 ? S::KW : 4, VL = S::VW < 4 ? S::VW : 4;  // words of one load
  constexpr int OPEN = kQ8Block / kQsWarps;  // tokens of the open block a warp
  static_assert(WO * 4 >= 2 * OPEN * HDP * (int)sizeof(T), "the open block's tokens fit");
  extern __shared__ __align__(128) unsigned char sm[];
  float* wo_all = reinterpret_cast<float*>(sm);
  float* res = wo_all + kQsWarps * WO;                  // [ROWS][ORow]
  uint2* qf = reinterpret_cast<uint2*>(res + WO);
  float* fac = reinterpret_cast<float*>(qf + S::KS * NT * QT * 32);  // [ROWS] row factors
  float* q_down = fac + ROWS;                                         // [ROWS] the power of two that q was raised by
  float* q_rest = q_down + ROWS;                                      // [ROWS] the rest of fac
  float* cm = q_rest + ROWS;                                          // [ROWS] the CTA's m, then l, then unit
  float* wm = cm + 3 * ROWS;                                          // [warps][ROWS] m, then l, then unit
  float* wl = wm + kQsWarps * ROWS;
  int* wx = reinterpret_cast<int*>(wl + kQsWarps * ROWS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, cq = lane & 3;
  const int csize = (int)cluster_size(), rank = (int)cluster_rank();
  // clusters are powers of two; the usual call has one group and one tile
  const int cluster = (int)(blockIdx.x >> (31 - __clz(csize)));
  const int i = groups == 1 ? cluster : (int)((unsigned)cluster / (unsigned)groups), group = cluster - i * groups;
  const int kvh = tiles == 1 ? (int)blockIdx.y : (int)(blockIdx.y / (unsigned)tiles);
  int len = __ldg(a.lens + i);
  const Seq s = seq_of(b, c.slots, i);
  const int G = a.group, R = s.nrow * G;
  if (s.slot == kSeqSkip || R == 0) return;
  // x / G of a row x by a product with 2^32 / G rounded up: exact while x * G < 2^32
  const bool small = R < 1 << 20 && G <= 4096;
  auto token_of = [&](int x) { return G == 1 ? x : small ? (int)__umulhi((unsigned)x, a.group_inv) : x / G; };
  if (s.slot == kSeqBad) len = -1;
  if (a.tiled && R > kQ8FewRows) return;
  T* const out0 = static_cast<T*>(const_cast<void*>(a.out.p));
  if (len < 0 || len > c.cap) {
    if (b.status && tid == 0) atomicOr(b.status, (int)kQ8BadRange);
    for (int x = ((blockIdx.y - kvh * tiles) * groups + group) * csize + rank; x < R; x += tiles * groups * csize)
      for (int d = tid; d < c.hd; d += kQsWarps * 32)
        out0[(int64_t)(s.row0 + x / G) * a.out.token + (int64_t)(kvh * G + x % G) * a.out.head + d] = E::from(NAN);
    return;
  }
  const int hd = EXACT ? HDP : c.hd, closed = len & ~(kQ8Block - 1);
  const int splits = min(qs_splits<HDP>(closed, R), groups * csize);
  const int split = group * kQsCluster + rank, ns = min(splits - group * kQsCluster, csize);  // ns: of the cluster
  if (rank >= ns) return;  // cluster barriers wait for the CTAs that are left
  const size_t sh = (size_t)s.slot * c.kvh + kvh;
  const unsigned char* kc = c.kc + sh * c.cap * hd;
  const unsigned char* vc = c.vc + sh * c.cap * hd;
  const float* ksc = c.ks + sh * (c.cap / kQ8Block);
  const float* vsc = c.vs + sh * (c.cap / kQ8Block);
  const unsigned char* hide = a.masked ? a.masked + (int64_t)i * a.mask_stride : nullptr;
  float* wo = wo_all + warp * WO;
  const int units = (closed + S::UNIT - 1) / S::UNIT;

  for (int tile = blockIdx.y - kvh * tiles; tile * ROWS < R; tile += tiles) {
    const int x0 = tile * ROWS;
    const int jlast = min(x0 + ROWS, R) - 1;
    // positions that the tile's last row sees bound the work of the tile
    const int most = a.causal ? min(len, len - (s.nrow - 1 - token_of(jlast))) : len;
    const int least = a.causal ? len - (s.nrow - 1 - token_of(x0)) : len;  // the first row's
    int u0 = 0, u1 = units;
    if (splits > 1) {
      u0 = (int)((unsigned)(units * split) / (unsigned)splits);
      u1 = (int)((unsigned)(units * (split + 1)) / (unsigned)splits);
    }
    const int t_end = min(min(closed, most), u1 * S::UNIT);
    const int t_first = u0 * S::UNIT + warp * S::TS;
    const int steps = t_end > t_first ? (t_end - t_first + S::UNIT - 1) / S::UNIT : 0;
    // positions of the open block that the warp adds: closed + warp, + kQsWarps, ...
    const int t_open = split == splits - 1 ? min(len, most) - closed - warp : 0;
    const int n_open = t_open > 0 ? (t_open + kQsWarps - 1) / kQsWarps : 0;

    // this thread's words of a step: K of rows r and r + 8, V of 4 positions, of each block
    uint32_t kw[S::NG][2][S::KW] = {}, vw[S::NG][4][S::VW] = {};
    float ks[S::NG] = {}, vs[S::NG] = {};
    const unsigned char* kp = kc + (size_t)(t_first + qs_row(r)) * hd + cq * (HDP >= 64 ? 16 : 8);
    const unsigned char* vp = vc + (size_t)(t_first + cq) * hd + r * (HDP / 8);
    const float *ksp = ksc + t_first / kQ8Block, *vsp = vsc + t_first / kQ8Block;
    // Loads of step `it`; nothing changes when there is none. closed is a
    // multiple of 16: a step of several blocks can end before its last one,
    // whose words are then an earlier step's and whose positions are hidden.
    auto load_k = [&](int it) {
      const int t0 = t_first + it * S::UNIT;
#pragma unroll
      for (int g = 0; g < S::NG; g++) {
        const int on = S::NG == 1 ? it < steps : t0 + g * kQ8Block < t_end;
        if (on) ks[g] = __ldg(ksp + g);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int w = 0; w < S::KW; w += KL)
            ld_words<KL>(kw[g][h] + w, kp + (size_t)(g * 16 + h * 8) * hd + w * 16,
                         on && (EXACT || (w / 4 * 4 + cq) * (HDP >= 64 ? 16 : 8) < hd));
      }
      kp += (size_t)S::UNIT * hd;
      ksp += S::UNIT / kQ8Block;
    };
    auto load_v = [&](int it) {
      const int t0 = t_first + it * S::UNIT;
#pragma unroll
      for (int g = 0; g < S::NG; g++) {
        const int on = S::NG == 1 ? it < steps : t0 + g * kQ8Block < t_end;
        if (on) vs[g] = __ldg(vsp + g);
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int w = 0; w < S::VW; w += VL)
            ld_words<VL>(vw[g][q] + w, vp + (size_t)(g * 16 + (q & 1) * 4 + (q >> 1) * 8) * hd + w * 4,
                         on && (EXACT || r * (HDP / 8) + w * 4 < hd));
      }
      vp += (size_t)S::UNIT * hd;
      vsp += S::UNIT / kQ8Block;
    };
    // The lines of step `it` towards L2, half the lanes K, half V; `it` goes up
    // by one a call. The last lines of a step of several blocks, or of
    // shorter rows, may lie behind the last block: those are left out.
    const int line = (lane & 15) * (S::TS * HDP / 16);
    const unsigned char* pf = (lane < 16 ? kc : vc) + (size_t)(t_first + S::UNIT) * hd + line;
    auto ahead = [&](int it) {
      bool on = it < steps, on2 = on;
      if constexpr (!EXACT || S::NG > 1) {
        const int64_t left = (int64_t)(t_end - t_first - it * S::UNIT) * hd;
        on = line < left;
        on2 = line + 128 < left;
      }
      if (on) asm volatile("prefetch.global.L2 [%0];" ::"l"(pf));
      if constexpr (HDP == 256) {
        if (on2) asm volatile("prefetch.global.L2 [%0];" ::"l"(pf + 128));
      }
      pf += (size_t)S::UNIT * hd;
    };
    load_k(0);
    load_v(0);
#pragma unroll
    for (int it = 1; it < S::AHEAD; it++) ahead(it);
    if (n_open) {
      const int row = hd * (int)sizeof(T) / 16;  // 16-byte chunks of a token
      const uint4* k16 = reinterpret_cast<const uint4*>(static_cast<const T*>(c.kt) + (sh * kQ8Block + warp) * hd);
      const uint4* v16 = reinterpret_cast<const uint4*>(static_cast<const T*>(c.vt) + (sh * kQ8Block + warp) * hd);
      for (int y = 0; y < n_open; y++)
        for (int x = lane; x < row; x += 32) {
          cp16(smem_u32(wo) + (y * row + x) * 16, k16 + y * kQsWarps * row + x);
          cp16(smem_u32(wo) + ((OPEN + y) * row + x) * 16, v16 + y * kQsWarps * row + x);
        }
    }

    // q rows of the tile as score operands, a row a warp
    for (int x = warp; x < ROWS; x += kQsWarps) {
      const bool on = x0 + x < R;
      const int tok = token_of(x0 + x);
      const T* q = static_cast<const T*>(a.q.p) + (int64_t)(s.row0 + tok) * a.q.token +
                   (int64_t)(kvh * G + x0 + x - tok * G) * a.q.head;
      float v[HDP / 32], mx = 0.0f;
#pragma unroll
      for (int e = 0; e < HDP / 32; e++) {
        const int d = e * 32 + lane;
        v[e] = on && d < hd ? E::to(q[d]) : 0.0f;
        mx = fmaxf(mx, fabsf(v[e]));
      }
      mx = warp_max_all(mx);
      // q times 2^up is in [2^14, 2^15) at its largest (less for subnormal
      // rows); a zero, infinite or NaN row is not scaled. The power is
      // applied in two steps: 2^up itself may exceed fp32's range.
      const int up = mx > 0.0f && mx <= FLT_MAX ? 141 - (__float_as_int(mx) >> 23) : 0;  // -113 .. 141
      const float up0 = __int_as_float((127 + up / 2) << 23), up1 = __int_as_float((127 + up - up / 2) << 23);
      if (lane == 0) {
        const float f = a.scale * 1.4426950408889634f;
        fac[x] = f * __int_as_float((127 - up / 2) << 23) * __int_as_float((127 - up + up / 2) << 23);
        q_down[x] = pow2(max(-up, -126));
        q_rest[x] = f * pow2(min(126 - up, 0));
      }
#pragma unroll
      for (int e = 0; e < HDP / 32; e++) {
        const int d = e * 32 + lane;
        const float y = v[e] * up0 * up1;
        const int cc = HDP >= 64 ? d / 16 % 4 : d / 8, w = HDP >= 64 ? d % 16 / 4 : d % 8 / 4, bb = d % 4;
        const int k = HDP >= 64 ? d / 64 * 4 + w : w;
        __half* dst = reinterpret_cast<__half*>(qf + ((k * NT + x / 8) * QT) * 32 + (x % 8) * 4 + cc) + bb;
        const __half hi = __float2half_rn(y);
        dst[0] = hi;
        if constexpr (QT == 2) {
          // an infinite or NaN row keeps it in the first term
          const float lo = y - __half2float(hi);
          dst[32 * 4] = __float2half_rn(lo == lo ? lo : 0.0f);
        }
      }
    }
    __syncthreads();

    float o[MT][NT][4] = {};
    float m[NT][2], l[NT][2], f[NT][2];
    int unit = 0;  // o is in units of 2^(unit - 14)
    int seen[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int x = n * 8 + 2 * cq + e;
        m[n][e] = -INFINITY;
        l[n][e] = 0.0f;
        f[n][e] = fac[x];
        seen[n][e] = x0 + x >= R ? 0 : a.causal ? len - (s.nrow - 1 - token_of(x0 + x)) : len;
      }

    // exponent of a scale over kQsRoom; the same in the whole warp
    auto unit_of_values = [](float v) { return (__float_as_int(v) >> 23) - 127 - kQsRoom; };
    auto move_unit = [&](int to) {
      if (to <= unit) return;
      const float f = pow2(unit - to);
      unit = to;
#pragma unroll
      for (int j = 0; j < MT; j++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[j][n][e] *= f;
    };
    for (int it = 0; it < steps; it++) {
      const int t0 = t_first + it * S::UNIT;
      ahead(it + S::AHEAD);
      // ---- scores of the step's blocks, in base 2
      float sc[S::NG][NT][4];
#pragma unroll
      for (int g = 0; g < S::NG; g++) {
        float s2[NT][4];
#pragma unroll
        for (int k = 0; k < S::KS; k++) {
          const uint32_t x = flip<KIND>(kw[g][0][k]), y = flip<KIND>(kw[g][1][k]);
          const uint32_t af[4] = {halves<KIND, false>(x), halves<KIND, false>(y), halves<KIND, true>(x),
                                  halves<KIND, true>(y)};
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int q = 0; q < QT; q++) {
              const uint2 bf = qf[((k * NT + n) * QT + q) * 32 + lane];
              // two chains: each product waits for the one before it
              if (k == 0 && q == 0) mma16816_zero(sc[g][n], af, bf.x, bf.y);
              else if (k == 1 && q == 0) mma16816_zero(s2[n], af, bf.x, bf.y);
              else mma16816(k & 1 ? s2[n] : sc[g][n], af, bf.x, bf.y);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[g][n][e] = (sc[g][n][e] + s2[n][e]) * (ks[g] * f[n][e & 1]);
      }
      load_k(it + 1);
      if (hide || t0 + S::TS > min(least, closed)) {
#pragma unroll
        for (int g = 0; g < S::NG; g++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int t = t0 + g * 16 + qs_row(r) + (e >> 1) * 8;
            const bool hid = t >= closed || (hide && hide[t]);
#pragma unroll
            for (int n = 0; n < NT; n++)
              if (hid || t >= seen[n][e & 1]) sc[g][n][e] = -INFINITY;
          }
      }
      // ---- the blocks' largest scores, the running maximum, weights, their sum
      uint32_t p[S::NG][NT][2][2];
      float co[S::NG][NT][2];  // what a product of the block counts in the row's output
      {
        float big = vs[0];
#pragma unroll
        for (int g = 1; g < S::NG; g++) big = fmaxf(big, vs[g]);
        if (big >= pow2(kQsRoom + 1)) move_unit(unit_of_values(big));
      }
      const float per_unit = pow2(-unit);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float mb[S::NG][2], al[2];
#pragma unroll
        for (int g = 0; g < S::NG; g++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float mx = fmaxf(sc[g][n][e], sc[g][n][e + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            mb[g][e] = mx;
          }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mn = m[n][e];
#pragma unroll
          for (int g = 0; g < S::NG; g++) mn = fmaxf(mn, mb[g][e]);
          const float ref = mn == -INFINITY ? 0.0f : mn;
          al[e] = ex2(m[n][e] - ref);
          m[n][e] = mn;
#pragma unroll
          for (int g = 0; g < S::NG; g++) co[g][n][e] = ex2(mb[g][e] - ref);
        }
        if (__any_sync(0xffffffffu, !(al[0] == 1.0f && al[1] == 1.0f))) {
#pragma unroll
          for (int e = 0; e < 2; e++) l[n][e] *= al[e];
#pragma unroll
          for (int j = 0; j < MT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[j][n][e] *= al[e & 1];
        }
#pragma unroll
        for (int g = 0; g < S::NG; g++) {
          const float ref0 = mb[g][0] == -INFINITY ? 0.0f : mb[g][0], ref1 = mb[g][1] == -INFINITY ? 0.0f : mb[g][1];
          float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; e += 2) {  // rows r, then r + 8
            float p0 = ex2(sc[g][n][e] - ref0), p1 = ex2(sc[g][n][e + 1] - ref1);
            sum0 += p0;
            sum1 += p1;
            p0 *= 16384.0f;
            p1 *= 16384.0f;
            const __half2 hi = __floats2half2_rn(p0, p1);
            p[g][n][0][e >> 1] = transpose8(h2_bits(hi));
            const float2 back = __half22float2(hi);
            p[g][n][1][e >> 1] = transpose8(h2_bits(__floats2half2_rn(p0 - back.x, p1 - back.y)));
          }
          l[n][0] = fmaf(sum0, co[g][n][0], l[n][0]);
          l[n][1] = fmaf(sum1, co[g][n][1], l[n][1]);
          co[g][n][0] *= vs[g] * per_unit;
          co[g][n][1] *= vs[g] * per_unit;
        }
      }
      // ---- values
#pragma unroll
      for (int g = 0; g < S::NG; g++) {
#pragma unroll
        for (int v = 0; v < S::VW; v++) {
          const uint32_t x0 = flip<KIND>(vw[g][0][v]), x1 = flip<KIND>(vw[g][1][v]);
          const uint32_t y0 = flip<KIND>(vw[g][2][v]), y1 = flip<KIND>(vw[g][3][v]);
#pragma unroll
          for (int h = 0; h < 2; h++) {  // dims 4v + 2h, 4v + 2h + 1 of the thread's
            const uint32_t x = __byte_perm(x0, x1, h ? 0x7362 : 0x5140);
            const uint32_t y = __byte_perm(y0, y1, h ? 0x7362 : 0x5140);
            const uint32_t af[4] = {halves<KIND, false>(x), halves<KIND, true>(x), halves<KIND, false>(y),
                                    halves<KIND, true>(y)};
            const int j = 2 * v + h;
#pragma unroll
            for (int n = 0; n < NT; n++) {
              float d[4];
              mma16816_zero(d, af, p[g][n][0][0], p[g][n][0][1]);
              mma16816(d, af, p[g][n][1][0], p[g][n][1][1]);
#pragma unroll
              for (int e = 0; e < 4; e++) o[j][n][e] = fmaf(d[e], co[g][n][e & 1], o[j][n][e]);
            }
          }
        }
      }
      load_v(it + 1);
    }
    cp_join();
    __syncwarp();

    // ---- the open block: the scores of the warp's tokens, one move of the
    // running maximum for all of them, then their values
    if (n_open) {
      const T* kb = reinterpret_cast<const T*>(wo);
      const T* vb = kb + OPEN * hd + r * (HDP / 8);
      auto quad = [](float (&f)[4], const T* p) {  // 4 elements, 8 or 16 bytes
        __align__(16) T x[4];
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p);
        else *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = E::to(x[e]);
      };
      float lam[OPEN];  // a token's largest value
      bool there[OPEN];
#pragma unroll
      for (int y = 0; y < OPEN; y++) {
        there[y] = y < n_open && !(hide && hide[closed + warp + y * kQsWarps]);
        float vmax = 0.0f;
        if (there[y]) {
#pragma unroll
          for (int d = 0; d < HDP / 8; d += 4)
            if (EXACT || r * (HDP / 8) + d < hd) {
              float f4[4];
              quad(f4, vb + y * hd + d);
#pragma unroll
              for (int e = 0; e < 4; e++) vmax = fmaxf(vmax, fabsf(f4[e]) <= FLT_MAX ? fabsf(f4[e]) : 0.0f);
            }
        }
        lam[y] = vmax;
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1)
#pragma unroll
        for (int y = 0; y < OPEN; y++) lam[y] = fmaxf(lam[y], __shfl_xor_sync(0xffffffffu, lam[y], d));
#pragma unroll
      for (int y = 0; y < OPEN; y++)
        if (lam[y] >= pow2(kQsRoom + 1)) move_unit(unit_of_values(lam[y]));
      const float scale_up = pow2(14 - unit);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float dot[OPEN];  // of row r, over the thread's dims
#pragma unroll
        for (int y = 0; y < OPEN; y++) dot[y] = 0.0f;
#pragma unroll
        for (int k = 0; k < S::KS; k++) {
          const int d0 = HDP >= 64 ? (k / 4 * 4 + cq) * 16 + k % 4 * 4 : cq * 8 + k * 4;
          float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // in its own size: raised, its products with large keys would overflow
          const float down = q_down[n * 8 + r];
#pragma unroll
          for (int x = QT - 1; x >= 0; x--) {
            const uint2 bf = qf[((k * NT + n) * QT + x) * 32 + lane];
            const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&bf.x));
            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&bf.y));
            q[0] += lo.x;
            q[1] += lo.y;
            q[2] += hi.x;
            q[3] += hi.y;
          }
#pragma unroll
          for (int e = 0; e < 4; e++) q[e] *= down;
          if (EXACT || d0 < hd) {
#pragma unroll
            for (int y = 0; y < OPEN; y++)
              if (there[y]) {
                float f4[4];
                quad(f4, kb + y * hd + d0);
#pragma unroll
                for (int e = 0; e < 4; e++) dot[y] = fmaf(q[e], f4[e], dot[y]);
              }
          }
        }
        float w[OPEN][2], al[2];
        bool on[OPEN][2];  // the row sees the token
#pragma unroll
        for (int y = 0; y < OPEN; y++) {
          dot[y] += __shfl_xor_sync(0xffffffffu, dot[y], 1);
          dot[y] += __shfl_xor_sync(0xffffffffu, dot[y], 2);
          dot[y] *= q_rest[n * 8 + r];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float x = __shfl_sync(0xffffffffu, dot[y], (2 * cq + e) * 4);
            on[y][e] = there[y] && closed + warp + y * kQsWarps < seen[n][e];
            w[y][e] = on[y][e] ? x : -INFINITY;
          }
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mn = m[n][e];
#pragma unroll
          for (int y = 0; y < OPEN; y++) mn = fmaxf(mn, w[y][e]);
          const float ref = mn == -INFINITY ? 0.0f : mn;
          al[e] = ex2(m[n][e] - ref);
          l[n][e] *= al[e];
          m[n][e] = mn;
#pragma unroll
          for (int y = 0; y < OPEN; y++) {
            w[y][e] = ex2(w[y][e] - ref);
            if (r == 0) l[n][e] += w[y][e];
            w[y][e] *= scale_up;
          }
        }
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[j][n][e] *= al[e & 1];
#pragma unroll
        for (int y = 0; y < OPEN; y++) {
          if (!there[y]) continue;
#pragma unroll
          for (int d = 0; d < HDP / 8; d += 4)
            if (EXACT || r * (HDP / 8) + d < hd) {
              float f4[4];
              quad(f4, vb + y * hd + d);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const int j = (d + e) / 2, z = e % 2 * 2;
                if (on[y][0]) o[j][n][z] = fmaf(w[y][0], f4[e], o[j][n][z]);
                if (on[y][1]) o[j][n][z + 1] = fmaf(w[y][1], f4[e], o[j][n][z + 1]);
              }
            }
        }
      }
    }

    // ---- merge of the warps, in order
    __syncwarp();  // every lane is done with the tokens in wo
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float x = l[n][e];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        const int row = n * 8 + 2 * cq + e;
        if (r == 0) {
          wm[warp * ROWS + row] = m[n][e];
          wl[warp * ROWS + row] = x;
          wx[warp * ROWS + row] = unit;
        }
#pragma unroll
        for (int j = 0; j < MT; j++)
          *reinterpret_cast<float2*>(wo + row * S::ORow + r * (HDP / 8) + 2 * j) =
              make_float2(o[j][n][e], o[j][n][e + 2]);
      }
    __syncthreads();
    const int rows = min(ROWS, R - x0);
    for (int x = tid; x < rows * (HDP / 4); x += kQsWarps * 32) {
      const int row = x / (HDP / 4), d = x % (HDP / 4) * 4;
      float M = -INFINITY;
      int X = 0;
#pragma unroll
      for (int w = 0; w < kQsWarps; w++) {
        M = fmaxf(M, wm[w * ROWS + row]);
        X = max(X, wx[w * ROWS + row]);
      }
      float L = 0.0f, O[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kQsWarps; w++) {
        float wt = part_weight(wm[w * ROWS + row], M);
        const float4 y = *reinterpret_cast<const float4*>(wo_all + w * WO + row * S::ORow + d);
        // a warp whose maximum is -inf holds zeros, or NaN from a NaN score
        L = fmaf(wt, wl[w * ROWS + row], L);
        wt *= pow2(wx[w * ROWS + row] - X);
        O[0] = fmaf(wt, y.x, O[0]);
        O[1] = fmaf(wt, y.y, O[1]);
        O[2] = fmaf(wt, y.z, O[2]);
        O[3] = fmaf(wt, y.w, O[3]);
      }
      *reinterpret_cast<float4*>(res + row * S::ORow + d) = make_float4(O[0], O[1], O[2], O[3]);
      if (d == 0) {
        cm[row] = M;
        cm[ROWS + row] = L;
        cm[2 * ROWS + row] = __int_as_float(X);
      }
    }
    // ---- merge of the splits, in order; the rows' dims are dealt out over the cluster
    if (csize > 1) cluster_arrive_wait();
    else __syncthreads();
    {
      const uint32_t res_u = smem_u32(res), cm_u = smem_u32(cm);
      for (int x = rank * kQsWarps * 32 + tid; x < rows * (HDP / 4); x += ns * kQsWarps * 32) {
        const int row = x / (HDP / 4), d = x % (HDP / 4) * 4;
        if (d >= hd) continue;
        float L, M, O[4];
        int X;
        if (ns > 1) {
          M = -INFINITY;
          X = 0;
#pragma unroll 4
          for (int q = 0; q < ns; q++) {
            M = fmaxf(M, ld_peer(peer_addr(cm_u + row * 4, q)));
            X = max(X, __float_as_int(ld_peer(peer_addr(cm_u + (2 * ROWS + row) * 4, q))));
          }
          L = O[0] = O[1] = O[2] = O[3] = 0.0f;
#pragma unroll 4
          for (int q = 0; q < ns; q++) {
            float wt = part_weight(ld_peer(peer_addr(cm_u + row * 4, q)), M);
            const float4 y = ld_peer4(peer_addr(res_u + (row * S::ORow + d) * 4, q));
            L = fmaf(wt, ld_peer(peer_addr(cm_u + (ROWS + row) * 4, q)), L);
            wt *= pow2(__float_as_int(ld_peer(peer_addr(cm_u + (2 * ROWS + row) * 4, q))) - X);
            O[0] = fmaf(wt, y.x, O[0]);
            O[1] = fmaf(wt, y.y, O[1]);
            O[2] = fmaf(wt, y.z, O[2]);
            O[3] = fmaf(wt, y.w, O[3]);
          }
        } else {
          M = cm[row];
          L = cm[ROWS + row];
          X = __float_as_int(cm[2 * ROWS + row]);
#pragma unroll
          for (int e = 0; e < 4; e++) O[e] = res[row * S::ORow + d + e];
        }
        const int tok = token_of(x0 + row), token = s.row0 + tok, head = kvh * G + x0 + row - tok * G;
        if (splits > kQsCluster) {  // merged with the other clusters' by k_q8_merge
          float* y = a.ws + (((size_t)token * a.heads + head) * groups + group) * (hd + 4);
          *reinterpret_cast<float4*>(y + d) = make_float4(O[0], O[1], O[2], O[3]);
          if (d == 0) {
            y[hd] = M;
            y[hd + 1] = L;
            y[hd + 2] = __int_as_float(X);
          }
          continue;
        }
        T* y = out0 + (int64_t)token * a.out.token + (int64_t)head * a.out.head + d;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = E::from(row_result(O[e], L, X));
      }
    }
    if (csize > 1) cluster_arrive_wait();  // peers are done with this CTA's result
    else __syncthreads();
  }
}

// Merge of the clusters' results of sequences of more than kQsCluster splits,
// in order: one warp per row and head, 4 dims a lane and step.
template <int TYPE, int HDP>
__global__ void __launch_bounds__(128) k_q8_merge(Q8View c, Q8Batch b, Q8Attend a, int groups) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (int64_t)b.tokens * a.heads) return;
  const int token = (int)(w / a.heads), head = (int)(w % a.heads);
  int i;
  if (b.q_start) {
    int lo = 0, hi = b.n;  // the last i with q_start[i] <= token
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (__ldg(b.q_start + mid) <= token) lo = mid;
      else hi = mid;
    }
    i = lo;
  } else {
    i = token / (b.tokens / b.n);
  }
  const Seq s = seq_of(b, c.slots, i);
  const int len = __ldg(a.lens + i);
  if (s.slot < 0 || token < s.row0 || token >= s.row0 + s.nrow || len < 0 || len > c.cap) return;
  if (a.tiled && s.nrow * (a.heads / c.kvh) > kQ8FewRows) return;
  const int splits =
      min(qs_splits<HDP>(len & ~(kQ8Block - 1), (int64_t)s.nrow * (a.heads / c.kvh)), groups * kQsCluster);
  if (splits <= kQsCluster) return;
  const int n = (splits + kQsCluster - 1) / kQsCluster;
  const float* y = a.ws + (size_t)w * groups * (c.hd + 4);
  float M = -INFINITY;
  int X = 0;
  for (int g = 0; g < n; g++) {
    M = fmaxf(M, y[g * (c.hd + 4) + c.hd]);
    X = max(X, __float_as_int(y[g * (c.hd + 4) + c.hd + 2]));
  }
  for (int d = lane * 4; d < c.hd; d += 128) {
    float L = 0.0f, O[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int g = 0; g < n; g++) {
      const float* z = y + g * (c.hd + 4);
      float wt = part_weight(z[c.hd], M);
      const float4 x = *reinterpret_cast<const float4*>(z + d);
      L = fmaf(wt, z[c.hd + 1], L);
      wt *= pow2(__float_as_int(z[c.hd + 2]) - X);
      O[0] = fmaf(wt, x.x, O[0]);
      O[1] = fmaf(wt, x.y, O[1]);
      O[2] = fmaf(wt, x.z, O[2]);
      O[3] = fmaf(wt, x.w, O[3]);
    }
    T* out = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)token * a.out.token + (int64_t)head * a.out.head + d;
#pragma unroll
    for (int e = 0; e < 4; e++) out[e] = E::from(row_result(O[e], L, X));
  }
}

// ------------------------------------------------------------------- host
bool aligned16(const void* p, int64_t s0, int64_t s1, int64_t s2, int esize) {
  return (reinterpret_cast<uintptr_t>(p) % 16 | (uint64_t)(s0 * esize) % 16 | (uint64_t)(s1 * esize) % 16 |
          (uint64_t)(s2 * esize) % 16) == 0;
}
int esize_of(int type) { return type == kQ8F32 ? 4 : 2; }

unsigned grid_of(int64_t warps) {
  if (warps >= INT32_MAX) fail(kInvalidArgument, "8-bit cache: too many sequences, heads and blocks in one call");
  return (unsigned)((warps + 3) / 4);
}

// f(type constant, kind constant)
template <int V>
struct Const {
  static constexpr int value = V;
};
template <class F>
void dispatch(const Q8View& c, F&& f) {
  auto by_kind = [&](auto type) {
    if (c.kind == kQ8Int8) f(type, Const<kQ8Int8>());
    else f(type, Const<kQ8E4m3>());
  };
  if (c.type == kQ8F32) by_kind(Const<kQ8F32>());
  else if (c.type == kQ8Bf16) by_kind(Const<kQ8Bf16>());
  else by_kind(Const<kQ8F16>());
}

}  // namespace

void q8_append(const Q8View& c, const Q8Batch& b, const int* pos, const Q8Rows& k, const Q8Rows& v, cudaStream_t st) {
  if (b.n == 0 || b.tokens == 0) return;
  const int es = esize_of(c.type);
  const int al = aligned16(k.p, k.token, k.head, 0, es) && aligned16(v.p, v.token, v.head, 0, es);
  // a sequence of q rows touches at most (q + 15 + 15) / 16 blocks
  const int per_seq = (std::min(b.max_q, c.cap) + 2 * kQ8Block - 2) / kQ8Block;
  const unsigned grid = grid_of((int64_t)b.n * 2 * c.kvh * per_seq);
  dispatch(c, [&](auto type, auto kind) {
    constexpr int TY = decltype(type)::value, KI = decltype(kind)::value;
    auto kern = c.hd == 64    ? k_q8_append<TY, KI, 64, true>
                : c.hd == 128 ? k_q8_append<TY, KI, 128, true>
                : c.hd <= 128 ? k_q8_append<TY, KI, 128, false>
                              : k_q8_append<TY, KI, 256, false>;
    kern<<<grid, 128, 0, st>>>(c, b, pos, k, v, al, per_seq);
  });
  DEFER_CUDA(cudaGetLastError());
}

void q8_read(const Q8View& c, int n, const int* lens, const int* start, const int* slots, int* status, int rows,
             const Q8Out& k, const Q8Out& v, cudaStream_t st) {
  if (n == 0 || rows == 0) return;
  const int es = esize_of(c.type);
  const int al = aligned16(k.p, k.seq, k.token, k.head, es) && aligned16(v.p, v.seq, v.token, v.head, es);
  const int most = std::min(rows, c.cap);
  const int per_seq = start ? (most + 2 * kQ8Block - 2) / kQ8Block : (most + kQ8Block - 1) / kQ8Block;
  const unsigned grid = grid_of((int64_t)n * 2 * c.kvh * per_seq);
  dispatch(c, [&](auto type, auto kind) {
    constexpr int TY = decltype(type)::value, KI = decltype(kind)::value;
    auto kern = c.hd == 64 ? k_q8_read<TY, KI, 64> : c.hd == 128 ? k_q8_read<TY, KI, 128> : k_q8_read<TY, KI, 0>;
    kern<<<grid, 128, 0, st>>>(c, n, lens, start, slots, status, rows, k, v, al, per_seq);
  });
  DEFER_CUDA(cudaGetLastError());
}

namespace {

template <int TYPE, int KIND, int HDP, int NT, bool EXACT>
void attend_few(const Q8View& c, const Q8Batch& b, const Q8Attend& a, cudaStream_t st) {
  auto kern = k_q8_attend<TYPE, KIND, HDP, NT, EXACT>;
  constexpr size_t smem = qs_smem<HDP, NT, TYPE == kQ8F32 ? 2 : 1>();
  static SmemLimit limit;
  limit.ensure([&] { SmemLimit::allow(kern, smem); });
  int64_t rows = (int64_t)std::max(b.max_q, 1) * (a.heads / c.kvh);
  if (a.tiled) rows = std::min<int64_t>(rows, kQ8FewRows);
  const int64_t tiles = std::min<int64_t>((rows + 8 * NT - 1) / (8 * NT), 65535 / c.kvh);
  // of the longest sequence, which with q_start may have few rows
  const int splits = qs_splits<HDP>(a.max_len / kQ8Block * kQ8Block, b.q_start ? 1 : rows);
  const int groups = (splits + kQsCluster - 1) / kQsCluster;
  int cl = 1;  // a power of two that holds its splits
  while (cl < std::min(splits, kQsCluster)) cl *= 2;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(b.n * groups * cl), (unsigned)(c.kvh * tiles), 1);
  cfg.blockDim = dim3(kQsWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  DEFER_CUDA(cudaLaunchKernelEx(&cfg, kern, c, b, a, (int)tiles, groups));
  if (groups > 1) k_q8_merge<TYPE, HDP><<<grid_of((int64_t)b.tokens * a.heads), 128, 0, st>>>(c, b, a, groups);
}

}  // namespace

namespace {
thread_local struct {
  int role;
  unsigned wait_us;
} drill;
}  // namespace

void q8_stall_next(int role, unsigned wait_us) {
  drill.role = role;
  drill.wait_us = wait_us;
}

size_t q8_attend_workspace(const Q8View& c, const Q8Batch& b, const Q8Attend& a) {
  if (!b.q_start && q8_tiles(c, b, a)) return 0;
  const int closed = a.max_len / kQ8Block * kQ8Block;
  const int64_t rows = b.q_start ? 1 : (int64_t)std::max(b.max_q, 1) * (a.heads / c.kvh);
  const int splits = c.hd <= 32    ? qs_splits<32>(closed, rows)
                     : c.hd <= 64  ? qs_splits<64>(closed, rows)
                     : c.hd <= 128 ? qs_splits<128>(closed, rows)
                                   : qs_splits<256>(closed, rows);
  if (splits <= kQsCluster) return 0;
  return (size_t)b.tokens * a.heads * ((splits + kQsCluster - 1) / kQsCluster) * (c.hd + 4) * sizeof(float);
}

void q8_attend(const Q8View& c, const Q8Batch& b, const Q8Attend& args, cudaStream_t st) {
  if (b.n == 0 || b.tokens == 0) return;
  Q8Attend a = args;
  a.out_aligned = aligned16(a.out.p, a.out.token, a.out.head, 0, esize_of(c.type));
  a.q_aligned = aligned16(a.q.p, a.q.token, a.q.head, 0, esize_of(c.type));
  a.group = a.heads / c.kvh;
  a.group_inv = (unsigned)(0xFFFFFFFFull / (unsigned)a.group + 1);
  a.tiled = q8_tiles(c, b, a);
  a.wait_ns = 2000000000ull;
  a.stall = 0;
  if (a.tiled) {
    if (drill.role) {
      a.stall = drill.role;
      a.wait_ns = drill.wait_us * 1000ull;
      drill.role = 0;
    }
    q8_attend_tiles(c, b, a, st);
    if (!b.q_start) return;  // every sequence has the same number of rows: none is left
  }
  const bool one = (int64_t)b.max_q * (a.heads / c.kvh) <= 8;
  dispatch(c, [&](auto type, auto kind) {
    constexpr int TY = decltype(type)::value, KI = decltype(kind)::value;
    auto go = [&](auto hdp, auto exact) {
      constexpr int HDP = decltype(hdp)::value;
      constexpr bool EX = decltype(exact)::value != 0;
      if (one || HDP == 256) attend_few<TY, KI, HDP, 1, EX>(c, b, a, st);
      else attend_few<TY, KI, HDP, HDP == 256 ? 1 : 2, EX>(c, b, a, st);
    };
    if (c.hd == 64) go(Const<64>(), Const<1>());
    else if (c.hd == 128) go(Const<128>(), Const<1>());
    else if (c.hd <= 32) go(Const<32>(), Const<0>());
    else if (c.hd <= 64) go(Const<64>(), Const<0>());
    else if (c.hd <= 128) go(Const<128>(), Const<0>());
    else go(Const<256>(), Const<0>());
  });
  DEFER_CUDA(cudaGetLastError());
}

}  // namespace defer
