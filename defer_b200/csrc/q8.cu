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
#include "q8.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "common.h"

namespace defer {
namespace {

constexpr float kQ8Tiny = 6.018531076210112e-36f;  // 2^-117

// ------------------------------------------------------------- elements
template <int TYPE>
struct Elem;
template <>
struct Elem<kQ8F32> {
  using T = float;
  static __device__ __forceinline__ float to(float x) { return x; }
  static __device__ __forceinline__ float from(float x) { return x; }
};
template <>
struct Elem<kQ8Bf16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to(T x) { return __bfloat162float(x); }
  static __device__ __forceinline__ T from(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Elem<kQ8F16> {
  using T = __half;
  static __device__ __forceinline__ float to(T x) { return __half2float(x); }
  static __device__ __forceinline__ T from(float x) { return __float2half_rn(x); }
};

// Code byte of t = x * r, and the value of a code byte.
template <int KIND>
__device__ __forceinline__ uint32_t encode(float t) {
  t = t == t ? t : 0.0f;
  if constexpr (KIND == kQ8Int8) {
    return (uint32_t)__float2int_rn(fminf(fmaxf(t, -127.0f), 127.0f)) & 0xFFu;
  } else {
    return (uint32_t)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
  }
}
template <int KIND>
__device__ __forceinline__ float decode(uint32_t byte) {
  if constexpr (KIND == kQ8Int8) {
    return (float)(int8_t)byte;
  } else {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
  }
}

__device__ __forceinline__ float warp_max_all(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// Sequence i of a call: its slot and its rows. kSeqSkip: padding or rows out
// of range, nothing is touched; kSeqBad: valid rows of a bad slot.
constexpr int kSeqSkip = -1, kSeqBad = -2;
struct Seq {
  int slot, row0, nrow;
};
__device__ __forceinline__ Seq seq_of(const Q8Batch& b, int slots, int i) {
  Seq s;
  s.slot = b.slots ? max(__ldg(b.slots + i), kSeqSkip) : i;
  if (s.slot >= slots) {
    if (b.status) atomicOr(b.status, (int)kQ8BadRange);
    s.slot = kSeqBad;
  }
  if (b.q_start) {
    s.row0 = __ldg(b.q_start + i);
    const int end = __ldg(b.q_start + i + 1);
    s.nrow = end - s.row0;
    if (s.row0 < 0 || end < s.row0 || end > b.tokens) {
      if (b.status) atomicOr(b.status, (int)kQ8BadRange);
      s.slot = kSeqSkip;
    }
  } else {
    s.nrow = b.tokens / b.n;
    s.row0 = i * s.nrow;
  }
  return s;
}

// ------------------------------------------------------------------ append
// One warp per (sequence, head, K or V, block). It holds the block in
// registers: 16 bytes of input a lane and step, so a step reads 512
// contiguous bytes, then the block's largest value by shuffles, then the
// codes. The warp of a sequence's first block also stores the open block
// (the tail): it is the only one that reads the old tail, and it does so
// before it writes.
template <int TYPE, int KIND, int HDMAX>
__global__ void __launch_bounds__(128) k_q8_append(Q8View c, Q8Batch b, const int* __restrict__ pos, Q8Rows rk,
                                                   Q8Rows rv, int aligned, int per_seq) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int VEC = 16 / (int)sizeof(T);             // elements of one step and lane
  constexpr int STEPS = kQ8Block * HDMAX / VEC / 32;  // at the widest head
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int heads2 = 2 * c.kvh;
  if (w >= (int64_t)b.n * heads2 * per_seq) return;
  const int blk0 = (int)(w % per_seq), h2 = (int)(w / per_seq % heads2), i = (int)(w / per_seq / heads2);
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
  const int h = h2 >> 1, hd = c.hd;
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
          a = fmaxf(a, f <= FLT_MAX ? f : 0.0f);
        }
      }
    }
    a = warp_max_all(a);
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
          o[e / 4] = encode<KIND>(__fmul_rn(E::to(x[j][e]), rc)) | encode<KIND>(__fmul_rn(E::to(x[j][e + 1]), rc)) << 8 |
                     encode<KIND>(__fmul_rn(E::to(x[j][e + 2]), rc)) << 16 |
                     encode<KIND>(__fmul_rn(E::to(x[j][e + 3]), rc)) << 24;
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
// One warp per (sequence, head, K or V, block); 16 bytes of output a lane
// and step, stored past L1.
template <int TYPE, int KIND>
__global__ void __launch_bounds__(128) k_q8_read(Q8View c, int n, const int* __restrict__ lens,
                                                 const int* __restrict__ start, const int* __restrict__ slots,
                                                 int* status, int rows, Q8Out ok, Q8Out ov, int aligned,
                                                 int per_seq) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int VEC = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int heads2 = 2 * c.kvh;
  if (w >= (int64_t)n * heads2 * per_seq) return;
  const int blk0 = (int)(w % per_seq), h2 = (int)(w / per_seq % heads2), i = (int)(w / per_seq / heads2);
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
  const int h = h2 >> 1, hd = c.hd;
  const bool is_v = h2 & 1;
  const Q8Out& o = is_v ? ov : ok;
  T* dst = static_cast<T*>(o.p) + (int64_t)i * o.seq + (int64_t)h * o.head;
  const size_t sh = (size_t)slot * c.kvh + h;
  const T* tail = static_cast<const T*>(is_v ? c.vt : c.kt) + sh * kQ8Block * hd;
  const unsigned char* cb = (is_v ? c.vc : c.kc) + (sh * c.cap + (size_t)blk * kQ8Block) * hd;
  const bool open = blk == len / kQ8Block;
  const float sc = open ? 0.0f : (is_v ? c.vs : c.ks)[sh * (c.cap / kQ8Block) + blk];
  const int vrow = hd / VEC, vblk = kQ8Block * vrow;
#pragma unroll 4
  for (int u = lane; u < vblk; u += 32) {
    const int r = u / vrow, d = (u - r * vrow) * VEC, p = blk * kQ8Block + r;
    if (p < p0 || p >= p1) continue;
    __align__(16) T x[VEC];
    if (open) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(tail + r * hd + d);
    } else {
      uint32_t q[VEC / 4];
      if constexpr (VEC == 4) {
        q[0] = __ldg(reinterpret_cast<const uint32_t*>(cb + (size_t)u * VEC));
      } else {
        const uint2 q2 = __ldg(reinterpret_cast<const uint2*>(cb + (size_t)u * VEC));
        q[0] = q2.x;
        q[1] = q2.y;
      }
#pragma unroll
      for (int e = 0; e < VEC; e++)
        x[e] = E::from(__fmul_rn(decode<KIND>(q[e / 4] >> (8 * (e & 3)) & 0xFFu), sc));
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

// ------------------------------------------------------------------ attend
// Attention of a few rows (q8_few_rows) of a sequence and key head: the cache
// is read once, and everything else is arranged around that stream.
//
// Mathematics. A code is a whole number (or an e4m3 number): exact in fp16,
// so the scores of a block are (codes . q) * s_K and its share of the output
// is (P . codes) * s_V with the scales outside the products, which run on the
// tensor cores (mma m16n8k16, fp32 sums). The other operand is made as exact
// as the cache's type asks: a q row is scaled by a power of two so that its
// largest element is in [2^14, 2^15) and held as one fp16 term (bf16 and fp16
// rows: no bit lost) or two (fp32: 22 bits); P is kept times 2^15, so that
// weights down to 2^-29 of the largest are full fp16 numbers, and held the
// same way. Products of one block of 16 positions are summed by the tensor
// core from zero and added to the running sums in fp32 registers: long chains
// inside the tensor core lose bits. Softmax: running maximum and sum per warp
// in base 2; warps, then splits, are merged in order.
//
// Work. The positions of the closed blocks are cut into units of 8 warp
// steps, the units into splits, one CTA each, the splits of a (sequence, key
// head, row tile) forming a cluster: partial results travel through
// distributed shared memory, so the call needs no workspace and no second
// launch. The number of splits follows from the sequence's length alone, so
// its result does not depend on the batch it runs in. Each warp streams its
// own steps (4 KB of K and V) through a ring of its own with 16-byte
// asynchronous copies, without any barrier; chunks are swizzled so that both
// the row-wise reads of K and the column-wise reads of V are free of bank
// conflicts. The open block (fp32 or 16-bit tokens) is added at the end by
// the last split, a token a warp, in fp32.
constexpr int kQsWarps = 8;
constexpr int kQsMaxSplits = 16;
constexpr int kQsMinUnits = 2;  // units of a split, when there are as many

template <int HDP>
struct QsShape {
  static constexpr int TS = HDP >= 128 ? 16 : 2048 / HDP;  // positions of a warp step
  static constexpr int NG = TS / kQ8Block;                 // blocks of a step
  static constexpr int CH = HDP / 16;                      // 16-byte chunks of a row
  static constexpr int KS = HDP / 16;                      // k steps of the score product
  static constexpr int STAGES = HDP == 256 ? 2 : 3;
  static constexpr int KBYTES = TS * HDP;
  static constexpr int STAGE = 2 * KBYTES + 2 * NG * 4 + (32 - 2 * NG * 4 % 32) % 32;  // codes, scales, pad
  static constexpr int OPENV = STAGE / 32 * 16;            // where the open block's values start
  static constexpr int UNIT = kQsWarps * TS;               // positions of one step of the CTA
  static constexpr int ORow = HDP + 4;                     // floats of a result row
};
template <int HDP, int NT, int QT>
constexpr size_t qs_smem() {
  using S = QsShape<HDP>;
  return (size_t)kQsWarps * S::STAGES * S::STAGE          // rings (later the warps' results)
         + (size_t)S::KS * NT * QT * 32 * 8               // q
         + (size_t)(8 * NT) * S::ORow * 4                 // the CTA's result
         + (size_t)(8 * NT) * (3 + 2 * kQsWarps) * 4;     // row factors, m and l of the CTA and of the warps
}

// Splits of a sequence with `closed` positions in closed blocks.
template <int HDP>
__host__ __device__ __forceinline__ int qs_splits(int closed) {
  const int n = (closed + QsShape<HDP>::UNIT - 1) / QsShape<HDP>::UNIT / kQsMinUnits;
  return n < 1 ? 1 : n > kQsMaxSplits ? kQsMaxSplits : n;
}

// Byte offset of 16-byte chunk `ch` of position `t` in a step's K or V. The
// exclusive-or keeps a 128-byte phase of both access patterns on 32 banks: K
// is read by 8 threads as 2 neighbouring rows x 4 chunks (or whole rows), V as
// rows 2c (or 2c + 1), c = 0..3, x neighbouring chunks.
template <int HDP>
__device__ __forceinline__ int qs_chunk(int t, int ch) {
  if constexpr (HDP == 256) return t * 256 + ((ch ^ ((t >> 1 & 1) | (((t >> 2) ^ t) & 1) << 2)) << 4);
  else if constexpr (HDP == 128) return t * 128 + ((ch ^ ((t & 6) ^ (t & 1) << 2)) << 4);
  else if constexpr (HDP == 64) return (t >> 1) * 128 + ((((t & 1) * 4 + ch) ^ ((t >> 1 & 3) * 2)) << 4);
  else return (t >> 2) * 128 + ((((t & 3) * 2 + ch) ^ ((t >> 2 & 1) * 2)) << 4);
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp16 numbers from code bytes (SEL: the prmt selector that puts two
// bytes x, y as x . y . into 16-bit lanes). int8: the byte with its sign bit
// flipped is x + 128; 0x6400 | u is 1024 + u, so one subtraction of 1152
// leaves x, exactly. `w` comes from flip<KIND>.
template <int KIND>
__device__ __forceinline__ uint32_t flip(uint32_t w) {
  return KIND == kQ8Int8 ? w ^ 0x80808080u : w;
}
template <int KIND, bool HI>
__device__ __forceinline__ uint32_t halves(uint32_t w) {
  if constexpr (KIND == kQ8Int8) {
    const uint32_t u = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
    return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480))));
  } else {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(HI ? w >> 16 : w & 0xFFFFu), __NV_E4M3);
    return h2_bits(__half2(h));
  }
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

// Weight of a partial result with maximum m under the total's maximum M.
__device__ __forceinline__ float part_weight(float m, float M) { return m == -INFINITY ? 0.0f : ex2(m - M); }

template <int TYPE, int KIND, int HDP, int NT>
__global__ void __launch_bounds__(kQsWarps * 32, HDP == 256 ? 1 : 2)
    k_q8_attend(const __grid_constant__ Q8View c, const __grid_constant__ Q8Batch b, const __grid_constant__ Q8Attend a,
                int tiles) {
  using S = QsShape<HDP>;
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int QT = TYPE == kQ8F32 ? 2 : 1, ROWS = 8 * NT, MT = HDP / 16, KW = HDP / 16;
  extern __shared__ __align__(128) unsigned char sm[];
  uint2* qf = reinterpret_cast<uint2*>(sm + (size_t)kQsWarps * S::STAGES * S::STAGE);
  float* res = reinterpret_cast<float*>(qf + S::KS * NT * QT * 32);  // [ROWS][ORow]
  float* fac = res + ROWS * S::ORow;                                  // [ROWS] row factors
  float* cm = fac + ROWS;                                             // [ROWS] the CTA's m, then l
  float* wm = cm + 2 * ROWS;                                          // [warps][ROWS] m, then [warps][ROWS] l
  float* wl = wm + kQsWarps * ROWS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, cq = lane & 3;
  const int csize = (int)cluster_size(), rank = (int)cluster_rank();
  const int i = blockIdx.x / csize;
  const int kvh = blockIdx.y / tiles;
  int len = __ldg(a.lens + i);
  const Seq s = seq_of(b, c.slots, i);
  const int G = a.heads / c.kvh, R = s.nrow * G;
  if (s.slot == kSeqSkip || R == 0) return;
  if (s.slot == kSeqBad) len = -1;
  T* const out0 = static_cast<T*>(const_cast<void*>(a.out.p));
  if (len < 0 || len > c.cap) {
    if (b.status && tid == 0) atomicOr(b.status, (int)kQ8BadRange);
    for (int x = (blockIdx.y - kvh * tiles) * csize + rank; x < R; x += tiles * csize)
      for (int d = tid; d < c.hd; d += kQsWarps * 32)
        out0[(int64_t)(s.row0 + x / G) * a.out.token + (int64_t)(kvh * G + x % G) * a.out.head + d] = E::from(NAN);
    return;
  }
  const int hd = c.hd, closed = len & ~(kQ8Block - 1);
  const int ns = min(qs_splits<HDP>(closed), csize);
  if (rank >= ns) return;  // cluster barriers wait for the CTAs that are left
  const size_t sh = (size_t)s.slot * c.kvh + kvh;
  const unsigned char* kc = c.kc + sh * c.cap * hd;
  const unsigned char* vc = c.vc + sh * c.cap * hd;
  const float* ksc = c.ks + sh * (c.cap / kQ8Block);
  const float* vsc = c.vs + sh * (c.cap / kQ8Block);
  const unsigned char* hide = a.masked ? a.masked + (int64_t)i * a.mask_stride : nullptr;
  unsigned char* ring = sm + (size_t)warp * S::STAGES * S::STAGE;
  const uint32_t ring_u = smem_u32(ring);
  const int units = (closed + S::UNIT - 1) / S::UNIT;

  for (int tile = blockIdx.y - kvh * tiles; tile * ROWS < R; tile += tiles) {
    const int x0 = tile * ROWS;
    const int jlast = min(x0 + ROWS, R) - 1;
    // positions that the tile's last row sees bound the work of the tile
    const int most = a.causal ? min(len, len - (s.nrow - 1 - jlast / G)) : len;
    const int least = a.causal ? len - (s.nrow - 1 - x0 / G) : len;  // the first row's
    const int u0 = (int)((int64_t)units * rank / ns), u1 = (int)((int64_t)units * (rank + 1) / ns);
    const int t_end = min(min(closed, most), u1 * S::UNIT);
    const int t_first = u0 * S::UNIT + warp * S::TS;
    const int steps = t_end > t_first ? (t_end - t_first + S::UNIT - 1) / S::UNIT : 0;
    // positions of the open block that the warp adds: closed + warp (+ 8)
    const int t_open = rank == ns - 1 ? min(len, most) - closed - warp : 0;
    const int n_open = t_open > kQsWarps ? 2 : t_open > 0 ? 1 : 0;

    // Step `it` of the warp into ring slot `st`; the last one is the open block's.
    const int lt = lane / S::CH, lch = lane % S::CH;  // the lane's position and chunk in a copy of 32 chunks
    const unsigned char* kp = kc + ((size_t)t_first + lt) * hd + lch * 16;
    const unsigned char* vp = vc + ((size_t)t_first + lt) * hd + lch * 16;
    const bool lane_on = lch * 16 < hd;
    auto issue = [&](int it, int st) {
      const uint32_t base = ring_u + st * S::STAGE;
      if (it < steps) {
        const int t0 = t_first + it * S::UNIT;
#pragma unroll
        for (int e = 0; e < S::TS * S::CH / 32; e++) {
          const int t = e * (32 / S::CH) + lt;
          // closed is a multiple of 16: only a step of several blocks can end before its last
          const bool on = lane_on && (S::NG == 1 || t0 + t < closed);
          const size_t o = on ? (size_t)(e * (32 / S::CH)) * hd : 0;
          const uint32_t d = base + qs_chunk<HDP>(t, lch);
          cp16(d, on ? kp + o : kc, on);
          cp16(d + S::KBYTES, on ? vp + o : vc, on);
        }
        kp += (size_t)S::UNIT * hd;
        vp += (size_t)S::UNIT * hd;
        if (lane < 2 * S::NG) {
          const int g = lane % S::NG;
          const bool on = t0 + g * kQ8Block < closed;
          cp4(base + 2 * S::KBYTES + lane * 4, (lane < S::NG ? ksc : vsc) + (on ? t0 / kQ8Block + g : 0), on);
        }
      } else if (it == steps && n_open) {
        const int row = hd * (int)sizeof(T) / 16;  // chunks of a token
        const uint4* k16 = reinterpret_cast<const uint4*>(static_cast<const T*>(c.kt) + (sh * kQ8Block + warp) * hd);
        const uint4* v16 = reinterpret_cast<const uint4*>(static_cast<const T*>(c.vt) + (sh * kQ8Block + warp) * hd);
        for (int x = lane; x < n_open * row; x += 32) {
          const int y = x < row ? x : x + (kQsWarps - 1) * row;  // the second token is 8 rows on
          cp16(base + x * 16, k16 + y, true);
          cp16(base + S::OPENV + x * 16, v16 + y, true);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int st = 0; st < S::STAGES - 1; st++) issue(st, st);

    // q rows of the tile as score operands: warp w takes rows w, w + 8
    for (int x = warp; x < ROWS; x += kQsWarps) {
      const bool on = x0 + x < R;
      const T* q = static_cast<const T*>(a.q.p) + (int64_t)(s.row0 + (x0 + x) / G) * a.q.token +
                   (int64_t)(kvh * G + (x0 + x) % G) * a.q.head;
      float v[HDP / 32], mx = 0.0f;
#pragma unroll
      for (int e = 0; e < HDP / 32; e++) {
        const int d = e * 32 + lane;
        v[e] = on && d < hd ? E::to(q[d]) : 0.0f;
        mx = fmaxf(mx, fabsf(v[e]));
      }
      mx = warp_max_all(mx);
      // up = 2^(14 - exponent of mx); a zero, infinite or NaN row is not scaled
      int ex = 0;
      if (mx > 0.0f && mx <= FLT_MAX) {
        frexpf(mx, &ex);  // mx in [2^(ex - 1), 2^ex)
        ex = 15 - ex;
      }
      // the power is applied in two steps: 2^ex itself may exceed fp32's range
      const float up0 = ldexpf(1.0f, ex / 2), up1 = ldexpf(1.0f, ex - ex / 2);
      if (lane == 0) fac[x] = a.scale * 1.4426950408889634f / up0 / up1;
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
    int seen[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int x = n * 8 + 2 * cq + e;
        m[n][e] = -INFINITY;
        l[n][e] = 0.0f;
        f[n][e] = fac[x];
        seen[n][e] = x0 + x >= R ? 0 : a.causal ? len - (s.nrow - 1 - (x0 + x) / G) : len;
      }

    int st = 0;
    for (int it = 0; it < steps; it++) {
      const int t0 = t_first + it * S::UNIT;
      cp_wait<S::STAGES - 2>();
      __syncwarp();  // the step has landed for every lane, and every lane is done with the last one
      issue(it + S::STAGES - 1, st == 0 ? S::STAGES - 1 : st - 1);
      const unsigned char* kb = ring + st * S::STAGE;
      const unsigned char* vb = kb + S::KBYTES;
      const float* scl = reinterpret_cast<const float*>(kb + 2 * S::KBYTES);
      st = st + 1 == S::STAGES ? 0 : st + 1;
      // ---- scores of the step's blocks, in base 2
      float sc[S::NG][NT][4];
#pragma unroll
      for (int g = 0; g < S::NG; g++) {
        uint32_t w0[KW < 4 ? KW : 4], w1[KW < 4 ? KW : 4];
#pragma unroll
        for (int k = 0; k < S::KS; k++) {
          if constexpr (HDP >= 64) {
            if (k % 4 == 0) {
              *reinterpret_cast<uint4*>(w0) =
                  *reinterpret_cast<const uint4*>(kb + qs_chunk<HDP>(g * 16 + r, k + cq));
              *reinterpret_cast<uint4*>(w1) =
                  *reinterpret_cast<const uint4*>(kb + qs_chunk<HDP>(g * 16 + r + 8, k + cq));
            }
          } else if (k == 0) {
            *reinterpret_cast<uint2*>(w0) =
                *reinterpret_cast<const uint2*>(kb + qs_chunk<HDP>(g * 16 + r, cq >> 1) + (cq & 1) * 8);
            *reinterpret_cast<uint2*>(w1) =
                *reinterpret_cast<const uint2*>(kb + qs_chunk<HDP>(g * 16 + r + 8, cq >> 1) + (cq & 1) * 8);
          }
          const uint32_t x = flip<KIND>(w0[k % 4]), y = flip<KIND>(w1[k % 4]);
          const uint32_t af[4] = {halves<KIND, false>(x), halves<KIND, false>(y), halves<KIND, true>(x),
                                  halves<KIND, true>(y)};
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int q = 0; q < QT; q++) {
              const uint2 bf = qf[((k * NT + n) * QT + q) * 32 + lane];
              if (k == 0 && q == 0) mma16816_zero(sc[g][n], af, bf.x, bf.y);
              else mma16816(sc[g][n], af, bf.x, bf.y);
            }
        }
        const float ks = scl[g];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[g][n][e] *= ks * f[n][e & 1];
      }
      if (hide || t0 + S::TS > min(least, closed)) {
#pragma unroll
        for (int g = 0; g < S::NG; g++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int t = t0 + g * 16 + r + (e >> 1) * 8;
            const bool hid = t >= closed || (hide && hide[t]);
#pragma unroll
            for (int n = 0; n < NT; n++)
              if (hid || t >= seen[n][e & 1]) sc[g][n][e] = -INFINITY;
          }
      }
      // ---- running maximum, weights (times 2^15) and their sum
      uint32_t p[S::NG][NT][QT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float ref[2], al[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mx = fmaxf(sc[0][n][e], sc[0][n][e + 2]);
#pragma unroll
          for (int g = 1; g < S::NG; g++) mx = fmaxf(mx, fmaxf(sc[g][n][e], sc[g][n][e + 2]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m[n][e], mx);
          ref[e] = mn == -INFINITY ? 0.0f : mn;
          al[e] = ex2(m[n][e] - ref[e]);
          m[n][e] = mn;
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
        for (int g = 0; g < S::NG; g++)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {  // position r, then r + 8
            const float p0 = ex2(sc[g][n][e] - ref[0]) * 32768.0f, p1 = ex2(sc[g][n][e + 1] - ref[1]) * 32768.0f;
            l[n][0] += p0;
            l[n][1] += p1;
            const __half2 hi = __floats2half2_rn(p0, p1);
            p[g][n][0][e >> 1] = transpose8(h2_bits(hi));
            if constexpr (QT == 2) {
              const float2 back = __half22float2(hi);
              p[g][n][1][e >> 1] = transpose8(h2_bits(__floats2half2_rn(p0 - back.x, p1 - back.y)));
            }
          }
      }
      // ---- values
#pragma unroll
      for (int g = 0; g < S::NG; g++) {
        const float vs15 = scl[S::NG + g] * 3.0517578125e-05f;
        constexpr int VW = HDP / 32;                 // words of a thread and position
        constexpr int VL = VW < 4 ? VW : 4;          // of one load
#pragma unroll
        for (int w0 = 0; w0 < VW; w0 += VL) {
          uint32_t w[4][VL];
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int t = g * 16 + 2 * cq + (q & 1) + (q >> 1) * 8;
            if constexpr (HDP == 256)
              *reinterpret_cast<uint4*>(w[q]) = *reinterpret_cast<const uint4*>(vb + qs_chunk<HDP>(t, 2 * r + w0 / 4));
            else if constexpr (HDP == 128)
              *reinterpret_cast<uint4*>(w[q]) = *reinterpret_cast<const uint4*>(vb + qs_chunk<HDP>(t, r));
            else if constexpr (HDP == 64)
              *reinterpret_cast<uint2*>(w[q]) =
                  *reinterpret_cast<const uint2*>(vb + qs_chunk<HDP>(t, r >> 1) + (r & 1) * 8);
            else
              w[q][0] = *reinterpret_cast<const uint32_t*>(vb + qs_chunk<HDP>(t, r >> 2) + (r & 3) * 4);
          }
#pragma unroll
          for (int v = 0; v < VL; v++) {
            const uint32_t x0 = flip<KIND>(w[0][v]), x1 = flip<KIND>(w[1][v]);
            const uint32_t y0 = flip<KIND>(w[2][v]), y1 = flip<KIND>(w[3][v]);
#pragma unroll
            for (int h = 0; h < 2; h++) {  // dims 4v + 2h, 4v + 2h + 1 of the thread's
              const uint32_t x = __byte_perm(x0, x1, h ? 0x7362 : 0x5140);
              const uint32_t y = __byte_perm(y0, y1, h ? 0x7362 : 0x5140);
              const uint32_t af[4] = {halves<KIND, false>(x), halves<KIND, true>(x), halves<KIND, false>(y),
                                      halves<KIND, true>(y)};
              const int j = 2 * (w0 + v) + h;
#pragma unroll
              for (int n = 0; n < NT; n++) {
                float d[4];
                mma16816_zero(d, af, p[g][n][0][0], p[g][n][0][1]);
                if constexpr (QT == 2) mma16816(d, af, p[g][n][1][0], p[g][n][1][1]);
#pragma unroll
                for (int e = 0; e < 4; e++) o[j][n][e] = fmaf(d[e], vs15, o[j][n][e]);
              }
            }
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();

    // ---- the open block
    {
      const T* kb = reinterpret_cast<const T*>(ring + st * S::STAGE);
      const T* vb = reinterpret_cast<const T*>(ring + st * S::STAGE + S::OPENV) + r * (HDP / 8);
      for (int y = 0; y < n_open; y++) {
        const int t = closed + warp + y * kQsWarps;
        if (hide && hide[t]) continue;
        const T *kr = kb + y * hd, *vr = vb + y * hd;
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float dot = 0.0f;  // of row r, over the thread's dims
#pragma unroll
          for (int k = 0; k < S::KS; k++) {
            const int d0 = HDP >= 64 ? (k / 4 * 4 + cq) * 16 + k % 4 * 4 : cq * 8 + k * 4;
            float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
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
            if (d0 < hd) {
#pragma unroll
              for (int e = 0; e < 4; e++) dot = fmaf(q[e], E::to(kr[d0 + e]), dot);
            }
          }
          dot += __shfl_xor_sync(0xffffffffu, dot, 1);
          dot += __shfl_xor_sync(0xffffffffu, dot, 2);
          dot *= fac[n * 8 + r];
          float w[2], al[2];
          bool on[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float x = __shfl_sync(0xffffffffu, dot, (2 * cq + e) * 4);
            on[e] = t < seen[n][e];
            const float mn = on[e] ? fmaxf(m[n][e], x) : m[n][e];
            const float ref = mn == -INFINITY ? 0.0f : mn;
            al[e] = ex2(m[n][e] - ref);
            w[e] = on[e] ? ex2(x - ref) : 0.0f;
            m[n][e] = mn;
            l[n][e] = l[n][e] * al[e] + (r == 0 ? w[e] * 32768.0f : 0.0f);
          }
#pragma unroll
          for (int j = 0; j < MT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int d = 2 * j + (e >> 1);
              const float v = r * (HDP / 8) + d < hd ? E::to(vr[d]) : 0.0f;
              const float y = o[j][n][e] * al[e & 1];
              o[j][n][e] = on[e & 1] ? fmaf(w[e & 1], v, y) : y;
            }
        }
      }
    }

    // ---- merge of the warps, in order
    __syncwarp();  // every lane is done with the ring
    float* wo = reinterpret_cast<float*>(ring);  // [ROWS][ORow]
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
#pragma unroll
      for (int w = 0; w < kQsWarps; w++) M = fmaxf(M, wm[w * ROWS + row]);
      float L = 0.0f, O[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kQsWarps; w++) {
        const float wt = part_weight(wm[w * ROWS + row], M);
        const float4 y = *reinterpret_cast<const float4*>(sm + (size_t)w * S::STAGES * S::STAGE +
                                                          (row * S::ORow + d) * sizeof(float));
        // a warp whose maximum is -inf holds zeros, or NaN from a NaN score
        L = fmaf(wt, wl[w * ROWS + row], L);
        O[0] = fmaf(wt, y.x, O[0]);
        O[1] = fmaf(wt, y.y, O[1]);
        O[2] = fmaf(wt, y.z, O[2]);
        O[3] = fmaf(wt, y.w, O[3]);
      }
      *reinterpret_cast<float4*>(res + row * S::ORow + d) = make_float4(O[0], O[1], O[2], O[3]);
      if (d == 0) {
        cm[row] = M;
        cm[ROWS + row] = L;
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
        float L, O[4];
        if (ns > 1) {
          float M = -INFINITY;
#pragma unroll 4
          for (int q = 0; q < ns; q++) M = fmaxf(M, ld_peer(peer_addr(cm_u + row * 4, q)));
          L = O[0] = O[1] = O[2] = O[3] = 0.0f;
#pragma unroll 4
          for (int q = 0; q < ns; q++) {
            const float wt = part_weight(ld_peer(peer_addr(cm_u + row * 4, q)), M);
            const float4 y = ld_peer4(peer_addr(res_u + (row * S::ORow + d) * 4, q));
            L = fmaf(wt, ld_peer(peer_addr(cm_u + (ROWS + row) * 4, q)), L);
            O[0] = fmaf(wt, y.x, O[0]);
            O[1] = fmaf(wt, y.y, O[1]);
            O[2] = fmaf(wt, y.z, O[2]);
            O[3] = fmaf(wt, y.w, O[3]);
          }
        } else {
          L = cm[ROWS + row];
#pragma unroll
          for (int e = 0; e < 4; e++) O[e] = res[row * S::ORow + d + e];
        }
        // O is sum p v, L is 2^15 sum p; nothing seen: L = 0
        T* y = out0 + (int64_t)(s.row0 + (x0 + row) / G) * a.out.token + (int64_t)(kvh * G + (x0 + row) % G) * a.out.head + d;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = E::from(L == 0.0f ? 0.0f : O[e] / (L * 3.0517578125e-05f));
      }
    }
    if (csize > 1) cluster_arrive_wait();  // peers are done with this CTA's result
    else __syncthreads();
  }
}

// ------------------------------------------------------------------- host
bool aligned16(const void* p, int64_t s0, int64_t s1, int64_t s2, int esize) {
  return (reinterpret_cast<uintptr_t>(p) % 16 | (uint64_t)(s0 * esize) % 16 | (uint64_t)(s1 * esize) % 16 |
          (uint64_t)(s2 * esize) % 16) == 0;
}
int esize_of(int type) { return type == kQ8F32 ? 4 : 2; }

unsigned grid_of(int64_t warps) {
  const int64_t g = (warps + 3) / 4;
  if (g > INT32_MAX) fail(kInvalidArgument, "8-bit cache: too many sequences and heads in one call");
  return (unsigned)g;
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
    if (c.hd <= 64) k_q8_append<TY, KI, 64><<<grid, 128, 0, st>>>(c, b, pos, k, v, al, per_seq);
    else if (c.hd <= 128) k_q8_append<TY, KI, 128><<<grid, 128, 0, st>>>(c, b, pos, k, v, al, per_seq);
    else k_q8_append<TY, KI, 256><<<grid, 128, 0, st>>>(c, b, pos, k, v, al, per_seq);
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
    k_q8_read<decltype(type)::value, decltype(kind)::value>
        <<<grid, 128, 0, st>>>(c, n, lens, start, slots, status, rows, k, v, al, per_seq);
  });
  DEFER_CUDA(cudaGetLastError());
}

namespace {

// Kernel attributes are set once per device.
bool first_on_device(unsigned long long& mask) {
  int dev = 0;
  DEFER_CUDA(cudaGetDevice(&dev));
  const unsigned long long bit = 1ull << (dev & 63);
  if (mask & bit) return false;
  mask |= bit;
  return true;
}

template <int TYPE, int KIND, int HDP, int NT>
void attend_few(const Q8View& c, const Q8Batch& b, const Q8Attend& a, cudaStream_t st) {
  auto kern = k_q8_attend<TYPE, KIND, HDP, NT>;
  constexpr size_t smem = qs_smem<HDP, NT, TYPE == kQ8F32 ? 2 : 1>();
  static unsigned long long attr = 0;
  if (first_on_device(attr)) {
    DEFER_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    DEFER_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  }
  const int64_t rows = (int64_t)std::max(b.max_q, 1) * (a.heads / c.kvh);
  const int64_t tiles = std::min<int64_t>((rows + 8 * NT - 1) / (8 * NT), 65535 / c.kvh);
  int cl = 1;  // a power of two that holds the splits of the longest sequence
  while (cl < qs_splits<HDP>(a.max_len / kQ8Block * kQ8Block)) cl *= 2;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  // a cluster's CTAs on as many SMs as there are, not two on one: a single
  // long sequence has fewer CTAs than the device has SMs
  at[1].id = cudaLaunchAttributeClusterSchedulingPolicyPreference;
  at[1].val.clusterSchedulingPolicyPreference = cudaClusterSchedulingPolicySpread;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(b.n * cl), (unsigned)(c.kvh * tiles), 1);
  cfg.blockDim = dim3(kQsWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  DEFER_CUDA(cudaLaunchKernelEx(&cfg, kern, c, b, a, (int)tiles));
}

}  // namespace

void q8_attend(const Q8View& c, const Q8Batch& b, const Q8Attend& a, cudaStream_t st) {
  if (b.n == 0 || b.tokens == 0) return;
  const bool one = (int64_t)b.max_q * (a.heads / c.kvh) <= 8;
  dispatch(c, [&](auto type, auto kind) {
    constexpr int TY = decltype(type)::value, KI = decltype(kind)::value;
    if (c.hd <= 32) one ? attend_few<TY, KI, 32, 1>(c, b, a, st) : attend_few<TY, KI, 32, 2>(c, b, a, st);
    else if (c.hd <= 64) one ? attend_few<TY, KI, 64, 1>(c, b, a, st) : attend_few<TY, KI, 64, 2>(c, b, a, st);
    else if (c.hd <= 128) one ? attend_few<TY, KI, 128, 1>(c, b, a, st) : attend_few<TY, KI, 128, 2>(c, b, a, st);
    else attend_few<TY, KI, 256, 1>(c, b, a, st);
  });
  DEFER_CUDA(cudaGetLastError());
}

}  // namespace defer
