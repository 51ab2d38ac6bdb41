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
// One CTA per query row and head: pieces of 128 positions, a score a thread,
// then the weighted values a dimension (or two) a thread, with the running
// maximum and sum of the softmax.
template <int TYPE, int KIND>
__global__ void __launch_bounds__(128) k_q8_attend(Q8View c, Q8Batch b, Q8Attend a) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  __shared__ float qs[kQ8MaxHeadDim], ps[128], red[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, head = blockIdx.y, hd = c.hd;
  int i;
  if (b.q_start) {
    int lo = 0, hi = b.n;  // the last i with q_start[i] <= row
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (__ldg(b.q_start + mid) <= row) lo = mid;
      else hi = mid;
    }
    i = lo;
  } else {
    i = row / (b.tokens / b.n);
  }
  const Seq s = seq_of(b, c.slots, i);
  const int j = row - s.row0;
  if (s.slot == kSeqSkip || j < 0 || j >= s.nrow) return;
  const int len = s.slot == kSeqBad ? -1 : __ldg(a.lens + i);
  T* out = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)row * a.out.token + (int64_t)head * a.out.head;
  if (len < 0 || len > c.cap) {
    if (b.status && tid == 0) atomicOr(b.status, (int)kQ8BadRange);
    for (int d = tid; d < hd; d += 128) out[d] = E::from(NAN);
    return;
  }
  const int seen = a.causal ? len - (s.nrow - 1 - j) : len;
  const T* q = static_cast<const T*>(a.q.p) + (int64_t)row * a.q.token + (int64_t)head * a.q.head;
  for (int d = tid; d < hd; d += 128) qs[d] = E::to(q[d]);
  __syncthreads();
  const size_t sh = (size_t)s.slot * c.kvh + head / (a.heads / c.kvh);
  const int closed = len / kQ8Block * kQ8Block;
  float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int t0 = 0; t0 < seen; t0 += 128) {
    const int t = t0 + tid;
    float sc = -INFINITY;
    if (t < seen && !(a.masked && a.masked[(int64_t)i * a.mask_stride + t])) {
      float dot = 0.0f;
      if (t < closed) {
        const unsigned char* k = c.kc + (sh * c.cap + t) * hd;
        for (int d = 0; d < hd; d++) dot = fmaf(qs[d], decode<KIND>(k[d]), dot);
        dot *= c.ks[sh * (c.cap / kQ8Block) + t / kQ8Block];
      } else {
        const T* k = static_cast<const T*>(c.kt) + (sh * kQ8Block + t - closed) * hd;
        for (int d = 0; d < hd; d++) dot = fmaf(qs[d], E::to(k[d]), dot);
      }
      sc = dot * a.scale;
    }
    float mx = warp_max_all(sc);
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(m, mx);
    const float w = m == -INFINITY ? 0.0f : expf(m - mn);
    ps[tid] = sc == -INFINITY ? 0.0f : expf(sc - mn);
    m = mn;
    __syncthreads();
    l *= w;
    acc[0] *= w;
    acc[1] *= w;
    const int tn = min(128, seen - t0);
    for (int u = 0; u < tn; u++) {
      const float p = ps[u];
      if (p == 0.0f) continue;  // a hidden position's value is not touched
      l += p;
      const int tt = t0 + u;
      for (int e = 0; e < 2; e++) {
        const int d = tid + e * 128;
        if (d >= hd) break;
        float v;
        if (tt < closed)
          v = decode<KIND>(c.vc[(sh * c.cap + tt) * hd + d]) * c.vs[sh * (c.cap / kQ8Block) + tt / kQ8Block];
        else
          v = E::to(static_cast<const T*>(c.vt)[(sh * kQ8Block + tt - closed) * hd + d]);
        acc[e] = fmaf(p, v, acc[e]);
      }
    }
    __syncthreads();
  }
  for (int e = 0; e < 2; e++)
    if (tid + e * 128 < hd) out[tid + e * 128] = E::from(l > 0.0f || l != l ? acc[e] / l : 0.0f);
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

void q8_attend(const Q8View& c, const Q8Batch& b, const Q8Attend& a, cudaStream_t st) {
  if (b.n == 0 || b.tokens == 0) return;
  const dim3 grid(b.tokens, a.heads);
  dispatch(c, [&](auto type, auto kind) {
    k_q8_attend<decltype(type)::value, decltype(kind)::value><<<grid, 128, 0, st>>>(c, b, a);
  });
  DEFER_CUDA(cudaGetLastError());
}

}  // namespace defer
