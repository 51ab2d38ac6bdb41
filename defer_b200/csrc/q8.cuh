// Device pieces that the kernels of the 8-bit cache share (q8.cu, q8_tile.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "q8.h"

namespace defer {
namespace {

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

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// Exponent of a value scale (floor of its base-2 logarithm), from -100 up.
__device__ __forceinline__ float scale_exponent(float v) {
  return (float)max((__float_as_int(v) >> 23) - 127, -100);
}

}  // namespace
}  // namespace defer
