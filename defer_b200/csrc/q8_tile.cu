// Attention over the 8-bit cache for many rows of a sequence (a prompt's
// piece): tiles of 128 rows x 128 positions on the 5th-generation tensor
// cores, 16-bit caches with head_dim up to 128.
//
// Mathematics: the one of k_q8_attend (q8.cu) at this size. Codes are exact
// fp16 operands; a q row is scaled by a power of two into fp16. The products
// with the values stay in tensor memory from block to block, so the weights
// carry the value scales: P' = 2^(x - m) s_V 2^(10 - D), where m follows the
// maximum of the scores x and m + D that of x + floor(log2 s_V). m is moved
// when the maximum has grown by 2^16, D when the other one has by 2^4 (P' stays
// below 2^15): the output is rescaled a few times a row instead of at every
// tile. The sum of the weights is relative to m alone, so no size of the values
// takes bits from it. A weight ends at 2^-25, 2^-35 of the row's largest weight
// times value scale: where one block's values are 2^20 times the others', those
// keep 15 bits, where they are 2^30 times, 5. The tokens of the open
// block are 16-bit numbers: scaled by a power of two for the block they are fp16
// operands like codes, values with their largest at 2^6, like a code, or as far
// up as 2^15 where their smallest need it. fp16 tokens lose no bit by that; of a
// bf16 token, an element 2^32 times smaller than the block's largest begins to
// (fp16 numbers end at 2^-24), as does an element of a bf16 q row 2^31 times
// smaller than the row's largest. At 2^15 the block's weights end 2^9 earlier
// than other blocks'. Weights are two fp16 terms (22 bits). Output and sums stay in fp32 (tensor memory, registers): the
// chain of 512 sums over 4096 positions may be some 2^-16 off, 2^-7 of a bf16
// result's rounding, 2^-4 of an fp16 one's.
//
// Work: a CTA takes two tiles of 128 rows (rows of the heads that share a key
// head, token after token), so that a converted block of 128 positions feeds
// two products and one tile's softmax runs beside the other's products. Warps
// 0-3 and 4-7: softmax of one tile each, a row a thread; warps 8-11 and 12-15
// turn the codes of K and of V into fp16 in shared memory (two stages each,
// no-swizzle core matrices: K read K-major, V MN-major, so both are stored
// alike and nothing is transposed); warp 16 issues the products. Tensor memory holds two
// score tiles and two outputs (512 columns); the weights overwrite the scores
// they came from and are the A operand from there. The order of the products
// (PV of tile 0, scores of tile 0 of the next block, the same of tile 1) keeps
// every buffer's reuse behind its last reader without a wait of its own.
// What bounds it: the way of a tile from its scores over the softmax to its
// products and back, with the other tile's products in between: a block of 128
// positions takes about 4.7 us for two tiles, of which the products are 2.2 at
// full rate (three products' worth: the weights have two terms). Four prompt
// pieces of 170 to 512 rows over 1024 to 4096 positions (8B heads, bf16): 278
// us, 279 TFLOP/s without the second term's products. With one term of the
// weights it was 194 us; then, converting warps shared by K and V took 230, one
// tile a CTA 277.
// Every wait is bounded: one that runs out fills the rows with NaN, sets
// kQ8Timeout in the status word and lets the CTA free its tensor memory.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "common.h"
#include "q8.cuh"
#include "smem.h"

namespace defer {
namespace {

constexpr int kQtM = 128;          // rows of a tile
constexpr int kQtN = 128;          // positions of a block
constexpr int kQtThreads = 17 * 32;
constexpr unsigned long long kQtDrainNs = 2000000000ull;
constexpr int kQtSlots = 4;        // ring of scales and masks
// A weight's operand is 2^(x - m) s_V 2^(kQtUnit - D), where x + log2 s_V is at
// most m + D + kQtLagD + 1: below 2^15.
constexpr int kQtUnit = 10;
constexpr float kQtLagD = 4.0f, kQtLagM = 16.0f;
constexpr float kQtLeast = -100.0f;  // D of a row that has seen nothing; scale_exponent's least

// Scales and masks of one block of positions.
struct QtScales {
  float ks[kQtN / kQ8Block];    // K scale
  float vs[kQtN / kQ8Block];    // V scale
  float lam[kQtN / kQ8Block];   // its exponent
  uint32_t show[kQtN / 32];     // bit per position: exists and is not hidden
};

// How long a wait of the CTA may take, and whether one has run out.
struct QtLimit {
  unsigned long long ns;
  int failed;
};
template <int HDT>
struct QtShared {
  unsigned char q[2][kQtM * HDT * 2];   // fp16 operands in core matrices
  unsigned char k[2][kQtN * HDT * 2];
  unsigned char v[2][kQtN * HDT * 2];
  QtScales sc[kQtSlots];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], sc_full[kQtSlots];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], drain;
  uint32_t tmem;
  QtLimit limit;
  int open_odd;          // the open block's values hold a NaN or an infinity
  float red[2][3][4];
  int red_odd[2][4];
  float fac[2 * kQtM];   // row factors
};

__device__ __forceinline__ unsigned long long qt_time() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void qb_init(uint64_t* b, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void qb_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ bool qb_try(uint64_t* b, unsigned parity) {
  unsigned ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait for the phase of `parity`; false when it ran out or another
// role of the CTA has given up.
__device__ __forceinline__ bool qb_wait(uint64_t* b, unsigned parity, QtLimit* limit) {
  if (qb_try(b, parity)) return true;
  const unsigned long long t0 = qt_time();
  for (unsigned spins = 1; !qb_try(b, parity); spins++) {
    if ((spins & 63u) == 0) {
      if (*(volatile int*)&limit->failed) return false;
      if (qt_time() - t0 > limit->ns) {
        *(volatile int*)&limit->failed = 1;
        return false;
      }
    }
  }
  return true;
}

// Shared-memory matrix descriptor without swizzle. K-major operands: lbo is
// the stride of 16-byte chunks along K, sbo of groups of 8 rows; MN-major: sbo
// is the stride of 16-byte chunks along N, lbo of groups of 8 along K.
__device__ __forceinline__ uint64_t qt_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
         (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46;
}
// Instruction descriptor of kind::f16: fp16 A and B, fp32 D, 128 rows, n columns.
template <int N, bool B_MN>
constexpr uint32_t kQtIdesc = (1u << 4) | (B_MN ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kQtM >> 4) << 24);
__device__ __forceinline__ void qt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void qt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void qt_commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b))
               : "memory");
}
__device__ __forceinline__ void qt_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void qt_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void qt_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define QT_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define QT_W8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
// 32 columns of the warp's 32 lanes; the registers hold them after tm_wait.
__device__ __forceinline__ void tm_ld32(uint32_t (&v)[32], uint32_t a) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : QT_R8(v, 0), QT_R8(v, 8), QT_R8(v, 16), QT_R8(v, 24)
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t (&v)[16], uint32_t a) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : QT_R8(v, 0), QT_R8(v, 8)
      : "r"(a)
      : "memory");
}
#define QT_RW8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
__device__ __forceinline__ void tm_wait(uint32_t (&v)[32]) {  // every load of the thread; v is used only behind it
  asm volatile("tcgen05.wait::ld.sync.aligned;" : QT_RW8(v, 0), QT_RW8(v, 8), QT_RW8(v, 16), QT_RW8(v, 24) : : "memory");
}
__device__ __forceinline__ void tm_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : QT_RW8(v, 0), QT_RW8(v, 8) : : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t a, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
      QT_W8(v, 0), QT_W8(v, 8), QT_W8(v, 16), QT_W8(v, 24)
      : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      QT_W8(v, 0), QT_W8(v, 8)
      : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two fp32 numbers in one register pair, and the operations on both at once.
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void f2_get(uint64_t d, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }
// Exponent of a positive finite number, subnormals as -126.
__device__ __forceinline__ int exponent_of(float x) { return max((__float_as_int(x) >> 23) - 127, -126); }

template <int TYPE, int KIND, int HDT>
__global__ void __launch_bounds__(kQtThreads, 1)
    k_q8_tile(const __grid_constant__ Q8View c, const __grid_constant__ Q8Batch b, const __grid_constant__ Q8Attend a,
              int tiles, int per_item) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int CH = HDT / 8;       // 16-byte chunks of an operand row
  constexpr uint32_t GROUP = CH * 128;  // bytes of 8 operand rows
  extern __shared__ __align__(1024) unsigned char qt_raw[];
  QtShared<HDT>& S = *reinterpret_cast<QtShared<HDT>*>(qt_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wg = warp >> 2;
  const int i = (int)((unsigned)blockIdx.x / (unsigned)tiles), kvh = blockIdx.y;
  const int len = __ldg(a.lens + i);
  const Seq s = seq_of(b, c.slots, i);
  const int G = a.heads / c.kvh, R = s.nrow * G, hd = c.hd;
  // sequences of few rows are k_q8_attend's
  if (s.slot == kSeqSkip || R <= kQ8FewRows) return;
  if (s.slot == kSeqBad || len < 0 || len > c.cap) {
    if (b.status && tid == 0) atomicOr(b.status, (int)kQ8BadRange);
    for (int x = (int)((unsigned)blockIdx.x % (unsigned)tiles); x < R; x += tiles)
      for (int d = tid; d < hd; d += kQtThreads)
        static_cast<T*>(const_cast<void*>(a.out.p))[(int64_t)(s.row0 + x / G) * a.out.token +
                                                    (int64_t)(kvh * G + x % G) * a.out.head + d] = E::from(NAN);
    return;
  }

  if (tid == 0) {
    for (int x = 0; x < 2; x++) {
      qb_init(&S.k_full[x], 128);
      qb_init(&S.v_full[x], 128);
      qb_init(&S.k_empty[x], 1);
      qb_init(&S.v_empty[x], 1);
      qb_init(&S.q_full[x], 128);
      qb_init(&S.s_full[x], 1);
      qb_init(&S.p_full[x], 128);
      qb_init(&S.o_full[x], 1);
    }
    for (int x = 0; x < kQtSlots; x++) qb_init(&S.sc_full[x], 128);
    qb_init(&S.drain, 1);
    S.limit.ns = a.wait_ns;
    S.limit.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  qt_before();
  __syncthreads();
  qt_after();
  const uint32_t tm = S.tmem;
  const uint32_t tm_s[2] = {tm, tm + 128}, tm_o[2] = {tm + 256, tm + 256 + HDT};
  QtLimit* const limit = &S.limit;

  const size_t sh = (size_t)s.slot * c.kvh + kvh;
  const int closed = len & ~(kQ8Block - 1);
  const T* kt = static_cast<const T*>(c.kt) + sh * kQ8Block * hd;
  const T* vt = static_cast<const T*>(c.vt) + sh * kQ8Block * hd;
  const unsigned char* hide = a.masked ? a.masked + (int64_t)i * a.mask_stride : nullptr;
  const int items = (R + per_item - 1) / per_item;
  const int first = tiles - 1 - (int)((unsigned)blockIdx.x % (unsigned)tiles);  // the longest causal items start first

  // Blocks of positions that the rows up to x (of the sequence) see.
  auto blocks_to = [&](int x) {
    const int most = a.causal ? min(len, len - (s.nrow - 1 - x / G)) : len;
    return most > 0 ? (most + kQtN - 1) / kQtN : 0;
  };

  if (wg < 2) {
    // ------------------------------------------------ softmax of one tile
    const int row = tid & 127;
    unsigned n_q = 0, n_s = 0, n_sc = 0;  // phases seen: items, score tiles, blocks of the CTA
    for (int item = first; item < items; item += tiles) {
      const int x0 = item * per_item, x_end = min(x0 + per_item, R);
      const int xt = x0 + wg * kQtM;  // the tile's first row
      const int nb0 = blocks_to(min(x0 + kQtM, x_end) - 1);
      const int nb1 = x0 + kQtM < x_end ? blocks_to(x_end - 1) : 0;
      const int nb = wg ? nb1 : nb0, nb_all = max(nb0, nb1);
      if (xt >= x_end) {
        n_sc += nb_all;
        continue;
      }
      const int x = xt + row;
      const bool on = x < x_end;
      const int token = s.row0 + (on ? x : x_end - 1) / G, head = kvh * G + (on ? x : x_end - 1) % G;
      const int seen = !on ? 0 : a.causal ? len - (s.nrow - 1 - x / G) : len;
      // The rows of q as operands, the warp's 32 rows a few at a time (16 bytes
      // of input a lane): times 2^up a row's largest element is in [2^14, 2^15).
      constexpr int RL = CH;             // lanes of a row
      constexpr int RI = 32 / RL;        // rows of a load
      // A tile that sees nothing has no products: no operands, and no arrival that
      // the issuing thread does not wait for (two in a row would pass it by).
      if (nb) {
#pragma unroll 4
        for (int r0 = 0; r0 < 32; r0 += RI) {
          const int rr = (warp & 3) * 32 + r0 + lane / RL, ch = lane % RL, y = xt + rr;
          const bool there = y < x_end && ch * 8 < hd;
          const T* q = static_cast<const T*>(a.q.p) + (int64_t)(s.row0 + (there ? y : 0) / G) * a.q.token +
                       (int64_t)(kvh * G + (there ? y : 0) % G) * a.q.head + (there ? ch * 8 : 0);
          __align__(16) T z[8];
          if (a.q_aligned) {
            *reinterpret_cast<uint4*>(z) = *reinterpret_cast<const uint4*>(q);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) z[e] = q[e];
          }
          float v[8], mx = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            v[e] = there ? E::to(z[e]) : 0.0f;
            mx = fmaxf(mx, fabsf(v[e]));
          }
#pragma unroll
          for (int d = RL / 2; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const int up = mx > 0.0f && mx <= FLT_MAX ? 14 - exponent_of(mx) : 0;
          const float up0 = exp2i(up / 2), up1 = exp2i(up - up / 2);
          // the sign of the scale goes into q: a block's largest score is then its largest product
          const float f = a.scale * 1.4426950408889634f * exp2i(-(up / 2)) * exp2i(up / 2 - up);
          const float u0 = f < 0.0f ? -up0 : up0;
          if (ch == 0) S.fac[wg * kQtM + rr] = fabsf(f);
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = h2_bits(__floats2half2_rn(v[2 * e] * u0 * up1, v[2 * e + 1] * u0 * up1));
          *reinterpret_cast<uint4*>(S.q[wg] + (rr >> 3) * GROUP + (rr & 7) * 16 + ch * 128) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        qt_proxy();
        if (a.stall != kQ8StallQ) qb_arrive(&S.q_full[wg]);
      }
      const float fs = S.fac[wg * kQtM + row];

      const uint32_t ts = tm_s[wg] + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t to = tm_o[wg] + ((uint32_t)((warp & 3) * 32) << 16);
      float m = -INFINITY, l = 0.0f, D = kQtLeast;  // references of the scores and of their products with values
      bool ok = true;
      for (int t = 0; t < nb; t++) {
        const unsigned blk = n_sc + t;
        const QtScales& sc = S.sc[blk % kQtSlots];
        // the scores first: only then is the slot's phase the last one that was completed
        ok = qb_wait(&S.s_full[wg], n_s & 1, limit) && qb_wait(&S.sc_full[blk % kQtSlots], (blk / kQtSlots) & 1, limit);
        n_s++;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        qt_after();
        // positions j * 32 .. + 31 of the block that the row sees
        auto shown = [&](int j) {
          const int n = seen - t * kQtN - j * 32;
          return sc.show[j] & (n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u);
        };
        const bool all = __all_sync(0xffffffffu, (shown(0) & shown(1) & shown(2) & shown(3)) == 0xffffffffu);
        // A row's scores from tensor memory, from position `at` of the block on; hidden ones are -inf.
        auto cover = [&](auto& v, int at) {
          if (all) return;
          const uint32_t w = shown(at >> 5) >> (at & 31);
#pragma unroll
          for (int e = 0; e < (int)(sizeof(v) / sizeof(v[0])); e++)
            if (!(w >> e & 1)) v[e] = 0xff800000u;
        };
        // Scale of a block's scores: never 0, which would turn -inf into NaN;
        // scores (below 2^38) times this least one are 0 to every bit that counts.
        auto scale_of = [&](int g) { return fmaxf(sc.ks[g] * fs, 1.0e-36f); };
        uint32_t z[2][16];  // one part is worked on while the next one comes
        // ---- the largest score mx, and the largest score with its value scale, mx + dx
        float mx = m, dx = D;
        tm_ld16(z[0], ts);
#pragma unroll 2
        for (int g = 0; g < kQtN / 16; g++) {
          uint32_t(&w)[16] = z[g & 1];
          tm_wait(w);
          tm_ld16(z[(g + 1) & 1], g + 1 < kQtN / 16 ? ts + (g + 1) * 16 : ts);  // the last one: for the second pass
          cover(w, g * 16);
          float y = __uint_as_float(w[0]);
#pragma unroll
          for (int e = 1; e < 15; e += 2) y = max3(y, __uint_as_float(w[e]), __uint_as_float(w[e + 1]));
          y = fmaxf(y, __uint_as_float(w[15]));
          y *= scale_of(g);
          const float old = mx;
          mx = fmaxf(mx, y);
          const float at = mx == -INFINITY ? 0.0f : mx;
          dx = fmaxf(dx + (old - at), sc.lam[g] + (y - at));
        }
        // ---- move the references when one has fallen far behind
        const bool move = mx > m + kQtLagM || dx + (mx - m) > D + kQtLagD;  // m of -inf: whenever mx is more
        const float dn = fmaxf(ceilf(dx), kQtLeast);
        if (__any_sync(0xffffffffu, move)) {
          const float al = move ? ex2((m - mx) + (D - dn)) : 1.0f;
          if (move) {
            l *= ex2(m - mx);
            m = mx;
            D = dn;
          }
          if (t) {
#pragma unroll 1
            for (int j = 0; j < HDT / 32; j++) {
              uint32_t w[32];
              tm_ld32(w, to + j * 32);
              tm_wait(w);
#pragma unroll
              for (int e = 0; e < 32; e++) w[e] = __float_as_uint(__uint_as_float(w[e]) * al);
              tm_st32(to + j * 32, w);
            }
            tm_wait_st();
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m, unit = exp2i(kQtUnit - (int)D);
        const bool far = __any_sync(0xffffffffu, fabsf(ref) > 1.0e6f);
        // ---- weights over the scores
        const uint64_t nref = f2(-ref, -ref);
        uint64_t l2 = f2(0.0f, 0.0f);
#pragma unroll 2
        for (int g = 0; g < kQtN / 16; g++) {
          uint32_t(&w)[16] = z[g & 1];
          tm_wait(w);
          if (g + 1 < kQtN / 16) tm_ld16(z[(g + 1) & 1], ts + (g + 1) * 16);
          cover(w, g * 16);
          const float cs = scale_of(g), vs = fminf(sc.vs[g] * unit, FLT_MAX);  // beyond that the weights are 0
          uint64_t cs2 = f2(cs, cs), vs2 = f2(vs, vs);
          if (far) {
            // products rounded as the reference was: what a fused step leaves of their
            // rounding is no longer small
#pragma unroll
            for (int e = 0; e < 16; e++) w[e] = __float_as_uint(__uint_as_float(w[e]) * cs);
            cs2 = f2(1.0f, 1.0f);
          }
          uint32_t p[16];  // the weights of 16 positions: 8 words of the first terms, 8 of the second ones
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float p0, p1;
            f2_get(f2_fma(f2(__uint_as_float(w[e]), __uint_as_float(w[e + 1])), cs2, nref), p0, p1);
            const uint64_t pp = f2(ex2(p0), ex2(p1));
            l2 = f2_add(l2, pp);
            f2_get(f2_mul(pp, vs2), p0, p1);
            const __half2 hi = __floats2half2_rn(p0, p1);
            p[e / 2] = h2_bits(hi);
            const float2 back = __half22float2(hi);
            p[8 + e / 2] = h2_bits(__floats2half2_rn(p0 - back.x, p1 - back.y));
          }
          tm_st16(ts + g * 16, p);  // in the place of their scores
        }
        {
          float l0, l1;
          f2_get(l2, l0, l1);
          l += l0 + l1;
        }
        tm_wait_st();
        qt_before();
        if (a.stall != kQ8StallWeights) qb_arrive(&S.p_full[wg]);
      }
      n_sc += nb_all;
      if (ok && nb) ok = __all_sync(0xffffffffu, qb_wait(&S.o_full[wg], n_q & 1, limit));
      if (nb) n_q++;
      T* out = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)token * a.out.token + (int64_t)head * a.out.head;
      const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l), back = exp2i((int)D - kQtUnit);
      qt_after();
#pragma unroll 1
      for (int j = 0; j < HDT / 32; j++) {
        uint32_t v[32];
        __syncwarp();
        if (ok && nb) {
          tm_ld32(v, to + j * 32);
          tm_wait(v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) v[e] = ok ? 0u : 0x7fc00000u;
        }
        if (ok && nb && S.open_odd) {
          // values of the open block that are no numbers: they count in the rows that see them
          for (int u = closed; u < min(len, seen); u++) {
            if (hide && hide[u]) continue;
#pragma unroll
            for (int e = 0; e < 32; e++) {
              const float y = j * 32 + e < hd ? E::to(vt[(u - closed) * hd + j * 32 + e]) : 0.0f;
              if (!(fabsf(y) <= FLT_MAX)) v[e] = __float_as_uint(__uint_as_float(v[e]) + y);
            }
          }
        }
        if (!on) continue;
        __align__(16) T y[32];
        const bool zero = ok && l == 0.0f;  // nothing seen
#pragma unroll
        for (int e = 0; e < 32; e++) y[e] = E::from(zero ? 0.0f : __uint_as_float(v[e]) * (ok ? inv : 1.0f) * back);
        if (a.out_aligned) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (j * 32 + e < hd) *reinterpret_cast<uint4*>(out + j * 32 + e) = *reinterpret_cast<const uint4*>(y + e);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (j * 32 + e < hd) out[j * 32 + e] = y[e];
        }
      }
      if (!ok) {
        if (b.status && lane == 0) atomicOr(b.status, (int)kQ8Timeout);
        // the rows of the items that were not reached
        for (int it = item + tiles; it < items; it += tiles) {
          const int y = it * per_item + wg * kQtM + row;
          if (y < min((it + 1) * per_item, R)) {
            T* o = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)(s.row0 + y / G) * a.out.token +
                   (int64_t)(kvh * G + y % G) * a.out.head;
            for (int d = 0; d < hd; d++) o[d] = E::from(NAN);
          }
        }
        break;
      }
      qt_before();  // this item's output is read before the next item's products
    }
  } else if (wg < 4) {
    // ------------- codes to fp16 operands (K and V by four warps each), scales and masks (K's)
    const bool is_v = wg == 3;
    const int ct = tid & 127, cw = ct >> 5, r8 = lane & 7, c4 = lane >> 3;
    constexpr int SETS = HDT / 64;  // sets of four 16-code chunks of a row
    const unsigned char* codes = (is_v ? c.vc : c.kc) + sh * c.cap * hd;
    const T* tail = is_v ? vt : kt;
    const float* ksc = c.ks + sh * (c.cap / kQ8Block);
    const float* vsc = c.vs + sh * (c.cap / kQ8Block);
    float open_k, open_v;
    {
      // The open block's power-of-two scales, from its finite elements that are
      // not hidden. Keys: the largest becomes [2^15, 2^16). Values: the largest
      // becomes [2^6, 2^7), as a code, so that the block's weights end where
      // other blocks' do; or as far up as [2^15, 2^16) when the last bits of the
      // smallest would else be below fp16's 2^-24.
      float ak = 0.0f, av = 0.0f, nv = FLT_MAX;
      bool odd = false;
      for (int x = ct; x < (len - closed) * hd; x += 128) {
        if (hide && hide[closed + x / hd]) continue;
        const float yk = fabsf(E::to(kt[x])), yv = fabsf(E::to(vt[x]));
        ak = fmaxf(ak, yk <= FLT_MAX ? yk : 0.0f);
        av = fmaxf(av, yv <= FLT_MAX ? yv : 0.0f);
        nv = fminf(nv, yv > 0.0f ? yv : FLT_MAX);
        odd |= !(yv <= FLT_MAX);
      }
      ak = warp_max_all(ak);
      av = warp_max_all(av);
      nv = -warp_max_all(-nv);
      odd = __any_sync(0xffffffffu, odd);
      if (lane == 0) {
        S.red[is_v][0][cw] = ak;
        S.red[is_v][1][cw] = av;
        S.red[is_v][2][cw] = nv;
        S.red_odd[is_v][cw] = odd;
      }
      asm volatile("bar.sync %0, 128;" ::"r"(1 + (int)is_v) : "memory");
      const float* rk = S.red[is_v][0];
      const float* rv = S.red[is_v][1];
      const float* rn = S.red[is_v][2];
      const float mk = fmaxf(fmaxf(rk[0], rk[1]), fmaxf(rk[2], rk[3]));
      const float mv = fmaxf(fmaxf(rv[0], rv[1]), fmaxf(rv[2], rv[3]));
      const int least = exponent_of(fminf(fminf(rn[0], rn[1]), fminf(rn[2], rn[3])));
      const int top = max(exponent_of(mv), -96), last = TYPE == kQ8F16 ? max(least - 10, -24) : least - 7;
      // exponents from -96: smaller blocks keep fewer than their own bits
      open_k = mk > 0.0f ? exp2i(max(exponent_of(mk), -96) - 15) : 1.0f;
      open_v = mv > 0.0f ? exp2i(top - min(max(top - last - 24, 6), 15)) : 1.0f;
      const int* ro = S.red_odd[is_v];
      if (ct == 0 && !is_v) S.open_odd = ro[0] | ro[1] | ro[2] | ro[3];
    }
    const float up = 1.0f / (is_v ? open_v : open_k);
    uint4 x[4 * SETS];
    auto load = [&](int t) {
#pragma unroll
      for (int g = 0; g < 4; g++)
#pragma unroll
        for (int z = 0; z < SETS; z++) {
          const int p = t * kQtN + (cw + 4 * g) * 8 + r8, ch = z * 4 + c4;
          x[g * SETS + z] = p < closed && ch * 16 < hd
                                ? __ldg(reinterpret_cast<const uint4*>(codes + (size_t)p * hd + ch * 16))
                                : make_uint4(0, 0, 0, 0);
        }
    };
    auto store = [&](unsigned char* dst, int t) {
#pragma unroll
      for (int g = 0; g < 4; g++)
#pragma unroll
        for (int z = 0; z < SETS; z++) {
          const int ch = z * 4 + c4;
          unsigned char* d = dst + (cw + 4 * g) * GROUP + ch * 256 + r8 * 16;
          uint32_t o[8];
          const uint4 w = x[g * SETS + z];
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t u = flip<KIND>(ww[e]);
            o[2 * e] = halves<KIND, false>(u);
            o[2 * e + 1] = halves<KIND, true>(u);
          }
          *reinterpret_cast<uint4*>(d) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(d + 128) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      if ((t + 1) * kQtN <= closed || t * kQtN >= len) return;
      // the open block's tokens, over the zeros that this warp has put in their
      // place: no warp waits for another, which may have given up
      __syncwarp();
#pragma unroll 1
      for (int u = lane; u < (len - closed) * (hd / 8); u += 32) {
        const int p = closed + u / (hd / 8) - t * kQtN, d8 = u % (hd / 8);
        if (p < 0 || p >= kQtN || ((p >> 3) & 3) != cw) continue;
        const T* y = tail + (u / (hd / 8)) * hd + d8 * 8;
        const bool hid = hide && hide[t * kQtN + p];
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float y0 = E::to(y[2 * e]), y1 = E::to(y[2 * e + 1]);
          if (is_v) {  // a weight of 0 times one of these would spread; they are added at the end
            y0 = fabsf(y0) <= FLT_MAX ? y0 : 0.0f;
            y1 = fabsf(y1) <= FLT_MAX ? y1 : 0.0f;
          }
          o[e] = hid ? 0u : h2_bits(__floats2half2_rn(y0 * up, y1 * up));
        }
        *reinterpret_cast<uint4*>(dst + (p >> 3) * GROUP + d8 * 128 + (p & 7) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    };
    unsigned n = 0;  // blocks of the CTA
    bool ok = true;
    for (int item = first; item < items && ok; item += tiles) {
      const int x0 = item * per_item, x_end = min(x0 + per_item, R);
      const int nb = max(blocks_to(min(x0 + kQtM, x_end) - 1), blocks_to(x_end - 1));
      if (nb) load(0);
      for (int t = 0; t < nb; t++, n++) {
        const unsigned st = n & 1, ph = (n >> 1) & 1;
        if (!is_v) {
          // scales and masks; the slot's last readers are behind: k_empty of
          // block n - 3 came after the products with block n - 4's weights
          QtScales& sc = S.sc[n % kQtSlots];
          const int p = t * kQtN + ct;
          const uint32_t show = __ballot_sync(0xffffffffu, p < len && !(hide && hide[p]));
          if (lane == 0) sc.show[cw] = show;
          if (ct < kQtN / kQ8Block) {
            const int p0 = t * kQtN + ct * kQ8Block;
            float ks = 0.0f, vs = 0.0f;
            if (p0 < closed) {
              ks = __ldg(ksc + p0 / kQ8Block);
              vs = __ldg(vsc + p0 / kQ8Block);
            } else if (p0 < len) {
              ks = open_k;
              vs = open_v;
            }
            sc.ks[ct] = ks;
            sc.vs[ct] = vs;
            sc.lam[ct] = scale_exponent(vs);
          }
          if (a.stall != kQ8StallScales) qb_arrive(&S.sc_full[n % kQtSlots]);
        }
        if (n >= 2) ok = qb_wait(is_v ? &S.v_empty[st] : &S.k_empty[st], ph ^ 1, limit);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        store(is_v ? S.v[st] : S.k[st], t);
        qt_proxy();
        // a drill withholds one warp's share: the others of the group go on
        if (a.stall != (is_v ? kQ8StallV : kQ8StallK) || cw) qb_arrive(is_v ? &S.v_full[st] : &S.k_full[st]);
        if (t + 1 < nb) load(t + 1);
      }
    }
  } else if (lane == 0) {
    // -------------------------------------------------------------- products
    const uint32_t qa[2] = {smem_u32(S.q[0]), smem_u32(S.q[1])};
    unsigned n = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
    bool ok = true;
    auto scores = [&](int w, unsigned blk) {
      const uint32_t ka = smem_u32(S.k[blk & 1]);
#pragma unroll
      for (int k = 0; k < HDT / 16; k++)
        qt_mma_ss(tm_s[w], qt_desc(qa[w] + k * 256, 128, GROUP), qt_desc(ka + k * 256, 128, GROUP), kQtIdesc<kQtN, false>,
                  k > 0);
      qt_commit(&S.s_full[w]);
    };
    auto values = [&](int w, unsigned blk, bool acc) {
      const uint32_t va = smem_u32(S.v[blk & 1]);
#pragma unroll
      for (int k = 0; k < kQtN / 16; k++)
#pragma unroll
        for (int z = 0; z < 2; z++)
          qt_mma_ts(tm_o[w], tm_s[w] + k * 16 + z * 8,
                    qt_desc(va + k * 2 * GROUP, GROUP, 128), kQtIdesc<HDT, true>, acc || k > 0 || z > 0);
    };
    for (int item = first; item < items && ok; item += tiles) {
      const int x0 = item * per_item, x_end = min(x0 + per_item, R);
      const int nb[2] = {blocks_to(min(x0 + kQtM, x_end) - 1), x0 + kQtM < x_end ? blocks_to(x_end - 1) : 0};
      const int all = max(nb[0], nb[1]);
      for (int w = 0; w < 2 && ok; w++)
        if (nb[w]) ok = qb_wait(&S.q_full[w], n_q[w]++ & 1, limit);
      if (!ok) break;
      qt_after();
      if (all) {
        ok = qb_wait(&S.k_full[n & 1], (n >> 1) & 1, limit);
        if (!ok) break;
        qt_after();
        for (int w = 0; w < 2; w++)
          if (nb[w]) scores(w, n);
        qt_commit(&S.k_empty[n & 1]);
      }
      for (int t = 0; t < all && ok; t++) {
        const unsigned blk = n + t;
        ok = qb_wait(&S.v_full[blk & 1], (blk >> 1) & 1, limit);
        if (ok && t + 1 < all) ok = qb_wait(&S.k_full[(blk + 1) & 1], ((blk + 1) >> 1) & 1, limit);
        for (int w = 0; w < 2 && ok; w++) {
          if (t >= nb[w]) continue;
          ok = qb_wait(&S.p_full[w], n_p[w]++ & 1, limit);
          if (!ok) break;
          qt_after();
          values(w, blk, t > 0);
          if (t + 1 < nb[w]) scores(w, blk + 1);
          else qt_commit(&S.o_full[w]);
        }
        if (!ok) break;
        qt_commit(&S.v_empty[blk & 1]);
        if (t + 1 < all) qt_commit(&S.k_empty[(blk + 1) & 1]);
      }
      n += all;
    }
    // every product issued has completed before tensor memory is freed
    qt_commit(&S.drain);
    const unsigned long long t0 = qt_time();
    while (!qb_try(&S.drain, 0))
      if (qt_time() - t0 > kQtDrainNs) {  // not the drill's limit: what was issued has to end
        limit->failed = 1;
        break;
      }
  }
  qt_before();
  __syncthreads();
  if (warp == 16) {
    qt_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512) : "memory");
  }
}

template <int TYPE, int KIND, int HDT>
void attend_tiles(const Q8View& c, const Q8Batch& b, const Q8Attend& a, int sms, cudaStream_t st) {
  auto kern = k_q8_tile<TYPE, KIND, HDT>;
  // all of tensor memory is taken, so one CTA an SM: with more than half of its shared memory too
  constexpr int smem = std::max((int)sizeof(QtShared<HDT>), 120 * 1024);
  static SmemLimit limit;
  limit.ensure([&] { SmemLimit::allow(kern, smem); });
  // One tile a CTA while there are SMs for all of them, else two.
  const int64_t rows = (int64_t)std::max(b.max_q, 1) * (a.heads / c.kvh);
  const int64_t single = (rows + kQtM - 1) / kQtM;
  const int per_item = single * b.n * c.kvh <= sms ? kQtM : 2 * kQtM;
  const int64_t tiles = std::min<int64_t>((rows + per_item - 1) / per_item, INT32_MAX / b.n);
  kern<<<dim3((unsigned)(b.n * tiles), (unsigned)c.kvh), kQtThreads, smem, st>>>(c, b, a, (int)tiles, per_item);
  DEFER_CUDA(cudaGetLastError());
}

}  // namespace

bool q8_tiles(const Q8View& c, const Q8Batch& b, const Q8Attend& a) {
  return c.type != kQ8F32 && c.hd <= 128 && (int64_t)b.max_q * (a.heads / c.kvh) > kQ8FewRows;
}

void q8_attend_tiles(const Q8View& c, const Q8Batch& b, const Q8Attend& a, cudaStream_t st) {
  int dev = 0, sms = 0;
  DEFER_CUDA(cudaGetDevice(&dev));
  DEFER_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  auto go = [&](auto f64, auto f128) { c.hd <= 64 ? f64(c, b, a, sms, st) : f128(c, b, a, sms, st); };
  if (c.type == kQ8Bf16) {
    if (c.kind == kQ8Int8) go(attend_tiles<kQ8Bf16, kQ8Int8, 64>, attend_tiles<kQ8Bf16, kQ8Int8, 128>);
    else go(attend_tiles<kQ8Bf16, kQ8E4m3, 64>, attend_tiles<kQ8Bf16, kQ8E4m3, 128>);
  } else {
    if (c.kind == kQ8Int8) go(attend_tiles<kQ8F16, kQ8Int8, 64>, attend_tiles<kQ8F16, kQ8Int8, 128>);
    else go(attend_tiles<kQ8F16, kQ8E4m3, 64>, attend_tiles<kQ8F16, kQ8E4m3, 128>);
  }
}

}  // namespace defer
