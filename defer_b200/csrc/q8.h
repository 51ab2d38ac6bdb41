// Key/value cache in 8 bits: host entry points of the kernels in q8.cu.
//
// One layer of a cache is held in the caller's device memory as
//   codes  [slots][kv_heads][cap][head_dim]  int8 or e4m3, for K and for V
//   scales [slots][kv_heads][cap / 16]       fp32, one per block and head
//   tail   [slots][kv_heads][16][head_dim]   the open block's tokens as given
// A block of 16 tokens is quantised when its last token arrives, so its
// codes depend on its tokens alone (not on how many came in one call) and no
// value is rounded twice.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace defer {

constexpr int kQ8Block = 16;        // tokens that share a scale
constexpr int kQ8MaxHeadDim = 256;  // head_dim is a multiple of 16 up to this

enum Q8Kind : int { kQ8Int8 = 0, kQ8E4m3 = 1 };
enum Q8Type : int { kQ8F32 = 0, kQ8Bf16 = 1, kQ8F16 = 2 };

// Bits of the optional status word (a sequence that sets one is skipped).
enum Q8Status : int {
  kQ8BadRange = 1,   // slot, length, position or row range outside its bounds
  kQ8SlotTwice = 2,  // append: the slot appears in an earlier sequence of the call
  kQ8Timeout = 4,    // attend: a bounded wait ran out; the rows are NaN
};

// One layer's buffers (every pointer 16-byte aligned device memory).
struct Q8View {
  unsigned char *kc, *vc;
  float *ks, *vs;
  void *kt, *vt;
  int slots, kvh, cap, hd;
  int kind, type;
};

// The rows of a call: sequence i has rows [q_start[i], q_start[i + 1]) of
// the k/v or q/out arrays (q_start null: tokens / n rows each) and is held
// in slot slots[i] (null: slot i; negative: skipped, its rows left alone).
struct Q8Batch {
  int n, tokens;
  int max_q;  // rows of the longest sequence (sizes the grid only)
  const int* q_start;
  const int* slots;
  int* status;  // or null
};

// Strides in elements; the head_dim elements of a row are contiguous.
struct Q8Rows {
  const void* p;
  int64_t token, head;
};

void q8_append(const Q8View& c, const Q8Batch& b, const int* pos, const Q8Rows& k, const Q8Rows& v, cudaStream_t st);

// Positions [start, min(len, start + rows)) of each sequence to output rows
// 0, 1, ...; rows behind them stay as they are.
struct Q8Out {
  void* p;
  int64_t seq, token, head;
};
void q8_read(const Q8View& c, int n, const int* lens, const int* start, const int* slots, int* status, int rows,
             const Q8Out& k, const Q8Out& v, cudaStream_t st);

struct Q8Attend {
  const int* lens;
  int max_len;  // longest sequence (sizes the grid only)
  int heads;
  Q8Rows q;
  Q8Rows out;  // p is written
  const unsigned char* masked;  // [n][mask_stride] nonzero hides a position, or null
  int64_t mask_stride;
  int causal;
  float scale;
  float* ws;  // q8_attend_workspace bytes (may be null when that is 0)
  // set by q8_attend
  int q_aligned, out_aligned;  // the rows start on 16 bytes
  int tiled;                   // sequences of more than kQ8FewRows rows are q8_attend_tiles'
  int group;                   // heads of a key head
  unsigned group_inv;          // 2^32 / group, rounded up
  unsigned long long wait_ns;  // limit of the tile kernel's waits
  int stall;                   // Q8Stall: an arrival of the tile kernel that is withheld (a drill), or 0
};
// Rows of a sequence and key head up to which the streaming kernel takes them
// all: 4 passes over the cache with 16 rows each.
constexpr int kQ8FewRows = 64;
// Whether a call may hold sequences for the tile kernel (q8_tile.cu), and that
// kernel's launch for them.
bool q8_tiles(const Q8View& c, const Q8Batch& b, const Q8Attend& a);
void q8_attend_tiles(const Q8View& c, const Q8Batch& b, const Q8Attend& a, cudaStream_t st);
// A role of the tile kernel whose arrivals the drill withholds: the operands of
// q, K or V, the scales, the weights.
enum Q8Stall : int { kQ8StallQ = 1, kQ8StallK, kQ8StallV, kQ8StallScales, kQ8StallWeights };
// The calling thread's next q8_attend that launches the tile kernel runs
// with `role` stalled and every wait limited to wait_us.
void q8_stall_next(int role, unsigned wait_us);
size_t q8_attend_workspace(const Q8View& c, const Q8Batch& b, const Q8Attend& a);
void q8_attend(const Q8View& c, const Q8Batch& b, const Q8Attend& a, cudaStream_t st);

}  // namespace defer
