/*
 * defer_b200 — C ABI of the B200 backend for convo-lang/defer's token loop.
 *
 * Every entry point replaces one item of the reference crate's public Rust
 * API (paths below are relative to the reference project root) and keeps
 * its meaning and error behaviour. Plain pointers and sizes only; no
 * framework types. Handles belong to one CUDA device; calls on one handle
 * must be serialised by the caller; different devices may be driven from
 * different host threads.
 *
 * Status codes mirror DeferError (src/error.rs:5-14):
 *   0 ok, 1 Io, 2 Parse, 3 Model, 4 Checkpoint, 5 Wal, 6 Tokenizer,
 *   7 Divergence, plus 8 Cuda, 9 DeviceTimeout, 10 InvalidArgument.
 * On a non-zero status defer_last_error() returns the message (per thread).
 */
#ifndef DEFER_B200_H
#define DEFER_B200_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define DEFER_API __attribute__((visibility("default")))
#else
#define DEFER_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef struct defer_model defer_model;
typedef struct defer_cache defer_cache;
typedef struct defer_session defer_session;
typedef struct defer_wal_writer defer_wal_writer;

/* Model::Config (src/model.rs:24-39) plus device facts. */
typedef struct {
  uint32_t vocab_size, hidden_size, intermediate_size, num_layers;
  uint32_t num_heads, num_kv_heads, head_dim, max_seq_len;
  float rms_norm_eps, rope_theta;
  int32_t tie_word_embeddings, gelu, has_bias, weights_bf16;
  int64_t bos_token_id; /* -1 when absent */
  uint64_t weight_bytes; /* bytes one token step streams from HBM */
  int32_t device, sm_count;
} defer_config;

/* Message of the last failed call on this thread (src/error.rs:16-27). */
DEFER_API const char* defer_last_error(void);

/* ------------------------------------------------------------- model ---- */
/* Model::load (src/model.rs:286-299): parses the safetensors file, hashes
 * every byte (the signature), uploads the weights to `device`. */
DEFER_API int defer_model_load(const char* path, int device, defer_model** out);
DEFER_API void defer_model_free(defer_model* m);
DEFER_API int defer_model_config(const defer_model* m, defer_config* out);
/* Model::signature (src/model.rs:273-274). */
DEFER_API int defer_model_signature(const defer_model* m, uint8_t out[32]);
/* Config::eos_token_ids (src/model.rs:85-89). */
DEFER_API int defer_model_eos_tokens(const defer_model* m, uint32_t* out, size_t cap, size_t* n);
/* Model::forward / forward_ext (src/model.rs:376-520): one token at
 * position defer_cache_len(c); `masked` positions (< len) are hidden from the
 * query; logits (vocab_size floats) are copied to `logits_out` unless NULL.
 * Tracing (forward_traced) is not offered by this backend. */
DEFER_API int defer_forward(defer_model* m, defer_cache* c, uint32_t token, const size_t* masked, size_t n_masked,
                            float* logits_out);

/* Allocation-free forward step. No counterpart in the reference: it exists
 * for callers that cannot allocate device memory while they run — e.g. a
 * server whose memory pool already holds all free HBM, or a latency-bound
 * loop that must not enter the driver's allocator — and therefore cannot
 * use defer_forward, whose first call on a model allocates its scratch.
 * Same arithmetic and result as defer_forward on a cache of `cap`
 * positions, with the caller's buffers: k_cache and v_cache each hold
 * num_layers * num_kv_heads * cap * head_dim floats laid out
 * [layer][kv_head][position][dim], positions < pos filled by earlier calls;
 * position `pos` is written; logits_out receives vocab_size floats. All
 * three are device pointers. `stream` is a cudaStream_t (NULL = legacy
 * default stream); the call returns after the step has finished.
 * Limits: the step's scratch lives in one 4 MiB array inside this library
 * (held by every GPU that loads it until the process exits); a model/cap
 * whose scratch would exceed it is rejected with InvalidArgument. The first
 * call on a device is its set-up: it looks up that array's device address
 * and loads this step's device code (CUDA loads code lazily, and loading it
 * takes device memory), so make that first call before a memory pool
 * reserves the free HBM and before any stream capture; later calls
 * allocate nothing. The address is kept for the life of the process: after
 * a cudaDeviceReset of that device do not call this entry point again.
 * All calls share the array and each call reinitialises it, so calls must
 * not overlap on the GPU (different streams or threads racing each other
 * corrupt each other's scratch). */
DEFER_API int defer_forward_noalloc(defer_model* m, float* k_cache, float* v_cache, uint32_t cap, uint32_t pos,
                                    uint32_t token, float* logits_out, void* stream);

/* ------------------------------------------------------------- cache ---- */
/* Model::new_cache / KvCache (src/model.rs:184-243, 370-372). `cap` = 0
 * means max_position_embeddings positions. */
DEFER_API int defer_cache_new(defer_model* m, uint32_t cap, defer_cache** out);
DEFER_API void defer_cache_free(defer_cache* c);
DEFER_API size_t defer_cache_len(const defer_cache* c);
/* KvCache::truncate (src/model.rs:211-220). */
DEFER_API int defer_cache_truncate(defer_cache* c, size_t n);
/* KvCache::clone (derive, src/model.rs:184). */
DEFER_API int defer_cache_clone(const defer_cache* c, defer_cache** out);
/* KvCache::keys[layer] / values[layer] (src/model.rs:186-188) in the
 * reference layout [len, kv_dim]; each buffer holds len * kv_dim floats. */
DEFER_API int defer_cache_download(const defer_cache* c, uint32_t layer, float* keys, float* values);
/* KvCache::fingerprint (src/model.rs:233-242). */
DEFER_API int defer_cache_fingerprint(const defer_cache* c, uint8_t out[32]);
/* KvCache::bit_eq (src/model.rs:223-230). */
DEFER_API int defer_cache_bit_eq(const defer_cache* a, const defer_cache* b, int* equal);

/* --------------------------------------------------------- sampler/PRNG -- */
/* engine::seed_from_u64 (src/engine.rs:19-21). */
DEFER_API void defer_seed_from_u64(uint64_t seed, uint8_t out[32]);
/* ChaCha8Rng words [start, start + n) of the stream keyed by `seed`
 * (the words sampler.rs:92 draws, one per sampled token). */
DEFER_API int defer_chacha8_words(const uint8_t seed[32], uint64_t start, size_t n, uint32_t* out);
/* sampler::words_per_sample (src/sampler.rs:15-21). */
DEFER_API uint64_t defer_words_per_sample(float temperature);
/* sampler::sample_token (src/sampler.rs:78-109) run by the device sampler
 * on host logits, with the PRNG word already drawn (ignored when T == 0).
 * `margin` (nullable) receives the distance of r to the nearest CDF edge. */
DEFER_API int defer_sample_logits(int device, const float* logits, size_t n, float temperature, uint32_t word,
                                  uint32_t* token, float* margin);

/* ----------------------------------------------------------- session ---- */
/* Session::new (src/engine.rs:44-60). */
DEFER_API int defer_session_new(defer_model* m, const uint8_t seed[32], float temperature, defer_session** out);
DEFER_API void defer_session_free(defer_session* s);
/* Session::prompt (src/engine.rs:62-71). */
DEFER_API int defer_session_prompt(defer_session* s, const uint32_t* tokens, size_t n);
/* Session::step (src/engine.rs:113-117). */
DEFER_API int defer_session_step(defer_session* s, uint32_t* token);
/* Called after each generated token with the PRNG word position after it;
 * a non-zero return stops generation and is returned as the status. */
typedef int (*defer_token_cb)(void* user, uint32_t token, uint64_t rng_word_pos);
/* Session::generate (src/engine.rs:121-137). out_tokens holds max_tokens. */
DEFER_API int defer_session_generate(defer_session* s, size_t max_tokens, const uint32_t* stop, size_t n_stop,
                                     defer_token_cb cb, void* user, uint32_t* out_tokens, size_t* n_out);
/* Session::checkout (src/engine.rs:241-274) from checkpoint bytes. */
DEFER_API int defer_session_checkout(defer_model* m, const uint8_t* ckpt, size_t len, defer_session** out);
/* Session::checkpoint (src/engine.rs:223-232) as checkpoint bytes; with
 * buf == NULL only *len is set. */
DEFER_API int defer_session_checkpoint(const defer_session* s, uint8_t* buf, size_t cap, size_t* len);
/* Session::history / prompt_len / rng_word_pos / last_logits / cache
 * (src/engine.rs:194-221). The cache handle is borrowed. */
DEFER_API int defer_session_history(const defer_session* s, uint32_t* out, size_t cap, size_t* n);
DEFER_API size_t defer_session_prompt_len(const defer_session* s);
DEFER_API uint64_t defer_session_rng_word_pos(const defer_session* s);
DEFER_API int defer_session_last_logits(const defer_session* s, float* out);
DEFER_API defer_cache* defer_session_cache(defer_session* s);
/* Sampler margins of the last generate / checkout (diagnostics). */
DEFER_API int defer_session_margins(const defer_session* s, float* out, size_t cap, size_t* n);

/* ---------------------------------------------- checkpoint / WAL formats -- */
/* DeferCheckpoint (src/checkpoint.rs:26-108) as fields <-> bytes. */
typedef struct {
  uint8_t model_signature[32];
  uint8_t base_seed[32];
  float temperature;
  uint32_t prompt_len;
  uint64_t rng_word_pos_lo, rng_word_pos_hi;
  const uint32_t* history_tokens;
  size_t n_tokens;
} defer_checkpoint_fields;
DEFER_API int defer_checkpoint_encode(const defer_checkpoint_fields* f, uint8_t* buf, size_t cap, size_t* len);
/* Decodes and verifies (magic, version, CRC, lengths); the token pointer
 * refers into `tokens_out` (capacity `tokens_cap`). */
DEFER_API int defer_checkpoint_decode(const uint8_t* b, size_t len, defer_checkpoint_fields* f, uint32_t* tokens_out,
                                      size_t tokens_cap);
/* DeferCheckpoint::save / load (src/checkpoint.rs:92-108). */
DEFER_API int defer_checkpoint_save(const uint8_t* bytes, size_t len, const char* path);
DEFER_API int defer_checkpoint_load(const char* path, uint8_t* buf, size_t cap, size_t* len);

/* WalHeader (src/wal.rs:45-84). */
typedef struct {
  uint8_t model_signature[32];
  uint8_t base_seed[32];
  float temperature;
  uint32_t prompt_len;
  uint64_t start_rng_word_pos_lo, start_rng_word_pos_hi;
  const uint32_t* prefix_tokens;
  size_t n_prefix;
} defer_wal_header;
/* WalWriter::create / resume / append (src/wal.rs:221-250). */
DEFER_API int defer_wal_create(const char* path, const defer_wal_header* h, int durable, defer_wal_writer** out);
DEFER_API int defer_wal_resume(const char* path, int durable, defer_wal_writer** out);
DEFER_API int defer_wal_append(defer_wal_writer* w, uint32_t token, uint64_t rng_lo, uint64_t rng_hi);
DEFER_API void defer_wal_close(defer_wal_writer* w);
/* WalLog::parse + to_checkpoint (src/wal.rs:123-209): WAL bytes to
 * checkpoint bytes; reports the record count and a discarded torn tail. */
DEFER_API int defer_wal_to_checkpoint(const uint8_t* wal, size_t len, uint8_t* ckpt, size_t cap, size_t* ckpt_len,
                                      size_t* n_records, int* torn_tail, uint64_t* valid_len);

/* `defer verify` (src/main.rs:620-666): `runs` identical sessions (seed,
 * temperature, prompt, then Session::generate of max_tokens with the stop
 * tokens) must give run 0's tokens and KV fingerprint, and Session::checkout
 * of run 0's checkpoint must reproduce that fingerprint; otherwise
 * Divergence (7) with "run N diverged from run 0" or "checkout KV cache
 * differs from live cache". out_tokens (max_tokens entries) and
 * fingerprint receive run 0's results. */
DEFER_API int defer_verify(defer_model* m, const uint8_t seed[32], float temperature, const uint32_t* prompt,
                           size_t n_prompt, uint32_t runs, size_t max_tokens, const uint32_t* stop, size_t n_stop,
                           uint32_t* out_tokens, size_t* n_out, uint8_t fingerprint[32]);

/* ----------------------------------------------------- batched drivers --- */
/* Session::checkout for n checkpoints at once, `batch` sessions advancing
 * one position per step on the device. Per session: status (0 or the
 * DeferError code), first diverging step / the token replay sampled there
 * (-1 / 0 when none), optional KV fingerprint (n * 32 bytes). device_ms:
 * device time of the replay steps. */
DEFER_API int defer_replay_batch(defer_model* m, const uint8_t* const* ckpts, const size_t* lens, size_t n, int batch,
                                 int32_t* status, int32_t* div_step, uint32_t* div_token, uint8_t* fingerprints,
                                 double* device_ms);
/* Session::new + prompt + generate for n sessions at once. out_tokens[i]
 * holds max_tokens[i] entries; n_out[i] receives the count. */
DEFER_API int defer_generate_batch(defer_model* m, const uint32_t* const* prompts, const size_t* prompt_lens,
                                   const uint8_t* seeds, const float* temperatures, const size_t* max_tokens, size_t n,
                                   int batch, uint32_t* const* out_tokens, size_t* n_out, double* device_ms);
/* attribution::ablation_attribution (src/attribution.rs:224-264): base
 * log p(target | context) and the ablated log-probability of each position,
 * variants batched `batch` at a time. */
DEFER_API int defer_ablation(defer_model* m, const uint32_t* context, size_t n, uint32_t target,
                             const size_t* positions, size_t n_pos, int batch, double* base_logprob,
                             double* ablated_logprobs);
/* Instrumentation (no counterpart in the reference, which only prints tok/s
 * at src/main.rs:303-313): totals over every token-loop run of this model
 * since the last reset — device milliseconds between CUDA events recorded
 * on the model's stream around each launch, runs, kernel launches, tokens
 * fed, and algorithmic HBM bytes (weights once per step plus KV read and
 * written). Any pointer may be NULL; reset != 0 zeroes the totals after
 * reading them. */
DEFER_API int defer_model_timing(defer_model* m, double* device_ms, uint64_t* runs, uint64_t* launches,
                                 uint64_t* tokens, double* hbm_bytes, int reset);
/* Instrumentation (no counterpart in the reference): arms a per-stage time
 * trace of step `step` (< 0 disarms) of the next dataflow token-loop run on
 * this model. For every CTA and stage of that step the kernel records
 * globaltimer nanoseconds in 24 slots: 0 stage entry, 1 inputs received
 * (after the poll), 2 + w phase warp w finished its share; warp 0 also
 * marks sub-stages in slots 10-21 (RMS statistic ready, first weight piece
 * in shared memory; attention rows staged, scores, softmax, weighted sum,
 * units, combines; in select the sampler's records published, polled,
 * decoded and walked for the sum and for the CDF). Stages: 0 select, then
 * per layer l: 1 + 5l QKV, 2 + 5l attention, 3 + 5l O, 4 + 5l gate/up,
 * 5 + 5l down; then head and two unused slots. */
DEFER_API int defer_debug_trace_arm(defer_model* m, int32_t step);
/* The last trace: n = ctas * stages * 24 stamps (0 = not reached). */
DEFER_API int defer_debug_trace_read(const defer_model* m, uint64_t* out, size_t cap, size_t* n, int32_t* ctas,
                                     int32_t* stages);
/* Fault drill (no counterpart in the reference; the test of the device
 * failure detection): the next token-loop run on this model has CTA 0
 * withhold its first hand-off of step 0 (the dataflow kernel's step header,
 * the grid-barrier kernel's first arrival) and limits every bounded wait to
 * wait_us microseconds, so the run ends with DeviceTimeout (9) and no GPU
 * fault; later runs are unaffected. */
DEFER_API int defer_debug_stall(defer_model* m, uint32_t wait_us);
/* The tensor-core contraction of the batched attribution step on its own
 * (no counterpart in the reference; its check): y [m][n] = x [m][k] .
 * w [n][k]^T with fp32 host buffers, m <= 128, computed as split-bf16
 * products accumulated in fp32 by tcgen05 MMAs on `device`; with w_bf16
 * the weights are bf16-exact values stored as bf16. */
DEFER_API int defer_debug_tc_gemm(int device, const float* x, uint32_t m, const float* w, uint32_t n, uint32_t k,
                                  int32_t w_bf16, float* y);
/* attribution::log_softmax_at (src/attribution.rs:71-85). */
DEFER_API double defer_log_softmax_at(const float* logits, size_t n, size_t idx);

/* -------------------------------------------- key/value cache in 8 bits --- */
/* No counterpart in the reference, whose cache is fp32 (src/model.rs:184-243):
 * a cache of a quarter of the bytes, for callers whose sessions no longer fit
 * or whose steps are bound by reading the cache. These operators work on the
 * caller's own device buffers (as defer_forward_noalloc does), allocate
 * nothing, synchronise nothing and may be captured into a CUDA graph (after
 * one such call outside the capture: CUDA loads device code at a kernel's
 * first launch). Calls that write one cache must be ordered by the caller
 * (one stream, events). A bounded wait that runs out in defer_q8_attend fills
 * the rows with NaN and sets bit 2 of the status word.
 *
 * One layer of the cache, every pointer 16-byte aligned memory of `device`:
 *   codes  [slots][kv_heads][cap][head_dim]   int8 (kind 0) or e4m3 (kind 1)
 *   scales [slots][kv_heads][cap / 16]        float
 *   tail   [slots][kv_heads][16][head_dim]    `dtype`: 0 float, 1 bf16, 2 fp16
 * for K and for V. cap is a multiple of 16, head_dim a multiple of 16 up to
 * 256. Blocks of 16 positions share one scale per head: a block is quantised
 * when its 16th position is written, with s = max|x| / Q (Q = 127 or 448) and
 * code = round(x * (1 / s)) in fp32 (s = 0 when max|x| < 2^-117); until then
 * its positions are held as given in the tail. So codes do not depend on how
 * many positions came in one call. An 8-bit code holds no NaN and no infinity:
 * when a block closes, the maximum is taken over its finite values, a NaN is
 * stored as 0 and an infinity as +-Q. The block of position len / 16 is the
 * open one of a sequence of len positions: to shorten a sequence, shorten it
 * inside that block, or to a multiple of 16. */
typedef struct {
  int32_t device, kind, dtype;
  uint32_t slots, kv_heads, cap, head_dim;
  void *k_codes, *v_codes;
  float *k_scales, *v_scales;
  void *k_tail, *v_tail;
} defer_q8_cache;

/* The sequences of a call. Sequence i has rows q_start[i] .. q_start[i + 1]
 * - 1 of the `tokens` rows of k/v or q/out (q_start NULL: tokens / n rows
 * each; rows behind q_start[n] are left as they were) and lives in slot
 * slots[i] (NULL: slot i; negative: the sequence is skipped and its rows are
 * left as they were). max_q: the largest number of rows of a sequence (0:
 * tokens). It sizes the launch: sequences of more rows are still taken as a
 * whole, with the same result of defer_q8_append and, of defer_q8_attend, one
 * whose sums may be taken in another order.
 * q_start, slots and status are device memory. A sequence whose slot, rows,
 * position or length is out of range is skipped (defer_q8_attend fills its
 * rows with NaN where the rows themselves are valid), as is, when appending,
 * one whose slot an earlier sequence of the call names; if `status` is not
 * NULL the kernel then sets bit 0 (range) or bit 1 (slot named twice) in it. */
typedef struct {
  uint32_t n, tokens, max_q;
  const int32_t* q_start;
  const int32_t* slots;
  int32_t* status;
} defer_q8_batch;

/* Writes rows k and v [tokens][kv_heads][head_dim] of the cache's dtype
 * (strides of rows and heads in elements) at positions pos[i], pos[i] + 1, ...
 * of each sequence; pos [n] is device memory. The cache holds pos[i]
 * positions already, those of the open block in the tail. With slots, at most
 * 2^16 sequences (the kernel compares them with one another). */
DEFER_API int defer_q8_append(const defer_q8_cache* c, const defer_q8_batch* b, const int32_t* pos, const void* k,
                              int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                              int64_t v_head_stride, void* stream);
/* Reads positions start[i] .. len - 1 (at most `rows`; start NULL: from 0)
 * of sequence i of lens[i] positions back: value = code * scale rounded once
 * to the cache's dtype, or the open block's value as given, to k_out and
 * v_out [n][kv_heads][rows][head_dim] with the element strides
 * {sequence, head, row}; rows behind the last position are left as they were.
 * slots and status as in defer_q8_batch. */
DEFER_API int defer_q8_read(const defer_q8_cache* c, uint32_t n, const int32_t* lens, const int32_t* start,
                            const int32_t* slots, int32_t* status, uint32_t rows, void* k_out,
                            const int64_t k_strides[3], void* v_out, const int64_t v_strides[3], void* stream);
/* Attention of q [tokens][heads][head_dim] over the cache into out, both of
 * the cache's dtype: head h reads key head h / (heads / kv_heads). lens[i] is
 * the length of sequence i with the call's own rows appended: with `causal`
 * row j of a sequence of r rows sees positions 0 .. lens[i] - r + j, else all
 * lens[i]. masked (NULL, or device bytes [n] with row stride mask_stride, 0 or
 * at least cap): position t of sequence i is hidden where masked[i *
 * mask_stride + t] is not 0. out = sum_t p_t V_t, p = softmax(scale * q . K_t)
 * over the positions seen, 0 when there are none; softmax and sums in fp32, the
 * weights rounded to 22 bits for the products with the values. Scores are sums
 * of products with q (of fp32 rows: 22 bits of each element). For more than 64
 * rows a key head of a 16-bit cache with head_dim up to 128, values that are
 * 2^20 times smaller than another visible block's count with 15 bits, 2^30
 * times smaller with 5. max_len: the longest length (0: cap). It sizes the
 * launch: a sequence that is longer is still attended as a whole, its sums taken
 * in another order. With max_q and max_len as they are or larger (or 0), a
 * sequence's result depends on its own rows, length and cache only, not on the
 * call's other sequences. */
DEFER_API int defer_q8_attend(const defer_q8_cache* c, const defer_q8_batch* b, const int32_t* lens,
                              uint32_t max_len, uint32_t heads, const void* q, int64_t q_token_stride,
                              int64_t q_head_stride, void* out, int64_t out_token_stride, int64_t out_head_stride,
                              const uint8_t* masked, int64_t mask_stride, int32_t causal, float scale,
                              void* workspace, size_t workspace_bytes, void* stream);
/* Bytes of 16-byte aligned device memory that such a call uses while it runs
 * (0 unless max_len is long); its contents need no preparation and mean
 * nothing afterwards. Calls that may run at the same time, captured graphs
 * among them, need one each. */
DEFER_API int defer_q8_attend_workspace(const defer_q8_cache* c, const defer_q8_batch* b, uint32_t max_len,
                                        uint32_t heads, size_t* bytes);

/* Fault drill (as defer_debug_stall): in the calling thread's next
 * defer_q8_attend of many 16-bit rows one role of the kernel withholds its
 * arrivals (1: q, 2: K, 3: V, 4: scales, 5: weights) and every bounded wait is
 * limited to wait_us microseconds. The rows become NaN, bit 2 of the status word
 * is set, nothing faults, and later calls are unaffected. */
DEFER_API int defer_debug_q8_stall(int32_t role, uint32_t wait_us);

/* A model's caches in 8 bits: `slots` sessions of up to `cap` positions (0:
 * max_position_embeddings; rounded up to 16), every layer, the open blocks in
 * fp32. For models whose head_dim is a multiple of 16 up to 256. */
typedef struct defer_qcache defer_qcache;
DEFER_API int defer_qcache_new(defer_model* m, uint32_t slots, uint32_t cap, int32_t kind, defer_qcache** out);
DEFER_API void defer_qcache_free(defer_qcache* c);
/* Positions of a slot (0 for a slot that does not exist). */
DEFER_API size_t defer_qcache_len(const defer_qcache* c, uint32_t slot);
/* Shortens a slot (as KvCache::truncate, src/model.rs:211-220). A block that
 * was closed and is shortened is opened again with its codes' values. */
DEFER_API int defer_qcache_truncate(defer_qcache* c, uint32_t slot, size_t n);
/* A cache of the same model into a slot, whose contents it replaces, and a
 * slot as a new cache holding the codes' values. */
DEFER_API int defer_qcache_store(defer_qcache* c, uint32_t slot, const defer_cache* src);
DEFER_API int defer_qcache_load(const defer_qcache* c, uint32_t slot, defer_cache** out);
/* Keys and values of a slot's layer as defer_cache_download gives them. */
DEFER_API int defer_qcache_download(const defer_qcache* c, uint32_t slot, uint32_t layer, float* keys, float* values);
/* One layer's buffers, for defer_q8_append, _read and _attend. A call that
 * writes them does not change the slots' lengths that the handle counts. */
DEFER_API int defer_qcache_view(const defer_qcache* c, uint32_t layer, defer_q8_cache* out);
/* Model::forward (src/model.rs:376-520) of tokens[i] in slot slots[i], i < n,
 * all in one step (of a model whose token loops run on the tensor cores: in
 * steps of 128 slots): each slot's K and V rows are appended to the 8-bit cache
 * and attention reads it; logits_out (NULL, or n * vocab_size floats) receives
 * the logits. No slot may be named twice. The projections are those of the
 * batched token loops; a slot's result does not depend on the other slots. */
DEFER_API int defer_forward_q8(defer_model* m, defer_qcache* c, const uint32_t* slots, const uint32_t* tokens,
                               size_t n, float* logits_out);

#ifdef __cplusplus
}
#endif
#endif
