/* rtgpu: MI355X (gfx950) GPT-2 token loop behind a C ABI.
 *
 * Each entry point mirrors one item of rusttorch's public GPT-2 API
 * (rusttorch-core/src/nn/gpt2.rs, re-exported at nn/mod.rs:50,94) and follows
 * the conventions of rusttorch's own C ABI (rusttorch-core/src/ffi/):
 * fallible calls return rtg_result {success, error_msg} like CResult
 * (ffi/tensor.rs:37-64); the message is owned by the library and released
 * with rtg_free_error_message (ffi/tensor.rs:66-72); host buffers are
 * caller-allocated and results are written into them (ffi/ops.rs:26-39).
 * Error strings are the reference's own (gpt2.rs:224-228, 269-279, 364-374,
 * 616-618).
 *
 * Threading: a model is immutable after construction and may be shared by
 * threads (gpt2.rs:358 takes &self); a cache binds one HIP stream and must not
 * be used from two threads at once (gpt2.rs:361 takes &mut KVCache). All calls
 * are synchronous from the host's point of view, as in the reference.
 *
 * There is no CPU fallback: creating a model without a usable gfx950 device
 * fails with an error. */
#ifndef RTGPU_H
#define RTGPU_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* CResult, ffi/tensor.rs:37-64. */
typedef struct {
  bool success;
  char* error_msg; /* NULL on success; free with rtg_free_error_message */
} rtg_result;

/* Gpt2Config, gpt2.rs:82-104. The fields are public in the reference, which
 * takes head_dim = n_embd / n_head (gpt2.rs:349-352). This build accepts the
 * configurations its kernels are written for and refuses the others when the
 * model is created, before anything is uploaded, with these errors:
 *   "n_embd <d> is not divisible by n_head <h>"   (the reference would
 *       truncate head_dim and read past its rows)
 *   "head_dim <hd> > 64 is not supported"         (head_dim <= 64 only)
 *   "n_embd <d> must be a multiple of 8"          (16-byte row vectors)
 * Every GPT-2 checkpoint (head_dim 64, n_embd 768 / 1024 / 1280 / 1600) and
 * the reference's own test configuration (n_embd 8, 2 heads) are accepted.
 * The fastest batch-1 decode step (one persistent kernel per token) is built
 * for n_embd 128 with vocab_size <= 512, and for vocab_size <= 50257 at
 * n_embd 768 and 1024 (f32 and bf16 storage), 1280 (f32) and 1600 (bf16);
 * other accepted shapes decode through the batched step's kernel graph at
 * batch 1 (same results within the logits tolerance, about 4.5 us per kernel
 * launch, 5 launches per layer: GPT-2 XL in f32 takes 2.19 ms per token that
 * way, against 1.67 ms for XL bf16 on the persistent step). */
typedef struct {
  size_t vocab_size;
  size_t n_positions;
  size_t n_embd;
  size_t n_layer;
  size_t n_head;
  float layer_norm_epsilon;
} rtg_config;

/* GenerationConfig, gpt2.rs:31-79, plus the seed of the sampler (the
 * reference draws from rand::thread_rng, gpt2.rs:978,1005, so its sampled ids
 * are not reproducible; greedy decoding ignores the seed). */
typedef struct {
  size_t max_new_tokens;
  float temperature;
  size_t top_k;
  float top_p;
  float repetition_penalty;
  uint64_t seed;
} rtg_gen_config;

/* Element type of a host tensor handed to rtg_model_from_host; decoded to
 * f32 as safetensors.rs:232-348 does (BF16 = bits << 16, :389-391). */
typedef enum { RTG_F32 = 0, RTG_BF16 = 1, RTG_F16 = 2, RTG_F64 = 3 } rtg_dtype;

/* How the weights are held in HBM. RTG_STORE_BF16 keeps GEMM/GEMV weights as
 * bfloat16 (round-to-nearest-even) and upcasts them in-kernel; the oracle is
 * fed the same rounded values. */
typedef enum { RTG_STORE_F32 = 0, RTG_STORE_BF16 = 1 } rtg_storage;

/* One StateDict entry (nn/state_dict.rs:35-56): name, dtype, shape, data. */
typedef struct {
  const char* name;
  const void* data;
  rtg_dtype dtype;
  size_t ndim;
  const size_t* shape;
} rtg_named_tensor;

typedef struct rtg_model rtg_model;
typedef struct rtg_cache rtg_cache;

/* Device-event timings of a generate call (HIP events on the cache's stream).
 * profile_kernels is an input: when nonzero and the decode step is the single
 * persistent kernel, the decode steps are replayed once more launch by launch
 * (identical inputs and results) with events around that kernel, filling
 * decode_kernel_ms / decode_kernel_launches. */
typedef struct {
  int profile_kernels;
  double prefill_ms;     /* forward_cached over the prompt + first argmax */
  double decode_ms;      /* the (max_new - 1) single-token steps */
  size_t decode_steps;
  double decode_kernel_ms;       /* summed duration of the decode-step kernel */
  size_t decode_kernel_launches;
} rtg_timing;

/* rusttorch_init / rusttorch_cleanup / rusttorch_version, ffi/mod.rs:24-48. */
void rtg_init(void);
void rtg_cleanup(void);
const char* rtg_version(void);
/* rusttorch_free_error_message, ffi/tensor.rs:66-72. */
void rtg_free_error_message(char* msg);

/* Gpt2Model::from_safetensors, gpt2.rs:214-220 (F32/F64/F16/BF16 tensors).
 * Error: "Failed to load safetensors: ..." or "Missing weight: <name>". */
rtg_result rtg_model_from_safetensors(const char* path, const rtg_config* cfg, rtg_storage storage,
                                      rtg_model** out);
/* Gpt2Model::from_state_dict, gpt2.rs:223-263. Tensors use the reference's
 * Conv1D layout [in, out]; the data is copied (uploaded) before returning. */
rtg_result rtg_model_from_host(const rtg_config* cfg, const rtg_named_tensor* tensors, size_t n,
                               rtg_storage storage, rtg_model** out);
void rtg_model_destroy(rtg_model* model);
/* Gpt2Model::num_parameters, gpt2.rs:541-563. */
size_t rtg_num_parameters(const rtg_model* model);

/* Gpt2Model::new_cache / KVCache::new, gpt2.rs:349-352, 125-134. The cache
 * holds `batch` sequences and preallocates n_layer*batch*2*n_head*n_positions*
 * head_dim f32 in HBM. batch = 1 is the reference's cache. */
rtg_result rtg_cache_new(const rtg_model* model, size_t batch, rtg_cache** out);
/* The same cache in 8 bits, a scale for every `block` (16, 32 or 64) tokens of a
 * head, keys and values apart (the rules stand with rtg_qcache below; no
 * counterpart in the reference). A quarter of the memory (and of what a decode
 * step reads of it), for logits that differ by what the rounding of keys and
 * values to 8 bits moves. Goes wherever a cache of this batch goes except
 * rtg_forward_cached_noalloc; one new token runs the batched step's kernel graph
 * at any batch, more run the prefill kernels. Behind a pass that failed the cache
 * goes on where it was, as an f32 one does; its last block's tokens may then count
 * as the values that they read back as. */
rtg_result rtg_cache_new_quantised(const rtg_model* model, size_t batch, size_t block, rtg_cache** out);
/* KVCache::len / is_empty / clear, gpt2.rs:137-161. */
size_t rtg_cache_len(const rtg_cache* cache);
bool rtg_cache_is_empty(const rtg_cache* cache);
void rtg_cache_clear(rtg_cache* cache);
void rtg_cache_destroy(rtg_cache* cache);
/* Copies cached keys (values != 0: values) of one layer/head/sequence for
 * positions [0, len) to out[len * head_dim]; a test hook with no reference
 * counterpart (the reference's LayerKVCache fields are private). */
rtg_result rtg_cache_read(const rtg_cache* cache, size_t layer, size_t head, size_t seq, int values, float* out);

/* Gpt2Model::forward, gpt2.rs:269-304: logits_out[n * vocab_size]. Here and
 * below, a call that returns an error leaves logits_out as it was, or with part
 * or all of what it had computed when the error was found. */
rtg_result rtg_forward(const rtg_model* model, const uint32_t* ids, size_t n, float* logits_out);
/* Gpt2Model::forward_cached, gpt2.rs:358-399: logits_out[n * vocab_size]
 * (may be NULL: nothing is copied, and a prompt of more than one token runs
 * without its LM head). The cache must have batch 1
 * and belong to model. One new token (n == 1) runs the persistent decode
 * step that generate_cached runs per token, where the model's shape has one;
 * 2..32 tokens run the multi-row forward in one launch (f32 weights, n_embd
 * 128, 768 or 1024); more tokens run the prefill kernels. */
rtg_result rtg_forward_cached(const rtg_model* model, rtg_cache* cache, const uint32_t* ids, size_t n,
                              float* logits_out);
/* forward_cached without device allocation. No counterpart in the reference:
 * it is for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc). Same
 * arguments as rtg_forward_cached and the kernels of its path for n >= 2
 * (the same results bit for bit; for n == 1 rtg_forward_cached runs the
 * persistent decode step instead, and the two agree within the logits
 * tolerance), but the pass's work rows and logits live in a fixed scratch
 * array of 16 MiB + 64 KiB per device inside the library instead of the
 * cache's buffers, and nothing is allocated. Up to 32 tokens run the
 * multi-row forward (its flags and epoch in the 64 KiB, kept between calls);
 * more run the prefill kernels, with the limit: n * (10 * n_embd +
 * vocab_size) floats (each of the six parts rounded up to 64) must fit in
 * 16 MiB, e.g. n <= 72 for GPT-2 small, n <= 63 for XL; a larger n returns
 * an error. The prefill GEMMs' split-k partials take what is left of the
 * array; where they do not fit the GEMMs run unsplit. All calls on one
 * device share the array and take turns on it (a per-device lock held until
 * the call's stream has drained). The cache must belong to model. */
rtg_result rtg_forward_cached_noalloc(const rtg_model* model, rtg_cache* cache, const uint32_t* ids, size_t n,
                                      float* logits_out);
/* Gpt2Model::generate (uncached, sliding window), gpt2.rs:311-346.
 * out receives n + max_new ids. */
rtg_result rtg_generate(const rtg_model* model, const uint32_t* prompt, size_t n, size_t max_new,
                        float temperature, uint64_t seed, uint32_t* out);
/* Gpt2Model::generate_cached, gpt2.rs:405-441. out receives n + max(1, max_new)
 * ids: like the reference, the prefill token is appended even if max_new == 0. */
rtg_result rtg_generate_cached(const rtg_model* model, const uint32_t* prompt, size_t n, size_t max_new,
                               float temperature, uint64_t seed, uint32_t* out);
/* Gpt2Model::generate_with_config, gpt2.rs:447-474 (+ sample_logits :871-906).
 * out receives n + max(1, cfg->max_new_tokens) ids. Non-greedy token choice
 * runs on the device for vocab_size <= 65536 (every GPT-2 vocabulary);
 * beyond it the call returns "vocabulary too large for the device sampler". */
rtg_result rtg_generate_with_config(const rtg_model* model, const uint32_t* prompt, size_t n,
                                    const rtg_gen_config* cfg, uint32_t* out);

/* Batched extension (new API: the reference is batch-1 only; its oracle for
 * batch B is B independent calls). ids/prompts are [batch][n] row-major. */
rtg_result rtg_forward_cached_batched(const rtg_model* model, rtg_cache* cache, const uint32_t* ids, size_t n,
                                      float* logits_out /* [batch][n][V] or NULL */);
/* Greedy generate_cached over `batch` equal-length prompts; out is
 * [batch][n + max(1, max_new)]. timing may be NULL. */
rtg_result rtg_generate_cached_batched(const rtg_model* model, const uint32_t* prompts, size_t batch, size_t n,
                                       size_t max_new, uint32_t* out, rtg_timing* timing);

/* The same over a cache of 8 bits (rtg_cache_new_quantised). */
rtg_result rtg_generate_cached_quantised(const rtg_model* model, const uint32_t* prompts, size_t batch, size_t n,
                                         size_t max_new, size_t block, uint32_t* out, rtg_timing* timing);

/* ---- 8-bit key/value cache over device tensors (no counterpart in the
 * reference, whose cache is f32 vectors on the host, gpt2.rs:111-175). For
 * programs that run their own layers: writing keys and values, reading them
 * back, and attention over them, for any number of sequences and of query
 * heads per key/value head. rtg_cache_new_quantised (above) is the same cache
 * under a GPT-2 model.
 *
 * For each (sequence, head), keys and values apart, every `block` consecutive
 * tokens (16, 32 or 64) share one scale:
 *   s = f32(max |x| over the block's tokens so far / 127)   (0 where a token's
 *       maximum is below 127 * 2^-126; NaN where a value is not finite)
 *   code = the integer nearest to x / s, ties to even; it reads back as code * s
 *       in f32 (the largest f32 of all as infinity).
 * The last token's block is quantised from its tokens' unrounded values, which
 * are kept in f32 until the next block begins: what the cache holds does not
 * depend on how the tokens were split over appends. 2 bytes per token, head and
 * column (columns padded to 64 or 128), 8 per block and head, and
 * 2 * block * columns f32 per sequence and head for the last block.
 *
 * Rows are [n_seq][tokens][heads][head_dim] in device memory of the device that
 * was current when the cache was made, in any strides (elements; a row's
 * head_dim columns contiguous); counts, start and first are device arrays of
 * n_seq int32, or NULL. Calls enqueue on `stream` (a hipStream_t of that device,
 * NULL for the default stream) and return without waiting; they allocate
 * nothing and may be captured into a graph, each replay acting on the cache as
 * it then is. Lengths live on the device. A cache must not be used by two
 * calls (or replays) at once, the reading ones included: they share a
 * workspace. Calls on different streams need the streams' own ordering, and a
 * cache has to live as long as the graphs that hold its calls. Making one and
 * destroying one (which waits for the device) leave captures under way alone. ---- */
typedef struct rtg_qcache rtg_qcache;
typedef struct {
  void* data;
  ptrdiff_t stride_seq, stride_token, stride_head;
} rtg_rows;
/* Errors: "head_dim <hd> is not supported (1 to 128)", "block <b> is not
 * supported (16, 32 or 64)", capacities over 4000000 tokens, more than 1000000
 * pairs of sequence and head. */
rtg_result rtg_qcache_new(size_t n_seq, size_t n_head, size_t head_dim, size_t capacity, size_t block,
                          rtg_qcache** out);
void rtg_qcache_destroy(rtg_qcache* cache);
/* n_new tokens to every sequence, or the first counts[s] (clamped to 0 ..
 * n_new) of its rows; behind its length, or with start from token start[s] on:
 * what lay there and behind is dropped (start of 0: the sequence begins anew;
 * n_new = 0: only dropped). Where the last token left lies in another block than
 * the last one did, its block's tokens count as the values they read back as
 * from then on (their unrounded ones are gone). A sequence whose start is
 * negative or behind its length, or whose tokens would pass the capacity, is
 * left as it was, and rtg_qcache_lengths reports it. */
rtg_result rtg_qcache_append(rtg_qcache* cache, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n_new,
                             const int32_t* counts, const int32_t* start, void* stream);
/* The values of tokens first[s] (0 for NULL) .. first[s] + n - 1 of every
 * sequence, rounded to dtype; rows that hold no token are set to 0. k or v may be NULL. */
rtg_result rtg_qcache_read(const rtg_qcache* cache, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n,
                           const int32_t* first, void* stream);
/* Causal attention of the last counts[s] (n_q for NULL, clamped to 0 .. n_q)
 * tokens of every sequence: query i of c sits at position len - c + i and sees
 * the keys up to its own; softmax of scale * q . k, in f32 or better, results
 * rounded to dtype once. Query head h reads key/value head h / (n_q_head /
 * n_head), at most 1024 of them one key/value head. A block that reads back as
 * NaN makes the rows NaN that see a key of it, and no others; a query with a
 * value that is not finite gives a row of NaN. Sums are f32 and divided last:
 * the largest |v| times the number of keys has to be below 3.4e38, and |v| below
 * 1e-31 lose digits. Rows i >= counts[s], and rows of queries before the
 * sequence's first token, are set to 0. out must not overlap the queries. */
rtg_result rtg_qcache_attend(rtg_qcache* cache, rtg_dtype dtype, const rtg_rows* queries, size_t n_q,
                             size_t n_q_head, const int32_t* counts, float scale, const rtg_rows* out, void* stream);
/* Waits for the stream and writes the n_seq lengths. Returns an error once
 * (the lengths are written all the same) where an append since the last call
 * left a sequence as it was. Not for a stream that is being captured. */
rtg_result rtg_qcache_lengths(rtg_qcache* cache, uint32_t* out, void* stream);

/* ---- 4-bit key/value cache over device tensors, and its eviction (no
 * counterpart in the reference). An eighth and a quarter of the memory of f32 and
 * bf16 rows and half of the 8-bit cache's, for contexts that are long or many; up to
 * half as much again, 17 MB at most, for attention's partial results.
 *
 * For each (sequence, head) and token, keys and values apart, 32 consecutive
 * channels are numbers of 4 bits (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times a
 * power of two:
 *   p = the largest power of two not above the channels' max |x|, twice that
 *       where the maximum is over 1.75 p; scale = p / 4, within 2^-100 .. 2^125
 *   the number nearest to x / scale, ties to the one of even code, 6 at most
 * It reads back as number * scale, which f32 and bf16 hold exactly; the 32
 * channels read back as NaN where one of them is not finite. A token's numbers
 * depend on its own values alone. (head_dim / 2 + head_dim / 32) bytes per token
 * and head for keys and as many for values (head_dim padded to 64 or 128), and 4
 * for the token's weight: what attention it has got.
 *
 * Rows, streams, captures, devices and the order of calls are as for rtg_qcache
 * above: one call or replay at a time on one cache. ---- */
typedef struct rtg_fourbit rtg_fourbit;
/* Errors: "head_dim <hd> is not supported (1 to 128)", capacities over 4000000
 * tokens, more than 1000000 pairs of sequence and head. */
rtg_result rtg_fourbit_new(size_t n_seq, size_t n_head, size_t head_dim, size_t capacity, rtg_fourbit** out);
void rtg_fourbit_destroy(rtg_fourbit* cache);
/* As rtg_qcache_append. The new tokens' weights are 0. */
rtg_result rtg_fourbit_append(rtg_fourbit* cache, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n_new,
                              const int32_t* counts, const int32_t* start, void* stream);
/* As rtg_qcache_read. */
rtg_result rtg_fourbit_read(const rtg_fourbit* cache, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n,
                            const int32_t* first, void* stream);
/* As rtg_qcache_attend: causal attention of the last counts[s] tokens of every
 * sequence, rows of padding and of queries before the first token 0. Sums are f32,
 * probabilities have 24 bits for f32 results and 16 for the others (2^-16 of each),
 * whatever the capacity; results are rounded to dtype once. Queries times scale,
 * scores, and 256 times the largest |v| times the number of keys have to be within
 * f32. A key that reads back as NaN makes the rows NaN that see it, a value their
 * channels of the same 32, and no others; a query that is not finite gives a row of
 * NaN.
 *
 * With stats (n_seq * n_q * n_q_head * 2 f32 to work in, not NULL) the weights of all
 * tokens then become decay (0 .. 1; 0 whatever they were) times what they are, plus
 * the probabilities that the counted queries of all heads of the token's head give
 * them: sums in f32, in a fixed order. */
rtg_result rtg_fourbit_attend(rtg_fourbit* cache, rtg_dtype dtype, const rtg_rows* queries, size_t n_q,
                              size_t n_q_head, const int32_t* counts, float scale, const rtg_rows* out, float* stats,
                              float decay, void* stream);
/* The weights of tokens 0 .. n - 1 to out [n_seq][n_head][n], 0 where there is no
 * token; and x [n_seq][n_head][n] added to those of the tokens that there are. */
rtg_result rtg_fourbit_weights(const rtg_fourbit* cache, float* out, size_t n, void* stream);
rtg_result rtg_fourbit_add_weights(rtg_fourbit* cache, const float* x, size_t n, void* stream);
/* Cuts every sequence longer than `keep` to that many tokens: each head keeps the
 * last `recent` and, of the others, the keep - recent of the largest weights (of
 * equal ones the first; NaN is larger than all), in their order and with their
 * weights. kept [n_seq][n_head][keep]: which tokens these were, ascending, -1
 * behind those of a shorter sequence. Positions count what is left from then on:
 * keys that hold rotary positions keep those they were written with. */
rtg_result rtg_fourbit_evict(rtg_fourbit* cache, size_t keep, size_t recent, int32_t* kept, void* stream);
/* As rtg_qcache_lengths. */
rtg_result rtg_fourbit_lengths(rtg_fourbit* cache, uint32_t* out, void* stream);

/* ---- Causal attention over packed prompts (no counterpart in the reference,
 * whose prompts are one sequence, gpt2.rs:639-770): rows of n_seq sequences one
 * behind the other, each attending to itself; query row i of a sequence sees its
 * rows 0 .. i. Rows are [n_rows][heads][head_dim] in device memory of the current
 * device (stride_seq is not used), offsets n_seq + 1 device int32: sequence s has
 * rows offsets[s] .. offsets[s + 1] - 1. Offsets are clamped to the rows there are,
 * and one that descends counts as the largest before it (its sequence has no row).
 * Rows of no sequence are set to 0. Query head h reads
 * key/value head h / (n_q_head / n_head), at most 1024 of them one.
 *
 * softmax of scale * q . k; sums are f32, results rounded to dtype once.
 * Probabilities have 24 bits for f32 rows, 16 for bf16 (2^-16 of each) and 22 for
 * f16, there in steps of 2^-30 of the row's largest. Queries times scale, scores, and
 * 256 times the largest |v| times the number of keys have to be within f32.
 * What is not finite: a query makes its row NaN, a value the channel not finite of the
 * rows that see it, a NaN in a key the rows NaN that see it. An infinity in a key does
 * the same for f32 rows; of bf16 and f16 ones it counts as the score that it gives, so
 * a score of -infinity takes no part in its row. No other results depend on them.
 * Enqueues one kernel on `stream`, allocates nothing, may be captured; out must
 * not overlap the others. ---- */
rtg_result rtg_attend_packed(rtg_dtype dtype, const rtg_rows* q, const rtg_rows* k, const rtg_rows* v, size_t n_rows,
                             size_t n_q_head, size_t n_head, size_t head_dim, const int32_t* offsets, size_t n_seq,
                             float scale, const rtg_rows* out, void* stream);

/* ---- BpeTokenizer, rusttorch-core/src/data/tokenizer.rs (host-side text in
 * and out; used by the reference's example at examples/gpt2.rs:77-95).
 * Text is UTF-8 with an explicit length (a Rust &str). Buffers that a call
 * returns (ids, text, spans) are owned by the caller and released with
 * rtg_free_buffer. Errors carry the reference's messages. ---- */
typedef struct rtg_tokenizer rtg_tokenizer;
/* BpeTokenizer::from_files, tokenizer.rs:45-53. Errors: "Failed to read
 * vocab.json: <io error>", "Failed to read merges.txt: <io error>", then those
 * of from_strings. */
rtg_result rtg_tokenizer_from_files(const char* vocab_json_path, const char* merges_txt_path, rtg_tokenizer** out);
/* BpeTokenizer::from_strings, tokenizer.rs:55-82 (parse_vocab_json :356-401,
 * parse_merges :486-514). */
rtg_result rtg_tokenizer_from_strings(const char* vocab_json, size_t vocab_len, const char* merges_txt,
                                      size_t merges_len, rtg_tokenizer** out);
/* BpeTokenizer::from_vocab_and_merges, tokenizer.rs:186-219: token i gets id
 * i, merge rule r gets rank r. Strings are NUL-terminated UTF-8. */
rtg_result rtg_tokenizer_from_vocab_and_merges(const char* const* vocab, size_t n_vocab, const char* const* merge_a,
                                               const char* const* merge_b, size_t n_merges, rtg_tokenizer** out);
void rtg_tokenizer_destroy(rtg_tokenizer* t);
/* BpeTokenizer::encode, tokenizer.rs:85-112: *ids receives *n token ids. */
rtg_result rtg_tokenizer_encode(const rtg_tokenizer* t, const char* text, size_t len, uint32_t** ids, size_t* n);
/* BpeTokenizer::decode, tokenizer.rs:115-130: *text receives *len bytes of
 * UTF-8 (from_utf8_lossy), NUL-terminated. */
rtg_result rtg_tokenizer_decode(const rtg_tokenizer* t, const uint32_t* ids, size_t n, char** text, size_t* len);
/* BpeTokenizer::vocab_size / token_to_id / id_to_token, tokenizer.rs:133-145.
 * id_to_token points *token at the tokenizer's own copy (valid while it
 * lives); false is Rust's None. */
size_t rtg_tokenizer_vocab_size(const rtg_tokenizer* t);
bool rtg_tokenizer_token_to_id(const rtg_tokenizer* t, const char* token, size_t len, uint32_t* id);
bool rtg_tokenizer_id_to_token(const rtg_tokenizer* t, uint32_t id, const char** token, size_t* len);
/* pre_tokenize, tokenizer.rs:260-331 (private in the reference; exported for
 * the parity tests): byte ranges of the words, (*spans)[2k] .. (*spans)[2k+1]. */
rtg_result rtg_tokenizer_pre_tokenize(const char* text, size_t len, size_t** spans, size_t* n_words);
/* build_byte_encoder, tokenizer.rs:223-241 (private in the reference;
 * exported for the parity tests): the code point of every byte. */
void rtg_tokenizer_byte_encoder(uint32_t out[256]);
/* Releases a buffer returned by rtg_tokenizer_encode / _decode / _pre_tokenize. */
void rtg_free_buffer(void* p);

#ifdef __cplusplus
}
#endif
#endif /* RTGPU_H */
