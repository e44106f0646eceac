/*
 * llmk_sampler.h — C ABI of the MI355X batched token-sampling engine for
 * llm-rs.  One call samples a whole batch on one GPU, asynchronously on a HIP
 * stream, and replaces the per-row host loop of
 *   llm-scheduler/src/scheduler.rs:138-145  (for each row: backend.sample(..))
 * whose body is
 *   llm-core/src/backend.rs:23-24           (LlmBackend::sample)
 *   llm-core/src/backends/candle.rs:2033-2035 (CandleBackend::sample)
 *   llm-core/src/sampler.rs:25-125          (sample_logits).
 *
 * Conventions follow llm-ffi/src/lib.rs: plain `extern "C"` symbols, an opaque
 * handle with explicit create/destroy (lib.rs:38-84), `#[repr(C)]`-compatible
 * structs (lib.rs:10-29).  Unlike llm-ffi's null/0 sentinels, every call
 * returns a status code (0 = success, negative = error) and
 * llmk_last_error() gives the message for the calling thread.
 *
 * Semantics per row (identical to sampler.rs when the extension fields are
 * at their defaults): repetition penalty (sampler.rs:128-147) -> presence and
 * frequency penalty -> allow-bitmask -> greedy if temperature <= 1e-5
 * (sampler.rs:40-50) -> temperature (sampler.rs:150-157) -> softmax
 * (sampler.rs:56-71) -> order by (probability desc, index asc) (sampler.rs:77)
 * -> min-p -> top-k (sampler.rs:80-89) -> top-p (sampler.rs:92-110) -> draw
 * with the caller's uniform (sampler.rs:113-124).
 *
 * Memory: every pointer in llmk_sample_batch_args is DEVICE memory owned by
 * the caller and must stay valid until the stream reaches the call.
 */
#ifndef LLMK_SAMPLER_H
#define LLMK_SAMPLER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LLMK_OK 0
#define LLMK_ERR_INVALID_ARGUMENT (-1)
#define LLMK_ERR_EMPTY_LOGITS (-2) /* sampler.rs:30-32 "Empty logits" */
#define LLMK_ERR_CAPACITY (-3)     /* batch/vocab above the handle's maxima */
#define LLMK_ERR_HIP (-4)
#define LLMK_ERR_ALIGNMENT (-5)
#define LLMK_ERR_UNSUPPORTED (-6)

/* Token written for a row whose parameters are invalid (NaN temperature,
 * negative top_k, non-finite penalties, ...). */
#define LLMK_INVALID_TOKEN 0xffffffffu

/* Bits of the device status word (llmk_sampler_status). */
#define LLMK_STATUS_INVALID_PARAMS 0x1u
/* More than 8192 distinct history tokens fell in one vocabulary segment of a
 * row (the fast path's LDS tables): the row was sampled by the slow path over
 * its materialised logits, every history token penalised by its count.  The
 * result is exact; the bit reports only that the row took the slower path. */
#define LLMK_STATUS_HISTORY_OVERFLOW 0x2u
#define LLMK_STATUS_SLOT_TIMEOUT 0x4u /* slow-path scratch slot not acquired */
/* llmk_history_append found a row's history buffer full (its token was not
 * appended). */
#define LLMK_STATUS_HISTORY_FULL 0x8u
/* A sampling row held a logit that makes the reference's probabilities NaN
 * (NaN itself, or +inf: l - max = inf - inf), outside the allow-mask's
 * disallowed tokens: the device analogue of sampler.rs's NAN_WARNED
 * warn-once flag (sampler.rs:7-9, :74-76).  The engine reads NaN as -inf
 * and samples on; results for such rows are outside the parity contract. */
#define LLMK_STATUS_NAN_LOGITS 0x10u
/* llmk_pages_update found too few free pages for a row (out_granted says
 * which rows were left as they were). */
#define LLMK_STATUS_PAGES_FULL 0x20u

typedef struct llmk_sampler llmk_sampler; /* opaque; owns device workspace */

/* Logit element types.  bf16 and f16 (IEEE half, the lm_head output of
 * half-precision models) are converted exactly to f32 as they are read, as
 * candle's to_dtype(F32) does before sampling (candle.rs:2007-2010). */
typedef enum { LLMK_F32 = 0, LLMK_BF16 = 1, LLMK_F16 = 2 } llmk_dtype;

typedef struct {
  /* logits[b * row_stride + v], v < vocab; row_stride in elements, rows at
   * any element offset.  Rows that do not start 16-byte aligned (fp32:
   * row_stride not a multiple of 4, bf16 and f16: not of 8, or a base
   * address off 16 bytes) are first copied to aligned rows in the handle's
   * staging buffer, which llmk_sample_batch allocates (once, and again when
   * a call needs more); llmk_sample_batch_static, which allocates nothing,
   * returns LLMK_ERR_ALIGNMENT for them. */
  const void* logits;
  int32_t dtype; /* llmk_dtype */
  uint32_t batch;
  uint32_t vocab;
  uint64_t row_stride;
  /* Per-row parameters, [batch] each; NULL = the SampleParams default
   * (llm-core/src/types.rs:186-195): temperature 1, top_k 0 (off), top_p 1,
   * repetition 1; extensions: min_p 0, presence 0, frequency 0. */
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* repetition_penalty;
  const float* presence_penalty;
  const float* frequency_penalty;
  /* Token history as CSR: hist_offsets[batch+1], hist_tokens[...].  NULL =
   * empty histories.  Ids >= vocab are ignored (sampler.rs:138). */
  const uint32_t* hist_offsets;
  const uint32_t* hist_tokens;
  /* Grammar allow-bitmask, [batch][mask_words_per_row] u32, LSB-first (token
   * t allowed iff bit t&31 of word t>>5 is set); NULL = everything allowed. */
  const uint32_t* allow_mask;
  uint32_t mask_words_per_row;
  /* One uniform in [0,1) per row; replaces rand::thread_rng (sampler.rs:113). */
  const float* uniforms;
  uint32_t* out_tokens; /* [batch] */
  /* Optional processed distribution: the kept candidates after top-p
   * renormalisation, in (p desc, idx asc) order, [batch][out_cap] each; and
   * the kept count per row.  NULL / out_cap 0 = not requested. */
  uint32_t* out_ids;
  float* out_probs;
  uint32_t out_cap;
  uint32_t* out_count;
  /* Optional, [batch]: row b's history is hist_tokens[hist_offsets[b] ..
   * hist_offsets[b] + hist_lengths[b]) (hist_offsets then needs [batch]
   * entries).  This lets the history live in per-row buffers with room to
   * grow, appended to on the device by llmk_history_append.  NULL = CSR. */
  const uint32_t* hist_lengths;
  /* final_logit_softcapping (candle.rs:1803-1807, models whose metadata sets
   * it, candle.rs:606): > 0 = the logits are the lm_head output before the
   * cap, and each is read as cap * tanh(l / cap) evaluated as candle's CPU
   * ops do in the logits' dtype (l * (1/cap) + 0, glibc's tanhf, * cap + 0,
   * each rounded to the dtype); 0 = off.  Fused into the sampling pass: the
   * capped logits are never written. */
  float softcap;
  /* Optional: the count-table form of the history (the per-row counts the
   * scheduler's token push, scheduler.rs:147, accumulates), indexed like
   * hist_tokens: entry i stands for hist_counts[i] occurrences of token
   * hist_tokens[i] (0 is read as 1).  Penalties are those of the history that
   * lists each token that many times (sampler.rs:128-147; the frequency
   * penalty's count).  Entries may come in any order; a token listed twice
   * has the sum of its counts.  llmk_history_count_append keeps such tables
   * sorted and distinct on the device, so a step reads each distinct token
   * once instead of every occurrence.  NULL = one occurrence per entry. */
  const uint32_t* hist_counts;
} llmk_sample_batch_args;

/* Create a sampler on `device` able to serve batches up to max_batch rows of
 * up to max_vocab logits; all device workspace is allocated here.
 * Replaces nothing in the reference (its sampler keeps no state). */
int llmk_sampler_create(llmk_sampler** out, int device, uint32_t max_batch,
                        uint32_t max_vocab);

/* Sample every row of the batch; enqueued on `hip_stream` (a hipStream_t, NULL
 * = default stream) and returns without waiting.  Allocates nothing.
 * Replaces the per-row loop scheduler.rs:138-145 over sampler.rs:25-125.
 * One handle serves one stream at a time (calls on a handle are serialised
 * by stream order; concurrent calls on two streams race on the workspace). */
int llmk_sample_batch(llmk_sampler* s, const llmk_sample_batch_args* args,
                      void* hip_stream);

/* llmk_sample_batch with no handle and no allocation of any kind.  It has no
 * counterpart in the reference: it is for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).  Same arguments, semantics and results as
 * llmk_sample_batch, on the current device; its workspace is a static
 * device array of 108 MiB that each GPU the library runs on holds
 * until the process ends, sized for batch <= 256 and vocab <= 262144 (larger
 * calls fail with LLMK_ERR_CAPACITY).  `status`: optional device u32 into
 * which the call ORs its LLMK_STATUS_* bits (the caller clears it); NULL =
 * the bits are dropped.  Every call on one GPU shares that workspace: calls
 * that overlap on one GPU (two streams, or two threads) race and give wrong
 * results; calls in one stream's order are safe. */
int llmk_sample_batch_static(const llmk_sample_batch_args* args, uint32_t* status,
                             void* hip_stream);

/* Mask-form top-k, batched and in place: replaces apply_top_k
 * (llm-core/src/sampler.rs:160-173) called on each row.  In row b every
 * logit below the top_k[b]-th largest value becomes -inf; values equal to
 * that threshold stay, so more than top_k[b] can remain.  Rows with
 * top_k[b] <= 0 or >= vocab are left as they are (sampler.rs:161-163).
 * logits: device f32 [batch][row_stride] (the reference's &mut [f32]; any
 * stride, no alignment beyond the f32 one); top_k: device [batch].  Enqueued on hip_stream;
 * allocates nothing; uses no workspace of the handle. */
int llmk_apply_top_k(llmk_sampler* s, float* logits, uint32_t batch, uint32_t vocab,
                     uint64_t row_stride, const int32_t* top_k, void* hip_stream);

/* Mask-form top-p, batched and in place: replaces apply_top_p
 * (llm-core/src/sampler.rs:176-216) called on each row.  Softmax of the row,
 * order by (probability desc, index asc), keep the shortest prefix whose
 * sequential f32 running sum reaches top_p[b], set every other logit to
 * -inf.  Rows with top_p[b] >= 1 or NaN, or whose probabilities sum to 0
 * (every logit -inf), are left as they are.  The probabilities are those of
 * llmk_sample_batch at temperature 1 (the same exp and normaliser), and the
 * kept set is what llmk_sample_batch keeps with that top_p alone.  f32 rows
 * at any element offset and stride; batch and vocab within the handle's
 * maxima; uses the handle's workspace (stream order, like
 * llmk_sample_batch).  Allocates nothing, except that rows not starting
 * 16-byte aligned are read through the handle's staging buffer, allocated
 * as llmk_sample_batch does. */
int llmk_apply_top_p(llmk_sampler* s, float* logits, uint32_t batch, uint32_t vocab,
                     uint64_t row_stride, const float* top_p, void* hip_stream);

/* Logit bias (the OpenAI logit_bias map), batched and in place: no
 * function of the reference has it; its formula is the one its test
 * llm-tests/tests/mlc_parity.rs:1060-1072 applies, logits[idx] += bias (f32).
 * Row b's pairs are bias_tokens[j], bias_values[j] for j in
 * [bias_offsets[b], bias_offsets[b+1]) (device CSR, like the history); ids
 * >= vocab are ignored.  The tokens of a row are the keys of a map: a token
 * listed twice gets both biases in an unspecified order.  Run it before
 * llmk_sample_batch on the same stream.  logits: device f32
 * [batch][row_stride], any stride.  Allocates nothing. */
int llmk_apply_logit_bias(llmk_sampler* s, float* logits, uint32_t batch, uint32_t vocab,
                          uint64_t row_stride, const uint32_t* bias_offsets,
                          const uint32_t* bias_tokens, const float* bias_values,
                          void* hip_stream);

/* Appends each row's sampled token to its device-resident history, as the
 * scheduler pushes it (llm-scheduler/src/scheduler.rs:147):
 * hist_tokens[hist_offsets[b] + hist_lengths[b]] = tokens[b] and
 * hist_lengths[b] += 1, for rows whose token is not LLMK_INVALID_TOKEN.  A
 * row already holding `capacity` tokens is left as it is and raises
 * LLMK_STATUS_HISTORY_FULL.  With hist_lengths in llmk_sample_batch_args
 * the next step then reads the grown histories without a host round trip.
 * Enqueued on hip_stream; allocates nothing. */
int llmk_history_append(llmk_sampler* s, uint32_t batch, const uint32_t* hist_offsets,
                        uint32_t* hist_lengths, uint32_t* hist_tokens, uint32_t capacity,
                        const uint32_t* tokens, void* hip_stream);

/* The token push of scheduler.rs:147 on a count-table history: row b's
 * entries hist_tokens/hist_counts[hist_offsets[b] .. + hist_lengths[b]) hold
 * its distinct tokens in ascending order with their occurrences.  A token
 * already listed gets count + 1; a new token is inserted in order with count
 * 1 (hist_lengths[b] += 1), or, when the row already holds `capacity`
 * entries, the row is left as it is and LLMK_STATUS_HISTORY_FULL is raised.
 * Rows whose token is LLMK_INVALID_TOKEN are left as they are.  Pass the same
 * arrays as hist_offsets / hist_tokens / hist_lengths / hist_counts of
 * llmk_sample_batch_args.  Enqueued on hip_stream; allocates nothing. */
int llmk_history_count_append(llmk_sampler* s, uint32_t batch, const uint32_t* hist_offsets,
                              uint32_t* hist_lengths, uint32_t* hist_tokens,
                              uint32_t* hist_counts, uint32_t capacity,
                              const uint32_t* tokens, void* hip_stream);

/* Speculative-decoding verification, batched: the residual resampling that
 * docs/mlc-contracts.md:83-84 describes (BatchVerifyDraftTokensWithProb-
 * AfterTopP) at the hook the reference leaves for it (llm-core/src/
 * backend.rs:20-22, "so the scheduler can apply speculative decoding"); the
 * reference itself has no implementation.  Row b verifies draft token
 * draft_tokens[b] against the target distribution p that llmk_sample_batch
 * returned for the row: its kept list ids/probs[b * list_cap ..] (in
 * (p desc, idx asc) order) and counts[b], i.e. out_ids/out_probs/out_count
 * with out_cap = list_cap; p is 0 outside the list.  draft_probs[b *
 * draft_stride + t] is the draft model's probability of token t (an id >= vocab
 * in a list, which the sampler never writes, reads q = 0).
 *   accept iff u_accept[b] * q(d) < p(d)  (the contract's reject when
 *   r >= p/q): out_tokens[b] = d, out_accepted[b] = 1;
 *   else out_accepted[b] = 0 and out_tokens[b] is drawn from the residual
 *   max(p - q, 0) over the kept list (one f32 subtraction each): R = its
 *   sequential f32 sum in list order; the first entry whose running sum of
 *   residual/R reaches u_resample[b] (the reference's `r <= cumulative`,
 *   sampler.rs:113-124), else the last entry with a positive residual; when
 *   R = 0, the same draw over p itself.
 * A chain of k draft tokens is k rows, one per position; the caller keeps
 * the accepted prefix and the first resampled token.  A row whose count is 0
 * or above list_cap (the list was cut) or whose draft token is >= vocab gets
 * LLMK_INVALID_TOKEN and raises LLMK_STATUS_INVALID_PARAMS.  Device arrays;
 * enqueued on hip_stream; allocates nothing. */
int llmk_verify_batch(llmk_sampler* s, uint32_t batch, uint32_t vocab, const uint32_t* ids,
                      const float* probs, uint32_t list_cap, const uint32_t* counts,
                      const uint32_t* draft_tokens, const float* draft_probs,
                      uint64_t draft_stride, const float* u_accept, const float* u_resample,
                      uint32_t* out_tokens, uint32_t* out_accepted, void* hip_stream);

/* Processed logits: the steps that llmk_sample_batch applies before its
 * softmax, written out (for log-probabilities of the distribution that is
 * sampled from, for other samplers, for speculative chains).  For row b of
 * sequence q = row_seq[b] and every token v < vocab, in this order:
 *   x = the logit as f32; softcap > 0: x = softcap * tanh(x / softcap);
 *   x += the sum of the sequence's biases of v, in listing order;
 *   n = occurrences of v in the sequence's history and the row's extra
 *   tokens; n > 0: x = x > 0 ? x / repetition : x * repetition
 *   (sampler.rs:128-147), x -= presence + n * frequency (mlc_parity.rs:1083);
 *   v not allowed by the row's mask: x = -inf;
 *   temperature > 1e-5: x /= temperature (sampler.rs:150-157).
 * Each step is one f32 operation, as in llmk_sample_batch: without a softcap
 * the f32 output gives llmk_sample_batch, with no penalties, the tokens that
 * the logits give with them, at temperature 1 for the rows divided here and at
 * temperature 0 for the greedy ones (temperature <= 1e-5, sampler.rs:40-50):
 * those are not divided, and at temperature 1 they would be drawn from.
 * The result is rounded once, to out_dtype.
 * NaN stays NaN.  (The softcap of 16-bit logits is computed in f32 here and
 * not rounded to 16 bits between its steps as llmk_sample_batch does.)
 * A softcap takes infinite logits to +-softcap, here and in llmk_sample_batch:
 * a token that the logits hold at -inf can be sampled again after it.  Tokens
 * are banned behind the softcap, by allow_mask or a bias of -inf.
 *
 * A row whose sequence is >= sequences, whose mask_index is >= mask_rows or
 * one of whose parameters is not finite is filled with NaN and raises
 * LLMK_STATUS_INVALID_PARAMS. */
typedef struct {
  /* logits[b * row_stride + v], rows at any element offset;
   * batch * row_stride <= 2^55. */
  const void* logits;
  int32_t dtype; /* llmk_dtype */
  uint32_t batch;
  uint32_t vocab;
  uint64_t row_stride;
  /* out[b * out_stride + v]; elements of a row past vocab are not written.
   * out_dtype is LLMK_F32 or dtype.  In place: out = logits with the same
   * dtype and stride; any other overlap of the rows is refused. */
  void* out;
  int32_t out_dtype;
  uint64_t out_stride;
  float softcap; /* 0 = off, or 2^-126 and above */
  /* The sequence of each row, [batch]: rows of one sequence share its
   * parameters, history and biases (a speculative chain's positions).
   * NULL: row b is sequence b, and sequences is not read. */
  const uint32_t* row_seq;
  uint32_t sequences;
  /* Per sequence; NULL = 1, 1, 0, 0 (types.rs:186-195). */
  const float* temperature;
  const float* repetition_penalty;
  const float* presence_penalty;
  const float* frequency_penalty;
  /* Histories, indexed by sequence, in any form llmk_sample_batch_args takes:
   * CSR, per-row buffers (hist_lengths), count tables (hist_counts).  A
   * token's occurrences are summed modulo 2^32. */
  const uint32_t* hist_offsets;
  const uint32_t* hist_tokens;
  const uint32_t* hist_lengths;
  const uint32_t* hist_counts;
  /* Tokens that join row b's history for this row alone (the drafts before
   * its position): extra_tokens[extra_begin[b] .. + extra_count[b]), [batch]
   * each; rows may share them.  NULL = none. */
  const uint32_t* extra_begin;
  const uint32_t* extra_count;
  const uint32_t* extra_tokens;
  /* Logit biases per sequence, CSR: bias_offsets[sequences + 1].  A list
   * holds at most 2^31 pairs, of which several may have one token; ids >=
   * vocab are ignored.  NULL = none. */
  const uint32_t* bias_offsets;
  const uint32_t* bias_tokens;
  const float* bias_values;
  /* Allow-masks, [mask_rows][mask_words_per_row] u32 as in
   * llmk_sample_batch_args.  Row b takes row mask_index[b], none if that is
   * negative; NULL mask_index: row b takes row b (mask_rows >= batch). */
  const uint32_t* allow_mask;
  uint32_t mask_words_per_row;
  uint32_t mask_rows;
  const int32_t* mask_index;
} llmk_process_logits_args;

/* Enqueued on hip_stream; allocates nothing and uses no workspace of the
 * handle, whose maxima do not bound batch and vocab.  batch * ceil(vocab / 4096)
 * < 2^24. */
int llmk_process_logits(llmk_sampler* s, const llmk_process_logits_args* args,
                        void* hip_stream);

/* Log-probabilities of a batch of rows (what an OpenAI-style `logprobs`
 * answer holds; no function of the reference has it).  With x = the logit as
 * f32 (softcapped as in llmk_process_logits, but for -inf, which stays -inf: a
 * banned token has no probability here, whatever the softcap), m = max x and S = sum
 * exp(x - m), both held in f32: log p(v) = (x_v - m) - log S.  For logits that
 * hold no -inf these are, to f32 accuracy, the log-probabilities of
 * llmk_process_logits' output with that softcap alone.  Tokens are
 * ordered by (raw logit descending, index ascending); NaN is read as -inf.
 *   out_logprobs[b] = log p(tokens[b]), out_ranks[b] = tokens before it in
 *   the order (0: the likeliest);
 *   out_top_ids / out_top_logprobs[b * top_n ..]: the first top_n tokens.
 * A token with a logit of -inf has -inf, also in a row that holds nothing
 * else; a row with a +inf logit has NaN for every other.  A token
 * >= vocab gives NaN and rank LLMK_INVALID_TOKEN; entries of the top list
 * past vocab are LLMK_INVALID_TOKEN and -inf. */
typedef struct {
  const void* logits; /* as in llmk_process_logits_args */
  int32_t dtype;
  uint32_t batch;
  uint32_t vocab; /* <= 2^20 */
  uint64_t row_stride;
  float softcap;
  const uint32_t* tokens; /* [batch]; NULL: the top list alone */
  float* out_logprobs;    /* [batch], with tokens */
  uint32_t* out_ranks;    /* [batch], with tokens; NULL: not wanted */
  uint32_t top_n;         /* 0 .. 32 */
  uint32_t* out_top_ids;  /* [batch][top_n] */
  float* out_top_logprobs;
} llmk_logprobs_args;

/* Enqueued on hip_stream; allocates nothing; uses the handle's workspace
 * (stream order, like llmk_sample_batch).  Batches above the handle's
 * max_batch run with one workgroup per row.  batch < 2^24; < 2^23 with a top
 * list and vocab above 39 * 1024.  A top list that has about as many entries as
 * the row has tiles of 1024 logits, or more, takes several times as long as a
 * shorter one. */
int llmk_logprobs(llmk_sampler* s, const llmk_logprobs_args* args, void* hip_stream);

/* A cache in pages: what the scheduler's block allocator keeps on the host
 * (llm-scheduler/src/block_allocator.rs, called at scheduler.rs:162-187), on
 * the device.  Row r holds lengths[r] tokens in the first
 * ceil(lengths[r] / page_tokens) pages of its table row; entries behind them
 * mean nothing and are left as they are.  refs[p] counts the rows that hold
 * page p, and bit p & 31 of used[p >> 5] says whether any does.  All arrays
 * are device memory of the caller; a zeroed cache is an empty one.  What the
 * pages hold lies in n_pools pools (a layer's keys, its values, their scales,
 * ...): page p of pool i is the pools[2 i + 1] bytes at address
 * pools[2 i] + p * pools[2 i + 1]. */
typedef struct {
  uint32_t rows;        /* <= 2^20 */
  uint32_t max_pages;   /* table entries per row */
  uint32_t page_tokens; /* tokens per page; max_pages * page_tokens < 2^31 */
  uint32_t num_pages;   /* <= 2^25 */
  uint32_t* table;      /* [rows][max_pages] */
  uint32_t* lengths;    /* [rows] */
  uint32_t* refs;       /* [num_pages] */
  uint32_t* used;       /* [ceil(num_pages / 32)] */
  uint32_t* work;       /* llmk_pages_work_words words, 8-byte aligned, zeroed once */
  uint32_t n_pools;     /* <= 65535 */
  uint64_t page_bytes;  /* the largest pools[2 i + 1], <= 2^40 */
  const uint64_t* pools; /* [n_pools][2], in device memory: address, bytes per page */
} llmk_page_cache;

/* The words of llmk_page_cache.work. */
int llmk_pages_work_words(uint32_t rows, uint32_t num_pages, uint64_t* words);

/* One step of a cache's rows.  parents and new_lengths: [rows], negative (or
 * a NULL array) = nothing asked of the row.  Every row states what it asks
 * for, and the result is that of these steps:
 *  1. forks: row r with parent p = parents[r] begins with p's first
 *     min(lengths[p], new_lengths[r] if >= 0) tokens: it shares their pages.
 *     The row must be empty, and p must be another row that has no parent in
 *     this call; p may end, shrink or grow in the same call.
 *  2. rows longer than new_lengths shrink to it; pages no row holds any more
 *     are free.
 *  3. rows shorter than new_lengths grow to it, in ascending order, each new
 *     page the lowest free one.  A row whose last page is partly filled and
 *     shared first gets a copy of it in a page of its own (the lowest free),
 *     unless every other row that holds it has left it so before.  From the
 *     first row on for which too few pages are left, rows that need a page
 *     or whose last page is shared stay as they are after steps 1 and 2.
 * out_granted[r] = 1, or 0 for a row that did not get what it asked for: too
 * few pages (LLMK_STATUS_PAGES_FULL), or an invalid request (a new length
 * above max_pages * page_tokens, a row that may not fork), which changes
 * nothing and raises LLMK_STATUS_INVALID_PARAMS.  Page contents move only
 * for the copies of step 3.  Enqueued on hip_stream; allocates nothing; calls
 * on one cache must not overlap. */
int llmk_pages_update(llmk_sampler* s, const llmk_page_cache* cache, const int32_t* parents,
                      const int32_t* new_lengths, uint32_t* out_granted, void* hip_stream);

/* Moves the M pages in use to pages 0 .. M - 1: the i-th used page at or
 * above M goes to the i-th free page below it, contents, counts and table
 * entries; no other page moves.  out_map[p] (required, [num_pages]) = the
 * place of page p's contents now, p for pages that did not move. */
int llmk_pages_compact(llmk_sampler* s, const llmk_page_cache* cache, uint32_t* out_map,
                       void* hip_stream);

/* Copies page src[i] to page dst[i] in every pool, i < n: n_pools pools of
 * num_pages pages, with page_bytes the most that a page of any has, as in
 * llmk_page_cache.  It copies rows of anything held
 * at a fixed pitch as well, per-row token histories and their lengths among
 * them.  A page may be the source of several copies; the destinations must
 * be distinct and none of them a source.  Pairs with a page >= num_pages are
 * left out and raise LLMK_STATUS_INVALID_PARAMS. */
int llmk_pages_copy(llmk_sampler* s, uint32_t n_pools, const uint64_t* pools,
                    uint64_t page_bytes, uint32_t num_pages, uint32_t n, const uint32_t* src,
                    const uint32_t* dst, void* hip_stream);

/* Reads and clears the device status word (OR of LLMK_STATUS_* bits raised by
 * calls since the last read).  Synchronises `hip_stream`. */
int llmk_sampler_status(llmk_sampler* s, void* hip_stream, uint32_t* status);

void llmk_sampler_destroy(llmk_sampler* s);

/* Message of the last error on the calling thread ("" if none). */
const char* llmk_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
