/*
 * vinfer_sampler.h — C ABI of the B200 (sm_100a) token sampler.
 *
 * One fused, memory-bound pass per batch of logits rows: repetition / presence / frequency
 * penalties from per-row token-count histograms, temperature, top-k, softmax, top-p, min-p,
 * and an inverse-CDF draw from a caller-supplied uniform. A vocab-sharded mode reduces each
 * rank's shard to a fixed-size candidate record for an all-gather and a merge.
 *
 * Every pointer is caller-owned memory. Device pointers unless stated otherwise; no pointer
 * is retained after a call returns. Calls are stream-ordered on the given CUDA stream
 * (`void*` is a `cudaStream_t`; NULL is the legacy default stream). Functions return
 * VINFER_OK or a VINFER_E_* code and never throw; a device-side problem is reported by OR-ing
 * VINFER_ST_* bits into `*status` (a device int32, may be NULL) and writing -1 as the row's id.
 *
 * The entry points replace these reference interfaces (vinfer, pure PyTorch):
 *   vinfer_sample        <- `sample(logits, params, seed, position) -> int`
 *                           (src/vinfer/runtime/sampler.py:68-77, called per decode step at
 *                           src/vinfer/runtime/generate.py:129), batched over rows, and
 *                           `filtered_probs(logits, params)` (sampler.py:50-65) through
 *                           the optional `out_probs`.
 *   vinfer_sampler_workspace_bytes / _init
 *                        <- per-device workspaces a backend sets up when the engine builds it
 *                           (src/vinfer/kernels/registry.py:9-11, BackendRegistry.resolve
 *                           registry.py:84-88 constructs it once).
 *   vinfer_sample_local / vinfer_sample_merge
 *                        <- no counterpart: the reference has no distributed code. They are
 *                           the vocab-sharded form of `vinfer_sample` (logits split along the
 *                           vocab as a tensor-parallel lm_head produces them,
 *                           src/vinfer/models/qwen/model.py:230-233).
 */
#ifndef VINFER_SAMPLER_H
#define VINFER_SAMPLER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VINFER_SAMPLER_ABI_VERSION 1

/* logits element types */
#define VINFER_DTYPE_F32 0
#define VINFER_DTYPE_BF16 1

/* return codes */
#define VINFER_OK 0
#define VINFER_E_ARG 1      /* a null pointer, a bad size, a dtype or stride out of range */
#define VINFER_E_LIMIT 2    /* a documented limit exceeded (vocab, batch, workspace too small) */
#define VINFER_E_CUDA 3     /* a CUDA runtime call failed (launch, attribute) */

/* bits OR-ed into *status by the device */
#define VINFER_ST_BAD_PARAM 1u   /* a row's parameters are invalid; its id is -1 */
#define VINFER_ST_NONFINITE 2u   /* a row has no finite maximum after processing */
#define VINFER_ST_HIST_FULL 4u   /* vinfer_hist_append: a slot had no room for a new token */
#define VINFER_ST_INTERNAL 8u    /* an internal check failed, or a kernel's wait reached its limit */
#define VINFER_ST_BAD_SCORE 16u  /* vinfer_beam_select: a beam's score is NaN or +inf */
#define VINFER_ST_BAD_PARENT 32u /* vinfer_reorder_states: a parent that cannot be copied from */
#define VINFER_ST_BAD_LIST 64u   /* vinfer_distill_*: an id or a log-probability out of range */

/* args.flags */
#define VINFER_FLAG_EXACT_ALL 1u /* resolve every row with the exact multi-pass search */

/* limits */
#define VINFER_MAX_VOCAB 262144   /* per call (per shard in sharded mode) and in total */
#define VINFER_MAX_BATCH 65535

typedef struct VinferSampleArgs {
  const void* logits;          /* [batch, ld] row-major; the first `vocab` columns are used */
  int32_t dtype;               /* VINFER_DTYPE_F32 or VINFER_DTYPE_BF16 */
  uint32_t flags;              /* VINFER_FLAG_* */
  int64_t batch;               /* rows */
  int64_t vocab;               /* columns processed (the local shard in sharded mode) */
  int64_t ld;                  /* row stride, in elements (>= vocab) */
  int64_t vocab_offset;        /* global id of column 0 (0 unless sharded) */
  int64_t vocab_total;         /* global vocabulary size (== vocab unless sharded) */
  /* per-row parameters, device float32 / int32 [batch]; NULL selects the default */
  const float* temperature;    /* 0 = greedy; default 1 */
  const int32_t* top_k;        /* 0 = off; default 0 */
  const float* top_p;          /* (0, 1], 1 = off; default 1 */
  const float* min_p;          /* [0, 1], 0 = off; default 0 */
  const float* repetition_penalty; /* > 0, 1 = off; default 1 */
  const float* presence_penalty;   /* 0 = off; default 0 */
  const float* frequency_penalty;  /* 0 = off; default 0 */
  /* token-count histograms, CSR over rows, global token ids; NULL row_ptr = no histories */
  const int64_t* hist_row_ptr; /* [batch + 1] */
  const int32_t* hist_ids;     /* [nnz], strictly ascending within each row */
  const int32_t* hist_counts;  /* [nnz]; entries with count <= 0 are ignored */
  const float* uniforms;       /* [batch] in [0, 1); required unless every row is greedy */
  int32_t* out_ids;            /* [batch] sampled global token ids */
  float* out_probs;            /* optional [batch, vocab] final probabilities (parity checks) */
  int32_t* status;             /* optional, one device int32 */
} VinferSampleArgs;

/* ABI version of the loaded library (VINFER_SAMPLER_ABI_VERSION). */
int vinfer_sampler_abi_version(void);

/* Workspace bytes `vinfer_sample` needs for this shape (independent of the device). A workspace
 * of N bytes serves every shape whose size is at most N: it starts with a header whose place and
 * size do not depend on the shape (per-row arrival counters for VINFER_MAX_BATCH rows), which
 * every call leaves at zero. */
size_t vinfer_sampler_workspace_bytes(int64_t batch, int64_t vocab, int32_t dtype);

/* Zero a workspace once after allocating it; calls leave it ready for the next call, of any
 * shape that fits. */
int vinfer_sampler_workspace_init(void* workspace, size_t bytes, void* stream);

/* Sample one token per row. One workspace serves one call at a time. */
int vinfer_sample(const VinferSampleArgs* args, void* workspace, size_t workspace_bytes,
                  void* stream);

/* Log-probability of each row's sampled token under the row's final distribution (after
 * penalties, temperature, top-k / top-p / min-p and renormalisation): the `logprobs` that
 * src/vinfer/server/protocol.py:131-132 rejects today. Call after vinfer_sample with the same
 * args and workspace (it reads the row results that call left there), before the next call on
 * that workspace. out_logprobs: float [batch]; greedy rows get 0 (a one-hot distribution),
 * rows without a result (invalid parameters, no finite logit) NaN. Unsharded calls only. */
int vinfer_sample_logprobs(const VinferSampleArgs* args, float* out_logprobs, void* workspace,
                           size_t workspace_bytes, void* stream);

/* The n most likely tokens of each row's final distribution with their log-probabilities: the
 * `top_logprobs` that src/vinfer/server/protocol.py:131-132 rejects today. Call after
 * vinfer_sample with the same args and workspace, before the next call on that workspace; it
 * streams the logits once more (the n largest processed values, by the candidate path) and
 * prices each token with the row's result that call left: out_ids / out_logprobs are
 * [batch, n] in descending probability (ties by ascending id); a token outside the kept set
 * gets -inf, a slot with no token id -1; a greedy row lists its token with 0 (its distribution
 * is one-hot); a row without a result (invalid parameters) gets -1 and NaN, and a row whose top
 * list ties flood (more than 1,024 equal values) gets -1. 1 <= n <= VINFER_TOP_LOGPROBS_MAX,
 * n < vocab. Unsharded calls only. */
#define VINFER_TOP_LOGPROBS_MAX 32
int vinfer_sample_top_logprobs(const VinferSampleArgs* args, int32_t n, int32_t* out_ids,
                               float* out_logprobs, void* workspace, size_t workspace_bytes,
                               void* stream);

/* ---- vocab-sharded mode -------------------------------------------------------------------
 * Each rank calls vinfer_sample_local on its shard (vocab_offset / vocab_total set), which
 * writes one fixed-size candidate record per row into `records` (this rank's slice of the
 * all-gather buffer). After an all-gather of those buffers in rank order, every rank calls
 * vinfer_sample_merge on the gathered [world][batch] records with identical parameters and
 * uniforms, and gets identical ids. A row whose cut or draw falls outside the candidates is
 * marked in `unresolved` (id -1); the caller resolves it with vinfer_sample on the full row.
 */
size_t vinfer_sample_record_bytes(int32_t record_cap);  /* bytes of one row's record */
int vinfer_sample_local(const VinferSampleArgs* args, int32_t record_cap, void* records,
                        void* workspace, size_t workspace_bytes, void* stream);
int vinfer_sample_merge(const VinferSampleArgs* args, int32_t record_cap, const void* records,
                        int32_t world_size, int32_t* unresolved, void* workspace,
                        size_t workspace_bytes, void* stream);

/* ---- allocation-free variant ---------------------------------------------------------------
 * No counterpart in the reference: an addition of this library. Some callers cannot allocate
 * device memory when they sample: a serving engine that has handed nearly all of HBM to its
 * KV-cache pool at start-up (a cudaMalloc then fails, or waits for the device), or a host
 * that links only this C library and owns no device allocator (a Go, Java or C runtime).
 * vinfer_sample_static is vinfer_sample without the workspace argument: its scratch is a
 * fixed array of VINFER_STATIC_SCRATCH_BYTES compiled into the library, which every device
 * that loads the library holds until the process exits. It allocates nothing.
 *  - Limit: the call returns VINFER_E_LIMIT when vinfer_sampler_workspace_bytes(batch, vocab,
 *    dtype) exceeds VINFER_STATIC_SCRATCH_BYTES (at least 63 rows fit at any vocabulary).
 *  - The first call on a device looks up the array's device address on that device (which
 *    may load the library's device code); make it before any stream capture. The address is
 *    kept for the life of the process: the library does not survive a cudaDeviceReset (or any
 *    other teardown of the device's primary context) in the same process.
 *  - All calls on one device share the array: calls that can overlap on the GPU (different
 *    streams or host threads without ordering) race and corrupt each other's results.
 */
#define VINFER_STATIC_SCRATCH_BYTES (32u << 20)
int vinfer_sample_static(const VinferSampleArgs* args, void* stream);

/* ---- slotted histories for a batched decode loop ----------------------------------------------
 * Replaces the host-side loop of src/vinfer/runtime/generate.py:127-143 (one sample() per step,
 * an int() host sync per token, no token counts kept) for a batch of decode slots, each owned
 * by one request as in src/vinfer/state/pool.py:70-82 (alloc / free of per-request state).
 * Slot s owns entries [s * cap, (s + 1) * cap) of hist_ids / hist_counts (int32): its first
 * hist_len[s] entries are its tokens (ids strictly ascending, counts > 0); the others are
 * padding with count 0 and id VINFER_HIST_PAD_ID - (cap - 1 - position), ascending and above
 * every vocabulary id. With row_ptr[s] = s * cap (int64 [slots + 1]) the arrays are a CSR
 * history that vinfer_sample reads as it is (padding entries are outside every vocabulary),
 * so sample -> append -> sample never leaves the device.
 *  - vinfer_hist_append: for every slot s with tokens[s] >= 0, count tokens[s] once more in
 *    slot s, or insert it in id order. A full slot (hist_len[s] == cap) keeps its counts and
 *    sets VINFER_ST_HIST_FULL in *status (may be NULL). tokens is typically the previous
 *    vinfer_sample's out_ids (an invalid row's id -1 changes nothing).
 *  - vinfer_hist_reset: empty the n slots listed in slot_list (a request leaving its slot);
 *    entries outside [0, slots) are skipped.
 * Both are stream-ordered, one CTA per slot, and allocate nothing. cap <= VINFER_HIST_MAX_CAP.
 *  - vinfer_sample_decode: vinfer_sample and vinfer_hist_append in one call. args' history
 *    is the slotted arrays (row_ptr[s] = s * cap) and is updated in place with each row's
 *    sampled id by the finishing kernel, after every read of it for this step; no out_probs.
 *    A log-probability call (which prices tokens with the counts of the step) must instead
 *    use vinfer_sample, vinfer_sample_logprobs, then vinfer_hist_append.
 */
#define VINFER_HIST_PAD_ID 0x7FFFFFFF
#define VINFER_HIST_MAX_CAP (1 << 20)
int vinfer_hist_append(const int32_t* tokens, int64_t slots, int32_t* hist_ids,
                       int32_t* hist_counts, int32_t* hist_len, int32_t cap, int32_t* status,
                       void* stream);
int vinfer_hist_reset(const int32_t* slot_list, int64_t n, int64_t slots, int32_t* hist_ids,
                      int32_t* hist_counts, int32_t* hist_len, int32_t cap, void* stream);
int vinfer_sample_decode(const VinferSampleArgs* args, int32_t* hist_len, int32_t cap,
                         void* workspace, size_t workspace_bytes, void* stream);

/* ---- beam search -----------------------------------------------------------------------------
 * No counterpart in the reference, which decodes one sequence a request
 * (src/vinfer/runtime/generate.py:105-146). One step over requests of W = `beams` rows each: beam w
 * of request r holds an accumulated log-probability scores[r, w] and row r * W + w of the logits.
 * A continuation's score is scores[r, w] + logits[token] - logsumexp(row).
 *  - out_scores / out_beams / out_tokens [requests, n]: the n best continuations over the request's
 *    beams and the vocabulary, in descending score, ties by beam, then token. Slots behind the last
 *    candidate get -inf, -1, -1. A beam with score -inf is dead and its row is not read; a token
 *    with logit -inf is no candidate.
 *  - next_scores / parents / next_tokens [requests, W] (all three or none): the first W of the
 *    candidates whose token is none of eos[0 .. n_eos), laid into the request's slots: the best
 *    child of a beam stays in the beam's slot, the others fill the slots without a child in
 *    ascending order. parents are slot numbers over all requests (r * W + beam), as
 *    vinfer_reorder_states takes them. A slot without a child gets -inf, itself and -1. n >=
 *    beams * (1 + n_eos) always finds every continuation. next_scores may be the scores array.
 *  - A score that is NaN or +inf sets VINFER_ST_BAD_SCORE, a live row whose logits hold a NaN or
 *    +inf or nothing above -inf VINFER_ST_NONFINITE; such a beam has no candidates.
 * The order is that of exact scores: scores too close for their streamed sums (2.5e-6) are
 * compared with sums taken in double.
 * The workspace needs no initialisation, holds nothing between calls and serves one call at a
 * time; 16-byte aligned. requests * beams <= VINFER_MAX_BATCH. */
#define VINFER_BEAM_MAX_WIDTH 32
#define VINFER_BEAM_MAX_N 128
#define VINFER_BEAM_MAX_EOS 16
typedef struct VinferBeamArgs {
  const void* logits;      /* [requests * beams, ld] row-major; the first `vocab` columns are used */
  int32_t dtype;           /* VINFER_DTYPE_F32 or VINFER_DTYPE_BF16 */
  int32_t beams;           /* W */
  int64_t requests;
  int64_t vocab;
  int64_t ld;              /* row stride, in elements (>= vocab) */
  const float* scores;     /* [requests, beams] */
  const int32_t* eos;      /* [n_eos] stop ids, device; may be NULL when n_eos is 0 */
  int32_t n_eos;
  int32_t n;               /* candidates listed for each request */
  float* out_scores;       /* [requests, n] */
  int32_t* out_beams;      /* [requests, n] */
  int32_t* out_tokens;     /* [requests, n] */
  float* next_scores;      /* [requests, beams], or NULL with the next two */
  int32_t* parents;        /* [requests, beams] */
  int32_t* next_tokens;    /* [requests, beams] */
  int32_t* status;         /* optional, one device int32 */
} VinferBeamArgs;
size_t vinfer_beam_workspace_bytes(int64_t requests, int32_t beams, int64_t vocab, int32_t dtype,
                                   int32_t n);
int vinfer_beam_select(const VinferBeamArgs* args, void* workspace, size_t workspace_bytes,
                       void* stream);

/* ---- decode states that follow the beams -------------------------------------------------------
 * The batched form of the state pool's copy from slot to slot (src/vinfer/state/pool.py): slot s of
 * every state takes the contents of slot parents[s]. A state is described by its runs of
 * contiguous bytes: slot s holds, for every index of the outer dimensions, run_bytes bytes at
 * base + s * slot_stride + sum(index * outer_stride) (strides in bytes).
 *  - In place (dst == src and equal strides, in all states or in none): parents[s] == s leaves the
 *    slot alone; any other parent must keep its own state (parents[parents[s]] == parents[s], as
 *    vinfer_beam_select lays beams out), else the slot is left alone and VINFER_ST_BAD_PARENT set.
 *  - Into another buffer (which must not overlap the source): every slot is copied, from any parent.
 *  - Neither parents nor lengths lie in memory that is written, no two destinations share a byte, and
 *    states copied in place share bytes of the same slot alone.
 *  - lengths (device int32 [slots]) with len_unit_bytes > 0 copies only the first lengths[s]
 *    positions (of len_unit_bytes each) of every run, with len_outer >= 0 only the first lengths[s]
 *    indices of that outer dimension; positions behind them are neither read nor written.
 * A parent outside [0, slots) leaves the slot alone and sets VINFER_ST_BAD_PARENT. `states` is a
 * host array, read during the call. slots <= VINFER_STATE_MAX_SLOTS. Copies go in vectors of up to
 * 16 bytes, the largest that divides every address, stride and size of the state; VINFER_E_LIMIT
 * when a slot has 2^31 of them or more. */
#define VINFER_STATE_MAX_OUTER 4
#define VINFER_STATE_MAX_SLOTS 8192
typedef struct VinferState {
  const void* src;
  void* dst;
  int64_t src_slot_stride;
  int64_t dst_slot_stride;
  int64_t run_bytes;
  int64_t len_unit_bytes;      /* bytes of one position within a run; 0: runs are copied whole */
  int32_t len_outer;           /* the outer dimension that lengths cut; -1: none */
  int32_t n_outer;
  int64_t outer_size[VINFER_STATE_MAX_OUTER];
  int64_t src_outer_stride[VINFER_STATE_MAX_OUTER];
  int64_t dst_outer_stride[VINFER_STATE_MAX_OUTER];
} VinferState;
int vinfer_reorder_states(const VinferState* states, int32_t n_states, const int32_t* parents,
                          int64_t slots, const int32_t* lengths, int32_t* status, void* stream);

/* ---- distillation from a teacher's top log-probabilities -----------------------------------------
 * The training side of vinfer_sample_top_logprobs: rows of a student's logits against the lists of
 * token ids and log-probabilities that a teacher left (natural logarithms, at the temperature of
 * the student's softmax). With q = softmax(logits / temperature) and p_j = exp(logprobs_j):
 *   loss[row] = weight * ( sum_j p_j (ln p_j - ln q_j)  [ + p_t (ln p_t - ln q_t) with tail ] )
 * tail == 0: the p_j are first divided by their sum. tail != 0: p_t = max(0, 1 - sum p_j) is matched
 * with q_t, the student's mass outside the list. The loss carries no factor temperature^2.
 * Entries with id < 0 are empty; an entry with log-probability -inf lists its token with mass 0. The
 * sum runs over entries: the masses of an id listed twice add up in all that depends on the logits, so
 * that the gradient is that of one entry with their sum; the teacher's own p_j ln p_j stay apart, so
 * that the loss is below that of the one entry by a constant. A row of weight 0 is not read: loss
 * and gradient 0; without tail, a list of no mass gives loss and gradient 0.
 * An id >= vocab or a log-probability that is NaN or +inf sets VINFER_ST_BAD_LIST, logits without a
 * finite log-sum VINFER_ST_NONFINITE; the row's loss and gradient are then NaN.
 *  - vinfer_distill_loss: losses [rows]; row_stats (float [rows, 2], 8-byte aligned) and list_grads
 *    (float [rows, k]) receive what the gradient needs, both or neither.
 *  - vinfer_distill_grad: d(sum_r grad_out[r] * loss[r]) / dlogits, of the logits' type, rounded once
 *    (grad_out NULL: ones; its stride in elements, 0 for one value shared by all rows). args as for
 *    the loss. grad may be the logits (then with their ld).
 *  - vinfer_distill_step: both in one call, grad_out all ones. grad may be the logits. Its one-pass
 *    kernel waits for its own copies and partners; a wait that reaches its limit (seconds) sets
 *    VINFER_ST_INTERNAL, and what that call leaves in loss and grad is not to be used.
 *  - vinfer_distill_step_within: the same with a limit of about wait_ns for each wait (0: one look;
 *    negative: the usual limit).
 * The workspace needs no initialisation and holds nothing between calls; 16-byte aligned. */
#define VINFER_DISTILL_MAX_K 128
#define VINFER_DISTILL_MAX_ROWS (1 << 22)
typedef struct VinferDistillArgs {
  const void* logits;      /* [rows, ld] row-major; the first `vocab` columns are used */
  int32_t dtype;           /* VINFER_DTYPE_F32 or VINFER_DTYPE_BF16 */
  int32_t k;               /* entries of each list */
  int64_t rows;
  int64_t vocab;
  int64_t ld;              /* row stride, in elements (>= vocab) */
  const int32_t* ids;      /* [rows, k] */
  const float* logprobs;   /* [rows, k] */
  const float* weights;    /* [rows], NULL: ones */
  float temperature;       /* in [1e-37, 1e37] */
  int32_t tail;
  int32_t* status;         /* optional, one device int32 */
} VinferDistillArgs;
size_t vinfer_distill_workspace_bytes(int64_t rows, int64_t vocab, int32_t dtype, int32_t k);
int vinfer_distill_loss(const VinferDistillArgs* args, float* loss, float* row_stats,
                        float* list_grads, void* workspace, size_t workspace_bytes, void* stream);
int vinfer_distill_grad(const VinferDistillArgs* args, const float* row_stats,
                        const float* list_grads, const float* grad_out, int64_t grad_out_stride,
                        void* grad, int64_t ld_grad, void* stream);
int vinfer_distill_step(const VinferDistillArgs* args, float* loss, void* grad, int64_t ld_grad,
                        void* workspace, size_t workspace_bytes, void* stream);
int vinfer_distill_step_within(const VinferDistillArgs* args, float* loss, void* grad,
                               int64_t ld_grad, void* workspace, size_t workspace_bytes,
                               int64_t wait_ns, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VINFER_SAMPLER_H */
