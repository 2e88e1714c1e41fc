/*
 * et_speculative.h -- C ABI of the verification of drafted tokens (speculative decoding, MI355X, gfx950).
 *
 * A draft model (or a lookup in the prompt) proposes up to K tokens for each of S sequences; the target
 * model is run once over all of them and leaves K + 1 rows of logits per sequence.  The verification
 * decides from GIVEN random numbers how many of the drafts are kept and draws the one token behind
 * them, so that the tokens are distributed as if the target model alone had been sampled with
 * temperature T from its full vocabulary.  For a sequence with drafts x_0 .. x_{L-1}:
 *
 *   p_i = softmax(target_i / T), i = 0..L;  q_i = softmax(draft_i / T), or all mass on x_i where no draft
 *                                           logits are given
 *   x_i is accepted  <=>  coin_i * q_i(x_i) < p_i(x_i);   n = the first i that is not accepted, or L
 *   n < L : the next token is drawn from max(p_n - q_n, 0), normalised (from p_n where the mass of that
 *           is at most 2^-30, which is rounding noise of two equal distributions)
 *   n == L: it is drawn from p_L
 *   a draw from weights w with coin c is the least v with w_0 + .. + w_v > c * sum(w)  (the last v with
 *           w_v > 0 where no v satisfies that, e.g. for c >= 1)
 *   T == 0: x_i is accepted <=> it is the arg-max of target_i; the next token is the arg-max of target_n
 *           (lowest index wins ties, NaN lowest: the rule of the sampler at temperature 0).  Draft logits
 *           and coins are not read.
 *
 * Decisions are those of 64-bit arithmetic: a token can differ from exact arithmetic only for a coin within
 * about 1e-10 of a border (of two nearly equal models, whose p - q has a mass of R: 1e-15 / R if that is more).
 * Masked tokens (logit -inf) have probability 0 and are never drawn; top-k and top-p are applied by masking the rows of both models
 * beforehand.  For T > 0 a row that holds NaN or +inf, or nothing but -inf, has no distribution; neither
 * has any row of a sequence whose temperature is NaN: a sequence that comes to such a row (the target's,
 * or the draft's beside it) gets -1 as its next token there.  A drafted token outside [0, vocab) is
 * never accepted, and takes nothing away from p where no draft logits are given.
 *
 * Nothing in the reference corresponds to this; status codes and dtype codes are those of et_sampler.h.
 */
#ifndef ET_SPECULATIVE_H_
#define ET_SPECULATIVE_H_

#include "et_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ets_verifier ets_verifier;

/* One call's tensors; every pointer is a DEVICE pointer.  Strides count elements. */
typedef struct ets_verify_batch {
  const void* target_logits; /* [sequences, drafts + 1, vocab], innermost stride 1 */
  const void* draft_logits;  /* [sequences, drafts, vocab] of the same element type, or NULL */
  int32_t dtype;             /* ETS_DTYPE_FLOAT, ETS_DTYPE_HALF or ETS_DTYPE_BFLOAT16 */
  int32_t sequences;         /* 0 .. max_sequences */
  int32_t drafts;            /* K: 0 .. max_drafts */
  float temperature;         /* of every sequence, where `temperatures` is NULL; negative means 0 */
  int64_t target_sequence_stride;
  int64_t target_position_stride;
  int64_t draft_sequence_stride; /* (not read without draft logits) */
  int64_t draft_position_stride;
  const int32_t* draft_tokens; /* [sequences, drafts] (may be NULL where drafts == 0) */
  int64_t draft_tokens_stride;
  const int32_t* draft_lengths; /* [sequences]: drafts of each sequence, clamped to 0 .. drafts; NULL: all `drafts`.
                                 * Rows, tokens and coins behind a sequence's length are not read. */
  const float* temperatures;    /* [sequences] or NULL.  Positive ones are taken between 1e-30 and 1e30. */
  const float* coins;           /* [sequences, drafts + 1] uniforms in [0, 1): one per draft, then the draw's */
  int64_t coins_stride;
  int32_t* tokens; /* out: [sequences, drafts + 1]: accepted drafts, the next token, then -1 */
  int64_t tokens_stride;
  int32_t* accepted; /* out: [sequences] drafts kept, 0 .. length */
} ets_verify_batch;

/* Work buffers for calls of at most max_sequences x max_drafts on the current HIP device (about
 * 16 x max_sequences x (2 max_drafts + 4) x vocab / 2048 bytes), allocated here: calls allocate
 * nothing and may be captured into a graph.  vocab_size is below 16777216. */
ETS_API ets_status ets_verifier_create(int32_t vocab_size, int32_t max_sequences, int32_t max_drafts, ets_verifier** out);
ETS_API ets_status ets_verifier_destroy(ets_verifier* v);

/* Verifies one batch, asynchronously on `hip_stream`.  The struct is read before the call returns.
 * The work buffers are shared by the calls of a handle: issue them, and the graphs that captured
 * them, on one stream at a time. */
ETS_API ets_status ets_verifier_verify(ets_verifier* v, const ets_verify_batch* batch, void* hip_stream);

/* Text of the last error on this handle (NULL: of the calling thread's last failed create). */
ETS_API const char* ets_verifier_last_error(const ets_verifier* v);

#ifdef __cplusplus
}
#endif

#endif /* ET_SPECULATIVE_H_ */
