/*
 * verbo_beam.h - beam search beside the B200 (sm_100a) token sampler, in the
 * same library as verbo_cuda.h and verbo_ops.h and with their conventions (C
 * types, 0 / -1 with verbo_cuda_last_error(), device arrays of the caller,
 * asynchronous calls on a stream of the current device, nothing allocated,
 * synchronised or kept between calls).
 *
 * A search keeps `beams` rows per request, row r*beams + b for beam b of
 * request r, in the logits and in every state.  A step: the model's logits
 * (verbo_ops_process_logits may change them), verbo_beam_select, then the
 * states in the order of the chosen parents (verbo_beam_reorder; for a cache
 * of pages verbo_cache_fork, verbo_cache.h).
 */
#ifndef VERBO_BEAM_H
#define VERBO_BEAM_H

#include "verbo_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest beams, and largest take, of a call. */
#define VERBO_BEAM_MAX_BEAMS 32
#define VERBO_BEAM_MAX_TAKE 64

/* The `take` best continuations of each request, out of its beams x vocab:
     value(b, i) = scores[b] + (x[b][i] - lse[b])
     lse[b] = m + log sum_j exp(x[b][j] - m),  m = max_j x[b][j]
   in the order of value descending (in 64 bits), then beam ascending, then
   logit descending, then token ascending.
   logits        requests*beams rows (row i at logits + i*ld, vocab columns of
                 `dtype`).  A NaN counts as -inf; columns at -inf are no
                 candidates.  Of a row with columns at +inf those alone are,
                 with -log(their number).
   scores        requests*beams floats: the beams' summed log-probabilities.  A
                 beam at -inf (or NaN) has no candidates, whatever its row holds;
                 so a request's first step, when all its beams hold the same
                 prompt, has 0 for one of them and -inf for the others.
   take          1..64.
   out_scores, parents, tokens   [requests][take]: the value rounded to fp32, the
                 beam (0..beams-1) and the token; where there are fewer candidates
                 -inf, -1 and -1.  out_scores may be scores only if take == beams.
   workspace     verbo_beam_workspace() bytes, 16-byte aligned, its own until the
                 call's work is done.
   lse is off by at most the sum of the columns' shares of the row times 2^-23
   (|x - m| + 7.5), where a column that stands out by more than 1 counts nothing: by
   some 1e-8 in a model's rows, and by less than 1e-7 in all that were measured.
   Candidates of two beams that lie nearer to each other may change places.  Equal rows
   have equal sums wherever they lie. */
VERBO_CUDA_API int verbo_beam_select(const void* logits, int dtype, int requests, int beams, int vocab, long long ld,
                                     const float* scores, int take, float* out_scores, int* parents, int* tokens,
                                     void* workspace, long long workspace_bytes, void* stream);
/* Bytes that a call of that size needs, or -1. */
VERBO_CUDA_API long long verbo_beam_workspace(int requests, int beams, int take);

/* One state: requests*beams rows of row_bytes, row i at data + i*stride_bytes. */
typedef struct {
  void* data;
  long long row_bytes;
  long long stride_bytes;
} verbo_beam_state;

/* Puts the rows of n states (n >= 0, host array) in the order of their parents,
   in place: row b of request r becomes what row parents[r*ld_parents + b] of that
   request was.  A parent outside [0, beams) leaves its row as it was.  One launch
   for up to 32 states of one alignment (rows whose address, length and stride are
   multiples of 16 bytes are moved fastest).  States must not overlap one another. */
VERBO_CUDA_API int verbo_beam_reorder(const verbo_beam_state* states, int n, int requests, int beams,
                                      const int* parents, long long ld_parents, void* stream);

#ifdef __cplusplus
}
#endif

#endif
