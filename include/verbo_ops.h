/*
 * verbo_ops.h - operators around the B200 (sm_100a) token sampler, in the same
 * library as verbo_cuda.h and with its conventions:
 *   - plain pointers and sizes, no C++ or torch types;
 *   - int functions return 0 on success and -1 on error, pointer functions
 *     NULL on error; the message is verbo_cuda_last_error();
 *   - arrays are DEVICE memory owned by the caller, calls are asynchronous on
 *     the given CUDA stream (NULL = legacy default stream), which has to be a
 *     stream of the current device, where the arrays live.
 * None of the calls allocates, synchronises or keeps anything between calls
 * (verbo_ops_q4_new and _free excepted), so they can be captured into CUDA
 * graphs, issued from several host threads and overlap on several streams.
 *
 * In the order of a decode step: a quantised layer's product with a few
 * hidden rows (verbo_ops_q4_*), what a request does to its logits before the
 * pick (verbo_ops_process_logits, then verbo_cuda_sample or
 * verbo_cuda_batch_step on its output with repeat = 1), and what a server
 * reports of the pick (verbo_ops_token_logprobs).
 */
#ifndef VERBO_OPS_H
#define VERBO_OPS_H

#include "verbo_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest vocab of the logits operators. */
#define VERBO_OPS_MAX_VOCAB 4194304

/* Element types of the caller's arrays. */
enum { VERBO_OPS_F32 = 0, VERBO_OPS_F16 = 1, VERBO_OPS_BF16 = 2 };

/* Penalties on the ids of a row's history.  `repeat` is verbo::Sampling's
   (include/verbo/verbo.hpp:60); frequency and presence are the usual additive
   ones; `last` is the window: the last `last` ids of the row, all if <= 0. */
typedef struct {
  float repeat;
  float frequency;
  float presence;
  int last;
} verbo_ops_penalties;

/* {repeat 1, frequency 0, presence 0, last 0}: no penalty. */
VERBO_CUDA_API verbo_ops_penalties verbo_ops_default_penalties(void);

/* Logits of `rows` rows (row r at logits + r*ld, `vocab` columns of `dtype`)
   -> fp32 rows (row r at out + r*ld_out), column by column in fp32:
     v = logits[r][i]
     c = how often i occurs in the window of row r's history; if c > 0:
       v = v > 0 ? v / repeat : v * repeat     (Sampler::pick, src/sampler.cpp:63)
       v = v - frequency * c
       v = v - presence
     if i is in row r's bias list:  v = v + its bias
     if i is not allowed by row r's mask:  v = -inf  (whatever it was, NaN too)
   every operation rounded to nearest.
   opts          NULL: no penalties, and hist is not read.
   row_penalties NULL, or rows x 3 floats {repeat, frequency, presence}: row r
                 takes these in place of opts' (opts->last still applies).
   hist          CSR like verbo_cuda_sample's; NULL: no history.
   bias_ids, bias, bias_off   row r's list is [bias_off[r], bias_off[r+1]);
                 of an id listed twice the last entry counts.  NULL: no biases.
   mask          row r's words at mask + r*ld_mask (words; 0: one row of words
                 for all rows), bit i%32 of word i/32 set = id i allowed.
                 NULL: all allowed.
   Ids outside [0, vocab) are ignored.
   out may be logits itself (F32, ld_out == ld): then only the columns that
   change are touched.  Any other overlap is refused.  Columns past vocab are
   neither read nor written. */
VERBO_CUDA_API int verbo_ops_process_logits(const void* logits, int dtype, int rows, int vocab, long long ld,
                                            const verbo_ops_penalties* opts, const float* row_penalties,
                                            const int* hist, const long long* hist_off, const int* bias_ids,
                                            const float* bias, const long long* bias_off, const unsigned* mask,
                                            long long ld_mask, float* out, long long ld_out, void* stream);

/* Log-probabilities of softmax(logits / temp), per row of `vocab` columns:
     logprob(i) = (v_i - m) / temp - log sum_j exp((v_j - m) / temp),  m = max v
   ids          one token per row, or NULL: then logprob and rank are not
                written.  logprob[r] is its log-probability, rank[r] the number
                of columns before it in the sampler's order (value descending,
                index ascending).  An id outside [0, vocab): -inf and -1.
   top          0..32: the `top` first columns of that order whose values are
                above -inf, top_ids and top_logprobs [rows][top]; where there
                are fewer, the rest is (-1, -inf).
   A NaN counts as -inf, as in verbo_cuda_sample; -0 equals +0.  A row of -inf
   alone has no probabilities: its log-probabilities are -inf.  Columns at
   +inf share the whole probability (the others' logarithm is -inf).  temp in [1e-4, 1e4]. */
VERBO_CUDA_API int verbo_ops_token_logprobs(const void* logits, int dtype, int rows, int vocab, long long ld,
                                            float temp, const int* ids, float* logprob, int* rank, int top,
                                            int* top_ids, float* top_logprobs, void* stream);

/* ---- products with 4-bit weights ------------------------------------------
   y = x W^T + b for a weight matrix of outs x ins in 4 bits with group scales:
     W[o][i] = s[o][g] * (q[o][i] - z[o][g]),  g = i / group
   The activations stay in their own type (the head of verbo_cuda_tail_*
   quantises them, as the reference does): fp16 x is taken as it is, bf16 and
   fp32 x to within 2^-23 of each value (or 2^-39 of its row's largest, for values
   that much smaller); the products with q - z are exact, the sums fp32.  The same
   call gives the same bits; the order of a sum goes by n, so a row's last bits can
   differ between batches of other sizes. */
typedef struct verbo_ops_q4 verbo_ops_q4;
/* Lays the matrix out on `device` (host or device arrays, read before the
   call returns; work on device arrays is ordered after `stream`).  Refused on a
   stream that is being captured, whose capture goes on.
   q      outs x ins/2 bytes, the reference's Q4 rows (src/kernels.hpp:13-23):
          byte j of a 32-block holds element j in its low half and element
          j+16 in its high half
   s      outs x ceil(ins / group) fp16 scales (the last group may be short)
   zeros  outs x ceil(ins / group) bytes 0..15 (the low half is taken), or
          NULL: 8 everywhere, the reference's
   bias   outs floats, or NULL
   ins a multiple of 32 in [32, 32768], outs in [1, 4194304], group a multiple
   of 32 (the reference's: 32). */
VERBO_CUDA_API verbo_ops_q4* verbo_ops_q4_new(int outs, int ins, int group, const unsigned char* q,
                                              const unsigned short* s, const unsigned char* zeros, const float* bias,
                                              int device, void* stream);
/* Waits for the device; a captured graph that uses the handle dies with it. */
VERBO_CUDA_API void verbo_ops_q4_free(verbo_ops_q4* h);
/* Largest n of a call. */
#define VERBO_OPS_MAX_ROWS 65535
/* Bytes of device memory that a call with n rows needs (16-byte aligned, its own
   until the call's work is done; 0 for a few rows), or -1. */
VERBO_CUDA_API long long verbo_ops_q4_workspace(const verbo_ops_q4* h, int x_type, int n);
/* n rows x (row i at x + i*ldx, ins elements of x_type) -> n rows y (row i at
   y + i*ldy, outs elements of y_type), on the handle's device.  If a copy inside the
   kernel has not come after a second, the call ends with y written in part only, and
   verbo_cuda_check() fails with it. */
VERBO_CUDA_API int verbo_ops_q4_matvec(const verbo_ops_q4* h, const void* x, int x_type, int n, long long ldx, void* y,
                                       int y_type, long long ldy, void* workspace, long long workspace_bytes,
                                       void* stream);

#ifdef __cplusplus
}
#endif

#endif
