/*
 * verbo_cache.h - a paged cache of keys and values in 8 bits, and the attention
 * that reads it, beside the B200 (sm_100a) token sampler: what the rows of a
 * decode step (the streams of verbo_cuda_batch_*, the beams of verbo_beam_select)
 * keep of their tokens.  In the same library as verbo_cuda.h and with the
 * conventions of verbo_ops.h: C types, 0 / -1 with verbo_cuda_last_error(),
 * device arrays of the caller, asynchronous calls on a stream of the current
 * device, nothing allocated, synchronised or kept between calls.
 *
 * Codes are e4m3 (NaN 0x7f, largest 448); a block of 16 tokens of one head has
 * one scale, and an element is code * scale.  A row's token i lies in page
 * table[row][i / page] at place i % page; rows may share pages: refs[p] counts
 * the entries of the tables that hold page p, 0 is a free page.  The calls keep
 *   - the entries behind a row's last page at -1,
 *   - refs in step with the tables,
 * and expect both.  What was not set that way is bounded, not checked: page ids
 * outside [0, pages) are taken for no page, lengths for at most width * page.
 *
 * A decode step: verbo_cache_reserve makes room for the rows' new tokens, then
 * per layer verbo_cache_append and verbo_cache_attend; a step of beam search ends
 * with verbo_cache_fork.  Two calls on one cache must not run at the same time,
 * but for appends and attends of different layers.
 */
#ifndef VERBO_CACHE_H
#define VERBO_CACHE_H

#include "verbo_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define VERBO_CACHE_BLOCK 16         /* tokens that share a scale */
#define VERBO_CACHE_MAX_ROWS 4096
#define VERBO_CACHE_MAX_PAGES 4194304
#define VERBO_CACHE_MAX_HEADS 256
#define VERBO_CACHE_MAX_DIM 128
#define VERBO_CACHE_MAX_PAGE 256
#define VERBO_CACHE_MAX_STEPS 32

typedef struct {
  int layers, pages;  /* pages of each layer: one table for all layers */
  int heads, dim;     /* of keys and values; dim a multiple of 16 up to 128 */
  int page;           /* tokens of a page, a multiple of 16 up to 256 */
  int rows, width;    /* width * page <= 2^30; rows * width * page, pages * heads * page < 2^35 */
  unsigned char* k;   /* [layers][pages][heads][page][dim] codes, 16-byte aligned */
  unsigned char* v;
  float* k_scale;     /* [layers][pages][heads][page / 16] */
  float* v_scale;
  int* table;         /* [rows][width] pages, -1 behind the last */
  int* lens;          /* [rows] tokens */
  int* refs;          /* [pages] */
} verbo_cache;

/* Bytes of device memory that verbo_cache_reserve and verbo_cache_compact need
   (16-byte aligned, its own until the call's work is done), or -1. */
VERBO_CUDA_API long long verbo_cache_workspace(const verbo_cache* c);

/* Room for add[r] more tokens of each row (add[r] <= 0: none): pages for them, the
   lowest free ones in the order of the rows, and lens[r] += add[r].  A row whose
   next token falls into a page that other rows hold too gets a copy of that page
   (all layers), the last of them that writes keeps it.
     start[r]   where the new tokens begin (the row's length before), -1: none
     status[0]  0; or the pages that were missing; or -(r + 1) for the lowest row
                that would be longer than width pages.  Unless it is 0 nothing was
                changed and every start is -1. */
VERBO_CUDA_API int verbo_cache_reserve(const verbo_cache* c, const int* add, int* start, int* status,
                                       void* workspace, long long workspace_bytes, void* stream);

/* Rows take over their parents' pages, in place: row b of group g (rows g*beams to
   g*beams + beams - 1) becomes what row parents[g*ld_parents + b] of its group was,
   and shares its pages.  A parent outside [0, beams) empties the row.  rows must be
   a multiple of beams, beams in [1, 32]. */
VERBO_CUDA_API int verbo_cache_fork(const verbo_cache* c, const int* parents, long long ld_parents, int beams,
                                    void* stream);

/* Row r keeps its first keep[r] tokens (all if keep[r] < 0 or above its length); the
   pages behind them are given back.  0 frees a row, its length less the rejected
   tokens undoes a speculation, but for its rounding: where a rejected token raised the
   scale of the block that it shares with kept ones, those stay rounded to that scale. */
VERBO_CUDA_API int verbo_cache_free(const verbo_cache* c, const int* keep, void* stream);

/* Moves the live pages to the front of the pools, all layers, and sets the tables
   and refs: the highest live page goes to the lowest free one, and so on, until
   pages [0, live) are the live ones.  info[0] = live, info[1] = pages that moved. */
VERBO_CUDA_API int verbo_cache_compact(const verbo_cache* c, int* info, void* workspace, long long workspace_bytes,
                                       void* stream);

/* Writes keys and values of `tokens` tokens (token i, head h at k + i*ld_k + h*hd_k,
   dim elements of `dtype`; v the same) into a layer.  Row r's are tokens off[r] to
   off[r + 1] - 1 (off[0] >= 0, ascending, at most `tokens`), or, off NULL, tokens /
   rows of them; they go to the places from start[r] on (start[r] < 0: none), which
   verbo_cache_reserve has made room for.
   A block's scale is the smallest power of two s >= 2^-64 with |x| <= 448 s for its
   finite new elements, but not below what it was where it holds tokens already; if
   it grows, their codes are rounded to the new scale.  A code is x / s rounded to
   nearest even, +-inf as +-448, NaN as NaN. */
VERBO_CUDA_API int verbo_cache_append(const verbo_cache* c, int layer, const void* k, long long ld_k, long long hd_k,
                                      const void* v, long long ld_v, long long hd_v, int dtype, int tokens,
                                      const int* start, const long long* off, void* stream);

/* Attention of the last `steps` tokens (1..32) of every row over a layer:
     out = softmax(scale * q k^T) v
   q             rows*steps tokens (token i, head h at q + i*ld_q + h*hd_q, dim
                 elements of q_type); row r's are tokens r*steps to r*steps + steps
                 - 1, the last one at place lens[r] - 1, each sees the places up to
                 its own.  `heads`: a multiple of the cache's, up to 64 times it; head
                 h reads the cache's head h / (heads / c->heads).
   out           likewise, of out_type.  A token that sees nothing (an empty row)
                 gets zeros.  Tokens in a page outside [0, pages) are left out.
   workspace     verbo_cache_attend_workspace() bytes, 16-byte aligned, its own
                 until the call's work is done.
   Scores' products are exact to 2^-22 of a row's largest element, sums fp32, whatever
   the types.  A weight e^(s - m) is off by at most 2^-22 of itself or, if that is more,
   2^-39 times the quotient of the largest scale among the values of the row's head, be
   their weights 0, and its own block's: 2e-9 where scales are within a factor of
   1000, 2e-6 where one block has values a million times as large as the others.  The same
   call gives the same bits. */
VERBO_CUDA_API int verbo_cache_attend(const verbo_cache* c, int layer, const void* q, int q_type, long long ld_q,
                                      long long hd_q, int heads, int steps, float scale, void* out, int out_type,
                                      long long ld_out, long long hd_out, void* workspace, long long workspace_bytes,
                                      void* stream);
/* Bytes of that call on the current device (0 for few rows and short tables), or -1. */
VERBO_CUDA_API long long verbo_cache_attend_workspace(const verbo_cache* c, int heads, int steps, int q_type);

#ifdef __cplusplus
}
#endif

#endif
