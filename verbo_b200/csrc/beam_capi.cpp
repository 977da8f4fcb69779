// C ABI of beam search (include/verbo_beam.h): argument checks and launches.
#include <cuda_runtime.h>

#include <climits>
#include <string>

#include "beam.cuh"
#include "capi_checks.hpp"
#include "capi_guard.hpp"
#include "ops.cuh"
#include "verbo_beam.h"

namespace {

using vb::check_aligned;
using vb::check_rows;
using vb::check_type;
using vb::cuda_ok;
using vb::fail;
using vb::guard;
using vb::overlap;

static_assert(VERBO_BEAM_MAX_BEAMS == vb::kBeamMaxBeams && VERBO_BEAM_MAX_TAKE == vb::kBeamMaxTake, "one limit");

void check_search(int requests, int beams) {
  if (requests < 0) fail("requests must be >= 0");
  if (beams < 1 || beams > VERBO_BEAM_MAX_BEAMS)
    fail("beams must be in [1, " + std::to_string(VERBO_BEAM_MAX_BEAMS) + "]");
  if (static_cast<long long>(requests) * beams > INT_MAX / vb::kBeamMaxTake) fail("too many rows");
}

void check_take(int take) {
  if (take < 1 || take > VERBO_BEAM_MAX_TAKE)
    fail("take must be in [1, " + std::to_string(VERBO_BEAM_MAX_TAKE) + "]");
}

bool touch(const void* a, long long la, const void* b, long long lb) { return overlap(a, la, la, b, lb, lb, 1, 1); }

}  // namespace

extern "C" {

VERBO_CUDA_API long long verbo_beam_workspace(int requests, int beams, int take) {
  return guard(
      [&]() -> long long {
        check_search(requests, beams);
        check_take(take);
        return static_cast<long long>(vb::beam_workspace_bytes(requests * beams, take));
      },
      -1);
}

VERBO_CUDA_API int verbo_beam_select(const void* logits, int dtype, int requests, int beams, int vocab, long long ld,
                                     const float* scores, int take, float* out_scores, int* parents, int* tokens,
                                     void* workspace, long long workspace_bytes, void* stream) {
  return guard(
      [&]() {
        check_type(dtype, "dtype");
        check_search(requests, beams);
        check_take(take);
        if (vocab < 1 || vocab > VERBO_OPS_MAX_VOCAB)
          fail("vocab must be in [1, " + std::to_string(VERBO_OPS_MAX_VOCAB) + "]");
        if (requests == 0) return 0;
        const int rows = requests * beams;
        check_rows(logits, dtype, rows, vocab, ld, "logits");
        if (!scores) fail("scores must not be NULL");
        if (!out_scores || !parents || !tokens) fail("out_scores, parents and tokens must not be NULL");
        check_aligned(scores, 4, "scores");
        check_aligned(out_scores, 4, "out_scores");
        check_aligned(parents, 4, "parents");
        check_aligned(tokens, 4, "tokens");
        const long long size = vb::ops_type_size(dtype), out = 4ll * requests * take;
        const long long need = static_cast<long long>(vb::beam_workspace_bytes(rows, take));
        if (!workspace || workspace_bytes < need)
          fail("the workspace must have " + std::to_string(need) + " bytes (verbo_beam_workspace)");
        check_aligned(workspace, 16, "workspace");
        if (touch(scores, 4ll * rows, out_scores, out) && !(out_scores == scores && take == beams))
          fail("out_scores overlaps scores");
        const void* outs[] = {out_scores, parents, tokens};
        for (int i = 0; i < 3; ++i) {
          if (overlap(logits, ld * size, vocab * size, outs[i], out, out, 1, rows)) fail("an output overlaps logits");
          if (touch(outs[i], out, workspace, need)) fail("an output overlaps the workspace");
          if (i > 0 && touch(outs[i], out, scores, 4ll * rows)) fail("an output overlaps scores");
          for (int j = 0; j < i; ++j)
            if (touch(outs[i], out, outs[j], out)) fail("two outputs overlap");
        }
        if (overlap(logits, ld * size, vocab * size, workspace, need, need, 1, rows) ||
            touch(scores, 4ll * rows, workspace, need))
          fail("the workspace overlaps logits or scores");
        vb::BeamSelectArgs a{};
        a.logits = logits;
        a.ld = ld;
        a.requests = requests;
        a.beams = beams;
        a.vocab = vocab;
        a.take = take;
        a.scores = scores;
        a.out_scores = out_scores;
        a.parents = parents;
        a.tokens = tokens;
        a.workspace = workspace;
        cuda_ok(vb::launch_beam_select(a, dtype, static_cast<cudaStream_t>(stream)), "kernel launch");
        return 0;
      },
      -1);
}

VERBO_CUDA_API int verbo_beam_reorder(const verbo_beam_state* states, int n, int requests, int beams,
                                      const int* parents, long long ld_parents, void* stream) {
  return guard(
      [&]() {
        check_search(requests, beams);
        if (n < 0) fail("n must be >= 0");
        if (n == 0 || requests == 0) return 0;
        if (!states || !parents) fail("states and parents must not be NULL");
        check_aligned(parents, 4, "parents");
        if (ld_parents < beams && requests > 1) fail("ld_parents must be at least beams");
        if (ld_parents > (1ll << 60) / requests) fail("ld_parents is too large");
        const int rows = requests * beams;
        const long long list = 4 * ((requests - 1) * ld_parents + beams);
        for (int i = 0; i < n; ++i) {
          const verbo_beam_state& s = states[i];
          if (s.row_bytes < 0) fail("row_bytes must be >= 0");
          if (s.row_bytes == 0) continue;
          if (!s.data) fail("a state's data must not be NULL");
          if (s.stride_bytes < s.row_bytes) fail("a state's stride must be at least its row's length");
          if (s.stride_bytes > (1ll << 60) / rows) fail("a state's stride is too large");
          if (overlap(s.data, s.stride_bytes, s.row_bytes, parents, list, list, 1, rows))
            fail("a state overlaps parents");
          for (int j = 0; j < i; ++j)
            if (states[j].row_bytes > 0 && overlap(s.data, s.stride_bytes, s.row_bytes, states[j].data,
                                                   states[j].stride_bytes, states[j].row_bytes, rows, rows))
              fail("two states overlap");
        }
        for (const int width : {16, 4, 1}) {
          vb::BeamReorderArgs a{};
          a.beams = beams;
          a.parents = parents;
          a.ld_parents = ld_parents;
          for (int i = 0; i <= n; ++i) {
            if (i < n && states[i].row_bytes > 0) {
              const unsigned long long all = reinterpret_cast<uintptr_t>(states[i].data) |
                                             static_cast<unsigned long long>(states[i].row_bytes) |
                                             static_cast<unsigned long long>(states[i].stride_bytes);
              if ((all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1) == width)
                a.states[a.n++] = {states[i].data, states[i].row_bytes, states[i].stride_bytes};
            }
            if (a.n == vb::kBeamMaxStates || (i == n && a.n > 0)) {
              cuda_ok(vb::launch_beam_reorder(a, requests, width, static_cast<cudaStream_t>(stream)), "kernel launch");
              a.n = 0;
            }
          }
        }
        return 0;
      },
      -1);
}

}  // extern "C"
