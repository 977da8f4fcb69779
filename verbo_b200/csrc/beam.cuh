// Launch-side view of beam search's operators (include/verbo_beam.h), shared by
// beam.cu and beam_capi.cpp.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace vb {

constexpr int kBeamMaxBeams = 32;
constexpr int kBeamMaxTake = 64;
constexpr int kBeamMaxStates = 32;  // of one launch

struct BeamSelectArgs {
  const void* logits;
  long long ld;
  int requests, beams, vocab, take;
  const float* scores;
  float* out_scores;
  int* parents;
  int* tokens;
  void* workspace;  // beam_workspace_bytes, 16-byte aligned
};
size_t beam_workspace_bytes(int rows, int take);
cudaError_t launch_beam_select(const BeamSelectArgs& a, int dtype, cudaStream_t s);

struct BeamState {
  void* data;
  long long row_bytes, stride_bytes;
};
struct BeamReorderArgs {
  BeamState states[kBeamMaxStates];
  unsigned first[kBeamMaxStates + 1];  // CTAs before each state's
  unsigned chunks[kBeamMaxStates];     // CTAs of a request
  int n, beams;
  const int* parents;
  long long ld_parents;
};
// States of one copying width: fills in first and chunks.
cudaError_t launch_beam_reorder(BeamReorderArgs a, int requests, int width, cudaStream_t s);

}  // namespace vb
