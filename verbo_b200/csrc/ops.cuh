// Launch-side view of the operators around the sampler (include/verbo_ops.h),
// shared by ops_logits.cu, ops_q4.cu and ops_capi.cpp.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace vb {

enum OpsType { kOpsF32 = 0, kOpsF16 = 1, kOpsBF16 = 2 };
inline int ops_type_size(int t) { return t == kOpsF32 ? 4 : 2; }

// SMs of the current device (the handle's, in the calls on one).
inline int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;  // a B200's; the launch that follows says what is wrong
  return sms;
}

// ------------------------------------------------------------ process -----
struct ProcArgs {
  const void* logits;
  long long ld;
  int rows, vocab;
  int parts;      // CTAs per row
  int part_cols;  // columns of a part
  float repeat, frequency, presence;
  int last;
  const float* row_pen;       // [rows][3] or null
  const int* hist;            // CSR or null
  const long long* hist_off;
  const int* bias_ids;        // CSR or null
  const float* bias;
  const long long* bias_off;
  const uint32_t* mask;       // or null
  long long ld_mask;
  float* out;
  long long ld_out;
};
// dtype: OpsType of the logits; in_place: out is the logits.
cudaError_t launch_process(ProcArgs a, int dtype, bool in_place, cudaStream_t s);

// ----------------------------------------------------------- logprobs -----
constexpr int kLpMaxTop = 32;
struct LogprobArgs {
  const void* logits;
  long long ld;
  int rows, vocab;
  float temp;
  const int* ids;  // or null
  float* logprob;
  int* rank;
  int top;
  int* top_ids;
  float* top_logprobs;
};
cudaError_t launch_logprobs(LogprobArgs a, int dtype, cudaStream_t s);

// ----------------------------------------------------------------- q4 -----
// Device layout of a matrix: tiles of kQ4Rows output rows; a tile is nkc
// chunks of kQ4Chunk weights of each of its rows, one after the other:
//   1024 B  nibbles in the order in which the lanes of a warp feed them to
//           mma.m16n8k16 (ops_q4.cu): two blocks of 32 lanes x 16 B
//   then    the chunk's fp16 scales, [8 row pairs][sets][row g, row g + 8]
//   then    its zero points (one byte each, the same order), if there are any,
//           filled up to a multiple of 32 bytes
// A set is `span` weights of one row that share a scale: gcd(group, 128).
// Rows past outs and weights past ins have scale 0.
constexpr int kQ4Rows = 16;
constexpr int kQ4Chunk = 128;
constexpr int kQ4MaxIns = 32768;
constexpr int kQ4MaxOuts = 1 << 22;
struct Q4Mat {
  int outs, ins, group;
  int span;         // 32, 64 or 128
  int nkc;          // chunks per tile
  int ntile;
  int chunk_bytes;
  bool zeros;
  const unsigned char* tiles;
  const float* bias;  // or null
};
// Scales of a row, without the sum ins + group: group is anything up to 2^31.
__host__ __device__ inline int q4_groups(const Q4Mat& m) { return (m.ins - 1) / m.group + 1; }
struct Q4Args {
  const void* x;
  long long ldx;
  int n;
  void* y;
  long long ldy;
  void* workspace;  // q4_workspace_bytes, 16-byte aligned
};
// Fills in span, nkc, ntile, chunk_bytes from outs, ins, group, zeros.
void q4_layout(Q4Mat& m);
size_t q4_tiles_bytes(const Q4Mat& m);
size_t q4_workspace_bytes(const Q4Mat& m, int n, int x_type);
// Lays device arrays out into `tiles` (m.zeros: whether zeros is given).
cudaError_t launch_q4_pack(const Q4Mat& m, const unsigned char* q, const uint16_t* s, const unsigned char* zeros,
                           unsigned char* tiles, cudaStream_t st);
cudaError_t launch_q4(const Q4Mat& m, const Q4Args& a, int x_type, int y_type, cudaStream_t st);

// Device-side failures of the operators (bounded waits that ran out).
constexpr unsigned kErrOpsWait = 1u;
cudaError_t ops_read_status(unsigned* st, bool clear);

}  // namespace vb
