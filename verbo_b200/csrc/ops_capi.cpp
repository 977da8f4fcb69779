// C ABI of the operators around the sampler (include/verbo_ops.h): argument
// checks and launches, no compute.
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "capi_guard.hpp"
#include "ops.cuh"
#include "verbo_ops.h"

struct verbo_ops_q4 {
  vb::Q4Mat m{};
  int device = 0;
  unsigned char* d_tiles = nullptr;
  float* d_bias = nullptr;
};

namespace {

using vb::cuda_ok;
using vb::fail;
using vb::guard;

// The calls on a handle run on its device and leave the caller's current.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    cuda_ok(cudaGetDevice(&before_), "cudaGetDevice");
    if (device != before_) {
      cuda_ok(cudaSetDevice(device), "cudaSetDevice");
      changed_ = true;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

// While a stream is being captured, CUDA refuses allocations and waits to the
// capturing thread (and to all threads, for some captures) and ends the capture.
// Those of a handle are no part of it: this thread's calls are let through.
class BesideCaptures {
 public:
  BesideCaptures() { changed_ = cudaThreadExchangeStreamCaptureMode(&mode_) == cudaSuccess; }
  ~BesideCaptures() {
    if (changed_) cudaThreadExchangeStreamCaptureMode(&mode_);
  }
  BesideCaptures(const BesideCaptures&) = delete;
  BesideCaptures& operator=(const BesideCaptures&) = delete;

 private:
  cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
  bool changed_ = false;
};

void check_type(int t, const char* what) {
  if (t != VERBO_OPS_F32 && t != VERBO_OPS_F16 && t != VERBO_OPS_BF16)
    fail(std::string(what) + " must be VERBO_OPS_F32, VERBO_OPS_F16 or VERBO_OPS_BF16");
}

void check_aligned(const void* p, int size, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) % static_cast<unsigned>(size))
    fail(std::string(what) + " must be aligned to its elements");
}

void check_rows(const void* p, int type, int rows, int cols, long long ld, const char* what) {
  if (!p) fail(std::string(what) + " must not be NULL");
  check_aligned(p, vb::ops_type_size(type), what);
  if (ld < cols) fail(std::string(what) + ": the row stride must be at least the row's length");
  if (ld > (1ll << 62) / (static_cast<long long>(rows) * 4)) fail(std::string(what) + ": the row stride is too large");
}

// Whether two sets of rows can touch the same byte.  Rows of one pitch that
// lie beside each other in it (two halves of one buffer) do not.
bool overlap(const void* a, long long pa, long long la, const void* b, long long pb, long long lb, int rows_b,
             int rows_a) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  const char *xe = x + (rows_a - 1) * pa + la, *ye = y + (rows_b - 1) * pb + lb;
  if (xe <= y || ye <= x) return false;
  if (pa != pb || rows_a != rows_b) return true;
  const long long d = ((y - x) % pa + pa) % pa;
  return !(d >= la && d + lb <= pa);
}

}  // namespace

extern "C" {

VERBO_CUDA_API verbo_ops_penalties verbo_ops_default_penalties(void) {
  verbo_ops_penalties p;
  p.repeat = 1.0f;
  p.frequency = 0.0f;
  p.presence = 0.0f;
  p.last = 0;
  return p;
}

VERBO_CUDA_API int verbo_ops_process_logits(const void* logits, int dtype, int rows, int vocab, long long ld,
                                            const verbo_ops_penalties* opts, const float* row_penalties,
                                            const int* hist, const long long* hist_off, const int* bias_ids,
                                            const float* bias, const long long* bias_off, const unsigned* mask,
                                            long long ld_mask, float* out, long long ld_out, void* stream) {
  return guard(
      [&]() {
        check_type(dtype, "dtype");
        if (rows < 0) fail("rows must be >= 0");
        if (vocab < 1 || vocab > VERBO_OPS_MAX_VOCAB)
          fail("vocab must be in [1, " + std::to_string(VERBO_OPS_MAX_VOCAB) + "]");
        if ((hist == nullptr) != (hist_off == nullptr)) fail("hist and hist_off must both be given or both be NULL");
        if ((bias_ids == nullptr) != (bias_off == nullptr) || (bias == nullptr) != (bias_off == nullptr))
          fail("bias_ids, bias and bias_off must all be given or all be NULL");
        if (row_penalties && !opts) fail("row_penalties need opts (for its window)");
        if (opts) {
          if (!std::isfinite(opts->repeat) || opts->repeat <= 0.0f) fail("repeat must be finite and > 0");
          if (!std::isfinite(opts->frequency)) fail("frequency must be finite");
          if (!std::isfinite(opts->presence)) fail("presence must be finite");
        }
        const long long words = (static_cast<long long>(vocab) + 31) / 32;
        if (mask && ld_mask != 0 && ld_mask < words) fail("ld_mask must be 0 or at least ceil(vocab / 32)");
        if (rows == 0) return 0;
        check_rows(logits, dtype, rows, vocab, ld, "logits");
        check_rows(out, VERBO_OPS_F32, rows, vocab, ld_out, "out");
        check_aligned(mask, 4, "mask");
        check_aligned(row_penalties, 4, "row_penalties");
        check_aligned(hist, 4, "hist");
        check_aligned(hist_off, 8, "hist_off");
        check_aligned(bias_ids, 4, "bias_ids");
        check_aligned(bias, 4, "bias");
        check_aligned(bias_off, 8, "bias_off");
        const bool in_place = static_cast<const void*>(out) == logits;
        if (in_place && (dtype != VERBO_OPS_F32 || (ld_out != ld && rows > 1)))
          fail("out may be logits only if they are F32 rows of the same stride");
        const long long size = vb::ops_type_size(dtype);
        if (!in_place && overlap(logits, ld * size, vocab * size, out, ld_out * 4, vocab * 4ll, rows, rows))
          fail("out overlaps logits without being the same rows");
        vb::ProcArgs a{};
        a.logits = logits;
        a.ld = ld;
        a.rows = rows;
        a.vocab = vocab;
        a.out = out;
        a.ld_out = ld_out;
        const bool pen = opts && hist &&
                         (row_penalties || opts->repeat != 1.0f || opts->frequency != 0.0f || opts->presence != 0.0f);
        if (pen) {
          a.repeat = opts->repeat;
          a.frequency = opts->frequency;
          a.presence = opts->presence;
          a.last = opts->last;
          a.row_pen = row_penalties;
          a.hist = hist;
          a.hist_off = hist_off;
        }
        a.bias_ids = bias_ids;
        a.bias = bias;
        a.bias_off = bias_off;
        a.mask = mask;
        a.ld_mask = ld_mask;
        if (in_place && !pen && !bias && !mask) return 0;
        cuda_ok(vb::launch_process(a, dtype, in_place, static_cast<cudaStream_t>(stream)), "kernel launch");
        return 0;
      },
      -1);
}

VERBO_CUDA_API int verbo_ops_token_logprobs(const void* logits, int dtype, int rows, int vocab, long long ld,
                                            float temp, const int* ids, float* logprob, int* rank, int top,
                                            int* top_ids, float* top_logprobs, void* stream) {
  return guard(
      [&]() {
        check_type(dtype, "dtype");
        if (rows < 0) fail("rows must be >= 0");
        if (vocab < 1 || vocab > VERBO_OPS_MAX_VOCAB)
          fail("vocab must be in [1, " + std::to_string(VERBO_OPS_MAX_VOCAB) + "]");
        if (!(temp >= 1e-4f && temp <= 1e4f)) fail("temp must be in [1e-4, 1e4]");
        if (top < 0 || top > vb::kLpMaxTop) fail("top must be in [0, " + std::to_string(vb::kLpMaxTop) + "]");
        if (rows == 0) return 0;
        check_rows(logits, dtype, rows, vocab, ld, "logits");
        if (ids && (!logprob || !rank)) fail("logprob and rank must not be NULL when ids are given");
        if (top > 0 && (!top_ids || !top_logprobs)) fail("top_ids and top_logprobs must not be NULL when top > 0");
        check_aligned(ids, 4, "ids");
        check_aligned(logprob, 4, "logprob");
        check_aligned(rank, 4, "rank");
        check_aligned(top_ids, 4, "top_ids");
        check_aligned(top_logprobs, 4, "top_logprobs");
        if (!ids && top == 0) return 0;
        vb::LogprobArgs a{};
        a.logits = logits;
        a.ld = ld;
        a.rows = rows;
        a.vocab = vocab;
        a.temp = temp;
        a.ids = ids;
        a.logprob = logprob;
        a.rank = rank;
        a.top = top;
        a.top_ids = top_ids;
        a.top_logprobs = top_logprobs;
        cuda_ok(vb::launch_logprobs(a, dtype, static_cast<cudaStream_t>(stream)), "kernel launch");
        return 0;
      },
      -1);
}

}  // extern "C"

namespace {

// A device view of a host or device array for the length of q4_new: device
// memory of the same device is read in place, the rest copied.
class Staged {
 public:
  Staged(const void* p, size_t bytes, int device, cudaStream_t s) : s_(s) {
    if (!p) return;
    cudaPointerAttributes pa{};
    cuda_ok(cudaPointerGetAttributes(&pa, p), "cudaPointerGetAttributes");
    if (pa.type == cudaMemoryTypeDevice && pa.device == device) {
      view_ = p;
      return;
    }
    cuda_ok(cudaMalloc(&own_, bytes), "cudaMalloc staging");
    view_ = own_;
    const cudaError_t e = cudaMemcpyAsync(own_, p, bytes, cudaMemcpyDefault, s);
    if (e != cudaSuccess) {
      cudaFree(own_);
      cuda_ok(e, "upload");
    }
  }
  ~Staged() {
    if (own_) {
      cudaStreamSynchronize(s_);
      cudaFree(own_);
    }
  }
  Staged(const Staged&) = delete;
  Staged& operator=(const Staged&) = delete;
  template <class T>
  const T* as() const {
    return static_cast<const T*>(view_);
  }

 private:
  cudaStream_t s_;
  void* own_ = nullptr;
  const void* view_ = nullptr;
};

// A language with garbage collection may free a handle during a capture.
void q4_release(verbo_ops_q4* h) {
  int before = 0;
  const bool known = cudaGetDevice(&before) == cudaSuccess;
  const BesideCaptures beside;
  cudaSetDevice(h->device);
  cudaFree(h->d_tiles);
  cudaFree(h->d_bias);
  if (known) cudaSetDevice(before);
  delete h;
}

}  // namespace

extern "C" {

VERBO_CUDA_API verbo_ops_q4* verbo_ops_q4_new(int outs, int ins, int group, const unsigned char* q,
                                              const unsigned short* s, const unsigned char* zeros, const float* bias,
                                              int device, void* stream) {
  return guard(
      [&]() -> verbo_ops_q4* {
        if (!q || !s) fail("q and s must not be NULL");
        if (outs < 1 || outs > vb::kQ4MaxOuts) fail("outs must be in [1, " + std::to_string(vb::kQ4MaxOuts) + "]");
        if (ins < 32 || ins > vb::kQ4MaxIns || ins % 32)
          fail("ins must be a multiple of 32 in [32, " + std::to_string(vb::kQ4MaxIns) + "]");
        if (group < 32 || group % 32) fail("group must be a multiple of 32, at least 32");
        check_aligned(s, 2, "s");
        check_aligned(bias, 4, "bias");
        int n = 0;
        cuda_ok(cudaGetDeviceCount(&n), "cudaGetDeviceCount");
        if (device < 0 || device >= n) fail("no CUDA device " + std::to_string(device));
        const DeviceScope scope(device);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        const cudaError_t e = cudaStreamIsCapturing(st, &capture);
        if (e != cudaErrorStreamCaptureImplicit) cuda_ok(e, "stream");
        if (e != cudaSuccess || capture != cudaStreamCaptureStatusNone) {
          (void)cudaGetLastError();
          fail("a layer cannot be made on a stream that is being captured");
        }
        const BesideCaptures beside;
        auto* h = new verbo_ops_q4();
        h->device = device;
        try {
          h->m.outs = outs;
          h->m.ins = ins;
          h->m.group = group;
          h->m.zeros = zeros != nullptr;
          vb::q4_layout(h->m);
          const size_t cells = static_cast<size_t>(outs) * vb::q4_groups(h->m);
          cuda_ok(cudaMalloc(&h->d_tiles, vb::q4_tiles_bytes(h->m)), "cudaMalloc weights");
          {
            const Staged dq(q, static_cast<size_t>(outs) * (ins / 2), device, st);
            const Staged ds(s, cells * 2, device, st);
            const Staged dz(zeros, cells, device, st);
            cuda_ok(vb::launch_q4_pack(h->m, dq.as<unsigned char>(), ds.as<uint16_t>(), dz.as<unsigned char>(),
                                       h->d_tiles, st),
                    "kernel launch");
            if (bias) {
              cuda_ok(cudaMalloc(&h->d_bias, outs * sizeof(float)), "cudaMalloc bias");
              cuda_ok(cudaMemcpyAsync(h->d_bias, bias, outs * sizeof(float), cudaMemcpyDefault, st), "upload bias");
            }
            cuda_ok(cudaStreamSynchronize(st), "stream");
          }
          h->m.tiles = h->d_tiles;
          h->m.bias = h->d_bias;
        } catch (...) {
          q4_release(h);
          throw;
        }
        return h;
      },
      nullptr);
}

VERBO_CUDA_API void verbo_ops_q4_free(verbo_ops_q4* h) {
  if (h) q4_release(h);
}

VERBO_CUDA_API long long verbo_ops_q4_workspace(const verbo_ops_q4* h, int x_type, int n) {
  return guard(
      [&]() -> long long {
        if (!h) fail("q4 handle is NULL");
        check_type(x_type, "x_type");
        if (n < 0 || n > VERBO_OPS_MAX_ROWS) fail("n must be in [0, " + std::to_string(VERBO_OPS_MAX_ROWS) + "]");
        const DeviceScope scope(h->device);
        return n == 0 ? 0 : static_cast<long long>(vb::q4_workspace_bytes(h->m, n, x_type));
      },
      -1);
}

VERBO_CUDA_API int verbo_ops_q4_matvec(const verbo_ops_q4* h, const void* x, int x_type, int n, long long ldx, void* y,
                                       int y_type, long long ldy, void* workspace, long long workspace_bytes,
                                       void* stream) {
  return guard(
      [&]() {
        if (!h) fail("q4 handle is NULL");
        check_type(x_type, "x_type");
        check_type(y_type, "y_type");
        if (n < 0 || n > VERBO_OPS_MAX_ROWS) fail("n must be in [0, " + std::to_string(VERBO_OPS_MAX_ROWS) + "]");
        if (n == 0) return 0;
        check_rows(x, x_type, n, h->m.ins, ldx, "x");
        check_rows(y, y_type, n, h->m.outs, ldy, "y");
        const DeviceScope scope(h->device);
        const long long sx = vb::ops_type_size(x_type), sy = vb::ops_type_size(y_type);
        if (overlap(x, ldx * sx, h->m.ins * sx, y, ldy * sy, h->m.outs * sy, n, n)) fail("y overlaps x");
        const long long need = static_cast<long long>(vb::q4_workspace_bytes(h->m, n, x_type));
        if (need) {
          if (!workspace || workspace_bytes < need)
            fail("the workspace must have " + std::to_string(need) + " bytes (verbo_ops_q4_workspace)");
          check_aligned(workspace, 16, "workspace");
          if (overlap(x, ldx * sx, h->m.ins * sx, workspace, need, need, 1, n) ||
              overlap(y, ldy * sy, h->m.outs * sy, workspace, need, need, 1, n))
            fail("workspace overlaps x or y");
        }
        vb::Q4Args a{};
        a.x = x;
        a.ldx = ldx;
        a.n = n;
        a.y = y;
        a.ldy = ldy;
        a.workspace = workspace;
        cuda_ok(vb::launch_q4(h->m, a, x_type, y_type, static_cast<cudaStream_t>(stream)), "kernel launch");
        return 0;
      },
      -1);
}

}  // extern "C"
