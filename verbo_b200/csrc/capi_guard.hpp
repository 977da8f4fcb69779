// Error handling shared by the C ABI's translation units: the thread's last
// message and the guard that turns exceptions into a failure value.
#pragma once

#include <cuda_runtime.h>

#include <exception>
#include <stdexcept>
#include <string>

namespace vb {

inline thread_local std::string g_err;

template <typename F>
auto guard(F&& fn, decltype(fn()) fail) -> decltype(fn()) {
  try {
    g_err.clear();
    return fn();
  } catch (const std::exception& e) {
    g_err = e.what();
  } catch (...) {
    g_err = "verbo_cuda: unknown error";
  }
  return fail;
}

[[noreturn]] inline void fail(const std::string& m) { throw std::runtime_error("verbo_cuda: " + m); }

// The runtime keeps a failed call's error until somebody takes it: taken here, or the
// next launch of the thread, which looks for errors that way, would answer with it.
inline void cuda_ok(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return;
  (void)cudaGetLastError();
  fail(std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace vb
