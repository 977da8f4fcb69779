// Checks of arguments that the C ABI's operators share.
#pragma once

#include <string>

#include "capi_guard.hpp"
#include "ops.cuh"
#include "verbo_ops.h"

namespace vb {

inline void check_type(int t, const char* what) {
  if (t != VERBO_OPS_F32 && t != VERBO_OPS_F16 && t != VERBO_OPS_BF16)
    fail(std::string(what) + " must be VERBO_OPS_F32, VERBO_OPS_F16 or VERBO_OPS_BF16");
}

inline void check_aligned(const void* p, int size, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) % static_cast<unsigned>(size))
    fail(std::string(what) + " must be aligned to its elements");
}

inline void check_rows(const void* p, int type, int rows, int cols, long long ld, const char* what) {
  if (!p) fail(std::string(what) + " must not be NULL");
  check_aligned(p, ops_type_size(type), what);
  if (ld < cols) fail(std::string(what) + ": the row stride must be at least the row's length");
  if (ld > (1ll << 62) / (static_cast<long long>(rows) * 4)) fail(std::string(what) + ": the row stride is too large");
}

// Whether two sets of rows can touch the same byte.  Rows of one pitch that
// lie beside each other in it (two halves of one buffer) do not.
inline bool overlap(const void* a, long long pa, long long la, const void* b, long long pb, long long lb, int rows_b,
                    int rows_a) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  const char *xe = x + (rows_a - 1) * pa + la, *ye = y + (rows_b - 1) * pb + lb;
  if (xe <= y || ye <= x) return false;
  if (pa != pb || rows_a != rows_b) return true;
  const long long d = ((y - x) % pa + pa) % pa;
  return !(d >= la && d + lb <= pa);
}

}  // namespace vb
