// C ABI of the paged cache (include/verbo_cache.h): argument checks and launches.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <string>

#include "cache.cuh"
#include "capi_checks.hpp"
#include "capi_guard.hpp"
#include "ops.cuh"

namespace {

using vb::check_aligned;
using vb::check_type;
using vb::cuda_ok;
using vb::fail;
using vb::guard;

// An array of the caller's as a range of bytes.
struct Range {
  const void* p;
  long long bytes;
  const char* what;
};
bool touch(const Range& a, const Range& b) {
  const char *x = static_cast<const char*>(a.p), *y = static_cast<const char*>(b.p);
  return a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}
void check_apart(const Range& a, const Range& b) {
  if (touch(a, b)) fail(std::string(a.what) + " overlaps " + b.what);
}

void check_number(int v, int low, int high, const char* what) {
  if (v < low || v > high)
    fail(std::string(what) + " must be in [" + std::to_string(low) + ", " + std::to_string(high) + "]");
}

void check_sizes(const verbo_cache* c) {
  if (!c) fail("cache must not be NULL");
  check_number(c->layers, 1, 65536, "layers");
  check_number(c->pages, 1, VERBO_CACHE_MAX_PAGES, "pages");
  check_number(c->heads, 1, VERBO_CACHE_MAX_HEADS, "heads");
  check_number(c->dim, 16, VERBO_CACHE_MAX_DIM, "dim");
  if (c->dim % 16) fail("dim must be a multiple of 16");
  check_number(c->page, VERBO_CACHE_BLOCK, VERBO_CACHE_MAX_PAGE, "page");
  if (c->page % VERBO_CACHE_BLOCK) fail("page must be a multiple of 16");
  check_number(c->rows, 0, VERBO_CACHE_MAX_ROWS, "rows");
  check_number(c->width, 1, (1 << 30) / c->page, "width");
  // blocks are counted in 32 bits: those of a layer, and those of all tables
  const long long per = c->page / VERBO_CACHE_BLOCK;
  if (static_cast<long long>(c->pages) * c->heads * per > INT_MAX)
    fail("pages * heads * page / 16 must be below 2^31");
  if (static_cast<long long>(c->rows) * (c->width * per + 16) > INT_MAX) fail("rows * width * page / 16 must be below 2^31");
}

struct CacheRanges {
  Range r[7];
};
CacheRanges ranges(const verbo_cache* c) {
  const long long cells = static_cast<long long>(c->layers) * c->pages * c->heads * c->page;
  return {{{c->k, cells * c->dim, "k"},
           {c->v, cells * c->dim, "v"},
           {c->k_scale, cells / VERBO_CACHE_BLOCK * 4, "k_scale"},
           {c->v_scale, cells / VERBO_CACHE_BLOCK * 4, "v_scale"},
           {c->table, static_cast<long long>(c->rows) * c->width * 4, "table"},
           {c->lens, c->rows * 4ll, "lens"},
           {c->refs, c->pages * 4ll, "refs"}}};
}
CacheRanges check_cache(const verbo_cache* c) {
  check_sizes(c);
  const CacheRanges all = ranges(c);
  for (int i = 0; i < 7; ++i) {
    if (!all.r[i].p && all.r[i].bytes > 0) fail(std::string(all.r[i].what) + " must not be NULL");
    check_aligned(all.r[i].p, i < 2 ? 16 : 4, all.r[i].what);
    for (int j = 0; j < i; ++j) check_apart(all.r[i], all.r[j]);
  }
  return all;
}

// An output: apart from the cache and from what `more` lists.
void check_output(const Range& out, const CacheRanges& c) {
  if (!out.p) fail(std::string(out.what) + " must not be NULL");
  for (const Range& r : c.r) check_apart(out, r);
}

Range check_workspace(void* ws, long long have, size_t need, const char* fn) {
  if (!ws || have < 0 || static_cast<unsigned long long>(have) < need)
    fail("the workspace must have " + std::to_string(need) + " bytes (" + fn + ")");
  check_aligned(ws, 16, "workspace");
  return {ws, static_cast<long long>(need), "the workspace"};
}

// Tokens of `heads` heads with their strides, as a range of bytes from their first
// element on.
Range check_tokens(const void* p, int type, long long tokens, long long ld, int heads, long long hd, int dim,
                   const char* what) {
  if (!p) fail(std::string(what) + " must not be NULL");
  const long long size = vb::ops_type_size(type);
  check_aligned(p, static_cast<int>(size), what);
  if (hd < dim && heads > 1) fail(std::string(what) + ": the head stride must be at least dim");
  if (ld < dim && tokens > 1) fail(std::string(what) + ": the token stride must be at least dim");
  if (hd < 0 || ld < 0 || hd > (1ll << 58) / heads || ld > (1ll << 58) / tokens)
    fail(std::string(what) + ": a stride is negative or too large");
  return {p, ((tokens - 1) * ld + (heads - 1) * hd + dim) * size, what};
}

}  // namespace

extern "C" {

VERBO_CUDA_API long long verbo_cache_workspace(const verbo_cache* c) {
  return guard(
      [&]() -> long long {
        check_sizes(c);
        return static_cast<long long>(vb::cache_workspace_bytes(*c));
      },
      -1);
}

VERBO_CUDA_API int verbo_cache_reserve(const verbo_cache* c, const int* add, int* start, int* status, void* workspace,
                                       long long workspace_bytes, void* stream) {
  return guard(
      [&]() {
        const CacheRanges all = check_cache(c);
        const Range list{add, c->rows * 4ll, "add"}, st{start, c->rows * 4ll, "start"}, so{status, 4, "status"};
        check_output(so, all);
        check_aligned(status, 4, "status");
        if (c->rows > 0) {
          if (!add) fail("add must not be NULL");
          check_aligned(add, 4, "add");
          check_output(st, all);
          check_aligned(start, 4, "start");
          check_apart(st, list);
          check_apart(so, list);
          check_apart(so, st);
        }
        const Range ws =
            check_workspace(workspace, workspace_bytes, vb::cache_workspace_bytes(*c), "verbo_cache_workspace");
        check_output(ws, all);
        for (const Range& r : {list, st, so}) check_apart(ws, r);
        cuda_ok(vb::launch_cache_reserve(*c, add, start, status, workspace, static_cast<cudaStream_t>(stream)),
                "kernel launch");
        return 0;
      },
      -1);
}

VERBO_CUDA_API int verbo_cache_fork(const verbo_cache* c, const int* parents, long long ld_parents, int beams,
                                    void* stream) {
  return guard(
      [&]() {
        const CacheRanges all = check_cache(c);
        check_number(beams, 1, 32, "beams");
        if (c->rows % beams) fail("rows must be a multiple of beams");
        if (c->rows == 0) return 0;
        const int groups = c->rows / beams;
        if (!parents) fail("parents must not be NULL");
        check_aligned(parents, 4, "parents");
        if (ld_parents < beams && groups > 1) fail("ld_parents must be at least beams");
        if (ld_parents > (1ll << 58) / groups) fail("ld_parents is too large");
        const Range list{parents, 4 * ((groups - 1) * ld_parents + beams), "parents"};
        for (const Range& r : all.r) check_apart(list, r);
        cuda_ok(vb::launch_cache_fork(*c, parents, ld_parents, beams, static_cast<cudaStream_t>(stream)),
                "kernel launch");
        return 0;
      },
      -1);
}

VERBO_CUDA_API int verbo_cache_free(const verbo_cache* c, const int* keep, void* stream) {
  return guard(
      [&]() {
        const CacheRanges all = check_cache(c);
        if (c->rows == 0) return 0;
        if (!keep) fail("keep must not be NULL");
        check_aligned(keep, 4, "keep");
        for (const Range& r : all.r) check_apart({keep, c->rows * 4ll, "keep"}, r);
        cuda_ok(vb::launch_cache_free(*c, keep, static_cast<cudaStream_t>(stream)), "kernel launch");
        return 0;
      },
      -1);
}

VERBO_CUDA_API int verbo_cache_compact(const verbo_cache* c, int* info, void* workspace, long long workspace_bytes,
                                       void* stream) {
  return guard(
      [&]() {
        const CacheRanges all = check_cache(c);
        const Range out{info, 8, "info"};
        check_output(out, all);
        check_aligned(info, 4, "info");
        const Range ws =
            check_workspace(workspace, workspace_bytes, vb::cache_workspace_bytes(*c), "verbo_cache_workspace");
        check_output(ws, all);
        check_apart(ws, out);
        cuda_ok(vb::launch_cache_compact(*c, info, workspace, static_cast<cudaStream_t>(stream)), "kernel launch");
        return 0;
      },
      -1);
}

VERBO_CUDA_API int verbo_cache_append(const verbo_cache* c, int layer, const void* k, long long ld_k, long long hd_k,
                                      const void* v, long long ld_v, long long hd_v, int dtype, int tokens,
                                      const int* start, const long long* off, void* stream) {
  return guard(
      [&]() {
        const CacheRanges all = check_cache(c);
        check_type(dtype, "dtype");
        check_number(layer, 0, c->layers - 1, "layer");
        check_number(tokens, 0, INT_MAX, "tokens");
        if (!off && (c->rows == 0 ? tokens != 0 : tokens % c->rows != 0))
          fail("tokens must be a multiple of rows without off");
        if (tokens == 0 || c->rows == 0) return 0;
        if (!start) fail("start must not be NULL");
        check_aligned(start, 4, "start");
        check_aligned(off, 8, "off");
        const Range in[] = {check_tokens(k, dtype, tokens, ld_k, c->heads, hd_k, c->dim, "new k"),
                            check_tokens(v, dtype, tokens, ld_v, c->heads, hd_v, c->dim, "new v"),
                            {start, c->rows * 4ll, "start"},
                            {off, off ? (c->rows + 1) * 8ll : 0, "off"}};
        for (const Range& a : in)
          for (const Range& r : all.r) check_apart(a, r);
        const vb::CacheNew x{k, v, ld_k, hd_k, ld_v, hd_v, tokens, start, off};
        cuda_ok(vb::launch_cache_append(*c, layer, x, dtype, static_cast<cudaStream_t>(stream)), "kernel launch");
        return 0;
      },
      -1);
}

namespace {
void check_attend(const verbo_cache* c, int heads, int steps) {
  check_number(steps, 1, VERBO_CACHE_MAX_STEPS, "steps");
  if (heads < 1 || heads % c->heads || heads / c->heads > 64)
    fail("heads must be a multiple of the cache's, at most 64 times it");
}
}  // namespace

VERBO_CUDA_API long long verbo_cache_attend_workspace(const verbo_cache* c, int heads, int steps, int q_type) {
  return guard(
      [&]() -> long long {
        check_sizes(c);
        check_attend(c, heads, steps);
        check_type(q_type, "q_type");
        return static_cast<long long>(vb::cache_attend_bytes(*c, heads, steps, q_type));
      },
      -1);
}

VERBO_CUDA_API int verbo_cache_attend(const verbo_cache* c, int layer, const void* q, int q_type, long long ld_q,
                                      long long hd_q, int heads, int steps, float scale, void* out, int out_type,
                                      long long ld_out, long long hd_out, void* workspace, long long workspace_bytes,
                                      void* stream) {
  return guard(
      [&]() {
        const CacheRanges all = check_cache(c);
        check_type(q_type, "q_type");
        check_type(out_type, "out_type");
        check_number(layer, 0, c->layers - 1, "layer");
        check_attend(c, heads, steps);
        if (!std::isfinite(scale)) fail("scale must be finite");
        if (c->rows == 0) return 0;
        const long long tokens = static_cast<long long>(c->rows) * steps;
        const Range rq = check_tokens(q, q_type, tokens, ld_q, heads, hd_q, c->dim, "q");
        const Range ro = check_tokens(out, out_type, tokens, ld_out, heads, hd_out, c->dim, "out");
        check_output(ro, all);
        check_apart(ro, rq);
        // rows of one output that lie in one another would be written twice
        const bool by_token = (heads - 1) * hd_out + c->dim <= ld_out || tokens == 1;
        const bool by_head = (tokens - 1) * ld_out + c->dim <= hd_out || heads == 1;
        if (!by_token && !by_head) fail("out: its tokens and heads overlap");
        if (const size_t need = vb::cache_attend_bytes(*c, heads, steps, q_type)) {
          const Range ws = check_workspace(workspace, workspace_bytes, need, "verbo_cache_attend_workspace");
          check_output(ws, all);
          check_apart(ws, rq);
          check_apart(ws, ro);
        }
        const vb::CacheQuery x{q, ld_q, hd_q, out, ld_out, hd_out, heads, steps, scale, workspace};
        cuda_ok(vb::launch_cache_attend(*c, layer, x, q_type, out_type, static_cast<cudaStream_t>(stream)),
                "kernel launch");
        return 0;
      },
      -1);
}

}  // extern "C"
