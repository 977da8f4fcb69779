// The paged cache's bookkeeping and its writes (include/verbo_cache.h): pages are
// reserved, forked, given back, compacted and copied; new keys and values are
// quantised into them.  Everything is decided on the device, by fixed rules, and
// counts are integers: the same calls leave the same pages.
#include <algorithm>
#include <climits>

#include "cache.cuh"
#include "device.cuh"
#include "ops.cuh"
#include "opsdev.cuh"

namespace vb {
namespace {

// ------------------------------------------------------------ workspace ---
constexpr int kChunk = 2048;  // pages that a CTA looks through
constexpr int kScanThreads = 256;
constexpr int kMaxChunks = VERBO_CACHE_MAX_PAGES / kChunk;

struct PageWs {
  int* head;   // [0] pages to copy, [1] live pages
  int* count;  // [chunks] free pages of each chunk
  int* list;   // [chunks][kChunk] them, ascending
  int* src;    // pages to copy
  int* dst;
  int* map;    // [pages] where a page goes
};
__host__ __device__ inline int chunks_of(const verbo_cache& c) { return (c.pages + kChunk - 1) / kChunk; }
inline size_t most_copies(const verbo_cache& c) {
  return std::max(static_cast<size_t>(c.rows), static_cast<size_t>(c.pages) / 2 + 1);
}
PageWs layout(const verbo_cache& c, void* ws) {
  PageWs w;
  int* p = static_cast<int*>(ws);
  w.head = p;
  w.count = p + 4;
  w.list = w.count + chunks_of(c);
  w.src = w.list + static_cast<size_t>(chunks_of(c)) * kChunk;
  w.dst = w.src + most_copies(c);
  w.map = w.dst + most_copies(c);
  return w;
}

__device__ __forceinline__ int length_of(const verbo_cache& c, int row) {
  return max(0, min(c.lens[row], c.width * c.page));
}
__device__ __forceinline__ int pages_for(int tokens, int page) { return tokens / page + (tokens % page > 0); }
__device__ __forceinline__ bool is_page(const verbo_cache& c, int id) { return id >= 0 && id < c.pages; }

// ----------------------------------------------------------- free pages ---
struct ScanArgs {
  verbo_cache c;
  PageWs w;
};
// A chunk's free pages, counted and listed in ascending order.
__global__ void __launch_bounds__(kScanThreads) cache_scan_kernel(const ScanArgs a) {
  constexpr int PER = kChunk / kScanThreads;
  __shared__ int ws[kScanThreads / 32];
  grid_wait();
  grid_release();
  const int first = blockIdx.x * kChunk + threadIdx.x * PER;
  int free_[PER], n = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    free_[i] = first + i < a.c.pages && a.c.refs[first + i] == 0;
    n += free_[i];
  }
  int total;
  int at = block_excl_scan<int, kScanThreads>(n, ws, &total);
  int* list = a.w.list + static_cast<size_t>(blockIdx.x) * kChunk;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (free_[i]) list[at++] = first + i;
  if (threadIdx.x == 0) a.w.count[blockIdx.x] = total;
}

// Free pages before each chunk into `pre` (shared, chunks + 1), by a whole CTA.
template <int NT>
__device__ __forceinline__ int scan_counts(const PageWs& w, int chunks, int* pre, int* ws) {
  constexpr int PER = (kMaxChunks + NT - 1) / NT;
  int v[PER], n = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = threadIdx.x * PER + i;
    v[i] = k < chunks ? w.count[k] : 0;
    n += v[i];
  }
  int total;
  int at = block_excl_scan<int, NT>(n, ws, &total);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = threadIdx.x * PER + i;
    if (k <= chunks) pre[k] = at;
    at += v[i];
  }
  if (threadIdx.x == 0) pre[chunks] = total;
  __syncthreads();
  return total;
}
// The i-th free page (i below the total).
__device__ __forceinline__ int free_page(const PageWs& w, int chunks, const int* pre, int i) {
  int lo = 0, hi = chunks - 1;
  while (lo < hi) {  // the last chunk that begins at or before i
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= i)
      lo = mid;
    else
      hi = mid - 1;
  }
  return w.list[static_cast<size_t>(lo) * kChunk + (i - pre[lo])];
}

// Pools of up to 16384 pages: the CTA that needs the list makes it, 16 pages to a
// thread: as long on the device as another kernel (5000 pages, 28 us for a fork and a
// reserve either way), and 3 us less of the calling thread's time.  `mask`: this thread's free
// pages, `before`: those before them.  Returns their number.
constexpr int kSmallPool = 16384;
constexpr int kSmallThreads = 1024;
constexpr int kSmallPer = kSmallPool / kSmallThreads;
__device__ __forceinline__ int scan_pool(const verbo_cache& c, const PageWs& w, int* ws, unsigned* mask, int* before) {
  const int first = threadIdx.x * kSmallPer;
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < kSmallPer; ++i)
    if (first + i < c.pages) m |= static_cast<unsigned>(c.refs[first + i] == 0) << i;
  int total;
  int at = block_excl_scan<int, kSmallThreads>(__popc(m), ws, &total);
  *mask = m;
  *before = at;
#pragma unroll
  for (int i = 0; i < kSmallPer; ++i)
    if (m >> i & 1u) w.list[at++] = first + i;
  __syncthreads();
  return total;
}

// --------------------------------------------------------------- reserve --
struct ReserveArgs {
  verbo_cache c;
  PageWs w;
  const int* add;
  int* start;
  int* status;
};
constexpr int kReserveThreads = 1024;

// One CTA for all rows, a thread to a row.  What a row needs is known when the
// rows before it are counted that write into the same page: with r references and
// i such rows, the row copies the page if r - i > 1.  Then pages are dealt out
// through the scan of the needs, one thread to a page.  Latency alone counts: the
// chain is lengths, tables, references, and the list of free pages.
template <bool SMALL>
__global__ void __launch_bounds__(kReserveThreads) cache_reserve_kernel(const ReserveArgs a) {
  constexpr int NT = kReserveThreads;
  static_assert(NT == kSmallThreads, "one thread layout");
  extern __shared__ __align__(16) int smem[];  // last, len, more, first, copied [rows + 3 each], then pre [chunks + 1]
  __shared__ int ws[NT / 32];
  __shared__ long long wide_ws[NT / 32];
  __shared__ int narrow;
  const verbo_cache& c = a.c;
  const int rows = c.rows, page = c.page, tid = threadIdx.x, chunks = chunks_of(c);
  const int most = c.width * page, pitch = (rows + 3) / 4 * 4;
  int* last = smem;            // the shared page that a row writes into, -1: none
  int* len = last + pitch;
  int* more = len + pitch;
  int* first = more + pitch;   // needs before the row
  int* copied = first + pitch; // 1 + its place among the copies, 0: none
  int* pre = copied + pitch;
  if (tid == 0) narrow = INT_MAX;
  __syncthreads();
  grid_wait();
  grid_release();

  for (int r = tid; r < pitch; r += NT) {
    int p = -1, n = 0, m = 0, shared = 0;
    if (r < rows) {
      n = length_of(c, r);
      m = max(0, a.add[r]);
      if (m > most - n) {
        atomicMin(&narrow, r);
        m = 0;
      }
      if (m > 0 && n % page > 0) {
        p = c.table[static_cast<long long>(r) * c.width + n / page];
        if (!is_page(c, p)) p = -1;
      }
      if (p >= 0) shared = c.refs[p];
      if (shared < 2) p = -1;
    }
    last[r] = p;
    len[r] = n;
    more[r] = m;
    copied[r] = shared;
  }
  unsigned mask;
  int before_mine;
  const int total_free = SMALL ? scan_pool(c, a.w, ws, &mask, &before_mine) : scan_counts<NT>(a.w, chunks, pre, ws);
  // a row needs up to 2^26 pages: sums in 64 bits, the copies' in the upper half
  long long sum = 0;
  for (int r0 = 0; r0 < rows; r0 += NT) {
    const int r = r0 + tid;
    long long need = 0;
    if (r < rows) {
      const int p = last[r];
      bool copy = false;
      if (p >= 0) {
        int before = 0;
        const int4* q = reinterpret_cast<const int4*>(last);
        for (int j = 0; j < r / 4; ++j) {
          const int4 v = q[j];
          before += (v.x == p) + (v.y == p) + (v.z == p) + (v.w == p);
        }
        for (int j = r / 4 * 4; j < r; ++j) before += last[j] == p;
        copy = copied[r] - before > 1;
      }
      const int n = len[r], m = more[r];
      need = copy + (m > 0 ? pages_for(n + m, page) - pages_for(n, page) : 0) + (static_cast<long long>(copy) << 40);
    }
    long long total;
    const long long at = sum + block_excl_scan<long long, NT>(need, wide_ws, &total);
    if (r < rows) {
      first[r] = static_cast<int>(min(at & ((1ll << 40) - 1), static_cast<long long>(INT_MAX)));
      copied[r] = need >> 40 ? static_cast<int>(at >> 40) + 1 : 0;
    }
    sum += total;
    __syncthreads();
  }
  const int total = static_cast<int>(min(sum & ((1ll << 40) - 1), static_cast<long long>(INT_MAX)));
  const int status = narrow != INT_MAX ? -(narrow + 1) : total > total_free ? total - total_free : 0;
  if (tid == 0) {
    *a.status = status;
    a.w.head[0] = status ? 0 : static_cast<int>(sum >> 40);
  }
  for (int r = tid; r < rows; r += NT) {
    const int m = status ? 0 : more[r];
    a.start[r] = m > 0 ? len[r] : -1;
    if (m > 0) c.lens[r] = len[r] + m;
  }
  if (status) return;
  for (int i = tid; i < total; i += NT) {
    int lo = 0, hi = rows - 1;
    while (lo < hi) {  // the last row whose pages begin at or before i
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= i)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int to = SMALL ? a.w.list[i] : free_page(a.w, chunks, pre, i);
    const int k = i - first[lo] - (copied[lo] > 0);
    int at = pages_for(len[lo], page) + k;
    if (k < 0) {  // a copy of the row's last page
      at = len[lo] / page;
      a.w.src[copied[lo] - 1] = last[lo];
      a.w.dst[copied[lo] - 1] = to;
      atomicSub(&c.refs[last[lo]], 1);
    }
    c.refs[to] = 1;
    c.table[static_cast<long long>(lo) * c.width + at] = to;
  }
}

// ------------------------------------------------------------------ copy --
struct CopyArgs {
  verbo_cache c;
  PageWs w;
  bool remap;  // compaction: tables and counts follow
};
constexpr int kCopyThreads = 256;
constexpr int kCopyPiece = kCopyThreads * 16 * 4;  // bytes of a CTA's step

// Pages src[i] -> dst[i] in all layers.  No page is both, so the order is free.
// Memory bound: each byte is read and written once, 64 bytes in flight per thread.
__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const CopyArgs a) {
  const verbo_cache& c = a.c;
  grid_wait();
  grid_release();
  const int tid = threadIdx.x;
  const long long n = a.w.head[0];
  if (a.remap) {
    const int live = a.w.head[1];
    const long long step = static_cast<long long>(gridDim.x) * kCopyThreads;
    for (long long i = static_cast<long long>(blockIdx.x) * kCopyThreads + tid; i < n; i += step) {
      const int s = a.w.src[i], d = a.w.dst[i];
      c.refs[d] = c.refs[s];
      c.refs[s] = 0;
    }
    if (n > 0)
      for (int r = blockIdx.x; r < c.rows; r += gridDim.x) {
        int* t = c.table + static_cast<long long>(r) * c.width;
        const int used = pages_for(length_of(c, r), c.page);
        for (int j = tid; j < used; j += kCopyThreads) {
          const int p = t[j];
          if (p >= live && p < c.pages) t[j] = a.w.map[p];
        }
      }
  }
  const long long bytes = static_cast<long long>(c.heads) * c.page * c.dim;
  const int pieces = static_cast<int>((bytes + kCopyPiece - 1) / kCopyPiece);
  const int scales = c.heads * (c.page / kCacheBlock);
  const long long units = n * c.layers * 2 * pieces;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int piece = static_cast<int>(u % pieces);
    const long long e = u / pieces;
    const bool value = e & 1;
    const int layer = static_cast<int>((e >> 1) % c.layers);
    const long long i = (e >> 1) / c.layers;
    const long long from = static_cast<long long>(layer) * c.pages + a.w.src[i];
    const long long to = static_cast<long long>(layer) * c.pages + a.w.dst[i];
    unsigned char* x = value ? c.v : c.k;
    const uint4* s = reinterpret_cast<const uint4*>(x + from * bytes);
    uint4* d = reinterpret_cast<uint4*>(x + to * bytes);
    const int end = static_cast<int>(bytes / 16);
    const int at = piece * (kCopyPiece / 16) + tid;
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j * kCopyThreads < end) v[j] = s[at + j * kCopyThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j * kCopyThreads < end) d[at + j * kCopyThreads] = v[j];
    if (piece == 0) {
      float* y = value ? c.v_scale : c.k_scale;
      for (int j = tid; j < scales; j += kCopyThreads) y[to * scales + j] = y[from * scales + j];
    }
  }
}

// --------------------------------------------------------------- compact --
struct MovesArgs {
  verbo_cache c;
  PageWs w;
  int* info;
};
// Where each page goes.  live = the pages in use; those at or above it move, the
// highest into the lowest free page: the i-th from the end of all live pages is
// taken by the i-th free one.
template <bool SMALL>
__global__ void __launch_bounds__(SMALL ? kSmallThreads : kScanThreads) cache_moves_kernel(const MovesArgs a) {
  constexpr int PER = SMALL ? kSmallPer : kChunk / kScanThreads;
  __shared__ int pre[SMALL ? 1 : kMaxChunks + 1];
  __shared__ int ws[32];
  const verbo_cache& c = a.c;
  grid_wait();
  grid_release();
  const int chunks = chunks_of(c);
  const int first = (SMALL ? 0 : blockIdx.x * kChunk) + threadIdx.x * PER;
  unsigned mask = 0;  // this thread's free pages
  int live, before;   // free pages before the thread's next one
  if constexpr (SMALL) {
    live = c.pages - scan_pool(c, a.w, ws, &mask, &before);
  } else {
    live = c.pages - scan_counts<kScanThreads>(a.w, chunks, pre, ws);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (first + i < c.pages) mask |= static_cast<unsigned>(c.refs[first + i] == 0) << i;
    int total;
    before = pre[blockIdx.x] + block_excl_scan<int, kScanThreads>(__popc(mask), ws, &total);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int p = first + i;
    if (p >= c.pages) break;
    const bool is_free = mask >> i & 1u;
    int to = p;
    if (p == live) {
      a.info[0] = live;
      a.info[1] = a.w.head[0] = before;
      a.w.head[1] = live;
    }
    if (p >= live && !is_free) {
      const int from_end = live - 1 - (p - before);
      to = SMALL ? a.w.list[from_end] : free_page(a.w, chunks, pre, from_end);
      a.w.src[from_end] = p;
      a.w.dst[from_end] = to;
    }
    a.w.map[p] = to;
    before += is_free;
  }
  if (live == c.pages && blockIdx.x == 0 && threadIdx.x == 0) {
    a.info[0] = live;
    a.info[1] = a.w.head[0] = 0;
    a.w.head[1] = live;
  }
}

// ------------------------------------------------------------------ fork --
struct ForkArgs {
  verbo_cache c;
  const int* parents;
  long long ld;
  int beams;
};
constexpr int kForkThreads = 256;

// A cluster per group; a thread owns columns of its tables: it reads all rows'
// entries of a column (into its own column of shared memory), writes the parents'
// and counts the difference.  Columns where all rows hold the same page, a common
// prompt's, change nothing.
__global__ void __launch_bounds__(kForkThreads) cache_fork_kernel(const ForkArgs a) {
  extern __shared__ int tile[];  // [beams][kForkThreads]
  __shared__ int used[32], from[32], len[32];
  const verbo_cache& c = a.c;
  cg::cluster_group cl = cg::this_cluster();
  const int C = cl.num_blocks(), rank = cl.block_rank();
  const int K = a.beams, tid = threadIdx.x;
  const int group = blockIdx.x / C;
  grid_wait();
  grid_release();
  if (tid < K) {
    const int n = length_of(c, group * K + tid);
    const int p = a.parents[group * a.ld + tid];
    len[tid] = n;
    used[tid] = pages_for(n, c.page);
    from[tid] = p >= 0 && p < K ? p : -1;
  }
  __syncthreads();
  // every CTA has read the lengths before one of them writes the new ones
  cluster_sync_all();
  if (rank == 0 && tid < K) c.lens[group * K + tid] = from[tid] < 0 ? 0 : len[from[tid]];
  int most = 0;
  for (int k = 0; k < K; ++k) most = max(most, used[k]);
  int* t = c.table + static_cast<long long>(group) * K * c.width;
  for (int j = rank * kForkThreads + tid; j < most; j += C * kForkThreads) {
    for (int k0 = 0; k0 < K; k0 += 8) {  // eight rows' entries on their way
      int v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = k0 + k < K && j < used[k0 + k] ? t[static_cast<long long>(k0 + k) * c.width + j] : -1;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < K) tile[(k0 + k) * kForkThreads + tid] = v[k];
    }
    for (int k = 0; k < K; ++k) {
      const int old = tile[k * kForkThreads + tid];
      const int now = from[k] < 0 ? -1 : tile[from[k] * kForkThreads + tid];
      if (now != old) {
        t[static_cast<long long>(k) * c.width + j] = now;
        if (is_page(c, old)) atomicSub(&c.refs[old], 1);
        if (is_page(c, now)) atomicAdd(&c.refs[now], 1);
      }
    }
  }
}

// ------------------------------------------------------------------ free --
struct FreeArgs {
  verbo_cache c;
  const int* keep;
};
constexpr int kFreeThreads = 128;

__global__ void __launch_bounds__(kFreeThreads) cache_free_kernel(const FreeArgs a) {
  const verbo_cache& c = a.c;
  grid_wait();
  grid_release();
  const int row = blockIdx.x;
  const int n = length_of(c, row), keep = a.keep[row];
  if (keep < 0 || keep >= n) return;
  int* t = c.table + static_cast<long long>(row) * c.width;
  const int end = pages_for(n, c.page);
  for (int j = pages_for(keep, c.page) + threadIdx.x; j < end; j += kFreeThreads) {
    if (is_page(c, t[j])) atomicSub(&c.refs[t[j]], 1);
    t[j] = -1;
  }
  __syncthreads();  // every thread has read the length
  if (threadIdx.x == 0) c.lens[row] = keep;
}

// ---------------------------------------------------------------- append --
// One warp per block of 16 tokens, head, and keys or values: the largest new
// element, the scale (an exponent: x / s and, between two scales, codes times a
// power of two are exact before their one rounding), then the codes.
struct AppendArgs {
  verbo_cache c;
  CacheNew x;
  int layer;
  int slots;  // blocks that are looked at
  int per;    // of a row, without offsets
  bool wide;  // 16 bytes at a time
};
constexpr int kAppendThreads = 256;

__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return lo | static_cast<uint32_t>(hi) << 16;
}
__device__ __forceinline__ float2 from_codes(uint32_t two) {  // the low 16 bits
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Eight elements as they lie, and as floats.
template <class T>
struct Eight {
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool wide) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (sizeof(T) == 4) {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(p);
      raw[0] = make_uint4(u[0], u[1], u[2], u[3]);
      raw[1] = make_uint4(u[4], u[5], u[6], u[7]);
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
      raw[0] = make_uint4(u[0] | static_cast<uint32_t>(u[1]) << 16, u[2] | static_cast<uint32_t>(u[3]) << 16,
                          u[4] | static_cast<uint32_t>(u[5]) << 16, u[6] | static_cast<uint32_t>(u[7]) << 16);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
    v.raw = raw[i / N];
    return v.get(i % N);
  }
};

__device__ __forceinline__ float divided(float x, float s, float inv) {
  return inv != 0.0f ? x * inv : __fdiv_rn(x, s);
}

template <class T>
__global__ void __launch_bounds__(kAppendThreads, sizeof(T) == 2 ? 3 : 2) cache_append_kernel(const AppendArgs a) {
  const verbo_cache& c = a.c;
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31;
  const unsigned w = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int slot = static_cast<int>(w / (c.heads * 2u));
  if (slot >= a.slots) return;
  const int rest = static_cast<int>(w - slot * (c.heads * 2u));
  const int head = rest >> 1;
  const bool value = rest & 1;

  // the row, its tokens, and which of its blocks this is
  int row, j;
  long long t0, t1;
  if (a.x.off) {
    // row r's slots begin at off[r] / 16 + 2 r: as many as it can have blocks.  The last
    // row that begins at or before this one, 32 rows looked at in one round trip.
    int lo = 0, count = c.rows;
    while (count > 1) {
      const int each = (count + 31) / 32, r = lo + lane * each;
      const bool before = lane * each < count && a.x.off[r] / kCacheBlock + 2ll * r <= slot;
      const unsigned which = __ballot_sync(0xffffffffu, before) | 1u;
      const int at = (31 - __clz(which)) * each;
      lo += at;
      count = min(each, count - at);
    }
    row = lo;
    t0 = max(0ll, min(a.x.off[row], static_cast<long long>(a.x.tokens)));
    t1 = max(t0, min(a.x.off[row + 1], static_cast<long long>(a.x.tokens)));
    j = static_cast<int>(slot - t0 / kCacheBlock - 2ll * row);
  } else {
    row = slot / a.per;
    j = slot - row * a.per;
    const int each = a.x.tokens / c.rows;
    t0 = static_cast<long long>(row) * each;
    t1 = t0 + each;
  }
  const int start = a.x.start[row];
  if (start < 0 || j < 0) return;
  const long long begin = static_cast<long long>(start) / kCacheBlock * kCacheBlock + static_cast<long long>(j) * kCacheBlock;
  const long long lo = max(begin, static_cast<long long>(start));
  const long long hi = min(begin + kCacheBlock, start + (t1 - t0));
  if (lo >= hi || begin >= static_cast<long long>(c.width) * c.page) return;
  const long long ld = value ? a.x.ld_v : a.x.ld_k;
  const T* x = static_cast<const T*>(value ? a.x.v : a.x.k) + head * (value ? a.x.hd_v : a.x.hd_k) +
               (t0 + (lo - start)) * ld;
  // a lane takes eight elements of a token, of every `side`-th one
  const int eights = c.dim / 8, side = 32 / eights;
  const int tok = lane / eights, col = (lane - tok * eights) * 8;
  const int n = tok < side ? static_cast<int>(hi - lo) : 0;
  constexpr int MOST = 8;  // of a lane, if two tokens lie side by side; up to 128 dims
  Eight<T> e[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i)
    if (tok + i * side < n) e[i].load(x + (tok + i * side) * ld + col, a.wide);
  const int place = static_cast<int>(begin);
  const int id = c.table[static_cast<long long>(row) * c.width + place / c.page];
  if (!is_page(c, id)) return;
  const int inside = place % c.page;
  const long long at = (static_cast<long long>(a.layer) * c.pages + id) * c.heads + head;
  uint32_t* codes = reinterpret_cast<uint32_t*>((value ? c.v : c.k) + (at * c.page + inside) * c.dim);
  float* scale = (value ? c.v_scale : c.k_scale) + at * (c.page / kCacheBlock) + inside / kCacheBlock;
  const bool held = begin < start;
  const float had = held ? *scale : 0.0f;

  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < MOST; ++i)
    if (tok + i * side < n) {
#pragma unroll
      for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(e[i].get(k)));  // NaNs left out
    }
  most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
  if (most > 3.402823466e38f) {  // rare: infinities are left out too
    most = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (tok + i * side < n) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float v = fabsf(e[i].get(k));
          most = fmaxf(most, v <= 3.402823466e38f ? v : 0.0f);
        }
      }
    most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
  }
  // most = 1.m 2^(e - 127); 448 = 1.75 * 2^8
  const uint32_t bits = __float_as_uint(most);
  const int q = max(static_cast<int>(bits >> 23) - ((bits & 0x7fffffu) > 0x600000u ? 134 : 135), -64);
  const float need = __uint_as_float(static_cast<uint32_t>(q + 127) << 23);
  const float s = fmaxf(need, had);
  // 1 / s is exact for a power of two; another scale is the caller's own
  const uint32_t sb = __float_as_uint(s);
  const float inv = (sb & 0x7fffffu) == 0 && sb < (247u << 23) ? __uint_as_float((254u << 23) - sb) : 0.0f;
  if (held && s != had) {
    for (int i = lane; i < static_cast<int>(lo - begin) * (c.dim / 4); i += 32) {
      const uint32_t old = codes[i];
      const float2 u = from_codes(old), v = from_codes(old >> 16);
      codes[i] = to_codes(divided(u.x * had, s, inv), divided(u.y * had, s, inv), divided(v.x * had, s, inv),
                          divided(v.y * had, s, inv));
    }
  }
  unsigned char* to = reinterpret_cast<unsigned char*>(codes) + (static_cast<int>(lo - begin) + tok) * c.dim + col;
  auto store = [&](auto&& coded) {
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (tok + i * side < n) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = coded(e[i].get(k));
        *reinterpret_cast<uint2*>(to + i * side * c.dim) =
            make_uint2(to_codes(v[0], v[1], v[2], v[3]), to_codes(v[4], v[5], v[6], v[7]));
      }
  };
  if (inv != 0.0f)
    store([&](float v) { return v * inv; });
  else
    store([&](float v) { return __fdiv_rn(v, s); });
  if (lane == 0 && !(held && s == had)) *scale = s;
}

template <class T>
cudaError_t run_append(AppendArgs a, cudaStream_t s) {
  const long long warps = static_cast<long long>(a.slots) * a.c.heads * 2;
  const long long grid = (warps + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (warps > INT_MAX) return cudaErrorInvalidConfiguration;
  // eight elements at once where every group of them is aligned to 16 bytes
  const long long all = a.x.ld_k | a.x.hd_k | a.x.ld_v | a.x.hd_v;
  a.wide = all % Vec<T>::N == 0 && reinterpret_cast<uintptr_t>(a.x.k) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(a.x.v) % 16 == 0;
  return launch_chained(cache_append_kernel<T>, static_cast<unsigned>(grid), kAppendThreads, 0, 1, s, a);
}

cudaError_t launch_copy(const verbo_cache& c, const PageWs& w, bool remap, cudaStream_t s) {
  return launch_chained(cache_copy_kernel, static_cast<unsigned>(sm_count()) * 8u, kCopyThreads, 0, 1, s,
                        CopyArgs{c, w, remap});
}

}  // namespace

size_t cache_workspace_bytes(const verbo_cache& c) {
  const size_t ints = 4 + chunks_of(c) + static_cast<size_t>(chunks_of(c)) * kChunk + 2 * most_copies(c) + c.pages;
  return (ints * 4 + 15) / 16 * 16;
}

cudaError_t launch_cache_reserve(const verbo_cache& c, const int* add, int* start, int* status, void* ws,
                                 cudaStream_t s) {
  const PageWs w = layout(c, ws);
  const ReserveArgs a{c, w, add, start, status};
  const size_t rows = 5 * ((static_cast<size_t>(c.rows) + 3) / 4 * 4) * 4;
  constexpr int most = (5 * VERBO_CACHE_MAX_ROWS + kMaxChunks + 1) * 4;
  cudaError_t e;
  if (c.pages <= kSmallPool) {
    e = allow_smem<cache_reserve_kernel<true>>(most);
    if (e == cudaSuccess) e = launch_chained(cache_reserve_kernel<true>, 1u, kReserveThreads, rows, 1, s, a);
  } else {
    e = launch_chained(cache_scan_kernel, static_cast<unsigned>(chunks_of(c)), kScanThreads, 0, 1, s, ScanArgs{c, w});
    if (e == cudaSuccess) e = allow_smem<cache_reserve_kernel<false>>(most);
    if (e == cudaSuccess)
      e = launch_chained(cache_reserve_kernel<false>, 1u, kReserveThreads, rows + (chunks_of(c) + 1) * 4, 1, s, a);
  }
  return e == cudaSuccess ? launch_copy(c, w, false, s) : e;
}

cudaError_t launch_cache_fork(const verbo_cache& c, const int* parents, long long ld_parents, int beams,
                              cudaStream_t s) {
  const int groups = c.rows / beams;
  // CTAs per group: as many as the columns give work to, while SMs are left (8 rows of 1024
  // pages 4.0 us, 8.7 with one; of 8192 pages 10 and 58)
  int C = 1;
  while (C < 8 && C * kForkThreads < c.width && groups * C * 2 <= sm_count()) C <<= 1;
  return launch_chained(cache_fork_kernel, static_cast<unsigned>(groups * C), kForkThreads,
                        static_cast<size_t>(beams) * kForkThreads * 4, C, s, ForkArgs{c, parents, ld_parents, beams});
}

cudaError_t launch_cache_free(const verbo_cache& c, const int* keep, cudaStream_t s) {
  return launch_chained(cache_free_kernel, static_cast<unsigned>(c.rows), kFreeThreads, 0, 1, s, FreeArgs{c, keep});
}

cudaError_t launch_cache_compact(const verbo_cache& c, int* info, void* ws, cudaStream_t s) {
  const PageWs w = layout(c, ws);
  const MovesArgs a{c, w, info};
  cudaError_t e;
  if (c.pages <= kSmallPool) {
    e = launch_chained(cache_moves_kernel<true>, 1u, kSmallThreads, 0, 1, s, a);
  } else {
    e = launch_chained(cache_scan_kernel, static_cast<unsigned>(chunks_of(c)), kScanThreads, 0, 1, s, ScanArgs{c, w});
    if (e == cudaSuccess)
      e = launch_chained(cache_moves_kernel<false>, static_cast<unsigned>(chunks_of(c)), kScanThreads, 0, 1, s, a);
  }
  return e == cudaSuccess ? launch_copy(c, w, true, s) : e;
}

cudaError_t launch_cache_append(const verbo_cache& c, int layer, const CacheNew& x, int dtype, cudaStream_t s) {
  AppendArgs a{c, x, layer, 0, 1, false};
  if (x.off) {
    const long long slots = static_cast<long long>(x.tokens) / kCacheBlock + 2ll * c.rows;
    if (slots > INT_MAX) return cudaErrorInvalidConfiguration;
    a.slots = static_cast<int>(slots);
  } else {
    a.per = (x.tokens / c.rows + 2 * kCacheBlock - 2) / kCacheBlock;
    const long long slots = static_cast<long long>(a.per) * c.rows;
    if (slots > INT_MAX) return cudaErrorInvalidConfiguration;
    a.slots = static_cast<int>(slots);
  }
  if (dtype == kOpsF16) return run_append<__half>(a, s);
  if (dtype == kOpsBF16) return run_append<__nv_bfloat16>(a, s);
  return run_append<float>(a, s);
}

}  // namespace vb
