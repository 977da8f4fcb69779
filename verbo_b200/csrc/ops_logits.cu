// Logits operators around the sampler (include/verbo_ops.h): penalties, biases
// and masks before the pick, log-probabilities after it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "device.cuh"
#include "ops.cuh"

namespace vb {
namespace {

constexpr float kNegInf = -__builtin_huge_valf();

template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_float(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

// Elements of a 16-byte vector as floats.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ float get(int i) const;
};
template <>
__device__ __forceinline__ float Vec<float>::get(int i) const {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  return __uint_as_float(w[i]);
}
template <>
__device__ __forceinline__ float Vec<__half>::get(int i) const {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  return __half2float(__ushort_as_half(static_cast<unsigned short>(w[i >> 1] >> (16 * (i & 1)))));
}
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::get(int i) const {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
}

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// The row's own 16-byte grid: a row of element stride ld starts anywhere, so a
// kernel counts columns from the 16-byte boundary at or before the row, u =
// column + row_shift, and vectors of N columns at u a multiple of N are aligned.
template <class T>
__device__ __forceinline__ int row_shift(const T* row) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % Vec<T>::N);
}

// =============================================================== process ==
// out = mask(bias(penalties(logits))), include/verbo_ops.h.  One pass: each CTA
// takes NT * V vectors of one row.  The loads of its logits go out first; while
// they are in flight it counts the row's window into one shared counter per
// column (integer atomics: exact in any order) and marks each biased column
// with the place of its last entry (atomicMax), so no later step depends on the
// order in which threads ran.  A CTA re-reads its row's whole window, from L2.
// In place nothing of the row is loaded but columns that change.
template <class T, int NT, int V, bool INPLACE>
__global__ void __launch_bounds__(NT, 2048 / NT / 2) process_kernel(const ProcArgs a) {
  constexpr int N = Vec<T>::N;
  constexpr int S = NT * V * N;
  extern __shared__ __align__(16) int smem_i[];  // counts [S], then bias places [S]: whichever the call has
  grid_wait();
  const int row = blockIdx.x / a.slices;
  const int u0 = (blockIdx.x - row * a.slices) * S;
  const int tid = threadIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.ld;
  float* out = a.out + row * a.ld_out;
  const int shift = row_shift(in);
  const int c0 = u0 - shift;  // column of the slice's first place
  if (c0 >= a.vocab) return;

  long long hb = 0, he = 0, bb = 0, be = 0;
  if (a.hist) {
    hb = a.hist_off[row];
    he = a.hist_off[row + 1];
    if (a.last > 0 && he - hb > a.last) hb = he - a.last;
  }
  if (a.bias) {
    bb = a.bias_off[row];
    be = a.bias_off[row + 1];
  }

  Vec<T> x[V];
  if (!INPLACE) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = c0 + (i * NT + tid) * N;
      if (c >= 0 && c + N <= a.vocab) x[i].raw = ld_stream16(in + c);
    }
  }

  int* cnt = smem_i;
  int* at = smem_i + (a.hist ? S : 0);
  const bool have_h = he > hb, have_b = be > bb;  // the same in every thread of the CTA
  float rep = a.repeat, freq = a.frequency, pres = a.presence;
  if (have_h || have_b) {
    if (have_h && a.row_pen) {
      rep = a.row_pen[3ll * row];
      freq = a.row_pen[3ll * row + 1];
      pres = a.row_pen[3ll * row + 2];
    }
#pragma unroll
    for (int i = 0; i < V * N / 4; ++i) {
      if (have_h) reinterpret_cast<int4*>(cnt)[i * NT + tid] = make_int4(0, 0, 0, 0);
      if (have_b) reinterpret_cast<int4*>(at)[i * NT + tid] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    for (long long i = hb + tid; i < he; i += NT) {
      const int id = a.hist[i];
      if (id < 0 || id >= a.vocab) continue;
      const int p = id - c0;
      if (p >= 0 && p < S) atomicAdd(&cnt[p], 1);
    }
    for (long long i = bb + tid; i < be; i += NT) {
      const int id = a.bias_ids[i];
      if (id < 0 || id >= a.vocab) continue;
      const int p = id - c0;
      if (p >= 0 && p < S) atomicMax(&at[p], static_cast<int>(i - bb) + 1);
    }
    __syncthreads();
  }
  const float* bias = a.bias + bb - 1;
  const uint32_t* mask = a.mask ? a.mask + row * a.ld_mask : nullptr;

#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int p = (i * NT + tid) * N;
    const int c = c0 + p;
    if (c >= a.vocab || c + N <= 0) continue;
    const bool full = c >= 0 && c + N <= a.vocab;
    uint32_t ok = (1u << N) - 1;  // bit j: column c + j is allowed
    if (mask) {
      if (full) {
        const int w = c >> 5, sh = c & 31;
        const uint32_t lo = __ldg(mask + w);
        const uint32_t hi = sh + N > 32 ? __ldg(mask + w + 1) : 0u;
        ok &= __funnelshift_r(lo, hi, sh);
      } else {
        for (int j = 0; j < N; ++j)
          if (c + j >= 0 && c + j < a.vocab && !((__ldg(mask + ((c + j) >> 5)) >> ((c + j) & 31)) & 1u))
            ok &= ~(1u << j);
      }
    }
    int k[N], b[N];
    int any = 0;
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      int4 t = make_int4(0, 0, 0, 0), s = t;
      if (have_h) t = *reinterpret_cast<const int4*>(cnt + p + j);
      if (have_b) s = *reinterpret_cast<const int4*>(at + p + j);
      k[j] = t.x, k[j + 1] = t.y, k[j + 2] = t.z, k[j + 3] = t.w;
      b[j] = s.x, b[j + 1] = s.y, b[j + 2] = s.z, b[j + 3] = s.w;
      any |= t.x | t.y | t.z | t.w | s.x | s.y | s.z | s.w;
    }
    if (INPLACE) {
      if (any == 0 && ok == (1u << N) - 1) continue;
      if (full && ok == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 4)
          *reinterpret_cast<float4*>(out + c + j) = make_float4(kNegInf, kNegInf, kNegInf, kNegInf);
        continue;
      }
    }
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const bool inside = full || (c + j >= 0 && c + j < a.vocab);
      const bool touched = (k[j] | b[j]) != 0;
      v[j] = 0.0f;
      if (INPLACE) {
        if (inside && touched && ((ok >> j) & 1u)) v[j] = out[c + j];
      } else if (full) {
        v[j] = x[i].get(j);
      } else if (inside) {
        v[j] = to_float(in[c + j]);
      }
      if (touched) {
        if (k[j] > 0) {
          v[j] = penalize(v[j], rep);
          v[j] = __fsub_rn(v[j], __fmul_rn(freq, static_cast<float>(k[j])));
          v[j] = __fsub_rn(v[j], pres);
        }
        if (b[j] > 0) v[j] = __fadd_rn(v[j], bias[b[j]]);
      }
      if (!((ok >> j) & 1u)) v[j] = kNegInf;
      if (INPLACE && inside && (touched || !((ok >> j) & 1u))) out[c + j] = v[j];
    }
    if (!INPLACE) {
      if (full && (reinterpret_cast<uintptr_t>(out + c) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 4)
          *reinterpret_cast<float4*>(out + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (full || (c + j >= 0 && c + j < a.vocab)) out[c + j] = v[j];
      }
    }
  }
}

template <class K, class A>
cudaError_t launch_chained(K kernel, unsigned grid, int threads, size_t smem, int cluster, cudaStream_t s, const A& a) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <class T, int NT, int V, bool INPLACE>
cudaError_t run_process(ProcArgs a, cudaStream_t s) {
  constexpr int N = Vec<T>::N;
  constexpr int S = NT * V * N;
  a.slices = static_cast<int>((static_cast<long long>(a.vocab) + N - 1 + S - 1) / S);
  const long long grid = static_cast<long long>(a.rows) * a.slices;
  if (grid > INT_MAX) return cudaErrorInvalidConfiguration;
  const size_t smem = (a.hist ? S * 4u : 0u) + (a.bias ? S * 4u : 0u);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(process_kernel<T, NT, V, INPLACE>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  return launch_chained(process_kernel<T, NT, V, INPLACE>, static_cast<unsigned>(grid), NT, smem, 1, s, a);
}

// Slices of 8192 columns, or of 2048 while those leave SMs idle.
template <class T, bool INPLACE>
cudaError_t pick_process(const ProcArgs& a, cudaStream_t s) {
  constexpr int V = 16 / Vec<T>::N;
  if (static_cast<long long>(a.rows) * a.vocab <= 148ll * 8192) return run_process<T, 256, V / 2, INPLACE>(a, s);
  return run_process<T, 512, V, INPLACE>(a, s);
}

// ============================================================== logprobs ==
// Log-probabilities, rank and the first columns of a row, one pass over it.
// A cluster of CTAs shares a row.  A thread keeps the maximum m of its columns
// and s = sum 2^(c (v - m)), c = log2(e) / temp.  In a batch the terms come from
// one fma each, 2^(c v + b) with b = -c m rounded; c v is exact inside the fma,
// so the rounding of b is one factor for the whole batch, 2^(-c m - b), which is
// multiplied back.
// The first columns: a bound T with at least `top` columns of the CTA at or
// above it comes from the maxima of the first batch (below); every column that
// reaches T is put into a shared list, from which the `top` first are ranked by
// counting.  A list that overflows is gathered anew with a sharper bound.
constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpBatch = 16;  // columns per thread and batch
constexpr int kLpCap = 2048;  // listed columns per CTA
constexpr int kLpMaxCluster = 8;

struct LpPart {
  float m, s;  // maximum, sum of 2^(c (v - m))
  int rank;    // columns before the chosen one
  int ninf;    // columns at +inf
  int ntop;    // keys in the slot
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// s seen from another maximum m >= the one it was taken at.
__device__ __forceinline__ float lp_scaled(float s, float from, float m, float c) {
  return s > 0.0f && m != -kNegInf ? s * ex2((from - m) * c) : 0.0f;
}

struct LpAcc {
  float m = kNegInf, s = 0.0f;
  int ninf = 0;
  // bm: the maximum of x[0, n)
  template <int n>
  __device__ __forceinline__ void add(const float (&x)[n], float bm, float c) {
    if (bm == -kNegInf) {  // +inf alone counts then
#pragma unroll
      for (int j = 0; j < n; ++j) ninf += x[j] == -kNegInf;
      m = bm;
    }
    if (m == -kNegInf) return;
    if (bm > m) {
      s = lp_scaled(s, m, bm, c);
      m = bm;
    }
    if (fabsf(m) < 1e30f) {
      const float b = -m * c;
      float t = 0.0f;
#pragma unroll
      for (int j = 0; j < n; ++j) t += ex2(fmaf(x[j], c, b));
      s += t * ex2(fmaf(-m, c, -b));
    } else if (m != kNegInf) {  // c m may overflow (rows masked with the type's lowest value)
#pragma unroll
      for (int j = 0; j < n; ++j) s += ex2((x[j] - m) * c);
    }
  }
};

template <class T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 2) logprob_kernel(const LogprobArgs a) {
  constexpr int N = Vec<T>::N;
  constexpr int NV = kLpBatch / N;  // vectors per thread and batch
  __shared__ LpPart parts[kLpWarps];
  __shared__ LpPart slots[kLpMaxCluster];  // the leader's: one per CTA
  __shared__ uint64_t slot_keys[TOP ? kLpMaxCluster * kLpMaxTop : 1];
  __shared__ uint64_t list[TOP ? kLpCap : 1];
  __shared__ uint64_t best[TOP ? kLpMaxTop : 1];
  __shared__ uint32_t offer[kLpWarps];
  __shared__ int count;
  __shared__ uint64_t bound_key;

  cg::cluster_group cl = cg::this_cluster();
  const int C = cl.num_blocks();
  const int rankc = cl.block_rank();
  if (C > 1) cluster_arrive();  // every CTA of the cluster has started before one writes to the leader
  grid_wait();
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* in = static_cast<const T*>(a.logits) + row * a.ld;
  const int shift = row_shift(in);
  const float c = 1.4426950408889634f / a.temp;
  const int top = a.top;
  // this CTA's columns [lo, hi), counted from the row's 16-byte boundary
  const long long ulo = static_cast<long long>(rankc) * a.slice;
  const int lo = static_cast<int>(max(0ll, ulo - shift));
  const int hi = static_cast<int>(min(static_cast<long long>(a.vocab), ulo + a.slice - shift));
  const int cu = static_cast<int>(min(ulo - shift, static_cast<long long>(a.vocab)));  // its first vector's column
  const int nbatch = hi > lo ? (hi - cu + kLpThreads * kLpBatch - 1) / (kLpThreads * kLpBatch) : 0;

  int id = -1;
  if (a.ids) {
    id = a.ids[row];
    if (id < 0 || id >= a.vocab) id = -1;
  }
  if (TOP && tid == 0) count = 0;

  Vec<T> x[NV], y[NV];
  auto load = [&](int batch, Vec<T>(&v)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = cu + ((batch * NV + i) * kLpThreads + tid) * N;
      if (col >= lo && col + N <= hi) {
        v[i].raw = ld_stream16(in + col);
      } else {
        const bool any = col + N > lo && col < hi;
        v[i].raw = make_uint4(0, 0, 0, 0);
        if (any) {  // the row's ragged ends, element by element
          uint32_t w[4] = {0, 0, 0, 0};
          for (int j = 0; j < N; ++j)
            if (col + j >= lo && col + j < hi) {
              const T e = in[col + j];
              if (sizeof(T) == 4)
                w[j & 3] = *reinterpret_cast<const uint32_t*>(&e);
              else
                w[(j >> 1) & 3] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&e)) << (16 * (j & 1));
            }
          v[i].raw = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  };
  if (nbatch > 0) load(0, x);
  const float chosen = id >= 0 ? fmaxf(to_float(in[id]), kNegInf) : 0.0f;  // a NaN counts as -inf

  LpAcc acc;
  int before = 0;
  float thr = kNegInf;  // T: columns at or above it are listed
  for (int bt = 0; bt < nbatch; ++bt) {
    if (bt + 1 < nbatch) load(bt + 1, y);
    float v[kLpBatch];
    float bm = kNegInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = cu + ((bt * NV + i) * kLpThreads + tid) * N;
      const bool full = col >= lo && col + N <= hi;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float e = fmaxf(x[i].get(j), kNegInf);
        if (!full && !(col + j >= lo && col + j < hi)) e = kNegInf;
        v[i * N + j] = e;
        bm = fmaxf(bm, e);
      }
      if (id >= 0) {
        if (full && col > id) {
#pragma unroll
          for (int j = 0; j < N; ++j) before += v[i * N + j] > chosen;
        } else if (full && col + N <= id) {
#pragma unroll
          for (int j = 0; j < N; ++j) before += v[i * N + j] >= chosen;
        } else {
          for (int j = 0; j < N; ++j)
            if (col + j >= lo && col + j < hi)
              before += v[i * N + j] > chosen || (v[i * N + j] == chosen && col + j < id);
        }
      }
    }
    acc.add(v, bm, c);
    if (TOP) {
      if (bt == 0) {
        // Every warp offers the q-th largest of its lanes' maxima: at least
        // q * kLpWarps >= top columns reach the lowest offer.  From there the
        // bound is raised, by halving, while `top` maxima still reach it.
        const int q = (top + kLpWarps - 1) / kLpWarps;
        uint32_t o = ord32(bm + 0.0f);
        const uint32_t mine = o;
        uint32_t w = __reduce_max_sync(0xffffffffu, o);
        if (q > 1) {
          const unsigned at = __ballot_sync(0xffffffffu, o == w);
          if (lane == __ffs(at) - 1) o = 0;
          w = __reduce_max_sync(0xffffffffu, o);
        }
        if (lane == 0) offer[warp] = w;
        __syncthreads();
        const uint32_t least = ord32(-3.402823466e38f);  // a column at -inf is never listed
        uint32_t low = offer[0], high = offer[0];
        for (int i = 1; i < kLpWarps; ++i) {
          low = min(low, offer[i]);
          high = max(high, offer[i]);
        }
        low = max(low, least);
        for (int it = 0; it < 12 && low < high; ++it) {
          const uint32_t mid = low + (high - low + 1) / 2;
          const int n = __syncthreads_count(mine >= mid);
          if (n >= top) {
            low = mid;
            if (n <= 2 * top) break;
          } else {
            high = mid - 1;
          }
        }
        thr = unord32(low);
      }
      if (bm >= thr) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (v[i * N + j] >= thr) {
              const int p = atomicAdd(&count, 1);
              if (p < kLpCap)
                list[p] = dkey(v[i * N + j], cu + ((bt * NV + i) * kLpThreads + tid) * N + j);
            }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = y[i];
  }

  // the CTA's part of the row
  LpPart p;
  p.m = unord32(__reduce_max_sync(0xffffffffu, ord32(acc.m + 0.0f)));
  p.s = lp_scaled(acc.s, acc.m, p.m, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) p.s += __shfl_xor_sync(0xffffffffu, p.s, o);
  p.rank = __reduce_add_sync(0xffffffffu, before);
  p.ninf = __reduce_add_sync(0xffffffffu, acc.ninf);
  p.ntop = 0;
  if (lane == 0) parts[warp] = p;
  __syncthreads();

  int ntop = 0;
  if (TOP) {
    int n = count;
    // Too many: the `top`-th of those that were kept is a bound that as many
    // columns reach; gather again from it on, in the order of the keys (distinct,
    // so at least kLpCap - top columns drop out each time).
    while (n > kLpCap) {
      for (int i = tid; i < kLpCap; i += kLpThreads) {
        int r = 0;
        const uint64_t k = list[i];
        for (int j = 0; j < kLpCap; ++j) r += list[j] < k;
        if (r == top - 1) bound_key = k;
      }
      __syncthreads();
      const uint64_t bk = bound_key;
      if (tid == 0) count = 0;
      __syncthreads();
      for (int col = lo + tid; col < hi; col += kLpThreads) {
        const float e = fmaxf(to_float(in[col]), kNegInf);
        const uint64_t k = dkey(e, col);
        if (e > kNegInf && k <= bk) {
          const int at = atomicAdd(&count, 1);
          if (at < kLpCap) list[at] = k;
        }
      }
      __syncthreads();
      n = count;
      __syncthreads();
    }
    ntop = min(n, top);
    for (int i = tid; i < n; i += kLpThreads) {
      int r = 0;
      const uint64_t k = list[i];
      for (int j = 0; j < n; ++j) r += list[j] < k;
      if (r < top) best[r] = k;
    }
    __syncthreads();
  }

  LpPart mine;
  if (warp == 0) {
    const LpPart w = lane < kLpWarps ? parts[lane] : LpPart{kNegInf, 0.0f, 0, 0, 0};
    mine.m = unord32(__reduce_max_sync(0xffffffffu, ord32(w.m + 0.0f)));
    mine.s = lp_scaled(w.s, w.m, mine.m, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine.s += __shfl_xor_sync(0xffffffffu, mine.s, o);
    mine.rank = __reduce_add_sync(0xffffffffu, w.rank);
    mine.ninf = __reduce_add_sync(0xffffffffu, w.ninf);
    mine.ntop = ntop;
  }
  if (C > 1) {
    cluster_wait();
    if (tid == 0) *cl.map_shared_rank(&slots[rankc], 0) = mine;
    if (TOP && tid < ntop) *cl.map_shared_rank(&slot_keys[rankc * kLpMaxTop + tid], 0) = best[tid];
    cluster_sync_all();
    if (rankc != 0) return;
  } else {
    if (tid == 0) slots[0] = mine;
    if (TOP && tid < ntop) slot_keys[tid] = best[tid];
    __syncthreads();
  }

  // the leader: the row's maximum and sum, then the outputs
  float m = kNegInf;
  int ninf = 0, rank = 0;
  for (int i = 0; i < C; ++i) {
    m = fmaxf(m, slots[i].m);
    ninf += slots[i].ninf;
    rank += slots[i].rank;
  }
  float s = 0.0f;
  if (m == -kNegInf)
    s = static_cast<float>(ninf);
  else
    for (int i = 0; i < C; ++i) s += lp_scaled(slots[i].s, slots[i].m, m, c);
  const float ls = logf(s);
  auto logp = [&](float v) {
    if (v == kNegInf) return kNegInf;
    if (v == m) return -ls;
    return __fdiv_rn(v - m, a.temp) - ls;
  };
  if (tid == 0 && a.ids) {
    a.logprob[row] = id >= 0 ? logp(chosen) : kNegInf;
    a.rank[row] = id >= 0 ? rank : -1;
  }
  if (TOP) {
    // a key's place: its own in its list, and what comes before it in the others
    for (int i = tid; i < C * top; i += kLpThreads) {
      const int l = i / top, at = i - l * top;
      if (at >= slots[l].ntop) continue;
      const uint64_t k = slot_keys[l * kLpMaxTop + at];
      int r = at;
      for (int o = 0; o < C; ++o) {
        if (o == l) continue;
        int b = 0, e = slots[o].ntop;
        while (b < e) {
          const int h = (b + e) >> 1;
          if (slot_keys[o * kLpMaxTop + h] < k)
            b = h + 1;
          else
            e = h;
        }
        r += b;
      }
      if (r < top) {
        a.top_ids[static_cast<long long>(row) * top + r] = static_cast<int>(did(k));
        a.top_logprobs[static_cast<long long>(row) * top + r] = logp(dval(k));
      }
    }
    int have = 0;
    for (int i = 0; i < C; ++i) have += slots[i].ntop;
    for (int i = have + tid; i < top; i += kLpThreads) {
      a.top_ids[static_cast<long long>(row) * top + i] = -1;
      a.top_logprobs[static_cast<long long>(row) * top + i] = kNegInf;
    }
  }
}

template <class T>
cudaError_t run_logprobs(LogprobArgs a, cudaStream_t s) {
  constexpr int N = Vec<T>::N;
  // enough CTAs for the SMs, in slices of a batch (8192 columns) or more
  int C = 1;
  while (C < kLpMaxCluster && static_cast<long long>(C) * kLpThreads * kLpBatch < a.vocab &&
         static_cast<long long>(a.rows) * C < 148 * 4)
    C <<= 1;
  const long long span = static_cast<long long>(a.vocab) + N - 1;
  a.slice = static_cast<int>(((span + C - 1) / C + N - 1) / N * N);
  const long long grid = static_cast<long long>(a.rows) * C;
  if (grid > INT_MAX) return cudaErrorInvalidConfiguration;
  return a.top > 0 ? launch_chained(logprob_kernel<T, true>, static_cast<unsigned>(grid), kLpThreads, 0, C, s, a)
                   : launch_chained(logprob_kernel<T, false>, static_cast<unsigned>(grid), kLpThreads, 0, C, s, a);
}

}  // namespace

cudaError_t launch_process(ProcArgs a, int dtype, bool in_place, cudaStream_t s) {
  if (dtype == kOpsF16) return pick_process<__half, false>(a, s);
  if (dtype == kOpsBF16) return pick_process<__nv_bfloat16, false>(a, s);
  return in_place ? pick_process<float, true>(a, s) : pick_process<float, false>(a, s);
}

cudaError_t launch_logprobs(LogprobArgs a, int dtype, cudaStream_t s) {
  if (dtype == kOpsF16) return run_logprobs<__half>(a, s);
  if (dtype == kOpsBF16) return run_logprobs<__nv_bfloat16>(a, s);
  return run_logprobs<float>(a, s);
}

}  // namespace vb
