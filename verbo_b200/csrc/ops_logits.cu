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
// out = mask(bias(penalties(logits))), include/verbo_ops.h.  One pass over the
// row; a CTA walks a part of it in slices of NT * 16 columns.  Per slice it
// counts the window's ids into one shared counter per column (integer atomics:
// exact in any order), with the top bit for a biased column, whose last entry
// is found by atomicMax; so nothing depends on the order in which threads ran.
// The thread that owns a column takes its counter back to 0.  The first ids of
// the window stay in registers over the slices, and the next slice's logits
// and mask words are on their way while a slice is counted and stored.
// In place nothing of the row is loaded but columns that change.
constexpr int kProcThreads = 256;
constexpr int kProcCols = 16;                         // columns per thread and slice
constexpr int kProcSlice = kProcThreads * kProcCols;  // 4096
constexpr int kProcHist = 4, kProcBias = 1;           // ids per thread in registers

template <class T, bool LISTS, bool INPLACE>
__global__ void __launch_bounds__(kProcThreads, 4) process_kernel(const ProcArgs a) {
  constexpr int N = Vec<T>::N, NT = kProcThreads, V = kProcCols / N, S = kProcSlice;
  constexpr uint32_t kAll = (1u << N) - 1;
  constexpr int kNone = -(1 << 30);  // an id that lies in no slice
  extern __shared__ __align__(16) int smem_i[];  // counters [S], then (with biases) last entries [S]
  grid_wait();
  const int row = blockIdx.x / a.parts;
  const int part = blockIdx.x - row * a.parts;
  const int tid = threadIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.ld;
  float* out = a.out + row * a.ld_out;
  const uint32_t* mask = a.mask ? a.mask + row * a.ld_mask : nullptr;
  const int shift = row_shift(in);
  const int c0 = part * a.part_cols - shift;
  const int c1 = min(a.vocab, c0 + a.part_cols);
  if (c0 >= c1) return;

  Vec<T> x[V];
  uint32_t ml[V], mh[V];
  auto load = [&](int cs) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = cs + (i * NT + tid) * N;
      if (c >= 0 && c + N <= a.vocab) {
        if (!INPLACE) x[i].raw = ld_stream16(in + c);
        if (mask) {
          const uint32_t* w = mask + (c >> 5);
          ml[i] = __ldg(w);
          mh[i] = (c & 31) + N > 32 ? __ldg(w + 1) : 0u;
        }
      }
    }
  };
  if (!LISTS) load(c0);

  int* cnt = smem_i;
  int* at = smem_i + S;
  long long hb = 0, hn = 0, bb = 0, bn = 0;
  int hid[kProcHist], bid[kProcBias];
  float rep = a.repeat, freq = a.frequency, pres = a.presence;
  if (LISTS) {
    if (a.hist) {
      hb = a.hist_off[row];
      hn = max(0ll, a.hist_off[row + 1] - hb);
    }
    if (a.bias) {
      bb = a.bias_off[row];
      bn = max(0ll, a.bias_off[row + 1] - bb);
    }
    load(c0);
    if (a.last > 0 && hn > a.last) {
      hb += hn - a.last;
      hn = a.last;
    }
    auto valid = [&](int id) { return id >= 0 && id < a.vocab ? id : kNone; };
#pragma unroll
    for (int i = 0; i < kProcHist; ++i) hid[i] = i * NT + tid < hn ? valid(a.hist[hb + i * NT + tid]) : kNone;
#pragma unroll
    for (int i = 0; i < kProcBias; ++i) bid[i] = i * NT + tid < bn ? valid(a.bias_ids[bb + i * NT + tid]) : kNone;
    if (hn > 0 && a.row_pen) {
      rep = a.row_pen[3ll * row];
      freq = a.row_pen[3ll * row + 1];
      pres = a.row_pen[3ll * row + 2];
    }
  }
  const bool lists = LISTS && (hn > 0 || bn > 0);  // the same in every thread of the CTA
  if (lists) {
#pragma unroll
    for (int i = 0; i < S / 4 / NT; ++i) {
      reinterpret_cast<int4*>(cnt)[i * NT + tid] = make_int4(0, 0, 0, 0);
      if (a.bias) reinterpret_cast<int4*>(at)[i * NT + tid] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
  }
  // one column: the whole of the operator but the mask
  auto apply = [&](float v, int k, int p) {
    if (k & 0x7fffffff) {
      v = penalize(v, rep);
      v = __fsub_rn(v, __fmul_rn(freq, static_cast<float>(k & 0x7fffffff)));
      v = __fsub_rn(v, pres);
    }
    if (k < 0) {
      v = __fadd_rn(v, a.bias[bb + at[p] - 1]);
      at[p] = 0;
    }
    return v;
  };

  for (int cs = c0; cs < c1; cs += S) {
    if (lists) {
#pragma unroll
      for (int i = 0; i < kProcHist; ++i) {
        const int p = hid[i] - cs;
        if (p >= 0 && p < S) atomicAdd(&cnt[p], 1);
      }
      for (long long i = kProcHist * NT + tid; i < hn; i += NT) {
        const int id = a.hist[hb + i];
        const int p = id >= 0 && id < a.vocab ? id - cs : -1;
        if (p >= 0 && p < S) atomicAdd(&cnt[p], 1);
      }
#pragma unroll
      for (int i = 0; i < kProcBias; ++i) {
        const int p = bid[i] - cs;
        if (p >= 0 && p < S) {
          atomicOr(&cnt[p], INT_MIN);
          atomicMax(&at[p], i * NT + tid + 1);
        }
      }
      for (long long i = kProcBias * NT + tid; i < bn; i += NT) {
        const int id = a.bias_ids[bb + i];
        const int p = id >= 0 && id < a.vocab ? id - cs : -1;
        if (p >= 0 && p < S) {
          atomicOr(&cnt[p], INT_MIN);
          atomicMax(&at[p], static_cast<int>(i) + 1);
        }
      }
      __syncthreads();
    }
    Vec<T> y[V];
    uint32_t ok[V];  // bit j: the vector's column j is allowed
#pragma unroll
    for (int i = 0; i < V; ++i) {
      y[i] = x[i];
      ok[i] = mask ? __funnelshift_r(ml[i], mh[i], (cs + (i * NT + tid) * N) & 31) & kAll : kAll;
    }
    if (cs + S < c1) load(cs + S);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int p = (i * NT + tid) * N;
      const int c = cs + p;
      if (c >= 0 && c + N <= a.vocab) {
        int k[N];
        int any = 0;
        if (lists) {
#pragma unroll
          for (int j = 0; j < N; j += 4) {
            const int4 t = *reinterpret_cast<const int4*>(cnt + p + j);
            k[j] = t.x, k[j + 1] = t.y, k[j + 2] = t.z, k[j + 3] = t.w;
            any |= t.x | t.y | t.z | t.w;
          }
          if (any) {
#pragma unroll
            for (int j = 0; j < N; j += 4) *reinterpret_cast<int4*>(cnt + p + j) = make_int4(0, 0, 0, 0);
          }
        }
        if (INPLACE) {
          if (any) {
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (k[j]) {
                const float v = apply((ok[i] >> j) & 1u ? out[c + j] : 0.0f, k[j], p + j);
                if ((ok[i] >> j) & 1u) out[c + j] = v;
              }
          }
          if (ok[i] == 0) {
#pragma unroll
            for (int j = 0; j < N; j += 4)
              *reinterpret_cast<float4*>(out + c + j) = make_float4(kNegInf, kNegInf, kNegInf, kNegInf);
          } else if (ok[i] != kAll) {
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (!((ok[i] >> j) & 1u)) out[c + j] = kNegInf;
          }
        } else {
          float v[N];
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] = y[i].get(j);
          if (any) {
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (k[j]) v[j] = apply(v[j], k[j], p + j);
          }
          if (ok[i] != kAll) {
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (!((ok[i] >> j) & 1u)) v[j] = kNegInf;
          }
          if ((reinterpret_cast<uintptr_t>(out + c) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < N; j += 4)
              *reinterpret_cast<float4*>(out + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < N; ++j) out[c + j] = v[j];
          }
        }
      } else if (c + N > 0 && c < a.vocab) {  // the row's ragged ends
        for (int j = max(0, -c); j < min(N, a.vocab - c); ++j) {
          const int k = lists ? cnt[p + j] : 0;
          const bool allowed = !mask || ((__ldg(mask + ((c + j) >> 5)) >> ((c + j) & 31)) & 1u);
          if (INPLACE && allowed && k == 0) continue;
          float v = to_float(in[c + j]);
          if (k) {
            v = apply(v, k, p + j);
            cnt[p + j] = 0;
          }
          out[c + j] = allowed ? v : kNegInf;
        }
      }
    }
    if (lists) __syncthreads();
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

// Parts of as many slices as leave at least four waves of CTAs, 8 at most.
template <class T, bool INPLACE>
cudaError_t run_process(ProcArgs a, cudaStream_t s) {
  const long long slices = (static_cast<long long>(a.vocab) + Vec<T>::N - 1 + kProcSlice - 1) / kProcSlice;
  long long per = std::max(1ll, std::min(8ll, a.rows * slices / (148 * 4 * 4)));
  a.part_cols = static_cast<int>(per) * kProcSlice;
  a.parts = static_cast<int>((slices + per - 1) / per);
  const long long grid = static_cast<long long>(a.rows) * a.parts;
  if (grid > INT_MAX) return cudaErrorInvalidConfiguration;
  const unsigned n = static_cast<unsigned>(grid);
  if (!a.hist && !a.bias) return launch_chained(process_kernel<T, false, INPLACE>, n, kProcThreads, 0, 1, s, a);
  const size_t smem = kProcSlice * 4u * (a.bias ? 2 : 1);
  return launch_chained(process_kernel<T, true, INPLACE>, n, kProcThreads, smem, 1, s, a);
}

// ============================================================== logprobs ==
// Log-probabilities, rank and the first columns of a row, one pass over it.
// A cluster of CTAs shares a row.  A thread keeps the maximum m of its columns
// and s = sum 2^(c (v - m)), c = log2(e) / temp.  In a batch the terms come from
// one fma each, 2^(c v + b) with b = -c m rounded; c v is exact inside the fma,
// so the rounding of b is one factor for the whole batch, 2^(-c m - b), which is
// multiplied back.
// The rank counts the columns v >= t, t the chosen value for columns before the
// chosen one and the next larger float for those after it.
// The first columns cost the pass nothing: of the threads' maxima, which it has
// anyway, a bound T is taken that `top` of them reach, so that `top` columns do;
// T is close to the `top`-th column itself, since two of the first columns
// seldom meet in one thread.  The few threads whose maximum reaches T have their
// columns read again (L2), and what reaches T is listed and ranked by counting.
// A list that overflows (ties) is gathered anew with a sharper bound.
constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 4;    // vectors per thread and batch
constexpr int kLpCap = 2048;  // listed columns per CTA
constexpr int kLpMaxCluster = 8;
constexpr float kLowest = -3.402823466e38f;

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
  // bm: the maximum of x[0, n), which may hold NaNs (they count as -inf)
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
    if (m == kNegInf) return;
    float t = 0.0f;
    if (fabsf(m) < 1e30f) {
      const float b = -m * c;
#pragma unroll
      for (int j = 0; j < n; ++j) t += ex2(fmaf(x[j], c, b));
      t *= ex2(fmaf(-m, c, -b));
    }
    // c m may overflow (rows masked with the type's lowest value), or a NaN was met
    if (!(fabsf(m) < 1e30f && t == t)) {
      t = 0.0f;
#pragma unroll
      for (int j = 0; j < n; ++j) t += ex2((fmaxf(x[j], kNegInf) - m) * c);
    }
    s += t;
  }
};

template <class T>
__device__ __forceinline__ uint4 all_neg_inf();
template <>
__device__ __forceinline__ uint4 all_neg_inf<float>() {
  return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
}
template <>
__device__ __forceinline__ uint4 all_neg_inf<__half>() {
  return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
}
template <>
__device__ __forceinline__ uint4 all_neg_inf<__nv_bfloat16>() {
  return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
}

template <class T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 2) logprob_kernel(const LogprobArgs a) {
  constexpr int N = Vec<T>::N, NV = kLpVecs, NT = kLpThreads;
  constexpr int SUB = 16 / N;  // vectors whose terms are summed together
  __shared__ LpPart parts[kLpWarps];
  __shared__ LpPart slots[kLpMaxCluster];  // the leader's: one per CTA
  __shared__ uint64_t slot_keys[TOP ? kLpMaxCluster * kLpMaxTop : 1];
  __shared__ uint64_t list[TOP ? kLpCap : 1];
  __shared__ uint64_t best[TOP ? kLpMaxTop : 1];
  __shared__ unsigned short hits[TOP ? NT : 1];
  __shared__ uint32_t offer[kLpWarps];
  __shared__ int count, nhits;
  __shared__ uint64_t bound_key;

  cg::cluster_group cl = cg::this_cluster();
  const int C = cl.num_blocks();
  const int rankc = cl.block_rank();
  if (C > 1) cluster_arrive();  // every CTA of the cluster has started before one writes to the leader
  grid_wait();
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* in = static_cast<const T*>(a.logits) + row * a.ld;
  const float c = 1.4426950408889634f / a.temp;
  const int top = a.top;
  // the row's aligned vectors [0, nvec) from column `head` on; the columns before
  // and after them go one to a thread of the first and of the last CTA
  const int head = min(a.vocab, (N - row_shift(in)) % N);
  const int nvec = (a.vocab - head) / N;
  const int tail = head + nvec * N;
  const int v0 = static_cast<int>(static_cast<long long>(nvec) * rankc / C);
  const int v1 = static_cast<int>(static_cast<long long>(nvec) * (rankc + 1) / C);
  const T* vin = in + head;
  int edge = -1;
  if (rankc == 0 && tid < head) edge = tid;
  if (rankc == C - 1 && tid >= N && tid - N < a.vocab - tail) edge = tail + tid - N;

  int id = -1;
  if (a.ids) {
    id = a.ids[row];
    if (id < 0 || id >= a.vocab) id = -1;
  }
  if (TOP && tid == 0) {
    count = 0;
    nhits = 0;
  }
  Vec<T> x[NV], y[NV];
  auto load = [&](int v, Vec<T>(&to)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (v + i * NT < v1)
        to[i].raw = ld_stream16(vin + static_cast<long long>(v + i * NT) * N);
      else
        to[i].raw = all_neg_inf<T>();
    }
  };
  load(v0 + tid, x);
  const float edge_value = edge >= 0 ? fmaxf(to_float(in[edge]), kNegInf) : kNegInf;
  // thresholds of the rank; nothing reaches a NaN
  const float nan = __uint_as_float(0x7fffffffu);
  float chosen = kNegInf, t_before = nan, t_after = nan;
  int before = 0;
  if (id >= 0) {
    chosen = fmaxf(to_float(in[id]), kNegInf) + 0.0f;  // a NaN counts as -inf, -0 as 0
    t_before = chosen;
    t_after = __uint_as_float(chosen >= 0.0f ? __float_as_uint(chosen) + 1u : __float_as_uint(chosen) - 1u);
    if (chosen == kNegInf) {  // every column before it counts, NaN and -inf among them
      t_before = nan;
      before = rankc == 0 && tid == 0 ? id : 0;
    }
  }

  LpAcc acc;
  for (int v = v0 + tid; v < v1; v += NV * NT) {
    if (v + NV * NT < v1) load(v + NV * NT, y);
#pragma unroll
    for (int i0 = 0; i0 < NV; i0 += SUB) {
      float e[SUB * N];
      float bm = kNegInf;
#pragma unroll
      for (int i = i0; i < i0 + SUB; ++i) {
        const int col = head + (v + i * NT) * N;
        const float t = col + N <= id ? t_before : t_after;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float w = x[i].get(j);
          e[(i - i0) * N + j] = w;
          bm = fmaxf(bm, w);
          before += w >= t;
        }
        if (col < id && id < col + N && v + i * NT < v1) {  // the chosen one's own vector: t_after does not count what is before it
          for (int j = 0; j < id - col; ++j) {
            const float w = to_float(in[col + j]);
            before += chosen > kNegInf ? w == chosen : -(w >= t_after);
          }
        }
      }
      acc.add(e, bm, c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = y[i];
  }
  if (edge >= 0) {
    const float e[1] = {edge_value};
    before += edge < id ? edge_value >= t_before : edge_value >= t_after;
    acc.add(e, edge_value, c);
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

  int ntop = 0;
  if (TOP) {
    // Every warp offers the q-th largest of its maxima: q * kLpWarps >= top
    // maxima reach the lowest offer.  From there the bound is raised by halving
    // while `top` maxima still reach it.
    const uint32_t mine = ord32(acc.m + 0.0f);
    uint32_t o = mine;
    uint32_t w = __reduce_max_sync(0xffffffffu, o);
    if (top > kLpWarps) {
      const unsigned at = __ballot_sync(0xffffffffu, o == w);
      if (lane == __ffs(at) - 1) o = 0;
      w = __reduce_max_sync(0xffffffffu, o);
    }
    if (lane == 0) offer[warp] = w;
    __syncthreads();
    const uint32_t least = ord32(kLowest);  // a column at -inf is never listed
    uint32_t low = offer[lane % kLpWarps];
    uint32_t high = ord32(parts[lane % kLpWarps].m);
    low = max(__reduce_min_sync(0xffffffffu, low), least);
    high = __reduce_max_sync(0xffffffffu, high);
    for (int it = 0; it < 16 && low < high; ++it) {
      const uint32_t mid = low + (high - low + 1) / 2;
      const int n = __syncthreads_count(mine >= mid);
      if (n >= top) {
        low = mid;
        if (n <= top + 4) break;
      } else {
        high = mid - 1;
      }
    }
    const float thr = unord32(low);
    if (mine >= low) hits[atomicAdd(&nhits, 1)] = static_cast<unsigned short>(tid);
    if (edge_value >= thr) list[atomicAdd(&count, 1)] = dkey(edge_value, edge);
    __syncthreads();
    const int per = (v1 - v0 + NT - 1) / NT;  // vectors of a thread
    for (int i = tid; i < nhits * per; i += NT) {
      const int h = i / per;
      const int v = v0 + (i - h * per) * NT + hits[h];
      if (v >= v1) continue;
      Vec<T> r;
      r.raw = *reinterpret_cast<const uint4*>(vin + static_cast<long long>(v) * N);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (r.get(j) >= thr) {
          const int at = atomicAdd(&count, 1);
          if (at < kLpCap) list[at] = dkey(r.get(j), head + v * N + j);
        }
    }
    __syncthreads();
    int n = count;
    // Too many: the `top`-th of those that were kept is a bound that as many
    // columns reach; gather again from it on, in the order of the keys (distinct,
    // so at least kLpCap - top columns drop out each time).
    while (n > kLpCap) {
      for (int i = tid; i < kLpCap; i += NT) {
        int r = 0;
        const uint64_t k = list[i];
        for (int j = 0; j < kLpCap; ++j) r += list[j] < k;
        if (r == top - 1) bound_key = k;
      }
      __syncthreads();
      const uint64_t bk = bound_key;
      if (tid == 0) count = 0;
      __syncthreads();
      const int lo = rankc == 0 ? 0 : head + v0 * N, hi = rankc == C - 1 ? a.vocab : head + v1 * N;
      for (int col = lo + tid; col < hi; col += NT) {
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
    for (int i = tid; i < n; i += NT) {
      int r = 0;
      const uint64_t k = list[i];
      for (int j = 0; j < n; ++j) r += list[j] < k;
      if (r < top) best[r] = k;
    }
  }
  __syncthreads();

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
    for (int i = tid; i < C * top; i += NT) {
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
    for (int i = have + tid; i < top; i += NT) {
      a.top_ids[static_cast<long long>(row) * top + i] = -1;
      a.top_logprobs[static_cast<long long>(row) * top + i] = kNegInf;
    }
  }
}

template <class T>
cudaError_t run_logprobs(LogprobArgs a, cudaStream_t s) {
  constexpr int N = Vec<T>::N;
  // enough CTAs for the SMs, in slices of a batch or more
  int C = 1;
  while (C < kLpMaxCluster && static_cast<long long>(C) * kLpThreads * kLpVecs * N < a.vocab &&
         static_cast<long long>(a.rows) * C < 148 * 4)
    C <<= 1;
  const long long grid = static_cast<long long>(a.rows) * C;
  if (grid > INT_MAX) return cudaErrorInvalidConfiguration;
  return a.top > 0 ? launch_chained(logprob_kernel<T, true>, static_cast<unsigned>(grid), kLpThreads, 0, C, s, a)
                   : launch_chained(logprob_kernel<T, false>, static_cast<unsigned>(grid), kLpThreads, 0, C, s, a);
}

}  // namespace

cudaError_t launch_process(ProcArgs a, int dtype, bool in_place, cudaStream_t s) {
  if (dtype == kOpsF16) return run_process<__half, false>(a, s);
  if (dtype == kOpsBF16) return run_process<__nv_bfloat16, false>(a, s);
  return in_place ? run_process<float, true>(a, s) : run_process<float, false>(a, s);
}

cudaError_t launch_logprobs(LogprobArgs a, int dtype, cudaStream_t s) {
  if (dtype == kOpsF16) return run_logprobs<__half>(a, s);
  if (dtype == kOpsBF16) return run_logprobs<__nv_bfloat16>(a, s);
  return run_logprobs<float>(a, s);
}

}  // namespace vb
