// Logits operators around the sampler (include/verbo_ops.h): penalties, biases
// and masks before the pick, log-probabilities after it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <type_traits>

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

// Not the read-only path: a kernel that is launched programmatically has begun
// before the grid whose rows it reads has ended.
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_word(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
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
//
// The bound is memory: the row in, the row out, the mask's bits.  Four CTAs of 256
// threads per SM with 16 columns per thread on their way; a slice of 4096 columns
// has 16 KB of counters, so that lists cost no occupancy.  Measured on B200: 512
// fp32 rows of 151936 with up to 1024 ids each 111 us, 5.6 TB/s (86% of the card's
// copy rate); 256 bf16 rows with ids, biases and masks 49 us, 4.9 TB/s.  One slice
// per CTA and the window read again for each took 160 and 92 us.
// 512 rows masked in place, a third of them free, a third nearly and a third with
// few columns left, take 48 us: 25 to look through the masks (issue slots 72%
// busy), the rest for the stores.  Those of masked columns beside allowed ones are
// 4 bytes each: half of all columns masked at random takes 206 us, all of them 59.
// The window's ids beyond the first 1024 are read again for each slice: 64 rows with
// 32768 ids each take 70 us.
constexpr int kProcThreads = 256;
constexpr int kProcCols = 16;                         // columns per thread and slice
constexpr int kProcSlice = kProcThreads * kProcCols;  // 4096
constexpr int kProcHist = 4, kProcBias = 1;           // ids per thread in registers

template <class T, bool LISTS, bool INPLACE>
__global__ void __launch_bounds__(kProcThreads, !LISTS && INPLACE ? 8 : 4) process_kernel(const ProcArgs a) {
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
          ml[i] = ld_word(w);
          mh[i] = (c & 31) + N > 32 ? ld_word(w + 1) : 0u;
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
          const bool allowed = !mask || ((mask[(c + j) >> 5] >> ((c + j) & 31)) & 1u);
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
  long long per = std::max(1ll, std::min(8ll, a.rows * slices / (sm_count() * 4 * 4)));
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
// The first columns cost the pass little: of the threads' maxima, which it has
// anyway, a bound T is taken that `top` of them reach, so that `top` columns do;
// T is close to the `top`-th column itself, since two of the first columns
// seldom meet in one thread.  The few batches whose maximum reaches T (kept in
// shared memory) are read again, from L2, and what reaches T is listed and
// ranked by counting.  A list that overflows (ties) is gathered anew with a
// sharper bound.
// Each thread copies its own vectors to shared memory (cp.async), two batches
// ahead, and reads them back itself: no registers for what is in flight and no
// barrier in the pass.
//
// Measured on B200: 512 fp32 rows of 151936 in 53 us, 5.9 TB/s (90% of the card's
// copy rate).  256 bf16 rows with the 20 first take 26 us, 3.0 TB/s: about ten
// instructions a column and an exponential unit of 16 lanes (9 us alone) bound it,
// and 256 rows leave 40 of 148 SMs half empty; two CTAs a row (a cluster's
// barriers, every first column found twice) take 34.7.  Clusters serve the few rows
// that would leave SMs without work: one row of 49152 with the 5 first 9.2 us, 5.4
// without them.
constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 4;    // vectors per thread and batch
constexpr int kLpStages = 2;  // batches in flight
constexpr int kLpGroups = 8;  // batches whose maxima are kept (the last: of all that follow)
constexpr int kLpCap = 1024;  // listed columns per CTA
constexpr int kLpOffers = 4;  // maxima a warp offers at most
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

// A value in T's own bits: the chosen column's, canonical (NaN as -inf, -0 as
// 0), and the next larger value (of +inf: a NaN, which nothing reaches).
template <class T>
struct Bits;
template <>
struct Bits<float> {
  using U = uint32_t;
  static constexpr U kSign = 0x80000000u, kInf = 0x7f800000u, kNan = 0x7fffffffu;
};
template <>
struct Bits<__half> {
  using U = uint16_t;
  static constexpr U kSign = 0x8000u, kInf = 0x7c00u, kNan = 0x7fffu;
};
template <>
struct Bits<__nv_bfloat16> {
  using U = uint16_t;
  static constexpr U kSign = 0x8000u, kInf = 0x7f80u, kNan = 0x7fffu;
};
template <class T>
__device__ __forceinline__ typename Bits<T>::U canon_bits(typename Bits<T>::U u) {
  using B = Bits<T>;
  if ((u & ~B::kSign) > B::kInf) return B::kSign | B::kInf;
  return u == B::kSign ? 0 : u;
}
template <class T>
__device__ __forceinline__ typename Bits<T>::U next_up(typename Bits<T>::U u) {
  return u & Bits<T>::kSign ? u - 1 : u + 1;
}

// NV vectors of one thread.
template <class T, int NV>
struct LpBatch {
  static constexpr int N = Vec<T>::N;
  Vec<T> x[NV];
  __device__ __forceinline__ const uint32_t& word(int i) const {  // i in [0, 4 NV)
    const uint4& r = x[i >> 2].raw;
    return (i & 3) == 0 ? r.x : (i & 3) == 1 ? r.y : (i & 3) == 2 ? r.z : r.w;
  }
  __device__ __forceinline__ float max() const {  // NaNs left out
    if constexpr (sizeof(T) == 4) {
      float m = kNegInf;
#pragma unroll
      for (int i = 0; i < 4 * NV; ++i) m = fmaxf(m, __uint_as_float(word(i)));
      return m;
    } else if constexpr (std::is_same_v<T, __half>) {
      uint32_t m = 0xfc00fc00u;
#pragma unroll
      for (int i = 0; i < 4 * NV; ++i) asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(word(i)));
      const __half2 h = *reinterpret_cast<const __half2*>(&m);
      return fmaxf(__low2float(h), __high2float(h));
    } else {
      uint32_t m = 0xff80ff80u;
#pragma unroll
      for (int i = 0; i < 4 * NV; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(word(i)));
      return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
  }
  // how many of vector i's values reach the value of bits u
  template <int I0, int I1>
  __device__ __forceinline__ int reach(typename Bits<T>::U u) const {
    if constexpr (sizeof(T) == 4) {
      int n = 0;
#pragma unroll
      for (int i = 4 * I0; i < 4 * I1; ++i) n += __uint_as_float(word(i)) >= __uint_as_float(u);
      return n;
    } else if constexpr (std::is_same_v<T, __half>) {
      const uint32_t t = u | static_cast<uint32_t>(u) << 16;
      __half2 n = __floats2half2_rn(0.0f, 0.0f);  // counts up to 4 NV: exact
#pragma unroll
      for (int i = 4 * I0; i < 4 * I1; ++i)
        n = __hadd2(n, __hge2(*reinterpret_cast<const __half2*>(&word(i)), *reinterpret_cast<const __half2*>(&t)));
      return static_cast<int>(__low2float(n) + __high2float(n));
    } else {
      const uint32_t t = u | static_cast<uint32_t>(u) << 16;
      __nv_bfloat162 n = __floats2bfloat162_rn(0.0f, 0.0f);
#pragma unroll
      for (int i = 4 * I0; i < 4 * I1; ++i)
        n = __hadd2(n, __hge2(*reinterpret_cast<const __nv_bfloat162*>(&word(i)),
                              *reinterpret_cast<const __nv_bfloat162*>(&t)));
      return static_cast<int>(__low2float(n) + __high2float(n));
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) f(x[i].get(j), j);
  }
};

struct LpAcc {
  float m = kNegInf, s = 0.0f;
  int ninf = 0;
  // bm: the maximum of the batch b, which may hold NaNs (they count as -inf)
  template <class B>
  __device__ __forceinline__ void add(const B& b, float bm, float c) {
    if (bm > m) {
      s = lp_scaled(s, m, bm, c);
      m = bm;
    }
    if (fabsf(m) < -kNegInf) {
      // fma(c, m, o) is the rounding of c m, exactly, and at most 2^6 below 2^31:
      // neither 2^(c v + o) nor the factor that takes it back leaves fp32's range.
      // A larger c m (rows masked with large finite values) counts the columns at m:
      // one step of fp32 below it (2^-24 |m| at least) is a factor of 2^-128.  So
      // does the power of two that takes |m| to [2^30, 2^31), where it is 2^-64.
      float k = c;
      if (fabsf(m * c) >= 2147483648.0f)
        k = __uint_as_float((284u << 23) - (__float_as_uint(m) & 0x7f800000u));
      const float o = -m * k;
      float t[2] = {0.0f, 0.0f};
      b.each([&](float v, int j) { t[j & 1] += ex2(fmaf(v, k, o)); });
      t[0] = (t[0] + t[1]) * ex2(fmaf(-m, k, -o));
      if (t[0] != t[0]) {  // rare: a NaN was met
        t[0] = 0.0f;
        b.each([&](float v, int) { t[0] += ex2((fmaxf(v, kNegInf) - m) * c); });
      }
      s += t[0];
    } else if (m == -kNegInf) {  // +inf alone counts then
      b.each([&](float v, int) { ninf += v == -kNegInf; });
    }
  }
};
struct LpOne {  // a single column
  float v;
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    f(v, 0);
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
  constexpr int N = Vec<T>::N, NT = kLpThreads, NV = kLpVecs;
  extern __shared__ __align__(16) uint4 ring[];  // [kLpStages][NV][NT]
  __shared__ LpPart parts[kLpWarps];
  __shared__ LpPart slots[kLpMaxCluster];  // the leader's: one per CTA
  __shared__ uint64_t slot_keys[TOP ? kLpMaxCluster * kLpMaxTop : 1];
  __shared__ uint64_t list[TOP ? kLpCap : 1];
  __shared__ uint64_t best[TOP ? kLpMaxTop : 1];
  __shared__ float group_max[TOP ? kLpGroups * NT : 1];
  __shared__ unsigned short hits[TOP ? kLpGroups * NT : 1];  // group * NT + thread
  __shared__ __align__(16) uint32_t offer[kLpWarps * kLpOffers];
  __shared__ int count, nhits;
  __shared__ uint32_t bound;
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
  const int nfull = (v1 - v0) / (NV * NT), rest = v1 - v0 - nfull * (NV * NT);
  const int nbatch = nfull + (rest > 0 ? 1 : 0);
  const T* next = vin + static_cast<long long>(v0 + tid) * N;  // of the batch to be copied next
  auto fetch = [&](int b) {
    uint4* to = ring + (b % kLpStages) * (NV * NT) + tid;
    if (b < nfull) {
#pragma unroll
      for (int i = 0; i < NV; ++i) cp_async16(to + i * NT, next + i * NT * N);
    } else if (b < nbatch) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid + i * NT < rest) cp_async16(to + i * NT, next + i * NT * N);
    }
    next += NV * NT * N;
    cp_async_commit();  // an empty group keeps the count
  };
#pragma unroll
  for (int b = 0; b < kLpStages; ++b) fetch(b);
  const float edge_value = edge >= 0 ? fmaxf(to_float(in[edge]), kNegInf) : kNegInf;
  // thresholds of the rank
  using U = typename Bits<T>::U;
  float chosen = kNegInf;
  U t_before = Bits<T>::kNan, t_after = Bits<T>::kNan;
  int before = 0;
  if (id >= 0) {
    t_before = canon_bits<T>(reinterpret_cast<const U*>(in)[id]);
    t_after = next_up<T>(t_before);
    const U bits = t_before;
    chosen = to_float(*reinterpret_cast<const T*>(&bits));
    if (chosen == kNegInf) {  // every column before it counts, NaN and -inf among them
      t_before = Bits<T>::kNan;
      before = rankc == 0 && tid == 0 ? id : 0;
    }
  }

  LpAcc acc;
  for (int b = 0; b < nbatch; ++b) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLpStages - 1) : "memory");
    LpBatch<T, NV> x;
    const uint4* from = ring + (b % kLpStages) * (NV * NT) + tid;
#pragma unroll
    for (int i = 0; i < NV; ++i) x.x[i].raw = from[i * NT];
    if (b >= nfull) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid + i * NT >= rest) x.x[i].raw = all_neg_inf<T>();
    }
    fetch(b + kLpStages);
    const float bm = x.max();
    const int col0 = head + (v0 + b * (NV * NT)) * N;
    if (id < col0) {
      before += x.template reach<0, NV>(t_after);
    } else if (id >= col0 + NV * NT * N) {
      before += x.template reach<0, NV>(t_before);
    } else {  // the batch that holds the chosen one
      auto vector = [&](auto i) {
        constexpr int I = decltype(i)::value;
        const int col = col0 + (I * NT + tid) * N;
        before += x.template reach<I, I + 1>(col + N <= id ? t_before : t_after);
        // its vector: t_after does not count what is before it
        if (col < id && id < col + N && I * NT + tid < v1 - v0 - b * (NV * NT)) {
          for (int j = 0; j < id - col; ++j) {
            const float w = to_float(in[col + j]);
            before += chosen > kNegInf ? w == chosen : -(w > kNegInf);
          }
        }
      };
      vector(std::integral_constant<int, 0>{});
      vector(std::integral_constant<int, 1>{});
      vector(std::integral_constant<int, 2>{});
      vector(std::integral_constant<int, 3>{});
      static_assert(NV == 4, "one call per vector");
    }
    acc.add(x, bm, c);
    if (TOP) {
      float* at = &group_max[min(b, kLpGroups - 1) * NT + tid];
      *at = b < kLpGroups ? bm : fmaxf(*at, bm);
    }
  }
  if (edge >= 0) {
    const U u = canon_bits<T>(reinterpret_cast<const U*>(in)[edge]);
    const float t = to_float(*reinterpret_cast<const T*>(edge < id ? &t_before : &t_after));
    before += to_float(*reinterpret_cast<const T*>(&u)) >= t;
    acc.add(LpOne{edge_value}, edge_value, c);
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
  LpPart sum;  // in warp 0
  auto total = [&]() {
    const LpPart w = lane < kLpWarps ? parts[lane] : LpPart{kNegInf, 0.0f, 0, 0, 0};
    sum.m = unord32(__reduce_max_sync(0xffffffffu, ord32(w.m + 0.0f)));
    sum.s = lp_scaled(w.s, w.m, sum.m, c);
#pragma unroll
    for (int o = kLpWarps / 2; o > 0; o >>= 1) sum.s += __shfl_xor_sync(0xffffffffu, sum.s, o);
    sum.rank = __reduce_add_sync(0xffffffffu, w.rank);
    sum.ninf = __reduce_add_sync(0xffffffffu, w.ninf);
  };

  int ntop = 0;
  if (TOP) {
    // Every warp offers its q largest maxima; the `top`-th of all offers is the
    // bound (q * kLpWarps >= top of them, each of another thread).
    const uint32_t mine = ord32(acc.m + 0.0f);
    const int q = min(kLpOffers, 2 * ((top + kLpWarps - 1) / kLpWarps));
    uint32_t o = mine;
    for (int i = 0; i < q; ++i) {
      const uint32_t w = __reduce_max_sync(0xffffffffu, o);
      const unsigned at = __ballot_sync(0xffffffffu, o == w);
      if (lane == __ffs(at) - 1) {
        offer[warp * q + i] = w;
        o = 0;
      }
    }
    __syncthreads();
    if (warp == 0) total();
    // the bound: an offer with fewer than `top` above it and `top` at or above it
    if (tid >= 32 && tid < 32 + q * kLpWarps) {
      const uint32_t w = offer[tid - 32];
      int gt = 0, ge = 0;
#pragma unroll 4
      for (int j = 0; j < q * kLpWarps; j += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(offer + j);
        gt += (v.x > w) + (v.y > w) + (v.z > w) + (v.w > w);
        ge += (v.x >= w) + (v.y >= w) + (v.z >= w) + (v.w >= w);
      }
      if (gt < top && top <= ge) bound = max(w, ord32(kLowest));  // a column at -inf is never listed
    }
    __syncthreads();
    const uint32_t low = bound;
    const float thr = unord32(low);
    if (mine >= low) {
      for (int g = 0; g < min(nbatch, kLpGroups); ++g)
        if (group_max[g * NT + tid] >= thr) hits[atomicAdd(&nhits, 1)] = static_cast<unsigned short>(g * NT + tid);
      if (edge_value >= thr) list[atomicAdd(&count, 1)] = dkey(edge_value, edge);
    }
    __syncthreads();
    const int lastn = max(1, nbatch - kLpGroups + 1);  // batches of the last group
    for (int i = tid; i < nhits * (NV * lastn); i += NT) {
      const int h = lastn == 1 ? i / NV : i / (NV * lastn);
      const int k = i - h * (NV * lastn);
      const int g = hits[h] / NT;
      if (k >= NV && g < kLpGroups - 1) continue;
      const int v = v0 + (g * NV + k) * NT + hits[h] % NT;
      if (v >= v1) continue;
      Vec<T> r;
      if (nbatch <= kLpStages)  // still in the ring
        r.raw = ring[(g * NV + k) * NT + hits[h] % NT];
      else
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

  if (!TOP && warp == 0) total();
  sum.ntop = ntop;
  if (C > 1) {
    cluster_wait();
    if (tid == 0) *cl.map_shared_rank(&slots[rankc], 0) = sum;
    if (TOP && tid < ntop) *cl.map_shared_rank(&slot_keys[rankc * kLpMaxTop + tid], 0) = best[tid];
    cluster_sync_all();
    if (rankc != 0) return;
  } else {
    if (tid == 0) slots[0] = sum;
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
    // halves: the difference of two large values of opposite sign stays finite
    return __fdiv_rn(0.5f * v - 0.5f * m, 0.5f * a.temp) - ls;
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
  // CTAs per row: one, or as many as give each SM one, with a batch each.
  const long long batches = (a.vocab / N + kLpThreads * kLpVecs - 1) / (kLpThreads * kLpVecs);
  const int sms = sm_count();
  int C = 1;
  while (C < kLpMaxCluster && C < batches && static_cast<long long>(a.rows) * C < sms) C <<= 1;
  const long long grid = static_cast<long long>(a.rows) * C;
  if (grid > INT_MAX) return cudaErrorInvalidConfiguration;
  constexpr int smem = kLpStages * kLpVecs * kLpThreads * 16;  // 64 KB
  const auto kernel = a.top > 0 ? logprob_kernel<T, true> : logprob_kernel<T, false>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_chained(kernel, static_cast<unsigned>(grid), kLpThreads, smem, C, s, a);
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
