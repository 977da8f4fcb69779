// Beam search's operators (include/verbo_beam.h): the best continuations of each
// request's beams, and the beams' states in the order of the chosen parents.
#include <climits>
#include <type_traits>

#include "beam.cuh"
#include "device.cuh"
#include "ops.cuh"
#include "opsdev.cuh"

namespace vb {
namespace {

// ================================================================ select ==
// value(b, i) = score[b] + (x[b][i] - lse[b]),  lse[b] = m + log sum_j e^(x[b][j] - m)
//
// Two beams' candidates are ordered by their values, so the sums have to be exact
// to below the distance of two candidates.  What makes up a row is its largest column: it
// is a 1 that is added in 64 bits, and the others' terms are seen from it.  Those are fp32
// (the factor log2(e) is taken in two parts, so a term is off by the roundings of x - m and of
// its product, 2^-23 |x - m| of itself, and by the exponential's 2^-22), eight to sixteen of them are
// added in fp32 and the rest in 64 bits.  Measured, lse is off by up to 6e-8: 4.5e-8 where
// thousands of columns share the row (the exponential is low by as much in the mean), 1e-8
// with deviations of 6, below 1e-9 where one column stands out by 10.  With a term of the first
// batch's maximum in the place of the 1, and fp32 sums, it was up to 3e-6.  A sum goes by
// the columns alone, not by where a row lies in memory: equal rows have equal sums
// to the last bit, and equal candidates are ordered by their beams.
//
// One pass over a row finds the sum and its first `take` columns (the bound from
// the threads' maxima, as in logprob_kernel); a cluster of CTAs shares a row where
// the rows are few.  A second, small kernel joins the beams of a request: a lane
// keeps the head of a beam's list, and the largest is taken `take` times.
//
// Measured on B200: 512 bf16 rows of 151936 with 16 taken 42 us, 3.7 TB/s: the exponential
// unit (16 lanes) is busy 57% of the time, issue slots 56%; fp32 65 us, 4.8 TB/s: 512 rows
// on 592 places leave SMs three or four.  CTAs of 512 threads, two to an SM, took 48 and 62;
// two CTAs to a row of a large batch 45 and 65.  One row of 49152 13 us, most of it
// round trips and barriers.
constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelVecs = 4;                         // vectors per thread and batch
constexpr int kSelStages = 2;                       // batches in flight
constexpr int kSelWarpVecs = kSelVecs * 32;         // a warp's vectors lie side by side
constexpr int kSelSlots = kSelWarpVecs + 1;         // one more for rows off the 16-byte grid
constexpr int kSelGroups = 8;  // groups of batches whose maxima are kept
constexpr int kSelCap = 512;  // listed columns per CTA
constexpr int kSelOffers = 32;  // maxima a warp offers at most
constexpr int kSelMaxCluster = 8;
constexpr float kSelLowest = -3.402823466e38f;
// log2(e) = kLog2eHi + kLog2eLo to 2^-49
constexpr double kLog2e = 1.4426950408889634;
constexpr float kLog2eHi = static_cast<float>(kLog2e);
constexpr float kLog2eLo = static_cast<float>(kLog2e - static_cast<double>(kLog2eHi));

// What a row leaves for the second kernel, before its keys.
struct SelRow {
  double lse;  // of a row with columns at +inf: the logarithm of their number
  int n;       // keys
  int inf;
};

struct SelPart {
  double s;  // sum of e^(x - m)
  float m;   // the reference
  int ninf;
};

__device__ __forceinline__ void cp_async16_part(void* dst, const void* src, int bytes) {  // the rest is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

template <class T>
struct SelBatch {
  static constexpr int N = Vec<T>::N, NV = kSelVecs;
  Vec<T> x[NV];
  __device__ __forceinline__ uint32_t word(int i) const {  // i in [0, 4 NV)
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
  // sum of e^(x - ref), NaNs left out
  __device__ __forceinline__ double sum(float ref) const {
    const Two away = two(-ref, -ref), c_hi = two(kLog2eHi, kLog2eHi), c_lo = two(kLog2eLo, kLog2eLo);
    Two t[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
#pragma unroll
    for (int i = 0; i < NV * N; i += 2) {
      const Two d = add2(two(x[i / N].get(i % N), x[i / N].get(i % N + 1)), away);
      const float2 e = parts_of(fma2(d, c_hi, mul2(d, c_lo)));
      t[i / 2 % 2] = add2(t[i / 2 % 2], two(ex2(e.x), ex2(e.y)));
    }
    const float2 p = parts_of(add2(t[0], t[1]));
    double s = static_cast<double>(p.x) + static_cast<double>(p.y);
    if (s != s) {  // rare: a NaN was met
      s = 0.0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float d = fmaxf(x[i].get(j), kNegInf) - ref;
          s += static_cast<double>(ex2(fmaf(d, kLog2eHi, d * kLog2eLo)));
        }
    }
    return s;
  }
  // How many columns are at v; they are at -inf after it.
  __device__ __forceinline__ int take_out(float v) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t w[4] = {x[i].raw.x, x[i].raw.y, x[i].raw.z, x[i].raw.w};
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (x[i].get(j) == v) {
          ++n;
          if constexpr (N == 4)
            w[j] = 0xff800000u;
          else
            w[j / 2] = j % 2 ? (w[j / 2] & 0xffffu) | (all_neg_inf<T>().x & 0xffff0000u)
                             : (w[j / 2] & 0xffff0000u) | (all_neg_inf<T>().x & 0xffffu);
        }
      x[i].raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return n;
  }
  __device__ __forceinline__ int count_inf() const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) n += x[i].get(j) == -kNegInf;
    return n;
  }
};

__device__ __forceinline__ double shfl_xor_double(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// A sum of e^(x - from), seen from another reference.
__device__ __forceinline__ double sel_scaled(double s, float from, float m) {
  return from == m || !(s > 0.0) ? s : s * exp(static_cast<double>(from) - static_cast<double>(m));
}

// SHIFT: a row need not begin on the 16-byte grid; a thread joins its vector from
// two that its warp copied.
template <class T, bool SHIFT>
__global__ void __launch_bounds__(kSelThreads, 4) beam_rows_kernel(const BeamSelectArgs a) {
  constexpr int N = Vec<T>::N, NT = kSelThreads, NV = kSelVecs, SLOTS = SHIFT ? kSelSlots : kSelWarpVecs;
  extern __shared__ __align__(16) uint4 ring[];  // [kSelStages][kSelWarps][SLOTS]
  __shared__ SelPart parts[kSelWarps];
  __shared__ SelPart slots[kSelMaxCluster];  // the leader's: one per CTA
  __shared__ int slot_n[kSelMaxCluster];
  __shared__ uint64_t slot_keys[kSelMaxCluster * kBeamMaxTake];
  __shared__ uint64_t list[kSelCap];
  __shared__ uint64_t best[kBeamMaxTake];
  __shared__ float group_max[kSelGroups * NT];
  __shared__ unsigned short hits[kSelGroups * NT];  // group * NT + thread
  __shared__ __align__(16) uint32_t offer[kSelWarps * kSelOffers];
  __shared__ uint32_t first_max[kSelWarps];
  __shared__ int count, nhits;
  __shared__ uint32_t bound;
  __shared__ uint64_t bound_key;

  cg::cluster_group cl = cg::this_cluster();
  const int C = cl.num_blocks();
  const int rankc = cl.block_rank();
  if (C > 1) cluster_arrive();  // every CTA of the cluster has started before one writes to the leader
  const int row = blockIdx.x >> (__ffs(C) - 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    count = 0;
    nhits = 0;
    bound = 0xffffffffu;
  }
  grid_wait();
  grid_release();
  const int top = a.take;
  const T* in = static_cast<const T*>(a.logits) + row * a.ld;
  const float score = a.scores[row];
  const int shift = SHIFT ? static_cast<int>(reinterpret_cast<uintptr_t>(in) & 15) : 0;  // bytes
  const char* grid = reinterpret_cast<const char*>(in) - shift;
  const long long last = static_cast<long long>(a.vocab) * sizeof(T) + shift;  // the row's end, from `grid`
  // vectors are counted by columns, whatever the row's place
  const int nvec = (a.vocab + N - 1) / N;
  const int cbits = __ffs(C) - 1;  // C is a power of two, and eight times the vectors are below 2^31
  const int v0 = nvec * rankc >> cbits;
  const int v1 = nvec * (rankc + 1) >> cbits;
  // vectors of a thread and batch: fewer where a part is short, so that all warps have some
  const int nv = min(NV, (v1 - v0 + NT - 1) / NT);
  const int step = nv * NT, mine0 = warp * nv * 32;  // of a batch; this warp's place in one
  int nbatch = nv == NV ? (v1 - v0 + NV * NT - 1) / (NV * NT) : v1 > v0;
  // batches of whole vectors: neither they nor, off the grid, the 16 bytes after them
  // reach the row's end
  const int whole = nv == NV ? (v1 - v0 - (SHIFT ? 2 : rankc == C - 1 && a.vocab % N ? 1 : 0)) / (NV * NT) : 0;

  auto copy = [&](uint4* to, int v) {  // the 16 bytes at v of the row's grid
    const long long at = static_cast<long long>(v) * 16;
    const int bytes = static_cast<int>(last - at < 16 ? (last - at > 0 ? last - at : 0) : 16);
    if (SHIFT && v == 0) {  // what lies before the row is not read
      T* t = reinterpret_cast<T*>(to);
      const int first = shift / static_cast<int>(sizeof(T));
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j >= first && j * static_cast<int>(sizeof(T)) < bytes) t[j] = in[j - first];
    } else {
      cp_async16_part(to, bytes > 0 ? grid + at : grid + 16 * (v0 + 1) - 16, bytes);
    }
  };
  const char* next = grid + (static_cast<long long>(v0) + mine0 + lane) * 16;  // of the batch to be copied next
  auto fetch = [&](int b) {
    uint4* to = ring + ((b % kSelStages) * kSelWarps + warp) * SLOTS;
    if (b < whole && !(SHIFT && v0 == 0 && b == 0)) {
#pragma unroll
      for (int i = 0; i < NV; ++i) cp_async16(to + i * 32 + lane, next + i * 512);
      if (SHIFT && lane == 0) cp_async16(to + kSelWarpVecs, next + kSelWarpVecs * 16);
    } else if (b < nbatch) {
      const int v = v0 + b * step + mine0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i < nv && v + i * 32 + lane < v1 + (SHIFT ? 1 : 0)) copy(to + i * 32 + lane, v + i * 32 + lane);
      if (SHIFT && lane == 0 && v + nv * 32 < v1 + 1) copy(to + nv * 32, v + nv * 32);
    }
    next += kSelVecs * NT * 16;
    cp_async_commit();  // an empty group keeps the count
  };
#pragma unroll
  for (int b = 0; b < kSelStages; ++b) fetch(b);
  if (!(score > kNegInf)) nbatch = 0;  // no candidates (the same in the whole cluster): nothing else is read

  const int per_group = max(1, (nbatch + kSelGroups - 1) / kSelGroups);
  float ref = kNegInf, mx = kNegInf, gm = kNegInf;
  double sum = 0.0;
  int ninf = 0, group = 0, in_group = 0;
  for (int b = 0; b < nbatch; ++b) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kSelStages - 1) : "memory");
    if (SHIFT) __syncwarp();
    SelBatch<T> x;
    const uint4* from = ring + ((b % kSelStages) * kSelWarps + warp) * SLOTS + lane;
    const int vb = v0 + b * step + mine0 + lane;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (SHIFT) {
        const uint4 p = from[i * 32], q = from[i * 32 + 1];
        uint32_t w[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
        if (shift & 8) {
#pragma unroll
          for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
        }
        if (shift & 4) {
#pragma unroll
          for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
        }
        const int bits = (shift & 3) * 8;
        x.x[i].raw = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                                __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
      } else {
        x.x[i].raw = from[i * 32];
      }
    }
    if (b >= whole) {  // the row's last, short vector, and what lies behind the part
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = vb + i * 32;
        if (i >= nv || v >= v1) {
          x.x[i].raw = all_neg_inf<T>();
        } else if (v == nvec - 1 && a.vocab % N) {
          const int have = a.vocab % N;
          const uint4 r = x.x[i].raw, none = all_neg_inf<T>();
          uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            constexpr int P = N / 4;  // columns of a word
            if (j * P >= have)
              w[j] = none.x;
            else if (P == 2 && j * P + 1 >= have)
              w[j] = (w[j] & 0xffffu) | (none.x & 0xffff0000u);
          }
          x.x[i].raw = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (SHIFT) __syncwarp();
    fetch(b + kSelStages);
    const float bm = x.max();
    mx = fmaxf(mx, bm);
    if (b == 0) {
      const uint32_t w = __reduce_max_sync(0xffffffffu, ord32(bm + 0.0f));
      if (lane == 0) first_max[warp] = w;
      __syncthreads();
      ref = unord32(__reduce_max_sync(0xffffffffu, lane < kSelWarps ? first_max[lane] : 0u));
      if (ref == -kNegInf) ref = kNegInf;
    }
    if (bm == -kNegInf) {
      ninf += x.count_inf();
    } else if (bm > kNegInf) {
      // The sum is seen from the largest column so far or one that is less than 1 below it: the
      // CTA's of the first batch, then the thread's own.  That column is a 1 added in 64 bits:
      // where it makes up the row, no fp32 rounding is left in the sum.
      const float up = bm - ref;
      if (up > 1.0f || (b == 0 && up == 0.0f)) {
        sum = sel_scaled(sum, ref, bm);
        ref = bm;
        sum += x.take_out(bm);
      }
      sum += x.sum(ref);
    }
    gm = fmaxf(gm, bm);
    if (++in_group == per_group || b == nbatch - 1) {
      group_max[group * NT + tid] = gm;
      gm = kNegInf;
      in_group = 0;
      ++group;
    }
  }

  cp_async_wait_all();  // a row without candidates has copies under way

  // the CTA's part of the row: sums of one reference are added as they are
  SelPart p;
  p.m = unord32(__reduce_max_sync(0xffffffffu, ord32(ref + 0.0f)));
  p.s = sel_scaled(sum, ref, p.m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) p.s += shfl_xor_double(p.s, o);
  p.ninf = __reduce_add_sync(0xffffffffu, ninf);
  if (lane == 0) parts[warp] = p;

  // Every warp offers its q largest maxima; the `top`-th of all offers is the
  // bound: `top` columns reach it, each of another thread.  The warps that have
  // columns offer twice as many in all; where there are not enough, all is listed.
  const uint32_t mine = ord32(mx + 0.0f);
  const int busy = nbatch > 1 ? kSelWarps : max(1, min(kSelWarps, (v1 - v0 + nv * 32 - 1) / max(1, nv * 32)));
  const int q = nbatch > 1 ? (2 * top + kSelWarps - 1) / kSelWarps : min(kSelOffers, (2 * top + busy - 1) / busy);
  uint32_t o = mine;
  if (q > 6) {  // the warp's maxima sorted, the largest first
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1) {
        const uint32_t w = __shfl_xor_sync(0xffffffffu, o, j);
        o = ((lane & j) == 0) == ((lane & k) == 0) ? max(o, w) : min(o, w);
      }
    if (lane < q) offer[warp * q + lane] = o;
  } else {
    for (int i = 0; i < q; ++i) {
      const uint32_t w = __reduce_max_sync(0xffffffffu, o);
      const unsigned at = __ballot_sync(0xffffffffu, o == w);
      if (lane == __ffs(at) - 1) {
        offer[warp * q + i] = w;
        o = 0;
      }
    }
  }
  __syncthreads();
  SelPart total;  // in warp 0
  if (warp == 0) {
    const SelPart w = lane < kSelWarps ? parts[lane] : SelPart{0.0, kNegInf, 0};
    total.m = unord32(__reduce_max_sync(0xffffffffu, ord32(w.m + 0.0f)));
    total.s = sel_scaled(w.s, w.m, total.m);
#pragma unroll
    for (int i = kSelWarps / 2; i > 0; i >>= 1) total.s += shfl_xor_double(total.s, i);
    total.ninf = __reduce_add_sync(0xffffffffu, w.ninf);
  }
  // the bound: an offer with fewer than `top` above it and `top` at or above it
  for (int i = tid; i < q * kSelWarps; i += NT) {
    const uint32_t w = offer[i];
    int gt = 0, ge = 0;
#pragma unroll 4
    for (int j = 0; j < q * kSelWarps; j += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(offer + j);
      gt += (v.x > w) + (v.y > w) + (v.z > w) + (v.w > w);
      ge += (v.x >= w) + (v.y >= w) + (v.z >= w) + (v.w >= w);
    }
    if (gt < top && top <= ge) bound = max(w, ord32(kSelLowest));  // a column at -inf is no candidate
  }
  __syncthreads();
  const uint32_t low = bound;
  const float thr = unord32(low);
  if (mine >= low) {
    for (int g = 0; g < group; ++g)
      if (group_max[g * NT + tid] >= thr) hits[atomicAdd(&nhits, 1)] = static_cast<unsigned short>(g * NT + tid);
  }
  __syncthreads();
  // a thread to a vector of the groups that were hit: read again, from L2
  const int per_hit = per_group * nv;
  for (int i = tid; i < nhits * per_hit; i += NT) {
    const int h = i / per_hit, k = i - h * per_hit;
    const int g = hits[h] / NT, t = hits[h] % NT;
    const int kb = nv == NV ? k / NV : k / nv;
    const int v = v0 + (g * per_group + kb) * step + (t >> 5) * nv * 32 + (k - kb * nv) * 32 + (t & 31);
    if (v >= v1) continue;
    const int col = v * N, have = min(N, a.vocab - col);
    if (!SHIFT && have == N) {
      Vec<T> r;
      r.raw = *reinterpret_cast<const uint4*>(in + col);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (r.get(j) >= thr) {
          const int at = atomicAdd(&count, 1);
          if (at < kSelCap) list[at] = dkey(r.get(j), col + j);
        }
    } else {
      for (int j = 0; j < have; ++j) {
        const float e = to_float(in[col + j]);
        if (e >= thr) {
          const int at = atomicAdd(&count, 1);
          if (at < kSelCap) list[at] = dkey(e, col + j);
        }
      }
    }
  }
  __syncthreads();
  int n = count;
  // Too many: the `top`-th of those that were kept is a bound that as many
  // columns reach; gather again from it on, in the order of the keys (distinct,
  // so at least kSelCap - top columns drop out each time).
  while (n > kSelCap) {
    for (int i = tid; i < kSelCap; i += NT) {
      int r = 0;
      const uint64_t k = list[i];
      for (int j = 0; j < kSelCap; ++j) r += list[j] < k;
      if (r == top - 1) bound_key = k;
    }
    __syncthreads();
    const uint64_t bk = bound_key;
    if (tid == 0) count = 0;
    __syncthreads();
    const int hi = min(a.vocab, v1 * N);
    for (int col = v0 * N + tid; col < hi; col += NT) {
      const float e = fmaxf(to_float(in[col]), kNegInf);
      const uint64_t k = dkey(e, col);
      if (e > kNegInf && k <= bk) {
        const int at = atomicAdd(&count, 1);
        if (at < kSelCap) list[at] = k;
      }
    }
    __syncthreads();
    n = count;
    __syncthreads();
  }
  const int ntop = min(n, top);
  for (int i = tid; i < n; i += NT) {
    int r = 0;
    const uint64_t k = list[i];
    for (int j = 0; j < n; ++j) r += list[j] < k;
    if (r < top) best[r] = k;
  }
  __syncthreads();

  if (C > 1) {
    cluster_wait();
    if (tid == 0) {
      *cl.map_shared_rank(&slots[rankc], 0) = total;
      *cl.map_shared_rank(&slot_n[rankc], 0) = ntop;
    }
    if (tid < ntop) *cl.map_shared_rank(&slot_keys[rankc * kBeamMaxTake + tid], 0) = best[tid];
    cluster_sync_all();
    if (rankc != 0) return;
  } else {
    if (tid == 0) {
      slots[0] = total;
      slot_n[0] = ntop;
    }
    if (tid < ntop) slot_keys[tid] = best[tid];
    __syncthreads();
  }

  // the leader: the row's sum, and a key's place: its own in its list and what
  // comes before it in the others
  uint64_t* keys = static_cast<uint64_t*>(a.workspace) + static_cast<long long>(row) * (top + 2);
  float m = kNegInf;
  int inf = 0, have = 0;
  for (int i = 0; i < C; ++i) {
    m = fmaxf(m, slots[i].m);
    inf += slots[i].ninf;
    have += slot_n[i];
  }
  if (tid == 0) {
    double s = 0.0;
    for (int i = 0; i < C; ++i) s += sel_scaled(slots[i].s, slots[i].m, m);
    SelRow r;
    r.inf = inf > 0;
    r.lse = inf > 0 ? log(static_cast<double>(inf)) : static_cast<double>(m) + log(s);
    r.n = min(top, inf > 0 ? min(inf, have) : have);
    *reinterpret_cast<SelRow*>(keys) = r;
  }
  for (int i = tid; i < C * top; i += NT) {
    const int l = i / top, at = i - l * top;
    if (at >= slot_n[l]) continue;
    const uint64_t k = slot_keys[l * kBeamMaxTake + at];
    int r = at;
    for (int c = 0; c < C; ++c) {
      if (c == l) continue;
      int b = 0, e = slot_n[c];
      while (b < e) {
        const int h = (b + e) >> 1;
        if (slot_keys[c * kBeamMaxTake + h] < k)
          b = h + 1;
        else
          e = h;
      }
      r += b;
    }
    if (r < top) keys[2 + r] = k;
  }
}

// Order-preserving code of a value in 64 bits (no NaN); larger value, larger code.
__device__ __forceinline__ uint64_t ord64(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b & 0x8000000000000000ull ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double unord64(uint64_t o) {
  return __longlong_as_double(static_cast<long long>(o & 0x8000000000000000ull ? o & 0x7fffffffffffffffull : ~o));
}

constexpr int kJoinThreads = 256;

// One CTA per request.  Codes of the lists' values in shared memory, then warp 0
// takes the largest head `take` times; equal values go by the beam.  A code of 0
// is no value's: the end of a list.
__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const BeamSelectArgs a) {
  extern __shared__ uint64_t codes[];  // [beams][take + 1], then tokens [beams][take]
  const int tid = threadIdx.x, lane = tid & 31;
  const int K = a.beams, top = a.take;
  uint32_t* toks = reinterpret_cast<uint32_t*>(codes + K * (top + 1));
  grid_wait();
  grid_release();
  const int req = blockIdx.x;
  const uint64_t* ws = static_cast<const uint64_t*>(a.workspace) + static_cast<long long>(req) * K * (top + 2);
  for (int i = tid; i < K * (top + 1); i += kJoinThreads) {
    const int b = i / (top + 1), j = i - b * (top + 1);
    const uint64_t* keys = ws + static_cast<long long>(b) * (top + 2);
    const SelRow r = *reinterpret_cast<const SelRow*>(keys);
    const float score = a.scores[static_cast<long long>(req) * K + b];
    uint64_t code = 0;
    if (score > kNegInf && j < r.n) {
      const uint64_t k = keys[2 + j];
      const double lp = r.inf ? -r.lse : static_cast<double>(dval(k)) - r.lse;
      const double v = static_cast<double>(score) + lp;
      if (v > -static_cast<double>(__int_as_float(0x7f800000))) code = ord64(v);
      toks[b * top + j] = did(k);
    }
    codes[i] = code;
  }
  __syncthreads();
  if (tid >= 32) return;
  int at = 0;
  uint64_t head = lane < K ? codes[lane * (top + 1)] : 0;
  const long long out = static_cast<long long>(req) * top;
  for (int i = 0; i < top; ++i) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(head >> 32));
    const uint32_t low = static_cast<uint32_t>(head >> 32) == hi ? static_cast<uint32_t>(head) : 0u;
    const uint32_t lo = __reduce_max_sync(0xffffffffu, low);
    const unsigned who =
        __ballot_sync(0xffffffffu, static_cast<uint32_t>(head >> 32) == hi && static_cast<uint32_t>(head) == lo);
    if (hi == 0 && lo == 0) {  // no candidates are left
      for (int j = i + lane; j < top; j += 32) {
        a.out_scores[out + j] = kNegInf;
        a.parents[out + j] = -1;
        a.tokens[out + j] = -1;
      }
      return;
    }
    if (lane == __ffs(who) - 1) {
      a.out_scores[out + i] = static_cast<float>(unord64(head));
      a.parents[out + i] = lane;
      a.tokens[out + i] = static_cast<int>(toks[lane * top + at]);
      ++at;
      head = codes[lane * (top + 1) + at];
    }
  }
}

template <class T, bool SHIFT>
cudaError_t run_select(const BeamSelectArgs& a, cudaStream_t s) {
  // CTAs per row: one, or as many as give each SM one, with a batch each.
  const long long batches = (a.vocab / Vec<T>::N + kSelVecs * kSelThreads - 1) / (kSelVecs * kSelThreads);
  const long long rows = static_cast<long long>(a.requests) * a.beams;
  const int sms = sm_count();
  int C = 1;
  while (C < kSelMaxCluster && C < batches && rows * C < sms) C <<= 1;
  const long long grid = rows * C;
  if (grid > INT_MAX) return cudaErrorInvalidConfiguration;
  constexpr int smem = kSelStages * kSelWarps * (SHIFT ? kSelSlots : kSelWarpVecs) * 16;
  cudaError_t e = allow_smem<beam_rows_kernel<T, SHIFT>>(smem);
  if (e != cudaSuccess) return e;
  e = launch_chained(beam_rows_kernel<T, SHIFT>, static_cast<unsigned>(grid), kSelThreads, smem, C, s, a);
  if (e != cudaSuccess) return e;
  const size_t lists = static_cast<size_t>(a.beams) * ((a.take + 1) * 8 + a.take * 4);
  return launch_chained(beam_join_kernel, static_cast<unsigned>(a.requests), kJoinThreads, lists, 1, s, a);
}

template <class T>
cudaError_t run_select(const BeamSelectArgs& a, cudaStream_t s) {
  const bool on_grid = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 &&
                       (static_cast<long long>(a.requests) * a.beams == 1 || a.ld % Vec<T>::N == 0);
  return on_grid ? run_select<T, false>(a, s) : run_select<T, true>(a, s);
}

// =============================================================== reorder ==
// state[r][k] <- state[r][parent[r][k]] in place.  A thread owns one column (W
// bytes) of a request's rows: it reads all rows' parents at that column, then
// writes them, so nothing is read after it was written and no copy is kept.
// Rows that are their own parents are neither read nor written.
constexpr int kReorderThreads = 256;

template <int W>
struct Piece;
template <>
struct Piece<16> {
  using type = uint4;
};
template <>
struct Piece<4> {
  using type = uint32_t;
};
template <>
struct Piece<1> {
  using type = unsigned char;
};

template <int K, int W>
__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const BeamReorderArgs a) {
  using P = typename Piece<W>::type;
  grid_wait();
  grid_release();
  int t = 0;
  while (t + 1 < a.n && blockIdx.x >= a.first[t + 1]) ++t;
  const unsigned i = blockIdx.x - a.first[t];
  const unsigned req = i / a.chunks[t];
  const long long col = (static_cast<long long>(i - req * a.chunks[t]) * kReorderThreads + threadIdx.x) * W;
  const BeamState st = a.states[t];
  if (col >= st.row_bytes) return;
  const int* parents = a.parents + req * a.ld_parents;
  char* at = static_cast<char*>(st.data) + static_cast<long long>(req) * a.beams * st.stride_bytes + col;
  int from[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    from[k] = k < a.beams ? parents[k] : k;
    if (from[k] < 0 || from[k] >= a.beams) from[k] = k;
  }
  P v[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (from[k] != k) v[k] = *reinterpret_cast<const P*>(at + from[k] * st.stride_bytes);
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (from[k] != k) *reinterpret_cast<P*>(at + k * st.stride_bytes) = v[k];
}

template <int W>
cudaError_t run_reorder(const BeamReorderArgs& a, unsigned grid, cudaStream_t s) {
  if (a.beams <= 4) return launch_chained(beam_reorder_kernel<4, W>, grid, kReorderThreads, 0, 1, s, a);
  if (a.beams <= 8) return launch_chained(beam_reorder_kernel<8, W>, grid, kReorderThreads, 0, 1, s, a);
  if (a.beams <= 16) return launch_chained(beam_reorder_kernel<16, W>, grid, kReorderThreads, 0, 1, s, a);
  return launch_chained(beam_reorder_kernel<32, W>, grid, kReorderThreads, 0, 1, s, a);
}

}  // namespace

size_t beam_workspace_bytes(int rows, int take) {
  static_assert(sizeof(SelRow) == 16, "a row's record is two keys long");
  return static_cast<size_t>(rows) * (take + 2) * 8;
}

cudaError_t launch_beam_select(const BeamSelectArgs& a, int dtype, cudaStream_t s) {
  if (dtype == kOpsF16) return run_select<__half>(a, s);
  if (dtype == kOpsBF16) return run_select<__nv_bfloat16>(a, s);
  return run_select<float>(a, s);
}

cudaError_t launch_beam_reorder(BeamReorderArgs a, int requests, int width, cudaStream_t s) {
  unsigned long long ctas = 0;
  for (int i = 0; i < a.n; ++i) {
    const long long per = static_cast<long long>(kReorderThreads) * width;
    const long long chunks = (a.states[i].row_bytes + per - 1) / per;
    if (chunks > INT_MAX) return cudaErrorInvalidConfiguration;
    a.first[i] = static_cast<unsigned>(ctas);
    a.chunks[i] = static_cast<unsigned>(chunks);
    ctas += static_cast<unsigned long long>(chunks) * requests;
    if (ctas > INT_MAX) return cudaErrorInvalidConfiguration;
  }
  if (ctas == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>(ctas);
  if (width == 16) return run_reorder<16>(a, grid, s);
  if (width == 4) return run_reorder<4>(a, grid, s);
  return run_reorder<1>(a, grid, s);
}

}  // namespace vb
