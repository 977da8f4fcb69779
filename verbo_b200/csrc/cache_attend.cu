// Attention of a row's last tokens over its pages of the 8-bit cache
// (include/verbo_cache.h).
//
//   out = sum_i e^(s_i - m) v_i / sum_i e^(s_i - m),  s_i = scale q . k_i
//
// Bound by memory: a token and head of the cache is 2 dim bytes, read once for all
// query heads that share it.  All rows' blocks of 16 tokens lie in one sequence,
// (row, head, block), of which every warp of the card takes an equal part, however
// the lengths are spread; a warp keeps the running maximum and sum of the softmax,
// and nothing but its own shared memory is waited for.  Where a (row, head) is
// split over warps a second kernel joins their parts.
//
// A warp copies its blocks (cp.async, several ahead) and multiplies them on
// mma.m16n8k16 with fp16 operands: codes are exact in fp16.  Of the 16 rows of A, 8
// hold the queries rounded to fp16 and 8 what the rounding left, so that products are
// exact to 2^-22 whatever the query's type at no extra instruction (8 rows are
// enough for the heads that share a token); the weights e^(s - m) are split the same
// way.  Sums on the tensor cores are cut, not rounded, so they are taken over to
// fp32 registers every few blocks.
#include <algorithm>
#include <climits>

#include "cache.cuh"
#include "device.cuh"
#include "ops.cuh"
#include "opsdev.cuh"

namespace vb {
namespace {

constexpr int kAttWarps = 8;
constexpr int kAttThreads = kAttWarps * 32;
constexpr int kAttRows = 8;      // query rows of a tile: heads that share a token, times steps
constexpr int kAttFlush = 8;     // blocks between two transfers of the sums
constexpr int kAttStages = 6;    // blocks in flight per warp, at most
constexpr float kUp = 14.0f;     // weights are held times 2^14: fp16's subnormals begin at 2^-28 of the largest
constexpr double kLog2e = 1.4426950408889634;

struct AttendArgs {
  const unsigned char* k;
  const unsigned char* v;
  const float* k_scale;
  const float* v_scale;
  const int* table;
  const int* lens;
  int rows, width, pages, heads, dim, page;
  const void* q;
  long long ld_q, hd_q;
  void* out;
  long long ld_out, hd_out;
  int group;  // query heads per head
  int steps;
  int tiles;      // of kAttRows query rows
  int teams;      // warps that share a part of the blocks, one tile each: grid warps / tiles
  int least;      // blocks that a warp takes at least
  int stages;
  int q_type, out_type;
  float c_hi, c_lo;  // scale * log2(e)
  float* parts;      // [teams][tiles][2][part_floats]
  long long* first;  // [rows + 1] blocks before each row
};
__host__ __device__ inline int part_floats(int dim) { return kAttRows * (dim + 2); }

// The part of the blocks that a team takes.
__device__ __forceinline__ long long blocks_each(const AttendArgs& a, long long all) {
  return max(static_cast<long long>(a.least), (all + a.teams - 1) / a.teams);
}

__device__ __forceinline__ float load_any(const void* p, long long i, int type) {
  if (type == kOpsF32) return static_cast<const float*>(p)[i];
  if (type == kOpsF16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, long long i, int type, float v) {
  if (type == kOpsF32)
    static_cast<float*>(p)[i] = v;
  else if (type == kOpsF16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t two_halves(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What the rounding of two values to fp16 left, in fp16.
__device__ __forceinline__ uint32_t two_rests(float lo, float hi, uint32_t rounded) {
  const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
  return two_halves(lo - r.x, hi - r.y);
}
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {  // codes 0, 1 of a word as fp16
  uint32_t h;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {  // codes 2, 3
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool take) {  // zeros otherwise
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// Blocks of 16 tokens before each row, in shared memory (rows + 1), by the CTA.
__device__ __forceinline__ void scan_rows(const AttendArgs& a, long long* first, long long* ws) {
  long long base = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kAttThreads) {
    const int r = r0 + threadIdx.x;
    long long n = 0;
    if (r < a.rows) {
      const int len = max(0, min(a.lens[r], a.width * a.page));
      n = (len + kCacheBlock - 1) / kCacheBlock;
    }
    long long total;
    const long long at = block_excl_scan<long long, kAttThreads>(n, ws, &total);
    if (r < a.rows) first[r] = base + at;
    base += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) first[a.rows] = base;
  __syncthreads();
}

struct __align__(16) SlotHead {
  float ks, vs;
  int valid;
  int pad;
};

// DP: the head dimension filled up with zeros.  Shared memory per warp: `stages`
// slots of a block's keys and values, rows of DP bytes whose 16-byte chunks are
// exchanged so that the fragment loads below meet no bank twice.
template <int DP>
__global__ void __launch_bounds__(kAttThreads, DP == 64 ? 2 : 1) cache_attend_kernel(const AttendArgs a) {
  constexpr int NJ = DP / 8;            // output tiles of 8 dims
  constexpr int KS = DP / 16;           // steps of 16 dims
  constexpr int CH = DP / 32;           // chunks that a lane copies of a block's keys
  constexpr int BLOCK_BYTES = 16 * DP;  // of keys, and of values
  constexpr int OWN = DP / 4;           // output dims of a lane
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long scan_ws[kAttWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + static_cast<size_t>(warp) * a.stages * (2 * BLOCK_BYTES + sizeof(SlotHead));
  SlotHead* heads_at = reinterpret_cast<SlotHead*>(ring + static_cast<size_t>(a.stages) * 2 * BLOCK_BYTES);
  long long* first =
      reinterpret_cast<long long*>(smem + static_cast<size_t>(kAttWarps) * a.stages * (2 * BLOCK_BYTES + sizeof(SlotHead)));
  if (a.dim < DP)  // the filled-up dims stay zero
    for (int i = lane; i < a.stages * 2 * BLOCK_BYTES / 16; i += 32)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
  grid_wait();
  grid_release();
  scan_rows(a, first, scan_ws);
  if (blockIdx.x == 0)
    for (int r = tid; r <= a.rows; r += kAttThreads) a.first[r] = first[r];

  const long long all = first[a.rows] * a.heads;
  const long long each = blocks_each(a, all);
  const int id = warp * gridDim.x + blockIdx.x;  // few blocks go to as many SMs as there are
  const int team = id / a.tiles, tile = id - team * a.tiles;
  if (team >= a.teams) return;
  long long i0 = team * each;
  const long long i1 = min(all, i0 + each);
  if (i0 >= i1) return;

  // a lane's chunks of a block: where they go, which token they belong to
  const int per_token = a.dim / 16;
  uint32_t to_k[CH], to_v[CH];
  int token_of[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = lane + 32 * i;
    const int tok = c / per_token, col = c - tok * per_token;
    token_of[i] = c < a.dim ? tok : 64;
    if (DP == 128) {
      to_k[i] = tok * 128 + ((col ^ ((tok & 1) << 2)) << 4);
      to_v[i] = tok * 128 + ((col ^ (((tok >> 1) & 3) << 1)) << 4);
    } else {
      to_k[i] = tok * 64 + (col << 4);
      const int line = tok >> 1, place = ((tok & 1) << 2) | col;
      to_v[i] = line * 128 + ((place ^ ((line & 3) << 1)) << 4);
    }
  }
  const uint32_t ring_at = smem_u32(ring), heads_smem = smem_u32(heads_at);

  int row;
  {
    const long long want = i0 / a.heads;  // a row's blocks come heads times in a row
    int lo = 0, hi = a.rows - 1;
    while (lo < hi) {  // the last row that begins at or before it (rows without blocks come first)
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= want)
        lo = mid;
      else
        hi = mid - 1;
    }
    row = lo;
  }
  int part = 0;  // parts that this warp has written
  while (i0 < i1) {
    while (first[row + 1] * a.heads <= i0) ++row;
    const int nb = static_cast<int>(first[row + 1] - first[row]);
    const long long in_row = i0 - first[row] * a.heads;
    const int head = static_cast<int>(in_row / nb);
    const int b0 = static_cast<int>(in_row - static_cast<long long>(head) * nb);
    const int n = static_cast<int>(min(static_cast<long long>(nb - b0), i1 - i0));
    const int len = max(0, min(a.lens[row], a.width * a.page));
    const int* pages = a.table + static_cast<long long>(row) * a.width;

    // ---- copies, `stages` blocks ahead
    int page_ids = -1;  // of 32 blocks, one per lane
    auto fetch = [&](int j) {
      if (j < n) {
        if ((j & 31) == 0) {
          const int b = b0 + j + lane;
          page_ids = b < nb ? pages[(b * kCacheBlock) / a.page] : -1;
        }
        int pid = __shfl_sync(0xffffffffu, page_ids, j & 31);
        const int b = b0 + j;
        int valid = min(kCacheBlock, len - b * kCacheBlock);
        if (pid < 0 || pid >= a.pages) {
          pid = 0;
          valid = 0;
        }
        const int inside = (b * kCacheBlock) % a.page;
        const long long at = static_cast<long long>(pid) * a.heads + head;
        const long long from = (at * a.page + inside) * a.dim + lane * 16;
        const int slot = j % a.stages;
        const uint32_t to = ring_at + slot * 2 * BLOCK_BYTES;
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (token_of[i] < 16) {
            const bool take = token_of[i] < valid;
            cp_async16_if(to + to_k[i], a.k + from + i * 512, take);
            cp_async16_if(to + BLOCK_BYTES + to_v[i], a.v + from + i * 512, take);
          }
        const long long sc = at * (a.page / kCacheBlock) + inside / kCacheBlock;
        if (lane == 0) {
          cp_async4(heads_smem + slot * sizeof(SlotHead), a.k_scale + sc);
          cp_async4(heads_smem + slot * sizeof(SlotHead) + 4, a.v_scale + sc);
          heads_at[slot].valid = valid;
        }
      }
      cp_async_commit();
    };
    for (int j = 0; j < a.stages - 1; ++j) fetch(j);

    // ---- the queries of this lane's row: row g of the tile, its own dims
    const int r = tile * kAttRows + g;  // step r / group, head r % group
    const bool live = r < a.steps * a.group;
    const int step = live ? r / a.group : 0;
    const long long q_at = (static_cast<long long>(row) * a.steps + step) * a.ld_q +
                           static_cast<long long>(head * a.group + (live ? r - step * a.group : 0)) * a.hd_q;
    uint32_t qa[KS][4];
    float row_scale;
    {
      float x[OWN];
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int d = (i / 16) * 64 + t * 16 + (i % 16);
        x[i] = live && d < a.dim ? load_any(a.q, q_at + d, a.q_type) : 0.0f;
      }
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < OWN; ++i) most = fmaxf(most, fabsf(x[i]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // the row times 2^e has its largest element in [2^14, 2^15)
      int e = 141 - static_cast<int>(__float_as_uint(most) >> 23);
      if (e < -113) e = 0;  // inf or NaN
      e = min(e, 126);
      const float up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
      row_scale = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float* y = x + 4 * s;
        qa[s][0] = two_halves(y[0] * up, y[1] * up);
        qa[s][1] = two_rests(y[0] * up, y[1] * up, qa[s][0]);
        qa[s][2] = two_halves(y[2] * up, y[3] * up);
        qa[s][3] = two_rests(y[2] * up, y[3] * up, qa[s][2]);
      }
    }
    const int end = len - (a.steps - 1 - step);  // places that the row sees

    float acc[NJ][4], sum[NJ][2];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
      sum[j][0] = sum[j][1] = 0.0f;
    }
    float m = kNegInf, l = 0.0f, vref = 0.0f;
    int since = 0;
    auto flush = [&]() {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        sum[j][0] += acc[j][0] + acc[j][2];
        sum[j][1] += acc[j][1] + acc[j][3];
        acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
      }
      since = 0;
    };

    for (int j = 0; j < n; ++j) {
      fetch(j + a.stages - 1);
      // all but the newest stages - 1 groups are here
      if (a.stages == 6)
        asm volatile("cp.async.wait_group 5;" ::: "memory");
      else if (a.stages == 5)
        asm volatile("cp.async.wait_group 4;" ::: "memory");
      else
        asm volatile("cp.async.wait_group 3;" ::: "memory");
      __syncwarp();
      const int slot = j % a.stages;
      const unsigned char* kt = ring + slot * 2 * BLOCK_BYTES;
      const unsigned char* vt = kt + BLOCK_BYTES;
      const SlotHead sh = heads_at[slot];

      // scores: tokens 8 h + g are the columns, this lane has columns 2 t and 2 t + 1
      float sc[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h][0] = sc[h][1] = sc[h][2] = sc[h][3] = 0.0f;
        const int tok = 8 * h + g;
        if (DP == 128) {
          const int flip = (tok & 1) << 2;
          const uint4 x = *reinterpret_cast<const uint4*>(kt + tok * 128 + ((t ^ flip) << 4));
          const uint4 y = *reinterpret_cast<const uint4*>(kt + tok * 128 + (((t + 4) ^ flip) << 4));
          const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
          for (int s = 0; s < KS; ++s) mma16816(sc[h], qa[s], codes_lo(w[s]), codes_hi(w[s]));
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(kt + tok * 64 + (t << 4));
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int s = 0; s < KS; ++s) mma16816(sc[h], qa[s], codes_lo(w[s]), codes_hi(w[s]));
        }
      }
      const int lim = min(sh.valid, end - (b0 + j) * kCacheBlock);
      const float f = row_scale * sh.ks;
      float p[2][2];
      float mx = kNegInf;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = (sc[h][i] + sc[h][i + 2]) * f;
          const float y = fmaf(x, a.c_hi, x * a.c_lo);
          p[h][i] = 8 * h + 2 * t + i < lim ? y : kNegInf;
          mx = fmaxf(mx, p[h][i]);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float vnew = sh.valid > 0 ? fmaxf(vref, fabsf(sh.vs)) : vref;
      if (__any_sync(0xffffffffu, mx > m || vnew != vref)) {
        const float mn = fmaxf(m, mx);
        const float alpha = m > kNegInf ? ex2(m - mn) : 0.0f;
        const float both = vnew != vref ? (vref > 0.0f ? alpha * __fdiv_rn(vref, vnew) : 0.0f) : alpha;
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
          acc[i][0] *= both, acc[i][1] *= both, acc[i][2] *= both, acc[i][3] *= both;
          sum[i][0] *= both, sum[i][1] *= both;
        }
        l *= alpha;
        m = mn;
        vref = vnew;
      }
      const float base = m > kNegInf ? m - kUp : 0.0f;
      const float ratio = vref > 0.0f && sh.valid > 0 ? __fdiv_rn(sh.vs, vref) : 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[h][i] = ex2(p[h][i] - base);
          l += p[h][i];
          p[h][i] *= ratio;
        }
      uint32_t pa[4];
      pa[0] = two_halves(p[0][0], p[0][1]);
      pa[1] = two_rests(p[0][0], p[0][1], pa[0]);
      pa[2] = two_halves(p[1][0], p[1][1]);
      pa[3] = two_rests(p[1][0], p[1][1], pa[2]);

      // values: this lane has tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 at the dims g DP / 8 ...
      constexpr int W = DP / 32;  // words of a token
      uint32_t v[4][W];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 2 * t + (i & 1) + 8 * (i >> 1);
        if (DP == 128) {
          const uint4 x = *reinterpret_cast<const uint4*>(vt + tok * 128 + ((g ^ (((tok >> 1) & 3) << 1)) << 4));
          v[i][0] = x.x, v[i][1] = x.y, v[i][W - 2] = x.z, v[i][W - 1] = x.w;
        } else {
          const int line = tok >> 1, place = ((tok & 1) << 2) | (g >> 1);
          const uint2 x = *reinterpret_cast<const uint2*>(vt + line * 128 + ((place ^ ((line & 3) << 1)) << 4) + (g & 1) * 8);
          v[i][0] = x.x, v[i][1] = x.y;
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5140), a1 = __byte_perm(v[0][w], v[1][w], 0x7362);
        const uint32_t c0 = __byte_perm(v[2][w], v[3][w], 0x5140), c1 = __byte_perm(v[2][w], v[3][w], 0x7362);
        mma16816(acc[4 * w], pa, codes_lo(a0), codes_lo(c0));
        mma16816(acc[4 * w + 1], pa, codes_hi(a0), codes_hi(c0));
        mma16816(acc[4 * w + 2], pa, codes_lo(a1), codes_lo(c1));
        mma16816(acc[4 * w + 3], pa, codes_hi(a1), codes_hi(c1));
      }
      if (++since == kAttFlush) flush();
      __syncwarp();  // the slot may be filled again
    }
    cp_async_wait_all();
    flush();
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);

    // this lane's dims: OWN t + i, from the tiles i % NJ and the columns 2 t, 2 t + 1
    const bool whole = n == nb;
    if (whole) {
      if (live) {
        const float inv = l > 0.0f || l != l ? __fdiv_rn(vref, l) : 0.0f;
        const long long o = (static_cast<long long>(row) * a.steps + step) * a.ld_out +
                            static_cast<long long>(head * a.group + r - step * a.group) * a.hd_out;
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          const int d = OWN * t + i;
          if (d < a.dim) store_any(a.out, o + d, a.out_type, sum[i % NJ][i / NJ] * inv);
        }
      }
    } else {
      float* to = a.parts + ((static_cast<long long>(team) * a.tiles + tile) * 2 + part) * part_floats(a.dim);
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int d = OWN * t + i;
        if (d < a.dim) to[g * a.dim + d] = sum[i % NJ][i / NJ] * vref;
      }
      if (t == 0) {
        to[kAttRows * a.dim + g] = m;
        to[kAttRows * a.dim + kAttRows + g] = l;
      }
    }
    part = 1;
    i0 += n;
  }
}

constexpr int kJoinThreads = 128;

// One CTA per (row, head, tile, query row): the parts of its blocks joined, in their
// order; nothing to do where one warp had them all.
__global__ void __launch_bounds__(kJoinThreads) cache_attend_join_kernel(const AttendArgs a) {
  constexpr int W = kJoinThreads / 32, PER = VERBO_CACHE_MAX_DIM / 32;
  __shared__ float ms[W], ls[W], os[W][VERBO_CACHE_MAX_DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int q_rows = a.steps * a.group;
  const int qr = blockIdx.x % q_rows;
  const int head = blockIdx.x / q_rows % a.heads;
  const int row = blockIdx.x / q_rows / a.heads;
  const int tile = qr / kAttRows, g = qr % kAttRows;
  grid_wait();
  grid_release();
  const int step = qr / a.group;
  const long long o = (static_cast<long long>(row) * a.steps + step) * a.ld_out +
                      static_cast<long long>(head * a.group + qr - step * a.group) * a.hd_out;
  const long long nb = a.first[row + 1] - a.first[row];
  if (nb == 0) {  // an empty row
    for (int d = threadIdx.x; d < a.dim; d += kJoinThreads) store_any(a.out, o + d, a.out_type, 0.0f);
    return;
  }
  const long long each = blocks_each(a, a.first[a.rows] * a.heads);
  const long long f = a.first[row] * a.heads + head * nb, e = f + nb - 1;
  const int w0 = static_cast<int>(f / each), w1 = static_cast<int>(e / each);
  if (w0 == w1) return;
  float m = kNegInf, l = 0.0f, x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = 0.0f;
  for (int w = w0 + warp; w <= w1; w += W) {
    const int which = w * each < f;  // its second part, after the end of another
    const float* from = a.parts + ((static_cast<long long>(w) * a.tiles + tile) * 2 + which) * part_floats(a.dim);
    const float pm = from[kAttRows * a.dim + g], pl = from[kAttRows * a.dim + kAttRows + g];
    float y[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) y[i] = lane + 32 * i < a.dim ? from[g * a.dim + lane + 32 * i] : 0.0f;
    if (pm == kNegInf && pl == 0.0f) continue;
    const float mn = fmaxf(m, pm);
    const float u = m > kNegInf ? ex2(m - mn) : 0.0f, t = pm > kNegInf ? ex2(pm - mn) : 1.0f;
    m = mn;
    l = l * u + pl * t;
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = x[i] * u + y[i] * t;
  }
  if (lane == 0) {
    ms[warp] = m;
    ls[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) os[warp][lane + 32 * i] = x[i];
  __syncthreads();
  float mn = kNegInf;
  for (int w = 0; w < W; ++w) mn = fmaxf(mn, ms[w]);
  float total = 0.0f, u[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    u[w] = ms[w] > kNegInf ? ex2(ms[w] - mn) : (ls[w] != ls[w] ? 1.0f : 0.0f);
    total += ls[w] * u[w];
  }
  const float inv = total > 0.0f || total != total ? __fdiv_rn(1.0f, total) : 0.0f;
  for (int d = threadIdx.x; d < a.dim; d += kJoinThreads) {
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) y += os[w][d] * u[w];
    store_any(a.out, o + d, a.out_type, y * inv);
  }
}

constexpr int kAttMaxSmem = 227 * 1024;

struct Plan {
  int dp, grid, stages, tiles, teams, least;
  size_t smem, parts_bytes;
};
Plan plan(const verbo_cache& c, int heads, int steps) {
  Plan p{};
  p.dp = c.dim <= 64 ? 64 : 128;
  const int per_sm = p.dp == 64 ? 2 : 1;
  p.grid = sm_count() * per_sm;
  p.tiles = (steps * (heads / c.heads) + kAttRows - 1) / kAttRows;
  p.teams = std::max(1, p.grid * kAttWarps / p.tiles);
  p.least = 2;
  const size_t rows = (static_cast<size_t>(c.rows) + 1) * 8;
  const size_t slot = static_cast<size_t>(kAttWarps) * (32 * p.dp + sizeof(SlotHead));
  const size_t room = (kAttMaxSmem - 1024 * (per_sm - 1)) / per_sm - 512;
  p.stages = std::min<int>(kAttStages, static_cast<int>((room - rows) / slot));
  p.smem = p.stages * slot + rows;
  p.parts_bytes = static_cast<size_t>(p.teams) * p.tiles * 2 * part_floats(c.dim) * 4;
  return p;
}

template <int DP>
cudaError_t run_attend(const AttendArgs& a, const Plan& p, cudaStream_t s) {
  const auto kernel = cache_attend_kernel<DP>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             DP == 64 ? kAttMaxSmem / 2 : kAttMaxSmem - 1024);
  if (e != cudaSuccess) return e;
  return launch_chained(kernel, static_cast<unsigned>(p.grid), kAttThreads, p.smem, 1, s, a);
}

}  // namespace

size_t cache_attend_bytes(const verbo_cache& c, int heads, int steps) {
  return (plan(c, heads, steps).parts_bytes + (static_cast<size_t>(c.rows) + 1) * 8 + 15) / 16 * 16;
}

cudaError_t launch_cache_attend(const verbo_cache& c, int layer, const CacheQuery& x, int q_type, int out_type,
                                cudaStream_t s) {
  const Plan p = plan(c, x.heads, x.steps);
  AttendArgs a{};
  const size_t per = static_cast<size_t>(c.pages) * c.heads * c.page;
  a.k = c.k + layer * per * c.dim;
  a.v = c.v + layer * per * c.dim;
  a.k_scale = c.k_scale + layer * (per / kCacheBlock);
  a.v_scale = c.v_scale + layer * (per / kCacheBlock);
  a.table = c.table;
  a.lens = c.lens;
  a.rows = c.rows;
  a.width = c.width;
  a.pages = c.pages;
  a.heads = c.heads;
  a.dim = c.dim;
  a.page = c.page;
  a.q = x.q;
  a.ld_q = x.ld_q;
  a.hd_q = x.hd_q;
  a.out = x.out;
  a.ld_out = x.ld_out;
  a.hd_out = x.hd_out;
  a.group = x.heads / c.heads;
  a.steps = x.steps;
  a.tiles = p.tiles;
  a.teams = p.teams;
  a.least = p.least;
  a.stages = p.stages;
  a.q_type = q_type;
  a.out_type = out_type;
  const double f = static_cast<double>(x.scale) * kLog2e;
  a.c_hi = static_cast<float>(f);
  a.c_lo = static_cast<float>(f - static_cast<double>(a.c_hi));
  a.parts = static_cast<float*>(x.workspace);
  a.first = reinterpret_cast<long long*>(static_cast<char*>(x.workspace) + p.parts_bytes);
  const long long joins = static_cast<long long>(c.rows) * c.heads * x.steps * a.group;
  if (joins > INT_MAX) return cudaErrorInvalidConfiguration;
  const cudaError_t e = p.dp == 64 ? run_attend<64>(a, p, s) : run_attend<128>(a, p, s);
  if (e != cudaSuccess) return e;
  return launch_chained(cache_attend_join_kernel, static_cast<unsigned>(joins), kJoinThreads, 0, 1, s, a);
}

}  // namespace vb
