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
// A warp copies its blocks (cp.async, a step or two ahead) and multiplies them on
// mma.m16n8k16 with fp16 operands: codes are exact in fp16.  Tokens, then dims, are the
// 16 rows of a product and the queries its 8 columns: scores K q^T, sums V^T p^T, the
// weights turned in between (movmatrix).  fp32 queries, and all weights e^(s - m), come
// in two parts, rounded to fp16 and what the rounding left, so that products are exact
// to 2^-22; weights have their block's scale in them, as a part of the largest that the warp has
// met, and the second part ends at 2^-39 of a weight of 1 there.  Sums on the tensor cores are cut, not rounded, so they are taken over to
// fp32 registers every few blocks (8 rows of 65536 tokens: off by 6e-7 with it, by 8e-6
// without).
//
// Measured on B200 (a card copies at 6.5 TB/s): 64 rows of 8192 tokens, 8 heads of 128,
// 32 query heads 188 us, 5.7 TB/s; of 4096 102 us; of 0 to 8192 108 us.  Each further
// byte comes at 6.2 TB/s; about 15 us are start, search, an uneven end (the slowest SM is
// busy 15% longer than the mean) and the join.
#include <algorithm>
#include <climits>

#include "cache.cuh"
#include "device.cuh"
#include "ops.cuh"
#include "opsdev.cuh"

namespace vb {
namespace {

constexpr int kAttPair = 2;    // blocks of a step
constexpr int kAttFlush = 4;   // steps between two transfers of the sums (a power of two)
constexpr int kAttHeads = 64;  // blocks that are known ahead, per warp
// What the beginning and the end of a (row, head) cost a warp, in blocks: parts are
// equal with it counted.  64 rows of 0 to 8192 tokens take 108 us with it, 127 without.
constexpr int kAttStart = 4;
constexpr float kUp = 14.0f;   // weights are held times 2^14: fp16's subnormals begin at 2^-28 of the largest
constexpr double kLog2e = 1.4426950408889634;
constexpr uint32_t kCodeBits = 0x7f7f7f7fu;  // of four codes, without their signs: all set in a NaN's

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
  int tile_rows;  // query rows of a tile (heads that share a token, times steps): 8 or 16
  int tiles;
  int teams;      // warps that share a part of the blocks, one tile each: grid warps / tiles
  int least;      // blocks that a warp takes at least
  int q_type, out_type;
  bool wide_q, wide_out;  // 16 bytes at a time
  float c_hi, c_lo;  // scale * log2(e)
  int members;       // CTAs of a cluster, where a cluster has a (row, head, tile)
  float* parts;      // [teams][tiles][2][part_floats]
  int* first;        // [rows + 1] blocks before each row
};
// A part: sums [tile_rows][dim], maxima [tile_rows], weights [tile_rows].
__host__ __device__ inline int part_floats(int rows, int dim) { return rows * (dim + 2); }

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
__device__ __forceinline__ float2 of_halves(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// An 8 x 8 matrix of 16-bit numbers, two of a row in a lane, turned.
__device__ __forceinline__ uint32_t turned(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
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
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool take) {  // zeros otherwise
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// N elements from `p` + i on, as floats, and back; `wide`: p is aligned to 16 bytes, i
// to N elements.
template <int N>
__device__ __forceinline__ void load_n(const void* p, long long i, int type, bool wide, float* x) {
  if (!wide) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = load_any(p, i + j, type);
  } else if (type == kOpsF32) {
    const float4* v = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const float4 y = v[j];
      x[4 * j] = y.x, x[4 * j + 1] = y.y, x[4 * j + 2] = y.z, x[4 * j + 3] = y.w;
    }
  } else {
    const uint4* v = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 8; ++j) {
      const uint4 y = v[j];
      const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = type == kOpsF16
                             ? of_halves(w[k])
                             : make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
        x[8 * j + 2 * k] = f.x, x[8 * j + 2 * k + 1] = f.y;
      }
    }
  }
}
template <int N>
__device__ __forceinline__ void store_n(void* p, long long i, int type, bool wide, const float* x) {
  if (!wide) {
#pragma unroll
    for (int j = 0; j < N; ++j) store_any(p, i + j, type, x[j]);
  } else if (type == kOpsF32) {
    float4* v = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) v[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
  } else {
    uint2* v = reinterpret_cast<uint2*>(static_cast<unsigned short*>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      uint32_t w[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float lo = x[4 * j + 2 * k], hi = x[4 * j + 2 * k + 1];
        if (type == kOpsF16) {
          w[k] = two_halves(lo, hi);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
          w[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      v[j] = make_uint2(w[0], w[1]);
    }
  }
}

// Blocks of 16 tokens before each row, kAttStart more for each row that has any, in
// shared memory (rows + 1), by the CTA.
template <int NT>
__device__ __forceinline__ void scan_rows(const AttendArgs& a, int* first, int* ws) {
  int base = 0;
  for (int r0 = 0; r0 < a.rows; r0 += NT) {
    const int r = r0 + threadIdx.x;
    int n = 0;
    if (r < a.rows) {
      const int len = max(0, min(a.lens[r], a.width * a.page));
      n = len > 0 ? (len - 1) / kCacheBlock + 1 + kAttStart : 0;
    }
    int total;
    const int at = block_excl_scan<int, NT>(n, ws, &total);
    if (r < a.rows) first[r] = base + at;
    base += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) first[a.rows] = base;
  __syncthreads();
}

// What is known of a block before it is copied.
struct __align__(16) BlockHead {
  float ks, vs;
  int valid;  // tokens, 0 where there is no page
  int block;  // of the layer's pool
};

// DP: the head dimension filled up with zeros.  RT: eights of query rows of a tile.
// Shared memory per warp: a ring of steps of two blocks' keys and values, rows of kRow
// bytes whose 16-byte chunks are exchanged so that the fragment loads below meet no
// bank twice, and what is known of the blocks.
// A warp's step is a chain of loads, products and exponentials, and two steps ahead
// cover the memory's latency: 8 warps with three steps of shared memory at 226 registers.
// With 96 dims 168 registers do, and 12 warps with two steps each take 148 us where 8
// with three take 157 (64 rows of 8192 tokens of 80 dims); with 128 dims those spill,
// and 64 rows of 4096 tokens take 124 us against 102.
template <int DP, int RT>
struct AttShape {
  static constexpr int kWarps = DP == 96 && RT == 1 ? 12 : 8;
  static constexpr int kCtas = DP == 64 && RT == 1 ? 2 : 1;  // per SM
  static constexpr int kStages = RT == 1 && DP != 96 ? 3 : 2;  // steps whose copies are in flight
  static constexpr int kRow = DP == 64 ? 64 : 128;
  static constexpr int kBlock = 16 * kRow;             // bytes of a block's keys, and of its values
  static constexpr int kStep = kAttPair * 2 * kBlock;  // of a step
  static constexpr int kRing = kStages * kStep;
  static constexpr int kKnown = kAttHeads * static_cast<int>(sizeof(BlockHead));
  static constexpr int kQuery = RT == 1 ? 0 : DP / 16 * 512;  // fragments of 16 queries
  static constexpr int kWarp = kRing + kKnown + kQuery;
};

// LO: queries in two parts (fp32).  CL: a cluster has one (row, head, tile), split evenly
// over its warps, and joins their parts itself.
template <int DP, int RT, bool LO, bool CL>
__global__ void __launch_bounds__(AttShape<DP, RT>::kWarps * 32, AttShape<DP, RT>::kCtas)
    cache_attend_kernel(const AttendArgs a) {
  using S = AttShape<DP, RT>;
  constexpr int NW = S::kWarps, NT = NW * 32;
  constexpr int MT = DP / 16;  // products of 16 dims
  constexpr int KS = DP / 16;  // steps of 16 dims
  constexpr int CH = DP / 32;  // chunks that a lane copies of a block's keys
  constexpr int VW = DP / 32;  // words of a token's values in a lane
  constexpr int ROWS = 8 * RT;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int scan_ws[NW];
  __shared__ float4 joined[CL ? NW : 1][VERBO_CACHE_MAX_DIM / 4];
  __shared__ float2 joined_ml[CL ? NW : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + warp * S::kWarp;
  BlockHead* known = reinterpret_cast<BlockHead*>(ring + S::kRing);
  uint4* query = reinterpret_cast<uint4*>(ring + S::kRing + S::kKnown) + lane;  // [KS][32], a lane's own
  int* first = reinterpret_cast<int*>(smem + NW * S::kWarp);
  if (a.dim < DP)  // the filled-up dims stay zero
    for (int i = lane; i < S::kRing / 16; i += 32) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
  grid_wait();
  grid_release();
  int team = 0, tile, row = 0, head = 0;
  long long i0 = 0, i1 = 1;
  if (CL) {
    const int unit = blockIdx.x / a.members;
    tile = unit % a.tiles;
    head = unit / a.tiles % a.heads;
    row = unit / a.tiles / a.heads;
  } else {
    scan_rows<NT>(a, first, scan_ws);
    if (blockIdx.x == 0)
      for (int r = tid; r <= a.rows; r += NT) a.first[r] = first[r];
    const long long all = static_cast<long long>(first[a.rows]) * a.heads;
    const long long each = blocks_each(a, all);
    const int id = warp * gridDim.x + blockIdx.x;  // few blocks go to as many SMs as there are
    team = id / a.tiles;
    tile = id - team * a.tiles;
    if (team >= a.teams) return;
    i0 = team * each;
    i1 = min(all, i0 + each);
    if (i0 >= i1) return;
  }

  // a lane's chunks of a block: where they go, which token they belong to
  const int per_token = a.dim / 16;
  uint32_t to_k[CH], to_v[CH];
  int token_of[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = lane + 32 * i;
    const int tok = c / per_token, col = c - tok * per_token;
    token_of[i] = c < a.dim ? tok : 64;
    if (S::kRow == 128) {
      to_k[i] = tok * 128 + ((col ^ ((tok & 1) << 2)) << 4);
      to_v[i] = tok * 128 + ((col ^ (((tok >> 1) & 3) << 1)) << 4);
    } else {
      to_k[i] = tok * 64 + (col << 4);
      const int line = tok >> 1, place = ((tok & 1) << 2) | col;
      to_v[i] = line * 128 + ((place ^ ((line & 3) << 1)) << 4);
    }
    to_v[i] += S::kBlock;
  }
  const uint32_t ring_at = smem_u32(ring);
  const long long block_bytes = 16ll * a.dim;
  // and where it reads fragments: of the keys of token g (and g + 8) the dims 16 t ... and
  // 64 + (DP - 64) / 4 t ...; of the values of tokens 2 t (v0, v2) and 2 t + 1 (v1, v3) (and
  // + 8) the dims N1 g ... and, of 96, 64 + 4 g ...
  uint32_t at_k0, at_k1 = 0, at_v0, at_v1, at_v2 = 0, at_v3 = 0;
  if (DP == 64) {
    at_k0 = g * 64 + (t << 4);
    at_v0 = S::kBlock + t * 128 + (((g >> 1) ^ (t << 1)) << 4) + (g & 1) * 8;
    at_v1 = S::kBlock + t * 128 + (((4 | (g >> 1)) ^ (t << 1)) << 4) + (g & 1) * 8;
  } else {
    const int flip = (g & 1) << 2;
    at_k0 = g * 128 + ((t ^ flip) << 4);
    if (DP == 128) {
      at_k1 = g * 128 + (((t + 4) ^ flip) << 4);
      at_v0 = S::kBlock + 2 * t * 128 + ((g ^ (t << 1)) << 4);
    } else {
      at_k1 = g * 128 + (((4 + (t >> 1)) ^ flip) << 4) + (t & 1) * 8;
      at_v0 = S::kBlock + 2 * t * 128 + (((g >> 1) ^ (t << 1)) << 4) + (g & 1) * 8;
      at_v2 = S::kBlock + 2 * t * 128 + (((4 + (g >> 2)) ^ (t << 1)) << 4) + (g & 3) * 4;
      at_v3 = at_v2 + 128;
    }
    at_v1 = at_v0 + 128;
  }

  if (!CL) {
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
    int nb, b0, n;
    if (CL) {
      nb = (max(0, min(a.lens[row], a.width * a.page)) + kCacheBlock - 1) / kCacheBlock;
      const int all = (nb + 1) / 2, warps = a.members * NW;
      const int w = blockIdx.x % a.members * NW + warp;
      b0 = 2 * (all * w / warps);
      n = max(0, min(nb, 2 * (all * (w + 1) / warps)) - b0);
      i0 = i1;
    } else {
      while (static_cast<long long>(first[row + 1]) * a.heads <= i0) ++row;
      const int counted = first[row + 1] - first[row];
      nb = counted - kAttStart;
      const long long in_row = i0 - static_cast<long long>(first[row]) * a.heads;
      head = static_cast<int>(in_row / counted);
      const int c0 = static_cast<int>(in_row - static_cast<long long>(head) * counted);
      const int c1 = static_cast<int>(min(static_cast<long long>(counted), c0 + (i1 - i0)));
      i0 += c1 - c0;
      b0 = max(0, c0 - kAttStart);
      n = max(0, c1 - kAttStart) - b0;
      if (n == 0) {  // its start alone
        part = 1;
        continue;
      }
    }
    const int len = max(0, min(a.lens[row], a.width * a.page));
    const int* pages = a.table + static_cast<long long>(row) * a.width;
    const int steps = (n + 1) / 2;

    // ---- copies, kStages - 1 steps ahead
    int slot_in = 0;
    int next_page = lane < n ? pages[(b0 + lane) * kCacheBlock / a.page] : -1;
    auto fetch = [&](int j) {
      if (j < steps) {
        if ((j & 15) == 0) {  // the next 32 blocks: one per lane
          const int i = 2 * j + lane, at = (b0 + i) * kCacheBlock;
          const int pid = next_page;
          next_page = i + 32 < n ? pages[(at + 32 * kCacheBlock) / a.page] : -1;
          BlockHead* h = &known[i & (kAttHeads - 1)];
          int2 v = make_int2(0, -1);
          __syncwarp();
          if (i < n && pid >= 0 && pid < a.pages) {
            v.y = (pid * a.heads + head) * (a.page / kCacheBlock) + (at % a.page) / kCacheBlock;
            v.x = min(kCacheBlock, len - at);
            cp_async4(smem_u32(&h->ks), a.k_scale + v.y);
            cp_async4(smem_u32(&h->vs), a.v_scale + v.y);
          } else {
            h->ks = h->vs = 0.0f;
          }
          *reinterpret_cast<int2*>(&h->valid) = v;
          __syncwarp();
        }
        const uint32_t to = ring_at + slot_in * S::kStep;
#pragma unroll
        for (int u = 0; u < kAttPair; ++u) {
          const int2 h = *reinterpret_cast<const int2*>(&known[(2 * j + u) & (kAttHeads - 1)].valid);
          const long long from = max(h.y, 0) * block_bytes + lane * 16;
          const unsigned char* fk = a.k + from;
          const unsigned char* fv = a.v + from;
#pragma unroll
          for (int i = 0; i < CH; ++i)
            if (token_of[i] < 16) {
              const bool take = token_of[i] < h.x;
              cp_async16_if(to + u * 2 * S::kBlock + to_k[i], fk + i * 512, take);
              cp_async16_if(to + u * 2 * S::kBlock + to_v[i], fv + i * 512, take);
            }
        }
      }
      slot_in = slot_in == S::kStages - 1 ? 0 : slot_in + 1;
      cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j < S::kStages - 1; ++j) fetch(j);

    // ---- the queries: this lane has column g (of each eight), the dims of its keys
    uint32_t qh[RT == 1 ? KS : 1][2], ql[LO ? KS : 1][2];
    Two c_hi[RT], c_lo[RT];  // factors of the rows 2 t and 2 t + 1
    int end[RT][2];          // places that they see
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const int r = tile * ROWS + 8 * u + g;  // step r / group, head r % group
      const bool live = r < a.steps * a.group;
      const int step = live ? r / a.group : 0;
      const long long q_at = (static_cast<long long>(row) * a.steps + step) * a.ld_q +
                             static_cast<long long>(head * a.group + (live ? r - step * a.group : 0)) * a.hd_q;
      float x[4 * KS];
#pragma unroll
      for (int i = 0; i < 4 * KS; ++i) x[i] = 0.0f;
      if (live && 16 * t < a.dim) load_n<16>(a.q, q_at + 16 * t, a.q_type, a.wide_q, x);
      if constexpr (DP > 64) {
        constexpr int N = (DP - 64) / 4;
        if (live && 64 + N * t < a.dim) load_n<N>(a.q, q_at + 64 + N * t, a.q_type, a.wide_q, x + 16);
      }
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < 4 * KS; ++i) most = fmaxf(most, fabsf(x[i]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // the row times 2^e has its largest element in [2^14, 2^15)
      int e = 141 - static_cast<int>(__float_as_uint(most) >> 23);
      if (e < -113) e = 0;  // inf or NaN
      e = min(e, 126);
      const float up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float y = x[4 * s + 2 * k] * up, z = x[4 * s + 2 * k + 1] * up;
          const uint32_t hi = two_halves(y, z);
          if (RT == 1)
            qh[RT == 1 ? s : 0][k] = hi;
          else
            reinterpret_cast<uint32_t*>(query + s * 32)[2 * u + k] = hi;
          if (LO) {
            const float2 back = of_halves(hi);
            ql[LO ? s : 0][k] = two_halves(y - back.x, z - back.y);
          }
        }
      const int sees = len - (a.steps - 1 - step);
      const float d0 = __shfl_sync(0xffffffffu, down, 8 * t), d1 = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      end[u][0] = __shfl_sync(0xffffffffu, sees, 8 * t);
      end[u][1] = __shfl_sync(0xffffffffu, sees, 8 * t + 4);
      c_hi[u] = two(a.c_hi * d0, a.c_hi * d1);
      c_lo[u] = two(a.c_lo * d0, a.c_lo * d1);
    }
    const int all_see = len - (a.steps - 1);  // places that every row sees

    // products: [even, odd dim] x [row 2 t, row 2 t + 1]
    float acc[MT][RT][4];
    Two sum[MT][RT][2];
    float m[RT][2], vref = 0.0f, vinv = 0.0f;
    Two l[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        acc[i][u][0] = acc[i][u][1] = acc[i][u][2] = acc[i][u][3] = 0.0f;
        sum[i][u][0] = sum[i][u][1] = two(0.0f, 0.0f);
      }
      m[u][0] = m[u][1] = kNegInf;
      l[u] = two(0.0f, 0.0f);
    }
    auto flush = [&]() {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          sum[i][u][0] = add2(sum[i][u][0], two(acc[i][u][0], acc[i][u][1]));
          sum[i][u][1] = add2(sum[i][u][1], two(acc[i][u][2], acc[i][u][3]));
          acc[i][u][0] = acc[i][u][1] = acc[i][u][2] = acc[i][u][3] = 0.0f;
        }
    };

    int slot = 0;
    for (int j = 0; j < steps; ++j) {
      fetch(j + S::kStages - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
      __syncwarp();
      unsigned char* at = ring + slot * S::kStep;
      slot = slot == S::kStages - 1 ? 0 : slot + 1;
      BlockHead h[kAttPair];
#pragma unroll
      for (int b = 0; b < kAttPair; ++b) h[b] = known[(2 * j + b) & (kAttHeads - 1)];

      const int place = (b0 + 2 * j) * kCacheBlock;
      // Several steps, and not every query row sees all of these tokens: a row's weight for
      // one that it does not see is 0, and 0 times a NaN is not.  So NaN codes (or all of a
      // block whose scale is none) become zeros here, and the sums that see one NaNs, in the
      // few registers that are left (64 rows of 4096 tokens with 16 query rows: of 128 dims 126
      // us with and without it, of 80 dims 116 and 113).
      if (a.steps > 1 && place + kAttPair * kCacheBlock > all_see) {
        bool any = false;
#pragma unroll
        for (int b = 0; b < kAttPair; ++b) {
          const bool no_scale = !(fabsf(h[b].vs) <= 3.402823466e38f);
          unsigned char* vt = at + b * 2 * S::kBlock + S::kBlock;
          any |= no_scale;
#pragma unroll 1
          for (int i = lane * 16; i < S::kBlock; i += 512) {
            const uint4 x = *reinterpret_cast<const uint4*>(vt + i);
            any |= (__vcmpeq4(x.x & kCodeBits, kCodeBits) | __vcmpeq4(x.y & kCodeBits, kCodeBits) |
                    __vcmpeq4(x.z & kCodeBits, kCodeBits) | __vcmpeq4(x.w & kCodeBits, kCodeBits)) != 0;
          }
        }
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll 1
          for (int i = 0; i < kAttPair * kCacheBlock; ++i) {
            const int tok = i % kCacheBlock, line = DP == 64 ? tok >> 1 : tok;
            const bool second = i >= kCacheBlock;
            const bool no_scale = !(fabsf(second ? h[1].vs : h[0].vs) <= 3.402823466e38f);
            unsigned char* vt = at + (second ? 3 : 1) * S::kBlock + line * 128;
            const int flip = DP == 64 ? (line & 3) << 1 : ((tok >> 1) & 3) << 1, first_of = DP == 64 ? (tok & 1) << 2 : 0;
#pragma unroll
            for (int w = 0; w < VW; ++w) {  // this lane's words of the token
              const int d = DP == 128 ? 16 * g + 4 * w : w < 2 ? 8 * g + 4 * w : 64 + 4 * g;
              uint32_t* word = reinterpret_cast<uint32_t*>(vt + (((first_of | (d >> 4)) ^ flip) << 4) + (d & 15));
              const uint32_t nan = no_scale ? 0xffffffffu : __vcmpeq4(*word & kCodeBits, kCodeBits);
              __syncwarp();  // four lanes have read the same word
              if (nan == 0) continue;
              *word &= ~nan;
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int u = 0; u < RT; ++u)
#pragma unroll
                  for (int k = 0; k < 2; ++k)
                    if ((nan >> 8 * c & 1u) && place + i < end[u][k])
                      acc[2 * w + c / 2][u][2 * (c & 1) + k] = __int_as_float(0x7fc00000);
            }
          }
          __syncwarp();
#pragma unroll
          for (int b = 0; b < kAttPair; ++b)
            if (!(fabsf(h[b].vs) <= 3.402823466e38f)) h[b].vs = 0.0f;
        }
      }

      // scores of the tokens g (0) and g + 8 (1) of each block for the rows 2 t and 2 t + 1
      Two p[kAttPair][RT][2];
#pragma unroll
      for (int b = 0; b < kAttPair; ++b) {
        uint32_t w[2][KS];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned char* kt = at + b * 2 * S::kBlock + i * 8 * S::kRow;
          const uint4 x = *reinterpret_cast<const uint4*>(kt + at_k0);
          w[i][0] = x.x, w[i][1] = x.y, w[i][2] = x.z, w[i][3] = x.w;
          if constexpr (DP == 128) {
            const uint4 y = *reinterpret_cast<const uint4*>(kt + at_k1);
            w[i][4] = y.x, w[i][5] = y.y, w[i][6] = y.z, w[i][7] = y.w;
          } else if constexpr (DP == 96) {
            const uint2 y = *reinterpret_cast<const uint2*>(kt + at_k1);
            w[i][4] = y.x, w[i][5] = y.y;
          }
        }
        float sc[RT][2][4];  // two chains each
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
          for (int k = 0; k < 2; ++k) sc[u][k][0] = sc[u][k][1] = sc[u][k][2] = sc[u][k][3] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint32_t a0 = codes_lo(w[0][s]), a1 = codes_lo(w[1][s]), a2 = codes_hi(w[0][s]), a3 = codes_hi(w[1][s]);
          if constexpr (RT == 1) {
            mma16816(sc[0][s & 1], a0, a1, a2, a3, qh[s][0], qh[s][1]);
            if (LO) mma16816(sc[0][s & 1], a0, a1, a2, a3, ql[LO ? s : 0][0], ql[LO ? s : 0][1]);
          } else {
            const uint4 q = query[s * 32];
            mma16816(sc[0][s & 1], a0, a1, a2, a3, q.x, q.y);
            mma16816(sc[RT - 1][s & 1], a0, a1, a2, a3, q.z, q.w);
          }
        }
        const Two ks = two(h[b].ks, h[b].ks);
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          const Two f_hi = mul2(c_hi[u], ks), f_lo = mul2(c_lo[u], ks);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const Two x = add2(two(sc[u][0][2 * i], sc[u][0][2 * i + 1]), two(sc[u][1][2 * i], sc[u][1][2 * i + 1]));
            p[b][u][i] = fma2(x, f_hi, mul2(x, f_lo));
          }
        }
      }
      if (h[0].valid + h[1].valid < 2 * kCacheBlock || place + 2 * kCacheBlock > all_see) {
#pragma unroll
        for (int b = 0; b < kAttPair; ++b)
#pragma unroll
          for (int u = 0; u < RT; ++u) {
            const int at0 = g + place + b * kCacheBlock, valid = h[b].valid - g;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 x = parts_of(p[b][u][i]);
              const bool there = 8 * i < valid;
              p[b][u][i] = two(there && at0 + 8 * i < end[u][0] ? x.x : kNegInf,
                               there && at0 + 8 * i < end[u][1] ? x.y : kNegInf);
            }
          }
      }
      float mx[RT][2];
      bool grows = false;
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        const float2 x = parts_of(p[0][u][0]), y = parts_of(p[0][u][1]);
        const float2 z = parts_of(p[1][u][0]), w = parts_of(p[1][u][1]);
        mx[u][0] = fmaxf(fmaxf(x.x, y.x), fmaxf(z.x, w.x));
        mx[u][1] = fmaxf(fmaxf(x.y, y.y), fmaxf(z.y, w.y));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          mx[u][0] = fmaxf(mx[u][0], __shfl_xor_sync(0xffffffffu, mx[u][0], o));
          mx[u][1] = fmaxf(mx[u][1], __shfl_xor_sync(0xffffffffu, mx[u][1], o));
        }
        grows |= mx[u][0] > m[u][0] || mx[u][1] > m[u][1];
      }
      const float vmax = fmaxf(fabsf(h[0].vs), fabsf(h[1].vs));  // 0 where there is no page
      if (__any_sync(0xffffffffu, grows || vmax > vref)) {
        const float vn = fmaxf(vref, vmax);
        const float less = vn > vref ? __fdiv_rn(vref, vn) : 1.0f;
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          float alpha[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float mn = fmaxf(m[u][k], mx[u][k]);
            alpha[k] = m[u][k] > kNegInf ? ex2(m[u][k] - mn) : 0.0f;
            m[u][k] = mn;
          }
          l[u] = mul2(l[u], two(alpha[0], alpha[1]));
          const float f0 = alpha[0] * less, f1 = alpha[1] * less;
          const Two both = two(f0, f1);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            acc[i][u][0] *= f0, acc[i][u][1] *= f1, acc[i][u][2] *= f0, acc[i][u][3] *= f1;
            sum[i][u][0] = mul2(sum[i][u][0], both);
            sum[i][u][1] = mul2(sum[i][u][1], both);
          }
        }
        if (vn > vref) vinv = __fdiv_rn(1.0f, vn);
        vref = vn;
      }
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        const Two base = two(m[u][0] > kNegInf ? kUp - m[u][0] : 0.0f, m[u][1] > kNegInf ? kUp - m[u][1] : 0.0f);
#pragma unroll
        for (int b = 0; b < kAttPair; ++b)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 x = parts_of(add2(p[b][u][i], base));
            p[b][u][i] = two(ex2(x.x), ex2(x.y));
          }
        l[u] = add2(l[u], add2(add2(p[0][u][0], p[0][u][1]), add2(p[1][u][0], p[1][u][1])));
      }

#pragma unroll
      for (int b = 0; b < kAttPair; ++b) {
        const float share = h[b].vs * vinv;
        const Two ratio = two(share, share), minus = two(-1.0f, -1.0f);
        uint32_t ph[RT][2], pl[RT][2];  // rounded, and what that left: of row g, tokens 2 t, 2 t + 1 (and + 8)
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const Two x = mul2(p[b][u][i], ratio);
            const float2 y = parts_of(x);
            const uint32_t hi = two_halves(y.x, y.y);
            const float2 back = of_halves(hi);
            const float2 rest = parts_of(fma2(two(back.x, back.y), minus, x));
            ph[u][i] = turned(hi);
            pl[u][i] = turned(two_halves(rest.x, rest.y));
          }
        // values: this lane has tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
        uint32_t v[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned char* vt = at + b * 2 * S::kBlock + (i >> 1) * 8 * S::kRow;
          if constexpr (DP == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(vt + (i & 1 ? at_v1 : at_v0));
            v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(vt + (i & 1 ? at_v1 : at_v0));
            v[i][0] = x.x, v[i][1] = x.y;
            if constexpr (DP == 96) v[i][2] = *reinterpret_cast<const uint32_t*>(vt + (i & 1 ? at_v3 : at_v2));
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5140), a1 = __byte_perm(v[0][w], v[1][w], 0x7362);
          const uint32_t e0 = __byte_perm(v[2][w], v[3][w], 0x5140), e1 = __byte_perm(v[2][w], v[3][w], 0x7362);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = i ? a1 : a0, y = i ? e1 : e0;
            const uint32_t c0 = codes_lo(x), c1 = codes_hi(x), c2 = codes_lo(y), c3 = codes_hi(y);
#pragma unroll
            for (int u = 0; u < RT; ++u) {
              mma16816(acc[2 * w + i][u], c0, c1, c2, c3, ph[u][0], ph[u][1]);
              mma16816(acc[2 * w + i][u], c0, c1, c2, c3, pl[u][0], pl[u][1]);
            }
          }
        }
      }
      if ((j & (kAttFlush - 1)) == kAttFlush - 1) flush();
      __syncwarp();  // the slot may be filled again
    }
    cp_async_wait_all();
    flush();

    // this lane's dims of the rows 2 t and 2 t + 1: 4 w + i of word w
    constexpr int N1 = DP == 128 ? 16 : 8, N2 = DP == 96 ? 4 : 0;
    const int d1 = N1 * g, d2 = 64 + 4 * g;
    const bool whole = !CL && n == nb;
    float* to = nullptr;
    if (CL) {
      __syncwarp();
      to = reinterpret_cast<float*>(ring);  // its copies are done
    } else if (!whole) {
      to = a.parts + ((static_cast<long long>(team) * a.tiles + tile) * 2 + part) * part_floats(ROWS, a.dim);
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const float2 l2 = parts_of(l[u]);
      float ls[2] = {l2.x, l2.y};
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        ls[0] += __shfl_xor_sync(0xffffffffu, ls[0], o);
        ls[1] += __shfl_xor_sync(0xffffffffu, ls[1], o);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int local = 8 * u + 2 * t + k, r = tile * ROWS + local;
        if (r >= a.steps * a.group) continue;
        const float by = whole ? (ls[k] > 0.0f || ls[k] != ls[k] ? __fdiv_rn(vref, ls[k]) : 0.0f) : vref;
        float y[4 * VW];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const float2 even = parts_of(sum[i][u][0]), odd = parts_of(sum[i][u][1]);
          y[2 * i] = (k ? even.y : even.x) * by;
          y[2 * i + 1] = (k ? odd.y : odd.x) * by;
        }
        if (!whole) {
          if (d1 < a.dim) store_n<N1>(to, local * a.dim + d1, kOpsF32, true, y);
          if constexpr (N2 > 0) {
            if (d2 < a.dim) store_n<N2>(to, local * a.dim + d2, kOpsF32, true, y + N1);
          }
          if (g == 0) {
            to[ROWS * a.dim + local] = m[u][k];
            to[ROWS * a.dim + ROWS + local] = ls[k];
          }
        } else {
          const int step = r / a.group;
          const long long o = (static_cast<long long>(row) * a.steps + step) * a.ld_out +
                              static_cast<long long>(head * a.group + r - step * a.group) * a.hd_out;
          if (d1 < a.dim) store_n<N1>(a.out, o + d1, a.out_type, a.wide_out, y);
          if constexpr (N2 > 0) {
            if (d2 < a.dim) store_n<N2>(a.out, o + d2, a.out_type, a.wide_out, y + N1);
          }
        }
      }
    }
    part = 1;
  }

  if constexpr (CL) {
    cg::cluster_group cl = cg::this_cluster();
    cluster_sync_all();  // every warp's part is there
    const int rows = min(ROWS, a.steps * a.group - tile * ROWS), quads = a.dim / 4;
    for (int r = cl.block_rank(); r < rows; r += a.members) {
      // this warp takes the parts of its likes in all CTAs, then warp 0 the warps'
      float pm = kNegInf, pl = 0.0f;
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      auto add = [&](float qm, float ql, float4 v) {
        const float mn = fmaxf(pm, qm);
        const float s = pm > kNegInf ? ex2(pm - mn) : 1.0f;
        const float u = qm > kNegInf ? ex2(qm - mn) : 1.0f;  // a part that sees nothing is zeros, or NaNs
        pm = mn;
        pl = pl * s + ql * u;
        y.x = y.x * s + v.x * u, y.y = y.y * s + v.y * u, y.z = y.z * s + v.z * u, y.w = y.w * s + v.w * u;
      };
#pragma unroll 4
      for (int c = 0; c < a.members; ++c) {
        const float* from = cl.map_shared_rank(reinterpret_cast<float*>(ring), c);
        add(from[ROWS * a.dim + r], from[ROWS * a.dim + ROWS + r],
            lane < quads ? reinterpret_cast<const float4*>(from + r * a.dim)[lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
      }
      if (lane < quads) joined[warp][lane] = y;
      if (lane == 0) joined_ml[warp] = make_float2(pm, pl);
      __syncthreads();
      if (warp == 0) {
        pm = kNegInf;
        pl = 0.0f;
        y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < NW; ++w)
          add(joined_ml[w].x, joined_ml[w].y, lane < quads ? joined[w][lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        if (lane < quads) {
          const float inv = pl > 0.0f || pl != pl ? __fdiv_rn(1.0f, pl) : 0.0f;
          const int qr = tile * ROWS + r, step = qr / a.group;
          const long long o = (static_cast<long long>(row) * a.steps + step) * a.ld_out +
                              static_cast<long long>(head * a.group + qr - step * a.group) * a.hd_out + 4 * lane;
          store_any(a.out, o, a.out_type, y.x * inv);
          store_any(a.out, o + 1, a.out_type, y.y * inv);
          store_any(a.out, o + 2, a.out_type, y.z * inv);
          store_any(a.out, o + 3, a.out_type, y.w * inv);
        }
      }
      __syncthreads();
    }
    cluster_sync_all();  // nobody reads another's shared memory any more
  }
}

// Of a join's CTA. Few warps where there are many (row, head) of few parts each (64 rows of
// 4096 tokens 102 us, 113 with many); many, with fewer query rows and more parts on their
// way, where a few are split over most of the card's warps (one row of 131072 tokens 58 us,
// 61 with as many rows and parts as the others).
template <bool MANY>
struct JoinShape {
  static constexpr int kWarps = MANY ? 16 : 4;
  static constexpr int kRows = MANY ? 2 : 4;   // query rows
  static constexpr int kAhead = MANY ? 6 : 2;  // a warp's parts on their way
};

// One CTA per (row, head, some rows of a tile): the parts of its blocks joined, in their
// order; nothing to do where one warp had them all.  A warp takes every W-th part.
template <bool MANY>
__global__ void __launch_bounds__(JoinShape<MANY>::kWarps * 32) cache_attend_join_kernel(const AttendArgs a) {
  using S = JoinShape<MANY>;
  constexpr int W = S::kWarps, R = S::kRows, AHEAD = S::kAhead;
  extern __shared__ float4 os[];  // [W][R][dim / 4]
  __shared__ float ms[W][R], ls[W][R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slices = a.tile_rows / R;
  const int slice = blockIdx.x % slices;
  const int tile = blockIdx.x / slices % a.tiles;
  const int head = blockIdx.x / (slices * a.tiles) % a.heads;
  const int row = blockIdx.x / (slices * a.tiles) / a.heads;
  grid_wait();
  grid_release();
  const int rows = min(R, a.steps * a.group - tile * a.tile_rows - slice * R);  // of this CTA
  if (rows <= 0) return;
  const int f0 = a.first[row], counted = a.first[row + 1] - f0, blocks = a.first[a.rows];
  const int quads = a.dim / 4;
  float total = 0.0f;
  int used = 0;
  if (counted > 0) {
    const long long all = static_cast<long long>(blocks) * a.heads;
    const long long each = blocks_each(a, all);
    const long long f = static_cast<long long>(f0) * a.heads + static_cast<long long>(head) * counted;
    int w0, w1;
    if (all < INT_MAX) {
      w0 = static_cast<int>(f + kAttStart) / static_cast<int>(each);
      w1 = static_cast<int>(f + counted - 1) / static_cast<int>(each);
    } else {
      w0 = static_cast<int>((f + kAttStart) / each);
      w1 = static_cast<int>((f + counted - 1) / each);
    }
    if (w0 == w1) return;  // teams w0 to w1 have blocks of it
    used = min(W, w1 - w0 + 1);
    float m[R], l[R];
    float4 x[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      m[i] = kNegInf;
      l[i] = 0.0f;
      x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (int w = w0 + warp; w <= w1; w += W * AHEAD) {
      float ml[AHEAD];
      float4 v[AHEAD][R];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int at = w + u * W;
        const int which = at * each < f;  // its second part, after the end of another
        const float* from = a.parts + ((static_cast<long long>(at) * a.tiles + tile) * 2 + which) * part_floats(a.tile_rows, a.dim);
        ml[u] = lane < R ? kNegInf : 0.0f;
        if (at <= w1 && lane < 2 * R && lane % R < rows)
          ml[u] = from[a.tile_rows * (a.dim + lane / R) + slice * R + lane % R];
#pragma unroll
        for (int i = 0; i < R; ++i)
          v[u][i] = at <= w1 && i < rows && lane < quads
                        ? reinterpret_cast<const float4*>(from)[(slice * R + i) * quads + lane]
                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float pm = __shfl_sync(0xffffffffu, ml[u], i), pl = __shfl_sync(0xffffffffu, ml[u], R + i);
          const float mn = fmaxf(m[i], pm);
          const float s = m[i] > kNegInf ? ex2(m[i] - mn) : 1.0f;
          const float t = pm > kNegInf ? ex2(pm - mn) : 1.0f;  // a part that sees nothing is zeros, or NaNs
          m[i] = mn;
          l[i] = l[i] * s + pl * t;
          x[i].x = x[i].x * s + v[u][i].x * t;
          x[i].y = x[i].y * s + v[u][i].y * t;
          x[i].z = x[i].z * s + v[u][i].z * t;
          x[i].w = x[i].w * s + v[u][i].w * t;
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (lane < quads) os[(warp * R + i) * quads + lane] = x[i];
      if (lane == i) {
        ms[warp][i] = m[i];
        ls[warp][i] = l[i];
      }
    }
    __syncthreads();
  }
  // a warp to a query row, four dims to a lane
  if (warp >= rows) return;
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // an empty row's
  float mn = kNegInf;
  for (int w = 0; w < used; ++w) mn = fmaxf(mn, ms[w][warp]);
  for (int w = 0; w < used; ++w) {
    const float t = ms[w][warp] > kNegInf ? ex2(ms[w][warp] - mn) : 1.0f;
    total += ls[w][warp] * t;
    if (lane < quads) {
      const float4 v = os[(w * R + warp) * quads + lane];
      y.x += v.x * t, y.y += v.y * t, y.z += v.z * t, y.w += v.w * t;
    }
  }
  if (lane >= quads) return;
  const float inv = total > 0.0f || total != total ? __fdiv_rn(1.0f, total) : 0.0f;
  const int qr = tile * a.tile_rows + slice * R + warp, step = qr / a.group;
  const long long o = (static_cast<long long>(row) * a.steps + step) * a.ld_out +
                      static_cast<long long>(head * a.group + qr - step * a.group) * a.hd_out + 4 * lane;
  store_any(a.out, o, a.out_type, y.x * inv);
  store_any(a.out, o + 1, a.out_type, y.y * inv);
  store_any(a.out, o + 2, a.out_type, y.z * inv);
  store_any(a.out, o + 3, a.out_type, y.w * inv);
}

constexpr int kAttMaxSmem = 227 * 1024;

// A warp of a cluster takes at most this many steps, whatever the lengths are: longer
// tables go to the parts, which are equal for any lengths.
constexpr int kClusterSteps = 32;

struct Plan {
  int dp, rt, warps, grid, tiles, teams, least, members;
  size_t smem, parts_bytes;
};
// Warps, their shared memory, and the largest cluster of which `units` run at once (0:
// they do not as single CTAs either).
template <int DP, int RT>
void shape(Plan* p, int* warp_bytes, int* ctas, long long units) {
  using S = AttShape<DP, RT>;
  p->warps = S::kWarps;
  *warp_bytes = S::kWarp;
  *ctas = S::kCtas;
  p->members = 8;
  while (p->members &&
         units > clusters_at_once<cache_attend_kernel<DP, RT, false, true>>(p->members, S::kWarps * 32, S::kWarps * S::kWarp))
    p->members /= 2;
}
Plan plan(const verbo_cache& c, int heads, int steps, int q_type) {
  Plan p{};
  const int rows = steps * (heads / c.heads), sms = sm_count();
  p.dp = c.dim <= 64 ? 64 : c.dim <= 96 ? 96 : 128;
  // More than 8 query rows: 16 at a time, twice the products for one conversion and one
  // copy of the keys and values: rows of 100003 and 131072 tokens with 16 query rows take
  // 107 us, 130 in two tiles of 8.  fp32 queries, in two parts, leave no registers for it.
  p.rt = rows > 8 && q_type != kOpsF32 ? 2 : 1;
  p.tiles = (rows + 8 * p.rt - 1) / (8 * p.rt);
  const long long units = static_cast<long long>(c.rows) * c.heads * p.tiles;
  int warp = 0, ctas = 1;
  if (p.dp == 64)
    p.rt == 1 ? shape<64, 1>(&p, &warp, &ctas, units) : shape<64, 2>(&p, &warp, &ctas, units);
  else if (p.dp == 96)
    p.rt == 1 ? shape<96, 1>(&p, &warp, &ctas, units) : shape<96, 2>(&p, &warp, &ctas, units);
  else
    p.rt == 1 ? shape<128, 1>(&p, &warp, &ctas, units) : shape<128, 2>(&p, &warp, &ctas, units);
  // Few (row, head, tile): a cluster for each, as large as all of them fit at once: no
  // second kernel and no search.  One row of 1500 tokens 6.8 us, 11.3 split over the card;
  // 18 rows of 8000 tokens, a CTA to a (row, head), 56 and 65.  Lengths are not known
  // before the launch: long or uneven rows lose by it, but not more than kClusterSteps
  // take.  One row of 49152 tokens 38 us, 34 split; with three of 100 beside it, on half
  // the CTAs, 66 and 36 (not taken: 49152 tokens are 48 steps then).
  const long long most = static_cast<long long>(c.width) * (c.page / kCacheBlock);  // blocks of a row
  if (p.members && most <= 2ll * kClusterSteps * p.warps * p.members) {
    p.grid = static_cast<int>(units) * p.members;
    p.smem = static_cast<size_t>(p.warps) * warp;
    return p;
  }
  p.members = 0;
  p.smem = static_cast<size_t>(p.warps) * warp + (static_cast<size_t>(c.rows) + 1) * 4;
  // very many rows leave room for one CTA an SM
  if (ctas * (p.smem + 1024) > kAttMaxSmem + 1024) ctas = 1;
  p.grid = sms * ctas;
  p.teams = std::max(1, p.grid * p.warps / p.tiles);
  p.least = 2;
  p.parts_bytes = static_cast<size_t>(p.teams) * p.tiles * 2 * part_floats(8 * p.rt, c.dim) * 4;
  return p;
}

template <int DP, int RT, bool LO>
cudaError_t run_attend(const AttendArgs& a, const Plan& p, cudaStream_t s) {
  constexpr int threads = AttShape<DP, RT>::kWarps * 32, warps = AttShape<DP, RT>::kWarps * AttShape<DP, RT>::kWarp;
  if (p.members) {
    const cudaError_t e = allow_smem<cache_attend_kernel<DP, RT, LO, true>>(warps);
    if (e != cudaSuccess) return e;
    return launch_chained(cache_attend_kernel<DP, RT, LO, true>, static_cast<unsigned>(p.grid), threads, p.smem,
                          p.members, s, a);
  }
  constexpr int most = warps + (VERBO_CACHE_MAX_ROWS + 1) * 4;
  static_assert(most + 64 <= kAttMaxSmem, "shared memory");
  const cudaError_t e = allow_smem<cache_attend_kernel<DP, RT, LO, false>>(most);
  if (e != cudaSuccess) return e;
  return launch_chained(cache_attend_kernel<DP, RT, LO, false>, static_cast<unsigned>(p.grid), threads, p.smem, 1, s, a);
}
template <int DP>
cudaError_t run_attend(const AttendArgs& a, const Plan& p, cudaStream_t s) {
  if (p.rt == 2) return run_attend<DP, 2, false>(a, p, s);
  return a.q_type == kOpsF32 ? run_attend<DP, 1, true>(a, p, s) : run_attend<DP, 1, false>(a, p, s);
}

template <bool MANY>
cudaError_t run_join(const AttendArgs& a, long long ctas, cudaStream_t s) {
  using S = JoinShape<MANY>;
  return launch_chained(cache_attend_join_kernel<MANY>, static_cast<unsigned>(ctas), S::kWarps * 32,
                        static_cast<size_t>(S::kWarps) * S::kRows * a.dim * 4, 1, s, a);
}

}  // namespace

size_t cache_attend_bytes(const verbo_cache& c, int heads, int steps, int q_type) {
  const Plan p = plan(c, heads, steps, q_type);
  return p.members || c.rows == 0 ? 0 : (p.parts_bytes + (static_cast<size_t>(c.rows) + 1) * 4 + 15) / 16 * 16;
}

cudaError_t launch_cache_attend(const verbo_cache& c, int layer, const CacheQuery& x, int q_type, int out_type,
                                cudaStream_t s) {
  const Plan p = plan(c, x.heads, x.steps, q_type);
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
  a.tile_rows = 8 * p.rt;
  a.tiles = p.tiles;
  a.teams = p.teams;
  a.least = p.least;
  a.members = p.members;
  a.q_type = q_type;
  a.out_type = out_type;
  const double f = static_cast<double>(x.scale) * kLog2e;
  a.c_hi = static_cast<float>(f);
  a.c_lo = static_cast<float>(f - static_cast<double>(a.c_hi));
  a.parts = static_cast<float*>(x.workspace);
  a.first = reinterpret_cast<int*>(static_cast<char*>(x.workspace) + p.parts_bytes);
  const auto wide = [](const void* p, long long ld, long long hd, int type) {
    const int n = type == kOpsF32 ? 4 : 8;  // elements of 16 bytes
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % n == 0 && hd % n == 0;
  };
  a.wide_q = wide(x.q, x.ld_q, x.hd_q, q_type);
  a.wide_out = wide(x.out, x.ld_out, x.hd_out, out_type);
  const long long tiles = static_cast<long long>(c.rows) * c.heads * p.tiles;
  const bool many = tiles * (a.tile_rows / JoinShape<false>::kRows) < 2 * sm_count();
  const long long joins = tiles * (a.tile_rows / (many ? JoinShape<true>::kRows : JoinShape<false>::kRows));
  if (joins > INT_MAX) return cudaErrorInvalidConfiguration;
  const cudaError_t e = p.dp == 64   ? run_attend<64>(a, p, s)
                        : p.dp == 96 ? run_attend<96>(a, p, s)
                                     : run_attend<128>(a, p, s);
  if (e != cudaSuccess || p.members) return e;
  return many ? run_join<true>(a, joins, s) : run_join<false>(a, joins, s);
}

}  // namespace vb
