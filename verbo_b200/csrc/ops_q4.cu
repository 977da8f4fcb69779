// Products with 4-bit weights (include/verbo_ops.h): y = x W^T + b with
// W[o][i] = s[o][g] (q[o][i] - z[o][g]) and the activations in their own type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "device.cuh"
#include "ops.cuh"

namespace vb {
namespace {

constexpr int kThreadsQ4 = 256;
constexpr int kWarpsQ4 = kThreadsQ4 / 32;
constexpr int kAhead = 4;  // chunks whose loads a warp keeps in flight

// ================================================================== pack ==
// One thread per 32-bit word of the chunks' nibbles.  Word j of lane (g, t) =
// (lane / 4, lane % 4) holds the lane's A fragment of k-step j: rows g and
// g + 8, and of the chunk's block p = j / 2 the four weights k, k + 1, k + 2,
// k + 3 from k = 32 p + 8 t + 4 (j % 2).  (The sum over k has no order, so the
// lane's share of a block is taken as 8 neighbouring weights, which lets x be
// read as it lies.)  Nibbles, low to high: (g, k), (g+8, k), (g, k+2),
// (g+8, k+2), (g, k+1), (g+8, k+1), (g, k+3), (g+8, k+3): four masks with
// 0x000f000f at shifts 0, 4, 8, 12 give the pairs of a0, a1, a2, a3.
__device__ __forceinline__ uint32_t q4_nibble(const Q4Mat& m, const unsigned char* q, int o, int i) {
  if (o >= m.outs || i >= m.ins) return 0;
  const int blk = i >> 5, e = i & 31;
  const unsigned char b = q[static_cast<size_t>(o) * (m.ins / 2) + blk * 16 + (e & 15)];
  return e < 16 ? b & 15u : b >> 4;
}

__global__ void q4_pack_kernel(Q4Mat m, const unsigned char* __restrict__ q, const uint16_t* __restrict__ s,
                               const unsigned char* __restrict__ z, unsigned char* __restrict__ tiles) {
  const long long nchunk = static_cast<long long>(m.ntile) * m.nkc;
  const int sets = kQ4Chunk / m.span;
  const int groups = (m.ins + m.group - 1) / m.group;
  for (long long c = blockIdx.x; c < nchunk; c += gridDim.x) {
    const int tile = static_cast<int>(c / m.nkc), kc = static_cast<int>(c % m.nkc);
    unsigned char* dst = tiles + c * m.chunk_bytes;
    const int w = threadIdx.x;  // 256 words of nibbles
    {
      const int half = w >> 7, lane = (w >> 2) & 31, j = half * 4 + (w & 3);
      const int g = lane >> 2, t = lane & 3;
      const int k = kc * kQ4Chunk + 32 * (j >> 1) + 8 * t + 4 * (j & 1);
      const int r = tile * kQ4Rows + g;
      uint32_t v = 0;
      const int dk[8] = {0, 0, 2, 2, 1, 1, 3, 3};
#pragma unroll
      for (int n = 0; n < 8; ++n) v |= q4_nibble(m, q, r + 8 * (n & 1), k + dk[n]) << (4 * n);
      reinterpret_cast<uint32_t*>(dst)[w] = v;
    }
    if (w < 16 * sets) {  // [g][set][row g, row g + 8]
      const int g = w / (2 * sets), set = (w / 2) % sets, o = tile * kQ4Rows + g + 8 * (w & 1);
      const int i = kc * kQ4Chunk + set * m.span;
      const bool in = o < m.outs && i < m.ins;
      const size_t at = in ? static_cast<size_t>(o) * groups + i / m.group : 0;
      reinterpret_cast<uint16_t*>(dst + 1024)[w] = in ? s[at] : uint16_t(0);
      if (m.zeros) dst[1024 + 32 * sets + w] = in ? z[at] & 15 : 0;
    }
  }
}

// ================================================================ matvec ==
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// d = a b + d, or a b with START.
template <bool BF16, bool START>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const float c0 = START ? 0.0f : d[0], c1 = START ? 0.0f : d[1], c2 = START ? 0.0f : d[2], c3 = START ? 0.0f : d[3];
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// The zero points of rows g and g + 8 as unpack() wants them.
template <bool BF16>
struct Q4Zero {
  uint32_t g, h;
  __device__ __forceinline__ Q4Zero(uint32_t zg, uint32_t zh) {
    zg |= zg << 16;
    zh |= zh << 16;
    g = (BF16 ? 0x43004300u : 0x64006400u) | zg;
    h = BF16 ? 0x43004300u | zh : 0xd400d400u | (zh << 4);
  }
};

// A word's eight weights minus their zero points: the A fragment of one k-step,
// exact.  0x6400 | q is the fp16 1024 + q, and with q four bits higher
// 1024 + 16 q, of which a sixteenth minus (64 + z) is q - z; 0x4300 | q is the
// bf16 128 + q, whose mantissa has no room for the second form.
template <bool BF16>
__device__ __forceinline__ void unpack(uint32_t w, const Q4Zero<BF16>& z, uint32_t (&a)[4]) {
  if (BF16) {
    a[0] = sub2((w & 0x000f000fu) | 0x43004300u, z.g, true);
    a[1] = sub2(((w >> 4) & 0x000f000fu) | 0x43004300u, z.h, true);
    a[2] = sub2(((w >> 8) & 0x000f000fu) | 0x43004300u, z.g, true);
    a[3] = sub2(((w >> 12) & 0x000f000fu) | 0x43004300u, z.h, true);
  } else {
    const uint32_t v = w >> 8, sixteenth = 0x2c002c00u;
    auto upper = [&](uint32_t u) {
      u = (u & 0x00f000f0u) | 0x64006400u;
      const __half2 d = __hfma2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&sixteenth),
                                *reinterpret_cast<const __half2*>(&z.h));
      return *reinterpret_cast<const uint32_t*>(&d);
    };
    a[0] = sub2((w & 0x000f000fu) | 0x64006400u, z.g, false);
    a[1] = upper(w);
    a[2] = sub2((v & 0x000f000fu) | 0x64006400u, z.g, false);
    a[3] = upper(v);
  }
}

// What one lane holds of a chunk.
template <int SETS, bool ZP>
struct Q4Buf {
  __device__ __forceinline__ uint32_t word(int j) const {
    const uint4& w = j < 4 ? w0 : w1;
    return (j & 3) == 0 ? w.x : (j & 3) == 1 ? w.y : (j & 3) == 2 ? w.z : w.w;
  }
  template <bool BF16>
  __device__ __forceinline__ Q4Zero<BF16> zero(int set) const {
    if (!ZP) return Q4Zero<BF16>(8u, 8u);
    const uint32_t v = z[set >> 1] >> (16 * (set & 1));
    return Q4Zero<BF16>(v & 15u, (v >> 8) & 15u);
  }
  __device__ __forceinline__ float2 scale(int set) const { return __half22float2(*reinterpret_cast<const __half2*>(&s[set])); }
  uint4 w0, w1;
  uint32_t s[SETS];                 // scales of rows g, g + 8 per set
  uint32_t z[ZP ? (SETS + 1) / 2 : 1];  // zero points, two bytes per set
  __device__ __forceinline__ void load(const unsigned char* p, int lane) {
    w0 = ld_stream16(p + lane * 16);
    w1 = ld_stream16(p + 512 + lane * 16);
    const unsigned char* sp = p + 1024 + (lane >> 2) * (4 * SETS);
    if (SETS == 4) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(sp));
      s[0] = v.x, s[1 % SETS] = v.y, s[2 % SETS] = v.z, s[3 % SETS] = v.w;
    } else if (SETS == 2) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(sp));
      s[0] = v.x, s[1 % SETS] = v.y;
    } else {
      s[0] = __ldg(reinterpret_cast<const unsigned*>(sp));
    }
    if (ZP) {
      const unsigned char* zp = p + 1024 + 32 * SETS + (lane >> 2) * (2 * SETS);
      if (SETS == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(zp));
        z[0] = v.x, z[(SETS + 1) / 2 - 1] = v.y;
      } else if (SETS == 2) {
        z[0] = __ldg(reinterpret_cast<const unsigned*>(zp));
      } else {
        z[0] = __ldg(reinterpret_cast<const unsigned short*>(zp));
      }
    }
  }
};

struct Q4Kernel {
  Q4Mat m;
  const void* x;   // the pass's first row
  long long ldx;
  int tokens;      // rows of x in this pass
  int cols;        // columns of B: tokens, or 3 per token for fp32 x
  int xstride;     // bytes from one column to the next in shared memory
  void* y;
  long long ldy;
  int y_type;
  bool wide;  // 16-bit x whose rows start on 16 bytes
  int kq;     // q4_tile_kernel: groups of warps along the inputs
};

// Three bf16 that sum to v exactly; an infinity or a NaN goes through the first.
__device__ __forceinline__ void split3(float v, uint16_t (&p)[3]) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    p[0] = v != v ? 0x7fc0u : static_cast<uint16_t>(u >> 16);
    p[1] = p[2] = 0;
    return;
  }
  const float r = v - __uint_as_float(u & 0xffff0000u);
  const float l = r - __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  p[0] = static_cast<uint16_t>(u >> 16);
  p[1] = static_cast<uint16_t>(__float_as_uint(r) >> 16);
  p[2] = static_cast<uint16_t>(__float_as_uint(l) >> 16);
}

__device__ __forceinline__ void q4_store(const Q4Kernel& a, int token, int o, float v) {
  const long long at = token * a.ldy + o;
  if (a.y_type == kOpsF32)
    static_cast<float*>(a.y)[at] = v;
  else if (a.y_type == kOpsF16)
    static_cast<__half*>(a.y)[at] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
}

// The bound is reading the matrix once.  A tile is 16 outputs times all inputs;
// a CTA takes a run of tiles and its warps equal shares of the run's chunks, so
// each warp streams one contiguous piece of memory, kAhead chunks ahead, in
// registers.  x lies in shared memory, one column after the other as in memory;
// a lane's B fragment of two k-steps is 16 neighbouring bytes of a column
// (columns 64 mod 128 bytes apart: the 8 lanes of a quarter warp hit 32 banks).
// The weights are unpacked to q - z, exact in 16 bits, and mma.sync sums a
// group's products in fp32; the group's scale multiplies that sum.  fp32 x is
// cut into three bf16 parts of 8 bits each (24 bits: exact), three columns of B
// that are added at the end.
// A tile whose chunks fall to several warps is summed over the warps' partial
// sums in shared memory, in the order of the warps.
template <bool BF16, bool SPLIT, int NT, int SETS, bool ZP>
__global__ void __launch_bounds__(kThreadsQ4, NT <= 2 ? 2 : 1) q4_kernel(const Q4Kernel a) {
  constexpr int PER = SPLIT ? 2 : 8;  // tokens per 8 columns
  extern __shared__ __align__(16) unsigned char smem_q4[];
  // slots: per warp the partial sums of its first tile, of its last, and one for
  // the tile at hand; [NT][8 columns][16 rows] each
  constexpr int SLOT = NT * 128;
  float* slots = reinterpret_cast<float*>(smem_q4);
  unsigned char* xs = smem_q4 + 3 * kWarpsQ4 * SLOT * 4;
  const Q4Mat& m = a.m;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  const int tile0 = static_cast<int>(static_cast<long long>(m.ntile) * blockIdx.x / gridDim.x);
  const int tile1 = static_cast<int>(static_cast<long long>(m.ntile) * (blockIdx.x + 1) / gridDim.x);
  const int run = (tile1 - tile0) * m.nkc;
  const int first = static_cast<int>(static_cast<long long>(run) * warp / kWarpsQ4);
  const int last = static_cast<int>(static_cast<long long>(run) * (warp + 1) / kWarpsQ4);
  const unsigned char* src = m.tiles + (static_cast<long long>(tile0) * m.nkc + first) * m.chunk_bytes;

  Q4Buf<SETS, ZP> buf[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (first + i < last) buf[i].load(src + static_cast<long long>(i) * m.chunk_bytes, lane);
  src += static_cast<long long>(kAhead) * m.chunk_bytes;

  grid_wait();  // the weights are the handle's; x comes from the grid before
  const int kp = m.nkc * kQ4Chunk;
  if (SPLIT) {
    const float* x = static_cast<const float*>(a.x);
    for (int tok = 0; tok < a.tokens; ++tok)
      for (int k = tid; k < kp; k += kThreadsQ4) {
        uint16_t part[3];
        split3(k < m.ins ? x[tok * a.ldx + k] : 0.0f, part);
        unsigned char* at = xs + static_cast<size_t>(3 * tok) * a.xstride + 2 * k;
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<uint16_t*>(at + i * a.xstride) = part[i];
      }
  } else {
    const uint16_t* x = static_cast<const uint16_t*>(a.x);
    for (int tok = 0; tok < a.tokens; ++tok) {
      unsigned char* at = xs + static_cast<size_t>(tok) * a.xstride;
      const uint16_t* row = x + tok * a.ldx;
      for (int k = tid * 8; k < kp; k += kThreadsQ4 * 8) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < m.ins) {  // ins is a multiple of 32
          if (a.wide) {
            v = *reinterpret_cast<const uint4*>(row + k);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = row[k + 2 * j] | static_cast<uint32_t>(row[k + 2 * j + 1]) << 16;
            v = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        *reinterpret_cast<uint4*>(at + 2 * k) = v;
      }
    }
  }
  __syncthreads();

  // column of B that this lane reads in each group of 8 (past the last one: the
  // last, whose sums are then not stored)
  const unsigned char* xcol[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    int c = SPLIT ? n * 6 + min(g, 5) : n * 8 + g;
    xcol[n] = xs + static_cast<size_t>(min(c, a.cols - 1)) * a.xstride + t * 16;
  }

  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

  float* mine = slots + warp * 3 * SLOT;
  auto spill = [&](float* slot) {  // acc -> [n][column][row]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      slot[n * 128 + (2 * t) * 16 + g] = acc[n][0];
      slot[n * 128 + (2 * t + 1) * 16 + g] = acc[n][1];
      slot[n * 128 + (2 * t) * 16 + g + 8] = acc[n][2];
      slot[n * 128 + (2 * t + 1) * 16 + g + 8] = acc[n][3];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
    }
  };
  auto finish = [&](int tile, int tok, int r, float v) {
    const int o = tile * kQ4Rows + r;
    if (o < m.outs) q4_store(a, tok, o, m.bias ? v + m.bias[o] : v);
  };
  // one warp stores a whole tile out of a slot
  auto store_tile = [&](int tile, const float* slot) {
    for (int e = lane; e < a.tokens * 16; e += 32) {
      const int tok = e >> 4, r = e & 15;
      const float* col = slot + (tok / PER) * 128 + (tok % PER) * (SPLIT ? 3 : 1) * 16 + r;
      finish(tile, tok, r, SPLIT ? col[0] + (col[16] + col[32]) : col[0]);
    }
  };

  int kc = first % m.nkc, tile = tile0 + first / m.nkc;
  const bool starts_inside = kc != 0;
  bool first_part = starts_inside;  // the tile at hand began in an earlier warp's share
  for (int i0 = first; i0 < last; i0 += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      if (i0 + d >= last) break;
      Q4Buf<SETS, ZP>& b = buf[d];
      const int xoff = kc * (kQ4Chunk * 2);
#pragma unroll
      for (int set = 0; set < SETS; ++set) {
        constexpr int BLK = 4 / SETS;  // 32-blocks per set
        const Q4Zero<BF16> z = b.template zero<BF16>(set);
        float part[NT][4];
#pragma unroll
        for (int p = set * BLK; p < (set + 1) * BLK; ++p) {
          uint32_t fa[2][4];
          unpack<BF16>(b.word(2 * p), z, fa[0]);
          unpack<BF16>(b.word(2 * p + 1), z, fa[1]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 f = *reinterpret_cast<const uint4*>(xcol[n] + xoff + p * 64);
            if (p == set * BLK)
              mma16816<BF16, true>(part[n], fa[0], f.x, f.y);
            else
              mma16816<BF16, false>(part[n], fa[0], f.x, f.y);
            mma16816<BF16, false>(part[n], fa[1], f.z, f.w);
          }
        }
        const float2 sc = b.scale(set);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(sc.x, part[n][0], acc[n][0]);
          acc[n][1] = fmaf(sc.x, part[n][1], acc[n][1]);
          acc[n][2] = fmaf(sc.y, part[n][2], acc[n][2]);
          acc[n][3] = fmaf(sc.y, part[n][3], acc[n][3]);
        }
      }
      if (i0 + d + kAhead < last) b.load(src, lane);
      src += m.chunk_bytes;
      if (++kc == m.nkc) {
        if (first_part) {
          spill(mine);
          first_part = false;
        } else {
          spill(mine + 2 * SLOT);
          __syncwarp();
          store_tile(tile, mine + 2 * SLOT);
          __syncwarp();
        }
        kc = 0;
        ++tile;
      }
    }
  }
  // what is left of a tile that the next warps finish; a share inside one tile
  // has this slot alone
  if (kc != 0 && last > first) spill(mine + SLOT);
  __syncthreads();

  // tiles cut by a boundary between shares: summed by the warp in whose share they begin
  if (last > first) {
    const int end_tile = tile0 + last / m.nkc;  // the tile the share ends in
    const int begin_at = (end_tile - tile0) * m.nkc;
    if (last % m.nkc != 0 && begin_at >= first) {
      for (int e = lane; e < a.tokens * 16; e += 32) {
        const int tok = e >> 4, r = e & 15;
        const int off = (tok / PER) * 128 + (tok % PER) * (SPLIT ? 3 : 1) * 16 + r;
        float v = 0.0f;
        for (int w = warp; w < kWarpsQ4; ++w) {
          const int wf = static_cast<int>(static_cast<long long>(run) * w / kWarpsQ4);
          const int wl = static_cast<int>(static_cast<long long>(run) * (w + 1) / kWarpsQ4);
          if (wf >= begin_at + m.nkc) break;
          if (wl <= wf) continue;
          // its part of this tile: the last slot if the share ends inside the
          // tile, the first slot if it ends at or past the tile's end
          const float* col = slots + (w * 3 + (wl < begin_at + m.nkc ? 1 : 0)) * SLOT + off;
          v += SPLIT ? col[0] + (col[16] + col[32]) : col[0];
        }
        finish(end_tile, tok, r, v);
      }
    }
  }
}

// ================================================================= tiles ==
// More columns than q4_kernel takes: the same products, with x streamed.  A CTA
// is kq groups of warps that split the inputs among them; in a group each warp
// has two tiles (32 outputs) at a time, and a chunk of x (128 inputs of every
// column) is staged for the group by cp.async, three buffers deep, one named
// barrier per chunk.  A warp's weights come straight to registers, a chunk
// ahead.  Reading x again for every 32 * (8 / kq) outputs costs L2 as many bytes
// as the weights at 16 * (8 / kq) * 2 columns.  A set's sums are scaled when it
// ends, 64 inputs at most, so that the fragments of a set stay in registers.
constexpr int kTileX = kQ4Chunk * 2 + 64;  // bytes of a column's chunk: 64 mod 128
constexpr int kTileBufs = 3;
constexpr int kTileRun = 2;  // tiles per warp at a time

__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(take ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <bool BF16, bool SPLIT, int NT, int SETS, bool ZP>
__global__ void __launch_bounds__(kThreadsQ4, NT <= 2 ? 2 : 1) q4_tile_kernel(const Q4Kernel a) {
  constexpr int COLS = NT * 8, R = kTileRun;
  extern __shared__ __align__(16) unsigned char smem_q4[];
  const Q4Mat& m = a.m;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wm_n = kWarpsQ4 / a.kq, kq = warp / wm_n, wm = warp % wm_n;
  const int gthreads = wm_n * 32, gt = tid - kq * gthreads;
  unsigned char* xs = smem_q4 + kq * (kTileBufs * COLS * kTileX);
  float* red = reinterpret_cast<float*>(smem_q4 + a.kq * (kTileBufs * COLS * kTileX));

  const int tile0 = static_cast<int>(static_cast<long long>(m.ntile) * blockIdx.x / gridDim.x);
  const int tile1 = static_cast<int>(static_cast<long long>(m.ntile) * (blockIdx.x + 1) / gridDim.x);
  const int c0 = m.nkc * kq / a.kq, nc = m.nkc * (kq + 1) / a.kq - c0;
  const int passes = (tile1 - tile0 + wm_n * R - 1) / (wm_n * R);
  const int total = passes * nc;

  auto stage = [&](int it) {  // chunk it % nc of x
    if (it < total) {
      unsigned char* to = xs + (it % kTileBufs) * (COLS * kTileX);
      const int k0 = (c0 + it % nc) * kQ4Chunk;
      if (SPLIT) {
        const float* x = static_cast<const float*>(a.x);
        for (int e = gt; e < a.tokens * (kQ4Chunk / 2); e += gthreads) {
          const int tok = e / (kQ4Chunk / 2), k = 2 * (e % (kQ4Chunk / 2));
          uint32_t h = 0, mi = 0, lo = 0;
          if (k0 + k < m.ins) {
            uint16_t p0[3], p1[3];
            split3(x[tok * a.ldx + k0 + k], p0);
            split3(x[tok * a.ldx + k0 + k + 1], p1);
            h = p0[0] | static_cast<uint32_t>(p1[0]) << 16;
            mi = p0[1] | static_cast<uint32_t>(p1[1]) << 16;
            lo = p0[2] | static_cast<uint32_t>(p1[2]) << 16;
          }
          unsigned char* at = to + ((tok >> 1) * 8 + (tok & 1) * 3) * kTileX + 2 * k;
          *reinterpret_cast<uint32_t*>(at) = h;
          *reinterpret_cast<uint32_t*>(at + kTileX) = mi;
          *reinterpret_cast<uint32_t*>(at + 2 * kTileX) = lo;
        }
      } else {
        const uint16_t* x = static_cast<const uint16_t*>(a.x);
        for (int e = gt; e < a.tokens * 16; e += gthreads) {
          const int tok = e >> 4, k = k0 + 8 * (e & 15);
          const uint16_t* from = x + tok * a.ldx + k;
          unsigned char* at = to + tok * kTileX + 16 * (e & 15);
          if (a.wide) {
            cp_async16_or_zero(at, k < m.ins ? from : x, k < m.ins);
          } else {
            uint32_t w[4] = {0, 0, 0, 0};
            if (k < m.ins) {
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = from[2 * j] | static_cast<uint32_t>(from[2 * j + 1]) << 16;
            }
            *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
    cp_async_commit();
  };
  Q4Buf<SETS, ZP> buf[2][R];
  auto load = [&](int it, Q4Buf<SETS, ZP>(&b)[R]) {
    if (it >= total) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int tile = tile0 + (it / nc * wm_n + wm) * R + r;
      if (tile < tile1) b[r].load(m.tiles + (static_cast<long long>(tile) * m.nkc + c0 + it % nc) * m.chunk_bytes, lane);
    }
  };
  load(0, buf[0]);
  grid_wait();  // the weights are the handle's; x comes from the grid before
  stage(0);
  stage(1);

  // columns past the pass's last are not stored; they read the last column
  int xcol[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    xcol[n] = (SPLIT ? n * 8 + min(g, 5) : min(n * 8 + g, a.tokens - 1)) * kTileX + t * 16;

  float acc[R][NT][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;

  int chunk = 0, pass = 0;
  for (int it0 = 0; it0 < total; it0 += 2) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int it = it0 + d;
      if (it >= total) break;
      load(it + 1, buf[d ^ 1]);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      group_sync(1 + kq, gthreads);  // the chunk is there, and the one before it is done with
      stage(it + 2);
      const unsigned char* xc = xs + (it % kTileBufs) * (COLS * kTileX);
      const int first = tile0 + (pass * wm_n + wm) * R;
      if (first < tile1) {
        constexpr int PARTS = SETS < 2 ? 2 : SETS;  // scaled together: at most 64 inputs
        constexpr int BLK = 4 / PARTS;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          const int set = q * SETS / PARTS;
          uint32_t fa[R][2 * BLK][4];
          float2 sc[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const Q4Zero<BF16> z = buf[d][r].template zero<BF16>(set);
#pragma unroll
            for (int j = 0; j < 2 * BLK; ++j) unpack<BF16>(buf[d][r].word(q * 2 * BLK + j), z, fa[r][j]);
            sc[r] = buf[d][r].scale(set);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float part[R][4];
#pragma unroll
            for (int p = 0; p < BLK; ++p) {
              const uint4 f = *reinterpret_cast<const uint4*>(xc + xcol[n] + (q * BLK + p) * 64);
#pragma unroll
              for (int r = 0; r < R; ++r) {
                if (p == 0)
                  mma16816<BF16, true>(part[r], fa[r][0], f.x, f.y);
                else
                  mma16816<BF16, false>(part[r], fa[r][2 * p], f.x, f.y);
              }
#pragma unroll
              for (int r = 0; r < R; ++r) mma16816<BF16, false>(part[r], fa[r][2 * p + 1], f.z, f.w);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
              acc[r][n][0] = fmaf(sc[r].x, part[r][0], acc[r][n][0]);
              acc[r][n][1] = fmaf(sc[r].x, part[r][1], acc[r][n][1]);
              acc[r][n][2] = fmaf(sc[r].y, part[r][2], acc[r][n][2]);
              acc[r][n][3] = fmaf(sc[r].y, part[r][3], acc[r][n][3]);
            }
          }
        }
      }
      if (++chunk < nc) continue;
      // the pass ends: the groups' sums are added in their order
      if (a.kq > 1) {
        float* mine = red + ((kq - 1) * wm_n + wm) * (R * NT * 4 * 32) + lane;
        __syncthreads();
        if (kq > 0) {
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) mine[((r * NT + n) * 4 + i) * 32] = acc[r][n][i];
        }
        __syncthreads();
        if (kq == 0) {
          for (int o = 1; o < a.kq; ++o) {
            const float* from = red + ((o - 1) * wm_n + wm) * (R * NT * 4 * 32) + lane;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[r][n][i] += from[((r * NT + n) * 4 + i) * 32];
          }
        }
      }
      if (kq == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int o = (first + r) * kQ4Rows + g + 8 * h;
            const bool in = first + r < tile1 && o < m.outs;
            const float bias = in && m.bias ? m.bias[o] : 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float u = acc[r][n][2 * h], v = acc[r][n][2 * h + 1];
              if (SPLIT) {  // columns 0, 1, 2 and 3, 4, 5 are the parts of one token each
                const float u1 = __shfl_down_sync(0xffffffffu, u, 1), v1 = __shfl_down_sync(0xffffffffu, v, 1);
                const float sum = t == 0 ? u + (v + u1) : v + (u1 + v1);
                const int tok = 2 * n + t;
                if (in && t < 2 && tok < a.tokens) q4_store(a, tok, o, sum + bias);
              } else {
                const int tok = n * 8 + 2 * t;
                if (in && tok < a.tokens) q4_store(a, tok, o, u + bias);
                if (in && tok + 1 < a.tokens) q4_store(a, tok + 1, o, v + bias);
              }
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;
      chunk = 0;
      ++pass;
    }
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

cudaError_t launch_q4_kernel(void (*kernel)(Q4Kernel), const Q4Kernel& a, int grid, int smem, cudaStream_t s) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreadsQ4);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <bool BF16, bool SPLIT, int NT, int SETS, bool ZP>
cudaError_t run_rows(const Q4Kernel& a, cudaStream_t s) {
  const int smem = 3 * kWarpsQ4 * NT * 512 + a.cols * a.xstride;
  const int per_sm = NT <= 2 && smem <= 110 * 1024 ? 2 : 1;
  return launch_q4_kernel(q4_kernel<BF16, SPLIT, NT, SETS, ZP>, a, std::min(a.m.ntile, sm_count() * per_sm), smem, s);
}

// Groups of warps along the inputs: the fewest that give every SM a CTA.
template <bool BF16, bool SPLIT, int NT, int SETS, bool ZP>
cudaError_t run_tiles(Q4Kernel a, cudaStream_t s) {
  const int sms = sm_count();
  auto ctas = [&](int kq) { return (a.m.ntile + kTileRun * kWarpsQ4 / kq - 1) / (kTileRun * kWarpsQ4 / kq); };
  auto bytes = [&](int kq) {
    return kq * kTileBufs * NT * 8 * kTileX + (kq - 1) * (kWarpsQ4 / kq) * kTileRun * NT * 512;
  };
  a.kq = 1;
  while (a.kq < kWarpsQ4 && 2 * a.kq <= a.m.nkc && ctas(a.kq) < sms && bytes(2 * a.kq) <= 220 * 1024) a.kq *= 2;
  const int per_sm = NT <= 2 && bytes(a.kq) <= 110 * 1024 ? 2 : 1;
  return launch_q4_kernel(q4_tile_kernel<BF16, SPLIT, NT, SETS, ZP>, a, std::min(ctas(a.kq), sms * per_sm), bytes(a.kq),
                          s);
}

template <bool BF16, bool SPLIT, int NT, bool TILES>
cudaError_t pick_sets(const Q4Kernel& a, cudaStream_t s) {
  const int sets = kQ4Chunk / a.m.span;
  auto run = [&](auto n, auto zp) {
    if constexpr (TILES)
      return run_tiles<BF16, SPLIT, NT, decltype(n)::value, decltype(zp)::value>(a, s);
    else
      return run_rows<BF16, SPLIT, NT, decltype(n)::value, decltype(zp)::value>(a, s);
  };
  using std::integral_constant;
  auto zeros = [&](auto n) {
    return a.m.zeros ? run(n, integral_constant<bool, true>{}) : run(n, integral_constant<bool, false>{});
  };
  return sets == 4   ? zeros(integral_constant<int, 4>{})
         : sets == 2 ? zeros(integral_constant<int, 2>{})
                     : zeros(integral_constant<int, 1>{});
}

template <bool BF16, bool SPLIT>
cudaError_t pick_cols(const Q4Kernel& a, bool tiles, cudaStream_t s) {
  const int nt = (a.tokens + (SPLIT ? 1 : 7)) / (SPLIT ? 2 : 8);
  if (!tiles) {
    if (nt <= 1) return pick_sets<BF16, SPLIT, 1, false>(a, s);
    return pick_sets<BF16, SPLIT, 2, false>(a, s);
  }
  if (nt <= 1) return pick_sets<BF16, SPLIT, 1, true>(a, s);
  if (nt <= 2) return pick_sets<BF16, SPLIT, 2, true>(a, s);
  if (nt <= 4) return pick_sets<BF16, SPLIT, 4, true>(a, s);
  return pick_sets<BF16, SPLIT, 8, true>(a, s);
}

}  // namespace

void q4_layout(Q4Mat& m) {
  m.span = m.group % 128 == 0 ? 128 : m.group % 64 == 0 ? 64 : 32;
  m.nkc = (m.ins + kQ4Chunk - 1) / kQ4Chunk;
  m.ntile = (m.outs + kQ4Rows - 1) / kQ4Rows;
  const int sets = kQ4Chunk / m.span;
  m.chunk_bytes = 1024 + 32 * sets + (m.zeros ? 16 * sets : 0);
}

size_t q4_tiles_bytes(const Q4Mat& m) { return static_cast<size_t>(m.ntile) * m.nkc * m.chunk_bytes; }

cudaError_t launch_q4_pack(const Q4Mat& m, const unsigned char* q, const uint16_t* s, const unsigned char* zeros,
                           unsigned char* tiles, cudaStream_t st) {
  const long long nchunk = static_cast<long long>(m.ntile) * m.nkc;
  q4_pack_kernel<<<static_cast<unsigned>(std::min(nchunk, 148ll * 64)), 256, 0, st>>>(m, q, s, zeros, tiles);
  return cudaGetLastError();
}

// Up to 8 columns (fp32: 16, 4 rows) whose x fits into shared memory take
// q4_kernel; more, and the inputs that are too long for it, q4_tile_kernel in
// passes of 64 columns (fp32: 16 rows).
cudaError_t launch_q4(const Q4Mat& m, const Q4Args& q, int x_type, int y_type, cudaStream_t st) {
  const bool split = x_type == kOpsF32;
  const int per = split ? 2 : 8, parts = split ? 3 : 1;
  Q4Kernel a{};
  a.m = m;
  a.xstride = m.nkc * kQ4Chunk * 2 + 64;
  a.ldx = q.ldx;
  a.ldy = q.ldy;
  a.y_type = y_type;
  a.wide = reinterpret_cast<uintptr_t>(q.x) % 16 == 0 && q.ldx % 8 == 0;
  const int nt = (q.n + per - 1) / per;
  const bool tiles = nt > (split ? 2 : 1) || 3 * kWarpsQ4 * nt * 512 + q.n * parts * a.xstride > 110 * 1024;
  const int most = 8 * per;
  for (int i = 0; i < q.n; i += most) {
    a.tokens = std::min(most, q.n - i);
    a.cols = a.tokens * parts;
    a.x = static_cast<const char*>(q.x) + i * q.ldx * ops_type_size(x_type);
    a.y = static_cast<char*>(q.y) + i * q.ldy * ops_type_size(y_type);
    const cudaError_t e = split                  ? pick_cols<true, true>(a, tiles, st)
                          : x_type == kOpsBF16 ? pick_cols<true, false>(a, tiles, st)
                                                 : pick_cols<false, false>(a, tiles, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace vb
