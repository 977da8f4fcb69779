// Products with 4-bit weights (include/verbo_ops.h): y = x W^T + b with
// W[o][i] = s[o][g] (q[o][i] - z[o][g]) and the activations in their own type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

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

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two nibbles (the low four bits of each half) minus two zero points, exact:
// 0x6400 | q is the fp16 1024 + q, 0x4300 | q the bf16 128 + q, and zc holds
// 1024 + z or 128 + z.
template <bool BF16>
__device__ __forceinline__ uint32_t unpack2(uint32_t v, uint32_t zc) {
  uint32_t u = (v & 0x000f000fu) | (BF16 ? 0x43004300u : 0x64006400u);
  if (BF16) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&u), *reinterpret_cast<__nv_bfloat162*>(&zc));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&u), *reinterpret_cast<__half2*>(&zc));
  return *reinterpret_cast<const uint32_t*>(&d);
}
template <bool BF16>
__device__ __forceinline__ uint32_t zero_const(uint32_t z) {  // z in both halves, above the base
  return (BF16 ? 0x43004300u : 0x64006400u) | z | (z << 16);
}

// What one lane holds of a chunk.
template <int SETS, bool ZP>
struct Q4Buf {
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
};

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
        const float v = k < m.ins ? x[tok * a.ldx + k] : 0.0f;
        const float hi = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
        const bool fin = fabsf(v) < __uint_as_float(0x7f800000u);
        const float r = fin ? v - hi : 0.0f;
        const float mid = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
        const float lo = r - mid;
        // an infinity or NaN goes through the first part alone
        const uint32_t h = fin ? __float_as_uint(hi) : (v != v ? 0x7fc00000u : __float_as_uint(v));
        unsigned char* at = xs + static_cast<size_t>(3 * tok) * a.xstride + 2 * k;
        *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(h >> 16);
        *reinterpret_cast<uint16_t*>(at + a.xstride) = static_cast<uint16_t>(__float_as_uint(mid) >> 16);
        *reinterpret_cast<uint16_t*>(at + 2 * a.xstride) = static_cast<uint16_t>(__float_as_uint(lo) >> 16);
      }
  } else {
    const uint16_t* x = static_cast<const uint16_t*>(a.x);
    const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (a.ldx & 7) == 0;
    for (int tok = 0; tok < a.tokens; ++tok) {
      unsigned char* at = xs + static_cast<size_t>(tok) * a.xstride;
      const uint16_t* row = x + tok * a.ldx;
      for (int k = tid * 8; k < kp; k += kThreadsQ4 * 8) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < m.ins) {  // ins is a multiple of 32
          if (wide) {
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
      const uint32_t words[8] = {b.w0.x, b.w0.y, b.w0.z, b.w0.w, b.w1.x, b.w1.y, b.w1.z, b.w1.w};
      const int xoff = kc * (kQ4Chunk * 2);
#pragma unroll
      for (int set = 0; set < SETS; ++set) {
        constexpr int BLK = 4 / SETS;  // 32-blocks per set
        uint32_t zg, zh;
        if (ZP) {
          const uint32_t zz = b.z[set >> 1] >> (16 * (set & 1));
          zg = zero_const<BF16>(zz & 15u);
          zh = zero_const<BF16>((zz >> 8) & 15u);
        } else {
          zg = zh = zero_const<BF16>(8u);
        }
        float part[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) part[n][i] = 0.0f;
#pragma unroll
        for (int p = set * BLK; p < (set + 1) * BLK; ++p) {
          uint32_t fa[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t w = words[2 * p + j];
            fa[j][0] = unpack2<BF16>(w, zg);
            fa[j][1] = unpack2<BF16>(w >> 4, zh);
            fa[j][2] = unpack2<BF16>(w >> 8, zg);
            fa[j][3] = unpack2<BF16>(w >> 12, zh);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 f = *reinterpret_cast<const uint4*>(xcol[n] + xoff + p * 64);
            mma16816<BF16>(part[n], fa[0], f.x, f.y);
            mma16816<BF16>(part[n], fa[1], f.z, f.w);
          }
        }
        const __half2 sc = *reinterpret_cast<const __half2*>(&b.s[set]);
        const float sg = __low2float(sc), sh = __high2float(sc);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(sg, part[n][0], acc[n][0]);
          acc[n][1] = fmaf(sg, part[n][1], acc[n][1]);
          acc[n][2] = fmaf(sh, part[n][2], acc[n][2]);
          acc[n][3] = fmaf(sh, part[n][3], acc[n][3]);
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

template <bool BF16, bool SPLIT, int NT, int SETS, bool ZP>
cudaError_t run_q4(const Q4Kernel& a, cudaStream_t s) {
  auto kernel = q4_kernel<BF16, SPLIT, NT, SETS, ZP>;
  const int smem = 3 * kWarpsQ4 * NT * 512 + a.cols * a.xstride;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  if (smem > 48 * 1024) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  const int per_sm = NT <= 2 && smem <= 110 * 1024 ? 2 : 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(std::min(a.m.ntile, sms * per_sm));
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

template <bool BF16, bool SPLIT, int NT>
cudaError_t pick_sets(const Q4Kernel& a, cudaStream_t s) {
  const int sets = kQ4Chunk / a.m.span;
  if (a.m.zeros)
    return sets == 4   ? run_q4<BF16, SPLIT, NT, 4, true>(a, s)
           : sets == 2 ? run_q4<BF16, SPLIT, NT, 2, true>(a, s)
                       : run_q4<BF16, SPLIT, NT, 1, true>(a, s);
  return sets == 4   ? run_q4<BF16, SPLIT, NT, 4, false>(a, s)
         : sets == 2 ? run_q4<BF16, SPLIT, NT, 2, false>(a, s)
                     : run_q4<BF16, SPLIT, NT, 1, false>(a, s);
}

template <bool BF16, bool SPLIT>
cudaError_t pick_cols(const Q4Kernel& a, cudaStream_t s) {
  const int per = SPLIT ? 2 : 8;
  if (a.tokens <= per) return pick_sets<BF16, SPLIT, 1>(a, s);
  if (a.tokens <= 2 * per) return pick_sets<BF16, SPLIT, 2>(a, s);
  return pick_sets<BF16, SPLIT, 4>(a, s);
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

// Rows of x go through in passes of as many as shared memory and the widest
// kernel take.
cudaError_t launch_q4(const Q4Mat& m, const Q4Args& q, int x_type, int y_type, cudaStream_t st) {
  const bool split = x_type == kOpsF32;
  const int per = split ? 2 : 8, parts = split ? 3 : 1;
  Q4Kernel a{};
  a.m = m;
  a.xstride = m.nkc * kQ4Chunk * 2 + 64;
  int most = 4 * per;
  // narrower kernels need less for their slots: the widest that holds its columns
  while (most > 1) {
    const int nt = most <= per ? 1 : most <= 2 * per ? 2 : 4;
    if (3 * kWarpsQ4 * nt * 512 + most * parts * a.xstride <= 225 * 1024) break;
    --most;
  }
  for (int i = 0; i < q.n; i += most) {
    a.tokens = std::min(most, q.n - i);
    a.cols = a.tokens * parts;
    a.x = static_cast<const char*>(q.x) + i * q.ldx * ops_type_size(x_type);
    a.ldx = q.ldx;
    a.y = static_cast<char*>(q.y) + i * q.ldy * ops_type_size(y_type);
    a.ldy = q.ldy;
    a.y_type = y_type;
    const cudaError_t e = split                  ? pick_cols<true, true>(a, st)
                          : x_type == kOpsBF16 ? pick_cols<true, false>(a, st)
                                                 : pick_cols<false, false>(a, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace vb
