// Products with 4-bit weights (include/verbo_ops.h): y = x W^T + b with
// W[o][i] = s[o][g] (q[o][i] - z[o][g]) and the activations at their own
// precision.
//
// Both kernels feed mma.sync.m16n8k16 with fp16: A is a tile of 16 outputs with
// the weights unpacked to q - z, exact, and B holds x as columns.  The products
// are exact, a group's sum is fp32, and the group's scale multiplies that sum.
//   fp16 x   is a column as it is.
//   bf16 x   is a column times a power of two that takes the token's largest
//            value to [2^14, 2^15): exact for all within 2^-31 of that value (8
//            bits above 2^-24), and off by 2^-39 of it at most for the rest.
//   fp32 x   is two columns, hi = fp16(v) and lo = fp16((v - hi) 2^11) of the
//            same scaled v: v - hi is at most 2^12 of v's last places, of which lo
//            holds 11 bits, so v is met to within one of its last places (2^-23).
// The sums are taken back by the inverse power.  Infinities and NaNs go through
// hi as they are and do not count for the largest value.
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
constexpr int kAhead = 2;  // chunks whose loads a warp of q4_kernel keeps in flight

__device__ unsigned g_ops_status;

// ================================================================== pack ==
// One thread per 32-bit word of the chunks' nibbles.  Word j of lane (g, t) =
// (lane / 4, lane % 4) holds the lane's A fragment of k-step j: rows g and
// g + 8, and of the chunk's block p = j / 2 the four weights k, k + 1, k + 2,
// k + 3 from k = 32 p + 8 t + 4 (j % 2).  (The sum over k has no order, so the
// lane's share of a block is taken as 8 neighbouring weights, which lets x be
// read as it lies.)  Nibbles, low to high: (g, k), (g+8, k), (g, k+2),
// (g+8, k+2), (g, k+1), (g+8, k+1), (g, k+3), (g+8, k+3): masks with 0x000f000f
// and 0x00f000f0 at shifts 0 and 8 give the pairs of a0, a1, a2, a3.
// Four neighbouring weights of output o from input i on (a multiple of 4) as the
// low halves of four bytes.
__device__ __forceinline__ uint32_t q4_four(const Q4Mat& m, const unsigned char* q, int o, int i) {
  if (o >= m.outs || i >= m.ins) return 0;
  const int e = i & 31;
  const unsigned char* p = q + static_cast<size_t>(o) * (m.ins / 2) + (i >> 5) * 16 + (e & 15);
  uint32_t v;
  if ((reinterpret_cast<uintptr_t>(q) & 3) == 0)
    v = *reinterpret_cast<const uint32_t*>(p);
  else
    v = p[0] | p[1] << 8 | p[2] << 16 | static_cast<uint32_t>(p[3]) << 24;
  return (e < 16 ? v : v >> 4) & 0x0f0f0f0fu;
}

__global__ void q4_pack_kernel(Q4Mat m, const unsigned char* __restrict__ q, const uint16_t* __restrict__ s,
                               const unsigned char* __restrict__ z, unsigned char* __restrict__ tiles) {
  const long long nchunk = static_cast<long long>(m.ntile) * m.nkc;
  const int sets = kQ4Chunk / m.span;
  const int groups = q4_groups(m);
  for (long long c = blockIdx.x; c < nchunk; c += gridDim.x) {
    const int tile = static_cast<int>(c / m.nkc), kc = static_cast<int>(c % m.nkc);
    unsigned char* dst = tiles + c * m.chunk_bytes;
    const int w = threadIdx.x;  // 256 words of nibbles
    {
      const int half = w >> 7, lane = (w >> 2) & 31, j = half * 4 + (w & 3);
      const int g = lane >> 2, t = lane & 3;
      const int k = kc * kQ4Chunk + 32 * (j >> 1) + 8 * t + 4 * (j & 1);
      const int r = tile * kQ4Rows + g;
      // k, k + 1, k + 2, k + 3 of row g to nibbles 0, 4, 2, 6, of row g + 8 to 1, 5, 3, 7
      const uint32_t lo = q4_four(m, q, r, k), up = q4_four(m, q, r + 8, k);
      const uint32_t both = lo | up << 4;
      const uint32_t v = __byte_perm(both, 0, 0x3120);
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

// ================================================================ pieces ==
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// d = a b + d, or a b with START.
template <bool START>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (START)
    asm("{\n .reg .f32 z;\n mov.f32 z, 0f00000000;\n"
        " mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {z,z,z,z};\n}"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (x, y) += s (px, py): the packed form of two fmas.
__device__ __forceinline__ void fma2(float& x, float& y, uint64_t s, float px, float py) {
  uint64_t a, p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(x), "f"(y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(px), "f"(py));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(s), "l"(p));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a));
}
__device__ __forceinline__ uint64_t twice(float s) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %1};" : "=l"(d) : "f"(s));
  return d;
}

// The zero points of rows g and g + 8 as unpack() wants them.
struct Q4Zero {
  uint32_t g, h;
  __device__ __forceinline__ Q4Zero(uint32_t zg, uint32_t zh) {
    g = 0x64006400u | zg | zg << 16;           // 1024 + z
    h = 0xd400d400u | zh << 4 | zh << 20;      // -(64 + z)
  }
};

// A word's eight weights minus their zero points: the A fragment of one k-step,
// exact.  0x6400 | q is the fp16 1024 + q, and with q four bits higher
// 1024 + 16 q, of which a sixteenth minus (64 + z) is q - z.
__device__ __forceinline__ void unpack(uint32_t w, const Q4Zero& z, uint32_t (&a)[4]) {
  const uint32_t v = w >> 8, sixteenth = 0x2c002c00u;
  auto h2 = [](const uint32_t& u) -> const __half2& { return *reinterpret_cast<const __half2*>(&u); };
  auto lower = [&](uint32_t u) {
    u = (u & 0x000f000fu) | 0x64006400u;
    const __half2 d = __hsub2(h2(u), h2(z.g));
    return *reinterpret_cast<const uint32_t*>(&d);
  };
  auto upper = [&](uint32_t u) {
    u = (u & 0x00f000f0u) | 0x64006400u;
    const __half2 d = __hfma2(h2(u), h2(sixteenth), h2(z.h));
    return *reinterpret_cast<const uint32_t*>(&d);
  };
  a[0] = lower(w);
  a[1] = upper(w);
  a[2] = lower(v);
  a[3] = upper(v);
}

// A chunk's scales and zero points for rows g and g + 8.
template <int SETS, bool ZP>
struct Q4Tail {
  uint32_t s[SETS];                     // two fp16 per set
  uint32_t z[ZP ? (SETS + 1) / 2 : 1];  // two bytes per set
  __device__ __forceinline__ void load(const unsigned char* p, int g) {
    const unsigned char* sp = p + g * (4 * SETS);
    if constexpr (SETS == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(sp);
      s[0] = v.x, s[1] = v.y, s[2] = v.z, s[3] = v.w;
    } else if constexpr (SETS == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(sp);
      s[0] = v.x, s[1] = v.y;
    } else {
      s[0] = *reinterpret_cast<const uint32_t*>(sp);
    }
    if constexpr (ZP) {
      const unsigned char* zp = p + 32 * SETS + g * (2 * SETS);
      if constexpr (SETS == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(zp);
        z[0] = v.x, z[1] = v.y;
      } else if constexpr (SETS == 2) {
        z[0] = *reinterpret_cast<const uint32_t*>(zp);
      } else {
        z[0] = *reinterpret_cast<const uint16_t*>(zp);
      }
    }
  }
  __device__ __forceinline__ Q4Zero zero(int set) const {
    if (!ZP) return Q4Zero(8u, 8u);
    const uint32_t v = z[set >> 1] >> (16 * (set & 1));
    return Q4Zero(v & 15u, (v >> 8) & 15u);
  }
  __device__ __forceinline__ float2 scale(int set) const {
    return __half22float2(*reinterpret_cast<const __half2*>(&s[set]));
  }
};

// What one lane holds of a chunk.
template <int SETS, bool ZP>
struct Q4Buf : Q4Tail<SETS, ZP> {
  uint4 w0, w1;
  __device__ __forceinline__ uint32_t word(int j) const {
    const uint4& w = j < 4 ? w0 : w1;
    return (j & 3) == 0 ? w.x : (j & 3) == 1 ? w.y : (j & 3) == 2 ? w.z : w.w;
  }
  __device__ __forceinline__ void load(const unsigned char* p, int lane) {
    w0 = ld_stream16(p + lane * 16);
    w1 = ld_stream16(p + 512 + lane * 16);
    Q4Tail<SETS, ZP>::load(p + 1024, lane >> 2);
  }
};

struct Q4Kernel {
  Q4Mat m;
  const void* x;
  long long ldx;
  int tokens;  // rows of x
  void* y;
  long long ldy;
  int y_type;
  bool wide;       // rows of x start on 16 bytes
  int xstride;     // q4_kernel: bytes from one column to the next in shared memory
  // q4_tile_kernel: x as q4_image_kernel lays it out, the factors that take its
  // sums back (per token), and the groups of warps along the inputs
  unsigned char* image;
  float2* back;
  int kq;
  int per_pass;  // tokens of a pass; blockIdx.y is the pass
};

template <int XT>
constexpr int kPartsOf = XT == kOpsF32 ? 2 : 1;  // columns per token

// Eight neighbouring values of a row (past `ins`: zeros).
template <int XT>
struct X8 {
  using E = std::conditional_t<XT == kOpsF32, uint32_t, uint16_t>;
  uint32_t v[XT == kOpsF32 ? 8 : 4];
  __device__ __forceinline__ void load(const void* row, int k, int ins, bool wide) {
    if (k >= ins) {  // ins is a multiple of 32
#pragma unroll
      for (uint32_t& w : v) w = 0;
      return;
    }
    const E* p = static_cast<const E*>(row) + k;
    if (wide) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(v) / 16); ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i];
        v[4 * i] = u.x, v[4 * i + 1] = u.y, v[4 * i + 2] = u.z, v[4 * i + 3] = u.w;
      }
    } else if constexpr (XT == kOpsF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = p[2 * i] | static_cast<uint32_t>(p[2 * i + 1]) << 16;
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (XT == kOpsF32)
      return __uint_as_float(v[i]);
    else if constexpr (XT == kOpsBF16)
      return __uint_as_float((i & 1) ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
    else
      return __half2float(__ushort_as_half(static_cast<unsigned short>(v[i >> 1] >> (16 * (i & 1)))));
  }
  // the largest magnitude among the finite values, as bits of a float
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
    if constexpr (XT == kOpsF32) {
#pragma unroll
      for (uint32_t u : v) m = max(m, u & 0x7fffffffu);
    } else {
#pragma unroll
      for (uint32_t u : v) m = __vmaxu2(m, u & 0x7fff7fffu);
      m = XT == kOpsBF16 ? max(m << 16, m & 0xffff0000u) : 0;
    }
    if (m < 0x7f800000u) return m;
    m = 0;  // an infinity or a NaN is among them
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(get(i)) & 0x7fffffffu;
      if (u < 0x7f800000u) m = max(m, u);
    }
    return m;
  }
  // the columns' 16 bytes
  __device__ __forceinline__ void columns(float up, float up2, uint4& hi, uint4& lo) const {
    if constexpr (XT == kOpsF16) {
      hi = make_uint4(v[0], v[1], v[2], v[3]);
    } else {
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = get(2 * i) * up, b = get(2 * i + 1) * up;
        if (up2 != 1.0f) {
          a *= up2;
          b *= up2;
        }
        const __half2 p = __floats2half2_rn(a, b);
        h[i] = *reinterpret_cast<const uint32_t*>(&p);
        const float2 q = __half22float2(p);
        // of an infinity or a NaN nothing is left over
        const __half2 r = __floats2half2_rn(fabsf(a) < __uint_as_float(0x7f800000u) ? (a - q.x) * 2048.0f : 0.0f,
                                            fabsf(b) < __uint_as_float(0x7f800000u) ? (b - q.y) * 2048.0f : 0.0f);
        l[i] = *reinterpret_cast<const uint32_t*>(&r);
      }
      hi = make_uint4(h[0], h[1], h[2], h[3]);
      if (XT == kOpsF32) lo = make_uint4(l[0], l[1], l[2], l[3]);
    }
  }
};

// The power of two that takes a largest magnitude (as bits) to [2^14, 2^15), and
// its inverse, each in two factors that fp32 holds, the second mostly 1.
struct Power {
  float up, up2, down, down2;
  __device__ __forceinline__ explicit Power(uint32_t largest) {
    int e = 0;
    if (largest) {
      int x;
      frexpf(__uint_as_float(largest), &x);  // value in [2^(x-1), 2^x)
      e = 15 - x;
    }
    const int h = e > 120 || e < -120 ? e / 2 : e;
    up = two(h), up2 = two(e - h), down = two(-h), down2 = two(h - e);
  }
  static __device__ __forceinline__ float two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
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

// ================================================================ matvec ==
// Up to 8 columns.  The bound is reading the matrix once.  A tile is 16 outputs
// times all inputs; a CTA takes a run of tiles and its warps equal shares of the
// run's chunks, so each warp streams one contiguous piece of memory, kAhead
// chunks ahead, in registers.  x lies in shared memory, one column after the
// other as in memory; a lane's B fragment of two k-steps is 16 neighbouring
// bytes of a column (columns 64 mod 128 bytes apart: the 8 lanes of a quarter
// warp hit 32 banks).  A tile whose chunks fall to several warps is summed over
// the warps' partial sums in shared memory, in the order of the warps.
//
// Measured on B200: a 151936 x 896 matrix in groups of 32 times one fp32 row 20.5
// us, 3.8 TB/s (57% of the card's copy rate): reading alone would take 11.8.  A
// chunk costs a warp about 190 instructions, 72 of them the unpacking, and its
// eight mma with their scaling 100 cycles of a quarter SM, against 198 in which memory
// delivers it.  About 4 us are start and end: 4096 x 4096 takes 6.4 us, 896 x 896
// 4.  Sixteen warps for small matrices, three CTAs per SM or more chunks ahead
// changed nothing or lost.  8 bf16 rows of 14336 x 4096 take 16.5 us, most of the
// difference to one row in laying x out in every CTA.
template <int XT, int SETS, bool ZP>
__global__ void __launch_bounds__(kThreadsQ4, 2) q4_kernel(const Q4Kernel a) {
  constexpr int PARTS = kPartsOf<XT>;
  extern __shared__ __align__(128) unsigned char smem_q4[];
  __shared__ uint32_t largest[8];
  __shared__ float2 back[8];
  // slots: per warp the partial sums of its first tile, of its last, and one for
  // the tile at hand; [8 columns][16 rows] each
  constexpr int SLOT = 128;
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

  grid_release();  // the next grid may start on its weights as SMs come free; it waits for this one's end as well
  if (XT != kOpsF16 && tid < 8) largest[tid] = 0;
  if (XT != kOpsF16) __syncthreads();
  grid_wait();  // the weights are the handle's; x comes from the grid before
  // x: eight inputs per thread at a time, a few loads in flight; the warps are dealt
  // to the tokens in equal numbers (of 3, 5, 6 and 7 tokens some warps have none)
  constexpr int ES = XT == kOpsF32 ? 4 : 2, FLY = 4;
  const int kp = m.nkc * kQ4Chunk;
  const int deal = a.tokens <= 1 ? 8 : a.tokens <= 2 ? 4 : a.tokens <= 4 ? 2 : 1;  // warps per token
  const int tok = warp / deal, k0 = ((warp % deal) * 32 + lane) * 8, dk = deal * 256;
  const char* row = static_cast<const char*>(a.x) + tok * a.ldx * ES;
  auto each_unit = [&](auto&& f) {
    for (int k = k0; k < kp; k += FLY * dk) {
      X8<XT> v[FLY];
#pragma unroll
      for (int i = 0; i < FLY; ++i) v[i].load(row, k + i * dk, m.ins, a.wide);
#pragma unroll
      for (int i = 0; i < FLY; ++i)
        if (k + i * dk < kp) f(v[i], k + i * dk);
    }
  };
  if (XT != kOpsF16) {
    if (tok < a.tokens) {
      uint32_t big = 0;
      each_unit([&](const X8<XT>& v, int) { big = max(big, v.largest()); });
      big = __reduce_max_sync(0xffffffffu, big);
      if (lane == 0) atomicMax(&largest[tok], big);
    }
    __syncthreads();
  }
  if (tok < a.tokens) {
    Power p(0);
    if (XT != kOpsF16) {
      p = Power(largest[tok]);
      if (k0 == 0) back[tok] = make_float2(p.down, p.down2);
    }
    unsigned char* at = xs + static_cast<size_t>(PARTS * tok) * a.xstride;
    each_unit([&](const X8<XT>& v, int k) {
      uint4 hi, lo;
      v.columns(p.up, p.up2, hi, lo);
      *reinterpret_cast<uint4*>(at + 2 * k) = hi;
      if (PARTS == 2) *reinterpret_cast<uint4*>(at + a.xstride + 2 * k) = lo;
    });
  }
  __syncthreads();

  // the column of B that this lane reads (past the last one: the last, whose sums
  // are then not stored)
  const unsigned char* xcol = xs + static_cast<size_t>(min(g, a.tokens * PARTS - 1)) * a.xstride + t * 16;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};

  float* mine = slots + warp * 3 * SLOT;
  auto spill = [&](float* slot) {  // acc -> [column][row]
    slot[(2 * t) * 16 + g] = acc[0];
    slot[(2 * t + 1) * 16 + g] = acc[1];
    slot[(2 * t) * 16 + g + 8] = acc[2];
    slot[(2 * t + 1) * 16 + g + 8] = acc[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.0f;
  };
  // a token's sum in a slot
  auto token_sum = [&](const float* slot, int tok, int r) {
    const float* col = slot + tok * (PARTS * 16) + r;
    return PARTS == 2 ? fmaf(col[16], 1.0f / 2048.0f, col[0]) : col[0];
  };
  auto finish = [&](int tile, int tok, int r, float v) {
    const int o = tile * kQ4Rows + r;
    if (XT != kOpsF16) v = v * back[tok].x * back[tok].y;
    if (o < m.outs) q4_store(a, tok, o, m.bias ? v + m.bias[o] : v);
  };

  int kc = first % m.nkc, tile = tile0 + first / m.nkc;
  bool first_part = kc != 0;  // the tile at hand began in an earlier warp's share
  const unsigned char* xk = xcol + kc * (kQ4Chunk * 2);
  for (int i0 = first; i0 < last; i0 += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      if (i0 + d >= last) break;
      Q4Buf<SETS, ZP>& b = buf[d];
#pragma unroll
      for (int set = 0; set < SETS; ++set) {
        constexpr int BLK = 4 / SETS;  // 32-blocks per set
        const Q4Zero z = b.zero(set);
        float part[4];
#pragma unroll
        for (int p = set * BLK; p < (set + 1) * BLK; ++p) {
          uint32_t fa[2][4];
          unpack(b.word(2 * p), z, fa[0]);
          unpack(b.word(2 * p + 1), z, fa[1]);
          const uint4 f = *reinterpret_cast<const uint4*>(xk + p * 64);
          if (p == set * BLK) {
            mma16816<true>(part, fa[0], f.x, f.y);
          } else {
            mma16816<false>(part, fa[0], f.x, f.y);
          }
          mma16816<false>(part, fa[1], f.z, f.w);
        }
        const float2 sc = b.scale(set);
        acc[0] = fmaf(sc.x, part[0], acc[0]);
        acc[1] = fmaf(sc.x, part[1], acc[1]);
        acc[2] = fmaf(sc.y, part[2], acc[2]);
        acc[3] = fmaf(sc.y, part[3], acc[3]);
      }
      if (i0 + d + kAhead < last) b.load(src, lane);
      src += m.chunk_bytes;
      xk += kQ4Chunk * 2;
      if (++kc == m.nkc) {
        if (first_part) {
          spill(mine);
          first_part = false;
        } else {  // the whole tile is this warp's
          spill(mine + 2 * SLOT);
          __syncwarp();
          for (int e = lane; e < a.tokens * 16; e += 32)
            finish(tile, e >> 4, e & 15, token_sum(mine + 2 * SLOT, e >> 4, e & 15));
          __syncwarp();
        }
        kc = 0;
        xk = xcol;
        ++tile;
      }
    }
  }
  // what is left of a tile that the next warps finish; a share inside one tile
  // has this slot alone
  if (kc != 0 && last > first) spill(mine + SLOT);
  __syncthreads();

  // tiles cut by a boundary between shares: summed by the warp in whose share they begin
  const int end_tile = last / m.nkc, begin_at = end_tile * m.nkc;  // the tile the share ends in
  if (last > first && last % m.nkc != 0 && begin_at >= first) {
    for (int e = lane; e < a.tokens * 16; e += 32) {
      float v = 0.0f;
      for (int w = warp; w < kWarpsQ4; ++w) {
        const int wf = static_cast<int>(static_cast<long long>(run) * w / kWarpsQ4);
        const int wl = static_cast<int>(static_cast<long long>(run) * (w + 1) / kWarpsQ4);
        if (wf >= begin_at + m.nkc) break;
        if (wl <= wf) continue;
        // its part of this tile: the last slot if the share ends inside the tile,
        // the first slot if it ends at or past the tile's end
        v += token_sum(slots + (w * 3 + (wl < begin_at + m.nkc ? 1 : 0)) * SLOT, e >> 4, e & 15);
      }
      finish(tile0 + end_tile, e >> 4, e & 15, v);
    }
  }
}

// ================================================================= image ==
// x for q4_tile_kernel, in passes of COLS columns: per chunk of 128 inputs, per
// tile of 8 columns and per 32-block the 16 bytes that each lane's B fragments of
// two k-steps are, so that a chunk is one contiguous copy and a fragment one
// 16-byte load.  One CTA per token; also its factors back.
template <int XT>
__global__ void __launch_bounds__(256) q4_image_kernel(const Q4Kernel a, int cols) {
  constexpr int PARTS = kPartsOf<XT>, ES = XT == kOpsF32 ? 4 : 2;
  __shared__ uint32_t largest[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_release();
  grid_wait();
  const int tok = blockIdx.x, per_pass = cols / PARTS;
  const int pass = tok / per_pass, col = (tok - pass * per_pass) * PARTS;
  const Q4Mat& m = a.m;
  const char* row = static_cast<const char*>(a.x) + tok * a.ldx * ES;
  float up = 1.0f, up2 = 1.0f;
  if (XT != kOpsF16) {
    uint32_t big = 0;
    for (int k = tid * 8; k < m.ins; k += 256 * 8) {
      X8<XT> v;
      v.load(row, k, m.ins, a.wide);
      big = max(big, v.largest());
    }
    big = __reduce_max_sync(0xffffffffu, big);
    if (lane == 0) largest[warp] = big;
    __syncthreads();
    big = largest[lane & 7];
    const Power p(__reduce_max_sync(0xffffffffu, big));
    up = p.up, up2 = p.up2;
    if (tid == 0) a.back[tok] = make_float2(p.down, p.down2);
  } else if (tid == 0) {
    a.back[tok] = make_float2(1.0f, 1.0f);
  }
  unsigned char* to = a.image + static_cast<size_t>(pass) * m.nkc * (cols * (kQ4Chunk * 2));
  for (int u = tid; u < m.nkc * 16; u += 256) {  // 8 inputs each: chunk, block p, t
    X8<XT> v;
    v.load(row, u * 8, m.ins, a.wide);
    uint4 hi, lo;
    v.columns(up, up2, hi, lo);
    unsigned char* at = to + static_cast<size_t>(u >> 4) * (cols * (kQ4Chunk * 2)) + (col >> 3) * 2048 +
                        ((u >> 2) & 3) * 512 + (col & 7) * 64 + (u & 3) * 16;
    *reinterpret_cast<uint4*>(at) = hi;
    if (PARTS == 2) *reinterpret_cast<uint4*>(at + 64) = lo;  // the next column, of the same eight
  }
}

// ================================================================= tiles ==
// More than 8 columns, or inputs too long for q4_kernel.  A CTA is kq groups of
// warps that split the inputs among them; in a group each warp has a tile (16
// outputs) times all columns at a time, its weights coming straight to registers,
// half a chunk at a time.  One thread of the group streams chunks of x (its image, one
// bulk copy each) through a ring of stages (full / empty barriers).  A set's sums
// are scaled when it ends, 64 inputs at most, so that its fragments stay in
// registers; up to four column tiles go through the tensor pipe side by side.
//
// What bounds it is not memory but the pipes behind mma.sync: measured on B200, an
// m16n8k16 takes 8.6 cycles of a quarter SM, and two of them (a group of 32) with
// their load and the fmas of their scale 19.6: 37 us of the 81 that 64 rows of a
// 151936 x 896 head take; unpacking and waiting make the rest.  tcgen05.mma does
// not help here: a group's sums have to leave tensor memory before the next scale,
// 2 values per weight at 64 columns and groups of 32, and weights that are unpacked
// into tensor memory went there at about 25 bytes per cycle and SM: a kernel built
// that way, five warps to 128 outputs, took 92 us for 64 rows of a 151936 x 896 head
// in groups of 32 (this one 81) and 43 us for 16 (this one 36).
constexpr int kTileStages = 3;
constexpr int kTileAhead = 2;  // half chunks of weights in flight per warp (four: 0 to 2 us slower)
// CTAs per SM.  More of them hide more, at fewer registers: 16 rows of a 151936 x
// 896 head in groups of 32 took 35.5 us with three and 39 with two, of a 14336 x
// 4096 matrix in groups of 64 (longer chains of fragments) 25.1 and 22.5.
// The widest forms (NT 8; NT 4 and 2 with four sets) spill 4 to 44 bytes of registers a
// thread.  How much goes by little: one more int in Q4Kernel made it 64 bytes in the
// loop of 64 rows of that head, which then took 140 us in place of 81.
template <int NT, int SETS>
constexpr int kTileCtas = NT <= 4 && SETS == 4 ? 3 : 2;

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mbar_arrive1(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// What one lane holds of half a chunk: 64 inputs, one set or two.
template <int SETS, bool ZP>
struct Q4Half {
  static constexpr int ND = SETS == 4 ? 2 : 1;
  uint4 w;
  uint32_t s[ND], z;
  __device__ __forceinline__ uint32_t word(int j) const { return j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w; }
  // half h of the chunk at p
  __device__ __forceinline__ void load(const unsigned char* p, int h, int lane) {
    w = ld_stream16(p + h * 512 + lane * 16);
    const unsigned char* tail = p + 1024;
    const int set = (lane >> 2) * SETS + (SETS == 1 ? 0 : h * ND);
    if constexpr (ND == 2) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(tail + set * 4));
      s[0] = v.x, s[1] = v.y;
      if constexpr (ZP) z = __ldg(reinterpret_cast<const unsigned*>(tail + 32 * SETS + set * 2));
    } else {
      s[0] = __ldg(reinterpret_cast<const unsigned*>(tail + set * 4));
      if constexpr (ZP) z = __ldg(reinterpret_cast<const unsigned short*>(tail + 32 * SETS + set * 2));
    }
  }
  __device__ __forceinline__ Q4Zero zero(int d) const {
    if (!ZP) return Q4Zero(8u, 8u);
    const uint32_t v = z >> (16 * d);
    return Q4Zero(v & 15u, (v >> 8) & 15u);
  }
  __device__ __forceinline__ float2 scale(int d) const {
    return __half22float2(*reinterpret_cast<const __half2*>(&s[d]));
  }
};

template <int XT, int NT, int SETS, bool ZP>
__global__ void __launch_bounds__(kThreadsQ4, kTileCtas<NT, SETS>) q4_tile_kernel(const Q4Kernel a) {
  constexpr int PARTS = kPartsOf<XT>;
  constexpr int XB = NT * 2048;  // a chunk of x
  extern __shared__ __align__(128) unsigned char smem_q4[];
  __shared__ uint64_t bars[kWarpsQ4][2 * kTileStages];  // per group: full, empty
  __shared__ float2 back[NT * 8 / PARTS];
  __shared__ int stop;
  const Q4Mat& m = a.m;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int group = kWarpsQ4 / a.kq, kq = warp / group, wm = warp % group;
  unsigned char* ring = smem_q4 + kq * (kTileStages * XB);
  float* red = reinterpret_cast<float*>(smem_q4 + a.kq * (kTileStages * XB));
  uint64_t* full = bars[kq];
  uint64_t* empty = bars[kq] + kTileStages;
  if (tid < a.kq * 2 * kTileStages)
    mbar_init(&bars[tid / (2 * kTileStages)][tid % (2 * kTileStages)], tid % (2 * kTileStages) < kTileStages ? 1 : group);
  if (tid == 0) stop = 0;

  const int tile0 = static_cast<int>(static_cast<long long>(m.ntile) * blockIdx.x / gridDim.x);
  const int tile1 = static_cast<int>(static_cast<long long>(m.ntile) * (blockIdx.x + 1) / gridDim.x);
  const int c0 = m.nkc * kq / a.kq, nc = m.nkc * (kq + 1) / a.kq - c0;
  const int passes = (tile1 - tile0 + group - 1) / group;
  const int total = passes * nc;
  const bool producer = wm == 0 && lane == 0;
  const int tok0 = blockIdx.y * a.per_pass, tokens = min(a.per_pass, a.tokens - tok0);
  const unsigned char* image = a.image + static_cast<size_t>(blockIdx.y) * m.nkc * XB;
  __syncthreads();

  // the weights are the handle's; x comes from the grid before
  constexpr int AHEAD = kTileAhead;
  Q4Half<SETS, ZP> buf[AHEAD];
  int load_tile = tile0 + wm, load_half = 0;
  const unsigned char* load_at = m.tiles + (static_cast<long long>(load_tile) * m.nkc + c0) * m.chunk_bytes;
  auto load = [&](Q4Half<SETS, ZP>& b, int h) {  // h: load_half & 1
    if (load_tile < tile1) b.load(load_at, h, lane);
    if (h == 1) load_at += m.chunk_bytes;
    if (++load_half == 2 * nc) {
      load_half = 0;
      load_tile += group;
      load_at += (static_cast<long long>(group) * m.nkc - nc) * m.chunk_bytes;
    }
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(buf[i], i & 1);
  int put = 0, put_chunk = 0;  // the next chunk of x
  auto inputs = [&]() {
    const int s = put % kTileStages;
    mbar_expect_tx(&full[s], XB);
    bulk_copy(ring + s * XB, image + static_cast<size_t>(c0 + put_chunk) * XB, XB, &full[s]);
    ++put;
    if (++put_chunk == nc) put_chunk = 0;
  };
  grid_release();
  grid_wait();
  if (producer)
    while (put < min(kTileStages, total)) inputs();
  if (tid < tokens) back[tid] = a.back[tok0 + tid];
  __syncthreads();

  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

  bool ok = true;
  int chunk = 0, tile = tile0 + wm, limit = total;  // limit: the chunks of x to copy
  // The tiles are through: the groups' sums are added in their order.
  auto finish = [&]() {
    if (a.kq > 1) {
      float* mine = red + ((kq - 1) * group + wm) * (NT * 4 * 32) + lane;
      __syncthreads();
      if (kq > 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) mine[(n * 4 + i) * 32] = acc[n][i];
      }
      __syncthreads();
      if (kq == 0) {
        for (int o = 1; o < a.kq; ++o) {
          const float* from = red + ((o - 1) * group + wm) * (NT * 4 * 32) + lane;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] += from[(n * 4 + i) * 32];
        }
      }
    }
    if (kq == 0 && ok && !*const_cast<volatile int*>(&stop) && tile < tile1) {
      const int o = tile * kQ4Rows + g;
      float bias[2] = {0.0f, 0.0f};
      if (m.bias) {
        if (o < m.outs) bias[0] = m.bias[o];
        if (o + 8 < m.outs) bias[1] = m.bias[o + 8];
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int u = 0; u < 2 / PARTS; ++u) {
          const int tok = PARTS == 2 ? n * 4 + t : n * 8 + 2 * t + u;
          if (tok >= tokens) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (o + 8 * h >= m.outs) continue;
            float v = PARTS == 2 ? fmaf(acc[n][2 * h + 1], 1.0f / 2048.0f, acc[n][2 * h]) : acc[n][2 * h + u];
            if (XT != kOpsF16) v = v * back[tok].x * back[tok].y;
            q4_store(a, tok0 + tok, o + 8 * h, m.bias ? v + bias[h] : v);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
  };
  for (int it0 = 0; it0 < total; it0 += AHEAD / 2) {
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
      const int it = it0 + d / 2, half = d & 1;
      if (it >= total) break;
      const int s = it % kTileStages;
      // After a wait that ran out the warp goes on without waiting (its lanes stay
      // together, and the barriers are met), but stores no tile any more, nor do
      // warps that see `stop`.  Tiles that were through before are in y: the call's
      // y is partly written then, and the status says so.
      if (half == 0 && ok && !mbar_wait_limited(&full[s], (it / kTileStages) & 1)) {
        ok = false;
        stop = 1;
      }
      if (tile < tile1) {
        const unsigned char* xc = ring + s * XB + half * 1024 + lane * 16;
        constexpr int ND = Q4Half<SETS, ZP>::ND, BLK = 2 / ND;  // sets, 32-blocks of each
        constexpr int NP = NT < 4 ? NT : 4;                      // column tiles side by side
#pragma unroll
        for (int q = 0; q < ND; ++q) {
          const Q4Zero z = buf[d].zero(q);
          uint32_t fa[2 * BLK][4];
#pragma unroll
          for (int j = 0; j < 2 * BLK; ++j) unpack(buf[d].word(2 * BLK * q + j), z, fa[j]);
          const float2 sc = buf[d].scale(q);
          const uint64_t sg = twice(sc.x), sh = twice(sc.y);
#pragma unroll
          for (int n = 0; n < NT; n += NP) {
            float part[NP][4];
#pragma unroll
            for (int p = 0; p < BLK; ++p) {
              uint4 f[NP];
#pragma unroll
              for (int u = 0; u < NP; ++u)
                f[u] = *reinterpret_cast<const uint4*>(xc + (n + u) * 2048 + (q * BLK + p) * 512);
#pragma unroll
              for (int u = 0; u < NP; ++u) {
                if (p == 0)
                  mma16816<true>(part[u], fa[0], f[u].x, f[u].y);
                else
                  mma16816<false>(part[u], fa[2 * p], f[u].x, f[u].y);
              }
#pragma unroll
              for (int u = 0; u < NP; ++u) mma16816<false>(part[u], fa[2 * p + 1], f[u].z, f[u].w);
            }
#pragma unroll
            for (int u = 0; u < NP; ++u) {
              fma2(acc[n + u][0], acc[n + u][1], sg, part[u][0], part[u][1]);
              fma2(acc[n + u][2], acc[n + u][3], sh, part[u][2], part[u][3]);
            }
          }
        }
      }
      load(buf[d], half);
      if (half == 0) continue;
      __syncwarp();
      if (lane == 0) mbar_arrive1(&empty[s]);  // this warp has read the stage
      // the stage that the group read a chunk ago takes the next chunk
      // (a refill that does not come off is the last one: the full waits then run out)
      if (producer && ok && it >= 1 && put < limit) {
        if (mbar_wait_limited(&empty[(it - 1) % kTileStages], ((it - 1) / kTileStages) & 1)) {
          inputs();
        } else {
          limit = put;
          stop = 1;
        }
      }
      if (++chunk == nc) {
        finish();
        chunk = 0;
        tile += group;
      }
    }
  }
  // No copy may be in flight when the CTA's shared memory goes away: those of
  // every chunk that was waited for have come; after a wait that ran out, the
  // rest is waited for, again with a limit.
  if (!ok) {
    atomicOr(&g_ops_status, kErrOpsWait);
    if (producer)
      for (int it = max(0, put - kTileStages); it < put; ++it)
        (void)mbar_wait_limited(&full[it % kTileStages], (it / kTileStages) & 1);
  }
}

// limit: the most shared memory that calls of the kernel ask for.  The attribute
// is set to it and not to the call's own size, which a call of another thread
// could lower between here and the launch.
template <class K, class... A>
cudaError_t launch_chained(K kernel, dim3 grid, int threads, int smem, int limit, cudaStream_t s, const A&... a) {
  if (limit > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a...);
}

size_t back_bytes(int n) { return (static_cast<size_t>(n) * sizeof(float2) + 1023) & ~static_cast<size_t>(1023); }

constexpr int kRowsSmem = 110 * 1024;  // two CTAs of q4_kernel per SM
constexpr int kTileSmem = 220 * 1024;  // of q4_tile_kernel
int rows_smem(const Q4Mat& m, int cols) { return 3 * kWarpsQ4 * 512 + cols * (m.nkc * kQ4Chunk * 2 + 64); }

// CTAs of q4_tile_kernel along the outputs, and their shared memory, with kq groups
// of warps and `cols` columns.
int tile_ctas(const Q4Mat& m, int kq) { return (m.ntile + kWarpsQ4 / kq - 1) / (kWarpsQ4 / kq); }
int tile_smem(int kq, int cols) { return kq * kTileStages * (cols * 256) + (kq - 1) * (kWarpsQ4 / kq) * cols * 64; }
bool tile_fits(const Q4Mat& m, int kq, int cols) {
  return kq <= kWarpsQ4 && kq <= m.nkc && tile_smem(kq, cols) <= kTileSmem;
}

// How a call goes: q4_kernel, or q4_tile_kernel in passes of `cols` columns with kq
// groups of warps.  The columns go in one pass, up to 64 of them; but where that
// leaves SMs without a CTA (few outputs), in more passes, which run side by side
// and each unpack the weights: 28 fp32 rows of a 2145 x 7328 matrix took 42 us in
// one pass and 22.7 in four.
struct Q4Plan {
  bool tiles;
  int cols, per_pass, passes, kq;
};
Q4Plan plan_q4(const Q4Mat& m, int n, int x_type, int sms) {
  const int per = x_type == kOpsF32 ? 2 : 1;
  Q4Plan p{};
  const long long cols = static_cast<long long>(n) * per;
  p.tiles = cols > 8 || rows_smem(m, static_cast<int>(cols)) > kRowsSmem;
  if (!p.tiles) return p;
  auto set = [&](int c) {
    p.cols = c;
    p.per_pass = c / per;
    p.passes = (n + p.per_pass - 1) / p.per_pass;
    int most = 1;
    while (tile_fits(m, 2 * most, c)) most *= 2;
    return static_cast<long long>(tile_ctas(m, most)) * p.passes;
  };
  int c = cols <= 8 ? 8 : cols <= 16 ? 16 : cols <= 32 ? 32 : 64;
  while (set(c) < sms && c > 8) c /= 2;
  // the fewest groups that give the SMs 3/2 CTAs each: more of them take more shared
  // memory (64 rows of 4096 x 4096: 16.6 us, and 27 with two CTAs each asked for)
  p.kq = 1;
  while (static_cast<long long>(tile_ctas(m, p.kq)) * p.passes * 2 < 3 * sms && tile_fits(m, 2 * p.kq, p.cols)) p.kq *= 2;
  return p;
}

template <int XT, int SETS, bool ZP>
cudaError_t run_rows(const Q4Kernel& a, int sms, cudaStream_t s) {
  const int smem = rows_smem(a.m, a.tokens * kPartsOf<XT>);
  return launch_chained(q4_kernel<XT, SETS, ZP>, std::min(a.m.ntile, sms * 2), kThreadsQ4, smem, kRowsSmem, s, a);
}

template <int XT, int NT, int SETS, bool ZP>
cudaError_t run_tiles(const Q4Kernel& a, const Q4Plan& p, int sms, cudaStream_t s) {
  const int smem = tile_smem(a.kq, p.cols);
  const int per_sm = std::max(1, std::min(kTileCtas<NT, SETS>, 226 * 1024 / (smem + 2048)));
  const int ctas = std::min(tile_ctas(a.m, a.kq), std::max(1, sms * per_sm / p.passes));
  return launch_chained(q4_tile_kernel<XT, NT, SETS, ZP>, dim3(ctas, p.passes), kThreadsQ4, smem, kTileSmem, s, a);
}

template <class F>
cudaError_t with_sets(const Q4Mat& m, F&& f) {
  using std::integral_constant;
  auto zeros = [&](auto sets) {
    return m.zeros ? f(sets, integral_constant<bool, true>{}) : f(sets, integral_constant<bool, false>{});
  };
  const int sets = kQ4Chunk / m.span;
  return sets == 4   ? zeros(integral_constant<int, 4>{})
         : sets == 2 ? zeros(integral_constant<int, 2>{})
                     : zeros(integral_constant<int, 1>{});
}

template <int XT>
cudaError_t launch_typed(Q4Kernel a, const Q4Args& q, const Q4Plan& p, int sms, cudaStream_t st) {
  if (!p.tiles) {
    a.tokens = q.n;
    return with_sets(a.m, [&](auto sets, auto zp) {
      return run_rows<XT, decltype(sets)::value, decltype(zp)::value>(a, sms, st);
    });
  }
  // the workspace: the factors, then the passes' images
  unsigned char* w = static_cast<unsigned char*>(q.workspace);
  a.back = reinterpret_cast<float2*>(w);
  a.image = w + back_bytes(q.n);
  a.tokens = q.n;
  a.per_pass = p.per_pass;
  a.kq = p.kq;
  const cudaError_t e = launch_chained(q4_image_kernel<XT>, q.n, 256, 0, 0, st, a, p.cols);
  if (e != cudaSuccess) return e;
  return with_sets(a.m, [&](auto sets, auto zp) {
    constexpr int S = decltype(sets)::value;
    constexpr bool Z = decltype(zp)::value;
    return p.cols == 8    ? run_tiles<XT, 1, S, Z>(a, p, sms, st)
           : p.cols == 16 ? run_tiles<XT, 2, S, Z>(a, p, sms, st)
           : p.cols == 32 ? run_tiles<XT, 4, S, Z>(a, p, sms, st)
                          : run_tiles<XT, 8, S, Z>(a, p, sms, st);
  });
}

}  // namespace

void q4_layout(Q4Mat& m) {
  m.span = m.group % 128 == 0 ? 128 : m.group % 64 == 0 ? 64 : 32;
  m.nkc = (m.ins + kQ4Chunk - 1) / kQ4Chunk;
  m.ntile = (m.outs + kQ4Rows - 1) / kQ4Rows;
  const int sets = kQ4Chunk / m.span;
  m.chunk_bytes = 1024 + 32 * sets + (m.zeros ? std::max(32, 16 * sets) : 0);
}

size_t q4_tiles_bytes(const Q4Mat& m) { return static_cast<size_t>(m.ntile) * m.nkc * m.chunk_bytes; }

size_t q4_workspace_bytes(const Q4Mat& m, int n, int x_type) {
  const Q4Plan p = plan_q4(m, n, x_type, sm_count());
  return p.tiles ? back_bytes(n) + static_cast<size_t>(p.passes) * m.nkc * (p.cols * (kQ4Chunk * 2)) : 0;
}

cudaError_t launch_q4_pack(const Q4Mat& m, const unsigned char* q, const uint16_t* s, const unsigned char* zeros,
                           unsigned char* tiles, cudaStream_t st) {
  const long long nchunk = static_cast<long long>(m.ntile) * m.nkc;
  q4_pack_kernel<<<static_cast<unsigned>(std::min(nchunk, sm_count() * 64ll)), 256, 0, st>>>(m, q, s, zeros, tiles);
  return cudaGetLastError();
}

cudaError_t launch_q4(const Q4Mat& m, const Q4Args& q, int x_type, int y_type, cudaStream_t st) {
  Q4Kernel a{};
  a.m = m;
  a.x = q.x;
  a.ldx = q.ldx;
  a.y = q.y;
  a.ldy = q.ldy;
  a.y_type = y_type;
  a.wide = reinterpret_cast<uintptr_t>(q.x) % 16 == 0 && q.ldx * ops_type_size(x_type) % 16 == 0;
  a.xstride = m.nkc * kQ4Chunk * 2 + 64;
  const int sms = sm_count();
  const Q4Plan p = plan_q4(m, q.n, x_type, sms);
  return x_type == kOpsF32    ? launch_typed<kOpsF32>(a, q, p, sms, st)
         : x_type == kOpsBF16 ? launch_typed<kOpsBF16>(a, q, p, sms, st)
                              : launch_typed<kOpsF16>(a, q, p, sms, st);
}

cudaError_t ops_read_status(unsigned* st, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(st, g_ops_status, sizeof(unsigned));
  if (e != cudaSuccess || !clear || !*st) return e;
  const unsigned z = 0;
  return cudaMemcpyToSymbol(g_ops_status, &z, sizeof(unsigned));
}

}  // namespace vb
