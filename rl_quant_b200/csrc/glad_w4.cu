// Rows times 4-bit weights with group scales:
//   y[m, n] = sum_g xs[m, g] * s[n, g] * sum_{k in group g} x[m, k] * q[n, k] + b[n]
//
// The weights are streamed once in the order the kernels read them (include/glad_b200.h: GladW4Weight):
// 8 KB for 128 rows x 128 inputs, in it 1 KB for 16 rows, 512 bytes a warp load: 16 rows x 64 inputs. A 32-bit word is
// one lane's share of the A operand of a 16x8x16 tensor-core product, so a word becomes
// four half2 registers with one logic operation and one half operation each:
// 0x6400 | u is the half 1024 + u, exact for 4-bit u. Products q * x are exact and the sum of
// a group is fp32; the scale multiplies the group's sum, so no weight is ever rounded.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <type_traits>

#include "glad_common.cuh"

namespace glad {
int set_last_error(int code, const char* msg);

namespace {

struct W4Params {
  const uint4* tiles;
  const __half* scales;
  int N, K, U, group;       // U: units of 128 inputs
  const void* x;
  int64_t M, ldx;
  const float* xs;          // scales of 8-bit rows or null
  int xs_rows, xs_groups;   // 0/0: none or one value; 1/1: a row; 1/G: a row and group
  int x_fast;               // rows can be read 8 inputs at a time
  int stream_warps;         // few rows: warps of a stream (2, 4, 8, 16)
  int splits;               // many rows: blocks that share a tile's inputs
  int x_tma;                // many rows: x is read by TMA
  const void* bias;
  void* y;
  int y_dtype;
  int y_vec;                // four columns of y can be stored at once
  uint32_t wait_ns;         // many rows: limit of a wait
  uint32_t hold;            // many rows: barriers that wait for an arrival that never comes (glad_debug_w4_wait; 0)
};

struct e4m3_t { uint8_t v; };

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t b2_sub(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// (w & mask) ^ flip in one logic operation: with both constants as literals the compiler takes two.
__device__ __forceinline__ uint32_t and_xor(uint32_t w, uint32_t mask, uint32_t flip) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(w), "r"(mask), "r"(flip));
  return d;
}
// Eight 4-bit weights -> the A registers of one 16x8x16 product. The two's-complement
// nibble with its top bit flipped is q + 8.
template <bool BF16>
__device__ __forceinline__ void unpack_w4(uint32_t w, uint32_t (&a)[4]) {
  if constexpr (BF16) {
    // 0x4300 | u is the bf16 128 + u (seven mantissa bits): each nibble is shifted to bit 0
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = b2_sub(and_xor(w >> (4 * i), 0x000f000fu, 0x43084308u), 0x43084308u);
  } else {
    a[0] = h2_sub(and_xor(w, 0x000f000fu, 0x64086408u), 0x64086408u);
    a[1] = h2_fma(and_xor(w, 0x00f000f0u, 0x64806480u), 0x2c002c00u, 0xd480d480u);   // (1024 + 16 u) / 16 - 72
    w >>= 8;
    a[2] = h2_sub(and_xor(w, 0x000f000fu, 0x64086408u), 0x64086408u);
    a[3] = h2_fma(and_xor(w, 0x00f000f0u, 0x64806480u), 0x2c002c00u, 0xd480d480u);
  }
}

// Inputs [k, k + 8) of one row as stored: 16 bytes of 16-bit inputs, 8 bytes of 8-bit ones (in
// .x, .y); zero at and past K.
template <typename T>
__device__ __forceinline__ uint4 load_raw8(const T* row, int k, int K, bool fast) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k >= K) return v;
  if constexpr (sizeof(T) == 2) {
    if (fast) {
      v = *reinterpret_cast<const uint4*>(row + k);
    } else {
      const uint16_t* s = reinterpret_cast<const uint16_t*>(row);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = k + 2 * i < K ? s[k + 2 * i] : 0u;
        const uint32_t hi = k + 2 * i + 1 < K ? s[k + 2 * i + 1] : 0u;
        w[i] = lo | (hi << 16);
      }
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    if (fast) {
      const uint2 u = *reinterpret_cast<const uint2*>(row + k);
      v.x = u.x, v.y = u.y;
    } else {
      const uint8_t* s = reinterpret_cast<const uint8_t*>(row);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (k + i < K) v.x |= (uint32_t)s[k + i] << (8 * i);
        if (k + 4 + i < K) v.y |= (uint32_t)s[k + 4 + i] << (8 * i);
      }
    }
  }
  return v;
}
// ... as the four half2 (bf16x2) the products take; e4m3 is exact in fp16.
template <typename T>
__device__ __forceinline__ uint4 to_halves(uint4 v) {
  if constexpr (sizeof(T) == 2) {
    return v;
  } else {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = i < 2 ? v.x : v.y;
      const __half2_raw h =
          __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(i & 1 ? w >> 16 : w & 0xffffu), __NV_E4M3);
      r[i] = (uint32_t)h.x | ((uint32_t)h.y << 16);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
}

__device__ __forceinline__ void store_y(const W4Params& p, int64_t m, int n, float v) {
  const int64_t at = m * p.N + n;
  if (p.y_dtype == GLAD_DTYPE_F16) {
    if (p.bias) v += __half2float(static_cast<const __half*>(p.bias)[n]);
    static_cast<__half*>(p.y)[at] = __float2half_rn(v);
  } else if (p.y_dtype == GLAD_DTYPE_BF16) {
    if (p.bias) v += __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
    static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  } else {
    if (p.bias) v += static_cast<const float*>(p.bias)[n];
    static_cast<float*>(p.y)[at] = v;
  }
}

// Four neighbouring columns; one store where the row allows it.
__device__ __forceinline__ void store_y4(const W4Params& p, int64_t m, int n, const float (&v)[4]) {
  if (!p.y_vec || n + 4 > p.N) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) store_y(p, m, n + e, v[e]);
    return;
  }
  float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t at = m * p.N + n;
  if (p.y_dtype == GLAD_DTYPE_F32) {
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = static_cast<const float*>(p.bias)[n + e];
    }
    *reinterpret_cast<float4*>(static_cast<float*>(p.y) + at) =
        make_float4(v[0] + b[0], v[1] + b[1], v[2] + b[2], v[3] + b[3]);
  } else if (p.y_dtype == GLAD_DTYPE_F16) {
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = __half2float(static_cast<const __half*>(p.bias)[n + e]);
    }
    __half2 h[2] = {__floats2half2_rn(v[0] + b[0], v[1] + b[1]), __floats2half2_rn(v[2] + b[2], v[3] + b[3])};
    *reinterpret_cast<uint2*>(static_cast<__half*>(p.y) + at) = *reinterpret_cast<uint2*>(h);
  } else {
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n + e]);
    }
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0] + b[0], v[1] + b[1]),
                           __floats2bfloat162_rn(v[2] + b[2], v[3] + b[3])};
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.y) + at) = *reinterpret_cast<uint2*>(h);
  }
}

// ---- few rows (up to 8 NT): weight streaming ------------------------------------------------
// One persistent block per SM. Its warps form streams of W warps; each stream walks tiles of 32 columns,
// its warps split the inputs in units of 128 and join their sums in warp order once a tile. Each warp
// brings its own units (2 KB of weights and 128/GROUP * 64 bytes of scales) through a private
// shared-memory ring of cp.async copies kRing - 1 units ahead, across tile borders, so about
// 70 KB are in flight on an SM with rings of three units (up to 8 rows, where x fits beside them) and half of that with two. x is staged once in shared memory, in the form
// the products take (e4m3 as fp16; int8 with the middle two of four inputs swapped, the order in which
// a word's nibbles come apart). Rows past M read row M - 1: their sums are never stored.
// A 32-bit word takes 9 instructions to unpack and one to multiply, so a unit is as
// large as registers allow, which spreads the rest (copies, x, scales, addresses) over more words. Instruction issue is the
// busiest part that a profile shows (59% of the slots at 1 x 28672 x 8192, 43% at 16 x 14336 x 4096 int8; HBM 45% and 22%), but
// not full: 16 warps an SM do not cover the waits between a unit's loads, products and scales.
// 1 x 28672 x 8192 bf16, groups of 128: 121 MB in 29.7 us, 4.1 TB/s, 64% of a copy's rate (f16, one operation less a
// pair: 8 rows 31.5 us; int8, whose words take 4 to unpack: 8 rows 25.8 us, 4.7 TB/s). 1 x 4096 x 4096 f16, groups of
// 64: 8.9 MB in 3.9 us, of which 1.6 us are a launch. 16 columns a step: 30.4 and 4.4 us; registers instead
// of the rings of copies: 76.8 and 7 us (the newest load held up the oldest).
template <int NT, int GROUP, int RING>
struct RowSmem {
  static constexpr int kWarps = 16, kRing = RING;
  static constexpr int kScales = 128 / GROUP;           // groups of a unit
  static constexpr int kWarpSlot = 2048 + kScales * 64;
  static constexpr int kRingBytes = kRing * kWarps * kWarpSlot;
  static constexpr int kBuffers = NT == 1 ? 2 : 1;      // of every warp's sums
  static constexpr int kPart = 8 * NT * 33;             // floats of a warp's sums
  static constexpr int kFixed = kRingBytes + kBuffers * kWarps * kPart * 4;
};

// D = A * B + 0 / D += A * B, m16n8k16 (f16, bf16 -> f32) and m16n8k32 (s8 -> s32).
template <bool BF16, bool FIRST>
__device__ __forceinline__ void mma_rows(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (FIRST) {
    if constexpr (BF16)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  } else {
    if constexpr (BF16)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
template <bool FIRST>
__device__ __forceinline__ void mma_rows_i8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (FIRST)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The 4-bit pieces of a word as int8 times 16 (the nibble in the byte's high half): rows r and r + 8.
__device__ __forceinline__ uint32_t w4_low16(uint32_t w) { return (w << 4) & 0xf0f0f0f0u; }
__device__ __forceinline__ uint32_t w4_high16(uint32_t w) { return w & 0xf0f0f0f0u; }
__device__ __forceinline__ uint32_t swap_mid(uint32_t v) { return __byte_perm(v, 0, 0x3120); }

template <typename TX, int NT, int GROUP, int RING>
__global__ void __launch_bounds__(512, 1) w4_rows_kernel(const __grid_constant__ W4Params p) {
  using L = RowSmem<NT, GROUP, RING>;
  constexpr bool BF16 = std::is_same<TX, __nv_bfloat16>::value, I8 = std::is_same<TX, int8_t>::value;
  constexpr int SG = L::kScales, XP = I8 ? 8 : 16;       // bytes of eight staged inputs
  constexpr int kRing = L::kRing, kThreads = L::kWarps * 32;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* xs = smem + L::kFixed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int T = (p.N + 31) / 32, U = p.U, M = (int)p.M, W = p.stream_warps;
  const int stream = warp / W, ws = warp - stream * W;   // the stream's tiles are first, first + step, ...
  const int first = stream * gridDim.x + blockIdx.x, step = gridDim.x * (L::kWarps / W);
  const int u0 = (int)((int64_t)ws * U / W), u1 = (int)((int64_t)(ws + 1) * U / W);
  uint8_t* ring = smem + warp * (kRing * L::kWarpSlot);
  float* part = reinterpret_cast<float*>(smem + L::kRingBytes) + stream * W * L::kPart;

  // the next unit to fetch: tile pt, unit pu
  int pt = u0 < u1 ? first : T, pu = u0;
  const uint4* wsrc = nullptr;
  const uint8_t* ssrc = nullptr;
  auto seek = [&]() {
    const int64_t at = ((int64_t)(pt >> 2) * U + pu) * 4 + (pt & 3);   // 2 KB blocks
    wsrc = p.tiles + at * 128 + lane;
    ssrc = reinterpret_cast<const uint8_t*>(p.scales) + at * (SG * 64) + lane * 16;
  };
  seek();
  auto fetch = [&](int slot) {
    if (pt < T) {
      uint8_t* dst = ring + slot * L::kWarpSlot + lane * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i) cp_async16(dst + i * 512, wsrc + i * 32);
      if (lane < SG * 4) cp_async16(dst + 2048, ssrc);
      wsrc += 4 * 128;
      ssrc += 4 * SG * 64;
      if (++pu == u1) {
        pu = u0;
        pt += step;
        seek();
      }
    }
    cp_async_commit();
  };
  grid_dep_wait();
  grid_dep_launch();
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) fetch(i);

  auto staged = [&](uint4 v) -> uint4 {
    if constexpr (I8) return make_uint4(swap_mid(v.x), swap_mid(v.y), 0, 0);
    else return to_halves<TX>(v);
  };
  {
    // [32-input block][row][lane c of four][inputs 4c..4c+3, 16+4c..]: a warp's reads of eight rows are contiguous
    const int pieces = U * 16 * M;
    for (int i = threadIdx.x; i < pieces; i += kThreads) {
      const int m = i / (U * 16), k8 = i - m * (U * 16);
      const uint4 v = staged(load_raw8<TX>(static_cast<const TX*>(p.x) + m * p.ldx, k8 * 8, p.K, p.x_fast));
      uint8_t* dst = xs + (((k8 >> 2) * M + m) * 4 + (k8 & 1) * 2) * XP + ((k8 >> 1) & 1) * (XP / 2);
      if constexpr (I8) {
        *reinterpret_cast<uint32_t*>(dst) = v.x;
        *reinterpret_cast<uint32_t*>(dst + XP) = v.y;
      } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(v.x, v.y);
        *reinterpret_cast<uint2*>(dst + XP) = make_uint2(v.z, v.w);
      }
    }
    __syncthreads();
  }
  const uint8_t* xrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int m = min(8 * j + r, M - 1);
    xrow[j] = xs + (m * 4 + c) * XP;
  }
  const int xstep = M * 4 * XP;                          // bytes of 32 inputs of all rows

  int slot = 0, buffer = 0;
  for (int t = first; t < T; t += step) {
    float acc[2][NT][4];                                 // [16 columns][8 rows]
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[h][j][e] = 0.0f;
    const uint8_t* xat[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) xat[j] = xrow[j] + 4 * u0 * xstep;
    for (int u = u0; u < u1; ++u) {
      cp_async_wait_group<kRing - 2>();
      __syncwarp();
      fetch(slot == 0 ? kRing - 1 : slot - 1);           // the slot that every lane has just left
      const uint8_t* in = ring + slot * L::kWarpSlot;
      slot = slot + 1 == kRing ? 0 : slot + 1;
      float g[2][NT][4];
      int gi8[2][NT][4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        uint4 w4[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) w4[h] = *reinterpret_cast<const uint4*>(in + h * 1024 + kb * 512 + lane * 16);
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2) {                 // 32 inputs at a time
          constexpr int QG = GROUP / 32;
          const int q = 2 * kb + q2;
          uint4 x[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if constexpr (I8) {
              const uint2 v = *reinterpret_cast<const uint2*>(xat[j]);
              x[j] = make_uint4(v.x, v.y, 0, 0);
            } else {
              x[j] = *reinterpret_cast<const uint4*>(xat[j]);
            }
            xat[j] += xstep;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w0 = q2 ? w4[h].z : w4[h].x, w1 = q2 ? w4[h].w : w4[h].y;
            if constexpr (I8) {
              const uint32_t a[4] = {w4_low16(w0), w4_high16(w0), w4_low16(w1), w4_high16(w1)};
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if (q % QG == 0) mma_rows_i8<true>(gi8[h][j], a, x[j].x, x[j].y);
                else mma_rows_i8<false>(gi8[h][j], a, x[j].x, x[j].y);
              }
            } else {
              uint32_t a0[4], a1[4];
              unpack_w4<BF16>(w0, a0);
              unpack_w4<BF16>(w1, a1);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if (q % QG == 0) mma_rows<BF16, true>(g[h][j], a0, x[j].x, x[j].y);
                else mma_rows<BF16, false>(g[h][j], a0, x[j].x, x[j].y);
                mma_rows<BF16, false>(g[h][j], a1, x[j].z, x[j].w);
              }
            }
          }
          if ((q + 1) % QG == 0) {
            const int gi = q / QG;
            float2 s[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[h] = __half22float2(*reinterpret_cast<const __half2*>(in + 2048 + h * (SG * 32) + gi * 32 + r * 4));
              if constexpr (I8) s[h].x *= 0.0625f, s[h].y *= 0.0625f;   // the codes were multiplied by 16
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              float x0 = 1.0f, x1 = 1.0f;
              const bool by_group = sizeof(TX) == 1 && p.xs_groups > 1;
              if (by_group) {
                const int m = 8 * j + 2 * c, xg = u * SG + gi;
                x0 = (m < M && xg < p.xs_groups) ? p.xs[m * p.xs_groups + xg] : 0.0f;
                x1 = (m + 1 < M && xg < p.xs_groups) ? p.xs[(m + 1) * p.xs_groups + xg] : 0.0f;
              }
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if constexpr (I8) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) g[h][j][e] = i2f_small(gi8[h][j][e]);   // at most 2^21
                }
                if (by_group) g[h][j][0] *= x0, g[h][j][1] *= x1, g[h][j][2] *= x0, g[h][j][3] *= x1;
                acc[h][j][0] = fmaf(s[h].x, g[h][j][0], acc[h][j][0]);
                acc[h][j][1] = fmaf(s[h].x, g[h][j][1], acc[h][j][1]);
                acc[h][j][2] = fmaf(s[h].y, g[h][j][2], acc[h][j][2]);
                acc[h][j][3] = fmaf(s[h].y, g[h][j][3], acc[h][j][3]);
              }
            }
          }
        }
      }
    }
    // with two buffers, the one written now was last read before the previous tile's barrier
    float* mine = part + (buffer * L::kWarps + ws) * L::kPart;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (8 * j + 2 * c + (e & 1) < M) mine[(8 * j + 2 * c + (e & 1)) * 33 + 16 * h + r + 8 * (e >> 1)] = acc[h][j][e];
    named_bar_sync(1 + stream, W * 32);
    for (int i = ws * 32 + lane; i < M * 32; i += W * 32) {
      const int row = i >> 5, col = i & 31, n = 32 * t + col;
      const float* all = part + buffer * L::kWarps * L::kPart + row * 33 + col;
      float v = 0.0f;
#pragma unroll 4
      for (int k = 0; k < W; ++k) v += all[k * L::kPart];
      if (p.xs != nullptr && p.xs_groups <= 1) v *= p.xs[p.xs_rows ? row : 0];
      if (n < p.N) store_y(p, row, n, v);
    }
    if constexpr (L::kBuffers == 2) buffer ^= 1;
    else named_bar_sync(1 + stream, W * 32);
  }
}

// ---- many rows: tcgen05 -----------------------------------------------------------------------
// A block computes 128 output columns x MT rows; D[n, m] lives in tensor memory, n its lanes. The
// inputs go in stages of 128 (one or two swizzle atoms of 128 bytes a row). Roles by
// warp: one brings the packed weights (bulk copies, PD units of 128 inputs ahead), one the x tile
// (TMA, NS stages ahead); teams of four unpack the weights of a unit each, in x's own type:
// f16 or bf16, int8 times 16, or e4m3 times 2^-9, all exact, and store them in tensor memory as the A operand (a
// warp's fragment order is the order of its 16x256b / 16x128b stores), so shared memory, whose
// bandwidth bounded the same kernel with A in it, carries only x; MW issue the products of
// groups in turn. Every group of inputs has an accumulator of its own (ND in rotation): SW warps
// read it back, scale it by s[n, g] (a lane's own row: one value a thread) and add it to fp32 sums in
// registers, so the weights need no rounding; that costs one multiply-add an output and group, at
// groups of 64 half of the tensor core's time for them at fp16 rate. Blocks of a cluster split the
// inputs when there are fewer tiles than SMs, send their sums to the rows' owners through
// distributed shared memory and add them in rank order.
// 1024 x 4096 x 4096 f16, groups of 64: 48.9 us, 0.70 PFLOP/s, 42% of a library product's rate (two rounds of tiles on 148
// SMs: 512 rows, one round, 25.0 us); groups of 128, 512 rows: 20.8 us, 0.82 PFLOP/s. 64 rows of e4m3 x 4096 x 14336,
// groups of 128 with scales of both: 30.8 MB in 20.5 us. Neither HBM (14% busy there) nor the tensor core (524 of
// 1250 clocks a unit at groups of 128) is the bound but the issue slots (57 to 71% busy) of unpacking and sums
// and the hand-offs between them. A deeper ring of x (54 us where four stages took 47.5), 16 unpacking warps, one or four
// product warps and tiles of 256 rows were slower or no faster.
__device__ unsigned int g_w4_status;
// Reads and clears the status word in one step, so that a bit set meanwhile is either returned or stays; the copies that
// calls at the same time bring to the host have words of their own.
constexpr int kStatusCalls = 64;
__device__ unsigned int g_w4_taken[kStatusCalls];
__global__ void w4_take_status_kernel(int slot) { g_w4_taken[slot] = atomicExch(&g_w4_status, 0u); }

template <int XB, int MT, int GROUP>                     // XB: bytes of an input
struct Tile {
  static constexpr int NS = 8 / XB;                      // stages: operands of a unit (128 inputs)
  static constexpr int PD = MT < 128 ? 12 : XB == 2 ? 8 : 4;       // units of packed weights in flight
  static constexpr int ND = MT == 128 ? 2 : 4;
  static constexpr int SG = 128 / GROUP;                 // groups of a unit
  static constexpr int SPG = GROUP * XB / 32;            // products (32 bytes of inputs) of a group
  static constexpr int ACOLS = 32 * XB;                  // tensor-memory columns of a stage's A
  static constexpr int MW = 2;                           // warps that issue products
  static constexpr int SW = MT == 128 ? 16 : 8;          // warps that take the sums
  static constexpr int DW = 8;                           // warps that unpack
  static constexpr int kThreads = (SW + DW + MW + 2) * 32;
  static constexpr int NC = MT * 4 / SW;                 // columns of a sums thread
  // Paired multiply-adds of the sums: 1024 x 4096 x 4096 f16, groups of 64: 53.9 -> 48.9 us. With one group a unit
  // they gain nothing (512 rows: 20.8 us alone, 22.3 us paired), and 8-bit rows spill (512 rows of e4m3,
  // groups of 32: 97 -> 119 us).
  static constexpr bool kPacked = XB == 2 && SG > 1;
  static constexpr int kBlock = MT * 128, kStage = XB * kBlock;    // x of a stage: 128 bytes a row and block
  static constexpr int kSlot = 8192;                     // packed weights of a unit
  static constexpr int SD = 4;                           // units of weight scales in flight, a copy a warp
  static constexpr int kWs = SG * 64;                    // weight scales of a unit and 32 rows
  // x scales: two blocks of eight groups (XF units), [group][NC + 4 columns] (no bank conflicts of the copies)
  static constexpr int XF = 8 / SG, XPITCH = NC + 4, kXs = XB == 1 ? 2 * 8 * XPITCH * 4 : 0;
  static constexpr int kSums = SD * kWs + kXs;           // scales of a sums warp
  static constexpr int kSmem = NS * kStage + PD * kSlot + SW * kSums + 512 + 1024;
  static constexpr int kACol = ND * MT;                  // first tensor-memory column of A
  static constexpr int kCols = ND * MT + NS * ACOLS <= 256 ? 256 : 512;
  static_assert(ND * MT + NS * ACOLS <= kCols, "tensor memory");
  static_assert(NS % MW == 0 && ND % MW == 0 && PD % (DW / 4) == 0 && NS % (DW / 4) == 0, "phases");
  static_assert(2 * MT * 512 <= NS * kStage, "the sums are sent and joined in the stage buffers");
  static_assert(kSmem <= 232448, "shared memory of one block");
  static_assert((2 * NS + 2 * PD + 2 * ND + 1 + MW) * 8 + 12 <= 512, "barrier area");
};

// Wait for a phase, abort[1] nanoseconds at most; then abort[0] is set, which ends every wait of the block. The timer
// is read only after many tries: a read costs more than most waits.
__device__ __noinline__ bool w4_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort) {
  for (int i = 0; i < 1000; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!*abort) {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (global_timer_ns() - t0 > (uint32_t)abort[1]) {
      *abort = 1;
      atomicOr(&g_w4_status, kDevErrMmaTimeout);
    }
  }
  return false;
}
__device__ __forceinline__ bool w4_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return mbar_try_wait(bar, parity) || w4_wait_slow(bar, parity, abort);
}
// The same by a whole warp: lanes may see a phase end, or the block give up, at different tries, and what follows
// (tensor-memory accesses, elections) takes all of them or none.
__device__ __forceinline__ bool w4_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) ||
         __all_sync(0xffffffffu, w4_wait_slow(bar, parity, abort));
}
// How long a warp waits at its end for copies and products that it issued: they take microseconds, but the barrier
// may also count arrivals of others, which do not come after a wait has run out.
constexpr uint64_t kDrainNs = 10000000;

// K-major operand with 128-byte swizzle: rows of 128 bytes, 8-row groups 1024 bytes apart, the 16-byte
// piece i of row r at i ^ (r & 7).
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// One lane of a converged warp, the same every time. With warp-uniform operands the single-thread
// instructions then take them from uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0;
}
// D (+)= A (tensor memory) * B^T, one thread issues: 32 bytes of inputs.
#define W4_MMA_TS(name, kind)                                                                                \
  __device__ __forceinline__ void name(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) { \
    asm volatile(                                                                                            \
        "{\n\t.reg .pred p;\n\t"                                                                              \
        "setp.ne.b32 p, %4, 0;\n\t"                                                                            \
        "tcgen05.mma.cta_group::1.kind::" kind " [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),                           \
        "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)                                                              \
        : "memory");                                                                                         \
  }
W4_MMA_TS(mma_ts_f16, "f16")
W4_MMA_TS(mma_ts_i8, "i8")
W4_MMA_TS(mma_ts_f8, "f8f6f4")
#undef W4_MMA_TS
// 16 lanes x 32 (16) columns: thread 4g + q gives, of every 8 (4) columns, lane g's columns 2q, 2q + 1
// (q) and the same of lane g + 8.
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void tmem_st_16x128b_x4(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// x tile: 128 bytes of MT rows, zero outside the tensor, swizzled as desc_sw128 reads it.
__device__ __forceinline__ void tma_x(uint32_t dst, const CUtensorMap* map, int k, int m, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(k), "r"(m), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void cp_async4_zfill(void* dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// acc += s * f, four values; PACKED: two multiply-adds an instruction (a pair of neighbouring registers).
template <bool PACKED>
__device__ __forceinline__ void add_scaled(float* acc, float s, const float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    if constexpr (PACKED)
      asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %2};\n\tmov.b64 b, {%3, %4};\n\tmov.b64 c, {%0, %1};\n\t"
          "fma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
          : "+f"(acc[i]), "+f"(acc[i + 1])
          : "f"(s), "f"(f[i]), "f"(f[i + 1]));
    else
      acc[i] = fmaf(s, f[i], acc[i]), acc[i + 1] = fmaf(s, f[i + 1], acc[i + 1]);
  }
}
// Cluster barrier in two halves, without ordering of memory accesses.
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// Shared memory of this block -> the same or another block of the cluster; counted on the receiver's barrier.
__device__ __forceinline__ void bulk_copy_s2c(uint32_t dst_cluster, uint32_t src, uint32_t bytes, uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst_cluster),
      "r"(src), "r"(bytes), "r"(bar_cluster)
      : "memory");
}

// Every byte's top bit in all eight of its bits.
__device__ __forceinline__ uint32_t byte_signs(uint32_t w) {
  uint32_t d;
  asm("prmt.b32 %0, %1, 0, 0xba98;" : "=r"(d) : "r"(w));
  return d;
}
// The eight weights of a word as bytes in the operand's type: lo = row r, hi = row r + 8, inputs
// k .. k + 3 in order.
template <bool E4M3>
__device__ __forceinline__ void unpack_w4_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (!E4M3) {
    lo = swap_mid(w4_low16(w));
    hi = swap_mid(w4_high16(w));
  } else {
    // sign and magnitude: the codes 0 to 8 are the magnitude times 2^-9 (subnormals and the first normal number), and
    // a negative nibble n has the magnitude 16 - n = (n ^ 15) + 1. Picking q's own codes from tables took a
    // quarter more instructions (17 x 4096 x 14336, groups of 128: 18.7 against 14.7 us).
    const uint32_t ml = byte_signs(w << 4), mh = byte_signs(w);
    lo = swap_mid(((w ^ ml) & 0x0f0f0f0fu) + (ml & 0x81818181u));
    hi = swap_mid((((w >> 4) ^ mh) & 0x0f0f0f0fu) + (mh & 0x81818181u));
  }
}

template <typename TX, int MT, int GROUP>
__global__ void __launch_bounds__(Tile<(int)sizeof(TX), MT, GROUP>::kThreads, 1)
    w4_tile_kernel(const __grid_constant__ W4Params p, const __grid_constant__ CUtensorMap xmap) {
  using L = Tile<(int)sizeof(TX), MT, GROUP>;
  constexpr bool BF16 = std::is_same<TX, __nv_bfloat16>::value, I8 = std::is_same<TX, int8_t>::value;
  constexpr bool E4M3 = std::is_same<TX, e4m3_t>::value;
  constexpr int XB = (int)sizeof(TX), SG = L::SG, NC = L::NC;
  constexpr int SW = L::SW, DW = L::DW, CTL = SW + DW;   // first control warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = smem + L::NS * L::kStage;
  uint8_t* scale_ring = slots + L::PD * L::kSlot;
  uint64_t* full = reinterpret_cast<uint64_t*>(scale_ring + L::SW * L::kSums);
  uint64_t* empty = full + L::NS;                        // [NS] products done; full: operands written
  uint64_t* wfull = empty + L::NS;                       // [PD]
  uint64_t* wempty = wfull + L::PD;                      // [PD]
  uint64_t* dfull = wempty + L::PD;                      // [ND]
  uint64_t* dempty = dfull + L::ND;                      // [ND]
  uint64_t* joined = dempty + L::ND;                     // sums of the cluster's other blocks are here
  uint64_t* drain = joined + 1;                          // [MW] all products of a warp are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + L::MW);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);   // {a wait ran out, the limit in ns}

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // warp-uniform
  const int S = p.splits, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int nt = blockIdx.x / S;
  const int64_t m0 = (int64_t)blockIdx.y * MT;
  const int U = p.U, un0 = (int)((int64_t)rank * U / S), un1 = (int)((int64_t)(rank + 1) * U / S);
  const int units = un1 - un0;

  if (warp == CTL) tmem_alloc(tmem_slot, L::kCols);
  if (tid == 0) {
    for (int i = 0; i < L::NS; ++i) {
      mbar_init(&full[i], 4 + (p.x_tma ? 1 : 0) + (p.hold & 1));
      mbar_init(&empty[i], SG < L::MW ? SG : L::MW);
    }
    for (int i = 0; i < L::PD; ++i) {
      mbar_init(&wfull[i], 1);
      mbar_init(&wempty[i], 4 + (p.hold >> 2 & 1));
    }
    for (int i = 0; i < L::ND; ++i) {
      mbar_init(&dfull[i], 1);
      mbar_init(&dempty[i], SW + (p.hold >> 1 & 1));
    }
    mbar_init(joined, 1 + (p.hold >> 3 & 1));
    for (int i = 0; i < L::MW; ++i) mbar_init(&drain[i], 1);
    fence_mbar_init();
    abort[0] = 0;
    abort[1] = (int)p.wait_ns;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  grid_dep_wait();
  grid_dep_launch();

  if (warp >= CTL) {
    if (warp == CTL + L::MW) {
      // ---- packed weights
      if (elect_one()) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(p.tiles) + ((int64_t)nt * U + un0) * 8192;
        int i = 0;
        for (; i < units; ++i, src += 8192) {
          const int slot = i % L::PD;
          if (i >= L::PD && !w4_wait(&wempty[slot], (i / L::PD - 1) & 1, abort)) break;
          mbar_arrive_expect_tx(&wfull[slot], 8192);
          bulk_copy_g2s(slots + slot * L::kSlot, src, 8192, &wfull[slot]);
        }
        // copies that were issued land before the block leaves, also where nobody waits for them any more
        for (int k = max(0, i - L::PD); k < i; ++k) mbar_wait_bounded(&wfull[k % L::PD], (k / L::PD) & 1, kDrainNs);
      }
    } else if (warp == CTL + L::MW + 1) {
      // ---- x tiles
      if (p.x_tma && elect_one()) {
        const uint32_t base = smem_u32(smem);
        int i = 0;
        for (; i < units; ++i) {
          const int st = i % L::NS;
          if (i >= L::NS && !w4_wait(&empty[st], (i / L::NS - 1) & 1, abort)) break;
          mbar_arrive_expect_tx(&full[st], L::kStage);
#pragma unroll
          for (int h = 0; h < XB; ++h)
            tma_x(base + st * L::kStage + h * L::kBlock, &xmap, (un0 + i) * 128 + h * 64, (int)m0, &full[st]);
        }
        for (int k = max(0, i - L::NS); k < i; ++k) mbar_wait_bounded(&full[k % L::NS], (k / L::NS) & 1, kDrainNs);
      }
    } else {
      // ---- products of every MW-th group. A wait must meet every phase of its barrier (phases are told apart
      // by parity alone): NS and ND being multiples of MW, a stage's and an accumulator's buffers are always
      // the same warps'.
      constexpr uint32_t idesc = I8 ? idesc_i8(128, MT) : idesc_f16(128, MT) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
      const uint32_t base = smem_u32(smem);
      const int me = warp - CTL;
      bool ok = true;
      for (int u = 0; ok && u < units; ++u) {
        const int st = u % L::NS;
        if (SG < L::MW && (me - u * SG % L::MW + L::MW) % L::MW >= SG) continue;   // none of this unit's groups
        ok = w4_wait_warp(&full[st], (u / L::NS) & 1, abort);
        const uint32_t a = tmem + L::kACol + st * L::ACOLS;
        const uint64_t b = desc_sw128(base + st * L::kStage);
#pragma unroll
        for (int j = 0; j < SG; ++j) {
          const int gi = u * SG + j, d = gi % L::ND;
          if (gi % L::MW != me) continue;
          if (ok && gi >= L::ND) ok = w4_wait_warp(&dempty[d], (gi / L::ND - 1) & 1, abort);
          tc_fence_after();
          if (ok && elect_one()) {
#pragma unroll
            for (int e = 0; e < L::SPG; ++e) {           // 32 bytes of inputs: 8 columns of A, 32 bytes of B's rows
              const int q = j * L::SPG + e;
              const uint64_t bq = b + (q >> 2) * (L::kBlock >> 4) + (q & 3) * 2;
              if constexpr (I8) mma_ts_i8(tmem + d * MT, a + 8 * q, bq, idesc, e > 0 ? 1u : 0u);
              else if constexpr (E4M3) mma_ts_f8(tmem + d * MT, a + 8 * q, bq, idesc, e > 0 ? 1u : 0u);
              else mma_ts_f16(tmem + d * MT, a + 8 * q, bq, idesc, e > 0 ? 1u : 0u);
            }
            mma_commit(&dfull[d]);
          }
          __syncwarp();
        }
        if (ok && elect_one()) mma_commit(&empty[st]);
        __syncwarp();
      }
      // products that were issued end before their operands and accumulators go, also where nobody waits for them any
      // more. A barrier of its own: the phases of dfull do not tell which use of an accumulator was the last.
      if (elect_one()) mma_commit(&drain[me]);
      __syncwarp();
      mbar_wait_bounded(&drain[me], 0, kDrainNs);
    }
  } else if (warp >= SW) {
    // ---- A operand
    const int dw = warp & 3;                             // SW is a multiple of four: also the lane quarter
    const uint32_t sbase = smem_u32(smem);
    bool ok = true;

    // x that TMA cannot read (rows off 16 bytes): 128 bytes a row of unit u by guarded loads
    auto copy_x = [&](int u, int h) {
      const uint32_t b = sbase + (u % L::NS) * L::kStage + h * L::kBlock;
#pragma unroll 1
      for (int id = dw * 32 + lane; id < MT * 8; id += 128) {
        const int row = id >> 3, piece = id & 7;
        const int k = (un0 + u) * 128 + h * 64 + piece * (16 / XB);
        const int64_t m = m0 + row;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (m < p.M) {
          const TX* src = static_cast<const TX*>(p.x) + m * p.ldx;
          v = load_raw8<TX>(src, k, p.K, false);
          if constexpr (XB == 1) {
            const uint4 u = load_raw8<TX>(src, k + 8, p.K, false);
            v.z = u.x, v.w = u.y;
          }
        }
        st_shared_v4(b + row * 128 + ((piece ^ (row & 7)) << 4), v.x, v.y, v.z, v.w);
      }
    };
    for (int u = (warp - SW) >> 2; u < units; u += DW / 4) {   // a team meets all phases of its slots
      const int slot = u % L::PD;
      if (ok) ok = w4_wait_warp(&wfull[slot], (u / L::PD) & 1, abort);
      if (ok && u >= L::NS) ok = w4_wait_warp(&empty[u % L::NS], (u / L::NS - 1) & 1, abort);
      if (!ok) break;
      tc_fence_after();
      const uint8_t* in = slots + slot * L::kSlot;
      uint4 packed[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        packed[e] = *reinterpret_cast<const uint4*>(in + (dw * 2 + (e & 1)) * 1024 + (e >> 1) * 512 + lane * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n16 = dw * 2 + (e & 1), kb = e >> 1;   // 16 rows x 64 inputs
        const uint4 w = packed[e];
        const uint32_t word[4] = {w.x, w.y, w.z, w.w};
        const uint32_t at = tmem + ((uint32_t)(16 * n16) << 16) + L::kACol;
        if constexpr (XB == 2) {
          uint32_t v[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) {                  // 16 inputs: (row r: 2 registers) (row r + 8: 2)
            uint32_t a[4];
            unpack_w4<BF16>(word[j], a);
            v[4 * j] = a[0], v[4 * j + 1] = a[2], v[4 * j + 2] = a[1], v[4 * j + 3] = a[3];
          }
          tmem_st_16x256b_x4(at + (u % L::NS) * L::ACOLS + kb * 32, v);
        } else {
          uint32_t v[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) unpack_w4_bytes<E4M3>(word[j], v[2 * j], v[2 * j + 1]);
          tmem_st_16x128b_x4(at + (u % L::NS) * L::ACOLS + kb * 16, v);
        }
      }
      if (!p.x_tma) {
#pragma unroll
        for (int h = 0; h < XB; ++h) copy_x(u, h);
        fence_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&wempty[slot]);
        mbar_arrive(&full[u % L::NS]);
      }
    }
  } else {
    // ---- sums
    const int q4 = warp & 3, col0 = (warp >> 2) * NC;
    const bool by_group = XB == 1 && p.xs_groups > 1;
    // the scales this warp multiplies by, in a ring of its own: the weights' are fetched SD - 1 units ahead, x's
    // in blocks of eight groups (one 32-byte sector a row: a group at a time, each copy was a sector of its own, which
    // bound the kernel: 512 x 4096 x 4096 int8 rows, groups of 64: 75 us) one block ahead
    uint8_t* ring = scale_ring + warp * L::kSums;
    float* xring = reinterpret_cast<float*>(ring + L::SD * L::kWs);
    const uint8_t* wsrc = reinterpret_cast<const uint8_t*>(p.scales) + (((int64_t)nt * U + un0) * 8 + q4 * 2) * (SG * 32);
    auto fetch_x = [&](int block) {
      if (by_group && block * L::XF < units) {
#pragma unroll
        for (int id = lane; id < 8 * NC; id += 32) {
          const int g = id & 7, xg = un0 * SG + block * 8 + g;
          const int64_t m = m0 + col0 + (id >> 3);
          const bool live = m < p.M && xg < p.xs_groups;
          cp_async4_zfill(xring + ((block & 1) * 8 + g) * L::XPITCH + (id >> 3),
                          p.xs + (live ? m * p.xs_groups + xg : 0), live);
        }
      }
    };
    auto fetch = [&](int u) {
      if (u < units && lane < SG * 4)
        cp_async16(ring + (u % L::SD) * L::kWs + lane * 16, wsrc + (int64_t)u * (8 * SG * 32) + lane * 16);
      cp_async_commit();
    };
    float acc[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = 0.0f;
    bool ok = true;
    if (XB == 1) fetch_x(0);
#pragma unroll
    for (int i = 0; i < L::SD - 1; ++i) fetch(i);
    for (int u = 0; ok && u < units; ++u) {
      // copies are committed with the unit SD - 1 ahead; a block of x scales is needed XF units after its commit
      cp_async_wait_group<XB == 1 && L::XF < L::SD - 1 ? L::XF - 1 : L::SD - 2>();
      __syncwarp();
      if (XB == 1 && u % L::XF == 0) fetch_x(u / L::XF + 1);   // the slots that every lane has just left
      fetch(u + L::SD - 1);
      const uint8_t* in = ring + (u % L::SD) * L::kWs;
      float sc[SG];
#pragma unroll
      for (int j = 0; j < SG; ++j) {
        sc[j] = __half2float(reinterpret_cast<const __half*>(in)[((lane >> 4) * SG + j) * 16 + (lane & 7) * 2 + ((lane >> 3) & 1)]);
        if (I8) sc[j] *= 0.0625f;                        // the int8 operand is 16 q
        if (E4M3) sc[j] *= 512.0f;                       // the e4m3 operand is 2^-9 q
      }
#pragma unroll
      for (int j = 0; j < SG; ++j) {
        const int gi = u * SG + j, d = gi % L::ND;
        if (ok) ok = w4_wait_warp(&dfull[d], (gi / L::ND) & 1, abort);
        tc_fence_after();
        // one piece of 16 columns is read while the one before is added, where registers allow it
        constexpr int CH = 16, PIECES = NC / CH, AHEAD = MT == 128 ? 0 : 1;
        const uint32_t at = tmem + ((uint32_t)(32 * q4) << 16) + d * MT + col0;
        uint32_t v[AHEAD + 1][CH];
        if (AHEAD) tmem_ld16(at, v[0]);
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          if (!AHEAD) tmem_ld16(at + k * CH, v[0]);
          tmem_ld_wait();
          if (AHEAD && k + 1 < PIECES) tmem_ld16(at + (k + 1) * CH, v[(k + 1) & AHEAD]);
          uint32_t (&w)[CH] = v[k & AHEAD];
#pragma unroll
          for (int e = 0; e < CH; e += 4) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = I8 ? i2f_small((int)w[e + i]) : __uint_as_float(w[e + i]);   // |int| <= 2^21
            if (by_group) {
              const float4 x = *reinterpret_cast<const float4*>(xring + (gi & 15) * L::XPITCH + k * CH + e);
              f[0] *= x.x, f[1] *= x.y, f[2] *= x.z, f[3] *= x.w;
            }
            add_scaled<L::kPacked>(&acc[k * CH + e], sc[j], f);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dempty[d]);
      }
    }
    cp_async_wait_all();
    // every product is done, so the stage buffers are free: [m][n]
    float* mine = reinterpret_cast<float*>(smem) + 32 * q4 + lane;
#pragma unroll
    for (int i = 0; i < NC; ++i) mine[(col0 + i) * 128] = acc[i];
    if (S > 1) fence_async_smem();
  }
  __syncwarp();
  // Rows m of rank k's share are contiguous: one copy a receiver, into [source rank][m of the owner][n]
  // behind the sums, once every block of the cluster has left its stage buffers.
  const int own = MT / S;
  const float* sums = reinterpret_cast<const float*>(smem) + lane * 4;
  if (S > 1) {
    cluster_sync_all();
    sums += MT * 128;
    if (tid == 0) mbar_arrive_expect_tx(joined, MT * 512);
    if (tid < S)
      bulk_copy_s2c(mapa_shared(smem_u32(smem) + (MT + rank * own) * 512, tid), smem_u32(smem) + tid * own * 512, own * 512,
                    mapa_shared(smem_u32(joined), tid));
    if (!w4_wait_warp(joined, 0, abort)) mbar_wait_bounded(joined, 0, kDrainNs);
    __syncwarp();
    cluster_arrive_relaxed();                            // this block has received all that is sent to it
  } else {
    __syncthreads();
  }
  if (!*abort) {
    const int n = nt * 128 + 4 * lane;
    for (int i = warp; i < own; i += L::kThreads / 32) {
      const int64_t m = m0 + rank * own + i;
      if (m >= p.M || n >= p.N) continue;
      float4 f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < S) f[k] = *reinterpret_cast<const float4*>(sums + (k * own + i) * 128);
      float v[4] = {f[0].x, f[0].y, f[0].z, f[0].w};
#pragma unroll
      for (int k = 1; k < 8; ++k)
        if (k < S) v[0] += f[k].x, v[1] += f[k].y, v[2] += f[k].z, v[3] += f[k].w;
      if (p.xs != nullptr && p.xs_groups <= 1) {
        const float s = p.xs[p.xs_rows ? m : 0];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= s;
      }
      store_y4(p, m, n, v);
    }
  }
  __syncwarp();
  if (S > 1) cluster_wait();                             // the others have received what this block sent
  tc_fence_before();
  __syncthreads();
  if (warp == CTL) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }
}

// ---- launch -------------------------------------------------------------------------------------
// Failure-path test hook (glad_debug_w4_wait): process-wide, read at launch.
uint32_t g_w4_hold = 0;
uint32_t g_w4_wait_ns = 2000000000u;

int current_device() {                                   // -1: none, or past the caches below
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : -1;
}
int w4_sms() {
  static int cache[64] = {0};
  const int dev = current_device();
  if (dev < 0) return 148;
  if (cache[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cache[dev] = n;
  }
  return cache[dev];
}

template <typename TX, int NT, int GROUP, int RING>
cudaError_t launch_rows(W4Params p, size_t x_bytes, cudaStream_t st) {
  using L = RowSmem<NT, GROUP, RING>;
  static bool done[64] = {false};
  const cudaError_t e = allow_max_smem((const void*)w4_rows_kernel<TX, NT, GROUP, RING>, done);
  if (e != cudaSuccess) return e;
  const int tiles = (p.N + 31) / 32, sms = w4_sms();
  // the stream width with the shortest longest stream: rounds of tiles x (units of a warp and half a unit's
  // time to join the sums)
  int64_t best = INT64_MAX;
  for (int w = 2; w <= L::kWarps; w *= 2) {
    const int64_t streams = (int64_t)sms * (L::kWarps / w);
    const int64_t cost = ((tiles + streams - 1) / streams) * (2 * ((p.U + w - 1) / w) + 1);
    if (cost <= best) {
      best = cost;
      p.stream_warps = w;
    }
  }
  return launch_k(w4_rows_kernel<TX, NT, GROUP, RING>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(L::kWarps * 32),
                  L::kFixed + x_bytes, st, true, p);
}

// The driver's tensor-map encoder, looked up once.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}
// x as a 2-d tensor read in boxes of 128 bytes x `rows`; false where TMA cannot read it (base or rows
// off 16 bytes).
bool x_tensor_map(CUtensorMap* map, const W4Params& p, size_t xb, CUtensorMapDataType type, int rows) {
  const int64_t pitch = p.M > 1 ? p.ldx * (int64_t)xb : (p.K * (int64_t)xb + 15) / 16 * 16;
  if ((reinterpret_cast<uintptr_t>(p.x) & 15) || pitch % 16 != 0 || encode_tiled() == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)p.K, (cuuint64_t)p.M}, strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / xb), (cuuint32_t)rows}, one[2] = {1, 1};
  return encode_tiled()(map, type, 2, const_cast<void*>(p.x), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename TX, int MT, int GROUP>
cudaError_t launch_tile(W4Params p, cudaStream_t st) {
  using L = Tile<(int)sizeof(TX), MT, GROUP>;
  static bool done[64] = {false};
  cudaError_t e = allow_max_smem((const void*)w4_tile_kernel<TX, MT, GROUP>, done);
  if (e != cudaSuccess) return e;
  const int nt = (p.N + 127) / 128, mt = (int)((p.M + MT - 1) / MT), units = p.U, sms = w4_sms();
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // As many blocks a tile as the GPU holds at once, four units of inputs each or more. Clusters are placed
  // within groups of SMs, so fewer blocks fit in large ones (16 clusters of 8 took two rounds, 17 x 2048 x 4096:
  // 9.7 us; 16 of 4: 6.3 us): the runtime tells how many do.
  auto fits = [&](int n) {
    static int cache[64][4] = {};                        // [device][log2 n]: clusters of n at once, plus one
    const int dev = current_device(), i = n == 2 ? 1 : n == 4 ? 2 : 3;
    if (dev < 0) return false;
    if (cache[dev][i] == 0) {
      int most = 0;
      attr[0].val.clusterDim = {(unsigned)n, 1, 1};
      cfg.gridDim = dim3((unsigned)n);
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&most, w4_tile_kernel<TX, MT, GROUP>, &cfg) != cudaSuccess) most = 0;
      cache[dev][i] = most + 1;
    }
    return (int64_t)nt * mt <= cache[dev][i] - 1;
  };
  int s = 1;
  while (s < 8 && (int64_t)nt * mt * s * 2 <= sms && units >= 4 * s && fits(2 * s)) s *= 2;
  p.splits = s;
  p.wait_ns = g_w4_wait_ns;
  p.hold = g_w4_hold;
  CUtensorMap map{};
  const CUtensorMapDataType type = sizeof(TX) == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : std::is_same<TX, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  p.x_tma = x_tensor_map(&map, p, sizeof(TX), type, MT);
  cfg.gridDim = dim3((unsigned)(nt * s), (unsigned)mt);
  attr[0].val.clusterDim = {(unsigned)s, 1, 1};
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, w4_tile_kernel<TX, MT, GROUP>, p, map);
}

template <typename TX, int GROUP>
cudaError_t launch_group(const W4Params& p, cudaStream_t st) {
  constexpr bool I8 = std::is_same<TX, int8_t>::value;
  // Rows of up to 16 are staged by every block, in shared memory as the products take them; the limit is the memory's
  // (16 rows of 4096 f16 inputs, groups of 64, take the tile kernel). At 16 | 17 rows, where the kernels change:
  // 28672 x 8192 f16 49.1 | 49.2 us, int8 35.8 | 49.7 us; 16384 x 1024 f16 5.9 | 6.1 us, groups of 32 6.1 | 8.7 us.
  const size_t x = (size_t)p.U * 128 * (I8 ? 1 : 2) * (size_t)p.M, limit = 232448;
  // Where four blocks can share a tile's inputs, staging 12 rows or more of 16 bits (e4m3 is staged as fp16) costs
  // more than the tile kernel (4096 x 4096 f16: 11 rows 6.7 us, 12 rows 7.2 | 6.8 us, 16 rows 8.1 | 6.9 us;
  // e4m3: 12 rows 7.4 | 6.8 us; 1024 x 4096 f16: 16 rows 8.0 | 5.0 us). Not with smaller groups (4096 x 4096, groups of 32: 14 rows 8.1 | 9.1 us), int8
  // (12 rows 6.0 | 6.5 us) or few inputs (777 x 1002: 5.0 | 5.2 us).
  const bool split = GROUP == 128 && !I8 && p.M > 11 && p.U >= 16 && (int64_t)((p.N + 127) / 128) * 4 <= w4_sms();
  if (p.M <= 8 && RowSmem<1, GROUP, 3>::kFixed + x <= limit) return launch_rows<TX, 1, GROUP, 3>(p, x, st);
  if (p.M <= 8 && RowSmem<1, GROUP, 2>::kFixed + x <= limit) return launch_rows<TX, 1, GROUP, 2>(p, x, st);
  if (p.M > 8 && p.M <= 16 && !split && RowSmem<2, GROUP, 2>::kFixed + x <= limit)
    return launch_rows<TX, 2, GROUP, 2>(p, x, st);
  // the smallest tile that holds all rows: 4096 x 4096 f16 at 32 | 33 rows 7.0 | 8.3 us, at 64 | 65 rows 8.6 | 12.1 us
  if (p.M <= 32) return launch_tile<TX, 32, GROUP>(p, st);
  if (p.M <= 64) return launch_tile<TX, 64, GROUP>(p, st);
  return launch_tile<TX, 128, GROUP>(p, st);
}
template <typename TX>
cudaError_t launch_w4(const W4Params& p, cudaStream_t st) {
  if (p.group == 32) return launch_group<TX, 32>(p, st);
  if (p.group == 64) return launch_group<TX, 64>(p, st);
  return launch_group<TX, 128>(p, st);
}

int bad(const char* what) {
  char msg[200];
  snprintf(msg, sizeof(msg), "glad_w4_linear_forward: %s", what);
  return set_last_error(GLAD_ERR_INVALID_ARG, msg);
}
bool on(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
bool shape_ok(int K, int N, int group) {
  return K >= 2 && K % 2 == 0 && K <= (1 << 20) && N >= 1 && N <= (1 << 20) &&
         (group == 32 || group == 64 || group == 128);
}
int units(int K) { return (K + 127) / 128; }

}  // namespace

// The status word of the current device, for the kernels of other files that report through it.
cudaError_t w4_status_word(uint32_t** word) {
  static void* cache[64] = {};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (cache[dev] == nullptr) {
    const cudaError_t e = cudaGetSymbolAddress(&cache[dev], g_w4_status);
    if (e != cudaSuccess) return e;
  }
  *word = static_cast<uint32_t*>(cache[dev]);
  return cudaSuccess;
}
}  // namespace glad

using namespace glad;

extern "C" {

size_t glad_w4_tiles_bytes(int in_features, int out_features, int group) {
  if (!shape_ok(in_features, out_features, group)) return 0;
  return (size_t)((out_features + 127) / 128) * (size_t)units(in_features) * 8192;
}

size_t glad_w4_scales_bytes(int in_features, int out_features, int group) {
  if (!shape_ok(in_features, out_features, group)) return 0;
  return (size_t)((out_features + 127) / 128) * (size_t)units(in_features) * 8 * (size_t)(128 / group) * 32;
}

int glad_w4_linear_status(uint32_t* status, void* stream) {
  if (!status) return set_last_error(GLAD_ERR_INVALID_ARG, "glad_w4_linear_status: status is NULL");
  const cudaStream_t st = (cudaStream_t)stream;
  static std::atomic<unsigned int> calls{0};
  const int slot = (int)(calls.fetch_add(1) % kStatusCalls);
  unsigned int word = 0;
  w4_take_status_kernel<<<1, 1, 0, st>>>(slot);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess)
    e = cudaMemcpyFromSymbolAsync(&word, g_w4_taken, sizeof(word), slot * sizeof(word), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) {
    char msg[200];
    snprintf(msg, sizeof(msg), "glad_w4_linear_status: %s", cudaGetErrorString(e));
    return set_last_error(GLAD_ERR_CUDA, msg);
  }
  *status = word;
  if (word != 0) return set_last_error(GLAD_ERR_DEVICE, "glad_w4_linear_status: a bounded wait inside a kernel ran out");
  return GLAD_OK;
}

int glad_debug_w4_wait(uint32_t hold, uint64_t limit_ns) {
  if (hold > 15 || limit_ns > 2000000000ull)
    return set_last_error(GLAD_ERR_INVALID_ARG, "glad_debug_w4_wait: hold above 15 or limit_ns above 2 s");
  g_w4_hold = hold;
  g_w4_wait_ns = limit_ns ? (uint32_t)limit_ns : 2000000000u;
  return GLAD_OK;
}

int glad_w4_linear_forward(const GladW4Weight* w, const void* x, int x_dtype, int64_t M, int64_t ldx,
                           const float* x_scale, int x_scale_rows, int x_scale_groups, const void* bias, void* y,
                           int y_dtype, void* stream) {
  if (!w || !w->tiles || !w->scales) return bad("the weight's tiles and scales must be set");
  const int K = w->in_features, N = w->out_features;
  if (!shape_ok(K, N, w->group)) return bad("in_features even in [2, 2^20], out_features in [1, 2^20], group 32, 64 or 128");
  if (!on(w->tiles, 16) || !on(w->scales, 16)) return bad("tiles and scales must be 16-byte aligned");
  const bool wide = x_dtype == GLAD_DTYPE_F16 || x_dtype == GLAD_DTYPE_BF16;
  if (!wide && x_dtype != GLAD_DTYPE_I8 && x_dtype != GLAD_DTYPE_E4M3) return bad("x must be f16, bf16, i8 or e4m3");
  if (y_dtype != GLAD_DTYPE_F16 && y_dtype != GLAD_DTYPE_BF16 && y_dtype != GLAD_DTYPE_F32)
    return bad("y must be f16, bf16 or f32");
  if (M < 0 || M > (1 << 20)) return bad("M must be in [0, 2^20]");
  if (M == 0) return GLAD_OK;
  if (!x || !y) return bad("x and y must be set");
  const size_t xb = wide ? 2 : 1, yb = y_dtype == GLAD_DTYPE_F32 ? 4 : 2;
  if (!on(x, xb) || !on(y, yb) || !on(bias, yb) || !on(x_scale, 4)) return bad("a tensor is not element-aligned");
  if (M > 1 && ldx < K) return bad("ldx is below in_features");
  if (wide && x_scale) return bad("x_scale is for 8-bit rows");
  if (!wide && !x_scale) return bad("8-bit rows need x_scale");
  const int G = (K + w->group - 1) / w->group;
  const bool one = x_scale_rows == 0 && x_scale_groups <= 1;
  if (x_scale && !one && !(x_scale_rows == 1 && (x_scale_groups == 1 || x_scale_groups == G)))
    return bad("x_scale is one value, one a row, or one a row and group");
  W4Params p{};
  p.tiles = static_cast<const uint4*>(w->tiles);
  p.scales = static_cast<const __half*>(w->scales);
  p.N = N;
  p.K = K;
  p.U = units(K);
  p.group = w->group;
  p.x = x;
  p.M = M;
  p.ldx = ldx;
  p.xs = x_scale;
  p.xs_rows = x_scale ? x_scale_rows : 0;
  p.xs_groups = x_scale ? x_scale_groups : 0;
  p.x_fast = K % 8 == 0 && on(x, 8 * xb) && (M == 1 || (ldx * (int64_t)xb) % (int64_t)(8 * xb) == 0);
  p.bias = bias;
  p.y = y;
  p.y_dtype = y_dtype;
  p.y_vec = N % 4 == 0 && on(y, 4 * yb);
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (x_dtype == GLAD_DTYPE_F16) e = launch_w4<__half>(p, st);
  else if (x_dtype == GLAD_DTYPE_BF16) e = launch_w4<__nv_bfloat16>(p, st);
  else if (x_dtype == GLAD_DTYPE_I8) e = launch_w4<int8_t>(p, st);
  else e = launch_w4<e4m3_t>(p, st);
  if (e != cudaSuccess) {
    char msg[200];
    snprintf(msg, sizeof(msg), "glad_w4_linear_forward: %s", cudaGetErrorString(e));
    return set_last_error(GLAD_ERR_CUDA, msg);
  }
  return GLAD_OK;
}

}  // extern "C"
