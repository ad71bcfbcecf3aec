// Rows times 4-bit weights with group scales:
//   y[m, n] = sum_g xs[m, g] * s[n, g] * sum_{k in group g} x[m, k] * q[n, k] + b[n]
//
// The weights are streamed once in the order the kernel reads them (include/glad_b200.h:
// GladW4Weight), 512 contiguous bytes a warp load: 16 rows x 64 inputs. A 32-bit word is
// one lane's share of the A operand of a 16x8x16 tensor-core product, so a word becomes
// four half2 registers with one logic operation and one half operation each:
// 0x6400 | u is the half 1024 + u, exact for 4-bit u. Products q * x are exact and the sum of
// a group is fp32; the scale multiplies the group's sum, so no weight is ever rounded.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <type_traits>

#include "glad_common.cuh"

namespace glad {
int set_last_error(int code, const char* msg);

namespace {

struct W4Params {
  const uint4* tiles;
  const __half* scales;
  int N, K, KB, group;      // KB: 64-input blocks, an even number
  const void* x;
  int64_t M, ldx;
  const float* xs;          // scales of 8-bit rows or null
  int xs_rows, xs_groups;   // 0/0: none or one value; 1/1: a row; 1/G: a row and group
  int x_fast;               // rows can be read 8 inputs at a time
  int x_smem;               // few rows: x is staged in shared memory
  int splits;               // many rows: blocks that share a tile's inputs
  const void* bias;
  void* y;
  int y_dtype;
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

// Eight 4-bit weights -> the A registers of one 16x8x16 product. The two's-complement
// nibble with its top bit flipped is q + 8.
template <bool BF16>
__device__ __forceinline__ void unpack_w4(uint32_t w, uint32_t (&a)[4]) {
  if constexpr (BF16) {
    // 0x4300 | u is the bf16 128 + u (seven mantissa bits): each nibble is shifted to bit 0
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = b2_sub(((w >> (4 * i)) & 0x000f000fu) ^ 0x43084308u, 0x43084308u);
  } else {
    a[0] = h2_sub((w & 0x000f000fu) ^ 0x64086408u, 0x64086408u);
    a[1] = h2_fma((w & 0x00f000f0u) ^ 0x64806480u, 0x2c002c00u, 0xd480d480u);   // (1024 + 16 u) / 16 - 72
    w >>= 8;
    a[2] = h2_sub((w & 0x000f000fu) ^ 0x64086408u, 0x64086408u);
    a[3] = h2_fma((w & 0x00f000f0u) ^ 0x64806480u, 0x2c002c00u, 0xd480d480u);
  }
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// ... as the four half2 (bf16x2) the products take; 8-bit inputs are exact in fp16.
template <typename T>
__device__ __forceinline__ uint4 to_halves(uint4 v) {
  if constexpr (sizeof(T) == 2) {
    return v;
  } else if constexpr (std::is_same<T, e4m3_t>::value) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = i < 2 ? v.x : v.y;
      const __half2_raw h =
          __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(i & 1 ? w >> 16 : w & 0xffffu), __NV_E4M3);
      r[i] = (uint32_t)h.x | ((uint32_t)h.y << 16);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  } else {
    // x + 128 in a byte; 0x6400 | u is the half 1024 + u = 1152 + x
    const uint32_t a = v.x ^ 0x80808080u, b = v.y ^ 0x80808080u;
    return make_uint4(h2_sub(__byte_perm(a, 0x64646464u, 0x4140), 0x64806480u),
                      h2_sub(__byte_perm(a, 0x64646464u, 0x4342), 0x64806480u),
                      h2_sub(__byte_perm(b, 0x64646464u, 0x4140), 0x64806480u),
                      h2_sub(__byte_perm(b, 0x64646464u, 0x4342), 0x64806480u));
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

// ---- few rows (up to 8 NT): weight streaming ------------------------------------------------
// One persistent block per SM walks 16-column tiles; its 16 warps split the inputs in units of
// 128 and join their sums in warp order once a tile. Each warp streams its own units (1 KB of
// weights and 128/GROUP * 32 bytes of scales) through a private shared-memory ring of
// cp.async copies kRing - 1 units ahead, across tile borders, so about 64 KB are in flight on
// an SM whatever the warps wait for. x is staged once in shared memory when it fits.
constexpr int kRowWarps = 16, kRing = 5;
constexpr int kRowThreads = kRowWarps * 32;

template <int GROUP>
struct RowRing {
  static constexpr int kScales = 128 / GROUP;           // groups of a unit
  static constexpr int kWarpSlot = 1024 + kScales * 32;
  static constexpr int kBytes = kRing * kRowWarps * kWarpSlot;
};
template <int NT>
struct RowPart {                                         // two buffers of every warp's sums
  static constexpr int kBytes = 2 * kRowWarps * 8 * NT * 17 * 4;
};

template <typename TX, int NT, int GROUP>
__global__ void __launch_bounds__(kRowThreads, 1) w4_rows_kernel(const __grid_constant__ W4Params p) {
  using Ring = RowRing<GROUP>;
  constexpr bool BF16 = std::is_same<TX, __nv_bfloat16>::value;
  constexpr int SG = Ring::kScales, XB = (int)sizeof(TX);
  extern __shared__ __align__(16) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem + Ring::kBytes);
  uint8_t* xs = smem + Ring::kBytes + RowPart<NT>::kBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int T = (p.N + 15) / 16, U = p.KB / 2, M = (int)p.M;
  const int u0 = (int)((int64_t)warp * U / kRowWarps), u1 = (int)((int64_t)(warp + 1) * U / kRowWarps);
  uint8_t* ring = smem + warp * (kRing * Ring::kWarpSlot);

  int pt = blockIdx.x, pu = u0;                          // the next unit to fetch
  auto fetch = [&](int slot) {
    if (pt < T && u0 < u1) {
      uint8_t* dst = ring + slot * Ring::kWarpSlot;
      const uint4* src = p.tiles + ((int64_t)pt * p.KB + 2 * pu) * 32 + lane;
      cp_async16(dst + lane * 16, src);
      cp_async16(dst + 512 + lane * 16, src + 32);
      if (lane < SG * 2) {
        const uint8_t* sc = reinterpret_cast<const uint8_t*>(p.scales) + ((int64_t)pt * U + pu) * (SG * 32);
        cp_async16(dst + 1024 + lane * 16, sc + lane * 16);
      }
      if (++pu == u1) {
        pu = u0;
        pt += gridDim.x;
      }
    }
    cp_async_commit();
  };
  grid_dep_wait();
  grid_dep_launch();
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) fetch(i);

  if (p.x_smem) {
    // [32-input block][row][32 inputs]: a warp's reads of eight rows are contiguous
    const int pieces = p.KB * 8 * M;
    for (int i = threadIdx.x; i < pieces; i += kRowThreads) {
      const int m = i / (p.KB * 8), k8 = i - m * (p.KB * 8);
      const uint4 v = load_raw8<TX>(static_cast<const TX*>(p.x) + m * p.ldx, k8 * 8, p.K, p.x_fast);
      uint8_t* dst = xs + (((k8 >> 2) * M + m) * 4 + (k8 & 3)) * (8 * XB);
      if constexpr (XB == 2) *reinterpret_cast<uint4*>(dst) = v;
      else *reinterpret_cast<uint2*>(dst) = make_uint2(v.x, v.y);
    }
    __syncthreads();
  }
  auto get_x = [&](int m, int k32) -> uint4 {            // inputs 32 k32 + 8 c .. + 7 of row m
    if (m >= M) return make_uint4(0, 0, 0, 0);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (p.x_smem) {
      const uint8_t* src = xs + ((k32 * M + m) * 4 + c) * (8 * XB);
      if constexpr (XB == 2) {
        v = *reinterpret_cast<const uint4*>(src);
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(src);
        v.x = u.x, v.y = u.y;
      }
    } else {
      v = load_raw8<TX>(static_cast<const TX*>(p.x) + m * p.ldx, k32 * 32 + 8 * c, p.K, p.x_fast);
    }
    return to_halves<TX>(v);
  };

  int slot = 0, parity = 0;
  for (int t = blockIdx.x; t < T; t += gridDim.x) {
    float acc[NT][4], g[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = g[j][e] = 0.0f;
    for (int u = u0; u < u1; ++u) {
      cp_async_wait_group<kRing - 2>();
      __syncwarp();
      fetch(slot == 0 ? kRing - 1 : slot - 1);           // the slot that every lane has just left
      const uint8_t* in = ring + slot * Ring::kWarpSlot;
      slot = slot + 1 == kRing ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {                      // 32 inputs at a time
        const uint2 w = *reinterpret_cast<const uint2*>(in + (q >> 1) * 512 + lane * 16 + (q & 1) * 8);
        uint32_t a0[4], a1[4];
        unpack_w4<BF16>(w.x, a0);
        unpack_w4<BF16>(w.y, a1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 x = get_x(8 * j + r, 4 * u + q);
          mma_16816<BF16>(g[j], a0, x.x, x.y);
          mma_16816<BF16>(g[j], a1, x.z, x.w);
        }
        if ((q + 1) % (GROUP / 32) == 0) {
          const int gi = q / (GROUP / 32);
          const float2 s = __half22float2(*reinterpret_cast<const __half2*>(in + 1024 + gi * 32 + r * 4));
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float x0 = 1.0f, x1 = 1.0f;
            if (p.xs_groups > 1) {
              const int m = 8 * j + 2 * c, xg = u * SG + gi;
              x0 = (m < M && xg < p.xs_groups) ? p.xs[m * p.xs_groups + xg] : 0.0f;
              x1 = (m + 1 < M && xg < p.xs_groups) ? p.xs[(m + 1) * p.xs_groups + xg] : 0.0f;
            }
            acc[j][0] = fmaf(__fmul_rn(s.x, x0), g[j][0], acc[j][0]);
            acc[j][1] = fmaf(__fmul_rn(s.x, x1), g[j][1], acc[j][1]);
            acc[j][2] = fmaf(__fmul_rn(s.y, x0), g[j][2], acc[j][2]);
            acc[j][3] = fmaf(__fmul_rn(s.y, x1), g[j][3], acc[j][3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) g[j][e] = 0.0f;
          }
        }
      }
    }
    // the buffer written now was last read two tiles ago, before the previous tile's barrier
    float* mine = part + (parity * kRowWarps + warp) * (8 * NT * 17);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      mine[(8 * j + 2 * c) * 17 + r] = acc[j][0];
      mine[(8 * j + 2 * c + 1) * 17 + r] = acc[j][1];
      mine[(8 * j + 2 * c) * 17 + r + 8] = acc[j][2];
      mine[(8 * j + 2 * c + 1) * 17 + r + 8] = acc[j][3];
    }
    __syncthreads();
    const int row = threadIdx.x >> 4, col = threadIdx.x & 15, n = 16 * t + col;
    if (row < 8 * NT && row < M && n < p.N) {
      const float* all = part + parity * kRowWarps * (8 * NT * 17) + row * 17 + col;
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < kRowWarps; ++k) v += all[k * (8 * NT * 17)];
      if (p.xs != nullptr && p.xs_groups <= 1) v *= p.xs[p.xs_rows ? row : 0];
      store_y(p, row, n, v);
    }
    parity ^= 1;
  }
}

// ---- many rows: tcgen05 -----------------------------------------------------------------------
// A block computes 128 output columns x MT rows; D[n, m] lives in tensor memory, n its lanes. Per
// stage of 128 inputs, 16 warps turn the packed weights into the fp16 (bf16) A operand in shared
// memory while one thread issues the products of the stage before. Every group of inputs has an
// accumulator of its own (ND in rotation): the warps read it back, scale it by s[n, g] (a lane's
// own row: one value a thread) and add it to fp32 sums in registers, so the weights need no
// rounding; that costs one multiply-add per output and group, as much issue time as the tensor
// core needs for 64 inputs at fp16 rate. The inputs of x are copied NS - 1 stages ahead, the
// packed weights PD stages ahead by bulk copies. Blocks of a cluster split the inputs when there are
// fewer tiles than SMs and join their sums through distributed shared memory in rank order.
constexpr int kTileWarps = 16;
constexpr int kTileThreads = (kTileWarps + 2) * 32;      // + the MMA warp + the weight loader

__device__ unsigned int g_w4_status;

template <int MT, int GROUP>
struct Tile {
  static constexpr int NS = MT == 256 ? 2 : 3;
  static constexpr int PD = MT == 256 ? 2 : MT == 128 ? 3 : 6;
  static constexpr int ND = MT == 256 ? 2 : 4;
  static constexpr int SG = 128 / GROUP;
  static constexpr int kA = 128 * 256, kB = MT * 256, kStage = kA + kB;
  static constexpr int kSlot = 8192 + 8 * SG * 32;       // packed weights and scales of a stage
  static constexpr int kXs = 3 * SG * MT * 4;            // x scales of three stages
  static constexpr int kRed = MT * 128 * 4;
  static constexpr int kSmem = NS * kStage + PD * kSlot + kXs + 256 + 1024;
  static constexpr int kCols = ND * MT;
  static_assert(kRed <= NS * kStage, "the sums are joined in the stage buffers");
  static_assert(kSmem <= 232448, "shared memory of one block");
};

__device__ __noinline__ bool w4_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!*abort) {
    if (mbar_try_wait(bar, parity)) return true;
    if (global_timer_ns() - t0 > 2000000000ull) {
      *abort = 1;
      atomicOr(&g_w4_status, kDevErrMmaTimeout);
    }
  }
  return false;
}

// K-major operand with 128-byte swizzle: rows of 128 bytes (64 halves), 8-row groups 1024 bytes apart,
// the 16-byte piece i of row r at i ^ (r & 7).
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <typename TX, int MT, int GROUP>
__global__ void __launch_bounds__(kTileThreads, 1) w4_tile_kernel(const __grid_constant__ W4Params p) {
  using L = Tile<MT, GROUP>;
  constexpr bool BF16 = std::is_same<TX, __nv_bfloat16>::value;
  constexpr int SG = L::SG, NC = MT / 4, XP = MT / 32;   // columns, 16-byte x pieces of a thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = smem + L::NS * L::kStage;
  float* xsc = reinterpret_cast<float*>(slots + L::PD * L::kSlot);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(xsc) + L::kXs);   // [NS]
  uint64_t* wfull = full + L::NS;                                                           // [PD]
  uint64_t* wempty = wfull + L::PD;                                                         // [PD]
  uint64_t* dfull = wempty + L::PD;                                                         // [ND]
  uint64_t* dempty = dfull + L::ND;                                                         // [ND]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dempty + L::ND);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((L::NS + 2 * L::PD + 2 * L::ND) * 8 + 8 <= 256, "barrier area");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.splits, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int nt = blockIdx.x / S;
  const int64_t m0 = (int64_t)blockIdx.y * MT;
  const int ST = p.KB / 2, st0 = (int)((int64_t)rank * ST / S), st1 = (int)((int64_t)(rank + 1) * ST / S);
  const int count = st1 - st0;
  const int live16 = min(8, (p.N + 15) / 16 - nt * 8);   // 16-column tiles that exist

  if (warp == kTileWarps) tmem_alloc(tmem_slot, L::kCols);
  if (tid == 0) {
    for (int i = 0; i < L::NS; ++i) mbar_init(&full[i], kTileWarps);
    for (int i = 0; i < L::PD; ++i) {
      mbar_init(&wfull[i], 1);
      mbar_init(&wempty[i], kTileWarps);
    }
    for (int i = 0; i < L::ND; ++i) {
      mbar_init(&dfull[i], 1);
      mbar_init(&dempty[i], kTileWarps);
    }
    fence_mbar_init();
    *abort = 0;
  }
  if (live16 < 8) {                                      // columns past the weight: zeros that nothing overwrites
    for (int i = tid; i < L::PD * L::kSlot / 16; i += kTileThreads)
      reinterpret_cast<uint4*>(slots)[i] = make_uint4(0, 0, 0, 0);
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();
  grid_dep_launch();

  if (warp == kTileWarps + 1) {
    // ---- packed weights and scales, PD stages ahead
    if (lane == 0) {
      const uint8_t* wsrc = reinterpret_cast<const uint8_t*>(p.tiles);
      const uint8_t* ssrc = reinterpret_cast<const uint8_t*>(p.scales);
      int issued = 0;
      for (int i = 0; i < count; ++i, ++issued) {
        const int slot = i % L::PD;
        if (i >= L::PD && !w4_wait(&wempty[slot], (i / L::PD - 1) & 1, abort)) break;
        uint8_t* dst = slots + slot * L::kSlot;
        mbar_arrive_expect_tx(&wfull[slot], (uint32_t)live16 * (1024 + SG * 32));
        for (int b = 0; b < live16; ++b) {
          const int64_t t = (int64_t)nt * 8 + b, st = st0 + i;
          bulk_copy_g2s(dst + b * 1024, wsrc + (t * p.KB + 2 * st) * 512, 1024, &wfull[slot]);
          bulk_copy_g2s(dst + 8192 + b * (SG * 32), ssrc + (t * ST + st) * (SG * 32), SG * 32, &wfull[slot]);
        }
      }
      // copies that were issued land before the block leaves
      for (int i = max(0, issued - L::PD); i < issued && *abort; ++i)
        mbar_wait_bounded(&wfull[i % L::PD], (i / L::PD) & 1);
    }
  } else if (warp == kTileWarps) {
    // ---- products
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_f16(128, MT) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
      const uint32_t base = smem_u32(smem);
      int gi = 0;
      for (int i = 0; i < count; ++i) {
        if (!w4_wait(&full[i % L::NS], (i / L::NS) & 1, abort)) break;
        tc_fence_after();
        const uint32_t a = base + (i % L::NS) * L::kStage, b = a + L::kA;
        bool ok = true;
#pragma unroll
        for (int j = 0; j < SG; ++j, ++gi) {
          const int d = gi % L::ND;
          if (gi >= L::ND && !(ok = w4_wait(&dempty[d], (gi / L::ND - 1) & 1, abort))) break;
          tc_fence_after();
#pragma unroll
          for (int q = 0; q < GROUP / 16; ++q) {
            const int k16 = j * (GROUP / 16) + q;
            mma_f16(tmem + d * MT, desc_sw128(a + (k16 >> 2) * 16384 + (k16 & 3) * 32),
                    desc_sw128(b + (k16 >> 2) * (MT * 128) + (k16 & 3) * 32), idesc, q > 0 ? 1u : 0u);
          }
          mma_commit(&dfull[d]);
        }
        if (!ok) break;
      }
      // after a failure: products that were issued end before their operands go
      for (int k = max(0, gi - L::ND); k < gi && *abort; ++k) mbar_wait_bounded(&dfull[k % L::ND], (k / L::ND) & 1);
    }
  } else {
    // ---- operands, sums
    const int r = lane >> 2, c = lane & 3, q4 = warp & 3, col0 = (warp >> 2) * NC;
    const uint32_t sbase = smem_u32(smem);
    const uint32_t a_row = (uint32_t)((warp >> 1) * 16 + r) * 128 + (warp & 1) * 16384;
    const int my_n16 = q4 * 2 + (lane >> 4), my_s = (lane & 7) * 2 + ((lane >> 3) & 1);
    float acc[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = 0.0f;
    float sc[SG], sc_next[SG];
    uint2 raw[sizeof(TX) == 1 ? XP : 1];
    float xs_reg[2] = {0.0f, 0.0f};
    constexpr int XD = L::NS - 1;

    auto x_dst = [&](int i, int piece) -> uint32_t {     // stage i, this thread's piece
      const int id = piece * 512 + tid, row = id >> 4, k8 = id & 15;
      return sbase + (i % L::NS) * L::kStage + L::kA + (k8 >> 3) * (MT * 128) + row * 128 + (((k8 & 7) ^ (row & 7)) << 4);
    };
    auto x_issue = [&](int i) {                          // 16-bit rows: asynchronous copies of stage i
      if constexpr (sizeof(TX) == 2) {
        if (p.x_fast && i < count) {
#pragma unroll
          for (int e = 0; e < XP; ++e) {
            const int id = e * 512 + tid;
            const int64_t m = m0 + (id >> 4);
            const int k = (st0 + i) * 128 + (id & 15) * 8;
            const bool live = m < p.M && k < p.K;
            cp_async16_zfill(x_dst(i, e), static_cast<const TX*>(p.x) + (live ? m * p.ldx + k : 0), live);
          }
        }
        cp_async_commit();
      }
    };
    auto x_load = [&](int i) {                           // 8-bit rows: stage i into registers
      if constexpr (sizeof(TX) == 1) {
        if (i < count) {
#pragma unroll
          for (int e = 0; e < XP; ++e) {
            const int id = e * 512 + tid;
            const int64_t m = m0 + (id >> 4);
            const int k = (st0 + i) * 128 + (id & 15) * 8;
            raw[e] = make_uint2(0, 0);
            if (m < p.M) {
              const uint4 v = load_raw8<TX>(static_cast<const TX*>(p.x) + m * p.ldx, k, p.K, p.x_fast);
              raw[e] = make_uint2(v.x, v.y);
            }
          }
          if (p.xs_groups > 1) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int id = e * 512 + tid, g = id / MT;
              const int64_t m = m0 + id % MT;
              const int xg = (st0 + i) * SG + g;
              xs_reg[e] = (g < SG && m < p.M && xg < p.xs_groups) ? p.xs[m * p.xs_groups + xg] : 0.0f;
            }
          }
        }
      }
    };
    auto x_finish = [&](int i) {                         // stage i of x is in shared memory
      if constexpr (sizeof(TX) == 1) {
#pragma unroll
        for (int e = 0; e < XP; ++e) {
          const uint4 h = to_halves<TX>(make_uint4(raw[e].x, raw[e].y, 0, 0));
          st_shared_v4(x_dst(i, e), h.x, h.y, h.z, h.w);
        }
        if (p.xs_groups > 1) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (e * 512 + tid < SG * MT) xsc[(i % 3) * (SG * MT) + e * 512 + tid] = xs_reg[e];
        }
      } else if (p.x_fast) {
        cp_async_wait_group<XD - 1>();
      } else {
#pragma unroll 1
        for (int e = 0; e < XP; ++e) {
          const int id = e * 512 + tid;
          const int64_t m = m0 + (id >> 4);
          uint4 v = make_uint4(0, 0, 0, 0);
          if (m < p.M)
            v = load_raw8<TX>(static_cast<const TX*>(p.x) + m * p.ldx, (st0 + i) * 128 + (id & 15) * 8, p.K, false);
          st_shared_v4(x_dst(i, e), v.x, v.y, v.z, v.w);
        }
      }
    };
    bool ok = true;
    auto sums = [&](int i) {                             // add the groups of stage i
#pragma unroll
      for (int j = 0; j < SG; ++j) {
        const int gi = i * SG + j, d = gi % L::ND;
        if (!ok || !(ok = w4_wait(&dfull[d], (gi / L::ND) & 1, abort))) return;
        tc_fence_after();
        constexpr int CH = NC < 16 ? NC : 16;
#pragma unroll
        for (int cb = 0; cb < NC; cb += CH) {
          uint32_t v[CH];
          const uint32_t at = tmem + ((uint32_t)(32 * q4) << 16) + d * MT + col0 + cb;
          if constexpr (CH == 16) tmem_ld16(at, v);
          else tmem_ld8(at, v);
          tmem_ld_wait();
          if (sizeof(TX) == 1 && p.xs_groups > 1) {
            const float4* xv = reinterpret_cast<const float4*>(xsc + (i % 3) * (SG * MT) + j * MT + col0 + cb);
#pragma unroll
            for (int e = 0; e < CH; e += 4) {
              const float4 f = xv[e / 4];
              acc[cb + e] = fmaf(__fmul_rn(sc[j], f.x), __uint_as_float(v[e]), acc[cb + e]);
              acc[cb + e + 1] = fmaf(__fmul_rn(sc[j], f.y), __uint_as_float(v[e + 1]), acc[cb + e + 1]);
              acc[cb + e + 2] = fmaf(__fmul_rn(sc[j], f.z), __uint_as_float(v[e + 2]), acc[cb + e + 2]);
              acc[cb + e + 3] = fmaf(__fmul_rn(sc[j], f.w), __uint_as_float(v[e + 3]), acc[cb + e + 3]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) acc[cb + e] = fmaf(sc[j], __uint_as_float(v[e]), acc[cb + e]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dempty[d]);
      }
    };

#pragma unroll
    for (int i = 0; i < XD; ++i) x_issue(i);
    x_load(0);
    for (int i = 0; i < count; ++i) {
      const int slot = i % L::PD;
      // after a failure the loop runs on without waiting, so that every warp meets the same barriers
      if (ok) ok = w4_wait(&wfull[slot], (i / L::PD) & 1, abort);
      const uint8_t* in = slots + slot * L::kSlot;
      const uint4 w4 = *reinterpret_cast<const uint4*>(in + warp * 512 + lane * 16);
#pragma unroll
      for (int j = 0; j < SG; ++j)
        sc_next[j] = __half2float(*reinterpret_cast<const __half*>(in + 8192 + my_n16 * (SG * 32) + j * 32 + my_s * 2));
      __syncwarp();
      if (lane == 0) mbar_arrive(&wempty[slot]);
      // odd rows store their two pieces in the other order: eight lanes then fill all banks
      const uint32_t a = sbase + (i % L::NS) * L::kStage + a_row;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int half = h ^ (r & 1);
        uint32_t b0[4], b1[4];
        unpack_w4<BF16>(half ? w4.z : w4.x, b0);
        unpack_w4<BF16>(half ? w4.w : w4.y, b1);
        const uint32_t at = a + (uint32_t)(((half * 4 + c) ^ r) << 4);
        st_shared_v4(at, b0[0], b0[2], b1[0], b1[2]);
        st_shared_v4(at + 1024, b0[1], b0[3], b1[1], b1[3]);
      }
      x_finish(i);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[i % L::NS]);
      if (sizeof(TX) == 1 && p.xs_groups > 1) named_bar_sync(1, kTileWarps * 32);
      if (i > 0) sums(i - 1);
#pragma unroll
      for (int j = 0; j < SG; ++j) sc[j] = sc_next[j];
      x_issue(i + XD);                                   // the products of stage i - 1 are done
      x_load(i + 1);
    }
    if (count > 0 && ok) sums(count - 1);
    cp_async_wait_all();
    // the stage buffers are free: every product is done
    float* red = reinterpret_cast<float*>(smem) + 32 * q4 + lane;
    named_bar_sync(1, kTileWarps * 32);
#pragma unroll
    for (int i = 0; i < NC; ++i) red[(col0 + i) * 128] = acc[i];
  }
  __syncthreads();
  if (S > 1) cluster_sync_all();
  if (warp < kTileWarps && !*abort) {
    const int rows = MT / S;
    const uint32_t red = smem_u32(smem) + lane * 16;
    const int n = nt * 128 + 4 * lane;
    for (int i = warp; i < rows; i += kTileWarps) {
      const int row = rank * rows + i;
      const int64_t m = m0 + row;
      if (m >= p.M || n >= p.N) continue;
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int k = 0; k < S; ++k) {
        const float4 f = ld_cluster_f4(S > 1 ? mapa_shared(red + row * 512, k) : red + row * 512);
        v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
      }
      if (p.xs != nullptr && p.xs_groups <= 1) {
        const float s = p.xs[p.xs_rows ? m : 0];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= s;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) store_y(p, m, n + e, v[e]);
    }
  }
  if (S > 1) cluster_sync_all();
  tc_fence_before();
  __syncthreads();
  if (warp == kTileWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }
}

// ---- launch -------------------------------------------------------------------------------------
int w4_sms() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cache[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cache[dev] = n;
  }
  return cache[dev];
}

template <typename TX, int NT, int GROUP>
cudaError_t launch_rows(W4Params p, cudaStream_t st) {
  static bool done[64] = {false};
  cudaError_t e = allow_max_smem((const void*)w4_rows_kernel<TX, NT, GROUP>, done);
  if (e != cudaSuccess) return e;
  const size_t fixed = RowRing<GROUP>::kBytes + RowPart<NT>::kBytes, limit = 232448;
  const size_t x = (size_t)p.KB * 64 * sizeof(TX) * (size_t)p.M;
  p.x_smem = fixed + x <= limit;
  const int tiles = (p.N + 15) / 16, sms = w4_sms();
  return launch_k(w4_rows_kernel<TX, NT, GROUP>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(kRowThreads),
                  fixed + (p.x_smem ? x : 0), st, true, p);
}

template <typename TX, int MT, int GROUP>
cudaError_t launch_tile(W4Params p, cudaStream_t st) {
  static bool done[64] = {false};
  cudaError_t e = allow_max_smem((const void*)w4_tile_kernel<TX, MT, GROUP>, done);
  if (e != cudaSuccess) return e;
  const int nt = (p.N + 127) / 128, mt = (int)((p.M + MT - 1) / MT), stages = p.KB / 2, sms = w4_sms();
  int s = 1;
  while (s < 8 && (int64_t)nt * mt * s * 2 <= sms && stages >= 8 * s) s *= 2;
  p.splits = s;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(nt * s), (unsigned)mt);
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = Tile<MT, GROUP>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)s, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, w4_tile_kernel<TX, MT, GROUP>, p);
}

template <typename TX, int GROUP>
cudaError_t launch_group(const W4Params& p, cudaStream_t st) {
  if (p.M <= 8) return launch_rows<TX, 1, GROUP>(p, st);
  if (p.M <= 16) return launch_rows<TX, 2, GROUP>(p, st);
  if (p.M <= 32) return launch_tile<TX, 32, GROUP>(p, st);
  if (p.M <= 64) return launch_tile<TX, 64, GROUP>(p, st);
  if (p.M <= 128) return launch_tile<TX, 128, GROUP>(p, st);
  return launch_tile<TX, 256, GROUP>(p, st);
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
int64_t blocks64(int K) { return (int64_t)((K + 127) / 128) * 2; }

}  // namespace
}  // namespace glad

using namespace glad;

extern "C" {

size_t glad_w4_tiles_bytes(int in_features, int out_features, int group) {
  if (!shape_ok(in_features, out_features, group)) return 0;
  return (size_t)((out_features + 15) / 16) * (size_t)blocks64(in_features) * 512;
}

size_t glad_w4_scales_bytes(int in_features, int out_features, int group) {
  if (!shape_ok(in_features, out_features, group)) return 0;
  return (size_t)((out_features + 15) / 16) * (size_t)(blocks64(in_features) * 64 / group) * 32;
}

int glad_w4_linear_status(uint32_t* status, void* stream) {
  if (!status) return set_last_error(GLAD_ERR_INVALID_ARG, "glad_w4_linear_status: status is NULL");
  const cudaStream_t st = (cudaStream_t)stream;
  const unsigned int zero = 0;
  unsigned int word = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&word, g_w4_status, sizeof(word), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && word != 0) {
    e = cudaMemcpyToSymbolAsync(g_w4_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  if (e != cudaSuccess) {
    char msg[200];
    snprintf(msg, sizeof(msg), "glad_w4_linear_status: %s", cudaGetErrorString(e));
    return set_last_error(GLAD_ERR_CUDA, msg);
  }
  *status = word;
  if (word != 0) return set_last_error(GLAD_ERR_DEVICE, "glad_w4_linear_status: a bounded wait inside a kernel ran out");
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
  p.KB = (int)blocks64(K);
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
