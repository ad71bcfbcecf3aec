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

constexpr int kW4Warps = 8;

struct W4Params {
  const uint4* tiles;
  const __half* scales;
  int N, K, KB, group;      // KB: 64-input blocks, padded to whole groups
  const void* x;
  int64_t M, ldx;
  const float* xs;          // scales of 8-bit rows or null
  int xs_rows, xs_groups;   // 0/0: none or one value; 1/1: a row; 1/G: a row and group
  int x_fast;               // rows can be read 8 inputs at a time
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

// Inputs [k, k + 8) of one row as four half2 (bf16x2) registers; zero at and past K. 8-bit
// inputs are exact in fp16.
template <typename T>
__device__ __forceinline__ void load_x8(const T* row, int k, int K, bool fast, uint32_t (&r)[4]) {
  if (k >= K) {
    r[0] = r[1] = r[2] = r[3] = 0;
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (fast) {
      const uint4 v = *reinterpret_cast<const uint4*>(row + k);
      r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
    } else {
      const uint16_t* s = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = k + 2 * i < K ? s[k + 2 * i] : 0u;
        const uint32_t hi = k + 2 * i + 1 < K ? s[k + 2 * i + 1] : 0u;
        r[i] = lo | (hi << 16);
      }
    }
  } else {
    uint32_t w[2];
    if (fast) {
      const uint2 v = *reinterpret_cast<const uint2*>(row + k);
      w[0] = v.x, w[1] = v.y;
    } else {
      const uint8_t* s = reinterpret_cast<const uint8_t*>(row);
      w[0] = w[1] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) w[i >> 2] |= (uint32_t)s[k + i] << (8 * (i & 3));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (sizeof(T) == 1 && !std::is_same<T, e4m3_t>::value) {
        const uint32_t u = w[i] ^ 0x80808080u;     // x + 128; 0x6400 | u is the half 1152 + x
        r[2 * i] = h2_sub(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u);
        r[2 * i + 1] = h2_sub(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u);
      } else {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] & 0xffffu), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> 16), __NV_E4M3);
        r[2 * i] = (uint32_t)a.x | ((uint32_t)a.y << 16);
        r[2 * i + 1] = (uint32_t)b.x | ((uint32_t)b.y << 16);
      }
    }
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

// One block: 16 output columns x 8 NT rows; its warps take the groups of inputs in turn and
// their sums are joined in warp order.
template <typename TX, int NT>
__global__ void __launch_bounds__(kW4Warps * 32) w4_rows_kernel(const __grid_constant__ W4Params p) {
  constexpr bool BF16 = std::is_same<TX, __nv_bfloat16>::value;
  __shared__ float part[kW4Warps][8 * NT][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int64_t m0 = (int64_t)blockIdx.y * (8 * NT);
  const int t = blockIdx.x;
  const uint4* tiles = p.tiles + (int64_t)t * p.KB * 32 + lane;
  const int groups = p.KB * 64 / p.group;
  const __half* scales = p.scales + (int64_t)t * groups * 16 + r;
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
  grid_dep_wait();
  grid_dep_launch();

  float g[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) g[j][e] = 0.0f;
  auto close_group = [&](int gi) {
    const float s0 = __half2float(scales[gi * 16]), s1 = __half2float(scales[gi * 16 + 8]);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float x0 = 1.0f, x1 = 1.0f;
      if (p.xs_groups > 1) {
        const int64_t m = m0 + 8 * j + 2 * c;
        x0 = (m < p.M && gi < p.xs_groups) ? p.xs[m * p.xs_groups + gi] : 0.0f;
        x1 = (m + 1 < p.M && gi < p.xs_groups) ? p.xs[(m + 1) * p.xs_groups + gi] : 0.0f;
      }
      acc[j][0] = fmaf(__fmul_rn(s0, x0), g[j][0], acc[j][0]);
      acc[j][1] = fmaf(__fmul_rn(s0, x1), g[j][1], acc[j][1]);
      acc[j][2] = fmaf(__fmul_rn(s1, x0), g[j][2], acc[j][2]);
      acc[j][3] = fmaf(__fmul_rn(s1, x1), g[j][3], acc[j][3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) g[j][e] = 0.0f;
    }
  };
  const int per = p.group == 128 ? 2 : 1;      // blocks of 64 that one warp must keep together
#pragma unroll 2
  for (int u = warp; u < p.KB / per; u += kW4Warps) {
    for (int b = 0; b < per; ++b) {
      const int kb = u * per + b;
      const uint4 w4 = __ldg(tiles + (int64_t)kb * 32);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t a0[4], a1[4];
        unpack_w4<BF16>(w[2 * half], a0);
        unpack_w4<BF16>(w[2 * half + 1], a1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int64_t m = m0 + 8 * j + r;
          uint32_t x[4] = {0, 0, 0, 0};
          if (m < p.M)
            load_x8<TX>(static_cast<const TX*>(p.x) + m * p.ldx, kb * 64 + half * 32 + 8 * c, p.K, p.x_fast, x);
          mma_16816<BF16>(g[j], a0, x[0], x[1]);
          mma_16816<BF16>(g[j], a1, x[2], x[3]);
        }
        if (p.group == 32) close_group(2 * kb + half);
      }
    }
    if (p.group != 32) close_group(u);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    part[warp][8 * j + 2 * c][r] = acc[j][0];
    part[warp][8 * j + 2 * c + 1][r] = acc[j][1];
    part[warp][8 * j + 2 * c][r + 8] = acc[j][2];
    part[warp][8 * j + 2 * c + 1][r + 8] = acc[j][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NT * 16; i += kW4Warps * 32) {
    const int row = i >> 4, col = i & 15, n = 16 * t + col;
    const int64_t m = m0 + row;
    if (m >= p.M || n >= p.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < kW4Warps; ++k) v += part[k][row][col];
    if (p.xs != nullptr && p.xs_groups <= 1) v *= p.xs[p.xs_rows ? m : 0];
    store_y(p, m, n, v);
  }
}

template <typename TX, int NT>
cudaError_t launch_rows(const W4Params& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.N + 15) / 16), (unsigned)((p.M + 8 * NT - 1) / (8 * NT)));
  return launch_k(w4_rows_kernel<TX, NT>, grid, dim3(kW4Warps * 32), 0, st, true, p);
}
template <typename TX>
cudaError_t launch_w4(const W4Params& p, cudaStream_t st) {
  if (p.M <= 8) return launch_rows<TX, 1>(p, st);
  if (p.M <= 16) return launch_rows<TX, 2>(p, st);
  return launch_rows<TX, 4>(p, st);
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
int64_t blocks64(int K, int group) {
  const int b = group == 128 ? 128 : 64;
  return (int64_t)((K + b - 1) / b) * (b / 64);
}

}  // namespace
}  // namespace glad

using namespace glad;

extern "C" {

size_t glad_w4_tiles_bytes(int in_features, int out_features, int group) {
  if (!shape_ok(in_features, out_features, group)) return 0;
  return (size_t)((out_features + 15) / 16) * (size_t)blocks64(in_features, group) * 512;
}

size_t glad_w4_scales_bytes(int in_features, int out_features, int group) {
  if (!shape_ok(in_features, out_features, group)) return 0;
  return (size_t)((out_features + 15) / 16) * (size_t)(blocks64(in_features, group) * 64 / group) * 32;
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
  p.KB = (int)blocks64(K, w->group);
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
