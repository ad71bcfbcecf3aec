// Root-mean-square norm with the residual's addition: 16/32-bit output (forward and
// backward) and 8-bit output with scales.
//
//   h = x + r, rounded to r's type (h = x without a residual)
//   rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * w
//   8 bits: s = max|y| / Q over a row or a group of columns (Q = 127 int8, 448 e4m3;
//           1 where the maximum is 0), q = round_half_even(y * (1/s)); or s is given.
//   backward, g = dy * w:  dh' = dh + rstd * (g - h * rstd^2 * mean(g * h)),
//           dx = dr = dh',  dw = sum over rows of dy * h * rstd
//
// Every operator reads its inputs once and keeps the row in registers between the
// reduction and the store, so DRAM bytes are the bound. Sums, statistics and the
// products are fp32; h is rounded because it is an output that the next layer (and the
// backward pass) reads, and the norm is of the value that is stored.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdio>

#include "glad_common.cuh"

namespace glad {
int set_last_error(int code, const char* msg);

namespace {

constexpr int kNormMaxCols = 32768;      // a row lives in the registers of one block
constexpr int kNormMaxPartials = 1184;   // dw partial rows of the backward pass (8 per SM)
constexpr int kNormRowsPerTeam = 4;      // rows a team sums before it may write a dw partial

struct NormParams {
  const void* x;        // forward: input rows; backward: dy
  const void* r;        // forward: residual or null; backward: dh or null
  const void* h;        // backward: the normalised rows
  const void* w;        // weight or null
  int64_t ldx, ldr, ldh;
  int64_t rows;
  int cols, team;       // team: threads of one row
  int w_f32;
  float eps;
  void* y;              // forward: output; backward: dx
  void* sum;            // forward: h out or null; backward: dr or null
  float* rstd;          // forward: out or null; backward: in
  int q_e4m3, group;    // 8-bit form: group 0 = one scale a row
  const float* given;   // given scale or null
  float* scales;
  float* partial;       // backward: dw partial rows [grid * teams, cols] or null
};

// ---- element access -------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_f(float v) { return v; }

// VEC consecutive elements, VEC 1 or 8 (8: 16-byte aligned).
template <int VEC, typename T>
__device__ __forceinline__ void load_v(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = to_f<T>(*p);
  } else {
    __align__(16) T v[VEC];
#pragma unroll
    for (int i = 0; i < (int)(VEC * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f<T>(v[i]);
  }
}
template <int VEC, typename T>
__device__ __forceinline__ void store_v(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f<T>(f[0]);
  } else {
    __align__(16) T v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = from_f<T>(f[i]);
#pragma unroll
    for (int i = 0; i < (int)(VEC * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
  }
}
// Weight elements [col, col + VEC): the input's type or fp32; ones without a weight.
template <int VEC, typename TX>
__device__ __forceinline__ void load_w(const NormParams& p, int64_t col, float (&f)[VEC]) {
  if (p.w == nullptr) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 1.0f;
  } else if (p.w_f32) {
    load_v<VEC, float>(static_cast<const float*>(p.w) + col, f);
  } else {
    load_v<VEC, TX>(static_cast<const TX*>(p.w) + col, f);
  }
}

// Sum / unsigned maximum over the `team` threads that share a row; `red` holds one word a
// warp. Every thread of the block calls it the same number of times.
__device__ __forceinline__ float team_sum(float v, int team, float* red) {
  v = warp_sum(v);
  if (team == 32) return v;
  const int warp = threadIdx.x >> 5, per = team >> 5, first = warp / per * per;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < per ? red[first + lane] : 0.0f);
}
__device__ __forceinline__ uint32_t team_max(uint32_t v, int team, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (team == 32) return v;
  const int warp = threadIdx.x >> 5, per = team >> 5, first = warp / per * per;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return __reduce_max_sync(0xffffffffu, lane < per ? red[first + lane] : 0u);
}

// ---- 8-bit rounding ---------------------------------------------------------------------
// The scale of a maximum held as the bits of |y| (a NaN has the largest bits and stays NaN).
__device__ __forceinline__ float q_scale(uint32_t amax_bits, float qmax) {
  return amax_bits == 0u ? 1.0f : __fdiv_rn(__uint_as_float(amax_bits), qmax);
}
// Multiplying by RN(1/s) instead of dividing moves a code only where y/s lies within two
// roundings of a border between two codes. Scales whose reciprocal may overflow divide.
struct QuantStep {
  float s, inv;
  __device__ __forceinline__ float operator()(float y) const {
    return fabsf(s) < 1e-36f ? __fdiv_rn(y, s) : __fmul_rn(y, inv);
  }
};
__device__ __forceinline__ QuantStep quant_step(float s) {
  QuantStep q;
  q.s = s;
  q.inv = __frcp_rn(s);
  return q;
}
__device__ __forceinline__ uint32_t code_i8(float t) {
  int q = __float2int_rn(t);                    // NaN -> 0, out of range saturates
  q = max(-127, min(127, q));
  return (uint32_t)q & 0xffu;
}
template <int VEC>
__device__ __forceinline__ void store_q(uint8_t* p, const float (&t)[VEC], bool e4m3) {
  if constexpr (VEC == 1) {
    *p = e4m3 ? (uint8_t)__nv_cvt_float_to_fp8(t[0], __NV_SATFINITE, __NV_E4M3) : (uint8_t)code_i8(t[0]);
  } else {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const uint32_t two = e4m3 ? (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(t[i], t[i + 1]), __NV_SATFINITE,
                                                                      __NV_E4M3)
                                : (code_i8(t[i]) | (code_i8(t[i + 1]) << 8));
      w[i >> 2] |= two << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

// ---- forward ------------------------------------------------------------------------------
// One team of threads per row, up to E = VEC * NV elements a thread.
template <typename TX, typename TH, int VEC, int NV, bool QUANT, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_fwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[32];
  __shared__ uint32_t gmax[VEC == 1 && QUANT ? 1024 + 32 : 1];
  const int t = threadIdx.x % p.team, teams = blockDim.x / p.team, who = threadIdx.x / p.team;
  const int64_t row = (int64_t)blockIdx.x * teams + who;
  const bool live = row < p.rows;
  const int nvec = (p.cols + VEC - 1) / VEC;
  float v[NV][VEC];
  grid_dep_wait();
  grid_dep_launch();

  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = i * p.team + t;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[i][e] = 0.0f;
    if (live && k < nvec) load_v<VEC, TX>(static_cast<const TX*>(p.x) + row * p.ldx + (int64_t)k * VEC, v[i]);
  }
  if (p.r != nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = i * p.team + t;
      if (live && k < nvec) {
        float r[VEC];
        load_v<VEC, TH>(static_cast<const TH*>(p.r) + row * p.ldr + (int64_t)k * VEC, r);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = to_f<TH>(from_f<TH>(__fadd_rn(v[i][e], r[e])));
        store_v<VEC, TH>(static_cast<TH*>(p.sum) + row * p.cols + (int64_t)k * VEC, v[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  ss = team_sum(ss, p.team, red);
  const float rstd = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)p.cols), p.eps)));
  if (p.rstd != nullptr && live && t == 0) p.rstd[row] = rstd;

  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = i * p.team + t;
    if (live && k < nvec) {
      float w[VEC];
      load_w<VEC, TX>(p, (int64_t)k * VEC, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = __fmul_rn(__fmul_rn(v[i][e], rstd), w[e]);
        if (QUANT) amax = max(amax, __float_as_uint(v[i][e]) & 0x7fffffffu);
      }
      if (!QUANT) store_v<VEC, TX>(static_cast<TX*>(p.y) + row * p.cols + (int64_t)k * VEC, v[i]);
    }
  }
  if constexpr (QUANT) {
    const float qmax = p.q_e4m3 ? 448.0f : 127.0f;
    uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.cols;
    if (p.group == 0) {
      float s;
      if (p.given != nullptr) {
        s = *p.given;
      } else {
        s = q_scale(team_max(amax, p.team, reinterpret_cast<uint32_t*>(red)), qmax);
        if (live && t == 0) p.scales[row] = s;
      }
      const QuantStep step = quant_step(s);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = i * p.team + t;
        if (live && k < nvec) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i][e] = step(v[i][e]);
          store_q<VEC>(q + (int64_t)k * VEC, v[i], p.q_e4m3);
        }
      }
    } else {
      const int groups = (p.cols + p.group - 1) / p.group;
      float* scales = p.scales + row * groups;
      if constexpr (VEC > 1) {
        // a group is 4, 8 or 16 neighbouring lanes
        const int lanes = p.group / VEC;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int k = i * p.team + t;
          uint32_t m = 0;
#pragma unroll
          for (int e = 0; e < VEC; ++e) m = max(m, __float_as_uint(v[i][e]) & 0x7fffffffu);
          for (int o = lanes >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          if (live && k < nvec) {
            const float s = q_scale(m, qmax);
            if ((k & (lanes - 1)) == 0) scales[k / lanes] = s;
            const QuantStep step = quant_step(s);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = step(v[i][e]);
            store_q<VEC>(q + (int64_t)k * VEC, v[i], p.q_e4m3);
          }
        }
      } else {
        // the 32 lanes of a step lie in one group: one shared-memory maximum a step
        uint32_t* gm = gmax + who * groups;
        for (int g = t; g < groups; g += p.team) gm[g] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int k = i * p.team + t;
          const uint32_t m = __reduce_max_sync(0xffffffffu, k < nvec ? __float_as_uint(v[i][0]) & 0x7fffffffu : 0u);
          if ((threadIdx.x & 31) == 0 && k < nvec) atomicMax(&gm[k / p.group], m);
        }
        __syncthreads();
        if (live)
          for (int g = t; g < groups; g += p.team) scales[g] = q_scale(gm[g], qmax);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int k = i * p.team + t;
          if (live && k < nvec) {
            const float one[1] = {quant_step(q_scale(gm[k / p.group], qmax))(v[i][0])};
            store_q<1>(q + k, one, p.q_e4m3);
          }
        }
      }
    }
  }
}

// ---- backward -----------------------------------------------------------------------------
// A team walks rows team_id, team_id + teams, ...; its columns' share of dw stays in
// registers and is written once as a partial row, which norm_dw_kernel sums in a fixed order.
template <typename TX, typename TH, int VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[32];
  const int t = threadIdx.x % p.team, teams = blockDim.x / p.team, who = threadIdx.x / p.team;
  const int nvec = (p.cols + VEC - 1) / VEC;
  float acc[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[i][e] = 0.0f;
  for (int64_t base = (int64_t)blockIdx.x * teams; base < p.rows; base += (int64_t)gridDim.x * teams) {
    const int64_t row = base + who;
    const bool live = row < p.rows;
    const float rstd = live ? p.rstd[row] : 0.0f;
    float h[NV][VEC], g[NV][VEC];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = i * p.team + t;
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i][e] = g[i][e] = 0.0f;
      if (live && k < nvec) {
        load_v<VEC, TH>(static_cast<const TH*>(p.h) + row * p.ldh + (int64_t)k * VEC, h[i]);
        load_v<VEC, TX>(static_cast<const TX*>(p.x) + row * p.ldx + (int64_t)k * VEC, g[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = i * p.team + t;
      if (live && k < nvec) {
        float w[VEC];
        load_w<VEC, TX>(p, (int64_t)k * VEC, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          acc[i][e] = fmaf(g[i][e], __fmul_rn(h[i][e], rstd), acc[i][e]);
          g[i][e] = __fmul_rn(g[i][e], w[e]);
          dot = fmaf(g[i][e], h[i][e], dot);
        }
      }
    }
    dot = team_sum(dot, p.team, red);
    const float c = __fmul_rn(__fmul_rn(rstd, rstd), __fdiv_rn(dot, (float)p.cols));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = i * p.team + t;
      if (live && k < nvec) {
        float d[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] = __fmul_rn(rstd, fmaf(-h[i][e], c, g[i][e]));
        if (p.r != nullptr) {
          float r[VEC];
          load_v<VEC, TH>(static_cast<const TH*>(p.r) + row * p.ldr + (int64_t)k * VEC, r);
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[e] = __fadd_rn(d[e], r[e]);
        }
        const int64_t at = row * p.cols + (int64_t)k * VEC;
        if (p.y != nullptr) store_v<VEC, TX>(static_cast<TX*>(p.y) + at, d);
        if (p.sum != nullptr) store_v<VEC, TH>(static_cast<TH*>(p.sum) + at, d);
      }
    }
  }
  if (p.partial != nullptr) {
    float* out = p.partial + ((int64_t)blockIdx.x * teams + who) * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = i * p.team + t;
      if (k < nvec) store_v<VEC, float>(out + (int64_t)k * VEC, acc[i]);
    }
  }
}

// dw[c] = sum of the partial rows: 32 columns x 32 row slices a block, slices joined in order.
template <typename TW>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* partial, int n, int cols, TW* dw) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.0f;
  if (c < cols)
    for (int i = threadIdx.y; i < n; i += 32) v += partial[(int64_t)i * cols + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = warp_sum(s[threadIdx.x][threadIdx.y]);
  const int c2 = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c2 < cols) dw[c2] = from_f<TW>(v);
}

// ---- launch -------------------------------------------------------------------------------
int num_sms() {
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

struct Shape {
  int team, threads;
  bool wide;            // 32 elements a thread instead of 8
};
Shape shape_of(int64_t rows, int cols) {
  Shape s;
  // few rows: as many threads a row as there are 8-element pieces (latency); many rows: 32
  // elements a thread, so that a thread has several loads in flight and a row fewer warps
  s.wide = rows > 2 * num_sms() || cols > 8192;
  const int e = s.wide ? 32 : 8;
  s.team = ((cols + e - 1) / e + 31) / 32 * 32;
  s.threads = s.team >= 256 ? s.team : 256 / s.team * s.team;
  if (!s.wide) s.threads = s.team;
  return s;
}

template <typename TX, typename TH, bool QUANT>
cudaError_t launch_fwd(NormParams p, bool vec, cudaStream_t st) {
  const Shape s = shape_of(p.rows, p.cols);
  p.team = s.team;
  const int teams = s.threads / s.team;
  const dim3 grid((unsigned)((p.rows + teams - 1) / teams)), block((unsigned)s.threads);
  if (!s.wide)
    return vec ? launch_k(norm_fwd_kernel<TX, TH, 8, 1, QUANT, 1024>, grid, block, 0, st, true, p)
               : launch_k(norm_fwd_kernel<TX, TH, 1, 8, QUANT, 1024>, grid, block, 0, st, true, p);
  if (s.threads <= 512)
    return vec ? launch_k(norm_fwd_kernel<TX, TH, 8, 4, QUANT, 512>, grid, block, 0, st, true, p)
               : launch_k(norm_fwd_kernel<TX, TH, 1, 32, QUANT, 512>, grid, block, 0, st, true, p);
  return vec ? launch_k(norm_fwd_kernel<TX, TH, 8, 4, QUANT, 1024>, grid, block, 0, st, true, p)
             : launch_k(norm_fwd_kernel<TX, TH, 1, 32, QUANT, 1024>, grid, block, 0, st, true, p);
}

int64_t bwd_teams(int64_t rows) {
  const int64_t t = (rows + kNormRowsPerTeam - 1) / kNormRowsPerTeam;
  return t < kNormMaxPartials ? t : kNormMaxPartials;
}

template <typename TX, typename TH>
cudaError_t launch_bwd(NormParams p, bool vec, void* dw, int dw_f32, cudaStream_t st) {
  const Shape s = shape_of(p.rows, p.cols);
  p.team = s.team;
  const int teams = s.threads / s.team;
  int64_t blocks = bwd_teams(p.rows) / teams;
  if (blocks < 1) blocks = 1;
  const dim3 grid((unsigned)blocks), block((unsigned)s.threads);
  cudaError_t e;
  if (!s.wide)
    e = vec ? launch_k(norm_bwd_kernel<TX, TH, 8, 1, 1024>, grid, block, 0, st, false, p)
            : launch_k(norm_bwd_kernel<TX, TH, 1, 8, 1024>, grid, block, 0, st, false, p);
  else if (s.threads <= 512)
    e = vec ? launch_k(norm_bwd_kernel<TX, TH, 8, 4, 512>, grid, block, 0, st, false, p)
            : launch_k(norm_bwd_kernel<TX, TH, 1, 32, 512>, grid, block, 0, st, false, p);
  else
    e = vec ? launch_k(norm_bwd_kernel<TX, TH, 8, 4, 1024>, grid, block, 0, st, false, p)
            : launch_k(norm_bwd_kernel<TX, TH, 1, 32, 1024>, grid, block, 0, st, false, p);
  if (e != cudaSuccess || dw == nullptr) return e;
  const dim3 g2((unsigned)((p.cols + 31) / 32)), b2(32, 32);
  const int n = (int)(blocks * teams);
  if (dw_f32) return launch_k(norm_dw_kernel<float>, g2, b2, 0, st, false, (const float*)p.partial, n, p.cols, (float*)dw);
  return launch_k(norm_dw_kernel<TX>, g2, b2, 0, st, false, (const float*)p.partial, n, p.cols, (TX*)dw);
}

// ---- argument checks ------------------------------------------------------------------------
int bad(const char* who, const char* what) {
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  return set_last_error(GLAD_ERR_INVALID_ARG, msg);
}
int cuda_bad(const char* who, cudaError_t e) {
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", who, cudaGetErrorString(e));
  return set_last_error(GLAD_ERR_CUDA, msg);
}
size_t width_of(int dtype) { return dtype == GLAD_DTYPE_F32 ? 4 : 2; }
bool is_float(int dtype) { return dtype == GLAD_DTYPE_F32 || dtype == GLAD_DTYPE_F16 || dtype == GLAD_DTYPE_BF16; }
bool on(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
// A row tensor: element-aligned, rows at least `cols` apart.
const char* rows_wrong(const void* p, int dtype, int64_t ld, int64_t rows, int cols) {
  if (!on(p, width_of(dtype))) return "a tensor is not element-aligned";
  if (rows > 1 && ld < cols) return "a row stride is below the number of columns";
  return nullptr;
}
// 8-element accesses: base and row pitch on 16 bytes.
bool vec_ok(const void* p, int dtype, int64_t ld, int64_t rows) {
  if (p == nullptr) return true;
  return on(p, 16) && (rows <= 1 || (ld * (int64_t)width_of(dtype)) % 16 == 0);
}

// Calls f(TX, TH) for the supported pairs.
template <typename F>
int for_types(int x_dtype, int h_dtype, F&& f) {
  if (x_dtype == GLAD_DTYPE_F16) return h_dtype == GLAD_DTYPE_F32 ? f(__half(), float()) : f(__half(), __half());
  if (x_dtype == GLAD_DTYPE_BF16)
    return h_dtype == GLAD_DTYPE_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
  return f(float(), float());
}

const char* common_wrong(int x_dtype, int h_dtype, const void* w, int w_dtype, int64_t rows, int cols) {
  if (!is_float(x_dtype)) return "x must be f32, f16 or bf16";
  if (h_dtype != x_dtype && h_dtype != GLAD_DTYPE_F32) return "the residual must have x's type or f32";
  if (w != nullptr && w_dtype != x_dtype && w_dtype != GLAD_DTYPE_F32) return "the weight must have x's type or f32";
  if (w != nullptr && !on(w, width_of(w_dtype))) return "the weight is not element-aligned";
  if (rows < 0 || rows > 0x7fffffffLL) return "rows must be in [0, 2^31)";
  if (cols < 1 || cols > kNormMaxCols) return "cols must be in [1, 32768]";
  return nullptr;
}

int forward_call(const char* who, const void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype,
                 int64_t ldr, const void* weight, int w_dtype, int64_t rows, int cols, float eps, void* sum_out,
                 NormParams p, bool quant, void* stream) {
  const int h_dtype = residual ? r_dtype : x_dtype;
  const char* why = common_wrong(x_dtype, h_dtype, weight, w_dtype, rows, cols);
  if (why) return bad(who, why);
  if (!(eps >= 0.0f)) return bad(who, "eps must be >= 0");
  if (rows == 0) return GLAD_OK;
  if (!x || !p.y) return bad(who, "x and the output must be set");
  if ((residual == nullptr) != (sum_out == nullptr)) return bad(who, "residual and sum_out go together");
  if ((why = rows_wrong(x, x_dtype, ldx, rows, cols))) return bad(who, why);
  if (residual && (why = rows_wrong(residual, h_dtype, ldr, rows, cols))) return bad(who, why);
  if (sum_out && !on(sum_out, width_of(h_dtype))) return bad(who, "sum_out is not element-aligned");
  if (!quant && !on(p.y, width_of(x_dtype))) return bad(who, "y is not element-aligned");
  p.x = x;
  p.r = residual;
  p.w = weight;
  p.ldx = ldx;
  p.ldr = ldr;
  p.rows = rows;
  p.cols = cols;
  p.w_f32 = w_dtype == GLAD_DTYPE_F32;
  p.eps = eps;
  p.sum = sum_out;
  const bool vec = cols % 8 == 0 && vec_ok(x, x_dtype, ldx, rows) && vec_ok(residual, h_dtype, ldr, rows) &&
                   on(weight, 16) && on(sum_out, 16) && on(p.y, quant ? 8 : 16);
  const cudaStream_t st = (cudaStream_t)stream;
  return for_types(x_dtype, h_dtype, [&](auto tx, auto th) {
    using TX = decltype(tx);
    using TH = decltype(th);
    const cudaError_t e = quant ? launch_fwd<TX, TH, true>(p, vec, st) : launch_fwd<TX, TH, false>(p, vec, st);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  });
}

}  // namespace
}  // namespace glad

using namespace glad;

extern "C" {

int glad_rms_norm_forward(const void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype, int64_t ldr,
                          const void* weight, int w_dtype, int64_t rows, int cols, float eps, void* y, void* sum_out,
                          float* rstd_out, void* stream) {
  NormParams p{};
  p.y = y;
  p.rstd = rstd_out;
  return forward_call("glad_rms_norm_forward", x, x_dtype, ldx, residual, r_dtype, ldr, weight, w_dtype, rows, cols,
                      eps, sum_out, p, false, stream);
}

int glad_rms_norm_quant(const void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype, int64_t ldr,
                        const void* weight, int w_dtype, int64_t rows, int cols, float eps, int q_dtype, int group,
                        const float* given_scale, void* q, float* scales, void* sum_out, void* stream) {
  const char* who = "glad_rms_norm_quant";
  if (q_dtype != GLAD_DTYPE_I8 && q_dtype != GLAD_DTYPE_E4M3) return bad(who, "the output must be i8 or e4m3");
  if (group != 0 && group != 32 && group != 64 && group != 128) return bad(who, "group must be 0, 32, 64 or 128");
  if (given_scale && group) return bad(who, "a given scale is one for the whole tensor (group 0)");
  if (rows > 0 && !given_scale && !scales) return bad(who, "scales must be set without a given scale");
  if (!on(given_scale, 4) || !on(scales, 4)) return bad(who, "scales must be 4-byte aligned");
  NormParams p{};
  p.y = q;
  p.q_e4m3 = q_dtype == GLAD_DTYPE_E4M3;
  p.group = group;
  p.given = given_scale;
  p.scales = scales;
  return forward_call(who, x, x_dtype, ldx, residual, r_dtype, ldr, weight, w_dtype, rows, cols, eps, sum_out, p, true,
                      stream);
}

size_t glad_rms_norm_backward_workspace_size(int64_t rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // a block holds up to eight teams, so the number of partial rows is at most this
  const int64_t teams = bwd_teams(rows);
  return (size_t)(teams < 8 ? 8 : teams) * (size_t)cols * sizeof(float);
}

int glad_rms_norm_backward(const void* dy, int x_dtype, int64_t lddy, const void* dsum, int h_dtype, int64_t lddsum,
                           const void* h, int64_t ldh, const void* weight, int w_dtype, const float* rstd,
                           int64_t rows, int cols, void* dx, void* dresidual, void* dweight, void* workspace,
                           size_t workspace_bytes, void* stream) {
  const char* who = "glad_rms_norm_backward";
  const char* why = common_wrong(x_dtype, h_dtype, weight, w_dtype, rows, cols);
  if (why) return bad(who, why);
  if (dweight && !weight) return bad(who, "dweight without a weight");
  if (!dweight && rows == 0) return GLAD_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    const cudaError_t e = cudaMemsetAsync(dweight, 0, (size_t)cols * width_of(w_dtype), st);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  }
  if (!dy || !h || !rstd) return bad(who, "dy, h and rstd must be set");
  if (!dx && !dresidual && !dweight) return bad(who, "no output is set");
  if ((why = rows_wrong(dy, x_dtype, lddy, rows, cols))) return bad(who, why);
  if ((why = rows_wrong(h, h_dtype, ldh, rows, cols))) return bad(who, why);
  if (dsum && (why = rows_wrong(dsum, h_dtype, lddsum, rows, cols))) return bad(who, why);
  if (!on(rstd, 4) || !on(dx, width_of(x_dtype)) || !on(dresidual, width_of(h_dtype)) ||
      !on(dweight, width_of(w_dtype)))
    return bad(who, "a tensor is not element-aligned");
  if (dweight && (!workspace || workspace_bytes < glad_rms_norm_backward_workspace_size(rows, cols) ||
                  !on(workspace, 16)))
    return set_last_error(GLAD_ERR_WORKSPACE,
                          "glad_rms_norm_backward: workspace of glad_rms_norm_backward_workspace_size bytes required");
  NormParams p{};
  p.x = dy;
  p.ldx = lddy;
  p.r = dsum;
  p.ldr = lddsum;
  p.h = h;
  p.ldh = ldh;
  p.w = weight;
  p.w_f32 = w_dtype == GLAD_DTYPE_F32;
  p.rows = rows;
  p.cols = cols;
  p.y = dx;
  p.sum = dresidual;
  p.rstd = const_cast<float*>(rstd);
  p.partial = dweight ? static_cast<float*>(workspace) : nullptr;
  const bool vec = cols % 8 == 0 && vec_ok(dy, x_dtype, lddy, rows) && vec_ok(dsum, h_dtype, lddsum, rows) &&
                   vec_ok(h, h_dtype, ldh, rows) && on(weight, 16) && on(dx, 16) && on(dresidual, 16);
  return for_types(x_dtype, h_dtype, [&](auto tx, auto th) {
    using TX = decltype(tx);
    using TH = decltype(th);
    const cudaError_t e = launch_bwd<TX, TH>(p, vec, dweight, p.w_f32, st);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  });
}

}  // extern "C"
