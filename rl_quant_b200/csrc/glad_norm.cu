// Root-mean-square norm with the residual's addition: 16/32-bit output (forward and
// backward) and 8-bit output with scales.
//
//   h = x + r, rounded to r's type (h = x without a residual)
//   rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * w
//   8 bits: s = max|y| / Q over a row or a group of columns (Q = 127 int8, 448 e4m3;
//           1 where that is 0 in fp32), q = round_half_even(y / s); or s is given.
//   backward, g = dy * w:  dh' = dh + rstd * (g - h * rstd^2 * mean(g * h)),
//           dx = dr = dh',  dw = sum over rows of dy * h * rstd
//
// Every operator reads its inputs once and keeps the row in registers between the
// reduction and the store, so DRAM bytes are the bound. Sums, statistics and the
// products are fp32; h is rounded because it is an output that the next layer (and the
// backward pass) reads, and the norm is of the value that is stored.
#include <cuda_fp8.h>

#include "glad_elem.cuh"
#include "glad_common.cuh"

namespace glad {
namespace {

constexpr int kNormMaxCols = 32768;      // a row lives in the registers of one block
// dw partial rows of the backward pass: rows in work at once, in teams of threads. Four blocks an SM where a block is one
// team (more than 2048 columns); narrow rows go up to eight teams a block, and the grid is as much smaller.
constexpr int kNormMaxPartials = 592;

struct NormParams {
  const void* x;        // forward: input rows; backward: dy
  const void* r;        // forward: residual or null; backward: dh or null
  const void* h;        // backward: the normalised rows
  const void* w;        // weight or null
  int64_t ldx, ldr, ldh;
  int64_t rows;
  int cols, team, teams;   // team: threads of one row; teams of a block
  int w_f32;
  float eps, inv_cols;
  void* y;              // forward: output; backward: dx
  void* sum;            // forward: h out or null; backward: dr or null
  float* rstd;          // forward: out or null; backward: in
  int group;            // 8-bit form: group 0 = one scale a row
  const float* given;   // given scale or null
  float* scales;
  float* partial;       // backward: dw partial rows [grid * teams, cols] or null
};

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
// warp and is used by one call between two barriers that follow it. Every thread of the block calls it
// the same number of times.
__device__ __forceinline__ float team_sum(float v, int team, float* red) {
  v = warp_sum(v);
  if (team == 32) return v;
  const int warp = threadIdx.x >> 5, per = team >> 5, first = team == (int)blockDim.x ? 0 : warp / per * per;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < per ? red[first + lane] : 0.0f);
}
__device__ __forceinline__ uint32_t team_max(uint32_t v, int team, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (team == 32) return v;
  const int warp = threadIdx.x >> 5, per = team >> 5, first = team == (int)blockDim.x ? 0 : warp / per * per;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return __reduce_max_sync(0xffffffffu, lane < per ? red[first + lane] : 0u);
}

// ---- 8-bit rounding ---------------------------------------------------------------------
// The largest of m and the |v|; a NaN stays.
template <int N>
__device__ __forceinline__ float max_abs(float m, const float (&v)[N]) {
  if constexpr (N == 1) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[0])));
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[e]), "f"(v[e + 1]));
  }
  return m;
}
// The 8-bit form finds its own scales with z = h * (Qz * 2^k) * w instead of y: 2^k is rstd without its mantissa m = rstd / 2^k,
// and Qz = Q / kUp, below 1 with few bits, so y = z / Qz * m. The scale is s = max|y| / Q and a code rounds y / s = z / d,
// d = max|z| / Q: rstd's own rounding cancels, and where h and w have 16 bits and z fits the 24 of fp32 (bf16 always), z
// and d are exact, so a quotient on a border between two codes is found there.
template <bool E4M3>
struct Q8 {
  static constexpr float kMax = E4M3 ? 448.0f : 127.0f;        // Q
  static constexpr float kUp = E4M3 ? 512.0f : 128.0f;
  static constexpr float kZ = kMax / kUp;                      // Qz
};
__device__ __forceinline__ float rcp_approx(float x) {   // x normal; within one unit in the last place
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two neighbouring elements in one instruction, the second operand (and the addend's) the same or a pair.
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y, float u, float v) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(a), "=f"(b) : "f"(x), "f"(y), "f"(u), "f"(v));
}
__device__ __forceinline__ void fma2(float& a, float& b, float x, float y, float u, float v, float s, float t) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%6, %7};\n\t"
      "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(a), "=f"(b) : "f"(x), "f"(y), "f"(u), "f"(v), "f"(s), "f"(t));
}
// y / s by a product with the reciprocal and STEPS correction steps (Markstein, "Computation of elementary functions on
// the IBM RISC System/6000 processor", 1990): a step takes the remainder, one fused multiply-add, times the reciprocal. The
// product is off by at most 1.5 * 2^-23 of the quotient; after one step with a reciprocal good to 2^-23 what is rounded
// is off by 2^-44, after a second one with the rounded reciprocal the result is the rounded quotient, always. `y` is
// given negated: the remainder q * s - y then needs no sign of its own, and a zero keeps its sign.
template <int STEPS>
__device__ __forceinline__ float corrected(float minus_y, float s, float inv) {
  float q = __fmul_rn(minus_y, -inv);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) q = fmaf(fmaf(q, s, minus_y), -inv, q);
  return q;
}
template <int STEPS, int N>
__device__ __forceinline__ void corrected_v(float (&v)[N], float s, float inv) {
  if constexpr (N == 1) {
    v[0] = corrected<STEPS>(v[0], s, inv);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float q0, q1, r0, r1;
      mul2(q0, q1, v[e], v[e + 1], -inv, -inv);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        fma2(r0, r1, q0, q1, s, s, v[e], v[e + 1]);
        fma2(q0, q1, r0, r1, -inv, -inv, q0, q1);
      }
      v[e] = q0, v[e + 1] = q1;
    }
  }
}
// rstd = 2^k * m, returns Qz * 2^k. A finite rstd other than 0 lies between 2^-65 and 2^75; 0, infinity and NaN go into
// z as they are.
template <bool E4M3>
__device__ __forceinline__ float split_rstd(float rstd, float& m) {
  m = 1.0f;
  if (!(rstd >= 0x1p-70f && rstd <= 0x1p80f)) return rstd;
  const uint32_t e = __float_as_uint(rstd) & 0x7f800000u;
  m = __fmul_rn(rstd, __uint_as_float(0x7f000000u - e));
  return __fmul_rn(__uint_as_float(e), Q8<E4M3>::kZ);
}
// Whether a maximum of |z| keeps d, s and every remainder that a code depends on among the normal numbers.
__device__ __forceinline__ bool plain_max(float top) { return top >= 0x1p-50f && top <= 0x1p90f; }
// max|z| / Q, and the scale, where plain_max holds.
template <bool E4M3>
__device__ __forceinline__ float plain_over_q(float v) {
  return corrected<1>(-v, Q8<E4M3>::kMax, (float)(1.0 / Q8<E4M3>::kMax));
}
template <bool E4M3>
__device__ __forceinline__ float plain_scale(float d, float m) {
  return plain_over_q<E4M3>(__fmul_rn(d, __fmul_rn(m, Q8<E4M3>::kUp)));
}
__device__ __forceinline__ uint32_t code_i8(float t) {
  int q = __float2int_rn(t);                    // NaN -> 0, out of range saturates
  q = max(-127, min(127, q));
  return (uint32_t)q & 0xffu;
}
template <int VEC, bool E4M3>
__device__ __forceinline__ void store_q(uint8_t* p, const float (&t)[VEC]) {
  if constexpr (VEC == 1) {
    *p = E4M3 ? (uint8_t)__nv_cvt_float_to_fp8(t[0], __NV_SATFINITE, __NV_E4M3) : (uint8_t)code_i8(t[0]);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const uint32_t two = E4M3 ? (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(t[i], t[i + 1]), __NV_SATFINITE,
                                                                      __NV_E4M3)
                                : (code_i8(t[i]) | (code_i8(t[i + 1]) << 8));
      w[i >> 2] |= two << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

// A thread's place: its row's team in the block, its index there.
__device__ __forceinline__ void place(int team, int& who, int& t) {
  if (team == (int)blockDim.x) {
    who = 0;
    t = threadIdx.x;
  } else {
    who = threadIdx.x / team;
    t = threadIdx.x - who * team;
  }
}

// Codes and scales where those of the fast form do not hold (a maximum or a given scale out of its range, an infinite
// quotient), which is rare: the pieces `slow` (bit i: piece i) of a thread, one element at a time, from memory and by division.
// row_top: the row's maximum of |z|.
template <typename TX, typename TH, int VEC, int NV, bool E4M3>
__device__ __noinline__ void quant_slow(const NormParams& p, uint32_t slow, float rstd, float row_top) {
  int who, t;
  place(p.team, who, t);
  const int64_t row = (int64_t)blockIdx.x * p.teams + who;
  const int groups = p.group != 0 ? (p.cols + p.group - 1) / p.group : 1;
  auto y_of = [&](int c) {
    const float h = p.r != nullptr ? to_f<TH>(static_cast<const TH*>(p.sum)[row * p.cols + c])
                                   : to_f<TX>(static_cast<const TX*>(p.x)[row * p.ldx + c]);
    float w[1];
    load_w<1, TX>(p, c, w);
    return __fmul_rn(__fmul_rn(h, rstd), w[0]);
  };
  float s = 1.0f, m;
  if (p.given != nullptr) {
    s = *p.given;
  } else if (p.group == 0) {
    split_rstd<E4M3>(rstd, m);
    s = __fdiv_rn(__fmul_rn(__fdiv_rn(row_top, Q8<E4M3>::kZ), m), Q8<E4M3>::kMax);
    if (s == 0.0f) s = 1.0f;                     // a scale that rounds to zero; a NaN stays
    if (t == 0) p.scales[row] = s;
  }
#pragma unroll 1
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * p.team + t) * VEC;
    if (!(slow >> i & 1) || c0 >= p.cols) continue;
    if (p.group != 0) {
      const int g0 = c0 / p.group * p.group;
      float top[1] = {0.0f}, y[1];
#pragma unroll 1
      for (int c = g0; c < min(g0 + p.group, p.cols); ++c) {
        y[0] = y_of(c);
        top[0] = max_abs<1>(top[0], y);
      }
      s = __fdiv_rn(top[0], Q8<E4M3>::kMax);
      if (s == 0.0f) s = 1.0f;
      if (c0 == g0) p.scales[row * groups + c0 / p.group] = s;
    }
#pragma unroll 1
    for (int c = c0; c < min(c0 + VEC, p.cols); ++c) {
      const float q[1] = {__fdiv_rn(y_of(c), s)};
      store_q<1, E4M3>(static_cast<uint8_t*>(p.y) + row * p.cols + c, q);
    }
  }
}

// ---- forward ------------------------------------------------------------------------------
// One team of threads per row, up to VEC * NV elements a thread. QUANT: 0 none, 1 int8, 2 e4m3.
// 8192 x 4096, bf16 with an fp32 residual: 403 MB in 63 us, 6.4 TB/s, what a plain copy reaches here. 8192 x 8192 bf16 to
// e4m3 with groups of 128: 472 MB in 91.6 us, 5.2 TB/s; there the instruction issue is busy for 77% of the time (a
// maximum, a scale, a quotient and a conversion an element on top; with a product by the reciprocal in place of the quotient
// 87.4 us, but other codes on borders). 1 x 2048 f16: 1.6 us, a launch.
// A persistent block that fetches its next row ahead gained nothing: with one row a block the
// scheduler already has five blocks' loads in flight on an SM.
// Blocks an SM of the 8-bit forms: three where a thread's elements fit 40 registers (8192 x 8192 e4m3, groups of 128: 91.6
// against 105 us with two).
template <typename TH, int VEC, int QUANT, int MAXT>
constexpr int kFwdBlocks = QUANT == 0 || VEC == 1 ? 0 : MAXT == 512 && sizeof(TH) == 2 ? 3 : 1;
template <typename TX, typename TH, int VEC, int NV, int QUANT, int MAXT>
__global__ void __launch_bounds__(MAXT, kFwdBlocks<TH, VEC, QUANT, MAXT>) norm_fwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[32];
  __shared__ uint32_t red_max[QUANT != 0 ? 32 : 1];
  __shared__ float red_rstd[QUANT != 0 ? 32 : 1];
  __shared__ uint32_t gmax[VEC == 1 && QUANT != 0 ? 1024 + 32 : 1];
  constexpr bool E4M3 = QUANT == 2;
  int who, t;
  place(p.team, who, t);
  const int nvec = (p.cols + VEC - 1) / VEC;
  const int64_t row = (int64_t)blockIdx.x * p.teams + who;
  const bool live = row < p.rows;
  grid_dep_wait();
  grid_dep_launch();

  // every load of the row is issued before the first is used
  Raw<VEC, TX> xn[NV];
  Raw<VEC, TH> rn[NV];
  if (live) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = i * p.team + t;
      if (k < nvec) {
        load_raw<VEC, TX>(static_cast<const TX*>(p.x) + row * p.ldx + (int64_t)k * VEC, xn[i]);
        if (p.r != nullptr) load_raw<VEC, TH>(static_cast<const TH*>(p.r) + row * p.ldr + (int64_t)k * VEC, rn[i]);
      }
    }
  }
  float v[NV][VEC];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = i * p.team + t;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[i][e] = 0.0f;
    if (live && k < nvec) {
      to_floats<VEC, TX>(xn[i], v[i]);
      if (p.r != nullptr) {
        float r[VEC];
        to_floats<VEC, TH>(rn[i], r);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = __fadd_rn(v[i][e], r[e]);
        store_v<VEC, TH, true>(static_cast<TH*>(p.sum) + row * p.cols + (int64_t)k * VEC, v[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  ss = team_sum(ss, p.team, red);
  const float rstd = rsqrtf(fmaf(ss, p.inv_cols, p.eps));   // within 2 units in the last place
  if (p.rstd != nullptr && live && t == 0) p.rstd[row] = rstd;
  float unit = rstd, m = 1.0f;                   // v becomes y; 8 bits: -y, or -z where the scale is found here
  if (QUANT != 0) unit = -(p.given == nullptr ? split_rstd<E4M3>(rstd, m) : rstd);

#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = i * p.team + t;
    if (live && k < nvec) {
      float w[VEC];
      load_w<VEC, TX>(p, (int64_t)k * VEC, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = __fmul_rn(__fmul_rn(v[i][e], unit), w[e]);
      if (QUANT == 0) store_v<VEC, TX>(static_cast<TX*>(p.y) + row * p.cols + (int64_t)k * VEC, v[i]);
    }
  }
  if constexpr (QUANT != 0) {
    uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.cols;
    // The fast form everywhere, without branches that would keep the pieces from overlapping; what it does not hold
    // for is written again at the end. A maximum of zero gives zeros by any divisor, and the scale 1.
    if ((threadIdx.x & 31) == 0) red_rstd[threadIdx.x >> 5] = rstd;      // for then, in no register
    float row_top = 0.0f;
    uint32_t slow = 0;
    if (p.group == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) row_top = max_abs<VEC>(row_top, v[i]);
      if (p.given != nullptr) {
        const float s = *p.given, inv = __frcp_rn(s);
        slow = s >= 0x1p-60f && s <= 0x1p60f && row_top <= s * 0x1p30f ? 0u : ~0u;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int k = i * p.team + t;
          if (live && k < nvec) {
            corrected_v<2>(v[i], s, inv);
            store_q<VEC, E4M3>(q + (int64_t)k * VEC, v[i]);
          }
        }
      } else {
        row_top = __uint_as_float(team_max(__float_as_uint(row_top), p.team, red_max));
        slow = plain_max(row_top) || row_top == 0.0f ? 0u : ~0u;
        const float d = row_top == 0.0f ? 1.0f : plain_over_q<E4M3>(row_top), inv = rcp_approx(d);
        if (live && t == 0) p.scales[row] = row_top == 0.0f ? 1.0f : plain_scale<E4M3>(d, m);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int k = i * p.team + t;
          if (live && k < nvec) {
            corrected_v<1>(v[i], d, inv);
            store_q<VEC, E4M3>(q + (int64_t)k * VEC, v[i]);
          }
        }
      }
    } else {
      const int groups = (p.cols + p.group - 1) / p.group;
      float* scales = p.scales + row * groups;
      if constexpr (VEC > 1) {
        // a group is 4 to 16 neighbouring lanes
        const int lanes = p.group / VEC;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int k = i * p.team + t;
          uint32_t u = __float_as_uint(max_abs<VEC>(0.0f, v[i]));
          for (int o = lanes >> 1; o > 0; o >>= 1) u = max(u, __shfl_xor_sync(0xffffffffu, u, o));
          if (live && k < nvec) {
            const float top = __uint_as_float(u), d = u == 0 ? 1.0f : plain_over_q<E4M3>(top);
            if (!plain_max(top) && u != 0) slow |= 1u << i;
            if ((k & (lanes - 1)) == 0) scales[k / lanes] = u == 0 ? 1.0f : plain_scale<E4M3>(d, m);
            corrected_v<1>(v[i], d, rcp_approx(d));
            store_q<VEC, E4M3>(q + (int64_t)k * VEC, v[i]);
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
          const uint32_t u = __reduce_max_sync(0xffffffffu, k < nvec ? __float_as_uint(v[i][0]) & 0x7fffffffu : 0u);
          if ((threadIdx.x & 31) == 0 && k < nvec) atomicMax(&gm[k / p.group], u);
        }
        __syncthreads();
        if (live) {
          for (int g = t; g < groups; g += p.team) {
            const float top = __uint_as_float(gm[g]);
            if (top == 0.0f) scales[g] = 1.0f;
            else if (plain_max(top)) scales[g] = plain_scale<E4M3>(plain_over_q<E4M3>(top), m);
          }                                      // the others by the thread of the group's first column
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int k = i * p.team + t;
          if (live && k < nvec) {
            const uint32_t u = gm[k / p.group];
            const float top = __uint_as_float(u), d = u == 0 ? 1.0f : plain_over_q<E4M3>(top);
            if (!plain_max(top) && u != 0) slow |= 1u << i;
            corrected_v<1>(v[i], d, rcp_approx(d));
            store_q<1, E4M3>(q + k, v[i]);
          }
        }
      }
    }
    __syncwarp();
    if (live && slow != 0) quant_slow<TX, TH, VEC, NV, E4M3>(p, slow, red_rstd[threadIdx.x >> 5], row_top);
  }
}

// ---- backward -----------------------------------------------------------------------------
// A team walks rows team_id, team_id + teams, ...; its columns' share of dw stays in
// registers and is written once as a partial row, which norm_dw_kernel sums in a fixed order.
// 8192 x 4096, bf16 with an fp32 sum, gradients of both and of the weight: 537 MB in 98 us, 5.5 TB/s, 86% of a copy's
// rate: 64 registers a thread for the row, its gradient and dw's share leave 32 warps an SM to hide the row's one
// barrier, and are not quite enough: this instance spills 29 words a thread. A ring of asynchronous copies ahead of the row
// and three blocks an SM (40 registers, more spills) were slower. Not timed: rows of more than 16384 columns (32 elements a
// thread, since a block could not hold the row otherwise: 150 to 900 words spilled) and many rows of few columns.
template <typename TX, typename TH, int VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT <= 512 ? 2 : 1) norm_bwd_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[2][32];                           // rows use them in turn: one barrier a row
  int who, t, parity = 0;
  place(p.team, who, t);
  const int teams = p.teams;
  const int nvec = (p.cols + VEC - 1) / VEC;
  grid_dep_wait();
  grid_dep_launch();
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
    dot = team_sum(dot, p.team, red[parity]);
    parity ^= 1;
    const float c = __fmul_rn(__fmul_rn(rstd, rstd), __fmul_rn(dot, p.inv_cols));
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

// dw[c] = sum of the partial rows: 32 columns x 32 row slices a block, slices joined in order. 592 x 4096: 9.7 MB from
// L2, 4 us behind the backward kernel.
template <typename TW>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* partial, int n, int cols, TW* dw) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.0f;
  grid_dep_wait();
  if (c < cols) {
    int i = threadIdx.y;
    for (; i + 7 * 32 < n; i += 8 * 32) {                // eight loads in flight
      float u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = partial[(int64_t)(i + k * 32) * cols + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) v += u[k];
    }
    for (; i < n; i += 32) v += partial[(int64_t)i * cols + c];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = warp_sum(s[threadIdx.x][threadIdx.y]);
  const int c2 = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c2 < cols) dw[c2] = from_f<TW>(v);
}

// ---- launch -------------------------------------------------------------------------------
struct Shape {
  int team, teams;      // threads of a row, rows of a block
  int elems;            // elements a thread holds: 8, 16 or 32
};
Shape shape_of(int64_t rows, int cols) {
  Shape s;
  // Up to one 8-element piece for each thread the GPU holds: as many threads a row as it has pieces
  // (latency). More: 16 elements a thread, so that a thread has several loads in flight and a row fewer
  // warps (8192 x 4096 forward, bf16 with an f32 sum: 69 us with 32, 63 us with 16 = the copy bandwidth;
  // 1003 x 1111 f16 forward + backward: 85 us with 32, 21 us with 8). 32 where a block could not hold the row.
  s.elems = cols > 16384 ? 32 : rows * cols > (int64_t)num_sms() * 2048 * 8 || cols > 8192 ? 16 : 8;
  s.team = ((cols + s.elems - 1) / s.elems + 31) / 32 * 32;
  s.teams = s.elems == 8 || s.team >= 256 ? 1 : 256 / s.team;
  return s;
}

template <typename TX, typename TH, int QUANT>
cudaError_t launch_fwd(NormParams p, bool vec, cudaStream_t st) {
  const Shape s = shape_of(p.rows, p.cols);
  p.team = s.team;
  p.teams = s.teams;
  const int threads = s.team * s.teams;
  const dim3 grid((unsigned)((p.rows + s.teams - 1) / s.teams)), block((unsigned)threads);
  if (s.elems == 8)
    return vec ? launch_k(norm_fwd_kernel<TX, TH, 8, 1, QUANT, 1024>, grid, block, 0, st, true, p)
               : launch_k(norm_fwd_kernel<TX, TH, 1, 8, QUANT, 1024>, grid, block, 0, st, true, p);
  if (s.elems == 16 && threads <= 512)
    return vec ? launch_k(norm_fwd_kernel<TX, TH, 8, 2, QUANT, 512>, grid, block, 0, st, true, p)
               : launch_k(norm_fwd_kernel<TX, TH, 1, 16, QUANT, 512>, grid, block, 0, st, true, p);
  if (s.elems == 16)
    return vec ? launch_k(norm_fwd_kernel<TX, TH, 8, 2, QUANT, 1024>, grid, block, 0, st, true, p)
               : launch_k(norm_fwd_kernel<TX, TH, 1, 16, QUANT, 1024>, grid, block, 0, st, true, p);
  return vec ? launch_k(norm_fwd_kernel<TX, TH, 8, 4, QUANT, 1024>, grid, block, 0, st, true, p)
             : launch_k(norm_fwd_kernel<TX, TH, 1, 32, QUANT, 1024>, grid, block, 0, st, true, p);
}

int64_t bwd_teams(int64_t rows) { return rows < kNormMaxPartials ? rows : kNormMaxPartials; }

template <typename TX, typename TH>
cudaError_t launch_bwd(NormParams p, bool vec, void* dw, int dw_f32, cudaStream_t st) {
  const Shape s = shape_of(p.rows, p.cols);
  p.team = s.team;
  p.teams = s.teams;
  const int threads = s.team * s.teams;
  int64_t blocks = bwd_teams(p.rows) / s.teams;
  if (blocks < 1) blocks = 1;
  const dim3 grid((unsigned)blocks), block((unsigned)threads);
  cudaError_t e;
  if (s.elems == 8)
    e = vec ? launch_k(norm_bwd_kernel<TX, TH, 8, 1, 1024>, grid, block, 0, st, true, p)
            : launch_k(norm_bwd_kernel<TX, TH, 1, 8, 1024>, grid, block, 0, st, true, p);
  else if (s.elems == 16 && threads <= 512)
    e = vec ? launch_k(norm_bwd_kernel<TX, TH, 8, 2, 512>, grid, block, 0, st, true, p)
            : launch_k(norm_bwd_kernel<TX, TH, 1, 16, 512>, grid, block, 0, st, true, p);
  else if (s.elems == 16)
    e = vec ? launch_k(norm_bwd_kernel<TX, TH, 8, 2, 1024>, grid, block, 0, st, true, p)
            : launch_k(norm_bwd_kernel<TX, TH, 1, 16, 1024>, grid, block, 0, st, true, p);
  else
    e = vec ? launch_k(norm_bwd_kernel<TX, TH, 8, 4, 1024>, grid, block, 0, st, true, p)
            : launch_k(norm_bwd_kernel<TX, TH, 1, 32, 1024>, grid, block, 0, st, true, p);
  if (e != cudaSuccess || dw == nullptr) return e;
  const dim3 g2((unsigned)((p.cols + 31) / 32)), b2(32, 32);
  const int n = (int)(blocks * s.teams);
  if (dw_f32) return launch_k(norm_dw_kernel<float>, g2, b2, 0, st, true, (const float*)p.partial, n, p.cols, (float*)dw);
  return launch_k(norm_dw_kernel<TX>, g2, b2, 0, st, true, (const float*)p.partial, n, p.cols, (TX*)dw);
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
                 NormParams p, int quant, void* stream) {
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
  p.inv_cols = 1.0f / (float)cols;
  p.sum = sum_out;
  const bool vec = cols % 8 == 0 && vec_ok(x, x_dtype, ldx, rows) && vec_ok(residual, h_dtype, ldr, rows) &&
                   on(weight, 16) && on(sum_out, 16) && on(p.y, quant ? 8 : 16);
  const cudaStream_t st = (cudaStream_t)stream;
  return for_types(x_dtype, h_dtype, [&](auto tx, auto th) {
    using TX = decltype(tx);
    using TH = decltype(th);
    const cudaError_t e = quant == 0   ? launch_fwd<TX, TH, 0>(p, vec, st)
                          : quant == 1 ? launch_fwd<TX, TH, 1>(p, vec, st)
                                       : launch_fwd<TX, TH, 2>(p, vec, st);
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
                      eps, sum_out, p, 0, stream);
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
  p.group = group;
  p.given = given_scale;
  p.scales = scales;
  return forward_call(who, x, x_dtype, ldx, residual, r_dtype, ldr, weight, w_dtype, rows, cols, eps, sum_out, p,
                      q_dtype == GLAD_DTYPE_E4M3 ? 2 : 1, stream);
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
  p.inv_cols = 1.0f / (float)cols;
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
