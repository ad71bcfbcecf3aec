// Elements of f32, f16 and bf16 rows: conversions, loads and stores of one or eight of them, and the host-side argument
// checks of the operators on such rows.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../include/glad_b200.h"

namespace glad {
int set_last_error(int code, const char* msg);   // glad_abi.cu

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

// Two elements of a 32-bit word of a 16-bit type (paired conversions: single ones run at a quarter of the rate).
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// VEC consecutive elements as stored, VEC 1 or 8 (8: 16-byte aligned).
template <int VEC, typename T>
struct Raw {
  uint32_t w[VEC == 1 ? 1 : VEC * (int)sizeof(T) / 4];
};
template <int VEC, typename T>
__device__ __forceinline__ void load_raw(const T* p, Raw<VEC, T>& r) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 4) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    else r.w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < (int)(VEC * sizeof(T) / 16); ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    }
  }
}
template <int VEC, typename T>
__device__ __forceinline__ void to_floats(const Raw<VEC, T>& r, float (&f)[VEC]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = __uint_as_float(r.w[i]);
  } else if constexpr (VEC == 1) {
    f[0] = unpack2<T>(r.w[0]).x;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 u = unpack2<T>(r.w[i]);
      f[2 * i] = u.x, f[2 * i + 1] = u.y;
    }
  }
}
template <int VEC, typename T>
__device__ __forceinline__ void load_v(const T* p, float (&f)[VEC]) {
  Raw<VEC, T> r;
  load_raw<VEC, T>(p, r);
  to_floats<VEC, T>(r, f);
}
// Stores f; with ROUND, f becomes what was stored.
template <int VEC, typename T, bool ROUND = false>
__device__ __forceinline__ void store_v(T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    const T v = from_f<T>(f[0]);
    *p = v;
    if (ROUND) f[0] = to_f<T>(v);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
      if (ROUND) {
        const float2 u = unpack2<T>(w[i]);
        f[2 * i] = u.x, f[2 * i + 1] = u.y;
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- launch ---------------------------------------------------------------------------
inline int num_sms() {
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

// ---- argument checks ------------------------------------------------------------------------
inline int bad(const char* who, const char* what) {
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", who, what);
  return set_last_error(GLAD_ERR_INVALID_ARG, msg);
}
inline int cuda_bad(const char* who, cudaError_t e) {
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", who, cudaGetErrorString(e));
  return set_last_error(GLAD_ERR_CUDA, msg);
}
inline size_t width_of(int dtype) { return dtype == GLAD_DTYPE_F32 ? 4 : 2; }
inline bool is_float(int dtype) { return dtype == GLAD_DTYPE_F32 || dtype == GLAD_DTYPE_F16 || dtype == GLAD_DTYPE_BF16; }
inline bool on(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
// A row tensor: element-aligned, rows at least `cols` apart.
inline const char* rows_wrong(const void* p, int dtype, int64_t ld, int64_t rows, int cols) {
  if (!on(p, width_of(dtype))) return "a tensor is not element-aligned";
  if (rows > 1 && ld < cols) return "a row stride is below the number of columns";
  return nullptr;
}
// 8-element accesses: base and row pitch on 16 bytes.
inline bool vec_ok(const void* p, int dtype, int64_t ld, int64_t rows) {
  if (p == nullptr) return true;
  return on(p, 16) && (rows <= 1 || (ld * (int64_t)width_of(dtype)) % 16 == 0);
}

}  // namespace glad
