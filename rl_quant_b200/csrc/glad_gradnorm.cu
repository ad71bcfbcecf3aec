// Global norm over many tensors, and the tensors scaled by it:
//   n = (sum |g|^2)^(1/2), sum |g| or max |g| over all tensors,  c = min(1, max_norm / (n + 1e-6)),  g' = c g
//
// The tensors are cut into units of 2048 elements, and a block takes a run of neighbouring units, twice, in two kernels (the
// scalar c needs all of them first): forwards for the sums, backwards to scale, so that what it read last is still in the L2.
// Partial results go to fixed places and are added in a fixed order: the same call gives the same bits. DRAM bytes are the
// bound of large calls, launch latency of small ones: 268 M bf16 elements in 290 tensors, clipped, 271 us, 1.61 GB read and written, 5.9 TB/s
// (1.07 GB would do if a first reading could stay on the chip: 164 us); 20 M in 448 within the limit 16.2 us, 40 MB; 613 K f32 in 39
// tensors 6.2 us, two launches.
#include "glad_elem.cuh"
#include "tc05.cuh"

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

namespace glad {
namespace {

constexpr int kThreads = 256, kPerSm = 4;
constexpr int kMaxBlocks = 640;          // partial results of one launch
constexpr int kUnit = 2048;              // elements; a call of few units has as many blocks, so small calls spread too
constexpr int kMost = 1024;              // tensors of one launch; the table travels in the kernel's parameters

enum Kind { kInf = 0, kOne = 1, kTwo = 2 };

template <int CAP>
struct Table {
  const void* src[CAP];
  void* dst[CAP];
  int64_t size[CAP];
  int32_t first[CAP + 1];    // first unit of each tensor; their number at the end
  uint8_t dtype[CAP];
  int32_t n;
};
static_assert(sizeof(Table<kMost>) <= 32000, "kernel parameters end at 32764 bytes");

// The tensor that unit u belongs to.
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& t, int u) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}
// Where block b's run of units starts.
template <int CAP>
__device__ __forceinline__ int first_unit(const Table<CAP>& t, unsigned b) {
  return (int)((int64_t)t.first[t.n] * b / gridDim.x);
}
// Calls f(pointer type, tensor, first element, elements) for the part of tensor i in units [lo, hi).
template <int CAP, typename F>
__device__ __forceinline__ void part_of(const Table<CAP>& t, int i, int lo, int hi, F&& f) {
  const int u0 = max(lo, t.first[i]) - t.first[i], u1 = min(hi, t.first[i + 1]) - t.first[i];
  const int64_t at = (int64_t)u0 * kUnit;
  const int n = (int)(min((int64_t)u1 * kUnit, t.size[i]) - at);
  if (t.dtype[i] == GLAD_DTYPE_F32) f(float(), at, n);
  else if (t.dtype[i] == GLAD_DTYPE_F16) f(__half(), at, n);
  else f(__nv_bfloat16(), at, n);
}

// Elements [p, p + n): head before the first 16-byte boundary, 16-byte pieces, and a tail.
template <typename T>
struct Cut {
  static constexpr int V = 16 / (int)sizeof(T);
  int head, vecs, rest;
  __device__ Cut(const T* p, int n) {
    const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    head = off ? min(n, V - off) : 0;
    vecs = (n - head) / V;
    rest = n - vecs * V;
  }
  __device__ int single(int i) const { return i < head ? i : vecs * V + i; }
};
constexpr int kBatch = 4;                // pieces a thread loads at once

__device__ __forceinline__ float max_nan(float a, float b) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
  return a;
}

// N values more. Squares (and magnitudes) of a few dozen are added in fp32; where they leave its range or its precise part, they
// are added again in 64 bits, so the norm is right for gradients of any magnitude. Between them the sums are 64-bit.
template <int KIND, int N>
__device__ __forceinline__ void add_values(const float (&v)[N], double& total) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < N; ++e) {
    if constexpr (KIND == kInf) s[e & 3] = max_nan(s[e & 3], fabsf(v[e]));
    else if constexpr (KIND == kOne) s[e & 3] += fabsf(v[e]);
    else s[e & 3] = fmaf(v[e], v[e], s[e & 3]);
  }
  if constexpr (KIND == kInf) {
    total = max_nan((float)total, max_nan(max_nan(s[0], s[1]), max_nan(s[2], s[3])));
  } else {
    const float sum = (s[0] + s[1]) + (s[2] + s[3]);
    if (sum > 1e-25f && sum < 1e30f) {
      total += sum;
    } else {
#pragma unroll 1
      for (int e = 0; e < N; e += 4) {
#pragma unroll
        for (int i = 0; i < 4 && i < N; ++i) {
          float x = v[i];
#pragma unroll
          for (int k = 4; k < N; k += 4) x = e == k ? v[k + i] : x;
          total += KIND == kOne ? fabs((double)x) : (double)x * x;
        }
      }
    }
  }
}

template <int KIND, typename T>
__device__ __forceinline__ void add_part(const T* p, int n, double& total) {
  constexpr int V = Cut<T>::V;
  const Cut<T> cut(p, n);
  const uint4* q = reinterpret_cast<const uint4*>(p + cut.head);
  for (int i = threadIdx.x; i < cut.vecs; i += kThreads * kBatch) {
    uint4 w[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) w[u] = i + u * kThreads < cut.vecs ? q[i + u * kThreads] : make_uint4(0, 0, 0, 0);
    float v[kBatch * V];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const Raw<V, T> r = {{w[u].x, w[u].y, w[u].z, w[u].w}};
      float f[V];
      to_floats<V, T>(r, f);
#pragma unroll
      for (int e = 0; e < V; ++e) v[u * V + e] = f[e];
    }
    add_values<KIND>(v, total);
  }
  if ((int)threadIdx.x < cut.rest) {
    const float v[1] = {to_f<T>(p[cut.single(threadIdx.x)])};
    add_values<KIND>(v, total);
  }
}

template <int KIND>
__device__ __forceinline__ double combine(double a, double b) {
  if constexpr (KIND == kInf) return max_nan((float)a, (float)b);
  else return a + b;
}

// Over the block, in a fixed order; the result in thread 0 (all: in every thread).
template <int KIND>
__device__ __forceinline__ double block_combine(double v, double* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = combine<KIND>(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = combine<KIND>(v, red[w]);
  return v;
}

template <int KIND, int CAP>
__global__ void __launch_bounds__(kThreads, kPerSm) grad_sum_kernel(const __grid_constant__ Table<CAP> t, double* partial) {
  __shared__ double red[kThreads / 32];
  grid_dep_wait();
  double total = 0.0;
  const int lo = first_unit(t, blockIdx.x), hi = first_unit(t, blockIdx.x + 1);
  for (int i = tensor_of(t, lo); i < t.n && t.first[i] < hi; ++i)
    part_of(t, i, lo, hi, [&](auto type, int64_t at, int n) {
      add_part<KIND>(static_cast<const decltype(type)*>(t.src[i]) + at, n, total);
    });
  total = block_combine<KIND>(total, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// q = c p (both may be the same), the last pieces first. Unlike alignments: elements one by one.
template <typename T>
__device__ __forceinline__ void scale_part(const T* p, T* q, int n, float c) {
  constexpr int V = Cut<T>::V;
  Cut<T> cut(p, n);
  if (((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15) != 0) cut.head = cut.rest = n, cut.vecs = 0;
  const uint4* pv = reinterpret_cast<const uint4*>(p + cut.head);
  uint4* qv = reinterpret_cast<uint4*>(q + cut.head);
  for (int b = (cut.vecs - 1) / (kThreads * kBatch) * (kThreads * kBatch); b >= 0; b -= kThreads * kBatch) {
    const int i = b + threadIdx.x;
    uint4 w[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (i + u * kThreads < cut.vecs) w[u] = pv[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (i + u * kThreads >= cut.vecs) continue;
      const Raw<V, T> r = {{w[u].x, w[u].y, w[u].z, w[u].w}};
      float v[V];
      to_floats<V, T>(r, v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] *= c;
      if constexpr (sizeof(T) == 4)
        qv[i + u * kThreads] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      else
        qv[i + u * kThreads] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
  }
  for (int i = threadIdx.x; i < cut.rest; i += kThreads) q[cut.single(i)] = from_f<T>(to_f<T>(p[cut.single(i)]) * c);
}

// The norm from the partial results, then every tensor times the coefficient. Tensors written in place are left alone
// where the coefficient is 1.
template <int KIND, int CAP>
__global__ void __launch_bounds__(kThreads, kPerSm) grad_scale_kernel(const __grid_constant__ Table<CAP> t, const double* partial,
                                                                      int parts, float max_norm, float* norm_out) {
  __shared__ double red[kThreads / 32];
  grid_dep_wait();
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) v = combine<KIND>(v, partial[i]);
  v = block_combine<KIND>(v, red);
  const float norm = KIND == kTwo ? (float)sqrt(v) : (float)v;
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  float c = max_norm / (norm + 1e-6f);
  c = c > 1.0f ? 1.0f : c;                               // a NaN stays
  const int lo = first_unit(t, blockIdx.x), hi = first_unit(t, blockIdx.x + 1);
  if (lo >= hi) return;
  for (int i = tensor_of(t, hi - 1); i >= 0 && t.first[i + 1] > lo; --i) {
    if (c == 1.0f && t.src[i] == t.dst[i]) continue;
    part_of(t, i, lo, hi, [&](auto type, int64_t at, int n) {
      using T = decltype(type);
      scale_part(static_cast<const T*>(t.src[i]) + at, static_cast<T*>(t.dst[i]) + at, n, c);
    });
  }
}

struct Call {
  const void* const* src;
  void* const* dst;          // null: the norm only
  const int64_t* sizes;
  const int32_t* dtypes;
  int n;
  float max_norm;
  float* norm;
  double* partial;
};

// Tensors [from, from + CAP) as a table; returns where the next one starts (empty tensors take no place).
template <int CAP>
int fill(Table<CAP>& t, const Call& c, int from) {
  int n = 0;
  int64_t units = 0;
  t.first[0] = 0;
  for (; from < c.n && n < CAP; ++from) {
    if (c.sizes[from] == 0) continue;
    units += (c.sizes[from] + kUnit - 1) / kUnit;
    t.src[n] = c.src[from];
    t.dst[n] = c.dst ? c.dst[from] : nullptr;
    t.size[n] = c.sizes[from];
    t.dtype[n] = (uint8_t)c.dtypes[from];
    t.first[++n] = (int32_t)units;
  }
  t.n = n;
  return from;
}

template <int KIND, int CAP>
cudaError_t launch(const Call& c, cudaStream_t st) {
  int limit = kPerSm * num_sms();
  if (limit > kMaxBlocks) limit = kMaxBlocks;
  Table<CAP> t;
  int parts = 0;
  cudaError_t e = cudaSuccess;
  for (int at = 0; at < c.n && e == cudaSuccess;) {
    at = fill(t, c, at);
    if (t.n == 0) break;
    const int blocks = t.first[t.n] < limit ? t.first[t.n] : limit;
    e = launch_k(grad_sum_kernel<KIND, CAP>, dim3(blocks), dim3(kThreads), 0, st, true, t, c.partial + parts);
    parts += blocks;
  }
  bool first = true;
  for (int at = 0; e == cudaSuccess && (first || (c.dst && at < c.n));) {
    if (c.dst) {
      at = fill(t, c, at);
    } else {
      t.n = 0;
      t.first[0] = 0;
    }
    if (!first && t.n == 0) break;
    const int units = t.first[t.n], blocks = units < 1 ? 1 : units < limit ? units : limit;
    e = launch_k(grad_scale_kernel<KIND, CAP>, dim3(blocks), dim3(kThreads), 0, st, true, t, (const double*)c.partial,
                 parts, c.max_norm, first ? c.norm : (float*)nullptr);
    first = false;
  }
  return e;
}

template <int KIND>
cudaError_t launch(const Call& c, cudaStream_t st) {
  // a table no larger than needed: its bytes are part of a launch
  return c.n <= 64 ? launch<KIND, 64>(c, st) : c.n <= 320 ? launch<KIND, 320>(c, st) : launch<KIND, kMost>(c, st);
}

// Whether a tensor that is written (or read) lies over another one; dst[i] may be src[i].
bool shared(const void* const* src, void* const* dst, const int64_t* sizes, const int32_t* dtypes, int n) {
  std::vector<std::pair<uintptr_t, uintptr_t>> blocks;
  blocks.reserve(2 * (size_t)n);
  for (int i = 0; i < n; ++i) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(src[i]), b = reinterpret_cast<uintptr_t>(dst[i]);
    const uintptr_t bytes = (uintptr_t)sizes[i] * width_of(dtypes[i]);
    if (bytes == 0) continue;
    blocks.emplace_back(a, a + bytes);
    if (a != b) blocks.emplace_back(b, b + bytes);
  }
  std::sort(blocks.begin(), blocks.end());
  for (size_t i = 1; i < blocks.size(); ++i)
    if (blocks[i].first < blocks[i - 1].second) return true;
  return false;
}

int call(const char* who, const void* const* src, void* const* dst, const int64_t* sizes, const int32_t* dtypes, int n,
         int norm_type, float max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (n < 0 || (n > 0 && (!src || !sizes || !dtypes))) return bad(who, "the tables must be set and n >= 0");
  if (norm_type < 0 || norm_type > 2) return bad(who, "norm_type must be 0 (maximum), 1 or 2");
  if (!norm || !on(norm, 4)) return bad(who, "norm must be set and 4-byte aligned");
  if (dst && !(max_norm >= 0.0f)) return bad(who, "max_norm must be >= 0");
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    if (!is_float(dtypes[i])) return bad(who, "a tensor is not f32, f16 or bf16");
    if (sizes[i] < 0 || sizes[i] > (int64_t)1 << 38) return bad(who, "a tensor's size must be in [0, 2^38]");
    if (sizes[i] && (!src[i] || (dst && !dst[i]))) return bad(who, "a tensor is not set");
    if (!on(src[i], width_of(dtypes[i])) || (dst && !on(dst[i], width_of(dtypes[i]))))
      return bad(who, "a tensor is not element-aligned");
    total += sizes[i];
    if (total > (int64_t)1 << 38) return bad(who, "more than 2^38 elements");
  }
  if (dst && shared(src, dst, sizes, dtypes, n)) return bad(who, "two of the tensors share memory");
  if (!workspace || workspace_bytes < glad_grad_norm_workspace_size(n) || !on(workspace, 8))
    return set_last_error(GLAD_ERR_WORKSPACE, "a workspace of glad_grad_norm_workspace_size bytes is required");
  const Call c{src, dst, sizes, dtypes, n, max_norm, norm, static_cast<double*>(workspace)};
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = norm_type == 0 ? launch<kInf>(c, st) : norm_type == 1 ? launch<kOne>(c, st) : launch<kTwo>(c, st);
  return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
}

}  // namespace
}  // namespace glad

using namespace glad;

extern "C" {

size_t glad_grad_norm_workspace_size(int n) {
  const int launches = (n + kMost - 1) / kMost;
  return (size_t)(launches + 1) * kMaxBlocks * sizeof(double);
}

int glad_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int n, int norm_type,
                   float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  return call("glad_grad_norm", grads, nullptr, sizes, dtypes, n, norm_type, 0.0f, norm, workspace, workspace_bytes,
              stream);
}

int glad_clip_grads(const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* dtypes, int n,
                    int norm_type, float max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (n > 0 && !outs) return bad("glad_clip_grads", "outs must be set");
  static void* const none[1] = {nullptr};
  try {
    return call("glad_clip_grads", grads, outs ? outs : none, sizes, dtypes, n, norm_type, max_norm, norm, workspace,
                workspace_bytes, stream);
  } catch (const std::bad_alloc&) {
    return bad("glad_clip_grads", "out of host memory");
  }
}

}  // extern "C"
