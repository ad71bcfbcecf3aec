// Global norm over many tensors, and the tensors scaled by it:
//   n = (sum |g|^2)^(1/2), sum |g| or max |g| over all tensors,  c = min(1, max_norm / (n + 1e-6)),  g' = c g
//
// The tensors are cut into chunks; a persistent grid walks the chunks twice, in two kernels (the scalar c needs all
// of them first). Partial results go to fixed places and are added in a fixed order: the same call gives the same bits.
// DRAM bytes are the bound of large calls, launch latency of small ones.
#include "glad_elem.cuh"
#include "tc05.cuh"

namespace glad {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 1280;         // partial results of one launch
constexpr int kBig = 1024, kSmall = 128; // tensors of one launch; the table travels in the kernel's parameters

enum Kind { kInf = 0, kOne = 1, kTwo = 2 };

template <int CAP>
struct Table {
  const void* src[CAP];
  void* dst[CAP];
  int64_t size[CAP];
  int32_t first[CAP + 1];    // first chunk of each tensor; their number at the end
  uint8_t dtype[CAP];
  int32_t n;
  int32_t chunk;             // elements
};
static_assert(sizeof(Table<kBig>) <= 32000, "kernel parameters end at 32764 bytes");

// The tensor that chunk c belongs to.
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& t, int c) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Calls f(value, slot) for the block's elements [p, p + n) that are this thread's: 16-byte loads between the first and the
// last 16-byte boundary, several at once.
template <typename T, typename F>
__device__ __forceinline__ void visit(const T* p, int n, F&& f) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  const int head = off ? min(n, V - off) : 0, vecs = (n - head) / V;
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
  for (int i = threadIdx.x; i < vecs; i += kThreads * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kThreads < vecs) w[u] = q[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kThreads < vecs) {
        Raw<V, T> r = {{w[u].x, w[u].y, w[u].z, w[u].w}};
        float v[V];
        to_floats<V, T>(r, v);
#pragma unroll
        for (int e = 0; e < V; ++e) f(v[e], e);
      }
    }
  }
  const int rest = n - vecs * V;                         // head and tail: fewer than 2 V elements
  if ((int)threadIdx.x < rest) {
    const int i = (int)threadIdx.x < head ? (int)threadIdx.x : vecs * V + (int)threadIdx.x;
    f(to_f<T>(p[i]), 0);
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
  return a;
}

// This thread's part of a chunk's sum (or maximum). A few dozen squares are added in fp32; where they leave its range or
// its precise part, they are added again in 64 bits, so the norm is right for gradients of any magnitude.
template <int KIND, typename T>
__device__ __forceinline__ void add_chunk(const T* p, int n, double& total) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  visit<T>(p, n, [&](float v, int e) {
    if constexpr (KIND == kInf) s[e & 3] = max_nan(s[e & 3], fabsf(v));
    else if constexpr (KIND == kOne) s[e & 3] += fabsf(v);
    else s[e & 3] = fmaf(v, v, s[e & 3]);
  });
  if constexpr (KIND == kInf) {
    total = max_nan((float)total, max_nan(max_nan(s[0], s[1]), max_nan(s[2], s[3])));
  } else {
    const float sum = (s[0] + s[1]) + (s[2] + s[3]);
    if (sum > 1e-25f && sum < 1e30f) {
      total += sum;
    } else {
      double d = 0.0;
      visit<T>(p, n, [&](float v, int) { d += KIND == kOne ? fabs((double)v) : (double)v * v; });
      total += d;
    }
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
__global__ void __launch_bounds__(kThreads) grad_sum_kernel(const __grid_constant__ Table<CAP> t, double* partial) {
  __shared__ double red[kThreads / 32];
  grid_dep_wait();
  double total = 0.0;
  const int chunks = t.first[t.n];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = tensor_of(t, c);
    const int64_t at = (int64_t)(c - t.first[i]) * t.chunk;
    const int n = (int)min((int64_t)t.chunk, t.size[i] - at);
    if (t.dtype[i] == GLAD_DTYPE_F32) add_chunk<KIND>(static_cast<const float*>(t.src[i]) + at, n, total);
    else if (t.dtype[i] == GLAD_DTYPE_F16) add_chunk<KIND>(static_cast<const __half*>(t.src[i]) + at, n, total);
    else add_chunk<KIND>(static_cast<const __nv_bfloat16*>(t.src[i]) + at, n, total);
  }
  total = block_combine<KIND>(total, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// dst = c src (both may be the same). Unlike alignments: elements one by one.
template <typename T>
__device__ __forceinline__ void scale_chunk(const T* p, T* q, int n, float c) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  const bool alike = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15) == 0;
  const int head = alike ? (off ? min(n, V - off) : 0) : n, vecs = (n - head) / V;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  uint4* qv = reinterpret_cast<uint4*>(q + head);
  for (int i = threadIdx.x; i < vecs; i += kThreads * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kThreads < vecs) w[u] = pv[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kThreads < vecs) {
        Raw<V, T> r = {{w[u].x, w[u].y, w[u].z, w[u].w}};
        float v[V];
        to_floats<V, T>(r, v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] *= c;
        if constexpr (sizeof(T) == 4) {
          qv[i + u * kThreads] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                            __float_as_uint(v[3]));
        } else {
          qv[i + u * kThreads] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                            pack2<T>(v[6], v[7]));
        }
      }
    }
  }
  for (int i = threadIdx.x; i < n - vecs * V; i += kThreads) {
    const int at = i < head ? i : vecs * V + i;
    q[at] = from_f<T>(to_f<T>(p[at]) * c);
  }
}

// The norm from the partial results, then every tensor times the coefficient. Tensors written in place are left alone
// where the coefficient is 1. The chunks are walked from the last one: those are still in the L2.
template <int KIND, int CAP>
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ Table<CAP> t, const double* partial,
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
  for (int k = t.first[t.n] - 1 - (int)blockIdx.x; k >= 0; k -= gridDim.x) {
    const int i = tensor_of(t, k);
    if (c == 1.0f && t.src[i] == t.dst[i]) continue;
    const int64_t at = (int64_t)(k - t.first[i]) * t.chunk;
    const int n = (int)min((int64_t)t.chunk, t.size[i] - at);
    if (t.dtype[i] == GLAD_DTYPE_F32)
      scale_chunk(static_cast<const float*>(t.src[i]) + at, static_cast<float*>(t.dst[i]) + at, n, c);
    else if (t.dtype[i] == GLAD_DTYPE_F16)
      scale_chunk(static_cast<const __half*>(t.src[i]) + at, static_cast<__half*>(t.dst[i]) + at, n, c);
    else
      scale_chunk(static_cast<const __nv_bfloat16*>(t.src[i]) + at, static_cast<__nv_bfloat16*>(t.dst[i]) + at, n, c);
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
  int chunk;
};

// Tensors [from, from + CAP) as a table; returns where the next one starts (empty tensors take no place).
template <int CAP>
int fill(Table<CAP>& t, const Call& c, int from) {
  int n = 0;
  int64_t chunks = 0;
  t.first[0] = 0;
  t.chunk = c.chunk;
  for (; from < c.n && n < CAP; ++from) {
    if (c.sizes[from] == 0) continue;
    const int64_t more = (c.sizes[from] + c.chunk - 1) / c.chunk;
    if (chunks + more > 0x7fffffff) break;
    t.src[n] = c.src[from];
    t.dst[n] = c.dst ? c.dst[from] : nullptr;
    t.size[n] = c.sizes[from];
    t.dtype[n] = (uint8_t)c.dtypes[from];
    chunks += more;
    t.first[++n] = (int32_t)chunks;
  }
  t.n = n;
  return from;
}

template <int KIND, int CAP>
cudaError_t launch(const Call& c, cudaStream_t st) {
  int limit = 8 * num_sms();
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
    const int chunks = t.first[t.n], blocks = chunks < 1 ? 1 : chunks < limit ? chunks : limit;
    e = launch_k(grad_scale_kernel<KIND, CAP>, dim3(blocks), dim3(kThreads), 0, st, true, t, (const double*)c.partial,
                 parts, c.max_norm, first ? c.norm : (float*)nullptr);
    first = false;
  }
  return e;
}

template <int KIND>
cudaError_t launch(const Call& c, cudaStream_t st) {
  return c.n <= kSmall ? launch<KIND, kSmall>(c, st) : launch<KIND, kBig>(c, st);
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
    if (sizes[i] < 0 || sizes[i] > (int64_t)1 << 40) return bad(who, "a tensor's size must be in [0, 2^40]");
    if (sizes[i] && (!src[i] || (dst && !dst[i]))) return bad(who, "a tensor is not set");
    if (!on(src[i], width_of(dtypes[i])) || (dst && !on(dst[i], width_of(dtypes[i]))))
      return bad(who, "a tensor is not element-aligned");
    total += sizes[i];
    if (total > (int64_t)1 << 50) return bad(who, "more than 2^50 elements");
  }
  if (!workspace || workspace_bytes < glad_grad_norm_workspace_size(n) || !on(workspace, 8))
    return set_last_error(GLAD_ERR_WORKSPACE, "a workspace of glad_grad_norm_workspace_size bytes is required");
  Call c{src, dst, sizes, dtypes, n, max_norm, norm, static_cast<double*>(workspace), 2048};
  // Chunks of 2048 elements spread small calls over the GPU; larger ones, up to 32768, have less to look up.
  while (c.chunk < 32768 && total / c.chunk > 8 * 1184) c.chunk *= 2;
  while (total / c.chunk > 0x40000000) c.chunk *= 2;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = norm_type == 0 ? launch<kInf>(c, st) : norm_type == 1 ? launch<kOne>(c, st) : launch<kTwo>(c, st);
  return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
}

}  // namespace
}  // namespace glad

using namespace glad;

extern "C" {

size_t glad_grad_norm_workspace_size(int n) {
  const int launches = n <= kSmall ? 1 : (n + kBig - 1) / kBig;
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
  return call("glad_clip_grads", grads, outs ? outs : none, sizes, dtypes, n, norm_type, max_norm, norm, workspace,
              workspace_bytes, stream);
}

}  // extern "C"
