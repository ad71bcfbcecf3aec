// Log probabilities of given tokens, entropy and the top alternatives of rows of logits, and their gradient:
//   z = (x - max x) / T,  S = sum e^z,  log p_j = z_j - ln S,  H = ln S - sum(e^z z) / S
//   dx_j = [ g [j = t] + sum_i gt_i [j = t_i] - p_j (g + sum gt) - gh p_j (ln p_j + H) ] / T
// Sums and statistics are fp32.
#include "glad_elem.cuh"
#include "tc05.cuh"

namespace glad {
namespace {

constexpr int kMaxTop = 32;

struct LogpParams {
  const void* x;
  const void* tokens;
  int64_t ldx, rows, ignore;
  int cols, top, tok64;
  float inv_t;
  float* logp;
  float* entropy;       // or null
  float* top_logp;      // [rows, top]
  int64_t* top_index;
  float2* stats;        // (max, ln S) or null
};

struct LogpGradParams {
  const void* x;
  const void* tokens;
  int64_t ldx, rows, ignore;
  int cols, top, tok64;
  float inv_t;
  const float* entropy;
  const float2* stats;
  const int64_t* top_index;
  const float* g;       // each or null
  const float* gh;
  const float* gt;
  void* dx;
};

__device__ __forceinline__ int64_t token_of(const void* tokens, int tok64, int64_t row) {
  return tok64 ? static_cast<const int64_t*>(tokens)[row] : (int64_t)static_cast<const int32_t*>(tokens)[row];
}
__device__ __forceinline__ float max_nan(float a, float b) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
  return a;
}
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// Order of the alternatives: the larger value first, the lower column among equals; a NaN before all, -0 equal to 0.
// Never 0, so 0 is "none".
__device__ __forceinline__ uint64_t rank_of(float v, int col) {
  uint32_t u = __float_as_uint(v + 0.0f);
  u = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)~col;
}

template <typename T>
__global__ void __launch_bounds__(256) logp_kernel(const LogpParams p) {
  __shared__ float red[3][8];
  __shared__ uint64_t best[8];
  grid_dep_wait();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const int64_t tok = token_of(p.tokens, p.tok64, row);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tok == p.ignore) {
    if (tid == 0) {
      p.logp[row] = 0.0f;
      if (p.entropy) p.entropy[row] = 0.0f;
      if (p.stats) p.stats[row] = make_float2(0.0f, INFINITY);
    }
    if (tid < p.top) p.top_logp[row * p.top + tid] = 0.0f, p.top_index[row * p.top + tid] = -1;
    return;
  }
  float m = -INFINITY;
  for (int j = tid; j < p.cols; j += 256) m = max_nan(m, to_f<T>(x[j]));
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
  m = red[0][0];
  for (int w = 1; w < 8; ++w) m = max_nan(m, red[0][w]);
  const float k = p.inv_t * kLog2e;
  float s = 0.0f, t = 0.0f;
  for (int j = tid; j < p.cols; j += 256) {
    const float d = to_f<T>(x[j]) - m, e = exp2_fast(d * k);
    s += e;
    t = fmaf(e, fmaxf(d, -1e30f), t);        // e = 0 where d is lower
  }
  s = warp_sum(s);
  t = warp_sum(t);
  if (lane == 0) red[1][warp] = s, red[2][warp] = t;
  __syncthreads();
  s = t = 0.0f;
  for (int w = 0; w < 8; ++w) s += red[1][w], t += red[2][w];
  const bool none = m == -INFINITY;          // every logit is -inf: no distribution
  const float ln_s = none ? INFINITY : logf(s);
  if (tid == 0) {
    const bool in = tok >= 0 && tok < p.cols;
    p.logp[row] = !in ? NAN : none ? -INFINITY : (to_f<T>(x[tok]) - m) * p.inv_t - ln_s;
    if (p.entropy) p.entropy[row] = none ? 0.0f : ln_s - t * p.inv_t / s;
    if (p.stats) p.stats[row] = make_float2(none ? 0.0f : m, ln_s);
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < p.top; ++i) {
    uint64_t b = 0;
    for (int j = tid; j < p.cols; j += 256) {
      const uint64_t r = rank_of(to_f<T>(x[j]), j);
      if (r < last && r > b) b = r;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const uint64_t q = __shfl_xor_sync(0xffffffffu, b, o);
      b = q > b ? q : b;
    }
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    b = best[0];
    for (int w = 1; w < 8; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (tid == 0) {
      const int col = (int)~(uint32_t)b;
      p.top_index[row * p.top + i] = col;
      p.top_logp[row * p.top + i] = none ? -INFINITY : (to_f<T>(x[col]) - m) * p.inv_t - ln_s;
    }
  }
}

// The gradient of column j without the given columns' own terms.
__device__ __forceinline__ float grad_at(float x, float m, float inv_t, float ln_s, float G, float gh, float H) {
  const float l = fmaf(x - m, inv_t, -ln_s), pr = exp2_fast(l * kLog2e);
  const float e = pr == 0.0f ? 0.0f : pr * (l + H);
  return -(pr * G + gh * e);
}

template <typename T>
__global__ void __launch_bounds__(256) logp_grad_kernel(const LogpGradParams p) {
  grid_dep_wait();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  T* dx = static_cast<T*>(p.dx) + row * p.cols;
  const int64_t tok = token_of(p.tokens, p.tok64, row);
  const int tid = threadIdx.x;
  const float2 st = p.stats[row];
  if (st.y == INFINITY) {                    // an ignored row, or one without a distribution
    for (int j = tid; j < p.cols; j += 256) dx[j] = from_f<T>(0.0f);
    return;
  }
  const bool in = tok >= 0 && tok < p.cols;
  float g = p.g ? p.g[row] : 0.0f;
  if (!in && p.g) g = NAN;
  const float gh = p.gh ? p.gh[row] : 0.0f, H = p.gh ? p.entropy[row] : 0.0f;
  float G = g;
  if (p.gt)
    for (int i = 0; i < p.top; ++i) G += p.gt[row * p.top + i];
  for (int j = tid; j < p.cols; j += 256)
    dx[j] = from_f<T>(grad_at(to_f<T>(x[j]), st.x, p.inv_t, st.y, G, gh, H) * p.inv_t);
  __syncthreads();
  const int given = p.gt ? p.top : 0;
  if (tid <= given) {                        // the given columns again, with their own terms
    const int64_t col = tid == given ? tok : p.top_index[row * p.top + tid];
    if (col >= 0 && col < p.cols) {
      float v = grad_at(to_f<T>(x[col]), st.x, p.inv_t, st.y, G, gh, H);
      if (col == tok) v += g;
      for (int i = 0; i < given; ++i)
        if (p.top_index[row * p.top + i] == col) v += p.gt[row * p.top + i];
      dx[col] = from_f<T>(v * p.inv_t);
    }
  }
}

template <typename F>
int for_type(int dtype, F&& f) {
  if (dtype == GLAD_DTYPE_F16) return f(__half());
  if (dtype == GLAD_DTYPE_BF16) return f(__nv_bfloat16());
  return f(float());
}

const char* common_wrong(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t cols, const void* tokens,
                         int tok_bytes, float temperature, int top) {
  if (!is_float(x_dtype)) return "logits must be f32, f16 or bf16";
  if (rows < 0 || rows > 0x7fffffffLL) return "rows must be in [0, 2^31)";
  if (cols < 1 || cols > 1 << 30) return "cols must be in [1, 2^30]";
  if (tok_bytes != 4 && tok_bytes != 8) return "tokens must have 4 or 8 bytes";
  if (!(temperature >= 1e-30f && temperature <= 1e30f)) return "temperature must be in [1e-30, 1e30]";
  if (top < 0 || top > kMaxTop || top > cols) return "top must be in [0, 32] and at most cols";
  if (rows == 0) return nullptr;
  if (!x || !tokens) return "logits and tokens must be set";
  if (!on(tokens, tok_bytes)) return "tokens are not element-aligned";
  return rows_wrong(x, x_dtype, ldx, rows, (int)cols);
}

}  // namespace
}  // namespace glad

using namespace glad;

extern "C" {

int glad_token_log_probs(const void* logits, int x_dtype, int64_t ldx, int64_t rows, int64_t cols, const void* tokens,
                         int token_bytes, int64_t ignore_index, float temperature, int top, float* log_prob,
                         float* entropy, float* top_log_prob, int64_t* top_index, float* stats, void* stream) {
  const char* who = "glad_token_log_probs";
  const char* why = common_wrong(logits, x_dtype, ldx, rows, cols, tokens, token_bytes, temperature, top);
  if (why) return bad(who, why);
  if (rows == 0) return GLAD_OK;
  if (!log_prob || (top && (!top_log_prob || !top_index))) return bad(who, "an output is not set");
  if (!on(log_prob, 4) || !on(entropy, 4) || !on(top_log_prob, 4) || !on(top_index, 8) || !on(stats, 8))
    return bad(who, "an output is not element-aligned");
  LogpParams p{};
  p.x = logits, p.ldx = ldx, p.rows = rows, p.cols = (int)cols, p.tokens = tokens, p.tok64 = token_bytes == 8;
  p.ignore = ignore_index, p.inv_t = 1.0f / temperature, p.top = top;
  p.logp = log_prob, p.entropy = entropy, p.top_logp = top_log_prob, p.top_index = top_index;
  p.stats = reinterpret_cast<float2*>(stats);
  return for_type(x_dtype, [&](auto t) {
    const cudaError_t e = launch_k(logp_kernel<decltype(t)>, dim3((unsigned)rows), dim3(256), 0, (cudaStream_t)stream,
                                   true, p);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  });
}

int glad_token_log_probs_backward(const void* logits, int x_dtype, int64_t ldx, int64_t rows, int64_t cols,
                                  const void* tokens, int token_bytes, int64_t ignore_index, float temperature, int top,
                                  const float* stats, const float* entropy, const int64_t* top_index, const float* d_log_prob,
                                  const float* d_entropy, const float* d_top, void* d_logits, void* stream) {
  const char* who = "glad_token_log_probs_backward";
  const char* why = common_wrong(logits, x_dtype, ldx, rows, cols, tokens, token_bytes, temperature, top);
  if (why) return bad(who, why);
  if (rows == 0) return GLAD_OK;
  if (!stats || !d_logits) return bad(who, "stats and d_logits must be set");
  if (d_entropy && !entropy) return bad(who, "d_entropy needs entropy");
  if (d_top && (!top || !top_index)) return bad(who, "d_top needs top and top_index");
  if (!on(stats, 8) || !on(entropy, 4) || !on(top_index, 8) || !on(d_log_prob, 4) || !on(d_entropy, 4) || !on(d_top, 4) ||
      !on(d_logits, width_of(x_dtype)))
    return bad(who, "a tensor is not element-aligned");
  LogpGradParams p{};
  p.x = logits, p.ldx = ldx, p.rows = rows, p.cols = (int)cols, p.tokens = tokens, p.tok64 = token_bytes == 8;
  p.ignore = ignore_index, p.inv_t = 1.0f / temperature, p.top = top;
  p.stats = reinterpret_cast<const float2*>(stats), p.entropy = entropy, p.top_index = top_index;
  p.g = d_log_prob, p.gh = d_entropy, p.gt = d_top, p.dx = d_logits;
  return for_type(x_dtype, [&](auto t) {
    const cudaError_t e = launch_k(logp_grad_kernel<decltype(t)>, dim3((unsigned)rows), dim3(256), 0,
                                   (cudaStream_t)stream, true, p);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  });
}

}  // extern "C"
