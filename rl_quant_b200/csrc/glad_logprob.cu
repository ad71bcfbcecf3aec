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
  int cols, top, tok64, cluster;
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
  int cols, top, tok64, chunks;
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

// The value back (-0 as 0, any NaN as one).
__device__ __forceinline__ float value_of(uint64_t rank) {
  const uint32_t u = (uint32_t)(rank >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// max, sum of e^z and sum of e^z d (d = x - max) of some of a row's logits, z = d / T.
struct Stats {
  float m, s, t;
};
// Log probability of logit x.
__device__ __forceinline__ float log_of(float x, const Stats& v, float ln_s, float inv_t) {
  return v.m == -INFINITY ? -INFINITY : (x - v.m) * inv_t - ln_s;
}
// ln S: -> inf where every logit is -inf (no distribution), NaN where one is +inf.
__device__ __forceinline__ float ln_sum(const Stats& v) {
  return v.m == -INFINITY ? INFINITY : v.m == INFINITY ? NAN : logf(v.s);
}
// d = x - m; a masked logit's stays finite, so that it adds e^z d = 0.
__device__ __forceinline__ float below(float x, float m) { return fmaxf(x - m, -1e30f); }

// v's sums relative to the larger maximum m (k = log2(e) / T).
__device__ __forceinline__ void raise(Stats& v, float m, float k) {
  m = max_nan(v.m, m);                         // a NaN on either side stays
  if (!(v.m >= m)) {
    const float d = below(v.m, m), f = exp2_fast(d * k);
    v.t = v.s == 0.0f ? 0.0f : f * fmaf(v.s, d, v.t);
    v.s = v.m == -INFINITY ? 0.0f : v.s * f;
    v.m = m;
  }
}

template <typename T>
__device__ __forceinline__ void write_row(const LogpParams& p, int64_t row, const T* x, int64_t tok, const Stats& v) {
  const float ln_s = ln_sum(v);
  p.logp[row] = tok >= 0 && tok < p.cols ? log_of(to_f<T>(x[tok]), v, ln_s, p.inv_t) : NAN;
  if (p.entropy) p.entropy[row] = v.m == -INFINITY ? 0.0f : ln_s - v.t * p.inv_t / v.s;
  if (p.stats) p.stats[row] = make_float2(v.m == -INFINITY ? 0.0f : v.m, ln_s);
}
__device__ __forceinline__ void write_top(const LogpParams& p, int64_t row, int i, uint64_t rank, const Stats& v) {
  p.top_index[row * p.top + i] = (int64_t)(int)~(uint32_t)rank;
  p.top_logp[row * p.top + i] = log_of(value_of(rank), v, ln_sum(v), p.inv_t);
}
__device__ __forceinline__ void write_ignored(const LogpParams& p, int64_t row, int i) {
  if (i == 0) {
    p.logp[row] = 0.0f;
    if (p.entropy) p.entropy[row] = 0.0f;
    if (p.stats) p.stats[row] = make_float2(0.0f, INFINITY);
  }
  if (i < p.top) p.top_logp[row * p.top + i] = 0.0f, p.top_index[row * p.top + i] = -1;
}

// ---- rows of up to 1024 columns: a warp each ---------------------------------------------------
// A lane holds E elements of a row, 16-byte pieces (VEC) or every 32nd. NR rows of a warp are loaded before the first is
// used: with one row a warp has 16 bytes a lane in flight and the row's latency (two shuffle trees) is not covered.
template <typename T, int E, bool VEC>
__device__ __forceinline__ int col_of(int e, int lane) {
  constexpr int EL = 16 / (int)sizeof(T);
  return VEC ? (e / EL * 32 + lane) * EL + e % EL : e * 32 + lane;
}
template <typename T, int E, bool VEC>
__device__ __forceinline__ void load_row(const T* x, int cols, int lane, bool on, float (&f)[E]) {
  constexpr int EL = 16 / (int)sizeof(T);
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < E / EL; ++j) {
      const int col = (j * 32 + lane) * EL;
      float v[EL];
      if (on && col < cols) {
        const uint4 w = *reinterpret_cast<const uint4*>(x + col);
        const Raw<EL, T> r = {{w.x, w.y, w.z, w.w}};
        to_floats<EL, T>(r, v);
      } else {
#pragma unroll
        for (int e = 0; e < EL; ++e) v[e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < EL; ++e) f[j * EL + e] = v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = on && e * 32 + lane < cols ? to_f<T>(x[e * 32 + lane]) : -INFINITY;
  }
}

template <typename T, int E, int NR, bool VEC>
__global__ void __launch_bounds__(256) logp_warp_kernel(const LogpParams p) {
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * NR;
  float f[NR][E];
  int64_t tok[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) tok[r] = row0 + r < p.rows ? token_of(p.tokens, p.tok64, row0 + r) : p.ignore;
#pragma unroll
  for (int r = 0; r < NR; ++r)
    load_row<T, E, VEC>(static_cast<const T*>(p.x) + (row0 + r) * p.ldx, p.cols, lane, tok[r] != p.ignore, f[r]);
  const float k = p.inv_t * kLog2e;
  Stats v[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float m = f[r][0];
#pragma unroll
    for (int e = 1; e < E; ++e) m = max_nan(m, f[r][e]);
    v[r].m = m;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int r = 0; r < NR; ++r) v[r].m = max_nan(v[r].m, __shfl_xor_sync(0xffffffffu, v[r].m, o));
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const float m = v[r].m == -INFINITY ? 0.0f : v[r].m;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = below(f[r][e], m), x = exp2_fast(d * k);
      s += x;
      t = fmaf(x, d, t);
    }
    v[r].s = s, v[r].t = t;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      v[r].s += __shfl_xor_sync(0xffffffffu, v[r].s, o);
      v[r].t += __shfl_xor_sync(0xffffffffu, v[r].t, o);
    }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int64_t row = row0 + r;
    if (row >= p.rows) break;
    if (tok[r] == p.ignore) {
      write_ignored(p, row, lane);
      continue;
    }
    if (v[r].m != v[r].m) v[r].s = v[r].t = NAN;
    if (lane == 0) write_row<T>(p, row, static_cast<const T*>(p.x) + row * p.ldx, tok[r], v[r]);
    if (p.top) {
      // rounds of: every lane's best that is not taken, the best of those, the lowest column among equals
      uint32_t taken = 0;
      for (int i = 0; i < p.top; ++i) {
        uint64_t best = 0;
        int at = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int col = col_of<T, E, VEC>(e, lane);
          const uint64_t q = rank_of(f[r][e], col);
          if (q > best && !(taken >> e & 1) && col < p.cols) best = q, at = e;
        }
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        const uint64_t won = (uint64_t)hi << 32 | lo;
        if (best == won) taken |= 1u << at;
        if (lane == i) write_top(p, row, i, won, v[r]);
      }
    }
  }
}

// ---- longer rows: a block or a cluster of blocks each ------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kCandidates = 1024;

// The 16-byte pieces of a row that are this block's, and its single elements before and behind them.
template <typename T>
struct Slice {
  static constexpr int EL = 16 / (int)sizeof(T);
  const T* x;
  const uint4* body;
  int head, vecs, lo, hi, extra;      // pieces lo <= i < hi; extra: single elements, of the first block
  __device__ Slice(const T* row, int cols, int rank, int blocks) : x(row) {
    const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = off ? min(cols, EL - off) : 0;
    vecs = (cols - head) / EL;
    body = reinterpret_cast<const uint4*>(row + head);
    const int per = (vecs + blocks - 1) / blocks;
    lo = min(vecs, rank * per), hi = min(vecs, lo + per);
    extra = rank == 0 ? cols - vecs * EL : 0;
  }
  __device__ int extra_col(int i) const { return i < head ? i : vecs * EL + i; }
};
template <typename T>
__device__ __forceinline__ uint4 masked_piece() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}
template <typename T>
__device__ __forceinline__ void piece(const uint4& w, float (&f)[16 / sizeof(T)]) {
  constexpr int EL = 16 / (int)sizeof(T);
  const Raw<EL, T> r = {{w.x, w.y, w.z, w.w}};
  to_floats<EL, T>(r, f);
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

struct RowShared {
  float red[kRowThreads / 32];
  float red2[2][kRowThreads / 32];
  Stats part;                         // this block's share of the row
  int count;
  uint32_t bar;                       // the threads' k-th largest maximum
  uint32_t keys[kRowThreads];
  uint64_t best[kRowThreads / 32];
  uint64_t top[kMaxTop];
  uint64_t list[kCandidates];
};

__device__ __forceinline__ uint64_t block_max(uint64_t v, RowShared& sh) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t q = __shfl_xor_sync(0xffffffffu, v, o);
    v = q > v ? q : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.best[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.best[0];
#pragma unroll
  for (int w = 1; w < kRowThreads / 32; ++w) v = sh.best[w] > v ? sh.best[w] : v;
  return v;
}

// This thread's best element that ranks below `last`. Elements come in rising columns, so the first of the value of `last` ends it.
template <typename T>
__device__ uint64_t next_best(const Slice<T>& sl, uint64_t last) {
  uint64_t best = 0;
  for (int i = sl.lo + threadIdx.x; i < sl.hi; i += kRowThreads) {
    float f[Slice<T>::EL];
    piece<T>(sl.body[i], f);
#pragma unroll
    for (int e = 0; e < Slice<T>::EL; ++e) {
      const uint64_t q = rank_of(f[e], sl.head + i * Slice<T>::EL + e);
      if (q < last && q > best) best = q;
    }
    if (best >> 32 == last >> 32) break;
  }
  if ((int)threadIdx.x < sl.extra) {
    const int col = sl.extra_col(threadIdx.x);
    const uint64_t q = rank_of(to_f<T>(sl.x[col]), col);
    if (q < last && q > best) best = q;
  }
  return best;
}

// The block's `top` first elements of its slice into sh.top (0: none), sorted. `m` is the thread's largest logit. At least `top` threads
// (all that have elements, if fewer) reach the top-th largest of the threads' maxima, so what lies below it is out, and only the
// threads at or above it look at their elements again. More candidates than the list holds (many equal ones): one by one.
template <typename T>
__device__ __forceinline__ void block_top(const Slice<T>& sl, int top, float m, RowShared& sh) {
  const int tid = threadIdx.x, lane = tid & 31;
  const bool some = sl.lo + tid < sl.hi || tid < sl.extra;
  const uint32_t key = some ? (uint32_t)(rank_of(m, 0) >> 32) : 0u;
  sh.keys[tid] = key;
  if (tid == 0) sh.count = 0;
  if (tid < kMaxTop) sh.top[tid] = 0;
  __syncthreads();
  if (tid < 32) {
    uint32_t k[kRowThreads / 32], bar = 0;
#pragma unroll
    for (int i = 0; i < kRowThreads / 32; ++i) k[i] = sh.keys[i * 32 + lane];
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {           // the largest value that `top` maxima reach
      const uint32_t c = bar | 1u << bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kRowThreads / 32; ++i) n += k[i] >= c;
      if (__reduce_add_sync(0xffffffffu, n) >= top) bar = c;
    }
    if (lane == 0) sh.bar = bar;
  }
  __syncthreads();
  const uint32_t bar = sh.bar;
  if (some && key >= bar) {
    auto offer = [&](float v, int col) {
      const uint64_t q = rank_of(v, col);
      if ((uint32_t)(q >> 32) >= bar) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kCandidates) sh.list[at] = q;
      }
    };
#pragma unroll 2
    for (int i = sl.lo + tid; i < sl.hi; i += kRowThreads) {
      float f[Slice<T>::EL];
      piece<T>(sl.body[i], f);
#pragma unroll
      for (int e = 0; e < Slice<T>::EL; ++e) offer(f[e], sl.head + i * Slice<T>::EL + e);
    }
    if (tid < sl.extra) offer(to_f<T>(sl.x[sl.extra_col(tid)]), sl.extra_col(tid));
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= kCandidates) {
    for (int i = tid; i < n; i += kRowThreads) {
      const uint64_t q = sh.list[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += sh.list[j] > q;
      if (before < top) sh.top[before] = q;
    }
  } else {
    uint64_t mine = next_best(sl, ~0ull);
    for (int i = 0; i < top; ++i) {
      const uint64_t won = block_max(mine, sh);
      if (won == 0) break;
      if (tid == 0) sh.top[i] = won;
      if (mine == won) mine = next_best(sl, won);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logp_row_kernel(const LogpParams p) {
  constexpr int EL = Slice<T>::EL, U = 4;
  __shared__ RowShared sh;
  grid_dep_wait();
  const int C = p.cluster, rank = (int)(blockIdx.x % (unsigned)C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / (unsigned)C;
  const int64_t tok = token_of(p.tokens, p.tok64, row);
  if (tok == p.ignore) {                               // all blocks of the row
    if (rank == 0) write_ignored(p, row, tid);
    return;
  }
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const Slice<T> sl(x, p.cols, rank, C);
  const float k = p.inv_t * kLog2e;
  Stats v = {-INFINITY, 0.0f, 0.0f};
  if (tid < sl.extra) v = {to_f<T>(x[sl.extra_col(tid)]), 1.0f, 0.0f};
  if (v.m == -INFINITY) v.s = 0.0f;
  for (int i = sl.lo + tid; i < sl.hi; i += kRowThreads * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = i + u * kRowThreads < sl.hi ? sl.body[i + u * kRowThreads] : masked_piece<T>();
    float f[U * EL];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float g[EL];
      piece<T>(w[u], g);
#pragma unroll
      for (int e = 0; e < EL; ++e) f[u * EL + e] = g[e];
    }
    float m = f[0];
#pragma unroll
    for (int e = 1; e < U * EL; ++e) m = max_nan(m, f[e]);
    raise(v, m, k);
    const float base = v.m == -INFINITY ? 0.0f : v.m;
    float s0 = 0.0f, s1 = 0.0f, t0 = 0.0f, t1 = 0.0f;
#pragma unroll
    for (int e = 0; e < U * EL; e += 2) {
      const float d0 = below(f[e], base), d1 = below(f[e + 1], base), e0 = exp2_fast(d0 * k), e1 = exp2_fast(d1 * k);
      s0 += e0, s1 += e1;
      t0 = fmaf(e0, d0, t0), t1 = fmaf(e1, d1, t1);
    }
    v.s += s0 + s1, v.t += t0 + t1;
  }
  const float own = v.m;
  float m = v.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sh.red[warp] = m;
  __syncthreads();
  m = sh.red[0];
#pragma unroll
  for (int i = 1; i < kRowThreads / 32; ++i) m = max_nan(m, sh.red[i]);
  raise(v, m, k);
  v.s = warp_sum(v.s);
  v.t = warp_sum(v.t);
  if (lane == 0) sh.red2[0][warp] = v.s, sh.red2[1][warp] = v.t;
  __syncthreads();
  if (tid == 0) {
    v.s = v.t = 0.0f;
    for (int i = 0; i < kRowThreads / 32; ++i) v.s += sh.red2[0][i], v.t += sh.red2[1][i];
    sh.part = v;
  }
  if (p.top) block_top<T>(sl, p.top, own, sh);
  if (C == 1) {
    __syncthreads();
    const Stats all = sh.part;
    if (tid == 0) write_row<T>(p, row, x, tok, all);
    if (tid < p.top) write_top(p, row, tid, sh.top[tid], all);
    return;
  }
  cluster_sync_all();
  if (rank == 0) {
    // the blocks' parts, in their order; the first of all their firsts
    Stats all = sh.part;
    const uint32_t here = smem_u32(&sh.part), tops = smem_u32(sh.top);
    float parts[8][3];
    for (int c = 1; c < C; ++c) {
      const uint32_t a = mapa_shared(here, c);
#pragma unroll
      for (int i = 0; i < 3; ++i) parts[c][i] = __uint_as_float(ld_cluster_u32(a + 4 * i));
    }
    for (int c = 1; c < C; ++c) {
      Stats u = {parts[c][0], parts[c][1], parts[c][2]};
      raise(all, u.m, k);
      raise(u, all.m, k);
      all.s += u.s, all.t += u.t;
    }
    if (tid == 0) write_row<T>(p, row, x, tok, all);
    if (p.top) {
      const int n = C * p.top;                         // at most 256: one a thread
      uint64_t q = 0;
      if (tid < n) {
        const uint32_t a = mapa_shared(tops + 8 * (tid % p.top), tid / p.top);
        q = (uint64_t)ld_cluster_u32(a + 4) << 32 | ld_cluster_u32(a);
      }
      sh.list[tid] = q;
      __syncthreads();
      if (q) {
        int before = 0;
        for (int j = 0; j < n; ++j) before += sh.list[j] > q;
        if (before < p.top) write_top(p, row, before, q, all);
      }
    }
  }
  cluster_sync_all();
}

// ---- gradient ----------------------------------------------------------------------------------
struct RowGrad {
  float m, ln_s, G, gh, H, inv_t;
  // of a logit's column without the given columns' own terms
  __device__ __forceinline__ float at(float x) const {
    const float l = fmaf(x - m, inv_t, -ln_s), pr = exp2_fast(l * kLog2e);
    return -pr * fmaf(gh, fmaxf(l, -200.0f) + H, G) * inv_t;     // p = 0 below -88
  }
};
__device__ __forceinline__ bool given_in(int64_t tok, int cols) { return tok >= 0 && tok < cols; }

__device__ __forceinline__ RowGrad row_grad(const LogpGradParams& p, int64_t row, int64_t tok) {
  const float2 st = p.stats[row];
  RowGrad r{st.x, st.y, p.g ? p.g[row] : 0.0f, p.gh ? p.gh[row] : 0.0f, p.gh ? p.entropy[row] : 0.0f, p.inv_t};
  if (!given_in(tok, p.cols) && p.g) r.G = NAN;
  if (p.gt)
    for (int i = 0; i < p.top; ++i) r.G += p.gt[row * p.top + i];
  return r;
}
// Column number i of the row's given ones (the top alternatives where they have gradients, then the token) again, with its own terms.
template <typename T>
__device__ __forceinline__ void given_column(const LogpGradParams& p, const RowGrad& r, int64_t row, int64_t tok, int i, int lo,
                                             int hi) {
  const int given = p.gt ? p.top : 0;
  const int64_t col = i == given ? tok : p.top_index[row * p.top + i];
  if (col < lo || col >= hi) return;
  float add = col == tok && p.g ? p.g[row] : 0.0f;
  for (int j = 0; j < given; ++j)
    if (p.top_index[row * p.top + j] == col) add += p.gt[row * p.top + j];
  const float v = r.at(to_f<T>(static_cast<const T*>(p.x)[row * p.ldx + col]));
  static_cast<T*>(p.dx)[row * p.cols + col] = from_f<T>(fmaf(add, p.inv_t, v));
}

template <typename T, int E, int NR, bool VEC>
__global__ void __launch_bounds__(256) logp_grad_warp_kernel(const LogpGradParams p) {
  constexpr int EL = 16 / (int)sizeof(T);
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * NR;
  float f[NR][E];
  int64_t tok[NR];
  RowGrad rg[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const bool on = row0 + r < p.rows;
    tok[r] = on ? token_of(p.tokens, p.tok64, row0 + r) : 0;
    rg[r] = row_grad(p, on ? row0 + r : p.rows - 1, tok[r]);
    load_row<T, E, VEC>(static_cast<const T*>(p.x) + (row0 + r) * p.ldx, p.cols, lane, on && tok[r] != p.ignore, f[r]);
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (row0 + r >= p.rows) break;
    T* dx = static_cast<T*>(p.dx) + (row0 + r) * p.cols;
    const bool none = rg[r].ln_s == INFINITY;          // an ignored row, or one without a distribution
#pragma unroll
    for (int e = 0; e < E; ++e) f[r][e] = none ? 0.0f : rg[r].at(f[r][e]);
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < E / EL; ++j) {
        const int col = (j * 32 + lane) * EL;
        if (col < p.cols) {
          if constexpr (EL == 4)
            *reinterpret_cast<float4*>(dx + col) = make_float4(f[r][4 * j], f[r][4 * j + 1], f[r][4 * j + 2], f[r][4 * j + 3]);
          else
            *reinterpret_cast<uint4*>(dx + col) =
                make_uint4(pack2<T>(f[r][8 * j], f[r][8 * j + 1]), pack2<T>(f[r][8 * j + 2], f[r][8 * j + 3]),
                           pack2<T>(f[r][8 * j + 4], f[r][8 * j + 5]), pack2<T>(f[r][8 * j + 6], f[r][8 * j + 7]));
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * 32 + lane < p.cols) dx[e * 32 + lane] = from_f<T>(f[r][e]);
    }
  }
  __syncwarp();
  const int given = (p.gt ? p.top : 0) + 1;
#pragma unroll
  for (int r = 0; r < NR; ++r)
    if (row0 + r < p.rows && rg[r].ln_s != INFINITY)
      for (int i = lane; i < given; i += 32) given_column<T>(p, rg[r], row0 + r, tok[r], i, 0, p.cols);
}

constexpr int kGradChunk = 16384;       // bytes of a row for a block

// A block takes a chunk of a row: kGradChunk bytes between 16-byte boundaries of x (the first chunk from the row's start).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) logp_grad_row_kernel(const LogpGradParams p) {
  constexpr int EL = 16 / (int)sizeof(T), U = 4, CH = kGradChunk / (int)sizeof(T);
  grid_dep_wait();
  const int64_t row = blockIdx.x / (unsigned)p.chunks;
  const int part = (int)(blockIdx.x % (unsigned)p.chunks), tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  T* dx = static_cast<T*>(p.dx) + row * p.cols;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  // chunk borders at multiples of CH less the row's offset
  const int lo = max(0, part * CH - off), hi = (int)min((int64_t)p.cols, (int64_t)(part + 1) * CH - off);
  if (lo >= hi) return;
  const int64_t tok = token_of(p.tokens, p.tok64, row);
  const RowGrad r = row_grad(p, row, tok);
  const bool none = r.ln_s == INFINITY;
  const int head = min(hi - lo, (part == 0 && off ? EL - off : 0)), vecs = alike ? (hi - lo - head) / EL : 0;
  const uint4* xv = reinterpret_cast<const uint4*>(x + lo + head);
  uint4* dv = reinterpret_cast<uint4*>(dx + lo + head);
  for (int i = tid; i < vecs; i += kRowThreads * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (!none && i + u * kRowThreads < vecs) w[u] = xv[i + u * kRowThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kRowThreads >= vecs) continue;
      float f[EL];
      piece<T>(w[u], f);
#pragma unroll
      for (int e = 0; e < EL; ++e) f[e] = none ? 0.0f : r.at(f[e]);
      if constexpr (EL == 4)
        dv[i + u * kRowThreads] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      else
        dv[i + u * kRowThreads] = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
    }
  }
  for (int i = tid; i < hi - lo - vecs * EL; i += kRowThreads) {
    const int col = lo + (i < head ? i : vecs * EL + i);
    dx[col] = from_f<T>(none ? 0.0f : r.at(to_f<T>(x[col])));
  }
  __syncthreads();
  if (!none && tid <= (p.gt ? p.top : 0)) given_column<T>(p, r, row, tok, tid, lo, hi);
}

// ---- launch ------------------------------------------------------------------------------------
constexpr int kWarpCols = 1024;

template <typename T>
cudaError_t launch_forward(LogpParams p, cudaStream_t st) {
  constexpr int EL = 16 / (int)sizeof(T);
  if (p.cols <= kWarpCols) {
    const bool vec = p.cols % EL == 0 && on(p.x, 16) && (p.rows <= 1 || p.ldx % EL == 0);
    const int NR = p.cols <= 256 ? 4 : p.cols <= 512 ? 2 : 1;
    const dim3 grid((unsigned)((p.rows + 8 * NR - 1) / (8 * NR)));
#define GLAD_LOGP(E, NR_) return launch_k(vec ? logp_warp_kernel<T, E, NR_, true> : logp_warp_kernel<T, E, NR_, false>, grid, \
                                          dim3(256), 0, st, true, p)
    if (NR == 4) GLAD_LOGP(8, 4);
    if (NR == 2) GLAD_LOGP(16, 2);
    GLAD_LOGP(32, 1);
#undef GLAD_LOGP
  }
  // Blocks of a row: while every thread keeps four 16-byte pieces and the rows alone do not fill the GPU several times over.
  p.cluster = 1;
  while (p.cluster < 8 && p.cols / (p.cluster * 2) >= kRowThreads * 4 * EL && p.rows * p.cluster < 56 * num_sms()) p.cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * p.cluster));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, logp_row_kernel<T>, p);
}

template <typename T>
cudaError_t launch_backward(LogpGradParams p, cudaStream_t st) {
  constexpr int EL = 16 / (int)sizeof(T);
  if (p.cols <= kWarpCols) {
    const bool vec = p.cols % EL == 0 && on(p.x, 16) && on(p.dx, 16) && (p.rows <= 1 || p.ldx % EL == 0);
    const int NR = p.cols <= 256 ? 4 : p.cols <= 512 ? 2 : 1;
    const dim3 grid((unsigned)((p.rows + 8 * NR - 1) / (8 * NR)));
#define GLAD_LOGP(E, NR_) return launch_k(vec ? logp_grad_warp_kernel<T, E, NR_, true> : logp_grad_warp_kernel<T, E, NR_, false>, \
                                          grid, dim3(256), 0, st, true, p)
    if (NR == 4) GLAD_LOGP(8, 4);
    if (NR == 2) GLAD_LOGP(16, 2);
    GLAD_LOGP(32, 1);
#undef GLAD_LOGP
  }
  constexpr int CH = kGradChunk / (int)sizeof(T);
  // a misaligned row ends up to EL - 1 elements later
  p.chunks = (int)(((int64_t)p.cols + EL - 1 + CH - 1) / CH);
  return launch_k(logp_grad_row_kernel<T>, dim3((unsigned)(p.rows * p.chunks)), dim3(kRowThreads), 0, st, true, p);
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
  if (!(temperature >= 1e-6f && temperature <= 1e6f)) return "temperature must be in [1e-6, 1e6]";
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
    const cudaError_t e = launch_forward<decltype(t)>(p, (cudaStream_t)stream);
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
    const cudaError_t e = launch_backward<decltype(t)>(p, (cudaStream_t)stream);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  });
}

}  // extern "C"
