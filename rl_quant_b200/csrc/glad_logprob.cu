// Log probabilities of given tokens, entropy and the top alternatives of rows of logits, and their gradient:
//   z = (x - max x) / T,  S = sum e^z,  log p_j = z_j - ln S,  H = ln S - sum(e^z z) / S
//   dx_j = [ g [j = t] + sum_i gt_i [j = t_i] - p_j (g + sum gt) - gh p_j (ln p_j + H) ] / T
// Sums and statistics are fp32 (the maximum and the sums of what has been seen, brought to a larger maximum as it comes up), so the logits
// are read once forward and once backward, and no probability is stored. Bytes are the bound of many rows, the exponentials
// (one a logit) come second, launch and latency bound a few rows.
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
  float inv_t, low;
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
// ln S; inf where every logit is -inf (no distribution), NaN where one is +inf or NaN.
__device__ __forceinline__ float ln_sum(const Stats& v) {
  return v.m == -INFINITY ? INFINITY : v.m < INFINITY ? logf(v.s) : NAN;
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

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The lanes' stats together, in every lane.
__device__ __forceinline__ Stats join_lanes(Stats v, float k) {
  raise(v, warp_max_nan(v.m), k);
  v.s = warp_sum(v.s);
  v.t = warp_sum(v.t);
  return v;
}
__device__ __forceinline__ Stats no_stats() { return {-INFINITY, 0.0f, 0.0f}; }

// The token's logit, NaN for one outside the row.
template <typename T>
__device__ __forceinline__ float token_logit(const LogpParams& p, const T* x, int64_t tok) {
  return tok >= 0 && tok < p.cols ? to_f<T>(x[tok]) : NAN;
}
__device__ __forceinline__ void write_row(const LogpParams& p, int64_t row, float at_token, const Stats& v) {
  const float ln_s = ln_sum(v);
  p.logp[row] = at_token != at_token ? NAN : log_of(at_token, v, ln_s, p.inv_t);
  if (p.entropy) p.entropy[row] = v.m == -INFINITY ? 0.0f : ln_s - v.t * p.inv_t / v.s;
  if (p.stats) p.stats[row] = make_float2(v.m == -INFINITY ? 0.0f : v.m, ln_s);
}
__device__ __forceinline__ void write_top(const LogpParams& p, int64_t row, int i, uint64_t rank, const Stats& v, float ln_s) {
  p.top_index[row * p.top + i] = (int64_t)(int)~(uint32_t)rank;
  p.top_logp[row * p.top + i] = log_of(value_of(rank), v, ln_s, p.inv_t);
}
__device__ __forceinline__ void write_ignored(const LogpParams& p, int64_t row, int i) {
  if (i == 0) {
    p.logp[row] = 0.0f;
    if (p.entropy) p.entropy[row] = 0.0f;
    if (p.stats) p.stats[row] = make_float2(0.0f, INFINITY);
  }
  if (i < p.top) p.top_logp[row * p.top + i] = 0.0f, p.top_index[row * p.top + i] = -1;
}

// How many of list[0 .. n) rank above q.
__device__ __forceinline__ int above(const uint64_t* list, int n, uint64_t q) {
  int before = 0, j = 0;
  for (; j + 8 <= n; j += 8) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(list + j + i);
      before += (u.x > q) + (u.y > q);
    }
  }
  for (; j < n; ++j) before += list[j] > q;
  return before;
}

// ---- rows of up to 1024 columns: a warp each ---------------------------------------------------
// A lane holds E elements of a row, 16-byte pieces (VEC) or every 32nd. NR rows of a warp are loaded before the first is
// used: with one row a warp has 16 bytes a lane in flight and the row's latency (two shuffle trees) is not covered. 118784 rows of 256 f16
// with entropy, forward and backward: 39 us, 178 MB, 4.5 TB/s (one row at a time: 100 us); issue slots are the bound.
template <typename T, int E, bool VEC>
__device__ __forceinline__ int col_of(int e, int lane) {
  constexpr int EL = 16 / (int)sizeof(T);
  return VEC ? (e / EL * 32 + lane) * EL + e % EL : e * 32 + lane;
}
// A lane's elements as stored (16-bit types: two a word); -inf past the row.
template <typename T, int E>
struct Held {
  uint32_t w[E * (int)sizeof(T) / 4];
  __device__ __forceinline__ void floats(float (&f)[E]) const {
#pragma unroll
    for (int i = 0; i < E * (int)sizeof(T) / 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 u = unpack2<T>(w[i]);
        f[2 * i] = u.x, f[2 * i + 1] = u.y;
      }
    }
  }
};
template <typename T, int E, bool VEC>
__device__ __forceinline__ Held<T, E> load_row(const T* x, int cols, int lane, bool on) {
  constexpr int EL = 16 / (int)sizeof(T);
  constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  Held<T, E> h;
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < E / EL; ++j) {
      const int col = (j * 32 + lane) * EL;
      uint4 v = make_uint4(kNone, kNone, kNone, kNone);
      if (on && col < cols) v = *reinterpret_cast<const uint4*>(x + col);
      h.w[4 * j] = v.x, h.w[4 * j + 1] = v.y, h.w[4 * j + 2] = v.z, h.w[4 * j + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < E; ++e) h.w[e] = on && e * 32 + lane < cols ? reinterpret_cast<const uint32_t*>(x)[e * 32 + lane] : kNone;
  } else {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(x);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const uint32_t lo = on && e * 32 + lane < cols ? u[e * 32 + lane] : kNone >> 16;
      const uint32_t hi = on && (e + 1) * 32 + lane < cols ? u[(e + 1) * 32 + lane] : kNone >> 16;
      h.w[e / 2] = lo | hi << 16;
    }
  }
  return h;
}

// Two at a time: these instructions have the rate of the single ones.
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(Two t, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.v)); }
__device__ __forceinline__ Two operator+(Two a, Two b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(a.v) : "l"(b.v), "l"(c.v));
  return a;
}
// Sums of e^z and (ENT) e^z d over N logits, d = x - m.
template <bool ENT, int N>
__device__ __forceinline__ void add_terms(const float (&f)[N], float m, float k, float& s, float& t) {
  const Two minus = two(-m, -m), kk = two(k, k);
  Two ss = two(0.0f, 0.0f), tt = two(0.0f, 0.0f);
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    Two d = two(f[e], f[e + 1]) + minus;
    if constexpr (ENT) {
      float a, b;
      apart(d, a, b);
      d = two(fmaxf(a, -1e30f), fmaxf(b, -1e30f));      // below()
    }
    float a, b;
    apart(d * kk, a, b);
    const Two x = two(exp2_fast(a), exp2_fast(b));
    ss = ss + x;
    if constexpr (ENT) tt = fma2(x, d, tt);
  }
  float a, b;
  apart(ss, a, b);
  s += a + b;
  if constexpr (ENT) {
    apart(tt, a, b);
    t += a + b;
  }
}

// Sums over the warp of N values at once, N a power of two: each step hands half of the open values to the partner. Lane l
// returns the sum of v[l / (32 / N)].
template <int N>
__device__ __forceinline__ float fold(float (&v)[N], int lane) {
  int o = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
    o /= 2;
  }
#pragma unroll
  for (; o; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

constexpr int kWarpList = 192;

// The `top` first columns of a warp's row. `top` lanes reach the top-th largest of the lanes' maxima (or there are fewer with
// columns), so what lies below it is out; the rest is ranked by counting. More than the list holds (many equal ones): one by one.
template <typename T, int E, bool VEC>
__device__ __forceinline__ void warp_top(const LogpParams& p, int64_t row, const float (&f)[E], const Stats& of, int lane,
                                         uint64_t* list, int* count) {
  const float ln_s = ln_sum(of);
  float m = f[0];
#pragma unroll
  for (int e = 1; e < E; ++e) m = max_nan(m, f[e]);
  uint32_t key = col_of<T, E, VEC>(0, lane) < p.cols ? (uint32_t)(rank_of(m, 0) >> 32) : 0u;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)            // the lanes' maxima, falling
#pragma unroll
    for (int o = size / 2; o; o /= 2) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, key, o);
      const bool larger = ((lane & o) == 0) == ((lane & size) == 0 || size == 32);
      key = larger ? max(key, other) : min(key, other);
    }
  const uint32_t bar_key = __shfl_sync(0xffffffffu, key, p.top - 1);
  const float bar = value_of((uint64_t)bar_key << 32);
  uint32_t in = 0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if ((bar_key == 0 || !(f[e] < bar)) && col_of<T, E, VEC>(e, lane) < p.cols) in |= 1u << e;
  __syncwarp();
  if (lane == 0) *count = 0;
  __syncwarp();
  const int mine = __popc(in);
  int at = mine ? atomicAdd(count, mine) : 0;
  __syncwarp();
  const int n = *count;
  if (n <= kWarpList) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (in >> e & 1) list[at++] = rank_of(f[e], col_of<T, E, VEC>(e, lane));
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
      const uint64_t q = list[i];
      const int before = above(list, n, q);
      if (before < p.top) write_top(p, row, before, q, of, ln_s);
    }
    __syncwarp();
    return;
  }
  // rounds of: every lane's best that is not taken, the best of those, the lowest column among equals
  uint32_t taken = 0;
  for (int i = 0; i < p.top; ++i) {
    uint64_t best = 0;
    int where = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int col = col_of<T, E, VEC>(e, lane);
      const uint64_t q = rank_of(f[e], col);
      if (q > best && !(taken >> e & 1) && col < p.cols) best = q, where = e;
    }
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    const uint64_t won = (uint64_t)hi << 32 | lo;
    if (best == won) taken |= 1u << where;
    if (lane == i) write_top(p, row, i, won, of, ln_s);
  }
}

// TOP: with alternatives.
template <typename T, int E, int NR, bool VEC, bool TOP>
__global__ void __launch_bounds__(256) logp_warp_kernel(const LogpParams p) {
  constexpr int LR = 32 / NR;                           // lanes of a row; the first of them finishes it
  __shared__ __align__(16) uint64_t lists[TOP ? 8 : 1][TOP ? kWarpList : 2];
  __shared__ int counts[8];
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * NR, mine = row0 + lane / LR;
  const int64_t tok = mine < p.rows ? token_of(p.tokens, p.tok64, mine) : p.ignore;
  const uint32_t live = __ballot_sync(0xffffffffu, tok != p.ignore);
  Held<T, E> h[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r)
    h[r] = load_row<T, E, VEC>(static_cast<const T*>(p.x) + (row0 + r) * p.ldx, p.cols, lane, row0 + r < p.rows);
  const float at_token = token_logit<T>(p, static_cast<const T*>(p.x) + mine * p.ldx, tok != p.ignore ? tok : -1);
  const float k = p.inv_t * kLog2e;
  float sums[2 * NR];
  Stats v = {0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float f[E];
    h[r].floats(f);
    float m = f[0];
#pragma unroll
    for (int e = 1; e < E; ++e) m = max_nan(m, f[e]);
    m = warp_max_nan(m);
    if (lane / LR == r) v.m = m;
    sums[2 * r] = sums[2 * r + 1] = 0.0f;
    if (p.entropy) add_terms<true>(f, m == -INFINITY ? 0.0f : m, k, sums[2 * r], sums[2 * r + 1]);
    else add_terms<false>(f, m == -INFINITY ? 0.0f : m, k, sums[2 * r], sums[2 * r + 1]);
  }
  v.s = fold(sums, lane);
  v.t = __shfl_xor_sync(0xffffffffu, v.s, LR / 2);
  if (lane % LR == 0 && mine < p.rows) {
    if (tok != p.ignore) write_row(p, mine, at_token, v);
    else write_ignored(p, mine, 0);
  }
  if constexpr (TOP) {
#pragma unroll 1
    for (int r = 0; r < NR; ++r) {
      const int64_t row = row0 + r;
      if (row >= p.rows) break;
      const Stats of = {__shfl_sync(0xffffffffu, v.m, r * LR), __shfl_sync(0xffffffffu, v.s, r * LR), 0.0f};
      if (!(live >> (r * LR) & 1)) {
        if (lane) write_ignored(p, row, lane);
        continue;
      }
      float f[E];
      h[r].floats(f);
      warp_top<T, E, VEC>(p, row, f, of, lane, lists[threadIdx.x >> 5], &counts[threadIdx.x >> 5]);
    }
  }
}

// ---- longer rows: a block or a cluster of blocks each ------------------------------------------
// A block holds a row, or a slice of one where there are few: 61 x 128001 bf16 with 20 alternatives on clusters of 8, 13.2 us (15.6 MB,
// mostly the alternatives' ranking and latency; without clusters' slices held in registers 22 us); 1 x 65536 f32 with entropy and 5
// alternatives 5.5 us (launch); 2048 x 131072 bf16 with entropy and its
// gradient 249 us, 1.54 GB (a few rows ignored), 6.2 TB/s: HBM.
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

// The largest of some pieces.
template <typename T, int U>
__device__ __forceinline__ float max_of(const uint4 (&w)[U]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      m = max_nan(max_nan(m, max_nan(__uint_as_float(w[u].x), __uint_as_float(w[u].y))),
                  max_nan(__uint_as_float(w[u].z), __uint_as_float(w[u].w)));
    return m;
  } else {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto as = [](const uint32_t& v) { return *reinterpret_cast<const P*>(&v); };
    P m = __hmax2_nan(__hmax2_nan(as(w[0].x), as(w[0].y)), __hmax2_nan(as(w[0].z), as(w[0].w)));
#pragma unroll
    for (int u = 1; u < U; ++u)
      m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(as(w[u].x), as(w[u].y)), __hmax2_nan(as(w[u].z), as(w[u].w))));
    const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(&m));
    return max_nan(f.x, f.y);
  }
}

constexpr int kGroups = kRowThreads / 4;
struct RowShared {
  Stats warps[kRowThreads / 32];
  Stats parts[8];                     // of the row's blocks, in the first one
  int count;
  uint32_t bar;                       // the groups' top-th largest maximum
  __align__(16) uint32_t keys[kGroups];
  uint64_t best[kRowThreads / 32];
  uint64_t top[8][kMaxTop + 1];       // of the row's blocks, in the first one (a list a bank)
  __align__(16) uint64_t list[kCandidates];
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

// The block's `top` first elements of its slice, best first, into out[0 .. top) (0: none). `m` is the thread's largest logit. `top` of
// the groups of four threads reach their top-th largest maximum (or there are fewer with elements), so what lies below it is out,
// and only threads at or above it look at their elements again: each(i, in) is their next piece from i on with one that is in. More candidates than the list holds (many equal ones): one by one.
template <typename T, typename V>
__device__ __forceinline__ void block_top(const Slice<T>& sl, int top, float m, RowShared& sh, uint64_t* out, V&& each) {
  const int tid = threadIdx.x;
  const bool some = sl.lo + tid < sl.hi || tid < sl.extra;
  const uint32_t key = some ? (uint32_t)(rank_of(m, 0) >> 32) : 0u;
  uint32_t high = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
  high = max(high, __shfl_xor_sync(0xffffffffu, high, 2));
  if (tid % 4 == 0) sh.keys[tid / 4] = high;
  if (tid == 0) sh.count = 0;
  if (tid < kMaxTop) out[tid] = 0;
  __syncthreads();
  {
    int more = 0, least = 0;                            // than the group's own, of a quarter of the groups
#pragma unroll
    for (int i = 0; i < kGroups / 4; i += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(sh.keys + tid % 4 * (kGroups / 4) + i);
      more += (u.x > high) + (u.y > high) + (u.z > high) + (u.w > high);
      least += (u.x >= high) + (u.y >= high) + (u.z >= high) + (u.w >= high);
    }
    int both = more << 16 | least;
    both += __shfl_xor_sync(0xffffffffu, both, 1);
    both += __shfl_xor_sync(0xffffffffu, both, 2);
    if ((both >> 16) < top && (both & 0xffff) >= top) sh.bar = high;       // equal keys write the same
  }
  __syncthreads();
  const uint32_t bar = sh.bar;
  const float low = value_of((uint64_t)bar << 32);
  auto in = [&](float v) { return bar == 0 || !(v < low); };      // a NaN is
  if (some && key >= bar) {
    auto offer = [&](uint32_t mask, const float (&f)[Slice<T>::EL], int col) {
      int at = atomicAdd(&sh.count, __popc(mask));
#pragma unroll
      for (int e = 0; e < Slice<T>::EL; ++e)
        if (mask >> e & 1) {
          if (at < kCandidates) sh.list[at] = rank_of(f[e], col + e);
          ++at;
        }
    };
    float f[Slice<T>::EL];
    for (int i = sl.lo + tid; i < sl.hi;) {
      i = each(i, in);
      if (i >= sl.hi) break;
      piece<T>(sl.body[i], f);
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < Slice<T>::EL; ++e) mask |= (uint32_t)in(f[e]) << e;
      offer(mask, f, sl.head + i * Slice<T>::EL);
      i += kRowThreads;
    }
    if (tid < sl.extra) {
      const int col = sl.extra_col(tid);
      f[0] = to_f<T>(sl.x[col]);
      if (in(f[0])) offer(1u, f, col);
    }
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= kCandidates) {
    // eight threads a candidate
    for (int i = tid / 8; i - tid / 8 < n; i += kRowThreads / 8) {
      const uint64_t q = i < n ? sh.list[i] : 0;
      int before = 0;
      for (int j = tid % 8; j < n; j += 8) before += sh.list[j] > q;
      before += __shfl_xor_sync(0xffffffffu, before, 1);
      before += __shfl_xor_sync(0xffffffffu, before, 2);
      before += __shfl_xor_sync(0xffffffffu, before, 4);
      if (tid % 8 == 0 && i < n && before < top) out[before] = q;
    }
  } else {
    uint64_t mine = next_best(sl, ~0ull);
    for (int i = 0; i < top; ++i) {
      const uint64_t won = block_max(mine, sh);
      if (won == 0) break;
      if (tid == 0) out[i] = won;
      if (mine == won) mine = next_best(sl, won);
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// HELD: the block's slice is at most kHeld pieces a thread, all loaded at once (one latency instead of two or more) and kept
// in registers for the alternatives. Else four pieces at a time, and the alternatives read them again.
constexpr int kHeld = 8;
template <typename T, bool ENT, bool HELD>
__global__ void __launch_bounds__(kRowThreads) logp_row_kernel(const LogpParams p) {
  constexpr int EL = Slice<T>::EL, U = HELD ? kHeld : 4;
  __shared__ RowShared sh;
  const int C = p.cluster, rank = (int)(blockIdx.x % (unsigned)C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (C > 1) cluster_arrive();                          // the first block is there to be written to
  grid_dep_wait();
  const int64_t row = blockIdx.x / (unsigned)C;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const Slice<T> sl(x, p.cols, rank, C);
  uint4 w[U];
  auto load = [&](int from) {
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = from + u * kRowThreads < sl.hi ? sl.body[from + u * kRowThreads] : masked_piece<T>();
  };
  int i = sl.lo + tid;
  if (HELD) load(i);                                   // on their way while the token arrives
  const int64_t tok = token_of(p.tokens, p.tok64, row);
  if (tok == p.ignore) {                               // all blocks of the row
    if (rank == 0) write_ignored(p, row, tid);
    if (C > 1) cluster_wait();
    return;
  }
  const float at_token = tid == 0 && rank == 0 ? token_logit<T>(p, x, tok) : 0.0f;
  const float k = p.inv_t * kLog2e;
  Stats v = no_stats();
  if (tid < sl.extra) v.m = to_f<T>(x[sl.extra_col(tid)]);
  if (v.m != -INFINITY) v.s = 1.0f;
  do {
    if (!HELD) load(i);
    raise(v, max_of<T>(w), k);
    const float base = v.m == -INFINITY ? 0.0f : v.m;
#pragma unroll
    for (int u = 0; u < U; u += 4) {
      if (HELD && sl.lo + u * kRowThreads >= sl.hi) break;
      float f[4 * EL];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float g[EL];
        piece<T>(w[u + h], g);
#pragma unroll
        for (int e = 0; e < EL; ++e) f[h * EL + e] = g[e];
      }
      add_terms<ENT>(f, base, k, v.s, v.t);
    }
    i += kRowThreads * U;
  } while (!HELD && i < sl.hi);
  const float own = v.m;
  v = join_lanes(v, k);
  if (lane == 0) sh.warps[warp] = v;
  __syncthreads();
  if (warp == 0) {
    v = join_lanes(lane < kRowThreads / 32 ? sh.warps[lane] : no_stats(), k);
    if (lane == 0) sh.parts[0] = v;
  }
  if (p.top)
    block_top<T>(sl, p.top, own, sh, sh.top[0], [&](int from, auto&& in) {
      if constexpr (HELD) {
        uint32_t mask = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint4 one[1] = {w[u]};
          mask |= (uint32_t)in(max_of<T>(one)) << u;
        }
        const int first = sl.lo + tid;
        mask &= ~0u << ((from - first) / kRowThreads);
        return mask ? first + (__ffs(mask) - 1) * kRowThreads : sl.hi;
      } else {
        for (; from < sl.hi; from += 4 * kRowThreads) {
          uint4 look[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            look[u] = from + u * kRowThreads < sl.hi ? sl.body[from + u * kRowThreads] : masked_piece<T>();
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint4 one[1] = {look[u]};
            if (in(max_of<T>(one))) return from + u * kRowThreads;
          }
        }
        return sl.hi;
      }
    });
  else __syncthreads();
  if (C > 1) {
    cluster_wait();
    if (rank > 0) {                                     // this block's part goes to the first one
      if (tid < 3) st_cluster_u32(mapa_shared(smem_u32(&sh.parts[rank]) + 4 * tid, 0),
                                  __float_as_uint(reinterpret_cast<const float*>(&sh.parts[0])[tid]));
      if (tid >= 32 && tid < 32 + 2 * p.top)
        st_cluster_u32(mapa_shared(smem_u32(sh.top[rank]) + 4 * (tid - 32), 0),
                       reinterpret_cast<const uint32_t*>(sh.top[0])[tid - 32]);
    }
    cluster_arrive();
    if (rank > 0) return;                               // a block that is gone is not waited for
    cluster_wait();
  }
  // the blocks' parts; the first of all their firsts, eight threads an entry
  const Stats all = join_lanes(lane < C ? sh.parts[lane] : no_stats(), k);
  const float ln_s = ln_sum(all);
  if (tid == 0) write_row(p, row, at_token, all);
  const int n = C * p.top;
  for (int i = tid / 8; i - tid / 8 < n; i += kRowThreads / 8) {
    const uint64_t q = i < n ? sh.top[i / p.top][i % p.top] : 0;
    int before = 0;                                     // in list tid % 8, which falls: by halving
    if (tid % 8 < C) {
#pragma unroll
      for (int step = kMaxTop; step; step /= 2)
        if (before + step <= p.top && sh.top[tid % 8][before + step - 1] > q) before += step;
    }
    before += __shfl_xor_sync(0xffffffffu, before, 1);
    before += __shfl_xor_sync(0xffffffffu, before, 2);
    before += __shfl_xor_sync(0xffffffffu, before, 4);
    if (tid % 8 == 0 && q && before < p.top) write_top(p, row, before, q, all, ln_s);
  }
}

// ---- gradient ----------------------------------------------------------------------------------
// A row's gradient without the given columns' own terms: with d = x - m, p = 2^(k d + c) and ln p + H = d / T + H - ln S it is
// p (a d + b), a = -gh / T^2, b = -(gh (H - ln S) + G) / T. d ends at `low`, where p is 2^-200 of the largest and less, which is
// 0 here: beyond it a d would reach infinity for masked logits at small T, and 0 times that is NaN.
struct RowGrad {
  float m, k, c, a, b, low;
  __device__ __forceinline__ float at(float x) const {
    const float d = fmaxf(x - m, low);
    return exp2_fast(fmaf(d, k, c)) * fmaf(d, a, b);
  }
  // of N logits, in place
  template <int N>
  __device__ __forceinline__ void over(float (&f)[N]) const {
    const Two minus = two(-m, -m), kk = two(k, k), cc = two(c, c), aa = two(a, a), bb = two(b, b);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float x, y;
      apart(two(f[e], f[e + 1]) + minus, x, y);
      const Two d = two(fmaxf(x, low), fmaxf(y, low));
      apart(fma2(d, kk, cc), x, y);
      apart(two(exp2_fast(x), exp2_fast(y)) * fma2(d, aa, bb), f[e], f[e + 1]);
    }
  }
};
__device__ __forceinline__ bool given_in(int64_t tok, int cols) { return tok >= 0 && tok < cols; }

// none: an ignored row, or one without a distribution; its gradient is 0.
__device__ __forceinline__ RowGrad row_grad(const LogpGradParams& p, int64_t row, int64_t tok, bool& none) {
  const float2 st = p.stats[row];
  float G = p.g ? p.g[row] : 0.0f;
  const float gh = p.gh ? p.gh[row] * p.inv_t : 0.0f, H = p.gh ? p.entropy[row] : 0.0f;
  none = st.y == INFINITY;
  if (!given_in(tok, p.cols) && p.g) G = NAN;
  if (p.gt)
    for (int i = 0; i < p.top; ++i) G += p.gt[row * p.top + i];
  if (none) return RowGrad{0.0f, 1.0f, -INFINITY, 0.0f, 0.0f, p.low};
  return RowGrad{st.x, p.inv_t * kLog2e, -st.y * kLog2e, -gh * p.inv_t, p.gh ? fmaf(-gh, H - st.y, -G * p.inv_t) : -G * p.inv_t,
                 p.low};
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
  constexpr int EL = 16 / (int)sizeof(T), LR = 32 / NR;
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * NR, mine = row0 + lane / LR;
  const int64_t tok = mine < p.rows ? token_of(p.tokens, p.tok64, mine) : p.ignore;
  Held<T, E> h[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r)
    h[r] = load_row<T, E, VEC>(static_cast<const T*>(p.x) + (row0 + r) * p.ldx, p.cols, lane, row0 + r < p.rows);
  bool none;
  const RowGrad rg = row_grad(p, mine < p.rows ? mine : p.rows - 1, tok, none);
  none |= mine >= p.rows;
  const uint32_t empty = __ballot_sync(0xffffffffu, none);
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (row0 + r >= p.rows) break;
    T* dx = static_cast<T*>(p.dx) + (row0 + r) * p.cols;
    const int from = r * LR;
    const RowGrad of{__shfl_sync(0xffffffffu, rg.m, from), p.inv_t * kLog2e, __shfl_sync(0xffffffffu, rg.c, from),
                     __shfl_sync(0xffffffffu, rg.a, from), __shfl_sync(0xffffffffu, rg.b, from), p.low};
    float f[E];
    h[r].floats(f);
    if (empty >> from & 1) {                            // 0 whatever the row holds: an infinity would make NaN of it
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = 0.0f;
    } else {
      of.over(f);
    }
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < E / EL; ++j) {
        const int col = (j * 32 + lane) * EL;
        if (col < p.cols) {
          if constexpr (EL == 4)
            *reinterpret_cast<float4*>(dx + col) = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
          else
            *reinterpret_cast<uint4*>(dx + col) =
                make_uint4(pack2<T>(f[8 * j], f[8 * j + 1]), pack2<T>(f[8 * j + 2], f[8 * j + 3]),
                           pack2<T>(f[8 * j + 4], f[8 * j + 5]), pack2<T>(f[8 * j + 6], f[8 * j + 7]));
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * 32 + lane < p.cols) dx[e * 32 + lane] = from_f<T>(f[e]);
    }
  }
  __syncwarp();
  if (!none)
    for (int i = lane % LR; i <= (p.gt ? p.top : 0); i += LR) given_column<T>(p, rg, mine, tok, i, 0, p.cols);
}

constexpr int kGradChunk = 16384;       // bytes of a row for a block

// A block takes a chunk of a row: kGradChunk bytes between 16-byte boundaries of x (the first chunk from the row's start). HBM is the
// bound (figures above).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) logp_grad_row_kernel(const LogpGradParams p) {
  constexpr int EL = 16 / (int)sizeof(T), U = 4, CH = kGradChunk / (int)sizeof(T);
  grid_dep_wait();
  // from the last row, which a forward pass just before read last: some of it is still in the L2
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const int64_t row = block / (unsigned)p.chunks;
  const int part = (int)(block % (unsigned)p.chunks), tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  T* dx = static_cast<T*>(p.dx) + row * p.cols;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  // chunk borders at multiples of CH less the row's offset
  const int lo = max(0, part * CH - off), hi = (int)min((int64_t)p.cols, (int64_t)(part + 1) * CH - off);
  if (lo >= hi) return;
  const int64_t tok = token_of(p.tokens, p.tok64, row);
  bool none;
  const RowGrad r = row_grad(p, row, tok, none);
  const int head = min(hi - lo, (part == 0 && off ? EL - off : 0)), vecs = alike ? (hi - lo - head) / EL : 0;
  const uint4* xv = reinterpret_cast<const uint4*>(x + lo + head);
  uint4* dv = reinterpret_cast<uint4*>(dx + lo + head);
  for (int i = tid; i < vecs; i += kRowThreads * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kRowThreads < vecs) w[u] = none ? masked_piece<T>() : xv[i + u * kRowThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kRowThreads >= vecs) continue;
      float f[EL];
      piece<T>(w[u], f);
      r.over(f);
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
    const int NR = p.cols <= 256 ? 8 : p.cols <= 512 ? 4 : 2;
    const dim3 grid((unsigned)((p.rows + 8 * NR - 1) / (8 * NR)));
    auto go = [&](auto k, auto k_top) { return launch_k(p.top ? k_top : k, grid, dim3(256), 0, st, true, p); };
#define GLAD_LOGP(E, NR_, V) return go(logp_warp_kernel<T, E, NR_, V, false>, logp_warp_kernel<T, E, NR_, V, true>)
    if (p.cols <= 64) GLAD_LOGP(2, 8, false);           // little to load: as many lanes as there are columns
    if (NR == 8 && vec) GLAD_LOGP(8, 8, true);
    if (NR == 8) GLAD_LOGP(8, 8, false);
    if (NR == 4 && vec) GLAD_LOGP(16, 4, true);
    if (NR == 4) GLAD_LOGP(16, 4, false);
    if (vec) GLAD_LOGP(32, 2, true);
    GLAD_LOGP(32, 2, false);
#undef GLAD_LOGP
  }
  // Blocks of a row: while every thread keeps four 16-byte pieces and the rows alone do not fill the GPU several times over.
  p.cluster = 1;
  while (p.cluster < 8 && p.cols / (p.cluster * 2) >= kRowThreads * 4 * EL && p.rows * p.cluster < 12 * num_sms()) p.cluster *= 2;
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
  const bool held = p.cols <= (int64_t)p.cluster * kRowThreads * kHeld * EL;
  if (held) return cudaLaunchKernelEx(&cfg, p.entropy ? logp_row_kernel<T, true, true> : logp_row_kernel<T, false, true>, p);
  return cudaLaunchKernelEx(&cfg, p.entropy ? logp_row_kernel<T, true, false> : logp_row_kernel<T, false, false>, p);
}

template <typename T>
cudaError_t launch_backward(LogpGradParams p, cudaStream_t st) {
  constexpr int EL = 16 / (int)sizeof(T);
  if (p.cols <= kWarpCols) {
    const bool vec = p.cols % EL == 0 && on(p.x, 16) && on(p.dx, 16) && (p.rows <= 1 || p.ldx % EL == 0);
    const int NR = p.cols <= 256 ? 8 : p.cols <= 512 ? 4 : 2;
    const dim3 grid((unsigned)((p.rows + 8 * NR - 1) / (8 * NR)));
#define GLAD_LOGP(E, NR_) return launch_k(vec ? logp_grad_warp_kernel<T, E, NR_, true> : logp_grad_warp_kernel<T, E, NR_, false>, \
                                          grid, dim3(256), 0, st, true, p)
    if (p.cols <= 64) return launch_k(logp_grad_warp_kernel<T, 2, 8, false>, grid, dim3(256), 0, st, true, p);
    if (NR == 8) GLAD_LOGP(8, 8);
    if (NR == 4) GLAD_LOGP(16, 4);
    GLAD_LOGP(32, 2);
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
  p.ignore = ignore_index, p.inv_t = 1.0f / temperature, p.top = top, p.low = -200.0f / (p.inv_t * kLog2e);
  p.stats = reinterpret_cast<const float2*>(stats), p.entropy = entropy, p.top_index = top_index;
  p.g = d_log_prob, p.gh = d_entropy, p.gt = d_top, p.dx = d_logits;
  return for_type(x_dtype, [&](auto t) {
    const cudaError_t e = launch_backward<decltype(t)>(p, (cudaStream_t)stream);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  });
}

}  // extern "C"
