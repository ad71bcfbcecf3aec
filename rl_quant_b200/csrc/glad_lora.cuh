// Low-rank adapters of many requests beside a shared projection:
//   forward   u[m] = s[i] A[i] x[m],  y[m] = base[m] + B[i] u[m]          (i: row m's adapter; none: y = base or 0)
//   backward  du[m] = s[i] B[i]^T dy[m],  dx[m] = A[i]^T du[m]            (the same kernel on transposed weights)
//             dA[i] = sum over i's rows of du[m] x[m]^T,  dB[i] = the same of dy[m] u[m]^T
//
// Few operations a byte (2 r of them), so at low ranks the bytes of x, base, y and the adapters in use are the bound. Rows of an adapter
// are taken in tiles of 16, 32 or 128; a cluster of blocks shares a tile: its warps split K for u, the parts are added through
// distributed shared memory in a fixed order, and the warps split N for y. u never leaves the chip unless a backward pass will need it.
//
// lora_kernel: mma.sync on rings of asynchronous copies, one a warp. A product's order of k is free as long as both operands share
//   it, so a lane takes 16 adjacent bytes of a row as its k of several instructions, and likewise 32 adjacent bytes of an output row.
//   Measured, forward: 64 requests with an adapter each, 4096 -> 14336 rank 16 bf16, 14.2 us, 42 MB, 2.95 TB/s (launch and three
//   latencies: x and A, the sum over the cluster, B); 8192 rows 4096 -> 4096 rank 16 bf16, one adapter, 32.8 us, 201 MB, 6.1 TB/s:
//   HBM; a token, rank 16, 5.5 us: launch and the same latencies.
// lora_tc_kernel: tcgen05, for many rows of ranks above 32, where mma.sync would be the bound.
// outer_kernel, outer_tc_kernel: the gradients of the adapters, the same two ways.
//
// u is fp32 and is added up as such. As an operand of the second product it is split into two numbers (16 bits together beside
// bf16 rows, 22 beside others), inputs of 16 bits are exact, and fp32 inputs are split the same way, three products each. The
// instruction cuts its fp32 sum off, which a chain of thousands of terms shows beside fp32 outputs: there every 8 or 16 terms start from 0
// and are added by rounding (4096 rows 2048 -> 2048 rank 64 with gradients: relative errors 1.3e-6 to 5.1e-6 became 2.6e-7 to 5.5e-7, fp32
// products of torch 5e-7 to 1e-6, for 191 us instead of 177; forward alone 63.1 and 61.7).
#pragma once
#include <utility>

#include "glad_elem.cuh"
#include "tc05.cuh"

namespace glad {
namespace lora {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kSelfRows = 256;        // up to so many rows the kernel finds the rows of an adapter itself, a cluster a row,
constexpr int kScanRows = 4096, kScanAdapters = 512;   // or, with few adapters, by counting all of them; above, plan_kernel does it once
// for all. Counting and a plan, us, 4096 -> 4096 rank 16 bf16: 2048 rows of 6 adapters 16.8 and 19.5, 3000 of 16 28.0 and 29.2, 4096 of 16
// 33.3 and 31.5, 8192 of 16 62.7 and 52.4; rank 64, 4096 of 16 43.2 and 46.0, 8192 65.8 and 65.7.
constexpr int kMaxAdapters = 16384, kMaxRank = 128;

// What plan_kernel leaves: rows in the order of their adapters, and tiles of them. In 32-bit words:
//   [0] tiles, [1 .. L+2] first place of each adapter's rows in the order (L: of the rows without one; L+1: M),
//   then the order [M], then the tiles (adapter or -1, first place) [2 * max]
struct Plan {
  const int32_t* w;
  int L, M;
  __device__ int tiles() const { return w[0]; }
  __device__ int first(int a) const { return w[1 + a]; }
  __device__ int row(int place) const { return w[3 + L + place]; }
  __device__ int2 tile(int t) const { return make_int2(w[3 + L + M + 2 * t], w[3 + L + M + 2 * t + 1]); }
};

struct Params {
  const void* x;        // [M, K]
  const void* w1;       // A [L, r, K]; transposed: B [L, K, r]
  const void* w2;       // B [L, N, r]; transposed: A [L, r, N]
  const void* base;     // [M, N] or null
  void* y;              // [M, N]
  float* u;             // [M, r] or null, as kept() gives it
  const float* scale;   // [L] or null: scale_value
  const void* index;    // null: adapter 0 for every row
  const int32_t* plan;  // null: the kernel looks at index itself
  int64_t ldx, ldb;
  float scale_value;
  int M, K, N, r, L, index64, cluster;
  int split;            // tiles of the kernel in a tile of the plan
  int half;             // some address off 4 bytes
  // of the tensor-core kernel: the device's status word, the longest wait, and arrivals to wait for that never come (tests)
  uint32_t* status;
  uint32_t wait_ns, hold;
};

struct OuterParams {    // out[a] = sum over a's rows of v[m]^T x[m]
  const void* x;        // [M, K]
  const float* v;       // [M, r], as kept() gives it
  void* out;            // element (rank, k) of adapter a at a * r * K + rank * step_r + k * step_k
  const int32_t* plan;  // null: all rows are adapter 0's
  int64_t ldx, step_r, step_k;
  int M, K, r, L, cluster;
  uint32_t pitch;       // of x in bytes, where it fits
  int blocks;
  int half;             // some address of x off 4 bytes
};
struct OuterPair {
  OuterParams of[2];
  int cluster;
  uint32_t* status;     // of the tensor-core kernel, as above
  uint32_t wait_ns, hold;
};

__device__ __forceinline__ float tf32(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return __uint_as_float(r);
}
// v = hi + lo, 11 bits each. Of an infinite v, lo is finite (the difference would be a NaN): the least that a finite v has, half a step of
// the largest number, so that products with it do not overflow beside the infinite ones. The 16-bit splits below alike.
__device__ __forceinline__ void split(float v, float& hi, float& lo) {
  hi = tf32(v);
  lo = tf32(fmaxf(v - hi, -1.7e35f));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const float4& a, float b0, float b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(__float_as_uint(a.x)), "r"(__float_as_uint(a.y)), "r"(__float_as_uint(a.z)), "r"(__float_as_uint(a.w)),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
template <typename T>
__device__ __forceinline__ void mma_16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a and b of the product with (hi, lo) parts each.
__device__ __forceinline__ void mma_split(float (&c)[4], const float4& ah, const float4& al, float b0, float b1) {
  float h0, l0, h1, l1;
  split(b0, h0, l0);
  split(b1, h1, l1);
  mma_tf32(c, al, h0, h1);
  mma_tf32(c, ah, l0, l1);
  mma_tf32(c, ah, h0, h1);
}
__device__ __forceinline__ void split4(const float4& v, float4& hi, float4& lo) {
  split(v.x, hi.x, lo.x);
  split(v.y, hi.y, lo.y);
  split(v.z, hi.z, lo.z);
  split(v.w, hi.w, lo.w);
}

// Element e of 32-bit words (16-bit types: two a word) as fp32.
template <typename T, int W>
__device__ __forceinline__ float elem(const uint32_t (&w)[W], int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w[e]);
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w[e >> 1]);
    return e & 1 ? __high2float(h) : __low2float(h);
  } else {
    return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
}
// The 16-bit elements number e of words a and b as a pair.
__device__ __forceinline__ uint32_t pair_of(uint32_t a, uint32_t b, int e) {
  return __byte_perm(a, b, e & 1 ? 0x7632 : 0x5410);
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ int adapter_of(const Params& p, int m) {
  const int64_t a = p.index64 ? static_cast<const int64_t*>(p.index)[m] : (int64_t)static_cast<const int32_t*>(p.index)[m];
  return a >= 0 && a < p.L ? (int)a : -1;
}

// Whether a call without a plan runs a cluster for every row, most of which end at once, rather than counts rows for every tile that there
// can be, which takes 1 us longer. Both sides, us, 4096 -> 4096 bf16 rank 16: 32 rows of 8 adapters 5.5 and 6.5, 64 of 2 7.4 and 8.4,
// 128 of 4 8.8 and 8.6, 128 of 16 7.2 and 8.0, 256 of 8 12.8 and 8.8, 256 of 128 12.2 and 13.4; rank 64: 256 of 8 28.3 and 15.6.
__host__ __device__ __forceinline__ bool finds_itself(int64_t M, int L, int R) {
  return M <= kSelfRows && (L > kScanAdapters || M <= 64 || M <= 8 * ((M + R - 1) / R + L + 1));
}
// The rows of this cluster's tile into rows[0 .. n); returns n (0: nothing to do) and the adapter. `scratch` is shared memory for
// kScanRows short numbers.
template <int R, int NT = kThreads>
__device__ __forceinline__ int find_rows(const Params& p, int tile, int* rows, int& adapter, void* scratch) {
  const int tid = threadIdx.x;
  int n;
  if (p.index == nullptr) {
    adapter = 0;
    n = min(R, p.M - tile * R);
    if (tid < n) rows[tid] = tile * R + tid;
  } else if (p.plan != nullptr) {
    const Plan plan{p.plan, p.L, p.M};
    const int whole = tile / p.split;
    if (whole >= plan.tiles()) return 0;
    const int2 t = plan.tile(whole);
    adapter = t.x;
    const int from = t.y + tile % p.split * R;
    n = min(R, plan.first((adapter < 0 ? p.L : adapter) + 1) - from);
    if (n <= 0) return 0;
    if (tid < n) rows[tid] = plan.row(from + tid);
  } else if (!finds_itself(p.M, p.L, R)) {
    // Count the rows of every adapter, look the tile up among their tiles, and collect the adapter's rows from the tile's first on.
    __shared__ int cnt[kScanAdapters + 1], sums[NT / 32], found[2];
    uint16_t* of = static_cast<uint16_t*>(scratch);
    const int lane = tid & 31, G = p.L + 1;
    for (int i = tid; i < G; i += NT) cnt[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < p.M; i0 += NT) {
      const int i = i0 + tid;
      int a = -1;
      if (i < p.M) {
        a = adapter_of(p, i);
        a = a < 0 ? p.L : a;
        of[i] = (uint16_t)a;
      }
      const uint32_t same = __match_any_sync(0xffffffffu, a);
      if (a >= 0 && lane == __ffs(same) - 1) atomicAdd(&cnt[a], __popc(same));
    }
    __syncthreads();
    if (tid < 32) {
      int carry = 0, a = -1, first = 0;
      for (int a0 = 0; a0 < G && a < 0; a0 += 32) {
        const int tiles = a0 + lane < G ? (cnt[a0 + lane] + R - 1) / R : 0;
        int t = tiles;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int u = __shfl_up_sync(0xffffffffu, t, o);
          if (lane >= o) t += u;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, carry + t > tile);
        if (past) {
          const int l = __ffs(past) - 1;
          a = a0 + l;
          first = (tile - carry - __shfl_sync(0xffffffffu, t - tiles, l)) * R;
        }
        carry += __shfl_sync(0xffffffffu, t, 31);
      }
      if (lane == 0) found[0] = a, found[1] = first;
    }
    __syncthreads();
    const int a = found[0], first = found[1];
    if (a < 0) return 0;
    adapter = a == p.L ? -1 : a;
    n = min(R, cnt[a] - first);
    const int run = (p.M + NT - 1) / NT, lo = tid * run, hi = min(p.M, lo + run);
    int mine = 0;
    for (int i = lo; i < hi; ++i) mine += of[i] == a;
    int at = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += u;
    }
    if (lane == 31) sums[tid >> 5] = at;
    __syncthreads();
    at -= mine;
    for (int w = 0; w < tid >> 5; ++w) at += sums[w];
    if (at < first + R && at + mine > first)
      for (int i = lo; i < hi; ++i)
        if (of[i] == a) {
          if (at >= first && at < first + R) rows[at - first] = i;
          ++at;
        }
  } else {
    // One cluster a row: it is the tile's where R, 2 R, ... rows of the same adapter (none) come before it.
    __shared__ int of[kSelfRows], counts[NT / 32];
    if (tid < p.M) of[tid] = adapter_of(p, tid);
    __syncthreads();
    adapter = of[tile];
    const bool same = tid < p.M && of[tid] == adapter;
    if (__syncthreads_count(same && tid < tile) % R != 0) return 0;
    const bool mine = same && tid >= tile;
    const uint32_t votes = __ballot_sync(0xffffffffu, mine);
    if ((tid & 31) == 0) counts[tid >> 5] = __popc(votes);
    __syncthreads();
    int at = __popc(votes & ((1u << (tid & 31)) - 1)), all = 0;
    for (int w = 0; w < NT / 32; ++w) {
      if (w < tid >> 5) at += counts[w];
      all += counts[w];
    }
    if (mine && at < R) rows[at] = tid;
    n = min(R, all);
  }
  __syncthreads();
  if (tid >= n && tid < R) rows[tid] = rows[0];       // read, not used
  __syncthreads();
  return n;
}

// fp32 numbers as an operand beside rows of T, whose products should run at the rate of T: two bf16 numbers (16 bits) for bf16;
// two fp16 numbers (22 bits) for fp16 where a power of two can bring them into its range: u, by row, and
// outer_tc_kernel's v, by rank (kHalves). Else two tf32 numbers (22 bits), at half the rate: fp32, and fp16's v in outer_kernel.
template <typename T>
constexpr bool kPairs = std::is_same<T, __nv_bfloat16>::value;
template <typename T>
constexpr bool kHalves = std::is_same<T, __half>::value;
__device__ __forceinline__ void split_bf16(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const float2 f = __bfloat1622float2(h);
  const __nv_bfloat162 l = __floats2bfloat162_rn(fmaxf(a - f.x, -6.7e35f), fmaxf(b - f.y, -6.7e35f));
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(fmaxf(a - f.x, -16.0f), fmaxf(b - f.y, -16.0f));
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// A row's power of two and its inverse: brings its largest number (as bits) to 2^14, so that the lower halves reach 2^-38 of it.
__device__ __forceinline__ void row_power(uint32_t most, float& up, float& down) {
  int e = 14 - ((int)(most >> 23) - 127);
  if (most == 0 || most >= 0x7f800000u) e = 0;
  e = min(max(e, -126), 126);
  up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
}
// u and du as they are kept: the two bf16 numbers side by side, or fp32.
template <typename T>
__device__ __forceinline__ float kept(float v) {
  if constexpr (kPairs<T>) {
    uint32_t hi, lo;
    split_bf16(v, 0.0f, hi, lo);
    return __uint_as_float(__byte_perm(hi, lo, 0x5410));
  } else {
    return v;
  }
}
// The warps' parts of a gradient tile, [RT][BW] each `step` floats apart, added up and, over the cluster, written.
template <typename T, int RT, int BW>
__device__ __forceinline__ void outer_end(const OuterParams& p, float* part, const float* red, int step, int a, int r0, int n0,
                                          int rank, int C) {
  const int tid = threadIdx.x;
  for (int i = tid; i < RT * BW; i += kThreads) {
    float s = red[i];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s += red[w * step + i];
    part[i] = s;
  }
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  T* out = static_cast<T*>(p.out) + (int64_t)a * p.r * p.K;
  const uint32_t here = smem_u32(part);
  const bool by_rank = p.step_r == 1;                  // adjacent threads write adjacent elements
  for (int i = rank * kThreads + tid; i < RT * BW; i += C * kThreads) {
    const int k = by_rank ? i % RT : i / BW, col = by_rank ? i / RT : i % BW;
    const uint32_t src = here + 4 * (k * BW + col);
    float v;
    if (C > 1) {
      v = ld_cluster(mapa_shared(src, 0));
      for (int c = 1; c < C; ++c) v += ld_cluster(mapa_shared(src, c));
    } else {
      v = part[k * BW + col];
    }
    if (r0 + k < p.r && n0 + col < p.K) out[(r0 + k) * p.step_r + (int64_t)(n0 + col) * p.step_k] = from_f<T>(v);
  }
  if (C > 1) cluster_sync_all();
}

// ---- rings of asynchronous copies ---------------------------------------------------------------
// Every warp copies what it needs next, by itself: 16-byte copies into a ring of its own while it works on the stage before, so
// the bytes in flight (up to 100 KB an SM) do not depend on registers or on other warps. The pieces are placed so that a
// fragment's reads touch every bank once.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {       // zeros where not live
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(live ? 8 : 0) : "memory");
}
// ROWS rows of ranks, src on the first's: COUNT 16-byte pieces of each, of which `ranks` ranks are there and the rest is zeros, as
// are rows from `there` on. Row i goes to place P::at(i), PITCH bytes each. P::at moves bits only, so a lane's places are its first
// one plus constants. Rows off 16 bytes are copied in halves.
template <typename T, int COUNT, int ROWS, int PITCH, typename P>
__device__ __forceinline__ void copy_rows(int lane, uint32_t dst, const T* src, int r, int ranks, int there) {
  constexpr int EL = 16 / (int)sizeof(T), STEP = 32 / COUNT;
  static_assert(COUNT <= 32 && ROWS % STEP == 0, "a lane's pieces are of one column");
  if (r % EL == 0) {
    const int row0 = lane / COUNT, c = lane % COUNT;
    const bool in = c * EL < ranks;
    const T* s = src + (in ? c * EL : 0);
    const uint32_t d = dst + P::at(row0) * PITCH + 16 * c;
    if (in && there >= ROWS) {
      s += (int64_t)row0 * r;
#pragma unroll
      for (int j = 0; j < ROWS / STEP; ++j) {
        copy16(d + P::at(STEP * j) * PITCH, s);
        s += STEP * r;
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < ROWS / STEP; ++j) {
        const int row = row0 + STEP * j;
        const bool live = in && row < there;
        copy16(dst + P::at(row) * PITCH + 16 * c, s + (live ? (int64_t)row * r : 0), live);
      }
    }
  } else {
#pragma unroll 1
    for (int id = lane; id < 2 * COUNT * ROWS; id += 32) {
      const int row = id / (2 * COUNT), c = id % (2 * COUNT);
      const bool live = row < there && c * (EL / 2) < ranks;
      copy8(dst + P::at(row) * PITCH + 8 * c, src + (live ? (int64_t)row * r + c * (EL / 2) : 0), live);
    }
  }
}

// The same for tensors off the 16-byte boundaries, one word of 4 bytes a lane: by asynchronous copies where every address is on 4 bytes
// (half == false), else, for 16-bit elements, by two loads and a store. `left` elements are there from src on (null: none).
template <typename T>
struct Word {
  uint32_t dst;
  const T* src;
  int left;
};
template <typename T, int COUNT, typename F>
__device__ __forceinline__ void copy_words(bool half, const T* any, F&& f) {
  constexpr int PER = 4 / (int)sizeof(T), BATCH = COUNT < 16 ? COUNT : 16;
  if (!half || sizeof(T) == 4) {
#pragma unroll 4
    for (int i = 0; i < COUNT; ++i) {
      const Word<T> w = f(i);
      const int bytes = w.src ? max(0, min(PER, w.left)) * (int)sizeof(T) : 0;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(w.dst), "l"(bytes ? w.src : any), "r"(bytes) : "memory");
    }
  } else {
#pragma unroll 1
    for (int i0 = 0; i0 < COUNT; i0 += BATCH) {
      uint32_t v[BATCH], at[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const Word<T> w = f(i0 + i);
        const uint16_t* u = reinterpret_cast<const uint16_t*>(w.src);
        const uint32_t lo = w.src && w.left > 0 ? __ldg(u) : 0u, hi = w.src && w.left > 1 ? __ldg(u + 1) : 0u;
        v[i] = lo | hi << 16, at[i] = w.dst;
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at[i]), "r"(v[i]) : "memory");
    }
  }
}

template <int N>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                   : "r"(addr + 4 * i));
  }
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint32_t w[4];
  lds(addr, w);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ void mma_pair(float (&c)[4], const uint4& hi, const uint4& lo, uint32_t b0, uint32_t b1) {
  mma_16<T>(c, lo.x, lo.y, lo.z, lo.w, b0, b1);
  mma_16<T>(c, hi.x, hi.y, hi.z, hi.w, b0, b1);
}
__device__ __forceinline__ float4 as_f4(const uint4& v) {
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
// One step of a product whose A operand is split, B operand elements b0, b1 of T.
template <typename T>
__device__ __forceinline__ void mma_step(float (&c)[4], const uint4& hi, const uint4& lo, float b0, float b1) {
  if constexpr (sizeof(T) == 4) {
    mma_split(c, as_f4(hi), as_f4(lo), b0, b1);
  } else {
    mma_tf32(c, as_f4(lo), b0, b1);
    mma_tf32(c, as_f4(hi), b0, b1);
  }
}

template <typename T, int RT, int MT>
struct Ring {
  static constexpr int SZ = (int)sizeof(T), R = 16 * MT;
  static constexpr int kStage1 = R * 128 + RT * 128;                  // 128 bytes of every row of x, and as much of A
  static constexpr int PB = RT * SZ < 64 ? RT * SZ : 64, PR = PB / SZ; // bytes and ranks of a piece of a row of B
  static constexpr int kW2 = 128 / SZ * PB, kBase = R * 128, kSlot = kW2 + kBase;
  // Two of each: a third changed nothing (64 requests at rank 16 13.4 us both ways, 2048 rows at rank 64 29.4 and 29.7).
  static constexpr int kSlots = 2, kStages = RT == 128 ? 1 : 2;
  static constexpr int kRed = (kSlots - 1) * kSlot;                   // a warp's part of u lies behind the slots that are filled before it is read
  static constexpr int kNeed = kRed + R * RT * 4 > kSlots * kSlot ? kRed + R * RT * 4 : kSlots * kSlot;
  static constexpr int kBytes = kStages * kStage1 > kNeed ? kStages * kStage1 : kNeed;               // of a warp
  static constexpr int kSmem = kWarps * kBytes + R * RT * 4 + R * RT * 8;
};

// Where 16-byte piece c of a 128-byte row lies: halves swapped in odd rows, so that eight lanes on half a row of two touch all banks.
__device__ __forceinline__ int swap(int c, int row) { return (c ^ ((row & 1) * 4)) * 16; }

// Places of a chunk's rows of B as k: the four lanes of a column read rows EL q + e of a half at once, which lie side by side.
template <int EL>
struct KPlace {
  __host__ __device__ static constexpr int at(int row) { return row / (4 * EL) * (4 * EL) + row % EL * 4 + row / EL % 4; }
};
// Places of a block's rows of B as columns: column 4 EL h + EL (g / 2) + 2 t + g % 2 is column g of the instruction of tile EL / 2 h + t
// and lies at 8 tile + g.
template <int EL>
struct NPlace {
  __host__ __device__ static constexpr int at(int row) {
    return (row / (4 * EL) * (EL / 2) + row % EL / 2) * 8 + row % (4 * EL) / EL * 2 + (row & 1);
  }
};

// RT: the rank, rounded up to 16, 32, 64 or 128; 16 MT rows a tile. RAGGED: some address off 16 bytes.
template <typename T, int RT, int MT, bool TRANS, bool RAGGED>
__global__ void __launch_bounds__(kThreads, RT == 16 ? 2 : 1) lora_kernel(const Params p) {
  using L = Ring<T, RT, MT>;
  constexpr int SZ = L::SZ, R = L::R, NT = RT / 8, EL = 16 / SZ, CH = 8 * EL, S1 = L::kStages, S2 = L::kSlots;
  constexpr int PR = L::PR, PB = L::PB, PIECES = RT / PR, E = PR / 4;           // E: a lane's ranks of a piece
  constexpr bool PAIRS = kPairs<T> || kHalves<T>;
  constexpr int SE = PAIRS ? 4 : 2, PS = E / SE, ST = PIECES * PS;          // ranks of a lane, and instructions, a step
  constexpr int TL = EL, BW = 8 * TL;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int rows[R];
  __shared__ int64_t base_at[R];                       // their places in base
  __shared__ float up[kHalves<T> ? R : 1], down[kHalves<T> ? R : 1];   // powers of two of the rows of u
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int C = p.cluster, rank = (int)blockIdx.x % C, tile = (int)blockIdx.x / C;
  const uint32_t ring = smem_u32(smem) + warp * L::kBytes;
  float* part = reinterpret_cast<float*>(smem + kWarps * L::kBytes);            // this block's part of u, [R][RT]
  uint4* frag = reinterpret_cast<uint4*>(part + R * RT);                        // u as split operands, [MT][ST][32][2]
  auto red = [&](int w) { return reinterpret_cast<float*>(smem + w * L::kBytes + L::kRed); };   // warp w's part, [R][RT]
  grid_dep_wait();
  int adapter;
  const int n = find_rows<R>(p, tile, rows, adapter, smem);
  if (n == 0) return;                                 // the whole cluster
  const int W = C * kWarps, w0 = rank * kWarps + warp;
  if (tid < R) base_at[tid] = (int64_t)rows[tid] * p.ldb;
  __syncthreads();

  if (adapter >= 0) {
    // the lane's piece lane % 8 of rows lane / 8 + 4 j, at its next chunk of K
    const T* w1 = static_cast<const T*>(p.w1) + (int64_t)adapter * p.r * p.K;
    const T* xp[4 * MT];
#pragma unroll
    for (int j = 0; j < 4 * MT; ++j)
      xp[j] = static_cast<const T*>(p.x) + (int64_t)rows[(lane >> 3) + 4 * j] * p.ldx + w0 * CH + (lane & 7) * EL;
    const T* wp = TRANS ? w1 + (int64_t)w0 * CH * p.r : w1 + (int64_t)(lane >> 3) * p.K + w0 * CH + (lane & 7) * EL;
    int from = w0 * CH, slot = 0;
    auto fetch = [&]() {
      if (from < p.K && RAGGED) {
        // a line of a row's 128 bytes at a time
        const uint32_t at = ring + slot * L::kStage1, wat = at + R * 128;
        const int e = lane * (4 / SZ);
        copy_words<T, R>(p.half, static_cast<const T*>(p.x), [&](int row) {
          return Word<T>{at + row * 128 + swap(lane >> 2, row) + 4 * (lane & 3),
                         row < n ? static_cast<const T*>(p.x) + (int64_t)rows[row] * p.ldx + from + e : nullptr, p.K - from - e};
        });
        if constexpr (!TRANS) {
          copy_words<T, RT>(p.half, w1, [&](int row) {
            return Word<T>{wat + row * 128 + swap(lane >> 2, row) + 4 * (lane & 3),
                           row < p.r ? w1 + (int64_t)row * p.K + from + e : nullptr, p.K - from - e};
          });
        } else {
          constexpr int WPR = RT * SZ / 4;             // words of a row
          copy_words<T, CH * WPR / 32>(p.half, w1, [&](int i) {
            const int id = lane + 32 * i, row = id / WPR, rk = id % WPR * (4 / SZ);
            return Word<T>{wat + KPlace<EL>::at(row) * (RT * SZ) + id % WPR * 4,
                           from + row < p.K ? w1 + (int64_t)(from + row) * p.r + rk : nullptr, p.r - rk};
          });
        }
        from += W * CH;
      } else if (from < p.K) {
        const uint32_t at = ring + slot * L::kStage1, to = at + (lane >> 3) * 128 + swap(lane & 7, lane >> 3), wat = at + R * 128;
        const bool whole = from + CH <= p.K && n == R, live = from + (lane & 7) * EL < p.K;
#pragma unroll
        for (int j = 0; j < 4 * MT; ++j) {
          if (whole) {
            copy16(to + j * 512, xp[j]);
          } else {
            const bool in = live && (lane >> 3) + 4 * j < n;
            copy16(to + j * 512, in ? xp[j] : static_cast<const T*>(p.x), in);
          }
          xp[j] += W * CH;
        }
        if constexpr (!TRANS) {
#pragma unroll
          for (int j = 0; j < RT / 4; ++j) {
            const T* src = wp + (int64_t)(4 * j) * p.K;
            const bool in = live && (lane >> 3) + 4 * j < p.r;
            copy16(to + R * 128 + j * 512, in ? src : w1, in);
          }
          wp += W * CH;
        } else {
          copy_rows<T, RT * SZ / 16, CH, RT * SZ, KPlace<EL>>(lane, wat, wp, p.r, p.r, p.K - from);
          wp += (int64_t)W * CH * p.r;
        }
        from += W * CH;
      }
      slot = slot + 1 == S1 ? 0 : slot + 1;
      cp_async_commit();
    };
    float acc[MT][NT][4] = {};
#pragma unroll
    for (int i = 0; i < S1 - 1; ++i) fetch();
    int stage = 0;
    for (int k0 = w0 * CH; k0 < p.K; k0 += W * CH) {
      fetch();
      cp_async_wait_group<S1 - 1>();
      __syncwarp();
      const uint32_t at = ring + stage * L::kStage1, wat = at + R * 128;
      stage = stage + 1 == S1 ? 0 : stage + 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {                    // a lane's k: pieces q and q + 4 of the row
        uint32_t xa[2 * MT][4];
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) lds(at + (g + 8 * j) * 128 + swap(q + 4 * h, g), xa[j]);
        auto products = [&](int t, const uint32_t (&wb)[4]) {
          if constexpr (SZ == 4) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              float c[4] = {};                         // added to the sum by rounding: the instruction cuts its sum off
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float4 ah, al;
                split4(make_float4(__uint_as_float(xa[2 * m][2 * j]), __uint_as_float(xa[2 * m + 1][2 * j]),
                                   __uint_as_float(xa[2 * m][2 * j + 1]), __uint_as_float(xa[2 * m + 1][2 * j + 1])), ah, al);
                mma_split(c, ah, al, __uint_as_float(wb[2 * j]), __uint_as_float(wb[2 * j + 1]));
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[m][t][e] += c[e];
            }
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int m = 0; m < MT; ++m)
                mma_16<T>(acc[m][t], xa[2 * m][2 * j], xa[2 * m + 1][2 * j], xa[2 * m][2 * j + 1], xa[2 * m + 1][2 * j + 1],
                          wb[2 * j], wb[2 * j + 1]);
          }
        };
        if constexpr (!TRANS) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t wb[4];
            lds(wat + (8 * t + g) * 128 + swap(q + 4 * h, g), wb);
            products(t, wb);
          }
        } else {
          constexpr int WN = NT * SZ / 4;              // words of a lane's ranks
          uint32_t raw[EL][WN];
#pragma unroll
          for (int e = 0; e < EL; ++e) lds(wat + (h * 4 * EL + e * 4 + q) * (RT * SZ) + g * NT * SZ, raw[e]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t wb[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if constexpr (SZ == 4) wb[w] = raw[w][t];
              else wb[w] = pair_of(raw[2 * w][t >> 1], raw[2 * w + 1][t >> 1], t);
            }
            products(t, wb);
          }
        }
      }
      __syncwarp();
    }
    cp_async_wait_all();
    __syncwarp();
    float* mine = red(warp);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = 2 * q + (c & 1), at = TRANS ? col * NT + t : 8 * t + col;
          mine[(16 * i + g + 8 * (c >> 1)) * RT + at] = acc[i][t][c];
        }
  }

  // The second product's operands: base and B of a step (a piece of the ranks of a block of columns).
  const T* w2 = static_cast<const T*>(p.w2) + (int64_t)(adapter < 0 ? 0 : adapter) * p.N * p.r;
  const bool any = adapter >= 0;
  int next_n = p.y == nullptr ? p.N : w0 * BW, next_piece = 0, w_slot = 0, b_slot = 0;       // what is copied next
  auto fetch2 = [&]() {
    if (next_n < p.N) {
      if (next_piece == 0) {
        if (p.base != nullptr && RAGGED) {
          const uint32_t at = ring + b_slot * L::kSlot + L::kW2;
          const T* src = static_cast<const T*>(p.base);
          const int col = next_n + lane * (4 / SZ);
          copy_words<T, R>(p.half, src, [&](int row) {
            return Word<T>{at + row * 128 + swap(lane >> 2, row) + 4 * (lane & 3), row < n ? src + base_at[row] + col : nullptr,
                           p.N - col};
          });
        } else if (p.base != nullptr) {
          const uint32_t at = ring + b_slot * L::kSlot + L::kW2 + (lane >> 3) * 128 + swap(lane & 7, lane >> 3);
          const int col = next_n + (lane & 7) * EL;
          const T* src = static_cast<const T*>(p.base);
          if (next_n + BW <= p.N && n == R) {
#pragma unroll
            for (int j = 0; j < 4 * MT; ++j) copy16(at + j * 512, src + base_at[(lane >> 3) + 4 * j] + col);
          } else {
#pragma unroll
            for (int j = 0; j < 4 * MT; ++j) {
              const bool live = (lane >> 3) + 4 * j < n && col < p.N;
              copy16(at + j * 512, live ? src + base_at[(lane >> 3) + 4 * j] + col : src, live);
            }
          }
        }
        b_slot = b_slot + 1 == S2 ? 0 : b_slot + 1;
      }
      if (any) {
        const uint32_t at = ring + w_slot * L::kSlot;
        if constexpr (RAGGED && !TRANS) {
          constexpr int WPR = PB / 4;
          copy_words<T, BW * WPR / 32>(p.half, w2, [&](int i) {
            const int id = lane + 32 * i, row = id / WPR, rk = next_piece * PR + id % WPR * (4 / SZ);
            return Word<T>{at + NPlace<EL>::at(row) * PB + id % WPR * 4,
                           next_n + row < p.N ? w2 + (int64_t)(next_n + row) * p.r + rk : nullptr, p.r - rk};
          });
        } else if constexpr (RAGGED) {
          const int col = next_n + lane * (4 / SZ);
          copy_words<T, PR>(p.half, w2, [&](int row) {
            const int rk = next_piece * PR + row;
            return Word<T>{at + row * 128 + (((lane >> 2) ^ (row / E)) * 16) + 4 * (lane & 3),
                           rk < p.r ? w2 + (int64_t)rk * p.N + col : nullptr, p.N - col};
          });
        } else if constexpr (!TRANS) {
          copy_rows<T, PB / 16, BW, PB, NPlace<EL>>(lane, at, w2 + (int64_t)next_n * p.r + (next_piece * PR < p.r ? next_piece * PR : 0),
                                                    p.r, p.r - next_piece * PR, p.N - next_n);
        } else {
          const int col = next_n + (lane & 7) * EL;
#pragma unroll
          for (int j = 0; j < PR / 4; ++j) {
            const int row = (lane >> 3) + 4 * j, rk = next_piece * PR + row;
            const bool live = rk < p.r && col < p.N;
            copy16(at + row * 128 + (((lane & 7) ^ (row / E)) * 16), live ? w2 + (int64_t)rk * p.N + col : w2, live);
          }
        }
        w_slot = w_slot + 1 == S2 ? 0 : w_slot + 1;
      }
      if (++next_piece >= (any ? PIECES : 1)) {
        next_piece = 0;
        next_n += W * BW;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S2 - 1; ++i) fetch2();           // on their way while u is added up
  if (adapter >= 0) {
    __syncthreads();
    for (int i = tid; i < R * RT; i += kThreads) {
      float s = red(0)[i];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) s += red(w)[i];
      part[i] = s;
    }
  }
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  if (adapter >= 0) {
    const float s = p.scale ? p.scale[adapter] : p.scale_value;
    const uint32_t here = smem_u32(part);
    float* whole = red(0);                             // [R][RT]
    for (int i = tid; i < R * RT; i += kThreads) {
      float v;
      if (C > 1) {
        v = ld_cluster(mapa_shared(here + 4 * i, 0));
        for (int c = 1; c < C; ++c) v += ld_cluster(mapa_shared(here + 4 * i, c));
      } else {
        v = part[i];
      }
      const int row = i / RT, at = i % RT;
      v = at < p.r ? v * s : 0.0f;                     // behind the ranks: 0 times an infinite x
      whole[i] = v;
      if (p.u && rank == 0 && row < n && at < p.r) p.u[(int64_t)rows[row] * p.r + at] = kept<T>(v);
    }
    __syncthreads();
    if constexpr (kHalves<T>) {
      for (int row = warp; row < R; row += kWarps) {
        float most = 0.0f;
        for (int i = lane; i < RT; i += 32) most = fmaxf(most, fabsf(whole[row * RT + i]));
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        if (lane == 0) row_power(bits, up[row], down[row]);
      }
      __syncthreads();
    }
    for (int i = tid; i < MT * ST * 32; i += kThreads) {
      const int l = i & 31, st = (i >> 5) % ST, m = (i >> 5) / ST;
      const float* v = whole + (16 * m + (l >> 2)) * RT + st / PS * PR + (l & 3) * E + st % PS * SE;
      uint4 hi, lo;
      if constexpr (kHalves<T>) {
        const float s0 = up[16 * m + (l >> 2)], s1 = up[16 * m + (l >> 2) + 8];
        split_f16(v[0] * s0, v[1] * s0, hi.x, lo.x);
        split_f16(v[8 * RT] * s1, v[8 * RT + 1] * s1, hi.y, lo.y);
        split_f16(v[2] * s0, v[3] * s0, hi.z, lo.z);
        split_f16(v[8 * RT + 2] * s1, v[8 * RT + 3] * s1, hi.w, lo.w);
      } else if constexpr (kPairs<T>) {
        split_bf16(v[0], v[1], hi.x, lo.x);
        split_bf16(v[8 * RT], v[8 * RT + 1], hi.y, lo.y);
        split_bf16(v[2], v[3], hi.z, lo.z);
        split_bf16(v[8 * RT + 2], v[8 * RT + 3], hi.w, lo.w);
      } else {
        float4 h, o;
        split4(make_float4(v[0], v[8 * RT], v[1], v[8 * RT + 1]), h, o);
        hi = make_uint4(__float_as_uint(h.x), __float_as_uint(h.y), __float_as_uint(h.z), __float_as_uint(h.w));
        lo = make_uint4(__float_as_uint(o.x), __float_as_uint(o.y), __float_as_uint(o.z), __float_as_uint(o.w));
      }
      frag[2 * i] = hi, frag[2 * i + 1] = lo;
    }
  }
  if (C > 1) cluster_sync_all();                       // nobody reads another block's part any more
  else __syncthreads();

  const uint32_t fr = smem_u32(frag);
  float c[MT][TL][4];
  T* yp[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) yp[i] = static_cast<T*>(p.y) + (int64_t)rows[g + 8 * i] * p.N + q * EL;
  int slot = 0, base_slot = 0, pi = 0;
  for (int n0 = p.y == nullptr ? p.N : w0 * BW; n0 < p.N;) {
    fetch2();
    cp_async_wait_group<S2 - 1>();
    __syncwarp();
    if (pi == 0) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < TL; ++t) c[m][t][0] = c[m][t][1] = c[m][t][2] = c[m][t][3] = 0.0f;
    }
    if (any) {
      const uint32_t at = ring + slot * L::kSlot;
      if constexpr (!TRANS) {
        uint32_t wv[TL][PB / 16];
#pragma unroll
        for (int t = 0; t < TL; ++t) lds(at + (t * 8 + g) * PB + q * (PB / 4), wv[t]);
#pragma unroll
        for (int j = 0; j < PS; ++j)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint32_t f = fr + 32 * ((m * ST + pi * PS + j) * 32 + lane);
            const uint4 hi = lds128(f), lo = lds128(f + 16);
#pragma unroll
            for (int t = 0; t < TL; ++t) {
              if constexpr (PAIRS) mma_pair<T>(c[m][t], hi, lo, wv[t][2 * j], wv[t][2 * j + 1]);
              else mma_step<T>(c[m][t], hi, lo, elem<T>(wv[t], 2 * j), elem<T>(wv[t], 2 * j + 1));
            }
          }
      } else {
#pragma unroll
        for (int j = 0; j < PS; ++j) {
          uint32_t wr[SE][4];
#pragma unroll
          for (int e = 0; e < SE; ++e) lds(at + (q * E + SE * j + e) * 128 + (((g / 2 + g % 2 * 4) ^ q) * 16), wr[e]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint32_t f = fr + 32 * ((m * ST + pi * PS + j) * 32 + lane);
            const uint4 hi = lds128(f), lo = lds128(f + 16);
#pragma unroll
            for (int t = 0; t < TL; ++t) {
              if constexpr (PAIRS)
                mma_pair<T>(c[m][t], hi, lo, pair_of(wr[0][t >> 1], wr[1][t >> 1], t), pair_of(wr[2][t >> 1], wr[3][t >> 1], t));
              else
                mma_step<T>(c[m][t], hi, lo, elem<T>(wr[0], t), elem<T>(wr[1], t));
            }
          }
        }
      }
    }
    slot = slot + 1 == S2 ? 0 : slot + 1;
    if (++pi >= (any ? PIECES : 1)) {
      const uint32_t at = ring + base_slot * L::kSlot + L::kW2;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        const int row = g + 8 * i;
        if (row >= n) continue;
        const float factor = kHalves<T> ? (any ? down[row] : 0.0f) : 1.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {                  // a lane's columns: pieces q and q + 4
          if (n0 + (q + 4 * h) * EL >= p.N) continue;
          T* y = yp[i] + n0 + 4 * h * EL;
          const uint32_t here = at + row * 128 + swap(q + 4 * h, row);
          uint32_t bw[4] = {0, 0, 0, 0};
          if (p.base != nullptr) lds(here, bw);
          float o[EL];
#pragma unroll
          for (int e = 0; e < EL; ++e) {
            const int t = TRANS ? e : h * (TL / 2) + (e >> 1), odd = TRANS ? h : e & 1;
            const float v = c[i >> 1][t][2 * (i & 1) + odd], b = elem<T>(bw, e);
            o[e] = kHalves<T> ? fmaf(v, factor, b) : v + b;
          }
          uint4 bits;
          if constexpr (SZ == 4)
            bits = make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
          else
            bits = make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]), pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
          if constexpr (RAGGED)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(here), "r"(bits.x), "r"(bits.y), "r"(bits.z), "r"(bits.w)
                         : "memory");
          else
            *reinterpret_cast<uint4*>(y) = bits;
        }
      }
      if constexpr (RAGGED) {                          // in place of base, and from there by rows
        __syncwarp();
        const int left = p.N - n0 - lane * (4 / SZ);
#pragma unroll 4
        for (int row = 0; row < n; ++row) {
          uint32_t w[1];
          lds(at + row * 128 + swap(lane >> 2, row) + 4 * (lane & 3), w);
          T* y = static_cast<T*>(p.y) + (int64_t)rows[row] * p.N + n0 + lane * (4 / SZ);
          if constexpr (SZ == 4) {
            if (left > 0) *reinterpret_cast<uint32_t*>(y) = w[0];
          } else {
            uint16_t* u = reinterpret_cast<uint16_t*>(y);
            if (!p.half && left > 1) {
              *reinterpret_cast<uint32_t*>(y) = w[0];
            } else {
              if (left > 0) u[0] = (uint16_t)w[0];
              if (left > 1) u[1] = (uint16_t)(w[0] >> 16);
            }
          }
        }
      }
      pi = 0;
      base_slot = base_slot + 1 == S2 ? 0 : base_slot + 1;
      n0 += W * BW;
    }
    __syncwarp();
  }
  cp_async_wait_all();
}

template <typename T, int RT>
struct OuterRing {
  static constexpr int kPitch = RT * 4 + (kPairs<T> ? 16 : 32);        // of a row of v: a fragment's reads touch every bank once
  static constexpr int kStage = 16 * 128 + 16 * kPitch, kStages = RT == 16 ? 3 : 2;
  static constexpr int kBytes = kStages * kStage;                      // of a warp
  static constexpr int BW = 128 / (int)sizeof(T);
  static constexpr int kSmem = kWarps * kBytes + RT * BW * 4;
  static_assert(RT * BW * 4 <= kBytes, "a warp's part of the gradient fits into its ring");
};

// out[a] = sum over a's rows of v[m]^T x[m], two gradients in one launch: the first blocks are of the first. RT: ranks of a block, 16 or
// 32 (blockIdx.z: which). A cluster shares 128 bytes of columns of an adapter's gradient; its warps split the rows, and
// the parts are added in a fixed order. Bound: at one block of ranks the bytes of x and dy, which every other one reads again (8192 rows
// 4096 -> 4096 rank 16 bf16, both gradients, 32 us with cold caches, 134 MB: 4.2 TB/s); with few rows an adapter the blocks' latency.
template <typename T, int RT, bool RAGGED>
__global__ void __launch_bounds__(kThreads, 2) outer_kernel(const __grid_constant__ OuterPair pair) {
  using L = OuterRing<T, RT>;
  const int second = (int)blockIdx.x >= pair.of[0].blocks;
  const OuterParams& p = pair.of[second];
  const int block = (int)blockIdx.x - (second ? pair.of[0].blocks : 0);
  constexpr int EL = 16 / (int)sizeof(T), TL = EL, BW = 8 * TL, RM = RT / 16, S = L::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int C = p.cluster, rank = block % C, n0 = block / C * BW;
  const int a = blockIdx.y, r0 = blockIdx.z * RT;
  const uint32_t ring = smem_u32(smem) + warp * L::kBytes;
  grid_dep_wait();
  const Plan plan{p.plan, p.L, p.M};
  const int from = p.plan ? plan.first(a) : 0, rows = p.plan ? plan.first(a + 1) - from : p.M;
  const int W = C * kWarps, w0 = rank * kWarps + warp;
  // lanes 0 .. 15: the rows of the warp's next group of 16 (-1: none)
  int group = w0 * 16, slot = 0;
  auto index_of = [&](int first) {
    const int at = first + lane;
    return lane < 16 && at < rows ? p.plan ? plan.row(from + at) : at : -1;
  };
  int next = index_of(group);
  const bool in = n0 + (lane & 7) * EL < p.K;
  const char* xc = static_cast<const char*>(p.x) + (in ? (n0 + (lane & 7) * EL) * (int)sizeof(T) : 0);
  constexpr int VC = RT / 4, VS = 32 / VC;             // pieces of a row of v, rows a step
  const bool v_in = r0 + 4 * (lane % VC) < p.r;
  const char* vc = reinterpret_cast<const char*>(p.v + (v_in ? r0 + 4 * (lane % VC) : 0));
  auto fetch = [&]() {
    if (group < rows) {
      const int mine = next;
      group += W * 16;
      next = index_of(group);
      const uint32_t at = ring + slot * L::kStage;
      if constexpr (RAGGED) {
        const T* x = static_cast<const T*>(p.x);
        const int col = n0 + lane * (4 / (int)sizeof(T));
        copy_words<T, 16>(p.half, x, [&](int row) {
          const int m = __shfl_sync(0xffffffffu, mine, row), turn = kPairs<T> ? row >> 1 & 3 : row & 3;
          return Word<T>{at + row * 128 + (((lane >> 2) ^ (2 * turn)) * 16) + 4 * (lane & 3),
                         m >= 0 ? x + (int64_t)m * p.ldx + col : nullptr, p.K - col};
        });
        copy_words<float, RT / 2>(false, p.v, [&](int i) {
          const int id = lane + 32 * i, row = id / RT, rk = id % RT, m = __shfl_sync(0xffffffffu, mine, row);
          return Word<float>{at + 2048 + row * L::kPitch + 4 * rk, m >= 0 ? p.v + (int64_t)m * p.r + r0 + rk : nullptr,
                             p.r - r0 - rk};
        });
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = (lane >> 3) + 4 * j;
          const int m = __shfl_sync(0xffffffffu, mine, row);
          const int turn = kPairs<T> ? row >> 1 & 3 : row & 3;         // a fragment's four rows at four places
          copy16(at + row * 128 + (((lane & 7) ^ (2 * turn)) * 16), xc + (uint64_t)(uint32_t)max(m, 0) * p.pitch, in && m >= 0);
        }
#pragma unroll
        for (int j = 0; j < 16 / VS; ++j) {
          const int row = lane / VC + VS * j;
          const int m = __shfl_sync(0xffffffffu, mine, row);
          copy16(at + 2048 + row * L::kPitch + 16 * (lane % VC), vc + (uint64_t)(uint32_t)max(m, 0) * (uint32_t)(4 * p.r),
                 v_in && m >= 0);
        }
      }
    }
    slot = slot + 1 == S ? 0 : slot + 1;
    cp_async_commit();
  };
  float acc[RM][TL][4] = {};
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch();
  int stage = 0;
  for (int i0 = w0 * 16; i0 < rows; i0 += W * 16) {
    fetch();
    cp_async_wait_group<S - 1>();
    __syncwarp();
    const uint32_t at = ring + stage * L::kStage, vat = at + 2048;
    stage = stage + 1 == S ? 0 : stage + 1;
    auto word_at = [&](int m, int rk) {
      uint32_t w[1];
      lds(vat + m * L::kPitch + 4 * rk, w);
      return w[0];
    };
    if constexpr (kPairs<T>) {
      uint32_t xw[4][4];                               // rows 2 q, 2 q + 1, 2 q + 8, 2 q + 9
#pragma unroll
      for (int e = 0; e < 4; ++e) lds(at + (2 * q + (e & 1) + 8 * (e >> 1)) * 128 + ((g ^ (2 * q)) * 16), xw[e]);
#pragma unroll
      for (int k = 0; k < RM; ++k) {
        uint4 hi, lo;
        const int rk = 16 * k + g;
        auto two_of = [&](int m, int rank_at, uint32_t& h, uint32_t& l) {
          const uint32_t u = word_at(m, rank_at), v = word_at(m + 1, rank_at);
          h = __byte_perm(u, v, 0x5410), l = __byte_perm(u, v, 0x7632);
        };
        two_of(2 * q, rk, hi.x, lo.x);
        two_of(2 * q, rk + 8, hi.y, lo.y);
        two_of(2 * q + 8, rk, hi.z, lo.z);
        two_of(2 * q + 8, rk + 8, hi.w, lo.w);
#pragma unroll
        for (int t = 0; t < TL; ++t)
          mma_pair<T>(acc[k][t], hi, lo, pair_of(xw[0][t >> 1], xw[1][t >> 1], t), pair_of(xw[2][t >> 1], xw[3][t >> 1], t));
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {                    // rows 8 h + q and 8 h + q + 4
        uint32_t x0[4], x1[4];
        lds(at + (8 * h + q) * 128 + ((g ^ (2 * q)) * 16), x0);
        lds(at + (8 * h + q + 4) * 128 + ((g ^ (2 * q)) * 16), x1);
#pragma unroll
        for (int k = 0; k < RM; ++k) {
          const int rk = 16 * k + g, m = 8 * h + q;
          float4 ah, al;
          auto v_at = [&](int mm, int kk) { return __uint_as_float(word_at(mm, kk)); };
          split4(make_float4(v_at(m, rk), v_at(m, rk + 8), v_at(m + 4, rk), v_at(m + 4, rk + 8)), ah, al);
#pragma unroll
          for (int t = 0; t < TL; ++t) {
            const float b0 = elem<T>(x0, t), b1 = elem<T>(x1, t);
            if constexpr (sizeof(T) == 4) {
              float c[4] = {};                         // as in lora_kernel
              mma_split(c, ah, al, b0, b1);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[k][t][e] += c[e];
            } else {
              mma_tf32(acc[k][t], al, b0, b1);
              mma_tf32(acc[k][t], ah, b0, b1);
            }
          }
        }
      }
    }
    __syncwarp();
  }
  cp_async_wait_all();
  __syncwarp();
  float* mine = reinterpret_cast<float*>(smem + warp * L::kBytes);
#pragma unroll
  for (int k = 0; k < RM; ++k)
#pragma unroll
    for (int t = 0; t < TL; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        mine[(16 * k + g + 8 * (c >> 1)) * BW + (2 * q + (c & 1)) * TL + t] = acc[k][t][c];
  __syncthreads();
  outer_end<T, RT, BW>(p, reinterpret_cast<float*>(smem + kWarps * L::kBytes), reinterpret_cast<const float*>(smem),
                       L::kBytes / 4, a, r0, n0, rank, C);
}

// ---- many rows an adapter, ranks above 32: both products on the tensor core's own memory -------------
// At these ranks mma.sync is the bound (8192 rows 4096 -> 4096 bf16: rank 64 73 us with the rings, rank 128 157), and a tile of 32 rows
// reads the adapter too often. So: tiles of 128 rows, u summed in tensor memory by tcgen05 while all warps keep three or four stages of x
// and A in flight; every block of the cluster adds up its share of u's rows and sends them, as two 16-bit numbers each (as in the
// rings), to the others; then u times 128 columns of B a step, base and y through shared memory. Two halves of eight warps take these steps
// in turn, so that one's stores go out while the other computes (one group of eight: rank 64 54 us, rank 128 61; with base and y as
// bulk copies of 256 bytes a row 67 and 72: issuing them took 3500 cycles a step). Operands lie K-major with the 128-byte
// swizzle; the backward pass gets its adapters transposed first (transpose_kernel), which are small.
// 8192 rows rank 64 50 us, rank 128 56, both 201 MB at least: 4.0 and 3.6 TB/s. Bound: the way into and out of an SM, 35 bytes a cycle
// in either phase; with few tiles latency (256 rows rank 64 17 us: launch, rows and setup 5, the rest x and A, u and columns alike).
template <int RT>
struct Tc {
  // a stage: 128 inputs of 128 rows of x and of A, in two blocks of 64 (128 bytes) each
  static constexpr int kThreads = 512, kStages = RT == 64 ? 4 : 3, kBlock = 128 * 128 + RT * 128, kStage = 2 * kBlock, NB = RT / 64;  // NB: blocks of 64 ranks
  static constexpr int kPart = 128 * RT * 4, kB = NB * 16384, kBase = 32768;
  // first the ring; then [B, two][base, two][u's operand], and this block's part of u behind it or, where that is too much, over base
  static constexpr int kBaseAt = 2 * kB, kA = 2 * kB + 2 * kBase, kBehind = kA + 2 * NB * 16384;
  static constexpr bool kApart = RT == 64;
  static constexpr int kPartAt = kApart ? kBehind : kBaseAt, kEnd = kApart ? kBehind + kPart : kBehind;
  static constexpr int kSmem = (kStages * kStage > kEnd ? kStages * kStage : kEnd) + 1024;
  static_assert(kPart <= 2 * kBase, "over base");
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {      // rows of 128 bytes, piece i of row r at i ^ (r & 7)
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ int turned(int piece, int row) { return (piece ^ (row & 7)) * 16; }
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void st_cluster1(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
// 32 consecutive columns of a warp's lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void half_sync(int half) { asm volatile("bar.sync %0, 256;" ::"r"(half + 1) : "memory"); }
// Waits for the products behind a phase; after one wait that ran out no other one waits, the bit is set and the kernel ends as usual.
template <typename P>
__device__ __forceinline__ void tc_wait(uint64_t* bar, uint32_t parity, const P& p, bool& dead) {
  if (dead || mbar_try_wait(bar, parity)) return;
  if (mbar_wait_bounded(bar, parity, p.wait_ns)) return;
  dead = true;
  atomicOr(p.status, kDevErrMmaTimeout);
}

template <typename T, int RT>
__global__ void __launch_bounds__(Tc<RT>::kThreads, 1) lora_tc_kernel(const Params p) {
  using L = Tc<RT>;
  constexpr int NTH = L::kThreads, R = 128, S = L::kStages, NB = L::NB;
  constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
  constexpr uint32_t kFirst = idesc_f16(128, RT) | kType, kSecond = idesc_f16(128, 128) | kType;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int rows[R];
  __shared__ float down[kHalves<T> ? R : 1];          // what the rows of u were divided by
  __shared__ __align__(8) uint64_t full[S], done[2], drain[2];
  __shared__ uint32_t tmem_at;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int half = warp >> 3, hw = warp & 7, ht = tid & 255;            // two halves of 8 warps take the second product's steps in turn
  const int C = p.cluster, rank = (int)blockIdx.x % C, tile = (int)blockIdx.x / C;
  grid_dep_wait();
  int adapter;
  const int n = find_rows<R, NTH>(p, tile, rows, adapter, smem);
  if (n == 0) return;                                 // the whole cluster
  const bool any = adapter >= 0;
  if (warp == 0) tmem_alloc(&tmem_at, 512);
  if (tid == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1 + p.hold);
    mbar_init(&done[0], 1 + p.hold);
    mbar_init(&done[1], 1 + p.hold);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at, base_addr = smem_u32(smem);
  bool dead = false;

  const T* w2 = static_cast<const T*>(p.w2) + (int64_t)(any ? adapter : 0) * p.N * p.r;
  const int tiles = (p.N + 127) / 128, steps = p.y != nullptr && rank < tiles ? (tiles - rank + C - 1) / C : 0;
  auto fetch_b = [&](int j) {
    if (j < steps && any) {
      const int n0 = (rank + j * C) * 128, row0 = ht >> 3, c = ht & 7;
      const uint32_t at = base_addr + half * L::kB + row0 * 128 + turned(c, row0);
      const T* src = w2 + (int64_t)(n0 + row0) * p.r + 8 * c;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = n0 + row0 + 32 * i < p.N && 64 * b + 8 * c < p.r;
          copy16(at + b * 16384 + i * 4096, in ? src + (int64_t)(32 * i) * p.r + 64 * b : w2, in);
        }
    }
    cp_async_commit();
  };
  auto fetch_base = [&](int j) {
    if (j < steps && p.base != nullptr) {
      const int n0 = (rank + j * C) * 128, row0 = ht >> 4, c = ht & 15;
      const uint32_t at = base_addr + L::kBaseAt + half * L::kBase + row0 * 256;
      const T* base = static_cast<const T*>(p.base);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = row0 + 16 * i;
        const bool in = row < n && n0 + 8 * c < p.N;
        copy16(at + i * 4096 + turned(c, row), in ? base + (int64_t)rows[row] * p.ldb + n0 + 8 * c : base, in);
      }
    }
    cp_async_commit();
  };
  if (any) {
    const T* w1 = static_cast<const T*>(p.w1) + (int64_t)adapter * p.r * p.K;
    const int row0 = tid >> 3, c = tid & 7;
    const T* xp[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) xp[j] = static_cast<const T*>(p.x) + (int64_t)rows[row0 + 64 * j] * p.ldx + c * 8;
    const int chunks = (p.K + 127) / 128, mine = rank < chunks ? (chunks - rank + C - 1) / C : 0;
    auto fetch = [&](int i) {
      if (i < mine) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int k = (rank + i * C) * 128 + 64 * b;
          const bool live = k + c * 8 < p.K;
          const uint32_t at = base_addr + i % S * L::kStage + b * L::kBlock + row0 * 128 + turned(c, row0);   // 64 rows on: the same turn
          if (k + 64 <= p.K && n == R && p.r == RT) {
#pragma unroll
            for (int j = 0; j < 2; ++j) copy16(at + j * 8192, xp[j] + k);
#pragma unroll
            for (int j = 0; j < RT / 64; ++j) copy16(at + 16384 + j * 8192, w1 + (int64_t)(row0 + 64 * j) * p.K + k + c * 8);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const bool in = live && row0 + 64 * j < n;
              copy16(at + j * 8192, in ? xp[j] + k : static_cast<const T*>(p.x), in);
            }
#pragma unroll
            for (int j = 0; j < RT / 64; ++j) {
              const bool in = live && row0 + 64 * j < p.r;
              copy16(at + 16384 + j * 8192, in ? w1 + (int64_t)(row0 + 64 * j) * p.K + k + c * 8 : w1, in);
            }
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch(i);
    for (int i = 0; i < mine; ++i) {
      cp_async_wait_group<S - 2>();
      fence_async_smem();
      __syncthreads();
      if (warp == 0) {
        tc_fence_after();
        const uint32_t at = base_addr + i % S * L::kStage;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16_warp(tmem, desc_sw128(at + b * L::kBlock) + 2 * k, desc_sw128(at + b * L::kBlock + 16384) + 2 * k, kFirst,
                         i > 0 || b > 0 || k > 0 ? 1u : 0u);
        mma_commit_warp(&full[i % S]);
      }
      if (i > 0) tc_wait(&full[(i - 1) % S], ((i - 1) / S) & 1, p, dead);      // its stage is filled next
      fetch(i + S - 1);
    }
    if (mine > 0) tc_wait(&full[(mine - 1) % S], ((mine - 1) / S) & 1, p, dead);
    cp_async_wait_all();
    tc_fence_after();
    __syncthreads();
    // this block's part of u: row 32 (warp % 4) + lane, a quarter of the ranks
    const int row = (warp & 3) * 32 + lane;
#pragma unroll 1
    for (int col = (warp >> 2) * (RT / 4); col < ((warp >> 2) + 1) * (RT / 4); col += 16) {
      uint32_t v[16] = {};
      if (mine > 0) {
        tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + col, v);
        tmem_ld_wait();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(smem + L::kPartAt + row * RT * 4 + turned(col / 4 + i, row)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
    tc_fence_before();
  }
  // the first operands of the second product are on their way while the others' parts are waited for
  if (C > 1) cluster_arrive();
  if (any) fetch_b(half);
  if (any && L::kApart) fetch_base(half);
  if (C > 1) cluster_wait();
  else __syncthreads();
  if (any) {
    // every block adds up its share of the rows, eight ranks a lane, and sends the operand to all
    const float s = p.scale ? p.scale[adapter] : p.scale_value;
    const int share = (R + C - 1) / C;
    for (int from = 0; from < share * (RT / 8); from += NTH) {
      const int i = from + tid, row = rank * share + i / (RT / 8), c8 = i % (RT / 8);
      const bool in = i < share * (RT / 8) && row < R;
      float f[8] = {};
      if (in) {
        const uint32_t line = base_addr + L::kPartAt + row * RT * 4;
        float4 o[16] = {};                             // all blocks' parts on their way
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c < C) {
            const uint32_t at = mapa_shared(line, c);
            o[2 * c] = ld_cluster4(at + turned(2 * c8, row)), o[2 * c + 1] = ld_cluster4(at + turned(2 * c8 + 1, row));
          }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          f[0] += o[2 * c].x, f[1] += o[2 * c].y, f[2] += o[2 * c].z, f[3] += o[2 * c].w;
          f[4] += o[2 * c + 1].x, f[5] += o[2 * c + 1].y, f[6] += o[2 * c + 1].z, f[7] += o[2 * c + 1].w;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 8 * c8 < p.r ? f[e] * s : 0.0f;      // as in the rings
        if (p.u && row < n && 8 * c8 < p.r) {
          float4* u = reinterpret_cast<float4*>(p.u + (int64_t)rows[row] * p.r + 8 * c8);
          u[0] = make_float4(kept<T>(f[0]), kept<T>(f[1]), kept<T>(f[2]), kept<T>(f[3]));
          u[1] = make_float4(kept<T>(f[4]), kept<T>(f[5]), kept<T>(f[6]), kept<T>(f[7]));
        }
      }
      uint4 hi, lo;
      float back = 1.0f;
      if constexpr (kHalves<T>) {                      // a row's power of two, as in the rings
        float most = 0.0f, to;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]));
#pragma unroll
        for (int d = 1; d < RT / 8; d *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        row_power(__float_as_uint(most), to, back);
        split_f16(f[0] * to, f[1] * to, hi.x, lo.x), split_f16(f[2] * to, f[3] * to, hi.y, lo.y);
        split_f16(f[4] * to, f[5] * to, hi.z, lo.z), split_f16(f[6] * to, f[7] * to, hi.w, lo.w);
      } else {
        split_bf16(f[0], f[1], hi.x, lo.x), split_bf16(f[2], f[3], hi.y, lo.y);
        split_bf16(f[4], f[5], hi.z, lo.z), split_bf16(f[6], f[7], hi.w, lo.w);
      }
      if (in) {
        const uint32_t at = base_addr + L::kA + c8 / 8 * 16384 + row * 128 + turned(c8 & 7, row);
        for (int c = 0; c < C; ++c) {
          const uint32_t to = mapa_shared(at, c);
          st_cluster4(to, hi);
          st_cluster4(to + NB * 16384, lo);
          if (kHalves<T> && c8 == 0) st_cluster1(mapa_shared(smem_u32(&down[kHalves<T> ? row : 0]), c), back);
        }
      }
    }
  }
  if (C > 1) cluster_sync_all();                       // u is there, and nobody reads another block's part any more
  else __syncthreads();

  if (!any) fetch_b(half);
  if (!any || !L::kApart) fetch_base(half);
  const uint32_t d = tmem + 128 + half * 128;
  for (int j = half; j < steps; j += 2) {
    cp_async_wait_group<1>();                          // B; base may be on its way
    fence_async_smem();
    half_sync(half);
    if (any) {
      if (hw == 0) {
        tc_fence_after();
        const uint32_t a = base_addr + L::kA, b = base_addr + half * L::kB;
#pragma unroll
        for (int part = 1; part >= 0; --part)          // the smaller numbers first
#pragma unroll
          for (int blk = 0; blk < NB; ++blk)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_f16_warp(d, desc_sw128(a + (part * NB + blk) * 16384) + 2 * k, desc_sw128(b + blk * 16384) + 2 * k, kSecond,
                           part == 1 && blk == 0 && k == 0 ? 0u : 1u);
        mma_commit_warp(&done[half]);
      }
      tc_wait(&done[half], (j >> 1) & 1, p, dead);
      __syncwarp();
      tc_fence_after();
    }
    fetch_b(j + 2);
    cp_async_wait_group<1>();                          // base
    half_sync(half);
    const int row = (warp & 3) * 32 + lane;
    const float f = kHalves<T> && any ? down[kHalves<T> ? row : 0] : 1.0f;
    uint8_t* line = smem + L::kBaseAt + half * L::kBase + row * 256;
    uint32_t v[2][32] = {};
    if (any) {
      const uint32_t at = d + ((uint32_t)((warp & 3) * 32) << 16) + (hw >> 2) * 64;
      tmem_ld32(at, v[0]);
      tmem_ld32(at + 32, v[1]);
      tmem_ld_wait();
    }
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      uint4* at = reinterpret_cast<uint4*>(line + turned((hw >> 2) * 8 + h, row));
      const uint4 b = p.base != nullptr ? *at : make_uint4(0, 0, 0, 0);
      const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = pack2<T>(fmaf(__uint_as_float(v[h / 4][h % 4 * 8 + 2 * e]), f, elem<T>(bw, 2 * e)),
                        fmaf(__uint_as_float(v[h / 4][h % 4 * 8 + 2 * e + 1]), f, elem<T>(bw, 2 * e + 1)));
      *at = make_uint4(o[0], o[1], o[2], o[3]);
    }
    tc_fence_before();
    half_sync(half);
    const int n0 = (rank + j * C) * 128, c = ht & 15;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = (ht >> 4) + 16 * i;
      if (row < n && n0 + 8 * c < p.N)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.y) + (int64_t)rows[row] * p.N + n0 + 8 * c) =
            *reinterpret_cast<const uint4*>(smem + L::kBaseAt + half * L::kBase + row * 256 + turned(c, row));
    }
    half_sync(half);
    fetch_base(j + 2);
  }
  cp_async_wait_all();
  dead = __any_sync(0xffffffffu, dead);               // whole warps
  if (dead) {                                          // products may still be on their way: they take microseconds
    if (hw == 0) mma_commit_warp(&drain[half]);
    mbar_wait_bounded(&drain[half], 0, 10000000);
  }
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// The gradients of adapters by tcgen05: out[a] = sum over a's rows of v[m]^T x[m] for 256 columns of x a block, both operands with the
// rows as k: 128 bytes of a row side by side (swizzled), 8 rows a group. 64 rows a stage: x by asynchronous copies, v through registers,
// taken apart on the way: bf16's two numbers as they are kept; fp16's split in two by a power of two for each rank, from the largest v of
// the block's rows (read once before: the backward pass of 8192 rows rank 128 takes 141 us, bf16's 106), which leaves an error of 2^-22 of a number or 2^-39 of the largest. A cluster's blocks take stages in turn and add up in a fixed order.
// Bound: the steps of a stage one after the other (copies there, products issued, the last ones done: 1700 cycles at rank 64, 2000 at 128,
// products alone 512). 8192 rows rank 64, both gradients of 4096 columns, 42 us: 3.2 TB/s. (Rows in core matrices of 16 bytes
// instead of 128 took 2800 cycles a stage: every 16 bytes are a write of their own.)
template <int RT>
struct OuterTc {
  static constexpr int kThreads = 512, BW = 256, kRows = 64, kStages = 4;
  static constexpr int kBlock = kRows * 128;                           // of 64 columns
  static constexpr int kX = BW / 64 * kBlock, kHalf = RT / 64 * kBlock, kV = 2 * kHalf;
  static constexpr int kNeed = kStages * kX + 2 * kV, kSmem = kNeed + 1024;
  static constexpr int kByRank = RT + 4, kByCol = BW + 4;              // pitch of the sums in floats: [BW][kByRank] or [RT][kByCol]
  static_assert(BW * kByRank * 4 <= kNeed && RT * kByCol * 4 <= kNeed, "the sums lie over all of it");
};
__device__ __forceinline__ uint64_t desc_rows(uint32_t saddr) {         // blocks of 64 columns by 64 rows, groups of 8 rows
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}

template <typename T, int RT>
__global__ void __launch_bounds__(OuterTc<RT>::kThreads, 1) outer_tc_kernel(const __grid_constant__ OuterPair pair) {
  using L = OuterTc<RT>;
  constexpr int S = L::kStages, BW = L::BW, NTH = L::kThreads, KR = L::kRows;
  constexpr int VI = RT / 8, VROWS = NTH / VI < KR ? NTH / VI : KR, VP = KR / VROWS;      // pieces of a row of v, rows a pass, passes
  constexpr uint32_t kDesc = idesc_f16(128, RT) | (kPairs<T> ? (1u << 7) | (1u << 10) : 0u) | (1u << 15) | (1u << 16);
  const int second = (int)blockIdx.x >= pair.of[0].blocks;
  const OuterParams& p = pair.of[second];
  const int block = (int)blockIdx.x - (second ? pair.of[0].blocks : 0);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[S], drain;
  __shared__ uint32_t tmem_at, most[kHalves<T> ? RT : 1];
  __shared__ float down[kHalves<T> ? RT : 1];          // what the ranks of v were divided by
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int C = p.cluster, rank = block % C, n0 = block / C * BW, a = blockIdx.y;
  grid_dep_wait();                                     // tensor memory is not held while others may need it
  if (warp == 0) tmem_alloc(&tmem_at, 2 * RT);
  if (tid == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1 + pair.hold);
    mbar_init(&drain, 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at, base = smem_u32(smem);
  bool dead = false;
  const Plan plan{p.plan, p.L, p.M};
  const int from = p.plan ? plan.first(a) : 0, rows = p.plan ? plan.first(a + 1) - from : p.M;
  const int chunks = (rows + KR - 1) / KR, mine = rank < chunks ? (chunks - rank + C - 1) / C : 0;
  auto row_of = [&](int i, int at) {                   // of the block's chunk i; -1: none
    at += (rank + i * C) * KR;
    return i < mine && at < rows ? p.plan ? plan.row(from + at) : at : -1;
  };
  // x: a warp's lanes hold a row's 256 columns, rows warp + 16 j; their numbers a chunk ahead
  const bool in = n0 + lane * 8 < p.K;
  const T* xc = static_cast<const T*>(p.x) + (in ? n0 + lane * 8 : 0);
  int xr[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) xr[j] = row_of(0, warp + 16 * j);
  auto fetch = [&](int i) {
    if (i < mine) {
      const uint32_t at = base + i % S * L::kX + (lane >> 3) * L::kBlock + warp * 128 + turned(lane & 7, warp);
#pragma unroll
      for (int j = 0; j < 4; ++j) copy16(at + j * 2048, xc + (int64_t)max(xr[j], 0) * p.ldx, in && xr[j] >= 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) xr[j] = row_of(i + 1, warp + 16 * j);
    }
    cp_async_commit();
  };
  // v: eight ranks of a row a thread, rows v0 + VROWS j
  const int v8 = tid % VI, v0 = tid / VI;
  const bool v_in = 8 * v8 < p.r && v0 < VROWS;
  int vr[VP];
  uint4 v[VP][2];
#pragma unroll
  for (int j = 0; j < VP; ++j) vr[j] = v_in ? row_of(0, v0 + VROWS * j) : -1;
  auto read = [&](int i) {                             // chunk i, whose row numbers are there
#pragma unroll
    for (int j = 0; j < VP; ++j) {
      const uint4* src = reinterpret_cast<const uint4*>(p.v + (int64_t)max(vr[j], 0) * p.r + 8 * v8);
      v[j][0] = vr[j] >= 0 ? src[0] : make_uint4(0, 0, 0, 0);
      v[j][1] = vr[j] >= 0 ? src[1] : make_uint4(0, 0, 0, 0);
      vr[j] = v_in ? row_of(i + 1, v0 + VROWS * j) : -1;
    }
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch(i);
  float up[8];
  if constexpr (kHalves<T>) {                          // a rank's power of two, from the block's rows
    for (int k = tid; k < RT; k += NTH) most[k] = 0;
    __syncthreads();
    uint32_t top[8] = {};
#pragma unroll 2
    for (int i = 0; i < mine; ++i)
#pragma unroll
      for (int j = 0; j < VP; ++j) {
        const int row = v_in ? row_of(i, v0 + VROWS * j) : -1;
        const uint4* src = reinterpret_cast<const uint4*>(p.v + (int64_t)max(row, 0) * p.r + 8 * v8);
        const uint4 f = row >= 0 ? src[0] : make_uint4(0, 0, 0, 0), g = row >= 0 ? src[1] : make_uint4(0, 0, 0, 0);
        const uint32_t w[8] = {f.x, f.y, f.z, f.w, g.x, g.y, g.z, g.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) top[e] = max(top[e], w[e] & 0x7fffffffu);
      }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (top[e]) atomicMax(&most[8 * v8 + e], top[e]);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float back;
      row_power(most[8 * v8 + e], up[e], back);
      if (v0 == 0) down[8 * v8 + e] = back;
    }
  }
  read(0);
  for (int i = 0; i < mine; ++i) {
    const int vat = S * L::kX + (i & 1) * L::kV;
    if (v0 < VROWS) {
#pragma unroll
      for (int j = 0; j < VP; ++j) {
        uint8_t* at = smem + vat + (v8 >> 3) * L::kBlock + (v0 + VROWS * j) * 128 + turned(v8 & 7, v0 + VROWS * j);
        const uint4 f = v[j][0], g = v[j][1];
        uint4 hi, lo;
        if constexpr (kHalves<T>) {
          auto two = [&](uint32_t a, uint32_t b, int e, uint32_t& h, uint32_t& l) {
            split_f16(__uint_as_float(a) * up[e], __uint_as_float(b) * up[e + 1], h, l);
          };
          two(f.x, f.y, 0, hi.x, lo.x), two(f.z, f.w, 2, hi.y, lo.y), two(g.x, g.y, 4, hi.z, lo.z), two(g.z, g.w, 6, hi.w, lo.w);
        } else {
          hi = make_uint4(__byte_perm(f.x, f.y, 0x5410), __byte_perm(f.z, f.w, 0x5410), __byte_perm(g.x, g.y, 0x5410),
                          __byte_perm(g.z, g.w, 0x5410));
          lo = make_uint4(__byte_perm(f.x, f.y, 0x7632), __byte_perm(f.z, f.w, 0x7632), __byte_perm(g.x, g.y, 0x7632),
                          __byte_perm(g.z, g.w, 0x7632));
        }
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + L::kHalf) = lo;
      }
    }
    read(i + 1);
    cp_async_wait_group<S - 2>();
    fence_async_smem();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      const uint32_t xs = base + i % S * L::kX, vs = base + vat;
#pragma unroll
      for (int half = 1; half >= 0; --half)            // the smaller numbers first
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < KR / 16; ++k)
            mma_f16_warp(tmem + c * RT, desc_rows(xs + c * 2 * L::kBlock + k * 2048), desc_rows(vs + half * L::kHalf + k * 2048), kDesc, i > 0 || half == 0 || k > 0 ? 1u : 0u);
      mma_commit_warp(&full[i % S]);
    }
    if (i > 0) tc_wait(&full[(i - 1) % S], ((i - 1) / S) & 1, pair, dead);       // its stage, and its v, are filled next
    fetch(i + S - 1);
  }
  if (mine > 0) tc_wait(&full[(mine - 1) % S], ((mine - 1) / S) & 1, pair, dead);
  cp_async_wait_all();
  tc_fence_after();
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  const bool by_rank = p.step_r == 1;                  // else columns lie side by side
  {
    const int c = (warp >> 2) & 1, col = c * 128 + (warp & 3) * 32 + lane;
#pragma unroll 1
    for (int k = (warp >> 3) * (RT / 2); k < ((warp >> 3) + 1) * (RT / 2); k += 16) {
      uint32_t w[16] = {};
      if (mine > 0) {
        tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c * RT + k, w);
        tmem_ld_wait();
      }
      if constexpr (kHalves<T>)
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * down[k + e]);
      if (by_rank) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<uint4*>(part + col * L::kByRank + k + 4 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) part[(k + e) * L::kByCol + col] = __uint_as_float(w[e]);
      }
    }
  }
  tc_fence_before();
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  // eight adjacent numbers of the gradient a thread
  T* out = static_cast<T*>(p.out) + (int64_t)a * p.r * p.K;
  for (int i = rank * NTH + tid; i < RT * BW / 8; i += C * NTH) {
    const int k = by_rank ? i % VI * 8 : i / (BW / 8), col = by_rank ? i / VI : i % (BW / 8) * 8;
    const uint32_t at = base + 4 * (by_rank ? col * L::kByRank + k : k * L::kByCol + col);
    float f[8] = {};
    for (int c0 = 0; c0 < C; c0 += 4) {                // in order, four blocks' parts on their way
      float4 o[8] = {};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + e < C) {
          const uint32_t src = mapa_shared(at, c0 + e);
          o[2 * e] = ld_cluster4(src), o[2 * e + 1] = ld_cluster4(src + 16);
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[0] += o[2 * e].x, f[1] += o[2 * e].y, f[2] += o[2 * e].z, f[3] += o[2 * e].w;
        f[4] += o[2 * e + 1].x, f[5] += o[2 * e + 1].y, f[6] += o[2 * e + 1].z, f[7] += o[2 * e + 1].w;
      }
    }
    if (k < p.r && n0 + col < p.K)
      *reinterpret_cast<uint4*>(out + k * p.step_r + (int64_t)(n0 + col) * p.step_k) =
          make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
  if (C > 1) cluster_sync_all();
  dead = __any_sync(0xffffffffu, dead);               // whole warps
  if (dead) {                                          // products may still be on their way: they take microseconds
    if (warp == 0) mma_commit_warp(&drain);
    mbar_wait_bounded(&drain, 0, 10000000);
  }
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 2 * RT);
}

// Allows a kernel its dynamic shared memory, once a device (the call costs as much as a launch). `limit`: 0 or what was allowed.
template <typename K>
cudaError_t allow_smem(K* kernel, size_t smem, size_t (&limit)[64]) {
  if (smem <= 40 * 1024) return cudaSuccess;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && limit[dev] >= smem)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess && dev < 64) limit[dev] = smem;
  return e;
}

// Clusters of n such blocks that the GPU holds at once. They are placed within groups of SMs, so that fewer blocks fit in
// larger ones: 16 clusters of 8 take two rounds (rings, 512 rows 4096 -> 4096 rank 64 bf16: 25.9 us, 16 of 4 16.5).
template <auto Kernel, int NT = kThreads>
int clusters_at_once(int n, size_t smem) {
  static int cache[64][9] = {};                        // plus one
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 0;
  if (cache[dev][n] == 0) {
    static size_t limit[64] = {};
    if (allow_smem(Kernel, smem, limit) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)n, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int most = 0;
    if (cudaOccupancyMaxActiveClusters(&most, Kernel, &cfg) != cudaSuccess) most = 0;
    cache[dev][n] = most + 1;
  }
  return cache[dev][n] - 1;
}

template <auto Kernel, int NT = kThreads, typename P>
cudaError_t launch_clusters(const P& p, dim3 grid, size_t smem, cudaStream_t st) {
  static size_t limit[64] = {};
  const cudaError_t e = allow_smem(Kernel, smem, limit);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = pdl_enabled() ? attr : attr + 1;
  cfg.numAttrs = (pdl_enabled() ? 1 : 0) + (p.cluster > 1 ? 1 : 0);
  return cudaLaunchKernelEx(&cfg, Kernel, p);
}

// Whether tiles of 16 rows are so few that the GPU holds `blocks` blocks or more of each at once (on 148 SMs).
inline bool few_tiles(int64_t M, int L, bool indexed, int blocks) { return M / 16 + (indexed ? L / 2 : 0) <= 144 / blocks; }
// Whether the tensor-core kernel takes the call (if every address is on 16 bytes; sides: inputs and outputs together): 16-bit rows, ranks
// above 32, half a tile an adapter on average, and more tiles than the rings hold in 16 rows or, above rank 64, 4096 rows or 1024 and
// 2^23 elements of x and y. Both sides, us, bf16, this kernel and the rings. Rank 64, 4096 -> 4096, one adapter: 256 rows 17.5 and
// 11.0, 1024 17.9 and 15.6, 2048 22 and 24, 8192 50 and 73; 8 adapters, 1024 rows 20.5 and 18.9, 16, 8192 rows 66 and 112. Rank 128,
// 4096 -> 4096: 256 rows 22.8 and 17.0, 1024 23.3 and 24.4, 8192 56 and 157; 1024 -> 1024, 1024 rows 16.2 and 11.5, 2048 16.0 and
// 13.7, 4096 16.9 and 26.4; 512 -> 512, 2048 rows 13.0 and 9.3, 4096 14.0 and 17.6.
inline bool tensor_sized(int64_t M, int64_t sides, int L, int r, bool indexed, bool wide16) {
  if (!wide16 || r <= 32 || M < 64 * (int64_t)(indexed ? L : 1)) return false;
  return r <= 64 ? !few_tiles(M, L, indexed, 2) : M >= 4096 || (M >= 1024 && M * sides >= 1 << 23);
}
// Rows of a ring kernel's tile: 32 need half of the reads of the adapters, 16 half of the shared memory and leave a block half of the
// work: 16 where an adapter has no more on average, above rank 64, and while the GPU holds several blocks of each tile at once
// (two, four at 32 bits above rank 16; up to rank 16 an SM holds two blocks). 32 rows and 16, us, 4096 -> 4096 bf16: rank 16, one adapter, 64 rows 6.8 and 5.1, 512 8.8 and 6.7, 1000
// 9.2 and 8.3, rank 8 1500 12.8 and 14.1; rank 64, 128 rows 13.5 and 9.2, 512 16.5 and 11.2, 1000 of 4 adapters 26.2 and 18.6; f32, rank
// 64, 200 rows of 2 25.2 and 17.8, 1000 40.8 and 46.9.
inline int ring_rows(int64_t M, int L, int r, bool indexed, bool wide16) {
  const bool few = few_tiles(M, L, indexed, r <= 16 || wide16 ? 2 : 4);
  return r <= 64 && M > 16 * (int64_t)(indexed ? L : 1) && !few ? 32 : 16;
}
// Rows of a tile of the plan: the larger of what the kernels of both directions may take.
inline int tile_rows(int64_t M, int64_t sides, int L, int r, bool indexed, bool wide16) {
  return tensor_sized(M, sides, L, r, indexed, wide16) ? 128 : ring_rows(M, L, r, indexed, wide16);
}
// Clusters for tiles of R rows.
inline int64_t max_tiles(int64_t M, int L, int R, bool indexed, bool planned) {
  if (!indexed) return (M + R - 1) / R;
  if (!planned && finds_itself(M, L, R)) return M;
  const int64_t all = (M + R - 1) / R + L + 1;
  return all < M ? all : M;
}

template <typename T, int RT, int MT, bool TRANS, bool RAGGED>
cudaError_t launch_ring(Params p, int64_t tiles, int64_t likely, cudaStream_t st) {
  // blocks of a tile: as many as the GPU holds at once
  constexpr auto kernel = lora_kernel<T, RT, MT, TRANS, RAGGED>;
  constexpr size_t smem = Ring<T, RT, MT>::kSmem;
  p.cluster = 1;
  while (p.cluster < 8 && likely <= clusters_at_once<kernel>(2 * p.cluster, smem)) p.cluster *= 2;
  return launch_clusters<kernel>(p, dim3((unsigned)(tiles * p.cluster)), smem, st);
}
// Whether every address is on 16 bytes (rows of ranks on 8).
template <typename T>
bool aligned(const Params& p) {
  constexpr int EL = 16 / (int)sizeof(T);
  return p.K % EL == 0 && p.N % EL == 0 && on(p.x, 16) && (p.M <= 1 || p.ldx % EL == 0) && on(p.w1, 16) && on(p.w2, 16) &&
         on(p.base, 16) && (p.M <= 1 || p.ldb % EL == 0) && on(p.y, 16) && p.r % (EL / 2) == 0;
}

// Whether some address is off 4 bytes.
template <typename T>
bool off_words(const Params& p) {
  return sizeof(T) == 2 && (p.K % 2 || p.N % 2 || p.r % 2 || !on(p.x, 4) || (p.M > 1 && p.ldx % 2) || !on(p.w1, 4) || !on(p.w2, 4) ||
                            !on(p.base, 4) || (p.M > 1 && p.ldb % 2) || !on(p.y, 4));
}

template <typename T, int RT>
cudaError_t launch_tc(Params p, int64_t tiles, int64_t likely, cudaStream_t st) {
  // blocks of a tile: as many as the GPU holds at once, and no more than shorten a block's work
  constexpr auto kernel = lora_tc_kernel<T, RT>;
  constexpr size_t smem = Tc<RT>::kSmem;
  auto steps = [&](int c) { return ((p.K + 127) / 128 + c - 1) / c + ((p.N + 127) / 128 + c - 1) / c; };
  p.cluster = 8;
  while (p.cluster > 1 && likely > clusters_at_once<kernel, Tc<RT>::kThreads>(p.cluster, smem)) --p.cluster;
  while (p.cluster > 1 && steps(p.cluster - 1) == steps(p.cluster)) --p.cluster;
  return launch_clusters<kernel, Tc<RT>::kThreads>(p, dim3((unsigned)(tiles * p.cluster)), smem, st);
}

template <typename T, bool TRANS>
cudaError_t run_as(Params p, cudaStream_t st) {
  const bool indexed = p.index != nullptr, planned = p.plan != nullptr;
  const int whole = tile_rows(p.M, (int64_t)p.K + p.N, p.L, p.r, indexed, sizeof(T) == 2);
  const bool on16 = aligned<T>(p);
  auto tiles_of = [&](int R) {             // and how many of them are likely to have rows
    p.split = planned ? whole / R : 1;
    const int64_t tiles = planned ? max_tiles(p.M, p.L, whole, indexed, true) * p.split : max_tiles(p.M, p.L, R, indexed, false);
    // an adapter of many tiles leaves half of its last one empty on average, one of one or two more than that; where most have fewer rows
    // than a tile, each is one
    const int64_t all = (int64_t)R * p.L;
    int64_t likely = (p.M + R - 1) / R + (!indexed ? 0 : p.M >= 2 * all ? p.L / 2 : p.M >= all ? 3 * p.L / 4 : p.L - 1);
    if (likely > p.M) likely = p.M;
    return std::pair<int64_t, int64_t>(tiles, likely < tiles ? likely : tiles);
  };
  if constexpr (!TRANS && sizeof(T) == 2) {
    if (on16 && p.r % 8 == 0 && on(p.u, 16) && tensor_sized(p.M, (int64_t)p.K + p.N, p.L, p.r, indexed, true)) {
      const auto t = tiles_of(128);
      return p.r <= 64 ? launch_tc<T, 64>(p, t.first, t.second, st) : launch_tc<T, 128>(p, t.first, t.second, st);
    }
  }
  const int R = on16 ? ring_rows(p.M, p.L, p.r, indexed, sizeof(T) == 2) : 16;
  const auto t = tiles_of(R);
  if (on16) {
#define GLAD_LORA(RT)                                                                        \
  return R == 32 ? launch_ring<T, RT, 2, TRANS, false>(p, t.first, t.second, st) \
                 : launch_ring<T, RT, 1, TRANS, false>(p, t.first, t.second, st)
    if (p.r <= 16) GLAD_LORA(16);
    if (p.r <= 32) GLAD_LORA(32);
    if (p.r <= 64) GLAD_LORA(64);
#undef GLAD_LORA
    return launch_ring<T, 128, 1, TRANS, false>(p, t.first, t.second, st);
  }
  p.half = off_words<T>(p);
  if (p.r <= 16) return launch_ring<T, 16, 1, TRANS, true>(p, t.first, t.second, st);
  if (p.r <= 32) return launch_ring<T, 32, 1, TRANS, true>(p, t.first, t.second, st);
  if (p.r <= 64) return launch_ring<T, 64, 1, TRANS, true>(p, t.first, t.second, st);
  return launch_ring<T, 128, 1, TRANS, true>(p, t.first, t.second, st);
}
// trans: w1 is B [L, K, r] and w2 A [L, r, N], else A [L, r, K] and B [L, N, r].
template <typename T>
cudaError_t run(Params p, bool trans, cudaStream_t st) {
  return trans ? run_as<T, true>(p, st) : run_as<T, false>(p, st);
}
// Whether a backward call goes to the tensor-core kernel once its adapters are transposed.
template <typename T>
bool wants_transposed(const Params& p) {
  return sizeof(T) == 2 && p.r % 8 == 0 && on(p.u, 16) && tensor_sized(p.M, (int64_t)p.K + p.N, p.L, p.r, p.index != nullptr, true) &&
         aligned<T>(p);
}

// Whether the gradients of adapters go to the tensor-core kernel: 16-bit rows, multiples of 8 ranks above 16. Backward passes 4096 -> 4096
// with the rings and with this kernel, us, bf16: rank 16, 8192 rows 65 and 76, 1024 rows and 16 adapters 42.6 and 42.7; rank 32, 87
// and 88, 65 and 48; rank 64, 117 and 88, 127 and 74; rank 128, 197 and 106, 221 and 101; 64 rows rank 32 13.3 and 14.9, rank 64 21.2 and
// 20.4. fp16: rank 32, 8192 rows 110 and 107, 1024 rows and 16 adapters 65 and 55; rank 128 289 and 141, 224 and 110.
inline bool outer_sized(int r) { return r > 16; }

template <typename T, int RT>
cudaError_t launch_outer_tc(OuterPair pair, int count, int64_t rows, cudaStream_t st) {
  constexpr auto kernel = outer_tc_kernel<T, RT>;
  constexpr size_t smem = OuterTc<RT>::kSmem;
  constexpr int BW = OuterTc<RT>::BW;
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) tiles += (int64_t)((pair.of[i].K + BW - 1) / BW) * pair.of[i].L;
  // blocks of a tile: as many as the GPU holds at once, two stages of rows each or more
  int C = 1;
  while (C < 8 && rows >= (int64_t)C * 4 * OuterTc<RT>::kRows && tiles <= clusters_at_once<kernel, OuterTc<RT>::kThreads>(2 * C, smem)) C *= 2;
  unsigned blocks = 0;
  for (int i = 0; i < count; ++i) {
    pair.of[i].cluster = C;
    pair.of[i].blocks = (pair.of[i].K + BW - 1) / BW * C;
    blocks += (unsigned)pair.of[i].blocks;
  }
  pair.cluster = C;
  return launch_clusters<kernel, OuterTc<RT>::kThreads>(pair, dim3(blocks, (unsigned)pair.of[0].L), smem, st);
}

// One or two gradients (count).
template <typename T>
cudaError_t run_outer(OuterPair pair, int count, cudaStream_t st) {
  constexpr int EL = 16 / (int)sizeof(T), BW = 8 * EL;
  const OuterParams& first = pair.of[0];
  const int RT = first.r <= 16 ? 16 : 32, ranks = (first.r + RT - 1) / RT;
  const int64_t rows = first.plan ? (first.M + first.L - 1) / first.L : first.M;       // of an adapter, on average
  int64_t tiles = 0;
  bool ring = first.r % 4 == 0, wide = true;
  for (int i = 0; i < count; ++i) {
    OuterParams& p = pair.of[i];
    tiles += (int64_t)((p.K + BW - 1) / BW) * p.L * ranks;
    wide = wide && on(p.out, 16);
    p.pitch = (uint32_t)(p.ldx * (int64_t)sizeof(T));
    p.half = sizeof(T) == 2 && (p.K % 2 || !on(p.x, 4) || (p.M > 1 && p.ldx % 2));
    ring = ring && p.K % EL == 0 && on(p.x, 16) && (p.M <= 1 || p.ldx % EL == 0) && p.ldx < (int64_t)1 << 29 && on(p.v, 16);
  }
  if constexpr (sizeof(T) == 2) {
    if (ring && wide && first.r % 8 == 0 && outer_sized(first.r)) {
      return first.r <= 64 ? launch_outer_tc<T, 64>(pair, count, rows, st) : launch_outer_tc<T, 128>(pair, count, rows, st);
    }
  }
  // blocks of a tile: while every warp keeps a few groups of 16 rows and the tiles alone do not fill the GPU
  int C = 1;
  while (C < 8 && rows >= (int64_t)C * 2 * kWarps * 16 && tiles * C * 2 <= 2 * num_sms()) C *= 2;
  unsigned blocks = 0;
  for (int i = 0; i < count; ++i) {
    pair.of[i].cluster = C;
    pair.of[i].blocks = (pair.of[i].K + BW - 1) / BW * C;
    blocks += (unsigned)pair.of[i].blocks;
  }
  pair.cluster = C;
  const dim3 grid(blocks, (unsigned)first.L, (unsigned)ranks);
  if (RT == 16)
    return ring ? launch_clusters<outer_kernel<T, 16, false>>(pair, grid, OuterRing<T, 16>::kSmem, st)
                : launch_clusters<outer_kernel<T, 16, true>>(pair, grid, OuterRing<T, 16>::kSmem, st);
  return ring ? launch_clusters<outer_kernel<T, 32, false>>(pair, grid, OuterRing<T, 32>::kSmem, st)
              : launch_clusters<outer_kernel<T, 32, true>>(pair, grid, OuterRing<T, 32>::kSmem, st);
}

}  // namespace lora
}  // namespace glad
