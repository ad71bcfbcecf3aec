// C entries of the low-rank adapters (glad_lora.cuh), and the order of rows by adapter that larger calls need.
#include "glad_lora.cuh"

#include <atomic>

namespace glad {
cudaError_t w4_status_word(uint32_t** word);          // glad_w4.cu: the device's status word

namespace lora {

extern template cudaError_t run<__half>(Params, bool, cudaStream_t);
extern template cudaError_t run<__nv_bfloat16>(Params, bool, cudaStream_t);
extern template cudaError_t run<float>(Params, bool, cudaStream_t);
extern template bool wants_transposed<__half>(const Params&);
extern template bool wants_transposed<__nv_bfloat16>(const Params&);
extern template bool wants_transposed<float>(const Params&);
extern template cudaError_t run_outer<__half>(OuterPair, int, cudaStream_t);
extern template cudaError_t run_outer<__nv_bfloat16>(OuterPair, int, cudaStream_t);
extern template cudaError_t run_outer<float>(OuterPair, int, cudaStream_t);

namespace {

constexpr int kPlanThreads = 1024;

// Counting warps, as many as shared memory has counters for, and its size with them, which is largest at the most adapters.
constexpr int plan_warps(int L) { return L < 1024 ? 32 : L < 4096 ? 8 : 2; }
constexpr size_t plan_smem(int warps, int L) { return (size_t)(warps * (L + 1) + L + 2) * 4; }
constexpr size_t kPlanSmem = plan_smem(plan_warps(kMaxAdapters), kMaxAdapters);
static_assert(kPlanSmem >= plan_smem(plan_warps(1023), 1023) && kPlanSmem >= plan_smem(plan_warps(4095), 4095) && kPlanSmem <= 226 * 1024,
              "the most of any call");

struct PlanParams {
  const void* index;
  int32_t* plan;
  int M, L, index64, warps, tile_rows;
};

// A stable counting sort by one block: the first `warps` warps count the adapters of a run of rows each, the counts are added up by
// adapter, then by warp, and the warps place their rows. Rows of an adapter stay in order, so sums over them repeat. Latency: three
// passes over the index by one block (300 rows, 5 adapters: 9.6 us with cold caches).
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  extern __shared__ int32_t sh[];
  const int G = p.L + 1;                                // groups: adapters, then the rows without one
  int32_t* cnt = sh;                                    // [warps][G]
  int32_t* tile0 = sh + p.warps * G;                    // [G + 1]
  __shared__ int32_t sums[2][kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < p.warps * G; i += kPlanThreads) cnt[i] = 0;
  grid_dep_wait();
  __syncthreads();
  const int run = ((p.M + p.warps - 1) / p.warps + 31) / 32 * 32;
  const int64_t lo = (int64_t)warp * run;
  const int64_t hi = warp >= p.warps ? lo : lo + run < p.M ? lo + run : p.M;
  // a lane's groups of the next kAhead steps of 32 rows (-1: past the end), loaded at once
  constexpr int kAhead = 8;
  int ahead[kAhead];
  auto load = [&](int64_t m0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t m = m0 + 32 * j + lane;
      int64_t a = -1;
      if (m < hi) {
        a = p.index64 ? static_cast<const int64_t*>(p.index)[m] : (int64_t)static_cast<const int32_t*>(p.index)[m];
        a = a >= 0 && a < p.L ? a : p.L;
      }
      ahead[j] = (int)a;
    }
  };
  // calls f(first row of a step, this lane's group, the lanes of the same group), in order
  auto steps = [&](auto&& f) {
    for (int64_t m0 = lo; m0 < hi; m0 += 32 * kAhead) {
      if (run > 32 * kAhead) load(m0);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (m0 + 32 * j < hi) f(m0 + 32 * j, ahead[j], __match_any_sync(0xffffffffu, ahead[j]));
    }
  };
  load(lo);
  steps([&](int64_t, int a, uint32_t same) {
    if (a >= 0 && lane == __ffs(same) - 1) cnt[warp * G + a] += __popc(same);
    __syncwarp();
  });
  __syncthreads();
  int row_carry = 0, tile_carry = 0;
  for (int a0 = 0; a0 < G; a0 += kPlanThreads) {        // exclusive sums over the groups, of rows and of tiles
    const int a = a0 + tid;
    int rows = 0;
    if (a < G)
      for (int w = 0; w < p.warps; ++w) rows += cnt[w * G + a];
    const int tiles = (rows + p.tile_rows - 1) / p.tile_rows;
    int r = rows, t = tiles;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int ur = __shfl_up_sync(0xffffffffu, r, o), ut = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) r += ur, t += ut;
    }
    if (lane == 31) sums[0][warp] = r, sums[1][warp] = t;
    __syncthreads();
    static_assert(kPlanThreads == 1024, "a lane a warp");
    int wr = sums[0][lane], wt = sums[1][lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int ur = __shfl_up_sync(0xffffffffu, wr, o), ut = __shfl_up_sync(0xffffffffu, wt, o);
      if (lane >= o) wr += ur, wt += ut;
    }
    const int before_r = row_carry + (warp ? __shfl_sync(0xffffffffu, wr, warp ? warp - 1 : 0) : 0);
    const int before_t = tile_carry + (warp ? __shfl_sync(0xffffffffu, wt, warp ? warp - 1 : 0) : 0);
    row_carry += __shfl_sync(0xffffffffu, wr, 31);
    tile_carry += __shfl_sync(0xffffffffu, wt, 31);
    if (a < G) {
      int at = before_r + r - rows;
      p.plan[1 + a] = at;
      tile0[a] = before_t + t - tiles;
      for (int w = 0; w < p.warps; ++w) {
        const int c = cnt[w * G + a];
        cnt[w * G + a] = at;
        at += c;
      }
    }
    __syncthreads();
  }
  if (tid == 0) p.plan[0] = tile_carry, p.plan[1 + G] = p.M, tile0[G] = tile_carry;
  __syncthreads();
  int32_t* order = p.plan + 3 + p.L;
  steps([&](int64_t m0, int a, uint32_t same) {
    if (a >= 0) order[cnt[warp * G + a] + __popc(same & ((1u << lane) - 1))] = (int32_t)(m0 + lane);
    __syncwarp();
    if (a >= 0 && lane == __ffs(same) - 1) cnt[warp * G + a] += __popc(same);
    __syncwarp();
  });
  int32_t* tiles = order + p.M;
  for (int t = tid; t < tile_carry; t += kPlanThreads) {
    int a = 0, b = G;                                   // the last group whose first tile is at or before t
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (tile0[mid] <= t) a = mid;
      else b = mid;
    }
    tiles[2 * t] = a == p.L ? -1 : a;
    tiles[2 * t + 1] = p.plan[1 + a] + (t - tile0[a]) * p.tile_rows;
  }
}

// dst[l] = src[l]^T for two sets of matrices of 16-bit elements, [rows, cols] each (multiples of 8, on 16 bytes), in one launch:
// 64 x 64 elements a block, 16 bytes a lane in and out.
struct Transposes {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int rows[2], cols[2];
};
__global__ void __launch_bounds__(256) transpose_kernel(const Transposes p) {
  __shared__ __align__(16) uint16_t tile[64][72];       // [column][row]
  const int which = blockIdx.z & 1, rows = p.rows[which], cols = p.cols[which];
  const int64_t at = (int64_t)(blockIdx.z >> 1) * rows * cols;
  const int tall = rows > cols;                         // the long side runs along blockIdx.x
  const int r0 = (tall ? blockIdx.x : blockIdx.y) * 64, c0 = (tall ? blockIdx.y : blockIdx.x) * 64;
  if (r0 >= rows || c0 >= cols) return;
  grid_dep_wait();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = (threadIdx.x >> 3) + 32 * j, c = (threadIdx.x & 7) * 8;
    if (r0 + row < rows && c0 + c < cols) {
      const uint4 v = *reinterpret_cast<const uint4*>(p.src[which] + at + (int64_t)(r0 + row) * cols + c0 + c);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[c + e][row] = (uint16_t)(w[e >> 1] >> 16 * (e & 1));
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int col = (threadIdx.x >> 3) + 32 * j, r = (threadIdx.x & 7) * 8;
    if (c0 + col < cols && r0 + r < rows)
      *reinterpret_cast<uint4*>(p.dst[which] + at + (int64_t)(c0 + col) * rows + r0 + r) = *reinterpret_cast<const uint4*>(&tile[col][r]);
  }
}

std::atomic<uint32_t> g_hold{0}, g_wait_ns{2000000000u};

// What the tensor-core kernel needs beside the operands.
template <typename P>
cudaError_t tensor_setup(P& p) {
  p.wait_ns = g_wait_ns, p.hold = g_hold;
  return w4_status_word(&p.status);
}

template <typename F>
cudaError_t for_type(int dtype, F&& f) {
  if (dtype == GLAD_DTYPE_F16) return f(__half());
  if (dtype == GLAD_DTYPE_BF16) return f(__nv_bfloat16());
  return f(float());
}

const char* shape_wrong(int dtype, int64_t M, int64_t K, int64_t N, int L, int r, const void* index, int index_bytes) {
  if (!is_float(dtype)) return "x must be f32, f16 or bf16";
  if (M < 0 || M > 1 << 24) return "rows must be in [0, 2^24]";
  if (K < 1 || K > 1 << 24 || N < 1 || N > 1 << 24) return "inputs and outputs must be in [1, 2^24]";
  if (L < 1 || L > kMaxAdapters) return "the number of adapters must be in [1, 16384]";
  if (r < 1 || r > kMaxRank) return "the rank must be in [1, 128]";
  if (!index && L != 1 && M > 0) return "several adapters need an index";
  if (index && index_bytes != 4 && index_bytes != 8) return "the index must have 4 or 8 bytes";
  if (!on(index, index_bytes ? index_bytes : 4)) return "the index is not element-aligned";
  return nullptr;
}

int64_t plan_words(int64_t M, int L) { return 3 + L + M + 2 * max_tiles(M, L, 16, true, true); }

cudaError_t make_plan(const void* index, int index_bytes, int64_t M, int64_t sides, int L, int r, bool wide16, void* plan,
                      cudaStream_t st) {
  static size_t limit[64] = {};
  // 256 rows a counting warp if possible, which it holds in registers
  int warps = plan_warps(L);
  if (M < 256 * warps) warps = (int)((M + 255) / 256);
  const PlanParams p{index, static_cast<int32_t*>(plan), (int)M, L, index_bytes == 8, warps, tile_rows(M, sides, L, r, true, wide16)};
  // the most of any call, so that the first calls of two threads allow the same whichever comes last
  const cudaError_t e = allow_smem(plan_kernel, kPlanSmem, limit);
  if (e != cudaSuccess) return e;
  return launch_k(plan_kernel, dim3(1), dim3(kPlanThreads), plan_smem(warps, L), st, true, p);
}

}  // namespace
}  // namespace lora
}  // namespace glad

using namespace glad;
using namespace glad::lora;

extern "C" {

size_t glad_lora_plan_size(int64_t M, int L) {
  if (M < 0 || M > 1 << 24 || L < 1 || L > kMaxAdapters) return 0;
  return (size_t)plan_words(M, L) * 4;
}

int glad_lora_forward(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, const void* a, const void* b, int64_t N,
                      int L, int r, const void* index, int index_bytes, void* plan, size_t plan_bytes, const float* scale,
                      float scale_value, const void* base, int64_t ldb, void* y, float* u, void* stream) {
  const char* who = "glad_lora_forward";
  const char* why = shape_wrong(dtype, M, K, N, L, r, index, index_bytes);
  if (why) return bad(who, why);
  if (M == 0) return GLAD_OK;
  if (!x || !a || !b || !y) return bad(who, "x, a, b and y must be set");
  if ((why = rows_wrong(x, dtype, ldx, M, (int)K))) return bad(who, why);
  if (base && (why = rows_wrong(base, dtype, ldb, M, (int)N))) return bad(who, why);
  if (!on(a, width_of(dtype)) || !on(b, width_of(dtype)) || !on(y, width_of(dtype)) || !on(u, 4) || !on(scale, 4) ||
      !on(plan, 16))
    return bad(who, "a tensor is not element-aligned");
  if (index && !plan && M > kSelfRows && (M > kScanRows || L > kScanAdapters))
    return bad(who, "so many rows (more than 256, with more than 512 adapters; more than 4096) with an index need a plan");
  if (!index) plan = nullptr;
  if (plan && plan_bytes < glad_lora_plan_size(M, L))
    return set_last_error(GLAD_ERR_WORKSPACE, "glad_lora_forward: a plan of glad_lora_plan_size bytes is required");
  Params p{};
  p.x = x, p.ldx = ldx, p.M = (int)M, p.K = (int)K, p.N = (int)N, p.w1 = a, p.w2 = b, p.L = L, p.r = r;
  p.index = index, p.index64 = index_bytes == 8, p.plan = static_cast<const int32_t*>(plan);
  p.scale = scale, p.scale_value = scale_value, p.base = base, p.ldb = base ? ldb : 0, p.y = y, p.u = u;
  cudaError_t e = tensor_setup(p);
  if (plan && e == cudaSuccess) e = make_plan(index, index_bytes, M, K + N, L, r, dtype != GLAD_DTYPE_F32, plan, (cudaStream_t)stream);
  if (e == cudaSuccess) e = for_type(dtype, [&](auto t) { return run<decltype(t)>(p, false, (cudaStream_t)stream); });
  return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
}

size_t glad_lora_backward_workspace_size(int64_t M, int64_t K, int64_t N, int L, int r, int dtype, int indexed) {
  if (M < 1 || K < 1 || N < 1 || L < 1 || L > kMaxAdapters || r < 1 || r > kMaxRank) return 0;
  if (r % 8 || !tensor_sized(M, K + N, L, r, indexed != 0, dtype != GLAD_DTYPE_F32)) return 0;
  return (size_t)L * (size_t)r * (size_t)(K + N) * 2;
}

int glad_debug_lora_wait(uint32_t hold, uint64_t limit_ns) {
  if (hold > 1 || limit_ns > 2000000000ull)
    return set_last_error(GLAD_ERR_INVALID_ARG, "glad_debug_lora_wait: hold above 1 or limit_ns above 2 s");
  g_hold = hold;
  g_wait_ns = limit_ns ? (uint32_t)limit_ns : 2000000000u;
  return GLAD_OK;
}

int glad_lora_backward(const void* dy, int dtype, int64_t lddy, const void* x, int64_t ldx, int64_t M, int64_t K, const void* a,
                       const void* b, int64_t N, int L, int r, const void* index, int index_bytes, const void* plan,
                       const float* scale, float scale_value, const float* u, float* du, void* dx, void* da, void* db,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "glad_lora_backward";
  const char* why = shape_wrong(dtype, M, K, N, L, r, index, index_bytes);
  if (why) return bad(who, why);
  const size_t e_bytes = width_of(dtype);
  if (!on(a, e_bytes) || !on(b, e_bytes) || !on(dx, e_bytes) || !on(da, e_bytes) || !on(db, e_bytes) || !on(u, 4) ||
      !on(du, 4) || !on(scale, 4) || !on(plan, 16))
    return bad(who, "a tensor is not element-aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  if (M == 0) {
    if (da) e = cudaMemsetAsync(da, 0, (size_t)L * r * K * e_bytes, st);
    if (db && e == cudaSuccess) e = cudaMemsetAsync(db, 0, (size_t)L * r * N * e_bytes, st);
    return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
  }
  if (!dy || !a || !b) return bad(who, "dy, a and b must be set");
  if (index && !plan) return bad(who, "an index needs the forward pass's plan");
  if (!index) plan = nullptr;
  if ((why = rows_wrong(dy, dtype, lddy, M, (int)N))) return bad(who, why);
  if (da && (!x || !du)) return bad(who, "da needs x and du");
  if (db && !u) return bad(who, "db needs u");
  if (da && (why = rows_wrong(x, dtype, ldx, M, (int)K))) return bad(who, why);
  if (dx || da) {
    Params p{};
    p.x = dy, p.ldx = lddy, p.M = (int)M, p.K = (int)N, p.N = (int)K, p.w1 = b, p.w2 = a, p.L = L, p.r = r;
    p.index = index, p.index64 = index_bytes == 8, p.plan = static_cast<const int32_t*>(plan);
    p.scale = scale, p.scale_value = scale_value, p.y = dx, p.u = da ? du : nullptr;
    e = tensor_setup(p);
    const size_t need = glad_lora_backward_workspace_size(M, K, N, L, r, dtype, index != nullptr);
    bool transposed = false;
    for_type(dtype, [&](auto t) {
      transposed = need && workspace && workspace_bytes >= need && on(workspace, 16) && wants_transposed<decltype(t)>(p);
      return cudaSuccess;
    });
    if (transposed && e == cudaSuccess) {              // b [L, N, r] -> [L, r, N], a [L, r, K] -> [L, K, r]
      Transposes t{};
      uint16_t* ws = static_cast<uint16_t*>(workspace);
      t.src[0] = static_cast<const uint16_t*>(b), t.dst[0] = ws, t.rows[0] = (int)N, t.cols[0] = r;
      t.src[1] = static_cast<const uint16_t*>(a), t.dst[1] = ws + (size_t)L * r * N, t.rows[1] = r, t.cols[1] = (int)K;
      const int64_t longest = N > K ? N : K;
      const unsigned wide = longest <= kMaxRank ? kMaxRank / 64 : (unsigned)((longest + 63) / 64);
      e = launch_k(transpose_kernel, dim3(wide, kMaxRank / 64, 2 * L), dim3(256), 0, st, true, t);
      p.w1 = t.dst[0], p.w2 = t.dst[1];
    }
    if (e == cudaSuccess) e = for_type(dtype, [&](auto t) { return run<decltype(t)>(p, !transposed, st); });
  }
  // db first: dy has just been read
  OuterPair pair{};
  int count = 0;
  auto add = [&](const void* rows, int64_t ld, const float* v, void* out, int64_t cols, int64_t step_r, int64_t step_k) {
    OuterParams& o = pair.of[count++];
    o.plan = static_cast<const int32_t*>(plan), o.M = (int)M, o.r = r, o.L = L;
    o.x = rows, o.ldx = ld, o.v = v, o.out = out, o.K = (int)cols, o.step_r = step_r, o.step_k = step_k;
  };
  if (db) add(dy, lddy, u, db, N, 1, r);
  if (da) add(x, ldx, du, da, K, K, 1);
  if (count && e == cudaSuccess) e = tensor_setup(pair);
  if (count && e == cudaSuccess)
    e = for_type(dtype, [&](auto t) { return run_outer<decltype(t)>(pair, count, st); });
  return e == cudaSuccess ? GLAD_OK : cuda_bad(who, e);
}

}  // extern "C"
