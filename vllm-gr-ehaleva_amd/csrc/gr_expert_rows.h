// The rows of routed experts, sorted by expert, and the sum over a token's experts:
// shared by the experts' layers with 16- and 8-bit weights (gr_experts.hip) and with
// 4-bit ones (gr_mx_experts.hip).
#pragma once

#include "gr_block_mm.h"

namespace gr {
namespace {

constexpr int MAX_EXPERTS = 1024;

// ---- the experts' rows ---------------------------------------------------------
constexpr int PLAN_THREADS = 1024;  // >= MAX_EXPERTS
constexpr int PLAN_ROWS = 8192;  // choices a workgroup sorts

struct PlanArgs {
  const int32_t* ids;
  int rows, E, bm, blocks;
  int32_t* hist;  // [blocks][E]
  int32_t* slot;
  int4* tiles;
  int32_t* num_tiles;
  int32_t* dev_status;
};

// exclusive prefix sum over the workgroup's 1024 threads
__device__ inline int block_excl_scan(int v, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = wave_incl_scan(v);
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < wave; ++i) before += part[i];
  __syncthreads();
  return before + incl - v;
}

constexpr int PLAN_PER = PLAN_ROWS / PLAN_THREADS;
// the workgroup's choices, PLAN_PER a thread; -1: none, or another rank's
__device__ inline void plan_load(const PlanArgs& a, int (&e)[PLAN_PER], bool flag) {
  const int r0 = blockIdx.x * PLAN_ROWS + threadIdx.x;
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i) {
    const int r = r0 + i * PLAN_THREADS;
    e[i] = r < a.rows ? a.ids[r] : -1;
  }
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i)
    if (e[i] >= a.E) {
      if (flag) flag_status(a.dev_status, GR_DEV_BAD_EXPERT);
      e[i] = -1;
    }
}
__device__ inline void plan_count(const PlanArgs& a, const int (&e)[PLAN_PER], int* n) {
  n[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i)
    if (e[i] >= 0) atomicAdd(&n[e[i]], 1);
  __syncthreads();
}

// more choices than one workgroup sorts: how many of each expert every one of them has
__device__ __forceinline__ void expert_count(const PlanArgs& a, int* n) {
  int e[PLAN_PER];
  plan_load(a, e, true);
  plan_count(a, e, n);
  if ((int)threadIdx.x < a.E) a.hist[(int64_t)blockIdx.x * a.E + threadIdx.x] = n[threadIdx.x];
}

// Sorts this workgroup's choices by expert into the rows of the experts' tiles.
// Where a row lands within its expert differs from run to run (an atomic in LDS
// hands out the places); its result does not.
__device__ __forceinline__ void expert_plan(const PlanArgs& a, int* next, int* part) {
  const int tid = threadIdx.x;
  int e[PLAN_PER];
  plan_load(a, e, a.blocks == 1);
  int total = 0, before = 0;
  if (a.blocks == 1) {
    plan_count(a, e, next);
    total = next[tid];
    __syncthreads();
  } else if (tid < a.E) {
#pragma unroll 8
    for (int b = 0; b < a.blocks; ++b) {  // (eight loads on their way)
      const int n = a.hist[(int64_t)b * a.E + tid];
      if (b < (int)blockIdx.x) before += n;
      total += n;
    }
  }
  const int first = block_excl_scan(total, part);
  next[tid] = first + before;
  if (blockIdx.x == 0) {
    const int tiles = (total + a.bm - 1) / a.bm;
    const int t0 = block_excl_scan(tiles, part);
    for (int i = 0; i < tiles; ++i)
      a.tiles[t0 + i] = make_int4(tid, first + i * a.bm, min(a.bm, total - i * a.bm), 0);
    if (tid == PLAN_THREADS - 1) *a.num_tiles = t0 + tiles;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i)
    if (e[i] >= 0) a.slot[atomicAdd(&next[e[i]], 1)] = blockIdx.x * PLAN_ROWS + i * PLAN_THREADS + tid;
}

__global__ __launch_bounds__(PLAN_THREADS) void expert_count_k(PlanArgs a) {
  __shared__ int n[MAX_EXPERTS];
  expert_count(a, n);
}
__global__ __launch_bounds__(PLAN_THREADS) void expert_plan_k(PlanArgs a) {
  __shared__ int next[MAX_EXPERTS], part[PLAN_THREADS / 64];
  expert_plan(a, next, part);
}

// ---- out[t] = sum_j weights[t, j] * y[t, j] ---------------------------------------
struct CombineArgs {
  void* out;
  int64_t out_stride;
  const void* y;         // float32, or MM_OUT_SCALED with the units' exponents
  const int8_t* y_exp;
  int exp_cols;          // columns of one exponent
  const float* weights;
  const int32_t* ids;
  int T, k, E, H;
};

// Bound by memory; a thread sums 8 columns over the token's choices, in order.
template <int DT, bool SCALED>
__global__ __launch_bounds__(256) void expert_combine_k(CombineArgs a) {
  const int64_t t = blockIdx.x;
  const int h = (blockIdx.y * 256 + threadIdx.x) * 8;
  if (h >= a.H) return;
  const int groups = SCALED ? (a.H + a.exp_cols - 1) / a.exp_cols : 0;
  float acc[8] = {};
#pragma unroll 8
  for (int j = 0; j < a.k; ++j) {
    const int64_t row = t * a.k + j;
    const int e = a.ids[row];
    const bool here = e >= 0 && e < a.E;  // (another's row holds anything: loaded all the same, so that nothing waits
    const float w = a.weights[row];       // for the id, and left out)
    float v[8];
    if constexpr (SCALED) {
      const u32x4_t d = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.y) + row * a.H + h);
      const float unit = __builtin_amdgcn_ldexpf(1.0f, a.y_exp[row * groups + h / a.exp_cols]);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        v[2 * u] = Mma<GR_DTYPE_F16>::lo(d[u]) * unit;
        v[2 * u + 1] = Mma<GR_DTYPE_F16>::hi(d[u]) * unit;
      }
    } else {
      const mm4_t* p = reinterpret_cast<const mm4_t*>(static_cast<const float*>(a.y) + row * a.H + h);
      const mm4_t lo = p[0], hi = p[1];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        v[u] = lo[u];
        v[u + 4] = hi[u];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) acc[u] = here ? fmaf(w, v[u], acc[u]) : acc[u];
  }
  const float lo[4] = {acc[0], acc[1], acc[2], acc[3]}, hi[4] = {acc[4], acc[5], acc[6], acc[7]};
  mm_store<DT>(a.out, t * a.out_stride + h, lo);
  mm_store<DT>(a.out, t * a.out_stride + h + 4, hi);
}

// Workgroups of a launch, of up to 512 threads: their threads are counted in 32 bits.
constexpr int GRID_MAX = (1 << 23) - 1;

}  // namespace
}  // namespace gr
