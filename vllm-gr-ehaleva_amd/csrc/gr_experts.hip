// Routing of tokens to experts, and the chosen experts' SwiGLU layers.
#include "gr_block_mm.h"

namespace gr {

gr_status_t launch_quant_fp8(void* out, int64_t out_stride, float* scale, int64_t scale_row, int64_t scale_group,
                             const void* x, int64_t x_stride, int num_tokens, int features, int dtype,
                             hipStream_t stream);

namespace {

// ---- routing -----------------------------------------------------------------
constexpr int RT_WAVES = 4;  // one token each
constexpr int MAX_EXPERTS = 1024;

struct RouteArgs {
  float* weights;
  int32_t* ids;
  const void* logits;
  int64_t stride;
  const float* bias;
  int T, E, k, score, groups, top_groups, renorm;
  float scale;
};

__device__ inline double wave_max_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmax(v, __shfl_xor(v, off, 64));
  return v;
}
__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// (v, i) before (w, j): larger value first, then lower index; a NaN after everything
__device__ inline bool ranks_before(double v, int i, double w, int j) {
  const bool vn = v != v, wn = w != w;
  if (vn || wn) return vn == wn ? i < j : wn;
  return v > w || (v == w && i < j);
}

// Expert i * 64 + lane in slot i of each lane.
template <int DT, int PER>
__global__ __launch_bounds__(64 * RT_WAVES) void route_experts_k(RouteArgs a) {
  using E = Elem<DT>;
  using S = typename E::storage;
  __shared__ double ch[RT_WAVES][64 * PER];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * RT_WAVES + wave;
  if (t >= a.T) return;  // no barrier below: a wave works on its own
  const S* row = static_cast<const S*>(a.logits) + t * a.stride;
  double s[PER], c[PER];
  double mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 64 + lane;
    s[i] = e < a.E ? (double)E::to_float(row[e]) : -INFINITY;
    c[i] = s[i];
    mx = fmax(mx, s[i]);
  }
  if (a.score == GR_SCORE_SOFTMAX) {
    mx = wave_max_f64(mx);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = mx == -INFINITY && s[i] == -INFINITY ? 0.0 : exp(s[i] - mx);
      sum += i * 64 + lane < a.E ? s[i] : 0.0;
    }
    sum = wave_sum_f64(sum);
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = sum == 0.0 ? 0.0 : s[i] / sum;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = 1.0 / (1.0 + exp(-s[i]));
  }
  if (a.bias)
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 64 + lane < a.E) c[i] = s[i] + (double)a.bias[i * 64 + lane];
  uint32_t open = 0;  // experts of this lane that may still be chosen
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (i * 64 + lane < a.E) open |= 1u << i;
  if (a.groups > 1) {
    double* mine = ch[wave];
#pragma unroll
    for (int i = 0; i < PER; ++i) mine[i * 64 + lane] = c[i];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int n = a.E / a.groups;
    double v = NAN;
    if (lane < a.groups) {
      double b0 = NAN, b1 = NAN;
      for (int i = 0; i < n; ++i) {
        const double d = mine[lane * n + i];
        if (i == 0 || ranks_before(d, 0, b0, 1)) { b1 = b0; b0 = d; }
        else if (i == 1 || ranks_before(d, 0, b1, 1)) b1 = d;
      }
      v = a.bias && n > 1 ? b0 + b1 : b0;
    }
    int before = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double w = __shfl(v, g, 64);
      before += ranks_before(w, g, v, lane) ? 1 : 0;
    }
    const uint64_t kept = __ballot(lane < a.groups && before < a.top_groups);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if ((open >> i & 1) && !(kept >> ((i * 64 + lane) / n) & 1)) open &= ~(1u << i);
  }
  double total = 0.0, mine_s = 0.0;
  int mine_e = 0;
  for (int j = 0; j < a.k; ++j) {
    // this lane's best, then the wave's
    double bv = NAN, bs = 0.0;
    int be = 1 << 30;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if ((open >> i & 1) && (be == 1 << 30 || ranks_before(c[i], i * 64 + lane, bv, be))) {
        bv = c[i];
        bs = s[i];
        be = i * 64 + lane;
      }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const double ov = __shfl_xor(bv, off, 64), os = __shfl_xor(bs, off, 64);
      const int oe = __shfl_xor(be, off, 64);
      if (oe != 1 << 30 && (be == 1 << 30 || ranks_before(ov, oe, bv, be))) { bv = ov; bs = os; be = oe; }
    }
    if ((be & 63) == lane) open &= ~(1u << (be >> 6));
    if (lane == j) { mine_s = bs; mine_e = be; }
    total += bs;
  }
  if (lane < a.k) {
    const double w = a.renorm ? (total == 0.0 ? 0.0 : mine_s / total) : mine_s;
    a.weights[t * a.k + lane] = (float)(w * (double)a.scale);
    a.ids[t * a.k + lane] = mine_e;
  }
}

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
__global__ __launch_bounds__(PLAN_THREADS) void expert_count_k(PlanArgs a) {
  __shared__ int n[MAX_EXPERTS];
  int e[PLAN_PER];
  plan_load(a, e, true);
  plan_count(a, e, n);
  if ((int)threadIdx.x < a.E) a.hist[(int64_t)blockIdx.x * a.E + threadIdx.x] = n[threadIdx.x];
}

// Sorts this workgroup's choices by expert into the rows of the experts' tiles.
// Where a row lands within its expert differs from run to run (an atomic in LDS
// hands out the places); its result does not.
__global__ __launch_bounds__(PLAN_THREADS) void expert_plan_k(PlanArgs a) {
  __shared__ int next[MAX_EXPERTS];
  __shared__ int part[PLAN_THREADS / 64];
  const int tid = threadIdx.x;
  int e[PLAN_PER];
  plan_load(a, e, a.blocks == 1);
  int total = 0, before = 0;
  if (a.blocks == 1) {
    plan_count(a, e, next);
    total = next[tid];
    __syncthreads();
  } else if (tid < a.E) {
    for (int b = 0; b < a.blocks; ++b) {
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

// ---- out[t] = sum_j weights[t, j] * y[t, j] ---------------------------------------
struct CombineArgs {
  void* out;
  int64_t out_stride;
  const float* y;
  const float* weights;
  const int32_t* ids;
  int T, k, E, H;
};

template <int DT>
__global__ __launch_bounds__(256) void expert_combine_k(CombineArgs a) {
  const int64_t t = blockIdx.x;
  const int h = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (h >= a.H) return;
  mm4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.k; ++j) {
    const int e = a.ids[t * a.k + j];
    if (e < 0 || e >= a.E) continue;
    const float w = a.weights[t * a.k + j];
    const mm4_t v = *reinterpret_cast<const mm4_t*>(a.y + (t * a.k + j) * a.H + h);
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] = fmaf(w, v[u], acc[u]);
  }
  const float v[4] = {acc[0], acc[1], acc[2], acc[3]};
  mm_store<DT>(a.out, t * a.out_stride + h, v);
}

// ---- workspace -----------------------------------------------------------------
struct Workspace {
  int64_t hist, slot, tiles, num_tiles, x8, xs, act, act_scale, y, bytes;
  int64_t max_tiles;
  int blocks;
};

// Rows of a tile, by the rows an expert gets on average.  Few rows are bound by the
// weights' way from memory: then more workgroups on a CU count, later the rows a
// weight is read for.  Measured (64 experts of 768 features, hidden 2048, 8 of them a
// token; us, by tile rows; 16-bit weights, then e4m3):
//   rows an expert   1             8              32              64              256             1024
//   16 / 64        86 / 96      145 / 143      285 / 159        - / 190         - / 432         -
//   128 / 256     105 / 120     162 / 186      172 / 190       197 / 213       300 / 322     934 / 867
//   32 / 128       61 / 78       82 / 124      104 / 132       126 / 147      (280 at 128)    - / 920
int expert_tile_rows(int64_t rows, int E, bool fp8) {
  if (fp8) return rows <= 112ll * E ? 32 : 128;
  return rows <= 4ll * E ? 16 : rows <= 80ll * E ? 64 : rows <= 512ll * E ? 128 : 256;
}

Workspace plan_workspace(int T, int k, int E, int H, int F, bool fp8, int bm) {
  Workspace w{};
  const int64_t rows = (int64_t)T * k;
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  w.blocks = (int)((rows + PLAN_ROWS - 1) / PLAN_ROWS);
  w.max_tiles = rows / bm + (rows < E ? rows : E);
  w.num_tiles = take(4);
  w.hist = take(4ll * w.blocks * E);
  w.slot = take(4 * rows);
  w.tiles = take(16 * w.max_tiles);
  if (fp8) {
    w.x8 = take((int64_t)T * H);
    w.xs = take(4ll * T * ((H + 127) / 128));
    w.act = take(rows * F);
    w.act_scale = take(4 * rows * ((F + 127) / 128));
  } else {
    w.act = take(2 * rows * F);
  }
  w.y = take(4 * rows * H);
  return w;
}

template <int XT>
void launch_experts(const MmArgs& up, const MmArgs& down, int tiles, int bm, hipStream_t stream) {
  if constexpr (XT == GR_DTYPE_FP8_E4M3) {
    // (down's float32 results are summed into 16 bits: the 8-bit instruction will do)
    if (bm == 32) {
      launch_mm<XT, 32, 256, 1, 4, 2, MM_SWIGLU_Q, true, true>(up, tiles, stream);
      launch_mm<XT, 32, 128, 1, 4, 3, MM_PLAIN, true, false>(down, tiles, stream);
    } else {
      launch_mm<XT, 128, 256, 2, 4, 3, MM_SWIGLU_Q, true, true>(up, tiles, stream);
      launch_mm<XT, 128, 128, 2, 2, 2, MM_PLAIN, true, false>(down, tiles, stream);
    }
  } else {
    if (bm == 16) {
      launch_few<XT, 1, 8, MM_SWIGLU, true>(up, tiles, stream);
      launch_few<XT, 1, 8, MM_PLAIN, true>(down, tiles, stream);
    } else if (bm == 64) {
      launch_mm<XT, 64, 64, 2, 2, 4, MM_SWIGLU, true, false>(up, tiles, stream);
      launch_mm<XT, 64, 64, 2, 2, 4, MM_PLAIN, true, false>(down, tiles, stream);
    } else if (bm == 128) {
      launch_mm<XT, 128, 256, 2, 4, 3, MM_SWIGLU, true, false>(up, tiles, stream);
      launch_mm<XT, 128, 256, 2, 4, 3, MM_PLAIN, true, false>(down, tiles, stream);
    } else {
      launch_mm<XT, 256, 256, 2, 4, 2, MM_SWIGLU, true, false>(up, tiles, stream);
      launch_mm<XT, 256, 256, 2, 4, 2, MM_PLAIN, true, false>(down, tiles, stream);
    }
  }
}

template <int DT>
void launch_route(const RouteArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.T + RT_WAVES - 1) / RT_WAVES)), block(64 * RT_WAVES);
  if (a.E <= 64) hipLaunchKernelGGL((route_experts_k<DT, 1>), grid, block, 0, stream, a);
  else if (a.E <= 256) hipLaunchKernelGGL((route_experts_k<DT, 4>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((route_experts_k<DT, 16>), grid, block, 0, stream, a);
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace gr

using namespace gr;

extern "C" gr_status_t gr_route_experts(float* weights, int32_t* ids, const void* logits, int64_t logits_stride,
                                        const float* bias, int num_tokens, int num_experts, int top_k, int score,
                                        int num_groups, int top_groups, int renormalize, float scale, int dtype,
                                        hipStream_t stream) {
  if (num_tokens < 0 || num_experts < 1 || top_k < 1 || num_groups < 1 || num_experts % num_groups != 0 ||
      top_groups < 1 || top_groups > num_groups || top_k > num_experts / num_groups * top_groups ||
      (score != GR_SCORE_SOFTMAX && score != GR_SCORE_SIGMOID) || !dtype_valid(dtype))
    return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  if (!weights || !ids || !logits || logits_stride < num_experts) return GR_ERR_INVALID_ARG;
  if (num_experts > MAX_EXPERTS || num_groups > 64 || top_k > 64 || num_tokens > (1 << 28)) return GR_ERR_UNSUPPORTED;
  const RouteArgs a{weights, ids, logits, logits_stride, bias, num_tokens, num_experts, top_k, score,
                    num_groups, num_groups > 1 ? top_groups : 1, renormalize, scale};
  if (dtype == GR_DTYPE_F32) launch_route<GR_DTYPE_F32>(a, stream);
  else if (dtype == GR_DTYPE_F16) launch_route<GR_DTYPE_F16>(a, stream);
  else launch_route<GR_DTYPE_BF16>(a, stream);
  return launch_status();
}

extern "C" size_t gr_expert_mlp_workspace_size(int num_tokens, int top_k, int num_experts, int hidden, int ffn,
                                               int fp8) {
  if (num_tokens < 1 || top_k < 1 || num_experts < 1 || hidden < 1 || ffn < 1) return 0;
  const int bm = expert_tile_rows((int64_t)num_tokens * top_k, num_experts, fp8 != 0);
  return (size_t)plan_workspace(num_tokens, top_k, num_experts, hidden, ffn, fp8 != 0, bm).bytes;
}

extern "C" gr_status_t gr_expert_mlp(void* out, int64_t out_stride, const void* x, int64_t x_stride,
                                     const void* gate_up, const float* gate_up_scale, const void* down,
                                     const float* down_scale, const float* weights, const int32_t* ids,
                                     int num_tokens, int top_k, int num_experts, int hidden, int ffn, int dtype,
                                     void* workspace, size_t workspace_bytes, int32_t* dev_status,
                                     hipStream_t stream) {
  if (num_tokens < 0 || top_k < 1 || num_experts < 1 || hidden < 1 || ffn < 1 || !dtype_valid(dtype))
    return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  if (!out || !x || !gate_up || !down || !weights || !ids || out_stride < hidden || x_stride < hidden ||
      (gate_up_scale == nullptr) != (down_scale == nullptr))
    return GR_ERR_INVALID_ARG;
  const bool fp8 = gate_up_scale != nullptr;
  const int T = num_tokens, H = hidden, F = ffn;
  if (dtype == GR_DTYPE_F32 || hidden % 16 != 0 || ffn % 16 != 0 || hidden > (1 << 21) || ffn > (1 << 21) ||
      num_experts > MAX_EXPERTS || (int64_t)T * top_k > (1 << 26) || !aligned(x, 16) || x_stride % 8 != 0 ||
      !aligned(gate_up, 16) || !aligned(down, 16) || !aligned(out, 8) || out_stride % 4 != 0 ||
      (fp8 && (!aligned(gate_up_scale, 4) || !aligned(down_scale, 4))) || (int64_t)T * x_stride > (1 << 30) - (1 << 24) ||
      (fp8 && (int64_t)T * H > (1ll << 31) - (1 << 24)))
    return GR_ERR_UNSUPPORTED;
  const int bm = expert_tile_rows((int64_t)T * top_k, num_experts, fp8);
  const Workspace l = plan_workspace(T, top_k, num_experts, H, F, fp8, bm);
  if (l.max_tiles * ((2ll * F + 15) / 16) > INT32_MAX - 8 || l.max_tiles * ((H + 15) / 16) > INT32_MAX - 8)
    return GR_ERR_UNSUPPORTED;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < (size_t)l.bytes) return GR_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int rows = T * top_k, hb = (H + 127) / 128, fb = (F + 127) / 128;

  PlanArgs p{ids, rows, num_experts, bm, l.blocks, reinterpret_cast<int32_t*>(ws + l.hist),
             reinterpret_cast<int32_t*>(ws + l.slot), reinterpret_cast<int4*>(ws + l.tiles),
             reinterpret_cast<int32_t*>(ws + l.num_tiles), dev_status};
  if (l.blocks > 1) hipLaunchKernelGGL(expert_count_k, dim3(l.blocks), dim3(PLAN_THREADS), 0, stream, p);
  hipLaunchKernelGGL(expert_plan_k, dim3(l.blocks), dim3(PLAN_THREADS), 0, stream, p);

  const int esize = fp8 ? 1 : 2;
  MmArgs up{};
  up.x = static_cast<const uint8_t*>(x);
  up.x_stride = x_stride * 2;
  up.w = static_cast<const uint8_t*>(gate_up);
  up.w_stride = (int64_t)H * esize;
  up.w_expert = 2ll * F * H * esize;
  up.out = ws + l.act;
  up.out_stride = F;
  up.M = rows;
  up.N = F;
  up.kbytes = H * esize;
  up.out_type = dtype;
  up.tiles = p.tiles;
  up.num_tiles = p.num_tiles;
  up.slot = p.slot;
  up.gather = top_k;
  if (fp8) {
    float* xs = reinterpret_cast<float*>(ws + l.xs);
    launch_quant_fp8(ws + l.x8, H, xs, 1, T, x, x_stride, T, H, dtype, stream);
    up.x = ws + l.x8;
    up.x_stride = H;
    up.xs = xs;
    up.xs_row = 1;
    up.xs_grp = T;
    up.ws = gate_up_scale;
    up.ws_expert = 2ll * fb * hb;
    up.out_scale = reinterpret_cast<float*>(ws + l.act_scale);
    up.os_row = 1;
    up.os_grp = rows;
  }
  MmArgs dn{};
  dn.x = ws + l.act;
  dn.x_stride = (int64_t)F * esize;
  dn.w = static_cast<const uint8_t*>(down);
  dn.w_stride = (int64_t)F * esize;
  dn.w_expert = (int64_t)H * F * esize;
  dn.out = ws + l.y;
  dn.out_stride = H;
  dn.M = rows;
  dn.N = H;
  dn.kbytes = F * esize;
  dn.out_type = GR_DTYPE_F32;
  dn.tiles = p.tiles;
  dn.num_tiles = p.num_tiles;
  dn.slot = p.slot;
  dn.scatter = 1;
  if (fp8) {
    dn.xs = up.out_scale;
    dn.xs_row = 1;
    dn.xs_grp = rows;
    dn.ws = down_scale;
    dn.ws_expert = (int64_t)hb * fb;
  }
  const int tiles = (int)l.max_tiles;
  if (fp8) launch_experts<GR_DTYPE_FP8_E4M3>(up, dn, tiles, bm, stream);
  else if (dtype == GR_DTYPE_BF16) launch_experts<GR_DTYPE_BF16>(up, dn, tiles, bm, stream);
  else launch_experts<GR_DTYPE_F16>(up, dn, tiles, bm, stream);

  const CombineArgs c{out, out_stride, reinterpret_cast<const float*>(ws + l.y), weights, ids, T, top_k,
                      num_experts, H};
  const dim3 grid((unsigned)T, (unsigned)((H + 1023) / 1024));
  if (dtype == GR_DTYPE_BF16) hipLaunchKernelGGL(expert_combine_k<GR_DTYPE_BF16>, grid, dim3(256), 0, stream, c);
  else hipLaunchKernelGGL(expert_combine_k<GR_DTYPE_F16>, grid, dim3(256), 0, stream, c);
  return launch_status();
}
