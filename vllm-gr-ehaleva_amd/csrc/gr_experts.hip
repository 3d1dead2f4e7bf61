// Routing of tokens to experts, and the chosen experts' SwiGLU layers.
#include <algorithm>

#include "gr_expert_rows.h"

namespace gr {

namespace {

// ---- routing -----------------------------------------------------------------
constexpr int RT_WAVES = 4;

struct RouteArgs {
  float* weights;
  int32_t* ids;
  const void* logits;
  int64_t stride;
  const float* bias;
  int T, E, k, score, groups, top_groups, renorm;
  float scale;
};

// Reductions over each L neighbouring lanes, the result in all of them: within a row
// of 16 by DPP moves (the xor of 1 and of 2, then mirrors of 8 and of 16, whose halves
// agree in themselves by then).
template <typename F> __device__ __forceinline__ uint32_t seg_step(uint32_t v, int step, F f) {
  switch (step) {
    case 1: return f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
    case 2: return f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
    case 4: return f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
    case 8: return f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
    default: return f(v, (uint32_t)__shfl_xor((int)v, step, 64));
  }
}
template <int L, typename F> __device__ __forceinline__ uint32_t seg_all(uint32_t v, F f) {
#pragma unroll
  for (int step = 1; step < L; step *= 2) v = seg_step(v, step, f);
  return v;
}
template <int L> __device__ __forceinline__ uint32_t seg_max(uint32_t v) {
  return seg_all<L>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int L> __device__ __forceinline__ uint64_t seg_max(uint64_t k) {
  const uint32_t hi = seg_max<L>((uint32_t)(k >> 32));
  return (uint64_t)hi << 32 | seg_max<L>((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
}
template <int L> __device__ __forceinline__ float seg_sum(float v) {
  return __uint_as_float(seg_all<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int L> __device__ __forceinline__ double seg_sum(double v) {
#pragma unroll
  for (int step = 1; step < L; step *= 2) v += __shfl_xor(v, step, 64);
  return v;
}
// Keys that rank as the values do: a NaN's is 1, 0 is left for what cannot be chosen.
__device__ __forceinline__ uint32_t rank_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 as 0)
  return v != v ? 1u : (int32_t)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_key(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return v != v ? 1u : (int64_t)b < 0 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ float rank_value(uint32_t k) {
  return k <= 1 ? NAN : __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k);
}
// a before b in rank (a NaN after everything)
template <typename T> __device__ __forceinline__ bool better(T a, T b) { return a > b || (b != b && a == a); }

__device__ __forceinline__ void wave_sync() {  // LDS written by this wave is read by other lanes of it
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// One row's logits (experts l * PER .. of it in lane l of its L lanes) and what its
// scores need.
template <int PER> struct RouteRow {
  float x[PER];  // -inf past the last
  float mx;      // softmax: the largest
  bool nan;      // softmax: every score is NaN (a NaN or +inf among the logits)
};
// A wave's room in LDS, by token: c of the experts, the groups' values and whether they
// are kept, the choices and their scores.
template <int PER, int L> struct RouteRoom {
  double c[64 / L][L * PER > 64 ? L * PER : 64];
  double group[64 / L][64];
  uint64_t kept[64 / L];
  int id[64 / L][64];
};

template <int PER, int L> __device__ __forceinline__ double route_sum(const RouteRow<PER>& r) {
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += r.x[i] == -INFINITY ? 0.0 : exp((double)r.x[i] - r.mx);
  return seg_sum<L>(sum);
}
template <int PER>
__device__ __forceinline__ double route_score(const RouteArgs& a, const RouteRow<PER>& r, float v, double sum) {
  if (a.score == GR_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-(double)v));
  if (r.nan) return NAN;
  return v == -INFINITY ? 0.0 : exp((double)v - r.mx) / sum;
}

// The k choices of each of the wave's rows, into room.id.  T: the type in which c is
// compared.  CHECK (float c of scores plus bias): two that had to be told apart are
// unsure where they are not further from each other than their error may be; float32
// scores are within 2^-22 (__expf's relative error grows with its argument, its share
// of a score shrinks faster), the sum with the bias adds a rounding.  `order`: choices
// are unsure; then the list goes on (`listed` entries) until the next is surely worse.
// `groups`: which groups are kept is.
struct RouteDoubt { bool order, groups; int listed; };
template <int PER, int L, bool CHECK, typename T>
__device__ __forceinline__ RouteDoubt route_choose(const RouteArgs& a, const T (&c)[PER], RouteRoom<PER, L>& room) {
  using U = decltype(rank_key(T()));
  const int lane = threadIdx.x & 63, l = lane % L, tok = lane / L, e0 = l * PER;
  auto apart = [](T p, T q, float times) { return fabs(p - q) > times * (0x1p-19f + (fabs(p) + fabs(q)) * 0x1p-22f); };
  RouteDoubt doubt{false, false, a.k};
  U key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = e0 + i < a.E ? rank_key(c[i]) : U(0);
  if (a.groups > 1) {
    T *mine = reinterpret_cast<T*>(room.c[tok]), *value = reinterpret_cast<T*>(room.group[tok]);
    const int n = a.E / a.groups;
    auto add = [](T d, T& b0, T& b1) __attribute__((always_inline)) {  // the two best
      const bool first = better(d, b0);
      const T rest = first ? b0 : d;
      b0 = first ? d : b0;
      b1 = better(rest, b1) ? rest : b1;
    };
    auto of = [&](T b0, T b1) { return a.bias && n > 1 ? b0 + b1 : b0; };
    // how group g ranks: groups ahead of it, and (CHECK) whether that is sure
    auto rank = [&](int g, T v) __attribute__((always_inline)) {
      int before = 0;
      T next = NAN;  // the next worse value, where this group is the last that is kept
#pragma unroll 4
      for (int h = 0; h < a.groups; ++h) {
        const T w = value[h];
        const bool ahead = h != g && (better(w, v) || (h < g && !better(v, w)));
        before += ahead ? 1 : 0;
        if (CHECK && h != g && !ahead) next = better(w, next) ? w : next;
      }
      if (CHECK && before == a.top_groups - 1 && a.top_groups < a.groups) doubt.groups = !apart(v, next, 2.f);
      return before < a.top_groups;
    };
    wave_sync();
    const int span = n / PER;
    if (n % PER == 0 && span <= L && (span & (span - 1)) == 0) {
      // a group is whole lanes, a power of two of them (and the groups fill the lanes from
      // the first on): its two best from registers
      T b0 = NAN, b1 = NAN;
#pragma unroll
      for (int i = 0; i < PER; ++i) add(c[i], b0, b1);
      for (int step = 1; step < span; step *= 2) {
        const T o0 = __shfl_xor(b0, step, 64), o1 = __shfl_xor(b1, step, 64);
        add(o0, b0, b1);
        add(o1, b0, b1);
      }
      const int g = l / span;
      const T v = of(b0, b1);
      if (l % span == 0 && g < a.groups) value[g] = v;
      wave_sync();
      if (g < a.groups && !rank(g, v))
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = 0;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) mine[e0 + i] = c[i];
      if (l == 0) room.kept[tok] = 0;
      wave_sync();
      for (int g = l; g < a.groups; g += L) {  // a lane scans whole groups, from its own place in them: its own banks
        T b0 = NAN, b1 = NAN;
        int at = g % n;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
          add(mine[g * n + at], b0, b1);
          at = at + 1 == n ? 0 : at + 1;
        }
        value[g] = of(b0, b1);
      }
      wave_sync();
      for (int g = l; g < a.groups; g += L)
        if (rank(g, value[g])) atomicOr(reinterpret_cast<unsigned long long*>(&room.kept[tok]), 1ull << g);
      wave_sync();
      const uint64_t kept = room.kept[tok];
      int ge = e0 / n, re = e0 - ge * n;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (e0 + i < a.E && !(kept >> ge & 1)) key[i] = 0;
        if (++re == n) {
          re = 0;
          ++ge;
        }
      }
    }
  }
  T prev = 0;
  bool open = true;  // CHECK: the list goes on
  for (int j = 0; CHECK ? __ballot(open) != 0 : j < a.k; ++j) {
    U best = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = max(best, key[i]);
    const U top = seg_max<L>(best);
    if constexpr (CHECK) {
      const T now = rank_value(top);
      const bool near = j > 0 && !apart(prev, now, 1.f);
      open = open && top != 0 && (j < a.k || near);
      if (open && j == 64) {  // (a list that does not end)
        doubt.groups = true;
        open = false;
      }
      doubt.order |= open && near;
      doubt.listed = open ? j + 1 : doubt.listed;
      prev = now;
    }
    // the first lane that has it, and its first slot: the lowest index
    const uint64_t mates = __ballot(best == top) >> (tok * L);
    const bool win = l == __builtin_ctzll(mates) && open;
    int at = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool hit = key[i] == top && !found;
      found |= hit;
      at = hit ? i : at;
      key[i] = hit && win ? U(0) : key[i];
    }
    if (win) room.id[tok][j] = e0 + at;
  }
  return doubt;
}

// L lanes a token, PER neighbouring experts a lane: a choice is one maximum over the L
// lanes, and among equal keys the first lane's first slot is the lowest index.  Without
// a bias the logits themselves rank.  With one, float32 sums of nearly equal ones could
// come out in the wrong order: they are tried first, and where two of them are too close
// to tell, the listed ones (groups: all) are ranked again in float64.
// Bound by instructions where there are many tokens: a choice costs its reduction and a
// few for each slot, so tokens share a wave (8 slots a lane: 8192 tokens of 256 experts
// in 8 groups, k = 8, with a bias 18.9 us; 16 slots 24.7, as a row that is done again is
// its wave's whole time; a wave a token, 4 slots a lane, all in float64 20.7; 8192 of 64
// without a bias 5.7).  Few tokens take the shorter chain of 4 slots (8 of 64: 3.8).
template <int DT, int PER, int L>
__global__ __launch_bounds__(64 * RT_WAVES) void route_experts_k(RouteArgs a) {
  using E = Elem<DT>;
  using S = typename E::storage;
  __shared__ RouteRoom<PER, L> rooms[RT_WAVES];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane % L, e0 = l * PER;
  const int64_t t0 = ((int64_t)blockIdx.x * RT_WAVES + wave) * (64 / L);
  if (t0 >= a.T) return;  // no barrier below: a wave works on its own
  const int64_t t = min(t0 + lane / L, (int64_t)a.T - 1);  // (past the last token: it again, not stored)
  const bool real = t0 + lane / L < a.T;
  RouteRoom<PER, L>& room = rooms[wave];
  const S* row = static_cast<const S*>(a.logits) + t * a.stride;
  const bool softmax = a.score == GR_SCORE_SOFTMAX;
  RouteRow<PER> r;
  r.mx = -INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    r.x[i] = e0 + i < a.E ? E::to_float(row[e0 + i]) : -INFINITY;
    r.mx = fmaxf(r.mx, r.x[i]);
    odd |= r.x[i] != r.x[i];
  }
  r.nan = false;
  if (softmax) {
    r.mx = rank_value(seg_max<L>(rank_key(r.mx)));
    r.nan = seg_max<L>(odd ? 1u : 0u) != 0 || r.mx == INFINITY;
  }
  if (!a.bias) {
    route_choose<PER, L, false>(a, r.x, room);
  } else {
    float bias[PER], c[PER], sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      bias[i] = e0 + i < a.E ? a.bias[e0 + i] : 0.f;
      c[i] = softmax ? __expf(r.x[i] - r.mx) : __builtin_amdgcn_rcpf(1.0f + __expf(-r.x[i]));
      sum += c[i];
    }
    const float inv = softmax ? 1.0f / seg_sum<L>(sum) : 1.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) c[i] = fmaf(c[i], inv, bias[i]);
    const RouteDoubt doubt = route_choose<PER, L, true>(a, c, room);
    if (__ballot(doubt.groups || (softmax && (doubt.order || r.nan || r.mx == -INFINITY)))) {
      const double all = softmax ? route_sum<PER, L>(r) : 1.0;
      double d[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) d[i] = route_score(a, r, r.x[i], all) + (double)bias[i];
      route_choose<PER, L, false>(a, d, room);
    } else if (__ballot(doubt.order)) {
      const int tok = lane / L, m = doubt.listed;
      double* v = room.c[tok];
      int* id = room.id[tok];
      wave_sync();
      for (int j = l; j < m; j += L) v[j] = route_score(a, r, E::to_float(row[id[j]]), 1.0) + (double)a.bias[id[j]];
      wave_sync();
      int to[64 / L], was[64 / L];
#pragma unroll
      for (int q = 0; q < 64 / L; ++q) {
        const int j = l + q * L;
        to[q] = 64;
        if (j >= m) continue;
        to[q] = 0;
        was[q] = id[j];
        for (int h = 0; h < m; ++h)
          to[q] += better(v[h], v[j]) || (!better(v[j], v[h]) && id[h] < was[q]) ? 1 : 0;
      }
      wave_sync();
#pragma unroll
      for (int q = 0; q < 64 / L; ++q)
        if (to[q] < a.k) id[to[q]] = was[q];
    }
  }
  wave_sync();
  // the chosen ones' scores, in float64 (a renormalised weight needs no sum of all)
  const double all = softmax && !a.renorm ? route_sum<PER, L>(r) : 1.0;
  const int* id = room.id[lane / L];
  double total = 0.0;
  for (int j = l; j < a.k; j += L) {
    const double s = route_score(a, r, E::to_float(row[id[j]]), all);
    room.c[lane / L][j] = s;  // (read by this lane alone)
    total += s;
  }
  total = a.renorm ? seg_sum<L>(total) : 1.0;
  if (!real) return;
  for (int j = l; j < a.k; j += L) {
    const double s = room.c[lane / L][j];
    a.weights[t * a.k + j] = (float)((total == 0.0 ? 0.0 : s / total) * (double)a.scale);
    a.ids[t * a.k + j] = id[j];
  }
}

// With e4m3 weights the tokens are quantised by the workgroups behind those that sort
// (or count, where several do): a launch less, and the sort's waits are theirs alone
// (512 tokens 6.1 us against 4.8 + 5.8 one after the other).
template <int DT, int ROWS> __global__ __launch_bounds__(PLAN_THREADS) void expert_start_k(PlanArgs a, QuantArgs q) {
  __shared__ int next[MAX_EXPERTS], part[PLAN_THREADS / 64];
  if ((int)blockIdx.x >= a.blocks)
    quant_group<DT, ROWS>(q, (blockIdx.x - a.blocks) * (PLAN_THREADS / 8) + (threadIdx.x >> 3), threadIdx.x & 7);
  else if (a.blocks > 1)
    expert_count(a, next);
  else
    expert_plan(a, next, part);
}


// ---- workspace -----------------------------------------------------------------
struct Workspace {
  int64_t hist, slot, tiles, num_tiles, x8, xs, act, act_scale, y, y_exp, bytes;
  int64_t max_tiles;
  int blocks;
};

// Rows of a tile, by the rows an expert gets on average.  Few rows are bound by the
// weights' way from memory: then more workgroups on a CU count, later the rows a
// weight is read for.  Measured (64 experts of 768 features, hidden 2048, 8 of them a
// token; us, by tile rows; 16-bit weights, then e4m3):
//   rows an expert    1            8            32           64           96          256          512         1024
//   16 / 64       95 / 107    139 / 139    296 / 146    511 / 182    724 / 206     - / 407     - / 696    - / 1216
//   128 / 256    140 / 165    156 / 181    164 / 187    175 / 197    183 / 208   280 / 310   448 / 435   808 / 744
//   32 / 128      58 / 75      77 / 119     97 / 123    113 / 127    151 / 132   294 / 255   495 / 415   923 / 763
int expert_tile_rows(int64_t rows, int E, bool fp8) {
  if (fp8) return rows <= 80ll * E ? 32 : 128;
  return rows <= 8ll * E ? 16 : rows <= 56ll * E ? 64 : rows <= 448ll * E ? 128 : 256;
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
  // (room for float32, whatever the results' type turns out to be)
  w.y = take(4 * rows * H);
  w.y_exp = take(rows * ((H + 15) / 16));
  return w;
}

// columns of a wave of the down product with tiles of bm rows (launch_experts)
int expert_wave_cols(int bm) { return bm == 16 ? 16 : bm == 64 ? 32 : 64; }

template <int XT>
void launch_experts(const MmArgs& up, const MmArgs& down, int tiles, int bm, hipStream_t stream) {
  if constexpr (XT == GR_DTYPE_FP8_E4M3) {
    // (down's float32 results are summed into 16 bits: the 8-bit instruction will do.  512 tokens, 64 rows an expert:
    // 256 columns of it 38.3 us, 128 columns 39.9)
    if (bm == 32) {
      launch_mm<XT, 32, 256, 1, 4, 2, MM_SWIGLU_Q, true, true>(up, tiles, stream);
      launch_mm<XT, 32, 256, 1, 4, 2, MM_PLAIN, true, false>(down, tiles, stream);
    } else {
      launch_mm<XT, 128, 256, 2, 4, 3, MM_SWIGLU_Q, true, true>(up, tiles, stream);
      launch_mm<XT, 128, 128, 2, 2, 2, MM_PLAIN, true, false>(down, tiles, stream);
    }
  } else {
    if (bm == 16) {
      launch_few<XT, 1, MM_SWIGLU, true>(up, tiles, stream);
      launch_few<XT, 1, MM_PLAIN, true>(down, tiles, stream);
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

template <int DT, int PER, int L> void launch_route_k(const RouteArgs& a, hipStream_t stream) {
  constexpr int PER_WG = RT_WAVES * (64 / L);
  hipLaunchKernelGGL((route_experts_k<DT, PER, L>), dim3((unsigned)(((int64_t)a.T + PER_WG - 1) / PER_WG)),
                     dim3(64 * RT_WAVES), 0, stream, a);
}
template <int DT> void launch_route(const RouteArgs& a, hipStream_t stream) {
  const int64_t lanes4 = (int64_t)a.T * a.E / 4;  // with 4 slots a lane
  if (a.E <= 256 && lanes4 <= 64 * 1024) {        // at most a wave for each of the 1024 SIMDs
    if (a.E <= 64) launch_route_k<DT, 4, 16>(a, stream);
    else if (a.E <= 128) launch_route_k<DT, 4, 32>(a, stream);
    else launch_route_k<DT, 4, 64>(a, stream);
  } else if (a.E <= 64) {
    launch_route_k<DT, 8, 8>(a, stream);
  } else if (a.E <= 128) {
    launch_route_k<DT, 8, 16>(a, stream);
  } else if (a.E <= 256) {
    launch_route_k<DT, 8, 32>(a, stream);
  } else if (a.E <= 512) {
    launch_route_k<DT, 8, 64>(a, stream);
  } else {
    launch_route_k<DT, 16, 64>(a, stream);
  }
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
  // (16 logits a thread at most, 8 up to 512 experts: their threads are counted in 32 bits)
  if (num_experts > MAX_EXPERTS || num_groups > 64 || top_k > 64 || num_tokens > (1 << 28) ||
      (int64_t)num_tokens * num_experts > (1ll << 34))
    return GR_ERR_UNSUPPORTED;
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
  const int cols = bm == 16 ? 16 : bm == 64 ? 32 : 128;  // results of a workgroup, in the narrower product
  if (l.max_tiles * ((std::max(F, H) + cols - 1) / cols) > GRID_MAX - 8 || T > GRID_MAX) return GR_ERR_UNSUPPORTED;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < (size_t)l.bytes) return GR_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int rows = T * top_k, hb = (H + 127) / 128, fb = (F + 127) / 128;

  PlanArgs p{ids, rows, num_experts, bm, l.blocks, reinterpret_cast<int32_t*>(ws + l.hist),
             reinterpret_cast<int32_t*>(ws + l.slot), reinterpret_cast<int4*>(ws + l.tiles),
             reinterpret_cast<int32_t*>(ws + l.num_tiles), dev_status};
  float* xs = reinterpret_cast<float*>(ws + l.xs);
  if (fp8) {
    const QuantArgs q{ws + l.x8, H, xs, 1, T, x, x_stride, T, H, hb};
    const int quant = quant_rows(T, hb);
    const int64_t items = ((int64_t)T + quant - 1) / quant * hb, per = PLAN_THREADS / 8;
    const dim3 grid((unsigned)(l.blocks + (items + per - 1) / per));
    auto go = [&](auto one, auto two) {
      hipLaunchKernelGGL(quant == 2 ? two : one, grid, dim3(PLAN_THREADS), 0, stream, p, q);
    };
    if (dtype == GR_DTYPE_F16) go(expert_start_k<GR_DTYPE_F16, 1>, expert_start_k<GR_DTYPE_F16, 2>);
    else go(expert_start_k<GR_DTYPE_BF16, 1>, expert_start_k<GR_DTYPE_BF16, 2>);
  } else if (l.blocks > 1) {
    hipLaunchKernelGGL(expert_count_k, dim3(l.blocks), dim3(PLAN_THREADS), 0, stream, p);
  }
  if (!fp8 || l.blocks > 1) hipLaunchKernelGGL(expert_plan_k, dim3(l.blocks), dim3(PLAN_THREADS), 0, stream, p);

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
  // (the gated product is the down product's operand: rounded to x's type, as the matrix core takes it.  Half a step for
  // each of F terms; of 8192 bf16 tokens' results 1.7e-3 of the norm is off with it in float32, 2.4e-3 so)
  up.out_type = dtype;
  up.tiles = p.tiles;
  up.num_tiles = p.num_tiles;
  up.slot = p.slot;
  up.gather = top_k;
  if (fp8) {
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
  // Rounding the experts' results to fp16 multiples costs up to 2^-11 of each: an eighth of the output's half step of
  // 2^-8 in bf16, and little beside the 2^-4 of e4m3 inputs; fp16 results of 16-bit weights are as exact as that
  // themselves, and keep float32.
  const bool scaled = fp8 || dtype == GR_DTYPE_BF16;
  dn.out_type = scaled ? MM_OUT_SCALED : GR_DTYPE_F32;
  dn.out_exp = reinterpret_cast<int8_t*>(ws + l.y_exp);
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

  const CombineArgs c{out, out_stride, ws + l.y, dn.out_exp, expert_wave_cols(bm), weights, ids, T, top_k,
                      num_experts, H};
  const dim3 grid((unsigned)T, (unsigned)((H + 2047) / 2048));
  auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, c); };
  if (dtype == GR_DTYPE_BF16) go(expert_combine_k<GR_DTYPE_BF16, true>);
  else if (scaled) go(expert_combine_k<GR_DTYPE_F16, true>);
  else go(expert_combine_k<GR_DTYPE_F16, false>);
  return launch_status();
}
