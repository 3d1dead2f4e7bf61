// The chosen experts' SwiGLU layers with 4-bit microscaled weights (gr_mx_mm.h): the
// tokens are quantised once, each expert's gated product is written in 4 bits, and its
// result waits for the sum over a token's experts in float32.
#include <algorithm>
#include <cmath>

#include "gr_expert_rows.h"
#include "gr_mx_mm.h"

#include "gr_mxfp4.h"

namespace gr {
namespace {

// The tokens are quantised by the workgroups behind those that sort (or count, where
// several do).
template <int DT> __global__ __launch_bounds__(PLAN_THREADS) void mx_expert_start_k(PlanArgs a, MxQuantArgs q) {
  __shared__ int next[MAX_EXPERTS], part[PLAN_THREADS / 64];
  if ((int)blockIdx.x >= a.blocks)
    mx_quant_item<DT>(q, (blockIdx.x - a.blocks) * PLAN_THREADS + threadIdx.x);
  else if (a.blocks > 1)
    expert_count(a, next);
  else
    expert_plan(a, next, part);
}

struct MxWorkspace {
  int64_t hist, slot, tiles, num_tiles, x4, xs, act, act_scale, y, bytes;
  int blocks;
};

// Rows of a tile.  By the rows an expert gets on average: few rows are bound by the weights'
// way from memory, many by the products and the results.  Measured (64 experts of 768
// features, hidden 2048, 8 of them a token; us of both products, by tile rows):
//   rows an expert    8    16    24    28    32    48    64    80    96   128   192   224   256   300   375   625
//    32            33.1  40.8  42.2  45.5  47.3  51.8  66.0
//    64            40.0  42.2  43.8  44.5  45.1  47.7  55.2  65.0  69.4  82.6
//   128                        49.9  50.8  50.9  55.3  58.8  64.5  67.3  81.5  99.1   112   119   139   163   252
//   256                                                                  93.0  99.4   119   125   137   143   222
// A tall tile is for many workgroups: where the gated product has fewer than 136 (some more than half the CUs),
// the next lower one is taken.  Over 76 sizes of 1 to 160 experts of 128 to 6144 features, hidden 512 to 4096, the pick
// is 1.3 % slower than the best tile in the mean and 17 % at most; by the rows alone 12 % and 131 % (us; E experts of F
// features, hidden H: tiles of 256, 128, 64 and 32 rows):
//   1200 rows, E 4, F 256, H 512     20.4  12.5  10.5   9.5    32 taken
//   1000 rows, E 8, F 512, H 2048    31.4  20.4  16.0  15.8    64
//   4000 rows, E 8, F 512, H 2048    35.5  27.9  31.4  33.4   128
//   4096 rows, E 8, F 1024, H 4096   67.9  72.2  69.2  93.0   256
int mx_up_cols(int bm) { return bm <= 64 ? 64 : 128; }  // results of the gated product that a workgroup has
int mx_tile_rows(int64_t rows, int E, int F) {
  int bm = rows <= 28ll * E ? 32 : rows <= 72ll * E ? 64 : rows <= 260ll * E ? 128 : 256;
  auto workgroups = [&] {  // (half of each expert's last tile is empty)
    return (rows / bm + (std::min<int64_t>(rows, E) + 1) / 2) * (((int64_t)F + mx_up_cols(bm) - 1) / mx_up_cols(bm));
  };
  while (bm > 32 && workgroups() < 136) bm /= 2;
  return bm;
}

int64_t mx_most_tiles(int64_t rows, int E, int bm) { return rows / bm + std::min<int64_t>(rows, E); }

// (H and F: sizes of which a call is refused too)
MxWorkspace plan_mx_workspace(int T, int k, int E, int64_t H, int64_t F) {
  MxWorkspace w{};
  const int64_t rows = (int64_t)T * k;
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  w.blocks = (int)((rows + PLAN_ROWS - 1) / PLAN_ROWS);
  w.num_tiles = take(4);
  w.hist = take(4ll * w.blocks * E);
  w.slot = take(4 * rows);
  w.tiles = take(16 * mx_most_tiles(rows, E, 32));  // (of the lowest ones: more tokens, of taller tiles, need no less)
  w.x4 = take((int64_t)T * ((H + 1) / 2));
  w.xs = take((int64_t)T * ((H + 31) / 32));
  w.act = take(rows * ((F + 1) / 2));
  w.act_scale = take(rows * ((F + 31) / 32));
  w.y = take(4 * rows * H);
  return w;
}

// The products' forms: rows of a tile, the gated product's stages on their way, the down product's columns.
struct MxForm { int bm, up_stages, down_cols; };
MxForm pick_mx_experts(int64_t rows, int E, int H, int F) {
  const int bm = mx_tile_rows(rows, E, F);
  if (bm > 32) return {bm, bm == 256 ? 2 : 3, bm == 256 ? 256 : 128};
  // Few rows: what counts is that all workgroups of a product are on the CUs at once.  Of the experts, choices
  // that fall evenly reach `reached`.  Up: 64 results a workgroup, two workgroups a CU with three stages each, or
  // three with two.  Down: 64 columns, six a CU, or 256, two a CU.  Where all fit in the second form only it is
  // taken, else the first (64 experts of 768 features, hidden 2048, 8 a token; us):
  //   tokens                     1     8    12    16    64    80    96   128
  //   workgroups up             96   483   619   680   768   768   768   768
  //   three stages             7.3  12.9  19.1  20.3  25.9  27.0  26.9  26.4
  //   two                      9.7  12.7  15.8  16.8  21.0  24.2  27.8  28.4
  //   down 64                  4.3   8.1   9.7  11.8  13.5  13.5  13.7  14.4
  //   down 256                 5.7   9.4   9.5   9.8  12.2  13.6  15.9  16.6
  const double reached = E * (1.0 - std::exp(-(double)rows / E));
  const double wgs = reached * ((F + 63) / 64), wide = reached * ((H + 255) / 256);
  const bool once = rows <= 10ll * E;  // (more rows give some experts a second tile)
  return {32, once && wgs > 512 && wgs <= 768 ? 2 : 3, once && wide <= 512 && reached * ((H + 63) / 64) > 1536 ? 256 : 64};
}

void launch_mx_experts(const MxArgs& up, const MxArgs& down, int tiles, const MxForm& f, hipStream_t stream) {
  if (f.bm == 32) {
    if (f.up_stages == 2) launch_mx<32, 128, 2, 2, 2, 2, MM_SWIGLU_Q, true>(up, tiles, stream);
    else launch_mx<32, 128, 2, 2, 3, 2, MM_SWIGLU_Q, true>(up, tiles, stream);
    if (f.down_cols == 256) launch_mx<32, 256, 1, 4, 2, 1, MM_PLAIN, true>(down, tiles, stream);
    else launch_mx<32, 64, 2, 1, 2, 1, MM_PLAIN, true>(down, tiles, stream);
  } else if (f.bm == 64) {
    launch_mx<64, 128, 2, 2, 3, 2, MM_SWIGLU_Q, true>(up, tiles, stream);
    launch_mx<64, 128, 2, 2, 2, 1, MM_PLAIN, true>(down, tiles, stream);
  } else if (f.bm == 128) {
    launch_mx<128, 256, 2, 4, 3, 2, MM_SWIGLU_Q, true>(up, tiles, stream);
    launch_mx<128, 128, 4, 2, 2, 1, MM_PLAIN, true>(down, tiles, stream);
  } else {
    launch_mx<256, 256, 2, 4, 2, 2, MM_SWIGLU_Q, true>(up, tiles, stream);
    launch_mx<256, 256, 2, 4, 2, 2, MM_PLAIN, true>(down, tiles, stream);
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace gr

using namespace gr;

extern "C" size_t gr_expert_mlp_mxfp4_workspace_size(int num_tokens, int top_k, int num_experts, int hidden, int ffn) {
  if (num_tokens < 1 || top_k < 1 || num_experts < 1 || hidden < 1 || ffn < 1) return 0;
  return (size_t)plan_mx_workspace(num_tokens, top_k, num_experts, hidden, ffn).bytes;
}

extern "C" int gr_expert_mlp_mxfp4_tile(int num_tokens, int top_k, int num_experts, int hidden, int ffn) {
  if (num_tokens < 1 || top_k < 1 || num_experts < 1 || hidden < 1 || ffn < 1 || hidden > (1 << 21) || ffn > (1 << 21)) return 0;
  const MxForm f = pick_mx_experts((int64_t)num_tokens * top_k, num_experts, hidden, ffn);
  return 1000000 * f.up_stages + 1000 * f.bm + f.down_cols;
}

extern "C" gr_status_t gr_expert_mlp_mxfp4(void* out, int64_t out_stride, const void* x, int64_t x_stride,
                                           const void* gate_up, const uint8_t* gate_up_scale, const void* down,
                                           const uint8_t* down_scale, const float* weights, const int32_t* ids,
                                           int num_tokens, int top_k, int num_experts, int hidden, int ffn, int dtype,
                                           void* workspace, size_t workspace_bytes, int32_t* dev_status,
                                           hipStream_t stream) {
  if (num_tokens < 0 || top_k < 1 || num_experts < 1 || hidden < 1 || ffn < 1 || !dtype_valid(dtype))
    return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  if (!out || !x || !gate_up || !gate_up_scale || !down || !down_scale || !weights || !ids || out_stride < hidden ||
      x_stride < hidden)
    return GR_ERR_INVALID_ARG;
  const int T = num_tokens, H = hidden, F = ffn;
  if (dtype == GR_DTYPE_F32 || hidden % 32 != 0 || ffn % 32 != 0 || hidden > (1 << 21) || ffn > (1 << 21) ||
      num_experts > MAX_EXPERTS || (int64_t)T * top_k > (1 << 26) || !aligned(x, 16) || x_stride % 8 != 0 ||
      !aligned(gate_up, 16) || !aligned(down, 16) || !aligned(out, 8) || out_stride % 4 != 0 ||
      (int64_t)T * H > (1ll << 32) - (1 << 24))
    return GR_ERR_UNSUPPORTED;
  const MxForm form = pick_mx_experts((int64_t)T * top_k, num_experts, H, F);
  const int bm = form.bm;
  const MxWorkspace l = plan_mx_workspace(T, top_k, num_experts, H, F);
  const int64_t tiles = mx_most_tiles((int64_t)T * top_k, num_experts, bm);
  const int cols = mx_up_cols(bm);  // (the down product's workgroups have as many or more)
  if (tiles * ((std::max(F, H) + cols - 1) / cols) > GRID_MAX - 8 || T > GRID_MAX) return GR_ERR_UNSUPPORTED;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < (size_t)l.bytes) return GR_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int rows = T * top_k;

  const PlanArgs p{ids, rows, num_experts, bm, l.blocks, reinterpret_cast<int32_t*>(ws + l.hist),
                   reinterpret_cast<int32_t*>(ws + l.slot), reinterpret_cast<int4*>(ws + l.tiles),
                   reinterpret_cast<int32_t*>(ws + l.num_tiles), dev_status};
  const MxQuantArgs q{ws + l.x4, H / 2, ws + l.xs, H / 32, x, x_stride, T, H};
  const int64_t items = (int64_t)T * (H / 16);
  const dim3 start((unsigned)(l.blocks + (items + PLAN_THREADS - 1) / PLAN_THREADS));
  auto first = [&](auto k) { hipLaunchKernelGGL(k, start, dim3(PLAN_THREADS), 0, stream, p, q); };
  if (dtype == GR_DTYPE_F16) first(mx_expert_start_k<GR_DTYPE_F16>);
  else first(mx_expert_start_k<GR_DTYPE_BF16>);
  if (l.blocks > 1) hipLaunchKernelGGL(expert_plan_k, dim3(l.blocks), dim3(PLAN_THREADS), 0, stream, p);

  MxArgs up{};
  up.x = q.out;
  up.x_stride = H / 2;
  up.xs4 = q.scale;
  up.xs4_row = H / 32;
  up.w = static_cast<const uint8_t*>(gate_up);
  up.w_stride = H / 2;
  up.w_expert = 2ll * F * (H / 2);
  up.ws4 = gate_up_scale;
  up.ws4_row = H / 32;
  up.ws4_expert = 2ll * F * (H / 32);
  up.out = ws + l.act;
  up.out_stride = F / 2;
  up.os4 = ws + l.act_scale;
  up.os4_row = F / 32;
  up.M = rows;
  up.N = F;
  up.kbytes = H / 2;
  up.blocks = H / 32;
  up.scale_piece = mx_scale_piece(up);
  up.tiles = p.tiles;
  up.num_tiles = p.num_tiles;
  up.slot = p.slot;
  up.gather = top_k;
  MxArgs dn{};
  dn.x = ws + l.act;
  dn.x_stride = F / 2;
  dn.xs4 = up.os4;
  dn.xs4_row = F / 32;
  dn.w = static_cast<const uint8_t*>(down);
  dn.w_stride = F / 2;
  dn.w_expert = (int64_t)H * (F / 2);
  dn.ws4 = down_scale;
  dn.ws4_row = F / 32;
  dn.ws4_expert = (int64_t)H * (F / 32);
  // float32 (fp16 multiples of a power of two would halve what the sum reads, 5001 tokens 246 us for 291, but a
  // token's sum would be off by 2^-11 of each of its terms, however near its terms' opposites bring it to 0)
  dn.out = ws + l.y;
  dn.out_stride = H;
  dn.M = rows;
  dn.N = H;
  dn.kbytes = F / 2;
  dn.blocks = F / 32;
  dn.scale_piece = mx_scale_piece(dn);
  dn.tiles = p.tiles;
  dn.num_tiles = p.num_tiles;
  dn.slot = p.slot;
  dn.scatter = 1;
  launch_mx_experts(up, dn, (int)tiles, form, stream);

  const CombineArgs c{out, out_stride, ws + l.y, nullptr, 0, weights, ids, T, top_k, num_experts, H};
  const dim3 grid((unsigned)T, (unsigned)((H + 2047) / 2048));
  auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, c); };
  if (dtype == GR_DTYPE_BF16) go(expert_combine_k<GR_DTYPE_BF16, false>);
  else go(expert_combine_k<GR_DTYPE_F16, false>);
  return launch_status();
}
