// Gated products: the choice of kernel, and the kernel with one thread for each result, which takes every tile shape, stride and
// alignment.
#include <cmath>

#include "gated_mmt4d.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

struct GenericArgs {
  GatedArgs p;
  Curve curve;
  int64_t results;
};

template <Float T>
__global__ __launch_bounds__(kThreads) void gated_mmt4d_generic(const GenericArgs g) {
  const GatedArgs& a = g.p;
  const int64_t tile = (int64_t)a.M0 * a.N0;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t o = n / tile, within = n % tile;
    const int64_t i = o / a.N, j = o % a.N;
    const int64_t i0 = within / a.N0, j0 = within % a.N0;
    const uint16_t* lhs = (const uint16_t*)a.lhs + i * a.lhs_stride0 + i0 * a.K0;
    const uint16_t* gate = (const uint16_t*)a.gate + j * a.gate_stride0 + j0 * a.K0;
    const uint16_t* up = (const uint16_t*)a.up + j * a.up_stride0 + j0 * a.K0;
    float sum_g = 0, sum_u = 0;
    for (int64_t k = 0; k < a.K; ++k) {
      for (int k0 = 0; k0 < a.K0; ++k0) {
        const float x = mx_widen<T>(lhs[k * a.M0 * a.K0 + k0]);
        sum_g += x * mx_widen<T>(gate[k * a.N0 * a.K0 + k0]);
        sum_u += x * mx_widen<T>(up[k * a.N0 * a.K0 + k0]);
      }
    }
    const int64_t in_row = j * tile + within;
    const int64_t gate_at = i * a.gate_pre_stride0 + in_row, up_at = i * a.up_pre_stride0 + in_row;
    if (a.pre_load) {
      sum_g += element(a.pre_type, a.gate_pre, gate_at);
      sum_u += element(a.pre_type, a.up_pre, up_at);
    }
    if (a.pre_store) {
      put_element(a.pre_type, a.gate_pre, gate_at, sum_g);
      put_element(a.pre_type, a.up_pre, up_at, sum_u);
    }
    put_element(a.out_type, a.out, i * a.out_stride0 + in_row, activated(g.curve, sum_g) * sum_u);
  }
}

hipError_t launch_generic(const GatedArgs& a, hipStream_t stream, const char** name) {
  GenericArgs g;
  g.p = a;
  g.curve = curve_of(a.activation);
  g.results = a.M * a.N * a.M0 * a.N0;
  const int64_t groups = (g.results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  *name = "gated_mmt4d_generic";
  return a.type == Float::kF16 ? launch_kernel(gated_mmt4d_generic<Float::kF16>, grid, kThreads, 0, stream, g)
                               : launch_kernel(gated_mmt4d_generic<Float::kBf16>, grid, kThreads, 0, stream, g);
}

// The problem as the fast kernels take it; false: they do not.
bool as_product(const GatedArgs& a, GatedProduct* p) {
  const int64_t depth = a.K * a.K0;
  if (depth == 0 || depth > 0x7FFFFFFF) return false;
  Operand16 up;
  if (!as_operand16(a.lhs, a.lhs_stride0, a.M, a.M0, a.K, a.K0, &p->lhs) ||
      !as_operand16(a.gate, a.gate_stride0, a.N, a.N0, a.K, a.K0, &p->gate) ||
      !as_operand16(a.up, a.up_stride0, a.N, a.N0, a.K, a.K0, &up))
    return false;
  p->up = a.up;
  p->up_stride0 = up.stride0;
  p->depth = (uint32_t)depth;
  GatedResults& r = p->results;
  r.out = a.out; r.gate_pre = a.gate_pre; r.up_pre = a.up_pre;
  r.out_at = layout_of(a.out_stride0, a.M0, a.N, a.N0);
  r.gate_at = layout_of(a.gate_pre_stride0, a.M0, a.N, a.N0);
  r.up_at = layout_of(a.up_pre_stride0, a.M0, a.N, a.N0);
  r.curve = curve_of(a.activation);
  r.out_type = a.out_type; r.pre_type = a.pre_type;
  r.pre_load = a.pre_load; r.pre_store = a.pre_store;
  const int e = float_bytes(a.out_type), pe = float_bytes(a.pre_type);
  r.runs = runs_of(r.out_at, a.out, a.M, e, 16 / e, 16) &&
           (!a.gate_pre || (runs_of(r.gate_at, a.gate_pre, a.M, pe, 4, 4 * pe) && runs_of(r.up_at, a.up_pre, a.M, pe, 4, 4 * pe)));
  return true;
}

// Whether the block kernels' 32-bit offsets inside a tile take the problem.
bool block_covers(const GatedProduct& p) {
  Operand16 up = p.gate;
  up.stride0 = p.up_stride0;
  return p.depth >= 32 && near16(p.lhs, 256) && near16(p.gate, 128) && near16(up, 128);
}

// Which kernel: the least of the times that a model gives, in microseconds.
//
// Block tiles: a start, and chunks of K times what one of them takes with one workgroup on a compute unit and, where LDS and
// registers hold two, with two; more workgroups than that follow each other. The weights come from memory beside that.
//
// Few rows: the workgroups of a compute unit one after the other, each its chunks times 18.4 ns for a fragment of gate and up and
// 1 to 25 ns for one of the lhs, by how many rows of a row-major matrix its neighbouring lanes read (18 through LDS); or the weights
// from memory at 6.5 TB/s, whichever is more, and a part of the other. With more than one and a half workgroups to a compute unit and
// more than 16 rows the block kernels, which read the lhs less often, are left to decide.
//
// Fitted to the times of every kernel in 530 problems drawn from 1 to 4096 rows, 64 to 28672 columns, K of 64 to 14336, row-major and
// tiled; over these the kernel taken is slower than the best one by 2.7 % in the mean, by more than 15 % in one of twenty. Those are times
// of product16_block.h's loop in every tile. Where rows of the lhs are whole cache lines nine of the tiles run product16_lines.h's, which
// is 2 to 13 % faster, each by another share: in 300 other problems like that, of 1 to 4096 rows, the kernel taken is slower than the best
// one by 3.8 % in the mean, by more than 15 % in one of twelve.
struct Choice {
  enum { kGeneric, kFew, kBlock } kernel;
  int number;
};
Choice choose(const GatedProduct& p) {
  struct Times { float start, one, two, start_again, memory; };  // two = 0: one workgroup on a compute unit; memory: TB/s
  static const Times kTimes[] = {{11.8f, .499f, 0, 19.9f, 4.14f},   {9.4f, .412f, 0, 14.1f, 4.81f},    {7.8f, .345f, 0, 11.3f, 5.75f},
                                 {9.8f, .409f, 0, 15.3f, 5.56f},    {7.3f, .325f, .888f, 3.4f, 5.47f}, {6.2f, .265f, .725f, 2.4f, 6.17f},
                                 {5.0f, .208f, .555f, 1.7f, 6.81f}, {5.2f, .254f, .613f, 1.8f, 6.93f}, {4.5f, .200f, .480f, 1.5f, 7.11f},
                                 {3.9f, .150f, .360f, 1.1f, 7.72f}, {3.1f, .124f, .229f, .8f, 8.12f}};
  static_assert(sizeof kTimes / sizeof kTimes[0] == sizeof kGatedTiles / sizeof kGatedTiles[0], "one for each tile");
  const int64_t rows = p.lhs.rows, cols = p.gate.rows;
  const float chunks = (float)((p.depth + 31) / 32), bytes = (float)cols * chunks * 128e-6f;  // of the weights, MB
  Choice best = {Choice::kGeneric, 0};
  float least = 0;
  auto consider = [&](float cost, Choice c) {
    if (best.kernel == Choice::kGeneric || cost < least) {
      least = cost;
      best = c;
    }
  };
  const float direct = p.lhs.tile_rows == 1 ? .0001f + .024f * (float)(rows < 16 ? rows - 1 : 15) / 15 : .011f;
  const float staged = p.lhs.tile_rows == 1 ? .018f : .016f;
  for (int i = 0; i < (int)(sizeof kGatedFewShapes / sizeof kGatedFewShapes[0]); ++i) {
    const GatedFewShape& s = kGatedFewShapes[i];
    const int64_t down = (rows + 16 * s.mt - 1) / (16 * s.mt), groups = down * ((cols + 16 * s.nt - 1) / (16 * s.nt));
    // (A grid has fewer than 2^32 threads, and 2^16 rows.)
    if (down > 65535 || groups > (1 << 22) || (s.staged && !near16(p.lhs, 64)) || (groups > 384 && rows > 16)) continue;
    const float rounds = (float)((groups + 255) / 256), start = 2.06f + .274f * s.mt * s.nt;
    const float loads = rounds * chunks * (s.mt * (s.staged ? staged : direct) + s.nt * .0184f), read = bytes / 6.5f;
    const float l2 = loads * loads, r2 = read * read;
    consider(start * (1 + .3f * (rounds - 1)) + sqrtf(sqrtf(l2 * l2 + r2 * r2)), {Choice::kFew, i});
  }
  if (!block_covers(p)) {
    // (With many rows and many workgroups, the plainest of the above.)
    const int64_t down = (rows + 15) / 16;
    if (best.kernel == Choice::kGeneric && down <= 65535 && down * ((cols + 15) / 16) <= (1 << 22)) return {Choice::kFew, 0};
    return best;
  }
  for (int i = 0; i < (int)(sizeof kGatedTiles / sizeof kGatedTiles[0]); ++i) {
    const GatedTile& t = kGatedTiles[i];
    const int64_t tiles = ((rows + t.rows - 1) / t.rows) * ((cols + t.cols - 1) / t.cols), rounds = (tiles + 255) / 256;
    if (tiles > (1 << 23)) continue;
    const Times& of = kTimes[i];
    const float steps = chunks * (of.two == 0 ? rounds * of.one : (rounds >> 1) * of.two + (rounds & 1) * of.one), read = bytes / of.memory;
    consider(of.start + (rounds - 1) * of.start_again + (steps > read ? steps + .15f * read : read + .15f * steps), {Choice::kBlock, i});
  }
  return best;
}

}  // namespace

hipError_t launch_gated_mmt4d(const GatedArgs& a, hipStream_t stream, const char** name) {
  GatedProduct p;
  if (!as_product(a, &p)) return launch_generic(a, stream, name);
  const Choice c = choose(p);
  if (c.kernel == Choice::kGeneric) return launch_generic(a, stream, name);
  if (c.kernel == Choice::kFew) {
    *name = kGatedFewShapes[c.number].name;
    return launch_gated_few(p, a.type, c.number, stream);
  }
  *name = kGatedTiles[c.number].name;
  return a.type == Float::kF16 ? launch_gated_block_f16(p, c.number, stream) : launch_gated_block_bf16(p, c.number, stream);
}

}  // namespace uk
