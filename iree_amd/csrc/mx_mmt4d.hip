// Products of microscaled operands: the choice of kernel, and the kernel with one thread for each result, which takes
// every tile shape, stride and alignment.
#include <type_traits>

#include "mx_mmt4d.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

struct MxGenericArgs {
  MxMmt4dArgs p;
  int64_t results;
};

// A block's 32 products are summed in f32, exactly (E2M1 times E2M1) or nearly so, then scaled and added to the total.
template <int LBITS>
__global__ __launch_bounds__(kThreads) void mx_mmt4d_generic(const MxGenericArgs g) {
  const MxMmt4dArgs& a = g.p;
  const int64_t tile = (int64_t)a.M0 * a.N0;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t o = n / tile, within = n % tile;
    const int64_t i = o / a.N, j = o % a.N;
    const int64_t i0 = within / a.N0, j0 = within % a.N0;
    const int blocks = a.K0 / 32;
    const uint8_t* lhs = a.lhs + i * a.lhs_stride0;
    const uint8_t* rhs = a.rhs + j * a.rhs_stride0;
    const uint8_t* lhs_scales = a.lhs_scales + i * a.lhs_scales_stride0;
    const uint8_t* rhs_scales = a.rhs_scales + j * a.rhs_scales_stride0;
    float sum = 0;
    for (int64_t k = 0; k < a.K; ++k) {
      for (int b = 0; b < blocks; ++b) {
        const int64_t l_at = (k * a.M0 + i0) * blocks + b, r_at = (k * a.N0 + j0) * blocks + b;
        float part = 0;
        for (int s = 0; s < 4; ++s) {  // eight values at a time
          uint32_t lw[LBITS / 4], rw[1];
          __builtin_memcpy(lw, lhs + l_at * (4 * LBITS) + s * LBITS, LBITS);
          __builtin_memcpy(rw, rhs + r_at * 16 + s * 4, 4);
          float x[8], y[8];
          mx_values<LBITS>(lw, 127, x);
          mx_values<4>(rw, 127, y);
          for (int e = 0; e < 8; ++e) part += x[e] * y[e];
        }
        const int ls = lhs_scales[l_at], rs = rhs_scales[r_at];
        sum += ls == 255 || rs == 255 ? __builtin_nanf("") : ldexpf(part, ls + rs - 254);
      }
    }
    const int64_t at = i * a.out_stride0 + j * tile + within;
    if (a.out_type == Float::kF32) {
      float* out = (float*)a.out + at;
      *out = a.accumulate ? *out + sum : sum;
    } else if (a.out_type == Float::kF16) {
      uint16_t* out = (uint16_t*)a.out + at;
      *out = mx_narrow<Float::kF16>(a.accumulate ? mx_widen<Float::kF16>(*out) + sum : sum);
    } else {
      uint16_t* out = (uint16_t*)a.out + at;
      *out = mx_narrow<Float::kBf16>(a.accumulate ? mx_widen<Float::kBf16>(*out) + sum : sum);
    }
  }
}

hipError_t launch_generic(const MxMmt4dArgs& a, hipStream_t stream, const char** name) {
  MxGenericArgs g;
  g.p = a;
  g.results = a.M * a.N * a.M0 * a.N0;
  const int64_t groups = (g.results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  *name = "mx_mmt4d_generic";
  return a.lhs_bits == 4 ? launch_kernel(mx_mmt4d_generic<4>, grid, kThreads, 0, stream, g)
                         : launch_kernel(mx_mmt4d_generic<8>, grid, kThreads, 0, stream, g);
}

// Whether a row of an operand's tiles has its K in chunks of 128 that lie a tile apart.
bool in_chunks(int32_t tile_rows, int32_t k0) { return tile_rows == 1 || k0 == 128; }

bool aligned(const void* p, int64_t stride, int64_t rows, int64_t to) {
  return (uintptr_t)p % to == 0 && (rows == 1 || stride % to == 0);
}

// The problem as the fast kernels take it; false: they do not.
bool as_product(const MxMmt4dArgs& a, MxProduct* p) {
  const int64_t rows = a.M * a.M0, cols = a.N * a.N0, depth = a.K * a.K0;
  if (depth == 0 || depth % 128 != 0 || depth / 128 > 0x7FFFFFFF || !in_chunks(a.M0, a.K0) || !in_chunks(a.N0, a.K0)) return false;
  if (rows > 0x7FFFFFFF - 256 || cols > 0x7FFFFFFF - 256) return false;
  if (!aligned(a.lhs, a.lhs_stride0, a.M, 16) || !aligned(a.rhs, a.rhs_stride0, a.N, 16) ||
      !aligned(a.lhs_scales, a.lhs_scales_stride0, a.M, 4) || !aligned(a.rhs_scales, a.rhs_scales_stride0, a.N, 4))
    return false;
  const int out_bytes = float_bytes(a.out_type);
  p->lhs = {a.lhs, a.lhs_scales, a.lhs_stride0, a.lhs_scales_stride0, (uint32_t)rows, (uint32_t)a.M0, reciprocal_of((uint32_t)a.M0)};
  p->rhs = {a.rhs, a.rhs_scales, a.rhs_stride0, a.rhs_scales_stride0, (uint32_t)cols, (uint32_t)a.N0, reciprocal_of((uint32_t)a.N0)};
  p->out = a.out;
  p->out_stride0 = a.out_stride0;
  p->chunks = (uint32_t)(depth / 128);
  p->n0 = (uint32_t)a.N0;
  p->n0_reciprocal = reciprocal_of((uint32_t)a.N0);
  p->out_tile = (uint32_t)a.M0 * (uint32_t)a.N0;
  p->out_type = a.out_type;
  p->accumulate = a.accumulate;
  // (Tiles one row tall and one column wide are a row-major result.)
  if (a.M0 == 1 && a.N0 == 1) {
    p->n0 = p->rhs.rows;
    p->n0_reciprocal = reciprocal_of(p->n0);
    p->out_tile = 0;
  }
  p->fours = (p->n0 % 4 == 0 || (a.M0 == 1 && a.N0 == 1)) && aligned(a.out, a.out_stride0 * out_bytes, a.M, 4 * out_bytes);
  return true;
}

// Whether rows up to 256 (or `apart`) apart lie within 32 bits of each other.
bool near(const MxOperand& o, int64_t apart = 256) {
  const int64_t panels = apart / o.tile_rows + 2, most = 1ll << 31;
  return o.stride0 < most / panels && o.scales_stride0 < most / panels;
}

// Whether the block kernels' 32-bit offsets inside a tile, and their stores of eight rows at a time, take the problem.
bool block_covers(const MxProduct& p) {
  const uint32_t m0 = p.lhs.tile_rows;
  if (m0 != 1 && m0 % 8 != 0) return false;
  return near(p.lhs) && near(p.rhs) && (m0 > 1 || p.out_stride0 < (1ll << 26)) && p.out_tile < (1ll << 28) / (256 / p.n0 + 2);
}

// Which kernel: the least of the times that a model gives, in microseconds.
//
// Block tiles: a start, and chunks of K times what one of them takes with one workgroup on a compute unit and, where LDS and
// registers hold two, with two; more workgroups than that follow each other. From the times of every tile with 128 to 1024 of
// them, row-major lhs, K = 1024 and 5120. The rhs comes from memory beside that.
//
// Few rows: a workgroup's loads and its matrix instructions (and, with more workgroups than compute units, what a start costs again),
// or the rhs from memory at 6.4 TB/s with a share of what the loads of the lhs take, whichever is more, and a part of the other.
// Sixteen rows of a chunk straight into registers take 19 to 23 ns a KiB where they lie in a tile, 5 to 20 where they are one row to
// sixteen rows of a matrix (30 of a rhs); through LDS 19 (4 bits) and 11 (8 bits). Fitted to the times of every shape in 880 problems.
//
// The lhs in registers: the rhs at 6.1 TB/s, less where wavefronts or workgroups have no part of it.
//
// Over these, drawn from 1 to 4096 rows, 64 to 32768 columns, K of 64 to 16384, with tiles and row-major, the kernel taken is
// slower than the best one by 2 % in the mean. For 16-bit results of an E4M3 lhs the constants are those of products with one matrix
// instruction each, not two: 3.5 % in the mean of 101 problems, from 1 to 4096 rows (1.4 % with those of f32 results).
struct Choice {
  enum { kGeneric, kFew, kResident, kBlock } kernel;
  int number;
};
Choice choose(const MxProduct& p, int lhs_bits) {
  struct Times { float start, one, two, start_again; };
  static const Times kE2m1[] = {{12.1f, .898f, 1.731f, 11}, {4.9f, .344f, .639f, 2.2f}, {5.8f, .444f, .817f, 2.7f},
                                {7.6f, .531f, 1.093f, 5}, {3.4f, .219f, .333f, 1}, {3.8f, .271f, .499f, 1.3f}, {3.9f, .265f, .457f, 1.4f}};
  static const Times kE4m3[] = {{12, 1.247f, 2.494f, 9.5f}, {4.6f, .441f, .813f, 2.5f}, {6.2f, .565f, 1.155f, 4},
                                {8, .710f, 1.456f, 5.7f}, {3.5f, .247f, .396f, 1}, {3.9f, .315f, .572f, 1.1f}, {3.9f, .288f, .501f, 1.3f}};
  static const Times kE4m3F32[] = {{14.4f, 2.67f, 5.42f, 11}, {6.6f, .929f, 1.544f, 2}, {7.5f, 1.169f, 2.339f, 4},
                                   {10.1f, 1.396f, 2.846f, 5}, {3.6f, .488f, .65f, 1}, {4.5f, .732f, 1.071f, 1.9f}, {4.5f, .537f, .871f, 1.4f}};
  const Times* times = lhs_bits == 4 ? kE2m1 : p.out_type == Float::kF32 ? kE4m3F32 : kE4m3;
  const int64_t rows = p.lhs.rows, cols = p.rhs.rows;
  Choice best = {Choice::kGeneric, 0};
  float least = 0;
  const bool eight = lhs_bits == 8, split = times == kE4m3F32, lhs_near = near(p.lhs);
  const float row_major = (eight ? 2 : 1) * (.0049f + .0151f * (float)(rows < 16 ? rows - 1 : 15) / 15);
  const float lhs_direct = p.lhs.tile_rows >= 16 && !eight ? .019f : row_major, lhs_staged = eight ? .0237f : .0188f;
  const float rhs_chunk = p.rhs.tile_rows >= 16 ? .0232f : .0295f, product = split ? .0105f : .0003f;
  const float memory = (float)cols * p.chunks * 68e-6f;
  for (int i = 0; i < (int)(sizeof kMxFewShapes / sizeof kMxFewShapes[0]); ++i) {
    const MxFewShape& s = kMxFewShapes[i];
    const int64_t down = (rows + 16 * s.mt - 1) / (16 * s.mt), across = (cols + 16 * s.nt - 1) / (16 * s.nt);
    // (A grid has fewer than 2^32 threads, and 2^16 rows.)
    if (down > 65535 || down * across > (1 << 22) || (s.staged && !lhs_near)) continue;
    const float rounds = (float)((down * across + 255) / 256), start = 1.94f + .286f * s.mt * s.nt;
    const float lhs = s.mt * (s.staged ? lhs_staged : lhs_direct) * p.chunks;
    const float loads = rounds * (lhs + (s.nt * rhs_chunk + s.mt * s.nt * product) * p.chunks) + (rounds - 1) * .321f * start;
    const float streamed = memory / 6.41f + .137f / 256 * (float)(down * across) * lhs;
    const float cost = start + (loads > streamed ? loads + .115f * streamed : streamed + .115f * loads);
    if (best.kernel == Choice::kGeneric || cost < least) {
      least = cost;
      best = {Choice::kFew, i};
    }
  }
  // (Up to three rows are read as quickly by every workgroup anew: one of E4M3 x 57008 x 4096 22.0 us, here 24.0; but not beside the
  // rows of a matrix: x 28672 x 8192 30.7 and 29.0.)
  if (rows <= 16 && (rows >= 4 || p.rhs.tile_rows < 16) && p.chunks <= kMxResidentChunks && comes_from_hbm(cols * p.chunks * 64)) {
    const int64_t panels = (cols + 15) / 16, most = (panels + kMxResidentGroups - 1) / kMxResidentGroups;
    if (lhs_near && near(p.rhs, 16 * most)) {
      // (32 or 64 chunks of every panel are loaded, the last one over and over where K has fewer, and some workgroups have a panel
      // less than the others.)
      const float fours = (float)((p.chunks + 3) / 4), held = p.chunks <= 32 ? 8 : 16;
      const float each = .5f * ((float)most + (float)panels / kMxResidentGroups);
      const float read = memory / (float)panels * kMxResidentGroups * each / 6.1f * held / fours;
      const float cost = 2 + 1.5f / most + (eight ? .5f : 0) + read + (split ? .004f * most * p.chunks : 0);
      if (best.kernel == Choice::kGeneric || cost < least) {
        least = cost;
        best = {Choice::kResident, 0};
      }
    }
  }
  if (!block_covers(p)) return best;
  for (int i = 0; i < (int)(sizeof kMxBlockTiles / sizeof kMxBlockTiles[0]); ++i) {
    const MxBlockTile& t = kMxBlockTiles[i];
    const int64_t tiles = ((rows + 64 * t.am - 1) / (64 * t.am)) * ((cols + 64 * t.bn - 1) / (64 * t.bn)), rounds = (tiles + 255) / 256;
    if (tiles > (1 << 23)) continue;
    const float steps = p.chunks * ((rounds >> 1) * times[i].two + (rounds & 1) * times[i].one);
    const float read = memory / 7.2f;
    const float cost = times[i].start + (rounds - 1) * times[i].start_again + (steps > read ? steps + .116f * read : read + .182f * steps);
    if (best.kernel == Choice::kGeneric || cost < least) {
      least = cost;
      best = {Choice::kBlock, i};
    }
  }
  return best;
}

}  // namespace

hipError_t launch_mx_mmt4d(const MxMmt4dArgs& a, hipStream_t stream, const char** name) {
  MxProduct p;
  if (!as_product(a, &p)) return launch_generic(a, stream, name);
  const Choice c = choose(p, a.lhs_bits);
  if (c.kernel == Choice::kGeneric) return launch_generic(a, stream, name);
  if (c.kernel == Choice::kFew) {
    *name = kMxFewShapes[c.number].name;
    return launch_mx_few(p, a.lhs_bits, c.number, stream);
  }
  if (c.kernel == Choice::kResident) {
    *name = "mx_mmt4d_resident";
    return launch_mx_resident(p, a.lhs_bits, stream);
  }
  *name = kMxBlockTiles[c.number].name;
  return a.lhs_bits == 4 ? launch_mx_block_e2m1(p, c.number, stream) : launch_mx_block_e4m3(p, c.number, stream);
}

}  // namespace uk
