// Quantisation into microscaled tiles and back: iree_uk_mi355x_mx_pack_p and iree_uk_mi355x_mx_unpack_p.
//
// Both are bound by memory: 2 or 4 bytes a value on the plain side, 0.53 or 1.03 on the other. A lane takes eight consecutive
// values of a row and four neighbouring lanes a block, so a block's maximum is two exchanges within a quad of lanes and
// nothing passes through LDS. Lanes follow each other in the order of the codes.
#include <type_traits>

#include "mx_device.h"
#include "uk_device.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

// Where the eight values of segment n (the n-th of the tiled order) lie.
struct MxPlace {
  int64_t row, col;      // in the matrix
  int64_t code, scale;   // bytes from the operand's start; of the block that the segment belongs to
};

template <typename INDEX>
struct MxShape {
  INDEX segments;             // of 8 values, in all
  INDEX row_segments, tile0, outer1;
  uint32_t row_reciprocal, tile0_reciprocal, outer1_reciprocal;
  int64_t codes_stride0, scales_stride0;
};

template <int BITS, typename INDEX>
__device__ __forceinline__ MxPlace mx_place(const MxShape<INDEX>& s, INDEX n) {
  INDEX q, seg, t0, o1, o0;
  if constexpr (sizeof(INDEX) == 4) {
    q = divide(n, s.row_segments, s.row_reciprocal);
    seg = n - q * s.row_segments;
    const INDEX tile = divide(q, s.tile0, s.tile0_reciprocal);
    t0 = q - tile * s.tile0;
    o0 = divide(tile, s.outer1, s.outer1_reciprocal);
    o1 = tile - o0 * s.outer1;
  } else {
    q = n / s.row_segments;
    seg = n - q * s.row_segments;
    const INDEX tile = q / s.tile0;
    t0 = q - tile * s.tile0;
    o0 = tile / s.outer1;
    o1 = tile - o0 * s.outer1;
  }
  MxPlace p;
  p.row = (int64_t)o0 * s.tile0 + t0;
  p.col = ((int64_t)o1 * s.row_segments + seg) * 8;
  const int64_t in_panel = ((int64_t)o1 * s.tile0 + t0) * s.row_segments + seg;
  p.code = (int64_t)o0 * s.codes_stride0 + in_panel * BITS;
  p.scale = (int64_t)o0 * s.scales_stride0 + in_panel / 4;
  return p;
}

template <typename INDEX>
struct MxPackKernelArgs {
  MxShape<INDEX> shape;
  const uint8_t* in;
  uint8_t* codes;
  uint8_t* scales;
  int64_t in_stride0, in_stride1, in_size0, in_size1;
  // mx_pack_transposed: rows and blocks of a row, padded; workgroups' rows.
  uint32_t rows, blocks, down, down_reciprocal, row_blocks_reciprocal;
};

template <typename INDEX>
struct MxUnpackKernelArgs {
  MxShape<INDEX> shape;
  const uint8_t* codes;
  const uint8_t* scales;
  uint8_t* out;
  int64_t out_stride0, out_stride1, out_size0, out_size1;
};

// A whole block: its scale byte, and its codes.
template <int BITS, Float T>
__device__ __forceinline__ uint32_t mx_block(const MxEight<T> (&v)[4], uint32_t codes[BITS]) {
  uint32_t largest = 0;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const uint32_t m = mx_largest<T>(v[h]);
    largest = m > largest ? m : largest;
  }
  const uint32_t b = mx_scale_byte<BITS>(largest);
#pragma unroll
  for (int h = 0; h < 4; ++h) mx_codes<BITS, T>(v[h], b, codes + h * (BITS / 4));
  return b;
}

// Rows whose values are next to each other (in_stride1 == 1). STREAM: past the caches. 14336 x 4096 f32 to E2M1 45.2 us, 5.9 TB/s.
template <Float T, int BITS, int AT_ONCE, bool STREAM, typename INDEX>
__global__ __launch_bounds__(kThreads) void mx_pack_rows(const MxPackKernelArgs<INDEX> a) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  const INDEX first = (INDEX)blockIdx.x * (kThreads * AT_ONCE) + threadIdx.x;
  MxEight<T> v[AT_ONCE];
  MxPlace p[AT_ONCE];
#pragma unroll
  for (int u = 0; u < AT_ONCE; ++u) {
    const INDEX n = first + (INDEX)(u * kThreads);
    if (n >= a.shape.segments) break;
    p[u] = mx_place<BITS>(a.shape, n);
    const int64_t left = p[u].row < a.in_size0 ? a.in_size1 - p[u].col : 0;
    mx_load<T, STREAM>(v[u], a.in + (p[u].row * a.in_stride0 + p[u].col) * SIZE, left);
  }
#pragma unroll
  for (int u = 0; u < AT_ONCE; ++u) {
    if (first + (INDEX)(u * kThreads) >= a.shape.segments) break;  // (segments come in fours: a block's lanes leave together)
    const uint32_t b = mx_scale_byte<BITS>(mx_largest_of_block(mx_largest<T>(v[u])));
    uint32_t codes[BITS / 4];
    mx_codes<BITS, T>(v[u], b, codes);
    __builtin_memcpy(a.codes + p[u].code, codes, BITS);
    if (threadIdx.x % 4 == 0) a.scales[p[u].scale] = (uint8_t)b;
  }
}

// Any strides: a lane takes a whole block and neighbouring lanes neighbouring rows, whose values are next to each other in a
// transposed matrix. A wavefront takes 64 rows and the four of a workgroup four blocks of them that follow each other, so that
// the codes of a row that share a cache line are written together.
template <Float T, int BITS>
__global__ __launch_bounds__(kThreads) void mx_pack_strided(const MxPackKernelArgs<uint64_t> a) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  const MxShape<uint64_t>& s = a.shape;
  const uint64_t row_blocks = s.row_segments / 4, blocks = s.outer1 * row_blocks, rows = s.segments / (4 * blocks);
  const uint64_t down = (rows + 63) / 64, across = (blocks + 3) / 4;
  for (uint64_t n = blockIdx.x; n < down * across; n += gridDim.x) {
    const uint64_t row = n % down * 64 + threadIdx.x % 64, block = n / down * 4 + threadIdx.x / 64;
    if (row >= rows || block >= blocks) continue;
    const uint64_t o0 = row / s.tile0, t0 = row - o0 * s.tile0, o1 = block / row_blocks, in_row = block - o1 * row_blocks;
    const int64_t left = (int64_t)row < a.in_size0 ? a.in_size1 - (int64_t)block * 32 : 0;
    const uint8_t* const from = a.in + ((int64_t)row * a.in_stride0 + (int64_t)block * 32 * a.in_stride1) * SIZE;
    const int64_t step = a.in_stride1 * SIZE;
    uint32_t x[32];
    if (left >= 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = SIZE == 4 ? *(const uint32_t*)(from + i * step) : *(const uint16_t*)(from + i * step);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        x[i] = i >= left ? 0u : SIZE == 4 ? *(const uint32_t*)(from + i * step) : *(const uint16_t*)(from + i * step);
    }
    MxEight<T> v[4];
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int i = 0; i < MxEight<T>::kWords; ++i)
        v[h].w[i] = SIZE == 4 ? x[8 * h + i] : x[8 * h + 2 * i] | x[8 * h + 2 * i + 1] << 16;
    uint32_t codes[BITS];
    const uint32_t b = mx_block<BITS, T>(v, codes);
    const int64_t in_panel = (int64_t)((o1 * s.tile0 + t0) * s.row_segments + in_row * 4);
    __builtin_memcpy(a.codes + (int64_t)o0 * s.codes_stride0 + in_panel * BITS, codes, 4 * BITS);
    a.scales[(int64_t)o0 * s.scales_stride0 + in_panel / 4] = (uint8_t)b;
  }
}

// A transposed matrix (in_stride0 == 1) whose columns and their distance are multiples of 16 bytes: 128 of K of 64 rows (128 of a
// 16-bit type) go straight to LDS, 16 bytes a lane along the rows, and lanes take whole blocks out of it, a word (one value, or
// two neighbouring rows' values) at a time, 64 of them next to each other. Codes go out through LDS too, 16 bytes a lane in the
// order of the tile. 14336 x 4096 f32 to E2M1 from memory: 46.3 us, 5.8 TB/s; a lane loading its own block 72.5 us. STREAM: past the
// caches.
template <Float T, int BITS, bool STREAM>
__global__ __launch_bounds__(kThreads) void mx_pack_transposed(const MxPackKernelArgs<uint32_t> a) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2, AT_ONCE = 4 / SIZE, ROWS = 64 * AT_ONCE;  // rows of a lane, of a workgroup
  constexpr int LOADS = 128 * 256 / (kThreads * 16), PIECES = BITS / 4;                     // of a lane; 16 bytes of a block's codes
  __shared__ uint4 values[128 * 16];                                                      // [k][ROWS]: 256 bytes each
  __shared__ uint32_t scales[ROWS];
  const MxShape<uint32_t>& s = a.shape;
  const uint32_t row_blocks = s.row_segments / 4;
  const uint32_t rows = a.rows, blocks = a.blocks, down = a.down;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = divide(blockIdx.x, down, a.down_reciprocal);
  const uint32_t first_row = (blockIdx.x - group * down) * ROWS, first_block = group * 4;
  const int64_t k0 = (int64_t)first_block * 32;

  // Load n of a wavefront: K (n * 4 + wave) * 4 + lane / 16, 16 lanes for the 256 bytes of its rows.
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)values;
  const int64_t load_row = first_row + (lane & 15) * (16 / SIZE);
#pragma unroll
  for (int n = 0; n < LOADS; ++n) {
    const int k = (n * 4 + wave) * 4 + (lane >> 4);
    if (load_row < a.in_size0 && k0 + k < a.in_size1) {
      const uint8_t* const from = a.in + ((k0 + k) * a.in_stride1 + load_row) * SIZE;
      const uint32_t to = lds + (n * 4 + wave) * 1024;
      if constexpr (STREAM) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(to), "v"(from) : "memory");
      else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  // A wavefront's block: words [k][lane].
  const uint32_t* const words = (const uint32_t*)values + (wave * 32) * 64 + lane;
  const int64_t left = a.in_size1 - k0 - wave * 32;
  uint32_t x[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = words[i * 64];
  if (left < 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = i < left ? x[i] : 0;
  }
  if (first_row + lane * AT_ONCE >= a.in_size0) {  // (rows come in whole loads)
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = 0;
  }
  uint32_t codes[AT_ONCE][BITS], b[AT_ONCE];
#pragma unroll
  for (int t = 0; t < AT_ONCE; ++t) {
    MxEight<T> v[4];
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int i = 0; i < MxEight<T>::kWords; ++i)
        v[h].w[i] = SIZE == 4 ? x[8 * h + i] : __builtin_amdgcn_perm(x[8 * h + 2 * i + 1], x[8 * h + 2 * i], t == 0 ? 0x05040100 : 0x07060302);
    b[t] = mx_block<BITS, T>(v, codes[t]);
  }
  __syncthreads();
  // [row][block][piece], the pieces of a row exchanged among themselves by its number so that lanes write to different banks.
  constexpr int ROW_PIECES = 4 * PIECES;
#pragma unroll
  for (int t = 0; t < AT_ONCE; ++t) {
    const int row = lane * AT_ONCE + t;
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      const int at = (wave * PIECES + c) ^ (row / AT_ONCE % ROW_PIECES);
      values[row * ROW_PIECES + at] = make_uint4(codes[t][4 * c], codes[t][4 * c + 1], codes[t][4 * c + 2], codes[t][4 * c + 3]);
    }
    ((uint8_t*)scales)[row * 4 + wave] = (uint8_t)b[t];
  }
  __syncthreads();
#pragma unroll
  for (int n = threadIdx.x; n < ROWS * ROW_PIECES; n += kThreads) {
    const int row = n / ROW_PIECES, piece = n % ROW_PIECES, block = piece / PIECES;
    const uint32_t r = first_row + row, k = first_block + block;
    if (r >= rows || k >= blocks) continue;
    const uint32_t o0 = divide(r, s.tile0, s.tile0_reciprocal), o1 = divide(k, row_blocks, a.row_blocks_reciprocal);
    const int64_t in_panel = (int64_t)(o1 * (uint64_t)s.tile0 + (r - o0 * s.tile0)) * row_blocks + (k - o1 * row_blocks);
    *(uint4*)(a.codes + (int64_t)o0 * s.codes_stride0 + in_panel * (4 * BITS) + piece % PIECES * 16) =
        values[row * ROW_PIECES + (piece ^ (row / AT_ONCE % ROW_PIECES))];
    if (piece % PIECES == 0) a.scales[(int64_t)o0 * s.scales_stride0 + in_panel] = ((const uint8_t*)scales)[row * 4 + block];
  }
}

// A lane's values make 16 bytes of the result, eight of a 16-bit type or four of f32 (with eight, whose stores leave every other
// 16 bytes to the next instruction, 14336 x 4096 E2M1 to f32 took 59.1 us, through the caches; now 48.2, and 38.9, 6.8 TB/s, with
// STREAM, past the caches).
template <Float T, int BITS, int AT_ONCE, bool STREAM, typename INDEX>
__global__ __launch_bounds__(kThreads) void mx_unpack_rows(const MxUnpackKernelArgs<INDEX> a) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2, VALUES = 16 / SIZE, SHARES = 8 / VALUES;
  const INDEX items = a.shape.segments * SHARES;
  // (One turn, but for operands of 2^33 values and more.)
  for (INDEX first = (INDEX)blockIdx.x * (kThreads * AT_ONCE) + threadIdx.x; first < items;
       first += (INDEX)gridDim.x * (kThreads * AT_ONCE)) {
    uint32_t codes[AT_ONCE][2], b[AT_ONCE];
    MxPlace p[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const INDEX n = first + (INDEX)(u * kThreads);
      if (n >= items) break;
      p[u] = mx_place<BITS>(a.shape, n / SHARES);
      const int share = SHARES == 1 ? 0 : (int)(n % SHARES);
      p[u].col += share * VALUES;
      codes[u][0] = codes[u][1] = 0;
      __builtin_memcpy(codes[u], a.codes + p[u].code + share * (VALUES * BITS / 8), VALUES * BITS / 8);
      b[u] = a.scales[p[u].scale];
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (first + (INDEX)(u * kThreads) >= items) break;
      int64_t left = p[u].row < a.out_size0 ? a.out_size1 - p[u].col : 0;
      if (left <= 0) continue;
      float f[8];
      mx_values<BITS>(codes[u], b[u], f);
      uint8_t* const at = a.out + (p[u].row * a.out_stride0 + p[u].col * a.out_stride1) * SIZE;
      if (a.out_stride1 == 1 && left >= VALUES) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (T == Float::kF32) w[i] = __builtin_bit_cast(uint32_t, f[i]);
          else w[i] = mx_narrow_pair<T>(f[2 * i], f[2 * i + 1]);
        }
        mx_store_sixteen<STREAM>(at, w);
      } else {
#pragma unroll
        for (int i = 0; i < VALUES; ++i)
          if (i < left) mx_store_eight<T>(at + i * a.out_stride1 * SIZE, f + i, 1);
      }
    }
  }
}

template <typename INDEX>
MxShape<INDEX> mx_shape(int64_t outer0, int64_t outer1, int64_t tile0, int64_t tile1, int64_t codes_stride0,
                        int64_t scales_stride0) {
  MxShape<INDEX> s;
  s.row_segments = (INDEX)(tile1 / 8);
  s.tile0 = (INDEX)tile0;
  s.outer1 = (INDEX)outer1;
  s.segments = (INDEX)(outer0 * outer1 * tile0 * (tile1 / 8));
  s.row_reciprocal = s.tile0_reciprocal = s.outer1_reciprocal = 0;
  if constexpr (sizeof(INDEX) == 4) {
    s.row_reciprocal = reciprocal_of(s.row_segments);
    s.tile0_reciprocal = reciprocal_of(s.tile0);
    s.outer1_reciprocal = reciprocal_of(s.outer1);
  }
  s.codes_stride0 = codes_stride0;
  s.scales_stride0 = scales_stride0;
  return s;
}

// (Fits: the tiles of a result lie apart in memory.)
int64_t segments_of(int64_t outer0, int64_t outer1, int64_t tile0, int64_t tile1) { return outer0 * outer1 * tile0 * (tile1 / 8); }

// Loads of a matrix past the caches: with a weight matrix from memory, up to 14336 x 4096 f32, in 46.3 us where loads through the
// caches take 51.2 (transposed; row by row 45.2 and 47.4), 14336 x 4096 bf16 27.4 and 30.7 (24.8 and 27.8). One that the
// last-level cache holds takes up to a quarter more (38.6 us of the first through the caches), and smaller ones it may hold.
bool streams_input(int64_t bytes) { return bytes > (96ll << 20); }

// Stores past the caches: 14336 x 4096 f32 in 38.9 us, through the caches 48.2, and with a kernel that reads the result 134.6 and 146.3.
// Smaller results are faster alone too (4096 x 4096 bf16 7.2 us, 9.1), but not with their reader (21.1, 19.6; 117 MB 72.3, 65.4), and
// rows that are not aligned are not (14336 x 4095 f32 73.0, 72.0; 4096 x 4095 20.3, 14.2).
bool streams_output(int64_t bytes, bool aligned) { return aligned && bytes > (192ll << 20); }

template <Float T, int BITS>
hipError_t pack(const MxPackArgs& a, hipStream_t stream, const char** name) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  const int64_t segments = segments_of(a.outer0, a.outer1, a.tile0, a.tile1);
  auto fill = [&](auto& k) {
    k.in = a.in; k.codes = a.codes; k.scales = a.scales;
    k.in_stride0 = a.in_stride0; k.in_stride1 = a.in_stride1;
    k.in_size0 = a.in_size0; k.in_size1 = a.in_size1;
  };
  if (a.in_stride1 == 1 && segments < (1ll << 31)) {
    MxPackKernelArgs<uint32_t> k;
    k.shape = mx_shape<uint32_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
    fill(k);
    *name = "mx_pack_rows";
    constexpr int MANY = 4;
    if (segments >= (int64_t)MANY * kThreads * 1024)
      return launch_kernel(streams_input(a.in_size0 * a.in_size1 * SIZE) ? mx_pack_rows<T, BITS, MANY, true, uint32_t>
                                                                         : mx_pack_rows<T, BITS, MANY, false, uint32_t>,
                           (unsigned)((segments + MANY * kThreads - 1) / (MANY * kThreads)), kThreads, 0, stream, k);
    return launch_kernel(mx_pack_rows<T, BITS, 1, false, uint32_t>, (unsigned)((segments + kThreads - 1) / kThreads), kThreads, 0,
                         stream, k);
  }
  auto sixteens = [](int64_t bytes) { return bytes % 16 == 0; };
  const int64_t rows = a.outer0 * a.tile0, blocks = a.outer1 * (a.tile1 / 32), fours = (blocks + 3) / 4;
  const int64_t down = (rows + 256 / SIZE - 1) / (256 / SIZE);
  if (a.in_stride0 == 1 && segments < (1ll << 31) && rows < (1ll << 31) - 256 && down * fours < (1ll << 23) &&
      sixteens((int64_t)(uintptr_t)a.in) && sixteens(a.in_stride1 * SIZE) && sixteens(a.in_size0 * SIZE) &&
      sixteens((int64_t)(uintptr_t)a.codes) && sixteens(a.codes_stride0)) {
    MxPackKernelArgs<uint32_t> k;
    k.shape = mx_shape<uint32_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
    fill(k);
    k.rows = (uint32_t)rows;
    k.blocks = (uint32_t)blocks;
    k.down = (uint32_t)down;
    k.down_reciprocal = reciprocal_of(k.down);
    k.row_blocks_reciprocal = reciprocal_of((uint32_t)(a.tile1 / 32));
    *name = "mx_pack_transposed";
    return launch_kernel(streams_input(a.in_size0 * a.in_size1 * SIZE) ? mx_pack_transposed<T, BITS, true> : mx_pack_transposed<T, BITS, false>,
                         (unsigned)(down * fours), kThreads, 0, stream, k);
  }
  MxPackKernelArgs<uint64_t> k;
  k.shape = mx_shape<uint64_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
  fill(k);
  *name = "mx_pack_strided";
  const int64_t groups = (rows + 63) / 64 * fours;
  return launch_kernel(mx_pack_strided<T, BITS>, (unsigned)(groups < (1 << 22) ? groups : 1 << 22), kThreads, 0, stream, k);
}

template <Float T, int BITS>
hipError_t unpack(const MxUnpackArgs& given, hipStream_t stream, const char** name) {
  // Tiles that hold nothing of the result are not visited (panels may coincide, so that their number says nothing).
  MxUnpackArgs a = given;
  a.outer0 = (a.out_size0 - 1) / a.tile0 + 1;
  a.outer1 = (a.out_size1 - 1) / a.tile1 + 1;
  const int64_t segments = segments_of(a.outer0, a.outer1, a.tile0, a.tile1);
  auto fill = [&](auto& k) {
    k.codes = a.codes; k.scales = a.scales; k.out = a.out;
    k.out_stride0 = a.out_stride0; k.out_stride1 = a.out_stride1;
    k.out_size0 = a.out_size0; k.out_size1 = a.out_size1;
  };
  *name = "mx_unpack_rows";
  constexpr int MANY = 4;
  const int64_t items = segments * (T == Float::kF32 ? 2 : 1);
  if (items < (1ll << 31)) {
    MxUnpackKernelArgs<uint32_t> k;
    k.shape = mx_shape<uint32_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
    fill(k);
    if (items >= (int64_t)MANY * kThreads * 1024) {
      constexpr int SIZE = T == Float::kF32 ? 4 : 2;
      const bool aligned = (uintptr_t)a.out % 16 == 0 && a.out_stride0 * SIZE % 16 == 0 && a.out_stride1 == 1;
      return launch_kernel(streams_output(a.out_size0 * a.out_size1 * SIZE, aligned) ? mx_unpack_rows<T, BITS, MANY, true, uint32_t>
                                                                                     : mx_unpack_rows<T, BITS, MANY, false, uint32_t>,
                           (unsigned)((items + MANY * kThreads - 1) / (MANY * kThreads)), kThreads, 0, stream, k);
    }
    return launch_kernel(mx_unpack_rows<T, BITS, 1, false, uint32_t>, (unsigned)((items + kThreads - 1) / kThreads), kThreads, 0,
                         stream, k);
  }
  MxUnpackKernelArgs<uint64_t> k;
  k.shape = mx_shape<uint64_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
  fill(k);
  return launch_kernel(mx_unpack_rows<T, BITS, MANY, false, uint64_t>, 1u << 21, kThreads, 0, stream, k);
}

}  // namespace

hipError_t launch_mx_pack(const MxPackArgs& a, hipStream_t stream, const char** name) {
  const bool four = a.bits == 4;
  switch (a.type) {
    case Float::kF32: return four ? pack<Float::kF32, 4>(a, stream, name) : pack<Float::kF32, 8>(a, stream, name);
    case Float::kF16: return four ? pack<Float::kF16, 4>(a, stream, name) : pack<Float::kF16, 8>(a, stream, name);
    default: return four ? pack<Float::kBf16, 4>(a, stream, name) : pack<Float::kBf16, 8>(a, stream, name);
  }
}

hipError_t launch_mx_unpack(const MxUnpackArgs& a, hipStream_t stream, const char** name) {
  const bool four = a.bits == 4;
  switch (a.type) {
    case Float::kF32: return four ? unpack<Float::kF32, 4>(a, stream, name) : unpack<Float::kF32, 8>(a, stream, name);
    case Float::kF16: return four ? unpack<Float::kF16, 4>(a, stream, name) : unpack<Float::kF16, 8>(a, stream, name);
    default: return four ? unpack<Float::kBf16, 4>(a, stream, name) : unpack<Float::kBf16, 8>(a, stream, name);
  }
}

}  // namespace uk
