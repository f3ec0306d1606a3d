// An update made orthogonal by Newton-Schulz products, and the optimiser's step around it.
//
//   X = U / (|U|_F + 1e-7), its shorter side as rows;  then `steps` times
//   G = X X^T,  P = b G + c G G,  X = a X + P X
//
// which takes every singular value s of X through s (a + b s^2 + c s^4) and leaves the vectors alone.  What small singular
// values there are grow by a factor a in each step (480 in five), and so does what rounding adds to them: operands of
// eleven bits leave 2 to 4 % of error in updates of low rank, so all operands are two fp16 planes (tile_product.hpp), 22 bits
// and more, with fp32 sums; the result is as near to float64 as fp32 products are, at three fp16 instructions per product.
// That holds for bf16 results too: Gram products of the hi planes alone add 1e-3 where roundings average out, but 5e-3 to an update
// whose entries have few different values, and 3.6e-2 in ten steps of steep coefficients.
//
// Planes hold kScale times their number: entries of an n x n matrix of norm one are about 1 / n, too near to the least
// fp16 numbers for a second plane; all numbers stay below 65504 / kScale (the entry points refuse coefficients that would not).  P's eigenvalues are
// b t + c t^2, which may be twice what the whole polynomial is: its planes hold half as much where they have to.
#include "tile_product.hpp"

#include <algorithm>
#include <memory>
#include <new>

namespace f2cgt {
namespace {

constexpr float kScale = 8192.f;
constexpr double kMost = 7.5;                  // of the polynomial's values; of P's before its planes hold half
constexpr int kGroup = 64;                     // matrices that one set of launches takes

// Several matrices of one shape; `rows` and `cols` as the caller has them, r <= l the sides as the products have them.
struct Matrices {
  const void* u[kGroup];                       // updates, or gradients
  void* out[kGroup];                           // results, or weights
  float* held[kGroup];                         // momenta, or null
};

struct Shape {
  int64_t rows, cols, r, l;
  int turned;                                  // rows > cols: X is the transposed update
  __host__ __device__ int64_t long_line() const { return ceil_div(l, 32) * kLine; }      // bytes of a row of X
  __host__ __device__ int64_t short_line() const { return ceil_div(r, 32) * kLine; }     // of a row of X^T, G and P
};

struct MuonArgs {
  Matrices at;
  Shape s;
  int u_dtype, out_dtype, nesterov;
  float momentum, keep, size;                  // weights: keep * w - size * o; results: keep 0
  double* partial;                             // [count][parts]
  int parts;
  char* x;                                     // [count][r] lines of X
  char* xt[2];                                 // [count][l] lines of X^T
  char* g;                                     // [count][r] lines of G
  char* p;                                     // of P
  float* sums;                                 // of parts of Gram products
  float a, b, c;
  float plane_b, plane_c, back;                // what makes P's planes of G's and of the sums of G G, and numbers of the sums of P X
  int whole;                                   // rows of the results start at multiples of four values
};

// The update's value i: the gradient, or what the momentum makes of it (held: after this step's change).
__device__ __forceinline__ float update_of(const MuonArgs& a, float grad, float held) {
  return a.nesterov ? a.momentum * held + (1.f - a.momentum) * grad : held;
}

// Four neighbours of memory, wherever they start, and fewer at its end.
template <typename T>
__device__ __forceinline__ fltx4 load_up_to_four(const void* p, int64_t i, int64_t end) {
  typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  fltx4 v = {0.f, 0.f, 0.f, 0.f};
  if (i + 4 <= end) {
    const four o = *reinterpret_cast<const four*>(static_cast<const T*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)o[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < end) v[e] = (float)static_cast<const T*>(p)[i + e];
  }
  return v;
}
__device__ __forceinline__ fltx4 load_up_to_four(const void* p, int dtype, int64_t i, int64_t end) {
  if (dtype == F2CGT_DT_F32) return load_up_to_four<float>(p, i, end);
  if (dtype == F2CGT_DT_F16) return load_up_to_four<_Float16>(p, i, end);
  return load_up_to_four<__bf16>(p, i, end);
}

// Momenta, and the sum of squares of the updates by parts, in 64 bits (a square of an fp32 number may be none).  Bound by memory:
// four bf16 gradients of 2048 x 512 and their momenta, 42 MB, 9.1 us (4.6 TB/s).
template <bool HELD>
__global__ __launch_bounds__(256) void muon_norm_kernel(MuonArgs a) {
  typedef fltx4 unaligned4 __attribute__((aligned(4)));
  constexpr int U = HELD ? 4 : 8;
  const int64_t count = a.s.rows * a.s.cols, z = blockIdx.y, step = (int64_t)gridDim.x * 1024;
  const void* u = a.at.u[z];
  float* held = a.at.held[z];
  double sum = 0.;
  for (int64_t i0 = (int64_t)blockIdx.x * 1024 + threadIdx.x * 4; i0 < count; i0 += U * step) {
    fltx4 v[U], h[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      v[k] = load_up_to_four(u, a.u_dtype, i0 + k * step, count);
      if (HELD) h[k] = load_up_to_four<float>(held, i0 + k * step, count);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (HELD) {
        const int64_t i = i0 + k * step;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[k][e] = a.momentum * h[k][e] + (1.f - a.momentum) * v[k][e];
        if (i + 4 <= count) {
          *reinterpret_cast<unaligned4*>(held + i) = h[k];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < count) held[i + e] = h[k][e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = update_of(a, v[k][e], h[k][e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += (double)v[k][e] * (double)v[k][e];
    }
  }
  __shared__ double s_sum[4];
#pragma unroll
  for (int by = 32; by > 0; by /= 2) sum += __shfl_xor(sum, by);
  if ((threadIdx.x & (kWave - 1)) == 0) s_sum[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.partial[z * a.parts + blockIdx.x] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// ---- planes ----------------------------------------------------------------------------------------------------------------
// v = hi + lo: a rounding, the exact rest rounded, and their sum.  The two ones are hidden from the compiler, so that it takes the
// instruction that multiplies and adds fp16 and fp32 numbers and does not convert them first (two instructions a value instead of
// three, one instead of three for the sum; same results: two of 256 x 128 82.9 -> 78.6 us then, with G kept in registers for P).
__device__ __forceinline__ float hidden(float one) {
  asm("" : "+s"(one));
  return one;
}
__device__ __forceinline__ _Float16 rest_of(float v, _Float16 hi) { return (_Float16)__builtin_fmaf((float)hi, hidden(-1.f), v); }
__device__ __forceinline__ float sum_of(_Float16 hi, _Float16 lo) { return __builtin_fmaf((float)hi, hidden(1.f), (float)lo); }

// ---- strips of finished tiles: 32 rows and WN columns of sums in LDS, in lanes' turns of eight neighbours -----------------
__device__ __forceinline__ void eight_of(const char* row, int64_t c, float (&v)[8]) {
  const char* line = row + (c >> 5) * kLine + 2 * (c & 31);
  const halfx8 hi = *reinterpret_cast<const halfx8*>(line), lo = *reinterpret_cast<const halfx8*>(line + 64);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = sum_of(hi[e], lo[e]);
}
__device__ __forceinline__ void put_eight(char* row, int64_t c, const float (&v)[8]) {
  halfx8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = (_Float16)v[e];
    lo[e] = rest_of(v[e], hi[e]);
  }
  char* line = row + (c >> 5) * kLine + 2 * (c & 31);
  *reinterpret_cast<halfx8*>(line) = hi;
  *reinterpret_cast<halfx8*>(line + 64) = lo;
}

// The update of length kScale in planes, both ways round: a 64 x 64 tile of the caller's matrix per workgroup.  Bound by memory, at
// 4096 x 4096 in bf16 168 MB in 34 to 41 us, and by a launch and two round trips at 1000 x 2051 (9.8 us).
__global__ __launch_bounds__(256) void muon_split_kernel(MuonArgs a) {
  __shared__ double s_sum[4];
  __shared__ float s_tile[64][65];
  const int t = threadIdx.x;
  const int64_t z = blockIdx.z, rows = a.s.rows, cols = a.s.cols;
  const int64_t row0 = (int64_t)blockIdx.x * 64, col0 = (int64_t)blockIdx.y * 64;
  const void* u = a.at.u[z];
  const float* held = a.at.held[z];
  fltx4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + t / 16 + 16 * i, col = col0 + 4 * (t % 16), end = row < rows ? (row + 1) * cols : 0;
    const int64_t from = col < cols ? row * cols + col : end;
    v[i] = load_up_to_four(u, a.u_dtype, from, end);
    if (held != nullptr) {
      const fltx4 h = load_up_to_four<float>(held, from, end);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = update_of(a, v[i][e], h[e]);
    }
  }
  double sum = 0.;
  for (int i = t; i < a.parts; i += 256) sum += a.partial[z * a.parts + i];
#pragma unroll
  for (int by = 32; by > 0; by /= 2) sum += __shfl_xor(sum, by);
  if ((t & (kWave - 1)) == 0) s_sum[t / kWave] = sum;
  __syncthreads();
  const double norm = sqrt((s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]));
  const float scale = (float)(kScale / (norm + 1e-7));
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s_tile[t / 16 + 16 * i][4 * (t % 16) + e] = v[i][e] * scale;
  __syncthreads();
  // the caller's rows are X's, or X^T's
  char* along = a.s.turned ? a.xt[0] + z * a.s.l * a.s.short_line() : a.x + z * a.s.r * a.s.long_line();
  char* across = a.s.turned ? a.x + z * a.s.r * a.s.long_line() : a.xt[0] + z * a.s.l * a.s.short_line();
  const int64_t along_line = a.s.turned ? a.s.short_line() : a.s.long_line();
  const int64_t across_line = a.s.turned ? a.s.long_line() : a.s.short_line();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = t / 8 + 32 * i, c = 8 * (t % 8);
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s_tile[r][c + e];
      y[e] = s_tile[c + e][r];
    }
    if (row0 + r < rows && (col0 + c) / 32 * 32 < cols) put_eight(along + (row0 + r) * along_line, col0 + c, x);
    if (col0 + r < cols && (row0 + c) / 32 * 32 < rows) put_eight(across + (col0 + r) * across_line, row0 + c, y);
  }
}

// change(row, col, v): eight neighbours of a row; then put(row, col, v) with them, and turned(row, col, v) with eight neighbours of
// a column from `row` on.  Rows and columns are whole eights, and may lie beyond the matrix.
template <int WN, class Change, class Turned>
__device__ __forceinline__ void strip_passes(float* strip, int64_t row0, int64_t col0, int lane, bool both, const Change& change,
                                             const Turned& turned) {
  constexpr int kLd = WN + 4, kAcross = WN / 8;
  static_assert(32 * kAcross % kWave == 0, "whole turns of the lanes");
#pragma unroll
  for (int i = 0; i < 32 * kAcross / kWave; ++i) {
    const int r = (i * kWave + lane) / kAcross, c = 8 * ((i * kWave + lane) % kAcross);
    fltx4* at = reinterpret_cast<fltx4*>(strip + r * kLd + c);
    const fltx4 a = at[0], b = at[1];
    float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    change(row0 + r, col0 + c, v);
    if (both) {
      at[0] = fltx4{v[0], v[1], v[2], v[3]};
      at[1] = fltx4{v[4], v[5], v[6], v[7]};
    }
  }
  if (!both) return;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < WN / 16; ++i) {
    const int c = i * 16 + lane / 4, r = 8 * (lane % 4);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = strip[(r + e) * kLd + c];
    turned(row0 + r, col0 + c, v);
  }
}

// G from X, or P = b G + c G G from G (g not null): the tiles on and below the diagonal, each written on both sides of it.
// At 4096 x 4096, where the card's power bounds them, G and P take 230 us each in a row of steps: 1.0e15 executed operations a second.
// At 1000 x 2051 there are 136 tiles of 64 x 64 for 256 CUs, each of whose LDS is read and written for most of the time (19.6 and
// 12.2 us); larger tiles leave more of the chip without one, and a third or fourth stage gained nothing.
template <int WN>
struct SymmetricEpilogue {
  const MuonArgs& a;
  char* out;
  const char* g;
  bool mirror;
  __device__ __forceinline__ void operator()(float* strip, int64_t row0, int64_t col0, int lane) const {
    const int64_t line = a.s.short_line(), r = a.s.r, padded = (r + 31) & ~31ll;
    strip_passes<WN>(strip, row0, col0, lane, mirror,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          if (row < r && col < padded) {
            if (g != nullptr) {
              float gv[8];
              eight_of(g + row * line, col, gv);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(a.plane_c, v[e], a.plane_b * gv[e]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] *= 1.f / kScale;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (col + e >= r) v[e] = 0.f;
            put_eight(out + row * line, col, v);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
          }
        },
        [&](int64_t row, int64_t col, const float (&v)[8]) {
          if (col < r && row < padded) put_eight(out + col * line, row, v);
        });
  }
};

template <bool SQUARE, int B, int W, int WJ, int GROUPS, int DEEP>
__global__ __launch_bounds__((B / W) * (B / WJ) * GROUPS * kWave) void muon_symmetric_kernel(MuonArgs a) {
  typedef TileProduct<SplitOp, B, B, W, WJ, GROUPS> Tile;
  __shared__ __attribute__((aligned(128))) char lds0[Tile::kStage], lds1[Tile::kStage];
  const uint32_t tiles = (uint32_t)ceil_div(a.s.r, B), each = tiles * (tiles + 1) / 2, at = place_of(blockIdx.x, gridDim.x);
  uint32_t i, j;
  lower_tile_of(at % each, tiles, DEEP, i, j);
  const int64_t z = at / each, row0 = (int64_t)B * i, col0 = (int64_t)B * j;
  const Shape& s = a.s;
  char* g = a.g + z * s.r * s.short_line();
  char* p = a.p + z * s.r * s.short_line();
  const Lines from = SQUARE ? Lines{g, s.short_line(), s.r, s.short_line()}
                            : Lines{a.x + z * s.r * s.long_line(), s.long_line(), s.r, s.long_line()};
  Tile::run({lds0, lds1}, from, from, row0, col0, SymmetricEpilogue<WJ>{a, SQUARE ? p : g, SQUARE ? g : nullptr, row0 != col0});
}

// G of a long X with few rows: its columns in `splits` parts for as many workgroups of a tile, whose sums of 64 x 64 go to memory...
struct PartEpilogue {
  float* sums;
  __device__ __forceinline__ void operator()(float* strip, int64_t row, int64_t col, int lane) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + lane / 8, c = 4 * (lane % 8);
      *reinterpret_cast<fltx4*>(sums + (row + r) * 64 + col + c) = *reinterpret_cast<const fltx4*>(strip + r * 36 + c);
    }
  }
};

__global__ __launch_bounds__(1024) void muon_gram_part_kernel(MuonArgs a, int splits) {
  typedef TileProduct<SplitOp, 64, 64, 32, 32, 4> Tile;
  __shared__ __attribute__((aligned(128))) char lds0[Tile::kStage], lds1[Tile::kStage];
  const Shape& s = a.s;
  // the parts of a tile go to different XCDs, tiles of a part to the same
  const uint32_t tiles = (uint32_t)ceil_div(s.r, 64), each = tiles * (tiles + 1) / 2, all = gridDim.x / splits, at = place_of(blockIdx.x, gridDim.x);
  const uint32_t part = at / all, tile = at % all;
  uint32_t i, j;
  lower_tile_of(tile % each, tiles, 8, i, j);
  const int64_t z = tile / each, steps = s.long_line() / kLine;
  const int64_t first = steps * part / splits, end = steps * (part + 1) / splits;
  const char* x = a.x + z * s.r * s.long_line() + first * kLine;
  const int64_t here = (end - first) * kLine;
  const Lines row_lines{x + 64 * i * s.long_line(), s.long_line(), s.r - 64 * i, here};
  const Lines col_lines{x + 64 * j * s.long_line(), s.long_line(), s.r - 64 * j, here};
  Tile::run({lds0, lds1}, row_lines, col_lines, 0, 0, PartEpilogue{a.sums + ((int64_t)tile * splits + part) * 4096});
}

// ... and are added, in their order, a quarter of a tile per wave.
__global__ __launch_bounds__(256) void muon_gram_add_kernel(MuonArgs a, int splits) {
  __shared__ __attribute__((aligned(16))) float s_strip[4][32 * 36];
  const Shape& s = a.s;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, wi = 32 * (wave >> 1), wj = 32 * (wave & 1);
  const uint32_t tiles = (uint32_t)ceil_div(s.r, 64), each = tiles * (tiles + 1) / 2, tile = blockIdx.x;
  uint32_t i, j;
  lower_tile_of(tile % each, tiles, 8, i, j);
  const int64_t z = tile / each;
  const float* sums = a.sums + (int64_t)tile * splits * 4096 + wi * 64 + wj;
  fltx4 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = fltx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < splits; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += *reinterpret_cast<const fltx4*>(sums + p * 4096 + (k * 8 + lane / 8) * 64 + 4 * (lane % 8));
#pragma unroll
  for (int k = 0; k < 4; ++k) *reinterpret_cast<fltx4*>(&s_strip[wave][(k * 8 + lane / 8) * 36 + 4 * (lane % 8)]) = v[k];
  __builtin_amdgcn_wave_barrier();
  SymmetricEpilogue<32>{a, a.g + z * s.r * s.short_line(), nullptr, i != j}(s_strip[wave], 64 * i + wi, 64 * j + wj, lane);
}

// How many parts: as many as make a workgroup per CU, of eight steps at least, where that saves more than the addition costs (4 us; a
// step 0.28).  99 x 2721: 24 us in one part.  1 where it does not.
int gram_splits(int64_t n, const Shape& s) {
  const int64_t tiles = n * ceil_div(s.r, 64) * (ceil_div(s.r, 64) + 1) / 2, steps = ceil_div(s.l, 32), cus = num_cus();
  int64_t splits = cus / tiles;
  if (splits > steps / 8) splits = steps / 8;
  return splits >= 2 && steps - steps / splits >= 20 ? (int)splits : 1;
}

// X = a X + P X in planes, both ways round, or the last one into the caller's matrix.  At 4096 x 4096 371 us in a row of steps, 1.1e15
// executed operations a second at the 1.5 GHz that the card's power leaves (the library's fp16 product of 8192 x 8192 x 8192 in a long run 1.32e15);
// 22 us at 1000 x 2051.  (a X from its own planes: with a in P's diagonal, which is rounded to 22 bits there, errors were half as much again.)
template <int WN>
struct UpdateEpilogue {
  const MuonArgs& a;
  int64_t z;
  char* xt;                                    // null: the last one
  __device__ __forceinline__ void operator()(float* strip, int64_t row0, int64_t col0, int lane) const {
    const Shape& s = a.s;
    const int64_t padded_r = (s.r + 31) & ~31ll, padded_l = (s.l + 31) & ~31ll;
    const bool last = xt == nullptr;
    strip_passes<WN>(strip, row0, col0, lane, !last || s.turned,
        [&](int64_t row, int64_t col, float (&v)[8]) {
          if (row < s.r && col < padded_l) {
            char* x = a.x + (z * s.r + row) * s.long_line();
            float xv[8];
            eight_of(x, col, xv);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = col + e < s.l ? __builtin_fmaf(v[e], a.back, a.a * xv[e]) : 0.f;
            if (!last) put_eight(x, col, v);
            else if (!s.turned) result(row, col, s.l, v);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
          }
        },
        [&](int64_t row, int64_t col, const float (&v)[8]) {
          if (col >= s.l || row >= padded_r) return;
          if (!last) put_eight(xt + (z * s.l + col) * s.short_line(), row, v);
          else result(col, row, s.r, v);
        });
  }
  // Eight neighbours of a row of the caller's matrix, of rows of `end` values.
  __device__ __forceinline__ void result(int64_t row, int64_t col, int64_t end, const float (&v)[8]) const {
    void* w = a.at.out[z];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const int64_t at = row * end + col + e;
      if (a.whole && col + e < end) {
        fltx4 o;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = v[e + d] * (1.f / kScale);
        if (a.keep != 0.f) {
          const fltx4 before = load_four(w, a.out_dtype, at);
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] = a.keep * before[d] - a.size * o[d];
        }
        store_four(w, a.out_dtype, at, o);
      } else {
#pragma unroll
        for (int d = 0; d < 4; ++d)
          if (col + e + d < end) {
            float o = v[e + d] * (1.f / kScale);
            if (a.keep != 0.f) o = a.keep * load_value(w, a.out_dtype, at + d) - a.size * o;
            store_value(w, a.out_dtype, at + d, o);
          }
      }
    }
  }
};

template <int BM, int BN, int WM, int WN, int GROUPS, int DEEP>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * GROUPS * kWave) void muon_update_kernel(MuonArgs a, int from, int last) {
  typedef TileProduct<SplitOp, BM, BN, WM, WN, GROUPS> Tile;
  __shared__ __attribute__((aligned(128))) char lds0[Tile::kStage], lds1[Tile::kStage];
  const Shape& s = a.s;
  const uint32_t tiles_r = (uint32_t)ceil_div(s.r, BM), tiles_l = (uint32_t)ceil_div(s.l, BN), at = place_of(blockIdx.x, gridDim.x);
  uint32_t i, j;
  tile_of(at % (tiles_r * tiles_l), tiles_r, tiles_l, DEEP, i, j);
  const int64_t z = at / (tiles_r * tiles_l);
  const Lines p{a.p + z * s.r * s.short_line(), s.short_line(), s.r, s.short_line()};
  const Lines x{a.xt[from] + z * s.l * s.short_line(), s.short_line(), s.l, s.short_line()};
  Tile::run({lds0, lds1}, p, x, (int64_t)BM * i, (int64_t)BN * j, UpdateEpilogue<WN>{a, z, last ? nullptr : a.xt[1 - from]});
}

template <int B, int W, int WJ, int GROUPS, int DEEP>
void launch_symmetric(const MuonArgs& a, int64_t n, bool square, hipStream_t st) {
  const int64_t tiles = ceil_div(a.s.r, B);
  const unsigned grid = (unsigned)(n * tiles * (tiles + 1) / 2);
  constexpr int kBlock = (B / W) * (B / WJ) * GROUPS * kWave;
  if (square) muon_symmetric_kernel<true, B, W, WJ, GROUPS, DEEP><<<grid, kBlock, 0, st>>>(a);
  else muon_symmetric_kernel<false, B, W, WJ, GROUPS, DEEP><<<grid, kBlock, 0, st>>>(a);
}

template <int BM, int BN, int WM, int WN, int GROUPS, int DEEP>
void launch_update(const MuonArgs& a, int64_t n, int from, int last, hipStream_t st) {
  const unsigned grid = (unsigned)(n * ceil_div(a.s.r, BM) * ceil_div(a.s.l, BN));
  muon_update_kernel<BM, BN, WM, WN, GROUPS, DEEP><<<grid, (BM / WM) * (BN / WN) * GROUPS * kWave, 0, st>>>(a, from, last);
}

// Which tiles.  Time of a step of 32 summed columns, in 10 ns, by tiles per CU, and steps' worth of a tile's begin and end:
//   128 x 128 in eight waves, two workgroups a CU: one tile 67, two 93, so 93 for each pair and 67 for a last one; 6 steps
//   192 x 192 in four waves (symmetric products): 133 each; 8 steps.  64 x 128 in eight waves (updates), three a CU: 30 each
//   64 x 64: 47 for one, 22 each for many; 2 steps.  With four groups of waves 31 for one
// us of Gram products of 1000 x 2051: 64 x 64 30, in four groups 19.5, 128 x 128 42; 2048 x 2048: 34, 54, 42; eight of 1000 x 700: 18, 27, 24;
// 3000 x 3000: 97, 128, 86, 192 x 192 128; 4096 x 4096: 195, 262, 169, 168 (528 and 253 tiles).
// Updates: 1000 x 2051: 64 x 64 20.8, 64 x 128 23.5, 128 x 128 27.1; 2048 x 2048: 50, 43, 49; 3000 x 3000: 160, 130, 142;
// 4096 x 4096: 349, 284, 237, 256 x 256 299.  (tests/test_gpu_dense_forms.py and test_gpu_muon.py have a shape for each.)
int64_t pairs_cost(int64_t tiles, int64_t cus) {
  const int64_t left = tiles % (2 * cus);
  return 93 * (tiles / (2 * cus)) + (left == 0 ? 0 : left <= cus ? 67 : 93);
}

void symmetric(const MuonArgs& a, int64_t n, bool square, hipStream_t st) {
  auto tiles = [&](int64_t b) { return n * ceil_div(a.s.r, b) * (ceil_div(a.s.r, b) + 1) / 2; };
  const int64_t cus = num_cus(), steps = ceil_div(square ? a.s.r : a.s.l, 32);
  const int64_t small = (steps + 2) * 22 * tiles(64) / cus;
  const int64_t middle = (steps + 6) * pairs_cost(tiles(128), cus), large = (steps + 8) * 133 * ceil_div(tiles(192), cus);
  if (tiles(64) <= cus) launch_symmetric<64, 32, 32, 4, 8>(a, n, square, st);
  else if (tiles(128) < cus || (small < middle && small < large)) launch_symmetric<64, 32, 32, 1, 8>(a, n, square, st);
  else if (middle <= large) launch_symmetric<128, 64, 32, 1, 8>(a, n, square, st);
  else launch_symmetric<192, 96, 96, 1, 6>(a, n, square, st);
}

void update(const MuonArgs& a, int64_t n, int from, int last, hipStream_t st) {
  const int64_t cus = num_cus(), middle = n * ceil_div(a.s.r, 128) * ceil_div(a.s.l, 128);
  const int64_t flat = n * ceil_div(a.s.r, 64) * ceil_div(a.s.l, 128);
  if (2 * flat <= 3 * cus) launch_update<64, 64, 32, 32, 1, 8>(a, n, from, last, st);
  else if (30 * ceil_div(flat, cus) <= pairs_cost(middle, cus)) launch_update<64, 128, 32, 32, 1, 8>(a, n, from, last, st);
  else launch_update<128, 128, 64, 32, 1, 8>(a, n, from, last, st);
}

// ---- small matrices: a workgroup each, from the update to the result in one launch --------------------------------------
// X stays in registers, in fp32: a wave has the 32-column strips wave, wave + 8, ... as the matrix instructions leave their sums
// (a lane: one column, of eight rows its side's four).  That is also what they take as a second operand, if the first
// one's columns are in the same order; so P X needs no X in LDS.
constexpr int kOneWaves = 8;

// Row v of a lane's sixteen values of a 32 x 32 tile.
__device__ __forceinline__ int tile_row(int v, int side) { return 8 * (v / 4) + 4 * side + v % 4; }

// Where a lane's sixteen values of tile (i, column tile c) lie in the caller's matrix: those outside it have the place of one
// inside.
struct TilePlaces {
  int from, down, rows;                                    // of its column; from a row to the next; rows from its first one on
  bool column;
  __device__ __forceinline__ TilePlaces(const Shape& m, int i, int c) {
    const int lane = threadIdx.x & (kWave - 1), col = 32 * c + (lane & 31), row = 32 * i + 4 * (lane >> 5);
    down = m.turned ? 1 : (int)m.cols;
    column = col < (int)m.l;
    rows = (int)m.r - row;
    from = (column ? col : (int)m.l - 1) * (m.turned ? (int)m.cols : 1) + row * down;
  }
  __device__ __forceinline__ bool whole(int q) const { return 8 * q + 4 <= rows; }       // rows of values 4 q to 4 q + 3
  __device__ __forceinline__ bool in(int v) const { return column && tile_row(v, 0) < rows; }
  __device__ __forceinline__ int at(int v) const { return from + (tile_row(v, 0) < rows ? tile_row(v, 0) : rows - 1) * down; }
};

// (four neighbours in memory at once where the columns of X are the caller's rows)
template <typename T>
__device__ __forceinline__ fltx16 load_tile(const void* m, const TilePlaces& p) {
  typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  fltx16 x;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const T* from = static_cast<const T*>(m) + p.at(4 * q);
    if (p.down == 1 && p.whole(q)) {
      const four o = *reinterpret_cast<const four*>(from);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * q + e] = (float)o[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * q + e] = (float)static_cast<const T*>(m)[p.at(4 * q + e)];
    }
  }
  return x;
}
__device__ __forceinline__ fltx16 load_tile(const void* m, int dtype, const TilePlaces& p) {
  if (dtype == F2CGT_DT_F32) return load_tile<float>(m, p);
  if (dtype == F2CGT_DT_F16) return load_tile<_Float16>(m, p);
  return load_tile<__bf16>(m, p);
}
template <typename T>
__device__ __forceinline__ void store_tile(void* m, const TilePlaces& p, const fltx16& x) {
  typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (p.down == 1 && p.whole(q)) {
      if (!p.column) continue;
      four o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (T)x[4 * q + e];
      *reinterpret_cast<four*>(static_cast<T*>(m) + p.at(4 * q)) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (p.in(4 * q + e)) static_cast<T*>(m)[p.at(4 * q + e)] = (T)x[4 * q + e];
    }
  }
}

// Strips of the update, of length `to` (momenta kept).
template <int RT, int S>
__device__ __forceinline__ void load_strips(const MuonArgs& a, int64_t z, double* s_sum, float to, fltx16 (&x)[S][RT]) {
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;
  double sum = 0.;
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const TilePlaces p(a.s, i, wave + kOneWaves * s);
      fltx16 o = load_tile(a.at.u[z], a.u_dtype, p);
      if (a.at.held[z] != nullptr) {
        fltx16 h = load_tile<float>(a.at.held[z], p);
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          h[v] = a.momentum * h[v] + (1.f - a.momentum) * o[v];
          o[v] = update_of(a, o[v], h[v]);
        }
        store_tile<float>(a.at.held[z], p, h);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        if (!p.in(v)) o[v] = 0.f;
        sum += (double)o[v] * (double)o[v];
      }
      x[s][i] = o;
    }
#pragma unroll
  for (int by = 32; by > 0; by /= 2) sum += __shfl_xor(sum, by);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  double all = 0.;
#pragma unroll
  for (int i = 0; i < kOneWaves; ++i) all += s_sum[i];
  const float scale = (float)((double)to / (sqrt(all) + 1e-7));
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) x[s][i][v] *= scale;
}

template <int RT, int S>
__device__ __forceinline__ void store_strips(const MuonArgs& a, int64_t z, float by, const fltx16 (&x)[S][RT]) {
  const int wave = threadIdx.x / kWave;
  void* w = a.at.out[z];
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const TilePlaces p(a.s, i, wave + kOneWaves * s);
      fltx16 o;
#pragma unroll
      for (int v = 0; v < 16; ++v) o[v] = x[s][i][v] * by;
      if (a.keep != 0.f) {
        const fltx16 before = load_tile(w, a.out_dtype, p);
#pragma unroll
        for (int v = 0; v < 16; ++v) o[v] = a.keep * before[v] - a.size * o[v];
      }
      if (a.out_dtype == F2CGT_DT_F32) store_tile<float>(w, p, o);
      else if (a.out_dtype == F2CGT_DT_F16) store_tile<_Float16>(w, p, o);
      else store_tile<__bf16>(w, p, o);
    }
}

// Up to 32 rows, all in fp32 (32 x 32 x 2 instructions): a product of this size is latency, not rate.  32 x 256 19 us, 20 x 300 27,
// 16 x 128 15, 48 of 32 x 128 16; of five steps, each three products that need each other, four barriers and a sum over the waves, 2.5 to 5
// us a step.  P, 32 x 32, is one wave's.
template <int S>
__global__ __launch_bounds__(kOneWaves * kWave) void muon_narrow_kernel(MuonArgs a, int steps) {
  constexpr int kRow = 32 + 4;                             // floats of a row of 32 in LDS
  __shared__ double s_sum[kOneWaves];
  __shared__ __attribute__((aligned(16))) float s_x[kOneWaves][S][32][kRow], s_g[kOneWaves][32][kRow], s_p[32][kRow];
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave), at = lane & 31, side = lane >> 5;
  const int64_t z = blockIdx.x;
  fltx16 x[S][1];
  load_strips<1, S>(a, z, s_sum, 1.f, x);
  for (int step = 0; step < steps; ++step) {
    // G: each wave the part of its own columns, in the order of a lane's reads
    fltx16 g;
#pragma unroll
    for (int v = 0; v < 16; ++v) g[v] = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (32 * (wave + kOneWaves * s) >= a.s.l) break;
#pragma unroll
      for (int v = 0; v < 16; ++v) s_x[wave][s][tile_row(v, side)][at] = x[s][0][v];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const fltx4 k = *reinterpret_cast<const fltx4*>(&s_x[wave][s][at][8 * q + 4 * side]);
#pragma unroll
        for (int e = 0; e < 4; ++e) g = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], k[e], g, 0, 0, 0);
      }
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) s_g[wave][tile_row(v, side)][at] = g[v];
    __syncthreads();
    for (int i = t; i < 1024; i += kOneWaves * kWave) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kOneWaves; ++w) sum += s_g[w][i / 32][i % 32];
      s_p[i / 32][i % 32] = sum;                           // (G, until it is P)
    }
    __syncthreads();
    if (wave == 0) {
      fltx16 square;
#pragma unroll
      for (int v = 0; v < 16; ++v) square[v] = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const fltx4 k = *reinterpret_cast<const fltx4*>(&s_p[at][8 * q + 4 * side]);
#pragma unroll
        for (int e = 0; e < 4; ++e) square = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], k[e], square, 0, 0, 0);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) square[v] = a.b * s_p[tile_row(v, side)][at] + a.c * square[v];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int v = 0; v < 16; ++v) s_p[tile_row(v, side)][at] = square[v];
    }
    __syncthreads();
    fltx16 sum[S];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < 16; ++v) sum[s][v] = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const fltx4 k = *reinterpret_cast<const fltx4*>(&s_p[at][8 * q + 4 * side]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int s = 0; s < S; ++s)
          if (32 * (wave + kOneWaves * s) < a.s.l) sum[s] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], x[s][0][4 * q + e], sum[s], 0, 0, 0);
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < 16; ++v) x[s][0][v] = a.a * x[s][0][v] + sum[s][v];
    // (s_p is written again behind the next step's first barrier, s_g in front of it: read before this step's second)
  }
  store_strips<1, S>(a, z, 1.f, x);
}

// Four neighbours of a row of 32 as planes in a line of LDS, from piece `piece`, half `half` on.
__device__ __forceinline__ void put_four(char* lds, int line, int piece, int half, const float (&v)[4]) {
  halfx4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hi[e] = (_Float16)v[e];
    lo[e] = rest_of(v[e], hi[e]);
  }
  *reinterpret_cast<halfx4*>(lds + piece_at(line, piece) + 8 * half) = hi;
  *reinterpret_cast<halfx4*>(lds + piece_at(line, piece + 4) + 8 * half) = lo;
}

// Two rows of a lane's column -> two columns of a row, an even lane's first, an odd one's second (turn: the bytes to take).
__device__ __forceinline__ uint32_t beside(halfx2 rows, uint32_t turn) {
  const uint32_t own = __builtin_bit_cast(uint32_t, rows);
  const uint32_t next = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xF, 0xF, true);      // (of lane ^ 1)
  return __builtin_amdgcn_perm(next, own, turn);
}

// 48 of 128 x 128 in bf16 48 us, two of 256 x 128 in fp32 74.  Of a step's 27 thousand clocks in the latter G takes 7500 and its planes
// 2200, P 5300, the update 8100 and the writing of X's lines 4100 (6000 value by value instead of by pairs); 15 400 of them issue matrix instructions on each SIMD,
// the rest is the splitting of values, reads and writes of LDS, and the waits between three products that need each other.  Tiles over the whole chip would
// be seventeen launches, 4 us and more each.  Up to 128 columns there are four strips of them, and half of the waves have none in the
// update and the writing of X's lines.
//
// From 33 to 32 RT rows: products of planes.  LDS: X's lines, a column tile of 32
// after the other, while G is made; then G's and P's, of 32 RT rows by RT column tiles each, in the same place.  Where there is
// room G's lie behind X's, and no wave waits for the others' products before it writes its part.
template <int RT, int S>
__global__ __launch_bounds__(kOneWaves * kWave) void muon_one_kernel(MuonArgs a, int steps) {
  constexpr int kRows = 32 * RT, kTile = kRows * kLine;    // a column tile
  constexpr int kTiles = S * kOneWaves > 2 * RT ? S * kOneWaves : 2 * RT;
  constexpr int TJ = (RT + 1) / 2;                         // column tiles of a wave, in products of square matrices
  __shared__ double s_sum[kOneWaves];
  __shared__ __attribute__((aligned(128))) char lds[kTiles * kTile];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t z = blockIdx.x;
  const int columns = (int)ceil_div(a.s.l, 32);
  const bool apart = columns + RT <= kTiles;
  char* gl = lds + (apart ? columns : 0) * kTile;
  char* pl = lds + (apart ? 0 : RT) * kTile;
  fltx16 x[S][RT];
  load_strips<RT, S>(a, z, s_sum, kScale, x);
  // tiles (i, j0 ...) of square products
  const int i0 = wave / 2, j0 = (wave & 1) * TJ;
  const bool squares = i0 < RT;
  // rows i of a times rows j of b, column tiles [0, n)
  auto product = [&](const char* of, int n, int at, int side, fltx16 (&sum)[TJ]) {
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) sum[j][v] = 0.f;
    for (int c = 0; c < n; ++c) {
      const char* tile = of + c * kTile;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        intx4 fa[2], fb[TJ][2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          fa[p] = *reinterpret_cast<const intx4*>(tile + piece_at(32 * i0 + at, 4 * p + 2 * g + side));
#pragma unroll
          for (int j = 0; j < TJ; ++j) {
            const int jj = j0 + j < RT ? j0 + j : RT - 1;
            fb[j][p] = *reinterpret_cast<const intx4*>(tile + piece_at(32 * jj + at, 4 * p + 2 * g + side));
          }
        }
#pragma unroll
        for (int m = 0; m < SplitOp::kTerms; ++m) {
#pragma unroll
          for (int j = 0; j < TJ; ++j) SplitOp::mma(sum[j], m, fa, fb[j]);
        }
      }
    }
  };
  for (int step = 0; step < steps; ++step) {
    // (places in LDS are made anew in each step: kept across all of it they are more than the registers hold)
    int lane_of = (int)threadIdx.x & (kWave - 1);
    asm volatile("" : "+v"(lane_of));
    const int at = lane_of & 31, side = lane_of >> 5;
    // X's lines: a lane has a column; of two rows each, neighbours exchange one
    const uint32_t turn = at & 1 ? 0x03020706 : 0x05040100;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int c = wave + kOneWaves * s;
      if (c < columns) {
        // (piece_at of row 8 q + 4 side + 2 e + (at & 1), which is piece at / 8 of the hi plane for one parity of q and of the lo
        // plane for the other)
        char* place[2][2];
#pragma unroll
        for (int odd = 0; odd < 2; ++odd)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            place[odd][e] = lds + c * kTile + (4 * side + (at & 1)) * kLine + ((at / 8 ^ (4 * odd + 2 * side + e)) << 4) + 2 * (at & 6);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              halfx2 hi, lo;
#pragma unroll
              for (int d = 0; d < 2; ++d) {
                const float v = x[s][i][4 * q + 2 * e + d];
                hi[d] = (_Float16)v;
                lo[d] = rest_of(v, hi[d]);
              }
              const int down = (32 * i + 8 * q + 2 * e) * kLine;
              *reinterpret_cast<uint32_t*>(place[q & 1][e] + down) = beside(hi, turn);
              *reinterpret_cast<uint32_t*>(place[~q & 1][e] + down) = beside(lo, turn);
            }
          __builtin_amdgcn_sched_barrier(0);                 // (so that no more values are under way than registers)
        }
      }
    }
    __syncthreads();
    fltx16 gram[TJ];                                       // (and P is made from these, not from their planes)
    if (squares) product(lds, columns, at, side, gram);
    if (!apart) __syncthreads();
    // A lane has, of tile (i, j), column j's `at` and four rows after four; G is symmetric: four neighbours of row `at`.
    if (squares) {
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        if (j0 + j < RT) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = gram[j][4 * q + e] *= 1.f / kScale;
            put_four(gl + i0 * kTile, 32 * (j0 + j) + at, q, side, v);
          }
        }
    }
    __syncthreads();
    if (squares) {
      fltx16 sum[TJ];
      product(gl, RT, at, side, sum);
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        if (j0 + j < RT) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(sum[j][4 * q + e], a.plane_c, a.plane_b * gram[j][4 * q + e]);
            // columns in the order in which a lane of x has its rows: 4 side ... of each eight
            put_four(pl + i0 * kTile, 32 * (j0 + j) + at, 2 * (q / 2) + side, q & 1, v);
          }
        }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (wave + kOneWaves * s >= columns) continue;
      // (X's planes are made once for its lines and once here: kept in between, both are more than the registers hold)
      if constexpr (RT == 4) {
#pragma unroll
        for (int i = 0; i < RT; ++i) asm volatile("" : "+v"(x[s][i]));
      }
      fltx16 next[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) next[i][v] = 0.f;
#pragma unroll
      for (int c = 0; c < RT; ++c)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          halfx8 hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            hi[e] = (_Float16)x[s][c][8 * g + e];
            lo[e] = rest_of(x[s][c][8 * g + e], hi[e]);
          }
          const intx4 fb[2] = {__builtin_bit_cast(intx4, hi), __builtin_bit_cast(intx4, lo)};
          intx4 fa[RT][2];
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              fa[i][p] = *reinterpret_cast<const intx4*>(pl + c * kTile + piece_at(32 * i + at, 4 * p + 2 * g + side));
#pragma unroll
          for (int m = 0; m < SplitOp::kTerms; ++m)
#pragma unroll
            for (int i = 0; i < RT; ++i) SplitOp::mma(next[i], m, fa[i], fb);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) x[s][i][v] = __builtin_fmaf(next[i][v], a.back, a.a * x[s][i][v]);
    }
    __syncthreads();
  }
  store_strips<RT, S>(a, z, 1.f / kScale, x);
}

// Whether a workgroup takes a matrix; and takes them.
bool one_workgroup(const Shape& m) {
  const int64_t rt = ceil_div(m.r, 32), s = ceil_div(ceil_div(m.l, 32), kOneWaves);
  return (rt <= 2 && s <= 2) || (rt <= 4 && s == 1);
}

template <int RT, int S>
void launch_one(const MuonArgs& a, int64_t n, int steps, hipStream_t st) {
  muon_one_kernel<RT, S><<<(unsigned)n, kOneWaves * kWave, 0, st>>>(a, steps);
}

bool one_launch(const MuonArgs& a, int64_t n, int steps, hipStream_t st) {
  const int64_t rt = ceil_div(a.s.r, 32), s = ceil_div(ceil_div(a.s.l, 32), kOneWaves);
  const unsigned grid = (unsigned)n, block = kOneWaves * kWave;
  if (rt == 1 && s == 1) muon_narrow_kernel<1><<<grid, block, 0, st>>>(a, steps);
  else if (rt == 1 && s == 2) muon_narrow_kernel<2><<<grid, block, 0, st>>>(a, steps);
  else if (rt == 2 && s == 1) launch_one<2, 1>(a, n, steps, st);
  else if (rt == 2 && s == 2) launch_one<2, 2>(a, n, steps, st);
  else if (rt == 3 && s == 1) launch_one<3, 1>(a, n, steps, st);
  else if (rt == 4 && s == 1) launch_one<4, 1>(a, n, steps, st);
  else return false;
  return true;
}

Shape shape_of(int64_t rows, int64_t cols) {
  const int turned = rows > cols;
  return Shape{rows, cols, turned ? cols : rows, turned ? rows : cols, turned};
}

int64_t parts_of(int64_t rows, int64_t cols) {
  const int64_t n = ceil_div(rows * cols, 4096);
  return n < 1024 ? n : 1024;
}

int64_t whole(int64_t bytes) { return ceil_div(bytes, 256) * 256; }

// Matrices that go through a set of launches together: enough for the chip's workgroups twice, so that the planes of
// those under way are not more than that takes.
int64_t group_of(int64_t count, int64_t rows, int64_t cols) {
  const int64_t tiles = ceil_div(rows, 64) * ceil_div(cols, 64), want = one_workgroup(shape_of(rows, cols)) ? kGroup : ceil_div(2048, tiles);
  const int64_t most = want < kGroup ? want : kGroup;
  return count < most ? count : most;
}

int64_t workspace_of(int64_t count, int64_t rows, int64_t cols) {
  const Shape s = shape_of(rows, cols);
  if (one_workgroup(s)) return 0;
  const int64_t n = group_of(count, rows, cols);
  return whole(n * parts_of(rows, cols) * 8) + whole(n * s.r * s.long_line()) + 2 * whole(n * s.l * s.short_line()) +
         2 * whole(n * s.r * s.short_line()) + (int64_t)num_cus() * 4096 * 4;
}

// most_p: what P's eigenvalues stay below.
int check_muon(const char* what, int64_t count, int64_t rows, int64_t cols, int steps, const float* coefficients, double& most_p) {
  F2CGT_REQUIRE(count >= 0 && rows >= 0 && cols >= 0, F2CGT_E_INVALID, "%s: sizes must not be negative", what);
  F2CGT_REQUIRE(rows <= 65536 && cols <= 65536, F2CGT_E_UNSUPPORTED, "%s: at most 65536 rows and columns", what);
  F2CGT_REQUIRE(steps >= 1 && steps <= 100, F2CGT_E_INVALID, "%s: from one to 100 steps", what);
  F2CGT_REQUIRE(coefficients != nullptr, F2CGT_E_INVALID, "%s: null coefficients", what);
  // How far singular values from [0, reach] get in a step, and what they are multiplied with: p(t) = a + b t + c t^2 of their
  // squares, and x p(x^2), at the ends and where a derivative is zero.
  const double a = coefficients[0], b = coefficients[1], c = coefficients[2];
  double reach = 1.;
  most_p = 0.;
  for (int s = 0; s < steps; ++s) {
    const double end = 1.002 * reach * reach, root = 9. * b * b - 20. * a * c;
    // the derivative a + 3 b t + 5 c t^2 of x p(x^2) is zero at q / 5 c and a / q: no difference of near numbers, whatever c is
    const double q = -0.5 * (3. * b + copysign(sqrt(root), b));
    const double at[5] = {0., end, c != 0. ? -b / (2. * c) : 0., root >= 0. && c != 0. ? q / (5. * c) : 0., root >= 0. && q != 0. ? a / q : 0.};
    double next = 0.;
    for (double t : at) {
      if (!(t >= 0. && t <= end) && t == t) continue;
      const double p = a + b * t + c * t * t, x = sqrt(t) * fabs(p);
      F2CGT_REQUIRE(p > -kMost && p < kMost && x < 2.5, F2CGT_E_UNSUPPORTED, "%s: these coefficients lead out of the range of the products", what);
      next = x > next ? x : next;
      most_p = fabs(p - a) > most_p ? fabs(p - a) : most_p;
    }
    reach = next;
  }
  return 0;
}

// Whether what a step writes shares no memory with anything else of its lists (of dense matrices of `values`).
int check_apart(const char* what, void* const* weights, int weight_size, const void* const* grads, int grad_size, float* const* momenta,
                int64_t count, int64_t values) {
  struct Range { uintptr_t from, end; bool written; };
  std::unique_ptr<Range[]> all(new (std::nothrow) Range[3 * count]);
  F2CGT_REQUIRE(all != nullptr, F2CGT_E_INVALID, "%s: out of host memory", what);
  auto put = [&](int64_t i, const void* p, int size, bool written) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(p);
    all[i] = Range{from, from + (uintptr_t)(values * size), written};
  };
  for (int64_t i = 0; i < count; ++i) {
    put(3 * i, weights[i], weight_size, true);
    put(3 * i + 1, grads[i], grad_size, false);
    put(3 * i + 2, momenta[i], 4, true);
  }
  std::sort(all.get(), all.get() + 3 * count, [](const Range& x, const Range& y) { return x.from < y.from; });
  uintptr_t end = 0, written_end = 0;                      // of those before
  for (int64_t i = 0; i < 3 * count; ++i) {
    const Range& r = all[i];
    F2CGT_REQUIRE(r.from >= (r.written ? end : written_end), F2CGT_E_INVALID, "%s: a weight or a momentum shares memory with another matrix", what);
    end = std::max(end, r.end);
    if (r.written) written_end = std::max(written_end, r.end);
  }
  return 0;
}

int run_muon(const char* what, MuonArgs a, int64_t count, int64_t rows, int64_t cols, int steps, const float* coefficients,
             double most_p, void* const* out, const void* const* u, float* const* held, int64_t u_step, void* workspace, hipStream_t st) {
  a.s = shape_of(rows, cols);
  const Shape& s = a.s;
  a.parts = (int)parts_of(rows, cols);
  a.a = coefficients[0]; a.b = coefficients[1]; a.c = coefficients[2];
  const float fit = most_p < kMost ? 1.f : 0.5f;           // (a and a + b t + c t^2 are below kMost: most_p is below twice that)
  a.plane_b = a.b * fit; a.plane_c = a.c * fit * (1.f / kScale); a.back = 1.f / (kScale * fit);
  const int64_t group = group_of(count, rows, cols);
  char* at = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) { char* p = at; at = p != nullptr ? p + whole(bytes) : p; return p; };
  a.partial = reinterpret_cast<double*>(take(group * a.parts * 8));
  a.x = take(group * s.r * s.long_line());
  a.xt[0] = take(group * s.l * s.short_line());
  a.xt[1] = take(group * s.l * s.short_line());
  a.g = take(group * s.r * s.short_line());
  a.p = take(group * s.r * s.short_line());
  a.sums = reinterpret_cast<float*>(take((int64_t)num_cus() * 4096 * 4));
  for (int64_t first = 0; first < count; first += group) {
    const int64_t n = count - first < group ? count - first : group;
    a.whole = cols % 4 == 0;
    for (int64_t i = 0; i < n; ++i) {
      a.at.u[i] = u_step ? static_cast<const char*>(u[0]) + (first + i) * u_step * type_size(a.u_dtype) : u[first + i];
      a.at.out[i] = u_step ? static_cast<char*>(out[0]) + (first + i) * u_step * type_size(a.out_dtype) : out[first + i];
      a.at.held[i] = held != nullptr ? held[first + i] : nullptr;
      a.whole = a.whole && aligned(a.at.out[i], 4 * type_size(a.out_dtype));
    }
    if (one_launch(a, n, steps, st)) {
      if (int rc = launch_status(what)) return rc;
      continue;
    }
    const int splits = gram_splits(n, s);
    const dim3 parts((unsigned)a.parts, (unsigned)n);
    if (held != nullptr) muon_norm_kernel<true><<<parts, 256, 0, st>>>(a);
    else muon_norm_kernel<false><<<parts, 256, 0, st>>>(a);
    muon_split_kernel<<<dim3((unsigned)ceil_div(rows, 64), (unsigned)ceil_div(cols, 64), (unsigned)n), 256, 0, st>>>(a);
    for (int step = 0; step < steps; ++step) {
      if (splits > 1) {
        const unsigned tiles = (unsigned)(n * ceil_div(s.r, 64) * (ceil_div(s.r, 64) + 1) / 2);
        muon_gram_part_kernel<<<tiles * splits, 1024, 0, st>>>(a, splits);
        muon_gram_add_kernel<<<tiles, 256, 0, st>>>(a, splits);
      } else {
        symmetric(a, n, false, st);
      }
      symmetric(a, n, true, st);
      update(a, n, step & 1, step == steps - 1, st);
    }
    if (int rc = launch_status(what)) return rc;
  }
  return 0;
}

}  // namespace
}  // namespace f2cgt

using namespace f2cgt;

extern "C" int64_t f2cgt_muon_workspace_bytes(int64_t count, int64_t rows, int64_t cols) {
  if (count <= 0 || rows <= 0 || cols <= 0 || rows > 65536 || cols > 65536) return 0;
  return workspace_of(count, rows, cols);
}

extern "C" int f2cgt_orthogonalize(const void* update, int dtype, void* out, int64_t count, int64_t rows, int64_t cols, int steps,
                                   const float* coefficients, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "orthogonalize";
  double most_p;
  if (int rc = check_muon(what, count, rows, cols, steps, coefficients, most_p)) return rc;
  F2CGT_REQUIRE(dense_type(dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 only", what);
  if (count == 0 || rows == 0 || cols == 0) return 0;
  F2CGT_REQUIRE(update && out && aligned(update, type_size(dtype)) && aligned(out, type_size(dtype)), F2CGT_E_INVALID,
                "%s: null or misaligned buffer", what);
  const int64_t bytes = workspace_of(count, rows, cols);
  F2CGT_REQUIRE(bytes == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= bytes), F2CGT_E_INVALID,
                "%s: workspace too small or misaligned", what);
  MuonArgs a{};
  a.u_dtype = a.out_dtype = dtype;
  a.keep = 0.f;
  void* outs[1] = {out};
  const void* ins[1] = {update};
  return run_muon(what, a, count, rows, cols, steps, coefficients, most_p, outs, ins, nullptr, rows * cols, workspace, as_stream(stream));
}

extern "C" int f2cgt_muon_step(void* const* weights, int weight_dtype, const void* const* grads, int grad_dtype, float* const* momenta,
                               int64_t count, int64_t rows, int64_t cols, float step_size, float decay, float momentum, int nesterov,
                               int steps, const float* coefficients, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "muon_step";
  double most_p;
  if (int rc = check_muon(what, count, rows, cols, steps, coefficients, most_p)) return rc;
  F2CGT_REQUIRE(dense_type(weight_dtype) && dense_type(grad_dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 only", what);
  if (count == 0 || rows == 0 || cols == 0) return 0;
  F2CGT_REQUIRE(weights && grads && momenta, F2CGT_E_INVALID, "%s: null list", what);
  for (int64_t i = 0; i < count; ++i)
    F2CGT_REQUIRE(weights[i] && grads[i] && momenta[i] && aligned(weights[i], type_size(weight_dtype)) &&
                      aligned(grads[i], type_size(grad_dtype)) && aligned(momenta[i], 4),
                  F2CGT_E_INVALID, "%s: null or misaligned buffer", what);
  if (int rc = check_apart(what, weights, type_size(weight_dtype), grads, type_size(grad_dtype), momenta, count, rows * cols)) return rc;
  const int64_t bytes = workspace_of(count, rows, cols);
  F2CGT_REQUIRE(bytes == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= bytes), F2CGT_E_INVALID,
                "%s: workspace too small or misaligned", what);
  MuonArgs a{};
  a.u_dtype = grad_dtype;
  a.out_dtype = weight_dtype;
  a.nesterov = nesterov;
  a.momentum = momentum;
  a.keep = 1.f - decay;
  a.size = step_size;
  F2CGT_REQUIRE(a.keep > 0.f && a.keep <= 1.f && momentum >= 0.f && momentum < 1.f, F2CGT_E_INVALID,
                "%s: decay must be in [0, 1), momentum too", what);
  return run_muon(what, a, count, rows, cols, steps, coefficients, most_p, weights, grads, momenta, 0, workspace, as_stream(stream));
}
