// Activations kept in 8 bits between the forward and the backward pass, and the products that are made with them.
//
// pack:   groups of 32 columns of a row, one exponent E a group, code = rint(x 2^(127 - E))      (the choice of E: rows.hpp)
// unpack: code 2^(E - 127)
// grad:   dW = g^T v, db = sum of g's rows, for a layer out = v W^T + b whose input v is held as codes
//
// Pack and unpack are bound by memory: 250 000 x 100 in fp32 31 to 33 us (126 MB, 4 TB/s) and 20.5 (6.1 TB/s), 262 144 x 128 5.8 TB/s
// either way, in 16 bits 4.8 and 6.1.  The product goes through bf16 matrix instructions: every v is a bf16 exactly, and g is one bf16
// plane (bf16), two (fp16: 11 bits in 8 + 8) or three (fp32: 24 bits in 8 + 8 + 8, cut off one after the other, exactly but for bits
// below 2^-133, bf16's least number), so all products are exact and only the fp32 sums round.  Large ones are bound by the matrix instructions at the card's power cap (16 384 x
// 4096 -> 4096 in bf16 500 to 550 us, 1.0 to 1.1e15 operations a second, 56 % of the clocks in which the CUs have waves; a library's
// product of bf16 operands in this layout 558), long sums for few outputs by splitting into planes and placing them (60 001 x 602 ->
// 128 in fp32 41 us, of which its matrix instructions are 41 %), small ones by a launch and latency (1024 x 128 -> 256 6.8 us).
#include "rows.hpp"
#include "tile_product.hpp"

#include <type_traits>

namespace f2cgt {
namespace {

// ---- into checkpoints and back -----------------------------------------------------------------------
struct PackArgs {
  const void* x;
  void* out;
  int8_t* codes;
  uint8_t* exponents;
  int64_t m, ld, code_stride;
  int k, groups;
  uint32_t pieces;           // of a row, those of whole groups
};

constexpr int kPackUnroll = 4;

// Piece `at` of the matrix as (row, first column): one 64-bit division for a workgroup, 32 bits from there.
struct PieceOf {
  int64_t row0;
  uint32_t over, pieces;
  int v;
  __device__ __forceinline__ PieceOf(uint32_t pieces_, int v_, int per_block) : pieces(pieces_), v(v_) {
    const int64_t first = (int64_t)blockIdx.x * per_block;
    row0 = first / pieces;
    over = (uint32_t)(first - row0 * pieces);
  }
  __device__ __forceinline__ void operator()(uint32_t i, int64_t& row, int& column) const {
    const uint32_t p = over + i, r = p / pieces;
    row = row0 + r;
    column = (int)(p - r * pieces) * v;
  }
};

template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
  constexpr int V = kPieceOf<T>, kShare = kCheckpointGroup / V;
  const PieceOf place(a.pieces, V, 256 * kPackUnroll);
  float v[kPackUnroll][V];
  int64_t row[kPackUnroll];
  int column[kPackUnroll];
#pragma unroll
  for (int u = 0; u < kPackUnroll; ++u) {
    place(u * 256 + threadIdx.x, row[u], column[u]);
    if (row[u] >= a.m) column[u] = a.k;                       // (nothing of it)
    const T* x = static_cast<const T*>(a.x) + row[u] * a.ld + column[u];
    if (column[u] + V <= a.k) {
      load_piece<T, V>(x, v[u]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[u][e] = 0.f;
        if (column[u] + e < a.k) v[u][e] = (float)x[e];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kPackUnroll; ++u) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t size = __float_as_uint(v[u][e]) & 0x7FFFFFFFu;
      most = size > most ? size : most;
    }
    const uint32_t exponent = exponent_of(most_lanes<kShare>(most));
    if (column[u] >= a.k) continue;
    uint32_t packed[V / 4] = {};
#pragma unroll
    for (int e = 0; e < V; ++e) packed[e / 4] |= (uint32_t)(code_of(v[u][e], exponent) & 255) << (8 * (e % 4));
    int8_t* codes = a.codes + row[u] * a.code_stride + column[u];
    if (column[u] + V <= a.k) {
      if constexpr (V == 8) *reinterpret_cast<uint2*>(codes) = uint2{packed[0], packed[1]};
      else *reinterpret_cast<uint32_t*>(codes) = packed[0];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (column[u] + e < a.k) codes[e] = (int8_t)(packed[e / 4] >> (8 * (e % 4)));
    }
    if (threadIdx.x % kShare == 0) a.exponents[row[u] * a.groups + column[u] / kCheckpointGroup] = (uint8_t)exponent;
  }
}

// (fp16 ends below what a step of fp16's largest values reaches: such a value becomes the largest one.)
template <typename T>
__device__ __forceinline__ float within(float v) {
  if constexpr (sizeof(T) == 2 && dtype_of<T>::tag == F2CGT_DT_F16) return v != v ? v : fminf(fmaxf(v, -65504.f), 65504.f);
  else return v;
}

template <typename T>
__global__ __launch_bounds__(256) void unpack_kernel(PackArgs a) {
  constexpr int V = kPieceOf<T>;
  const PieceOf place(a.pieces, V, 256 * kPackUnroll);
  uint32_t words[kPackUnroll][V / 4];
  float step[kPackUnroll];
  int64_t row[kPackUnroll];
  int column[kPackUnroll];
#pragma unroll
  for (int u = 0; u < kPackUnroll; ++u) {
    place(u * 256 + threadIdx.x, row[u], column[u]);
    if (row[u] >= a.m) column[u] = a.k;
    step[u] = 0.f;
#pragma unroll
    for (int e = 0; e < V / 4; ++e) words[u][e] = 0;
    if (column[u] < a.k) {                                    // (a row's codes are readable in whole pieces)
      const int8_t* codes = a.codes + row[u] * a.code_stride + column[u];
#pragma unroll
      for (int e = 0; e < V / 4; ++e) words[u][e] = reinterpret_cast<const uint32_t*>(codes)[e];
      step[u] = step_of(a.exponents[row[u] * a.groups + column[u] / kCheckpointGroup]);
    }
  }
#pragma unroll
  for (int u = 0; u < kPackUnroll; ++u) {
    if (column[u] >= a.k) continue;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = within<T>(coded_value(words[u][e / 4], e % 4, step[u]));
    T* out = static_cast<T*>(a.out) + row[u] * a.k + column[u];
    if (column[u] + V <= a.k) {
      store_piece<T, V>(out, v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (column[u] + e < a.k) out[e] = (T)v[e];
    }
  }
}

// ---- the weight's gradient -----------------------------------------------------------------------------
typedef __bf16 bfx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));

struct GradArgs {
  const void* grad;          // [m, n], rows ld apart
  const int8_t* codes;       // [m, k]
  const uint8_t* exponents;  // [m, groups]
  float* parts;              // [splits][n][k], then [splits][n] of the bias; or null: one split, straight to `out` and `bias`
  void* out;
  void* bias;                // or null
  int64_t m, ld, code_stride;
  int n, k, groups, out_tag;
  int64_t steps;             // of rows, in all
  uint32_t splits, tiles_n, tiles_k;
};

template <typename T> constexpr int kPlanes = dtype_of<T>::tag == F2CGT_DT_F32 ? 3 : dtype_of<T>::tag == F2CGT_DT_F16 ? 2 : 1;

// Eight numbers of T, as memory holds them.
template <typename T> struct Eight {
  static constexpr int kWords = 2 * (int)sizeof(T);
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const char* p) {
    typedef typename piece_words<T, kPieceOf<T>>::type words;
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const words v = reinterpret_cast<const words*>(p)[i / 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[i + e] = v[e];
    }
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    else if constexpr (dtype_of<T>::tag == F2CGT_DT_BF16) return __uint_as_float(e % 2 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e / 2] >> 16 * (e % 2)));
  }
  __device__ __forceinline__ void set(int e, T v) {
    if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(v);
    else w[e / 2] = e % 2 ? w[e / 2] | (uint32_t)__builtin_bit_cast(uint16_t, v) << 16 : (uint32_t)__builtin_bit_cast(uint16_t, v);
  }
  // As bf16 planes, whose sum the numbers are.  Each plane is the upper half of what is left: no rounding, 8 bits each.  (An infinity
  // leaves a NaN.)
  __device__ __forceinline__ void planes(intx4 (&p)[kPlanes<T>]) const {
    if constexpr (kPlanes<T> == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) p[0][e] = (int)w[e];
    } else {
      float left[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) left[e] = (*this)[e];
#pragma unroll
      for (int i = 0; i < kPlanes<T>; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p[i][e] = (int)__builtin_amdgcn_perm(__float_as_uint(left[2 * e + 1]), __float_as_uint(left[2 * e]), 0x07060302);
        if (i + 1 < kPlanes<T>)
#pragma unroll
          for (int e = 0; e < 8; ++e) left[e] -= __uint_as_float(__float_as_uint(left[e]) & 0xFFFF0000u);
      }
    }
  }
};

typedef uint32_t word_any __attribute__((aligned(1)));

// A tile of dW: BN outputs by BK inputs, WN x WK to a wave, BM rows of g and v a step; GROUPS groups of waves take the steps in turn
// and add their sums in the end (two groups on 128 squared, for eight waves on a CU).  Rows lie in LDS as they do in memory, one line
// of BN or BK bf16 a row, and matrix operands, which hold eight rows of one column a lane, are read through the transposing LDS loads:
// sixteen lanes give the addresses of 4 rows x 16 columns in four pieces a row, and get a column each.  Units of 64 bytes of a line
// change places by the row's last two bits, so the four rows of such a read lie in different banks.
template <typename T, int BN, int BK, int WN, int WK, int BM, int GROUPS>
struct GradTile {
  static constexpr int P = kPlanes<T>;
  static constexpr int kThreads = (BN / WN) * (BK / WK) * kWave, kBlock = kThreads * GROUPS;
  static constexpr int TI = WN / 32, TJ = WK / 32;
  static constexpr int kLineG = BN * 2, kLineX = BK * 2;               // bytes
  static constexpr int kPlaneG = BM * kLineG;
  static constexpr int kStage = P * kPlaneG + BM * kLineX;
  static constexpr int kPiecesG = BM * BN / 8 / kThreads, kPiecesX = BM * BK / 8 / kThreads;      // of a thread
  static_assert(kPiecesG * kThreads * 8 == BM * BN && kPiecesX * kThreads * 8 == BM * BK, "whole pieces per thread");
  static_assert(kThreads % (BN / 8) == 0 && kThreads % (BK / 8) == 0, "a thread's pieces are of the same columns");
  static constexpr int kRowsG = kThreads / (BN / 8), kRowsX = kThreads / (BK / 8);                // rows between a thread's pieces
  static constexpr int kParts = BM / 16;
  static_assert(kPiecesG % kParts == 0 || kPiecesG < kParts, "pieces in turn with products");

  // (64 banks hold one line of 256 bytes or half of a longer one, and two lines of 128)
  static __device__ __forceinline__ int line_at(int row, int byte, int line) {
    return row * line + (byte ^ (line == 128 ? (row >> 1 & 1) << 6 : (row & 3) << 6));
  }
  struct Held {
    Eight<T> g[kPiecesG];
    uint2 x[kPiecesX];
    uint32_t e[kPiecesX];      // exponents, each the lowest byte of four
  };
};

template <typename T, int BN, int BK, int WN, int WK, int BM, int GROUPS>
__global__ __launch_bounds__((BN / WN) * (BK / WK) * kWave * GROUPS) void packed_linear_grad_kernel(GradArgs a) {
  typedef GradTile<T, BN, BK, WN, WK, BM, GROUPS> Tile;
  constexpr int P = Tile::P, TI = Tile::TI, TJ = Tile::TJ, kThreads = Tile::kThreads;
  constexpr int kLd = WK + 1, kStrips = 32 * kLd * 4 * (kThreads / kWave) * GROUPS;      // a strip of sums for each wave on its way out
  constexpr int kStages = 2 * Tile::kStage * GROUPS, kLds = kStages > kStrips ? kStages : kStrips;
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  const int group = GROUPS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads) : 0;
  const int t = threadIdx.x - group * kThreads, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int wi = (wave % (BN / WN)) * WN, wj = (wave / (BN / WN)) * WK;
  char* stages = lds + group * 2 * Tile::kStage;
  // neighbours in time share rows: all tiles of a split are one XCD's
  const uint32_t tiles = a.tiles_n * a.tiles_k, place = place_of(blockIdx.x, tiles * a.splits);
  const uint32_t split = place / tiles;
  uint32_t ti, tj;
  tile_of(place - split * tiles, a.tiles_n, a.tiles_k, 4, ti, tj);
  const int col_n = (int)ti * BN, col_k = (int)tj * BK;
  // (whole rounds to every split but the last)
  const int64_t shares = (a.steps + GROUPS - 1) / GROUPS, from = shares * split / a.splits * GROUPS;
  const int64_t ahead = shares * (split + 1) / a.splits * GROUPS, to = ahead < a.steps ? ahead : a.steps;

  // this thread's columns: those beyond the operand's end repeat its first ones (what they give is not kept)
  const int pg = t % (BN / 8) * 8, px = t % (BK / 8) * 8, rg = t / (BN / 8), rx = t / (BK / 8);
  const int cg = col_n + pg < a.n ? col_n + pg : 0, cx = col_k + px < a.k ? col_k + px : 0;
  // (32 bits from a step's first row: strides are below 2^24)
  const uint32_t off_g = (uint32_t)(rg * (int)a.ld + cg) * (uint32_t)sizeof(T), off_x = (uint32_t)(rx * (int)a.code_stride + cx);
  const uint32_t off_e = (uint32_t)(rx * a.groups + cx / kCheckpointGroup);
  typedef typename Tile::Held Held;

  // A piece that runs over its row's end reads on in the next one, and four exponents at a time, of which the first counts, in the next
  // ones: the steps of the last four rows are not among these, and with fewer than eight outputs, whose pieces run over more rows, no step
  // is (250 000 x 128 -> 1 to 7 in fp32 32 us, -> 8 26; in bf16 27 and 19).  (Of a single exponent's byte the compiler makes a word where
  // the loop ends, behind a wait.)
  const int64_t whole = a.n >= 8 && a.m > 4 ? (a.m - 4) / BM : 0;
  const int64_t rounds = (whole < to ? (whole > from ? whole - from : 0) : to - from) / GROUPS, end = from + rounds * GROUPS;
  // Pieces of one of kParts parts of a step into registers.
  auto load_part = [&](Held& h, int64_t step, int part) {
    const int64_t row0 = step * BM;
    const char* grad = static_cast<const char*>(a.grad) + row0 * a.ld * (int64_t)sizeof(T);
    const int8_t* codes = a.codes + row0 * a.code_stride;
    const uint8_t* exponents = a.exponents + row0 * a.groups;
    uint32_t og = off_g, ox = off_x, oe = off_e;
    asm("" : "+v"(og), "+v"(ox), "+v"(oe));       // (32 bits beside a scalar base, which the compiler would widen ahead of the loop)
#pragma unroll
    for (int i = 0; i < Tile::kPiecesG; ++i)
      if (i % Tile::kParts == part) h.g[i].load(grad + (int64_t)i * Tile::kRowsG * a.ld * (int64_t)sizeof(T) + og);
#pragma unroll
    for (int i = 0; i < Tile::kPiecesX; ++i) {
      if (i % Tile::kParts != part) continue;
      h.x[i] = *reinterpret_cast<const uint2*>(codes + i * Tile::kRowsX * a.code_stride + ox);
      h.e[i] = *reinterpret_cast<const word_any*>(exponents + (int64_t)i * Tile::kRowsX * a.groups + oe);
    }
  };
  const bool sums = a.bias != nullptr && tj == 0;
  float db[8] = {};
  auto place_g = [&](auto with_sums, const Eight<T>& g, char* stage, int row, bool count) {
    if constexpr (decltype(with_sums)::value)
#pragma unroll
      for (int e = 0; e < 8; ++e) db[e] += count ? g[e] : 0.f;
    intx4 planes[P];
    g.planes(planes);
#pragma unroll
    for (int p = 0; p < P; ++p)
      *reinterpret_cast<intx4*>(stage + p * Tile::kPlaneG + Tile::line_at(row, pg * 2, Tile::kLineG)) = planes[p];
  };
  auto place_x = [&](const uint2& x, uint32_t exponent, char* stage, int row) {
    const float step = __uint_as_float(exponent << 24 >> 1);
    intx4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t word = e < 2 ? x.x : x.y;
      v[e] = (int)__builtin_amdgcn_perm(__float_as_uint(coded_value(word, 2 * (e % 2) + 1, step)),
                                        __float_as_uint(coded_value(word, 2 * (e % 2), step)), 0x07060302);
    }
    *reinterpret_cast<intx4*>(stage + P * Tile::kPlaneG + Tile::line_at(row, px * 2, Tile::kLineX)) = v;
  };
  // What load_part loaded into a stage.
  auto place_part = [&](auto with_sums, const Held& h, char* stage, int part, bool count) {
#pragma unroll
    for (int i = 0; i < Tile::kPiecesG; ++i)
      if (i % Tile::kParts == part) place_g(with_sums, h.g[i], stage, rg + i * Tile::kRowsG, count);
#pragma unroll
    for (int i = 0; i < Tile::kPiecesX; ++i)
      if (i % Tile::kParts == part) place_x(h.x[i], h.e[i], stage, rx + i * Tile::kRowsX);
  };
  // The matrix's last rows, value by value, at places that exist, into a stage; what is not theirs is made zero.
  auto place_last = [&](auto with_sums, int64_t step, char* stage) {
    const int64_t row0 = step * BM;
    constexpr int kAtOnce = BN > 128 ? 1 : 4;      // (large tiles have no registers for more)
#pragma unroll kAtOnce
    for (int i = 0; i < Tile::kPiecesX; ++i) {
      const int64_t row = row0 + rx + i * Tile::kRowsX, held_row = row < a.m ? row : a.m - 1;
      uint2 x = *reinterpret_cast<const uint2*>(a.codes + held_row * a.code_stride + cx);
      const uint32_t exponent = a.exponents[held_row * a.groups + cx / kCheckpointGroup];
      if (row >= a.m) x = uint2{0, 0};
      place_x(x, row < a.m ? exponent : 127, stage, rx + i * Tile::kRowsX);
    }
#pragma unroll kAtOnce
    for (int i = 0; i < Tile::kPiecesG; ++i) {
      const int64_t row = row0 + rg + i * Tile::kRowsG;
      const T* p = static_cast<const T*>(a.grad) + (row < a.m ? row : a.m - 1) * a.ld;
      T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p[cg + e < a.n ? cg + e : a.n - 1];
      Eight<T> g;
#pragma unroll
      for (int e = 0; e < 8; ++e) g.set(e, row < a.m && cg + e < a.n ? v[e] : (T)0.f);
      place_g(with_sums, g, stage, rg + i * Tile::kRowsG, true);
    }
  };

  fltx16 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  // A lane's part of an operand: eight rows of column lane % 32, the rows 8 (lane / 32) on of a group of sixteen.
  const int tr_row = (lane >> 5) * 8 + (lane >> 2 & 3), tr_byte = ((lane >> 4 & 1) * 16 + (lane & 3) * 4) * 2;
  auto operand = [&](const char* plane, int part, int column, int line) {
    shortx4 half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) shortx4*)(plane + Tile::line_at(part * 16 + tr_row + 4 * h, column * 2 + tr_byte, line)));
    const shortx8 both = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bfx8, both);
  };
  // Operands of a part of a stage; those of the next part are read while one is multiplied.
  bfx8 fx[2][TJ], fg[2][P][TI];
  auto read_part = [&](const char* stage, int s) {
#pragma unroll
    for (int j = 0; j < TJ; ++j) fx[s & 1][j] = operand(stage + P * Tile::kPlaneG, s, wj + 32 * j, Tile::kLineX);
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
#pragma unroll
      for (int i = 0; i < TI; ++i) fg[s & 1][p][i] = operand(stage + p * Tile::kPlaneG, s, wi + 32 * i, Tile::kLineG);
  };
  auto multiply_part = [&](int s) {
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fg[s & 1][p][i], fx[s & 1][j], acc[i][j], 0, 0, 0);
  };
  // A group's step s is multiplied out of stage s % 2 while its next one goes from registers into the other stage, a part at a time, and the
  // registers of each part take the step after that: its loads have a whole round for their way.  (One copy of the round, and no branch in
  // it: what a short call waits for is the kernel's code, and where paths meet the compiler would wait for every load.)
  auto go = [&](auto with_sums) {
    auto held_step = [&](int64_t step) { return step < end ? step : from; };       // (behind the last one: the first one again)
    if (rounds > 0) {
      Held h;
#pragma unroll
      for (int part = 0; part < Tile::kParts; ++part) load_part(h, from + group, part);
#pragma unroll
      for (int part = 0; part < Tile::kParts; ++part) {
        place_part(with_sums, h, stages, part, true);
        load_part(h, held_step(from + group + GROUPS), part);
      }
      __syncthreads();
      int turn = 0;
      for (int64_t step = from + group; step < end; step += GROUPS, turn ^= 1) {
        const char* now = stages + turn * Tile::kStage;
        char* next = stages + (turn ^ 1) * Tile::kStage;
        const int64_t after = held_step(step + 2 * GROUPS);
        read_part(now, 0);
#pragma unroll
        for (int part = 0; part < Tile::kParts; ++part) {
          if (part + 1 < Tile::kParts) read_part(now, part + 1);
          multiply_part(part);
          place_part(with_sums, h, next, part, step + GROUPS < end);
          load_part(h, after, part);
        }
        __syncthreads();
      }
    }
    for (int64_t at = end; at < to; at += GROUPS) {          // what is left of the steps: a few, or all with fewer than eight outputs
      const int64_t step = at + group;
      if (step < to) place_last(with_sums, step, stages);
      __syncthreads();
      if (step < to)
#pragma unroll
        for (int part = 0; part < Tile::kParts; ++part) {
          read_part(stages, part);
          multiply_part(part);
        }
      __syncthreads();
    }
  };
  if (sums) go(std::true_type{});
  else go(std::false_type{});

  // Sums out, 32 rows of each wave's tile at a time by way of LDS, where the groups' sums are added in their order; a row of WK columns to a
  // store.  (A lane holds, of column lane % 32, rows 4 (lane / 32) to + 3 after every eight.)
  constexpr int kWaves = kThreads / kWave, kStrip = 32 * kLd;
  float* strips = reinterpret_cast<float*>(lds);
  float* strip = strips + (group * kWaves + wave) * kStrip;
#pragma unroll
  for (int i = 0; i < TI; ++i) {
    if (GROUPS > 1 && i > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) strip[(8 * (v / 4) + 4 * (lane >> 5) + v % 4) * kLd + 32 * j + (lane & 31)] = acc[i][j][v];
    if (GROUPS > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    // (each group stores a share of the strip's rows)
    const int row0 = col_n + wi + 32 * i, column0 = col_k + wj;
    const int rows = a.n - row0 < 32 ? a.n - row0 : 32;
    constexpr int kWide = WK < kWave ? WK : kWave, kAtOnce = kWave / kWide;       // columns and rows to a pass of the lanes
    for (int r = group * kAtOnce + lane / kWide; r < rows; r += GROUPS * kAtOnce)
#pragma unroll
      for (int c = lane % kWide; c < WK; c += kWide)
        if (column0 + c < a.k) {
          float sum = strips[wave * kStrip + r * kLd + c];
#pragma unroll
          for (int o = 1; o < GROUPS; ++o) sum += strips[(o * kWaves + wave) * kStrip + r * kLd + c];
          const int64_t at = (int64_t)(row0 + r) * a.k + column0 + c;
          if (a.parts != nullptr) a.parts[(int64_t)split * a.n * a.k + at] = sum;
          else store_value(a.out, a.out_tag, at, sum);
        }
    if (GROUPS == 1) __builtin_amdgcn_wave_barrier();
  }
  if (!sums) return;
  __syncthreads();
  constexpr int kRows = Tile::kRowsG * GROUPS;
  static_assert(kRows * BN * 4 <= kLds, "the bias' sums fit");
  float* room = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int e = 0; e < 8; ++e) room[(group * Tile::kRowsG + rg) * BN + pg + e] = db[e];
  __syncthreads();
  if (threadIdx.x < BN && col_n + (int)threadIdx.x < a.n) {
    float sum = 0.f;
    for (int r = 0; r < kRows; ++r) sum += room[r * BN + threadIdx.x];
    if (a.parts != nullptr) a.parts[(int64_t)a.splits * a.n * a.k + (int64_t)split * a.n + col_n + threadIdx.x] = sum;
    else store_value(a.bias, a.out_tag, col_n + threadIdx.x, sum);
  }
}

// Sums of a gradient's columns alone, of a layer without inputs: sixteen waves with every sixteenth row of 64 columns, a thousand rows of a
// wave to a part and the parts to a sum.  (One sum for all rows stands still at 2^24 equal values.)
struct ColumnArgs {
  const void* grad;
  void* bias;
  int64_t m, ld;
  int n, out_tag;
};
constexpr int kColumnWaves = 16, kColumnPart = 1024;
template <typename T>
__global__ __launch_bounds__(kColumnWaves * kWave) void column_sums_kernel(ColumnArgs a) {
  __shared__ float room[kColumnWaves][kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, column = blockIdx.x * kWave + lane;
  float sum = 0.f;
  if (column < a.n) {
    const T* from = static_cast<const T*>(a.grad) + column;
    for (int64_t row = wave; row < a.m;) {
      const int64_t left = (a.m - row + kColumnWaves - 1) / kColumnWaves;
      const int rows = left < kColumnPart ? (int)left : kColumnPart;
      float part = 0.f;
#pragma unroll 8
      for (int r = 0; r < rows; ++r, row += kColumnWaves) part += (float)from[row * a.ld];
      sum += part;
    }
  }
  room[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || column >= a.n) return;
#pragma unroll
  for (int w = 1; w < kColumnWaves; ++w) sum += room[w][lane];
  store_value(a.bias, a.out_tag, column, sum);
}

// Sums over the splits: SHARE waves have 64 E outputs, each of them every SHAREth split, then the waves' sums are added in order; the bias'
// in workgroups behind the weight's.  (No splits: zeros, of no rows.)
struct JoinArgs {
  const float* parts;
  void* out;
  void* bias;
  int64_t count;             // n k
  int n, tag;
  uint32_t splits, blocks;   // blocks: those of the weight
};
template <int WAVES, int SHARE, int E>
__global__ __launch_bounds__(WAVES * kWave) void join_splits_kernel(JoinArgs a) {
  constexpr int kOuts = 64 * E;
  __shared__ float room[SHARE > 1 ? WAVES : 1][kOuts];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, share = wave % SHARE;
  const bool weight = blockIdx.x < a.blocks;
  const int64_t count = weight ? a.count : a.n;
  const int64_t first = ((int64_t)(weight ? blockIdx.x : blockIdx.x - a.blocks) * (WAVES / SHARE) + wave / SHARE) * kOuts;
  const float* parts = (weight ? a.parts : a.parts + (int64_t)a.splits * a.count) + first;
  void* out = weight ? a.out : a.bias;
  const int64_t left = count - first;
  constexpr int kAtOnce = 16 / E;
  float sum[E] = {};
  for (uint32_t s = share; s < a.splits; s += kAtOnce * SHARE) {
    float v[kAtOnce][E];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[u][e] = 0.f;
        if (s + u * SHARE < a.splits && lane + 64 * e < left) v[u][e] = parts[(int64_t)(s + u * SHARE) * count + lane + 64 * e];
      }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) sum[e] += v[u][e];
  }
  if constexpr (SHARE > 1) {
    static_assert(WAVES == SHARE, "one set of outputs to a workgroup");
#pragma unroll
    for (int e = 0; e < E; ++e) room[wave][lane + 64 * e] = sum[e];
    __syncthreads();
    if (threadIdx.x >= kOuts || (int64_t)threadIdx.x >= left) return;
    float all = room[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < SHARE; ++w) all += room[w][threadIdx.x];
    store_value(out, a.tag, first + threadIdx.x, all);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 64 * e < left) store_value(out, a.tag, first + lane + 64 * e, sum[e]);
  }
}

constexpr int rows_of_step(int dtype, int size) {
  return size > 64 && dtype == F2CGT_DT_BF16 ? 64 : 32;
}

// How a product is cut: tiles of `size` squared, rows in `splits`.
struct Cut {
  int size;
  int64_t tiles, steps, splits;
};
// The shortest of the cuts that are tried, by times that were measured (us; planes of one, two and three): a launch with the begin and end
// of a tile of 64, 128 and 256 squared 2.5, 7 and 9; 32 rows of a tile of 64 squared 0.45, 0.55 and 0.65 where it is alone on its CU, 0.17,
// 0.20 and 0.275 for each of many, of 128 squared 0.43, 0.62 and 0.78, of 256 squared 0.95, 1.8 and 2.45, those alone on their CUs; splits'
// sums a launch more, 3.5, and 5 MB a us both ways.  What it decides, bf16 and fp32: 1000 x 1000 -> 1000 64 squared 18.5 and 24, 128 squared
// 22.8 and 25.1; 8192 x 2048 -> 2048 256 squared in four splits 94 and 187, 128 squared 120 and 207; 60 001 x 602 -> 128 128 squared 33.7 and
// 46.2, 64 squared 35.7 and 56.0; 30 000 x 64 -> 1024 64 squared in 48 or 64 splits 24.3 and 31.6, in 32 26.9 and 33.1, 128 squared 28.9 and
// 38.9.  (Fewer than eight outputs, whose steps are not on their way ahead, are cut by the same times.)
Cut cut_of(int dtype, int64_t m, int64_t n, int64_t k) {
  static constexpr float kAlone[3][3] = {{0.45f, 0.55f, 0.65f}, {0.43f, 0.62f, 0.78f}, {0.95f, 1.8f, 2.45f}};
  static constexpr float kShared[3] = {0.17f, 0.20f, 0.275f}, kBegin[3] = {2.5f, 7.f, 9.f};
  const int planes = dtype == F2CGT_DT_BF16 ? 0 : dtype == F2CGT_DT_F16 ? 1 : 2;
  const int64_t cus = num_cus();
  Cut best{};
  float least = 0.f;
  for (int i = 0; i < 3; ++i) {
    const int size = 64 << i;
    if (i == 2 && (n <= 128 || k <= 128)) continue;
    const int64_t tiles = ceil_div(n, size) * ceil_div(k, size), steps = ceil_div(m, rows_of_step(dtype, size));
    const float each = (float)rows_of_step(dtype, size) / 32;
    auto take = [&](int64_t splits) {
      if (splits < 1 || splits > steps || splits > 1024 || (splits > 1 && (splits * tiles > 8 * cus || splits * n * k > (1ll << 28)))) return;
      const int64_t rounds = ceil_div(tiles * splits, cus);
      float step = kAlone[i][planes] * (i == 0 ? 1.f : (float)rounds);
      if (i == 0 && kShared[planes] * (float)rounds > step) step = kShared[planes] * (float)rounds;
      float time = kBegin[i] + (float)ceil_div(steps, splits) * each * step;
      if (splits > 1) time += 3.5f + (float)(splits * n * k) * 8e-6f / 5.f;
      if (best.size != 0 && time >= least) return;
      least = time;
      best = Cut{size, tiles, steps, splits};
    };
    // one, two and three to the power of two, and as many as fill the chip
    take(1);
    for (int64_t s = 2; s <= 1024; s *= 2) {
      take(s);
      take(s + s / 2);
    }
    for (int64_t s = 1; s <= 4; s *= 2) take(s * cus / tiles);
  }
  return best;
}

int check_codes(const char* what, const int8_t* codes, int64_t stride, const uint8_t* exponents, int64_t k) {
  F2CGT_REQUIRE(codes && exponents, F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(stride % 16 == 0 && stride >= k && aligned(codes, 16), F2CGT_E_UNSUPPORTED,
                "%s: rows of codes must start at multiples of 16 bytes and not overlap", what);
  return 0;
}
int check_sizes(const char* what, int64_t m, int64_t n, int64_t k) {
  F2CGT_REQUIRE(m >= 0 && n >= 0 && k >= 0, F2CGT_E_INVALID, "%s: sizes must not be negative", what);
  F2CGT_REQUIRE(m < (1ll << 31) && n < (1ll << 22) && k < (1ll << 22), F2CGT_E_UNSUPPORTED,
                "%s: at most 2^31 - 1 rows and 2^22 - 1 columns", what);
  return 0;
}

// Pieces of all rows in workgroups of 1024.
template <typename T>
int pieces_launch(const char* what, PackArgs& a, unsigned& blocks) {
  a.groups = (int)ceil_div(a.k, kCheckpointGroup);
  a.pieces = (uint32_t)a.groups * (kCheckpointGroup / kPieceOf<T>);
  const int64_t all = ceil_div(a.m * a.pieces, 256 * kPackUnroll);
  F2CGT_REQUIRE(all < (1ll << 24), F2CGT_E_UNSUPPORTED, "%s: too many values for a launch", what);     // (2^32 threads)
  blocks = (unsigned)all;
  return 0;
}

}  // namespace
}  // namespace f2cgt

using namespace f2cgt;

extern "C" int f2cgt_pack_activations(const void* x, int dtype, int64_t ld, int8_t* codes, int64_t code_stride,
                                      uint8_t* exponents, int64_t m, int64_t k, void* stream) {
  const char* what = "pack_activations";
  if (int rc = check_sizes(what, m, 0, k)) return rc;
  F2CGT_REQUIRE(dense_type(dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 rows only", what);
  F2CGT_REQUIRE(m <= 1 || ld >= k, F2CGT_E_INVALID, "%s: rows overlap", what);
  if (m == 0 || k == 0) return 0;
  if (int rc = check_codes(what, codes, code_stride, exponents, k)) return rc;
  F2CGT_REQUIRE(x && aligned(x, type_size(dtype)), F2CGT_E_INVALID, "%s: null or misaligned rows", what);
  PackArgs a{x, nullptr, codes, exponents, m, ld, code_stride, (int)k, 0, 0};
  return with_type(dtype, [&](auto t) {
    unsigned blocks;
    if (int rc = pieces_launch<decltype(t)>(what, a, blocks)) return rc;
    pack_kernel<decltype(t)><<<dim3(blocks), dim3(256), 0, as_stream(stream)>>>(a);
    return launch_status(what);
  });
}

extern "C" int f2cgt_unpack_activations(const int8_t* codes, int64_t code_stride, const uint8_t* exponents, void* out, int dtype,
                                        int64_t m, int64_t k, void* stream) {
  const char* what = "unpack_activations";
  if (int rc = check_sizes(what, m, 0, k)) return rc;
  F2CGT_REQUIRE(dense_type(dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 output only", what);
  if (m == 0 || k == 0) return 0;
  if (int rc = check_codes(what, codes, code_stride, exponents, k)) return rc;
  F2CGT_REQUIRE(out && aligned(out, type_size(dtype)), F2CGT_E_INVALID, "%s: null or misaligned output", what);
  PackArgs a{nullptr, out, const_cast<int8_t*>(codes), const_cast<uint8_t*>(exponents), m, k, code_stride, (int)k, 0, 0};
  return with_type(dtype, [&](auto t) {
    unsigned blocks;
    if (int rc = pieces_launch<decltype(t)>(what, a, blocks)) return rc;
    unpack_kernel<decltype(t)><<<dim3(blocks), dim3(256), 0, as_stream(stream)>>>(a);
    return launch_status(what);
  });
}

extern "C" int64_t f2cgt_packed_linear_grad_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || !dense_type(dtype)) return 0;
  const Cut c = cut_of(dtype, m, n, k);
  return c.splits > 1 ? c.splits * n * (k + 1) * 4 : 0;
}

extern "C" int f2cgt_packed_linear_grad(const void* grad, int dtype, int64_t ld, const int8_t* codes, int64_t code_stride,
                                        const uint8_t* exponents, void* dweight, void* dbias, int out_dtype, void* workspace,
                                        int64_t workspace_bytes, int64_t m, int64_t n, int64_t k, void* stream) {
  const char* what = "packed_linear_grad";
  if (int rc = check_sizes(what, m, n, k)) return rc;
  F2CGT_REQUIRE(dense_type(dtype) && dense_type(out_dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 only", what);
  F2CGT_REQUIRE(m <= 1 || ld >= n, F2CGT_E_INVALID, "%s: rows overlap", what);
  F2CGT_REQUIRE(m <= 1 || (ld < (1ll << 24) && code_stride < (1ll << 24)), F2CGT_E_UNSUPPORTED, "%s: rows 2^24 and more apart", what);
  if (n == 0 || (k == 0 && !dbias)) return 0;
  F2CGT_REQUIRE(dweight || k == 0, F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(aligned(grad, type_size(dtype)) && aligned(dweight, type_size(out_dtype)) && aligned(dbias, type_size(out_dtype)),
                F2CGT_E_INVALID, "%s: misaligned buffer", what);
  if (m > 0) {
    F2CGT_REQUIRE(grad, F2CGT_E_INVALID, "%s: null buffer", what);
    if (k > 0)
      if (int rc = check_codes(what, codes, code_stride, exponents, k)) return rc;
  }
  hipStream_t st = as_stream(stream);
  if (k == 0) {
    const ColumnArgs a{grad, dbias, m, ld, (int)n, out_dtype};
    return with_type(dtype, [&](auto t) {
      column_sums_kernel<decltype(t)><<<dim3((unsigned)ceil_div(n, kWave)), dim3(kColumnWaves * kWave), 0, st>>>(a);
      return launch_status(what);
    });
  }
  Cut c{};
  if (m > 0) {
    c = cut_of(dtype, m, n, k);
    const int64_t need = f2cgt_packed_linear_grad_workspace_bytes(dtype, m, n, k);
    F2CGT_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), F2CGT_E_INVALID,
                  "%s: workspace too small or misaligned", what);
    F2CGT_REQUIRE(c.tiles * c.splits < (1ll << 22), F2CGT_E_UNSUPPORTED, "%s: too many tiles", what);
    const GradArgs a{grad, codes, exponents, c.splits > 1 ? static_cast<float*>(workspace) : nullptr, dweight, dbias, m, ld,
                     code_stride, (int)n, (int)k, (int)ceil_div(k, kCheckpointGroup), out_dtype, c.steps, (uint32_t)c.splits,
                     (uint32_t)ceil_div(n, c.size), (uint32_t)ceil_div(k, c.size)};
    const dim3 grid((unsigned)(c.tiles * c.splits));
    const int rc = with_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      constexpr int tag = dtype_of<T>::tag;
      if (c.size == 256) packed_linear_grad_kernel<T, 256, 256, 128, 64, rows_of_step(tag, 256), 1><<<grid, dim3(512), 0, st>>>(a);
      else if (c.size == 128) packed_linear_grad_kernel<T, 128, 128, 64, 64, rows_of_step(tag, 128), 2><<<grid, dim3(512), 0, st>>>(a);
      else packed_linear_grad_kernel<T, 64, 64, 32, 32, rows_of_step(tag, 64), 1><<<grid, dim3(256), 0, st>>>(a);
      return launch_status(what);
    });
    if (rc || c.splits == 1) return rc;
  }
  // Few splits: a wave for 256 outputs.  Many: sixteen waves for 256, or for 64 until there is a workgroup for each CU (128 x 128 of 255
  // splits 8 us in 64 workgroups, 6 in 256).
  const bool few = c.splits <= 8;
  const int outs = few ? 1024 : n * k <= 64 * (int64_t)num_cus() ? 64 : 256;
  F2CGT_REQUIRE(ceil_div(n * k, outs) < (1ll << 21), F2CGT_E_UNSUPPORTED, "%s: too many outputs", what);
  const JoinArgs j{static_cast<const float*>(workspace), dweight, dbias, n * k, (int)n, out_dtype, (uint32_t)c.splits,
                   (uint32_t)ceil_div(n * k, outs)};
  const dim3 join_grid(j.blocks + (dbias ? (unsigned)ceil_div(n, outs) : 0u));
  if (few) join_splits_kernel<4, 1, 4><<<join_grid, dim3(256), 0, st>>>(j);
  else if (outs == 64) join_splits_kernel<16, 16, 1><<<join_grid, dim3(1024), 0, st>>>(j);
  else join_splits_kernel<16, 16, 4><<<join_grid, dim3(1024), 0, st>>>(j);
  return launch_status(what);
}
