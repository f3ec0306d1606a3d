// Activations kept in 8 bits between the forward and the backward pass, and the products that are made with them.
//
// pack:   groups of 32 columns of a row, one exponent E a group, code = rint(x 2^(127 - E))      (the choice of E: rows.hpp)
// unpack: code 2^(E - 127)
// grad:   dW = g^T v, db = sum of g's rows, for a layer out = v W^T + b whose input v is held as codes
//
// Pack and unpack are bound by memory.  The product goes through bf16 matrix instructions: every v is a bf16 exactly, and g is one
// bf16 plane (bf16), two (fp16: 11 bits in 8 + 8) or three (fp32: 24 bits in 8 + 8 + 8, cut off one after the other, exactly), so all
// products are exact and only the fp32 sums round.
#include "rows.hpp"
#include "tile_product.hpp"

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

// A tile of dW: BN outputs by BK inputs, WN x WK to a wave, BM rows of g and v a step; GROUPS groups of waves take the steps in turn and
// add their sums in the end.  Rows lie in LDS as they do in memory, one line of BN or BK bf16 a row, and matrix operands, which hold
// eight rows of one column a lane, are read through the transposing LDS loads: sixteen lanes give the addresses of 4 rows x 16
// columns in four pieces a row, and get a column each.  Units of 64 bytes of a line change places by the row's last two bits, so the four
// rows of such a read lie in different banks.
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
    uint32_t e[kPiecesX];
  };
};

template <typename T, int BN, int BK, int WN, int WK, int BM, int GROUPS>
__global__ __launch_bounds__((BN / WN) * (BK / WK) * kWave * GROUPS) void packed_linear_grad_kernel(GradArgs a) {
  typedef GradTile<T, BN, BK, WN, WK, BM, GROUPS> Tile;
  constexpr int P = Tile::P, TI = Tile::TI, TJ = Tile::TJ, kThreads = Tile::kThreads;
  constexpr int kAcross = (BN * BK * 4) * (GROUPS - 1);                 // the groups' sums on their way to the first one
  constexpr int kLds = 2 * Tile::kStage * GROUPS > kAcross ? 2 * Tile::kStage * GROUPS : kAcross;
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
  const int64_t from = a.steps * split / a.splits, to = a.steps * (split + 1) / a.splits;

  // this thread's columns: those beyond the operand's end repeat its first ones (what they give is not kept)
  const int pg = t % (BN / 8) * 8, px = t % (BK / 8) * 8, rg = t / (BN / 8), rx = t / (BK / 8);
  const int cg = col_n + pg < a.n ? col_n + pg : 0, cx = col_k + px < a.k ? col_k + px : 0;
  // (32 bits from a step's first row: strides are below 2^24)
  const uint32_t off_g = (uint32_t)(rg * (int)a.ld + cg) * (uint32_t)sizeof(T), off_x = (uint32_t)(rx * (int)a.code_stride + cx);
  const uint32_t off_e = (uint32_t)(rx * a.groups + cx / kCheckpointGroup);
  typedef typename Tile::Held Held;

  // A piece that runs over its row's end reads on in the next one; the last rows, which have none, are read value by value.  Steps behind
  // the last one read it again.
  const bool pieces = a.n >= 8 && a.k > 0;
  auto load = [&](Held& h, int64_t step) {
    const int64_t row0 = (step < to ? step : to - 1) * BM;
    const char* grad = static_cast<const char*>(a.grad) + row0 * a.ld * (int64_t)sizeof(T);
    const int8_t* codes = a.codes + row0 * a.code_stride;
    const uint8_t* exponents = a.exponents + row0 * a.groups;
    if (row0 + BM < a.m && pieces) {
#pragma unroll
      for (int i = 0; i < Tile::kPiecesG; ++i) h.g[i].load(grad + (int64_t)i * Tile::kRowsG * a.ld * (int64_t)sizeof(T) + off_g);
#pragma unroll
      for (int i = 0; i < Tile::kPiecesX; ++i) {
        h.x[i] = *reinterpret_cast<const uint2*>(codes + i * Tile::kRowsX * a.code_stride + off_x);
        h.e[i] = exponents[(int64_t)i * Tile::kRowsX * a.groups + off_e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < Tile::kPiecesG; ++i) {
        const bool in = row0 + rg + i * Tile::kRowsG < a.m;
        const T* p = reinterpret_cast<const T*>(grad + (int64_t)i * Tile::kRowsG * a.ld * (int64_t)sizeof(T) + off_g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          T v = (T)0.f;
          if (in && cg + e < a.n) v = p[e];
          h.g[i].set(e, v);
        }
      }
#pragma unroll
      for (int i = 0; i < Tile::kPiecesX; ++i) {
        h.x[i] = uint2{0, 0};
        h.e[i] = 127;
        if (row0 + rx + i * Tile::kRowsX < a.m && a.k > 0) {
          h.x[i] = *reinterpret_cast<const uint2*>(codes + i * Tile::kRowsX * a.code_stride + off_x);
          h.e[i] = exponents[(int64_t)i * Tile::kRowsX * a.groups + off_e];
        }
      }
    }
  };
  const bool sums = a.bias != nullptr && tj == 0;
  float db[8] = {};
  // Pieces of one of kParts parts into a stage.
  auto place_part = [&](const Held& h, char* stage, int part, bool count) {
#pragma unroll
    for (int i = 0; i < Tile::kPiecesG; ++i) {
      if (i % Tile::kParts != part) continue;
      if (sums && count)
#pragma unroll
        for (int e = 0; e < 8; ++e) db[e] += h.g[i][e];
      intx4 planes[P];
      h.g[i].planes(planes);
#pragma unroll
      for (int p = 0; p < P; ++p)
        *reinterpret_cast<intx4*>(stage + p * Tile::kPlaneG + Tile::line_at(rg + i * Tile::kRowsG, pg * 2, Tile::kLineG)) = planes[p];
    }
#pragma unroll
    for (int i = 0; i < Tile::kPiecesX; ++i) {
      if (i % Tile::kParts != part) continue;
      const float step = step_of(h.e[i]);
      intx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t word = e < 2 ? h.x[i].x : h.x[i].y;
        v[e] = (int)__builtin_amdgcn_perm(__float_as_uint(coded_value(word, 2 * (e % 2) + 1, step)),
                                          __float_as_uint(coded_value(word, 2 * (e % 2), step)), 0x07060302);
      }
      *reinterpret_cast<intx4*>(stage + P * Tile::kPlaneG + Tile::line_at(rx + i * Tile::kRowsX, px * 2, Tile::kLineX)) = v;
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
  auto multiply_part = [&](const char* stage, int s) {
    bfx8 fx[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) fx[j] = operand(stage + P * Tile::kPlaneG, s, wj + 32 * j, Tile::kLineX);
#pragma unroll
    for (int p = P - 1; p >= 0; --p) {
      bfx8 fg[TI];
#pragma unroll
      for (int i = 0; i < TI; ++i) fg[i] = operand(stage + p * Tile::kPlaneG, s, wi + 32 * i, Tile::kLineG);
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fg[i], fx[j], acc[i][j], 0, 0, 0);
    }
  };
  // Two steps of each group are on their way from memory while one is multiplied: a round trip is longer than a step.
  // Step s is multiplied out of stage s % 2 while the next one is placed in the other; then the registers of that take the step after the next two.
  const int64_t rounds = (to - from + GROUPS - 1) / GROUPS;
  Held held[2];
  load(held[0], from + group);
  load(held[1], from + group + GROUPS);
#pragma unroll
  for (int part = 0; part < Tile::kParts; ++part) place_part(held[0], stages, part, from + group < to);
  load(held[0], from + group + 2 * GROUPS);
  __syncthreads();
  for (int64_t r = 0; r < rounds; r += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (r + u < rounds) {
        const int64_t step = from + group + (r + u) * GROUPS;
        char* now = stages + u * Tile::kStage;
        char* next = stages + (u ^ 1) * Tile::kStage;
        Held& h = held[u ^ 1];
#pragma unroll
        for (int part = 0; part < Tile::kParts; ++part) {
          if (GROUPS == 1 || step < to) multiply_part(now, part);
          place_part(h, next, part, step + GROUPS < to);
        }
        load(h, step + 3 * GROUPS);
        __syncthreads();
      }
    }
  }
  if constexpr (GROUPS > 1) {
    // the other groups' sums, in their order
    float* across = reinterpret_cast<float*>(lds);
    if (group > 0) {
      float* to_first = across + (group - 1) * BN * BK;
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) to_first[((i * TJ + j) * 16 + v) * kThreads + t] = acc[i][j][v];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int g = 0; g < GROUPS - 1; ++g)
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
          for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] += across[g * BN * BK + ((i * TJ + j) * 16 + v) * kThreads + t];
    }
  }
  // Sums out: a lane holds, of column lane % 32, rows 4 (lane / 32) to + 3 after every eight.
  if (group == 0) {
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int row = col_n + wi + 32 * i + 8 * (v / 4) + 4 * (lane >> 5) + v % 4, column = col_k + wj + 32 * j + (lane & 31);
          if (row < a.n && column < a.k) {
            const int64_t at = (int64_t)row * a.k + column;
            if (a.parts != nullptr) a.parts[(int64_t)split * a.n * a.k + at] = acc[i][j][v];
            else store_value(a.out, a.out_tag, at, acc[i][j][v]);
          }
        }
  }
  if (!sums) return;
  if constexpr (GROUPS > 1) __syncthreads();
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

// Sums over the splits: a workgroup has 256 outputs, each of its waves every fourth split, then the waves' sums in order; the bias' in
// workgroups behind the weight's.  (No splits: zeros, of no rows.)
struct JoinArgs {
  const float* parts;
  void* out;
  void* bias;
  int64_t count;             // n k
  int n, tag, whole;         // whole: four values at a time
  uint32_t splits, blocks;   // blocks: those of the weight
};
__global__ __launch_bounds__(256) void join_splits_kernel(JoinArgs a) {
  __shared__ __attribute__((aligned(16))) float room[4][256];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const bool weight = blockIdx.x < a.blocks;
  const int64_t count = weight ? a.count : a.n, first = (int64_t)(weight ? blockIdx.x : blockIdx.x - a.blocks) * 256;
  const float* parts = weight ? a.parts : a.parts + (int64_t)a.splits * a.count;
  void* out = weight ? a.out : a.bias;
  const int64_t at = first + 4 * lane;
  fltx4 sum = {0.f, 0.f, 0.f, 0.f};
  if (weight && a.whole) {
    if (at < count) {
      uint32_t s = wave;
      for (; s + 12 < a.splits; s += 16) {
        fltx4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const fltx4*>(parts + (int64_t)(s + 4 * u) * count + at);
#pragma unroll
        for (int u = 0; u < 4; ++u) sum += v[u];
      }
      for (; s < a.splits; s += 4) sum += *reinterpret_cast<const fltx4*>(parts + (int64_t)s * count + at);
    }
  } else {
    for (uint32_t s = wave; s < a.splits; s += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += at + e < count ? parts[(int64_t)s * count + at + e] : 0.f;
  }
  *reinterpret_cast<fltx4*>(&room[wave][4 * lane]) = sum;
  __syncthreads();
  if (first + threadIdx.x >= count) return;
  const float all = room[0][threadIdx.x] + room[1][threadIdx.x] + room[2][threadIdx.x] + room[3][threadIdx.x];
  store_value(out, a.tag, first + threadIdx.x, all);
}

// How a product is cut: tiles of `size` squared, rows in `splits`.
struct Cut {
  int size;
  int64_t tiles, steps, splits;
};
Cut cut_of(int dtype, int64_t m, int64_t n, int64_t k) {
  const int64_t cus = num_cus();
  Cut c;
  auto tiles = [&](int size) { return ceil_div(n, size) * (k > 0 ? ceil_div(k, size) : 1); };     // (a bias has rows without columns too)
  c.size = tiles(256) >= cus ? 256 : tiles(64) * ceil_div(m, 32) <= 4 * cus ? 64 : n * k > 64 * 64 ? 128 : 64;
  const int bm = dtype == F2CGT_DT_BF16 && c.size != 64 ? 64 : 32;
  c.tiles = tiles(c.size);
  c.steps = ceil_div(m, bm);
  const int64_t most = c.steps, want = c.size == 256 ? 1 : c.size == 128 ? cus / c.tiles : 2 * cus / c.tiles;
  c.splits = want < 1 ? 1 : want > most ? most : want;
  return c;
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
  if (m <= 0 || n <= 0 || k < 0 || !dense_type(dtype)) return 0;
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
  Cut c{};
  if (m > 0) {
    c = cut_of(dtype, m, n, k);
    const int64_t need = f2cgt_packed_linear_grad_workspace_bytes(dtype, m, n, k);
    F2CGT_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), F2CGT_E_INVALID,
                  "%s: workspace too small or misaligned", what);
    F2CGT_REQUIRE(c.tiles * c.splits < (1ll << 22), F2CGT_E_UNSUPPORTED, "%s: too many tiles", what);
    const GradArgs a{grad, codes, exponents, c.splits > 1 ? static_cast<float*>(workspace) : nullptr, dweight, dbias, m, ld,
                     code_stride, (int)n, (int)k, (int)ceil_div(k, kCheckpointGroup), out_dtype, c.steps, (uint32_t)c.splits,
                     (uint32_t)ceil_div(n, c.size), (uint32_t)(k > 0 ? ceil_div(k, c.size) : 1)};
    const dim3 grid((unsigned)(c.tiles * c.splits));
    const int rc = with_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      constexpr int BM = kPlanes<T> == 1 ? 64 : 32;
      if (c.size == 256) packed_linear_grad_kernel<T, 256, 256, 128, 64, BM, 1><<<grid, dim3(512), 0, st>>>(a);
      else if (c.size == 128) packed_linear_grad_kernel<T, 128, 128, 64, 64, BM, 2><<<grid, dim3(512), 0, st>>>(a);
      else packed_linear_grad_kernel<T, 64, 64, 32, 32, 32, 1><<<grid, dim3(256), 0, st>>>(a);
      return launch_status(what);
    });
    if (rc || c.splits == 1) return rc;
  }
  JoinArgs j{static_cast<const float*>(workspace), dweight, dbias, n * k, (int)n, out_dtype,
             n * k % 4 == 0 && aligned(dweight, 4 * type_size(out_dtype)), (uint32_t)c.splits, (uint32_t)ceil_div(n * k, 256)};
  F2CGT_REQUIRE(ceil_div(n * k, 256) < (1ll << 23), F2CGT_E_UNSUPPORTED, "%s: too many outputs", what);
  join_splits_kernel<<<dim3(j.blocks + (dbias ? (unsigned)ceil_div(n, 256) : 0u)), dim3(256), 0, st>>>(j);
  return launch_status(what);
}
