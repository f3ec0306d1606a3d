// A tile of C = A B^T on the matrix instructions, from operands whose rows are lines of 128 bytes along the summed dimension:
// 128 codes of 8 bits, or 32 numbers as two fp16 planes (hi, then lo).  Both products of this library that are bound by
// matrix instructions, the one of 8-bit codes and the Newton-Schulz products, share it; they differ in what they do
// with a line (an Op) and with a finished strip of the tile (an epilogue).
#pragma once

#include "common.hpp"

namespace f2cgt {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
typedef float fltx4 __attribute__((ext_vector_type(4)));
typedef float fltx16 __attribute__((ext_vector_type(16)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));

constexpr int kLine = 128;                 // bytes of a row that a step of the main loop takes

// Rows of one operand: row r at base + r * stride (a multiple of 16), `bytes` of it are summed over.
struct Lines {
  const char* base;
  int64_t stride;
  int64_t rows;
  int64_t bytes;
};

// 8-bit codes: a group is one 32 x 32 x 32 instruction over 32 codes.
struct Int8Op {
  typedef intx16 Acc;
  static constexpr int kGroups = 4, kParts = 1;
  static __device__ __forceinline__ int chunk(int group, int) { return 2 * group; }
  static __device__ __forceinline__ void mma(Acc& acc, const intx4 (&p)[1], const intx4 (&q)[1]) {
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(p[0], q[0], acc, 0, 0, 0);
  }
};

// Two fp16 planes: x = hi + lo to 2^-23 of x, and of the four products hi hi, hi lo and lo hi (the fourth is 2^-23 of the
// first): a group is three 32 x 32 x 16 instructions over 16 numbers.
struct SplitOp {
  typedef fltx16 Acc;
  static constexpr int kGroups = 2, kParts = 2;
  static __device__ __forceinline__ int chunk(int group, int part) { return 4 * part + 2 * group; }
  static __device__ __forceinline__ void mma(Acc& acc, const intx4 (&p)[2], const intx4 (&q)[2]) {
    const halfx8 p0 = __builtin_bit_cast(halfx8, p[0]), p1 = __builtin_bit_cast(halfx8, p[1]);
    const halfx8 q0 = __builtin_bit_cast(halfx8, q[0]), q1 = __builtin_bit_cast(halfx8, q[1]);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(p1, q0, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(p0, q1, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(p0, q0, acc, 0, 0, 0);
  }
};

// 16 bytes of row r from byte k0 on, zeros behind the operand's end.  Rows beyond the last one repeat it (what they give is not kept).
__device__ __forceinline__ intx4 line_piece(const Lines& x, int64_t r, int64_t k0) {
  const char* p = x.base + (r < x.rows ? r : x.rows - 1) * x.stride + k0;
  intx4 v = {0, 0, 0, 0};
  if (k0 + 16 <= x.bytes) {
    v = *reinterpret_cast<const intx4*>(p);
  } else if (k0 < x.bytes) {
    const int left = (int)(x.bytes - k0);
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < left) v[i >> 2] |= (int)(uint8_t)p[i] << (8 * (i & 3));
  }
  return v;
}

// A piece's place in LDS: rows of 128 bytes, the eight pieces of a row in another order in each of eight rows, so that the
// lanes of a read, which take the same piece of consecutive rows, spread over the banks.
__device__ __forceinline__ int piece_at(int r, int c) { return r * kLine + ((c ^ (r & 7)) << 4); }

// A sum as a word of LDS.  (By value: a bit cast of a vector's element itself takes the vector's first one.)
__device__ __forceinline__ float word_of(float v) { return v; }
__device__ __forceinline__ float word_of(int v) { return __builtin_bit_cast(float, v); }

template <class Op, int BM, int BN, int WM, int WN>
struct TileProduct {
  static constexpr int kWaves = (BM / WM) * (BN / WN), kThreads = kWaves * kWave;
  static constexpr int TI = WM / 32, TJ = WN / 32;
  static constexpr int kLd = WN + 4;                                   // floats of a strip's row in LDS
  static constexpr int kStrip = 32 * kLd * 4;
  static constexpr int kStage = (BM + BN) * kLine;
  static constexpr int kLds = kStage > kWaves * kStrip ? kStage : kWaves * kStrip;
  typedef typename Op::Acc Acc;

  // Rows [row0, row0 + BM) of a against rows [col0, col0 + BN) of b.  epilogue(strip, row, col, lane): strip [32][kLd] holds
  // the sums of 32 rows from `row` on and WN columns from `col` on.
  template <class Epilogue>
  static __device__ __forceinline__ void run(char* lds, const Lines& a, const Lines& b, int64_t row0, int64_t col0, const Epilogue& epilogue) {
    const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int wi = (wave % (BM / WM)) * WM, wj = (wave / (BM / WM)) * WN;
    constexpr int PA = BM * 8 / kThreads, PB = BN * 8 / kThreads;
    static_assert(BM * 8 % kThreads == 0 && BN * 8 % kThreads == 0, "whole pieces per thread");
    intx4 va[PA], vb[PB];
    auto load = [&](int64_t k0) {
#pragma unroll
      for (int i = 0; i < PA; ++i) {
        const int q = t + i * kThreads;
        va[i] = line_piece(a, row0 + (q >> 3), k0 + 16 * (q & 7));
      }
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        const int q = t + i * kThreads;
        vb[i] = line_piece(b, col0 + (q >> 3), k0 + 16 * (q & 7));
      }
    };
    Acc acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
    const int at = lane & 31, side = lane >> 5;
    load(0);
    for (int64_t k0 = 0; k0 < a.bytes; k0 += kLine) {
#pragma unroll
      for (int i = 0; i < PA; ++i) {
        const int q = t + i * kThreads;
        *reinterpret_cast<intx4*>(lds + piece_at(q >> 3, q & 7)) = va[i];
      }
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        const int q = t + i * kThreads;
        *reinterpret_cast<intx4*>(lds + BM * kLine + piece_at(q >> 3, q & 7)) = vb[i];
      }
      __syncthreads();
      if (k0 + kLine < a.bytes) load(k0 + kLine);
#pragma unroll
      for (int g = 0; g < Op::kGroups; ++g) {
        intx4 fa[TI][Op::kParts], fb[TJ][Op::kParts];
#pragma unroll
        for (int p = 0; p < Op::kParts; ++p) {
#pragma unroll
          for (int i = 0; i < TI; ++i)
            fa[i][p] = *reinterpret_cast<const intx4*>(lds + piece_at(wi + 32 * i + at, Op::chunk(g, p) + side));
#pragma unroll
          for (int j = 0; j < TJ; ++j)
            fb[j][p] = *reinterpret_cast<const intx4*>(lds + BM * kLine + piece_at(wj + 32 * j + at, Op::chunk(g, p) + side));
        }
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
          for (int j = 0; j < TJ; ++j) Op::mma(acc[i][j], fb[j], fa[i]);
      }
      __syncthreads();
    }
    // The columns' operand came first: a lane holds, of one row, four columns after four.
    float* strip = reinterpret_cast<float*>(lds + wave * kStrip);
#pragma unroll
    for (int i = 0; i < TI; ++i) {
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          fltx4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = word_of(acc[i][j][4 * q + e]);
          *reinterpret_cast<fltx4*>(strip + at * kLd + 32 * j + 8 * q + 4 * side) = v;
        }
      __builtin_amdgcn_wave_barrier();
      epilogue(strip, row0 + wi + 32 * i, col0 + wj, lane);
      __builtin_amdgcn_wave_barrier();
    }
  }
};

// ---- values of the types that the dense operators take ---------------------------------------------------
__device__ __forceinline__ float load_value(const void* p, int dtype, int64_t i) {
  if (dtype == F2CGT_DT_F32) return static_cast<const float*>(p)[i];
  if (dtype == F2CGT_DT_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void store_value(void* p, int dtype, int64_t i, float v) {
  if (dtype == F2CGT_DT_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == F2CGT_DT_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
  else static_cast<__bf16*>(p)[i] = (__bf16)v;
}
inline bool dense_type(int dtype) { return dtype == F2CGT_DT_F32 || dtype == F2CGT_DT_F16 || dtype == F2CGT_DT_BF16; }
inline int type_size(int dtype) { return dtype == F2CGT_DT_F32 ? 4 : 2; }

}  // namespace f2cgt
