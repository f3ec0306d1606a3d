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
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));

constexpr int kLine = 128;                 // bytes of a row that a step of the main loop takes

// Rows of one operand: row r at base + r * stride (a multiple of 16), `bytes` of it are summed over.
// The 16-byte piece with a row's last byte is read as a whole.
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
  static constexpr bool kTrim = true;        // a row may end within a line
  static __device__ __forceinline__ int chunk(int group, int) { return 2 * group; }
  static constexpr int kTerms = 1;
  static __device__ __forceinline__ void mma(Acc& acc, int, const intx4 (&p)[1], const intx4 (&q)[1]) {
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(p[0], q[0], acc, 0, 0, 0);
  }
};

// Two fp16 planes: x = hi + lo to 2^-23 of x, and of the four products hi hi, hi lo and lo hi (the fourth is 2^-23 of the
// first): a group is three 32 x 32 x 16 instructions over 16 numbers.
struct SplitOp {
  typedef fltx16 Acc;
  static constexpr int kGroups = 2, kParts = 2;
  static constexpr bool kTrim = false;       // rows are whole lines
  static __device__ __forceinline__ int chunk(int group, int part) { return 4 * part + 2 * group; }
  static constexpr int kTerms = 3;             // (one after the other over all tiles: in a row on one they wait for each other)
  static __device__ __forceinline__ void mma(Acc& acc, int term, const intx4 (&p)[2], const intx4 (&q)[2]) {
    const halfx8 a = __builtin_bit_cast(halfx8, p[term == 0 ? 1 : 0]), b = __builtin_bit_cast(halfx8, q[term == 1 ? 1 : 0]);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
  }
};

// A piece's place in LDS: rows of 128 bytes, the eight pieces of a row in another order in each of eight pairs of rows (64 banks
// hold two rows), so that the lanes of a read, which take the same piece of consecutive rows, spread over the banks.
__device__ __forceinline__ int piece_at(int r, int c) { return r * kLine + ((c ^ (r >> 1 & 7)) << 4); }

// A sum as a word of LDS.  (By value: a bit cast of a vector's element itself takes the vector's first one.)
__device__ __forceinline__ float word_of(float v) { return v; }
__device__ __forceinline__ float word_of(int v) { return __builtin_bit_cast(float, v); }
__device__ __forceinline__ void add_word(fltx16& sums, int i, float word) { sums[i] += word; }
__device__ __forceinline__ void add_word(intx16& sums, int i, float word) { sums[i] += __builtin_bit_cast(int, word); }

// Waits until this wave's copies into LDS and its reads of LDS are done.
__device__ __forceinline__ void wait_copies() { __builtin_amdgcn_s_waitcnt(7 << 4); }

// The pieces of a tile go from memory into LDS without a stop in registers, a step ahead of the one that is multiplied; a step
// costs one barrier.  The two stages are LDS arrays of their own (Buffers), which is how the compiler knows that a read of one need not
// wait for the copies into the other.
//
// GROUPS > 1: groups of waves take the steps in turn, each into its own part of the stages, and add their sums in the end: for
// tiles that are fewer than the chip's CUs (256 x 4096 x 4096 in 8 bits: four groups 12.8 us, two 14.3, one 20.6).
//
// With three stages or four the same tiles took as long or longer (fp16 planes, 1000 x 2051: 19.6 us with two, 20.1 and 22.2), for the time of a step is the LDS's, which writes each byte once and reads it once for every wave beside or
// below, and a stage more is a workgroup less on a CU.
template <class Op, int BM, int BN, int WM, int WN, int GROUPS = 1>
struct TileProduct {
  static constexpr int kWaves = (BM / WM) * (BN / WN), kThreads = kWaves * kWave;      // of a group
  static constexpr int kBlock = kThreads * GROUPS;
  static constexpr int TI = WM / 32, TJ = WN / 32;
  static constexpr int kLd = WN + 4;                                   // floats of a strip's row in LDS
  static constexpr int kStrip = 32 * kLd * 4;
  static constexpr int kPart = (BM + BN) * kLine;                      // bytes of a group's stage
  static constexpr int kStage = GROUPS * kPart;                        // of a buffer
  static constexpr int kPieces = (BM + BN) * 8 / kThreads;             // copies of a thread in a step
  static_assert((BM + BN) * 8 % kThreads == 0 && BM * 8 % kThreads == 0, "whole pieces per thread");
  static constexpr int kStripsPerStage = kStage / kStrip;
  static_assert(kStripsPerStage * 2 >= kWaves * GROUPS, "a strip per wave");
  typedef typename Op::Acc Acc;
  typedef char* Buffers[2];

  // Rows [row0, row0 + BM) of a against rows [col0, col0 + BN) of b.  epilogue(strip, row, col, lane): strip [32][kLd] holds
  // the sums of 32 rows from `row` on and WN columns from `col` on.
  template <class Epilogue>
  static __device__ __forceinline__ void run(const Buffers& lds, const Lines& a, const Lines& b, int64_t row0, int64_t col0,
                                             const Epilogue& epilogue) {
    const int group = GROUPS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads) : 0;
    const int t = threadIdx.x - group * kThreads, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int wi = (wave % (BM / WM)) * WM, wj = (wave / (BM / WM)) * WN;
    const int at = lane & 31, side = lane >> 5;
    const int steps = (int)((a.bytes + kLine - 1) / kLine);
    const int left = (int)(a.bytes - (int64_t)(steps - 1) * kLine);     // bytes of the last step

    // Thread t copies the pieces of places t + i kThreads: place q holds, of row q / 8, piece (q % 8) ^ (row / 2 % 8), and the rows
    // of a thread are whole sixteens apart: the same piece of each.  Rows beyond the operand's end repeat its last one: what they give
    // is not kept.  Offsets are 32 bits from a tile's first row (strides are below 2^23 here).
    const int piece = ((t & 7) ^ (t >> 4 & 7)) << 4;
    static_assert(kThreads % 128 == 0, "rows of a thread sixteen apart");
    const char* base_a = a.base + row0 * a.stride;
    const char* base_b = b.base + col0 * b.stride;
    uint32_t from[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const bool first = i * kThreads < BM * 8;
      const int r = (t + i * kThreads) / 8 - (first ? 0 : BM);
      const int64_t rows = first ? a.rows - row0 : b.rows - col0;
      from[i] = (uint32_t)(r < rows ? r : (int)rows - 1) * (uint32_t)(first ? a.stride : b.stride) + piece;
    }
    auto copy = [&](char* to, int step) {
      // (pieces of the last step that begin behind the end: the row's first one of this step, which is made zero below)
      const int back = step == steps - 1 && piece >= left ? piece : 0;
      const char* pa = base_a + (int64_t)step * kLine;
      const char* pb = base_b + (int64_t)step * kLine;
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)((i * kThreads < BM * 8 ? pa : pb) + (from[i] - back)),
            (__attribute__((address_space(3))) void*)(to + (wave * kWave + i * kThreads) * 16), 16, 0, 0);
    };
    // The first operand's bytes behind the end made zero, by the thread that copied them (the second's then do not count).
    auto trim = [&](char* stage) {
      const int in = left - piece;
      intx4 mask;
#pragma unroll
      for (int e = 0; e < 4; ++e) mask[e] = in >= 4 * e + 4 ? -1 : in <= 4 * e ? 0 : (1 << (8 * (in - 4 * e))) - 1;
#pragma unroll
      for (int i = 0; i * kThreads < BM * 8; ++i) {
        intx4* at_piece = reinterpret_cast<intx4*>(stage + (t + i * kThreads) * 16);
        *at_piece &= mask;
      }
      __builtin_amdgcn_s_waitcnt(63 | 3 << 14 | 7 << 4 | 0 << 8);      // (LDS only)
    };
    Acc acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
    // Products of a stage, a group's operands read while the group before is multiplied.
    auto multiply = [&](const char* stage) {
      intx4 fa[2][TI][Op::kParts], fb[2][TJ][Op::kParts];
      auto read = [&](int g) {
#pragma unroll
        for (int p = 0; p < Op::kParts; ++p) {
#pragma unroll
          for (int j = 0; j < TJ; ++j)
            fb[g & 1][j][p] = *reinterpret_cast<const intx4*>(stage + BM * kLine + piece_at(wj + 32 * j + at, Op::chunk(g, p) + side));
#pragma unroll
          for (int i = 0; i < TI; ++i)
            fa[g & 1][i][p] = *reinterpret_cast<const intx4*>(stage + piece_at(wi + 32 * i + at, Op::chunk(g, p) + side));
        }
      };
      read(0);
#pragma unroll
      for (int g = 0; g < Op::kGroups; ++g) {
        if (g + 1 < Op::kGroups) read(g + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < Op::kTerms; ++m)
#pragma unroll
          for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) Op::mma(acc[i][j], m, fb[g & 1][j], fa[g & 1][i]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (steps > 0) {
      // Step `step` from stage s: this wave's copies are done, then all waves' are, and nobody reads the other stage any more, into
      // which the next step's go.  (There always are some: behind the last step it is copied again, into a stage that nobody reads.)
      auto held = [&](int step) { return step < steps ? step : steps - 1; };
      const int part = group * kPart;
      copy(lds[0] + part, held(group));
      int step = group;
      while (true) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          wait_copies();
          if (Op::kTrim && left < kLine && step == steps - 1) trim(lds[s] + part);
          __builtin_amdgcn_s_barrier();
          copy(lds[1 - s] + part, held(step + GROUPS));
          __builtin_amdgcn_sched_barrier(0);             // (the compiler would sink them to the step's end)
          if (GROUPS == 1 || step < steps) multiply(lds[s] + part);
          step += GROUPS;
          if (step - group >= steps) goto done;
        }
      }
    }
  done:
    wait_copies();
    __builtin_amdgcn_s_barrier();
    // The columns' operand came first: a lane holds, of one row, four columns after four.
    auto strip_of = [&](int of) {
      const int n = of * kWaves + wave;
      char* at_stage = nullptr;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (n / kStripsPerStage == s) at_stage = lds[s] + (n % kStripsPerStage) * kStrip;
      return reinterpret_cast<float*>(at_stage);
    };
    float* strip = strip_of(group);
    auto place = [&](float* of, int j, int q) { return reinterpret_cast<fltx4*>(of + at * kLd + 32 * j + 8 * q + 4 * side); };
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      if (GROUPS > 1 && i > 0) __syncthreads();
      if (GROUPS == 1 || group > 0) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            fltx4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = word_of(acc[i][j][4 * q + e]);
            *place(strip, j, q) = v;
          }
      }
      if constexpr (GROUPS > 1) {
        __syncthreads();
        if (group > 0) continue;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int o = 1; o < GROUPS; ++o) {
              const fltx4 v = *place(strip_of(o), j, q);
#pragma unroll
              for (int e = 0; e < 4; ++e) add_word(acc[i][j], 4 * q + e, v[e]);
            }
            fltx4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = word_of(acc[i][j][4 * q + e]);
            *place(strip, j, q) = v;
          }
      }
      __builtin_amdgcn_wave_barrier();
      epilogue(strip, row0 + wi + 32 * i, col0 + wj, lane);
      __builtin_amdgcn_wave_barrier();
    }
  }
};

// Neighbours in time share operands: workgroups go round the eight XCDs, each with an L2 of its own, so an XCD gets one run of the
// tiles' order.  Workgroup `id` of `all` -> its place in that order.
__device__ __forceinline__ uint32_t place_of(uint32_t id, uint32_t all) {
  const uint32_t xcd = id & 7, share = all >> 3, more = all & 7;
  return xcd * share + (xcd < more ? xcd : more) + (id >> 3);
}
// Place `at` among tiles_m x tiles_n, which are gone through in bands of `deep` rows, a band column by column.
__device__ __forceinline__ void tile_of(uint32_t at, uint32_t tiles_m, uint32_t tiles_n, uint32_t deep, uint32_t& i, uint32_t& j) {
  const uint32_t band = at / (deep * tiles_n), first = band * deep, in = at - band * deep * tiles_n;
  const uint32_t rows = tiles_m - first < deep ? tiles_m - first : deep;
  j = in / rows;
  i = first + in - j * rows;
}
// The same of the tiles on and below the diagonal of `tiles` rows.
__device__ __forceinline__ void lower_tile_of(uint32_t at, uint32_t tiles, uint32_t deep, uint32_t& i, uint32_t& j) {
  uint32_t first = 0;
  while (true) {
    const uint32_t rows = tiles - first < deep ? tiles - first : deep, square = rows * first, all = square + rows * (rows + 1) / 2;
    if (at < square) {
      j = at / rows;
      i = first + at - j * rows;
      return;
    }
    if (at < all) {
      at -= square;
      i = 0;
      while (at > i) at -= ++i;
      j = first + at;
      i += first;
      return;
    }
    at -= all;
    first += rows;
  }
}

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
// Four neighbours at once, at an address that is a multiple of four values.
__device__ __forceinline__ void store_four(void* p, int dtype, int64_t i, const fltx4& v) {
  typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
  if (dtype == F2CGT_DT_F32) *reinterpret_cast<fltx4*>(static_cast<float*>(p) + i) = v;
  else if (dtype == F2CGT_DT_F16) *reinterpret_cast<halfx4*>(static_cast<_Float16*>(p) + i) = __builtin_convertvector(v, halfx4);
  else *reinterpret_cast<bf4*>(static_cast<__bf16*>(p) + i) = __builtin_convertvector(v, bf4);
}
__device__ __forceinline__ fltx4 load_four(const void* p, int dtype, int64_t i) {
  typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
  if (dtype == F2CGT_DT_F32) return *reinterpret_cast<const fltx4*>(static_cast<const float*>(p) + i);
  if (dtype == F2CGT_DT_F16) return __builtin_convertvector(*reinterpret_cast<const halfx4*>(static_cast<const _Float16*>(p) + i), fltx4);
  return __builtin_convertvector(*reinterpret_cast<const bf4*>(static_cast<const __bf16*>(p) + i), fltx4);
}
inline bool dense_type(int dtype) { return dtype == F2CGT_DT_F32 || dtype == F2CGT_DT_F16 || dtype == F2CGT_DT_BF16; }
inline int type_size(int dtype) { return dtype == F2CGT_DT_F32 ? 4 : 2; }

}  // namespace f2cgt
