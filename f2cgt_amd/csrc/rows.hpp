// What the operators on rows of floating values share: pieces of 16 bytes, sums over groups of lanes, and the 8-bit
// checkpoint's arithmetic.
#pragma once

#include "common.hpp"

namespace f2cgt {

// ---- pieces ----------------------------------------------------------------------------------------
// V values side by side, at any address that is a multiple of one value's size (global memory takes wide loads and stores
// at any byte).
template <typename T, int V> struct piece_words {
  typedef uint32_t type __attribute__((ext_vector_type(V * sizeof(T) / 4), aligned(sizeof(T))));
};
template <> struct piece_words<float, 1> { typedef uint32_t type; };
template <> struct piece_words<_Float16, 1> { typedef uint16_t type; };
template <> struct piece_words<__bf16, 1> { typedef uint16_t type; };

template <typename T> constexpr int kPieceOf = 16 / (int)sizeof(T);

// The words of a piece as values, and back with one rounding to nearest.
template <typename T, int V>
__device__ __forceinline__ void values_of(const typename piece_words<T, V>::type& words, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = (float)__builtin_bit_cast(T, words);
  } else {
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef uint32_t plain __attribute__((ext_vector_type(V * sizeof(T) / 4)));
    const vec t = __builtin_bit_cast(vec, (plain)words);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)t[e];
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_piece(const T* p, float (&v)[V]) {
  typedef typename piece_words<T, V>::type words;
  values_of<T, V>(*reinterpret_cast<const words*>(p), v);
}
template <typename T, int V>
__device__ __forceinline__ typename piece_words<T, V>::type words_of(const float (&v)[V]) {
  typedef typename piece_words<T, V>::type words;
  if constexpr (V == 1) {
    return __builtin_bit_cast(words, (T)v[0]);
  } else {
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef uint32_t plain __attribute__((ext_vector_type(V * sizeof(T) / 4)));
    vec t;
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = (T)v[e];
    return (words)__builtin_bit_cast(plain, t);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_piece(T* p, const float (&v)[V]) {
  *reinterpret_cast<typename piece_words<T, V>::type*>(p) = words_of<T, V>(v);
}

// ---- over groups of lanes --------------------------------------------------------------------------
template <int CONTROL>
__device__ __forceinline__ uint32_t other_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true);
}
// join(a, b) over each N neighbouring lanes (a power of two up to 64), in all of them, in one order.
template <int N, typename Join>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, const Join& join) {
  if constexpr (N >= 2) v = join(v, other_lane<0xB1>(v));          // of lane ^ 1
  if constexpr (N >= 4) v = join(v, other_lane<0x4E>(v));          // of lane ^ 2
  if constexpr (N >= 8) v = join(v, other_lane<0x141>(v));         // of lane 7 - i of its eight
  if constexpr (N >= 16) v = join(v, other_lane<0x140>(v));        // of lane 15 - i of its sixteen
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = join(r[0], r[1]);
  }
  if constexpr (N >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = join(r[0], r[1]);
  }
  return v;
}
template <int N>
__device__ __forceinline__ float sum_lanes(float v) {
  return __uint_as_float(over_lanes<N>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int N>
__device__ __forceinline__ uint32_t most_lanes(uint32_t v) {
  return over_lanes<N>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// ---- checkpoints -----------------------------------------------------------------------------------
// A group of 32 columns of a row has one exponent E: a value is code * 2^(E - 127), codes within +-127.  The step is the
// least power of two of which 127 reach the group's largest size, and 2^-126 at least: a power of two, because a code of 8 bits
// times it is a bf16 (and products with it need no rounding), and because coding is then exact arithmetic up to its one
// rounding.  127 is 1.984375 * 2^6, so a size with a larger fraction takes the next step; its top is E = 249, at which codes
// stay within +-63: 64 * 2^122 is beyond fp32.  A group with a NaN or an infinity has E = 255 and codes of zero: NaN.
constexpr int kCheckpointGroup = 32;

// most: the bits of the group's largest |x|.
__device__ __forceinline__ uint32_t exponent_of(uint32_t most) {
  if (most >= 0x7F800000u) return 255;
  const int e = (int)((most + 0x1FFFFu) >> 23) - 6;
  return e < 1 ? 1 : (uint32_t)e;
}
__device__ __forceinline__ int code_of(float x, uint32_t exponent) {
  const float limit = exponent >= 249 ? 63.f : 127.f;
  const float code = rintf(x * __uint_as_float((254 - exponent) << 23));     // (of 255: not used)
  return exponent == 255 ? 0 : (int)fminf(fmaxf(code, -limit), limit);
}
__device__ __forceinline__ float step_of(uint32_t exponent) { return __uint_as_float(exponent << 23); }
// Byte `at` of four codes as its value.  (E = 255 is an infinity here, and its codes are zeros: NaN.)
__device__ __forceinline__ float coded_value(uint32_t codes, int at, float step) {
  return (float)(int)(int8_t)(codes >> (8 * at)) * step;
}

template <typename T> struct dtype_of;
template <> struct dtype_of<float> { static constexpr int tag = F2CGT_DT_F32; };
template <> struct dtype_of<_Float16> { static constexpr int tag = F2CGT_DT_F16; };
template <> struct dtype_of<__bf16> { static constexpr int tag = F2CGT_DT_BF16; };

// f with a value of the type that the tag stands for.
template <typename F>
int with_type(int dtype, const F& f) {
  if (dtype == F2CGT_DT_F32) return f(float{});
  if (dtype == F2CGT_DT_F16) return f(_Float16{});
  return f(__bf16{});
}

}  // namespace f2cgt
