// Dense layers in 8 bits: rows coded with a scale each, and the product of coded tokens with coded weights.
//
//   scale_i = max(max_j |x_ij|, 1e-30) * fl(1 / 127)       code_ij = rint(x_ij * fl(1 / scale_i)) within +-127
//   out_ij  = (sum_t code_it weight_jt) * fl(scale_i * weight_scale_j) + bias_j, through max(., 0), rounded once
//
// The sum is one of whole numbers: it is exact in 32 bits up to 2^17 - 1 columns whatever the order.
#include "tile_product.hpp"

namespace f2cgt {
namespace {

constexpr float kLeast = 1e-30f;           // (its scale and the reciprocal of that are normal numbers)

struct QuantizeArgs {
  const void* x;
  int8_t* codes;
  float* scales;
  int64_t m, k, ld, stride;
};

// Magnitudes are compared as the whole numbers of their bits: the order is the same, and a NaN is above infinity and stays.
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// What the codes of a row are made with, from its largest magnitude.
struct RowCode {
  float scale, inverse;
  uint32_t keep;                             // no bit where a NaN is among the row's values: its codes are zero
  __device__ __forceinline__ explicit RowCode(uint32_t bits) {
    const float most = __builtin_bit_cast(float, bits);
    scale = (most < kLeast ? kLeast : most) * (1.f / 127.f);
    inverse = 1.f / scale;
    keep = most == most ? ~0u : 0u;
  }
  // rint(x * inverse) in the low byte.  Adding 3 * 2^22 rounds to a whole number in the place of the last bit.  No magnitude
  // is above 127: x <= most, and three roundings on the way are not half a code.  (Infinities: inverse 0, inf * 0 is the NaN without payload.)
  __device__ __forceinline__ uint32_t operator()(float x) const { return __builtin_bit_cast(uint32_t, x * inverse + 12582912.f); }
  __device__ __forceinline__ uint32_t four(float a, float b, float c, float d) const {
    const uint32_t low = __builtin_amdgcn_perm((*this)(b), (*this)(a), 0x0c0c0400), high = __builtin_amdgcn_perm((*this)(d), (*this)(c), 0x04000c0c);
    return (low | high) & keep;
  }
};

template <typename X>
constexpr int piece_values() { return 16 / sizeof(X); }

// V neighbours of a row of k values from column c on, wherever they start in memory (which takes 16 bytes at any address): zeros
// for those behind the row's end, but for a piece that begins there others of the row.  `last`: behind this row is
// nothing that may be read.  One load without a branch around it, so that a caller's loads are under way together.
template <typename X, int V>
__device__ __forceinline__ void load_piece(const X* row, int64_t c, int64_t k, bool last, X (&v)[V]) {
  typedef X values __attribute__((ext_vector_type(V), aligned(sizeof(X))));
  if (k < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c + e < k ? row[c + e] : (X)0.f;
    return;
  }
  const int64_t from = c < k ? c : 0;
  const bool over = last && from + V > k;
  const values p = *reinterpret_cast<const values*>(row + (over ? k - V : from));
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = p[e];
  if (k % V != 0) {
    if (over) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = from + e < k ? row[from + e] : (X)0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = from + e < k ? v[e] : (X)0.f;
  }
}

template <typename X, int V>
__device__ __forceinline__ uint32_t largest(const X (&v)[V], uint32_t most) {
#pragma unroll
  for (int e = 0; e < V; ++e) most = larger(most, magnitude((float)v[e]));
  return most;
}

// A piece's codes, four in a word.
template <int V>
struct Words {
  uint32_t w[V / 4] = {};
  __device__ __forceinline__ Words() {}
  template <typename X>
  __device__ __forceinline__ Words(const RowCode& code, const X (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) w[i] = code.four((float)v[4 * i], (float)v[4 * i + 1], (float)v[4 * i + 2], (float)v[4 * i + 3]);
  }
};

// A row per LANES lanes (16, 64, or 256: a workgroup), read once: up to HELD pieces of 16 bytes a lane stay in registers, what is
// beyond them is read again for the codes.
template <typename X, int LANES, int HELD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a) {
  constexpr int V = piece_values<X>();
  const int t = threadIdx.x, lane = t % LANES;
  __shared__ uint32_t s_most[4];
  for (int64_t r0 = (int64_t)blockIdx.x * (256 / LANES); r0 < a.m; r0 += (int64_t)gridDim.x * (256 / LANES)) {
    const int64_t r = r0 + t / LANES, rr = r < a.m ? r : a.m - 1;
    const bool last = rr == a.m - 1;
    const X* x = static_cast<const X*>(a.x) + rr * a.ld;
    X v[HELD][V];
    uint32_t most = 0;
    auto any = [&](int i) { return i == 0 || i * LANES * V < a.k; };         // (for all lanes)
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (any(i)) load_piece<X, V>(x, (int64_t)(lane + i * LANES) * V, a.k, last, v[i]);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (any(i)) most = largest(v[i], most);
    for (int64_t c = (int64_t)(lane + HELD * LANES) * V; c < a.k; c += LANES * V) {
      X w[V];
      load_piece<X, V>(x, c, a.k, last, w);
      most = largest(w, most);
    }
#pragma unroll
    for (int by = 1; by < (LANES < kWave ? LANES : kWave); by *= 2) most = larger(most, (uint32_t)__shfl_xor((int)most, by));
    if (LANES > kWave) {
      __syncthreads();                         // (of the row before)
      if (t % kWave == 0) s_most[t / kWave] = most;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) most = larger(most, s_most[i]);
    }
    const RowCode code(most);
    if (r >= a.m) continue;
    int8_t* codes = a.codes + r * a.stride;
    auto put = [&](int64_t c, const X (&w)[V]) {
      const Words<V> q(code, w);
      if (c + V <= a.k) {
        typedef uint32_t words __attribute__((ext_vector_type(V / 4), aligned(1)));
        words o;
#pragma unroll
        for (int e = 0; e < V / 4; ++e) o[e] = q.w[e];
        *reinterpret_cast<words*>(codes + c) = o;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c + e < a.k) codes[c + e] = (int8_t)(q.w[e / 4] >> (8 * (e % 4)));
      }
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (any(i)) put((int64_t)(lane + i * LANES) * V, v[i]);
    for (int64_t c = (int64_t)(lane + HELD * LANES) * V; c < a.k; c += LANES * V) {
      X w[V];
      load_piece<X, V>(x, c, a.k, last, w);
      put(c, w);
    }
    if (lane == 0) a.scales[r] = code.scale;
  }
}

template <typename X, int LANES, int HELD>
void launch_quantize(const QuantizeArgs& a, hipStream_t st) {
  const int64_t blocks = ceil_div(a.m, 256 / LANES);
  quantize_rows_kernel<X, LANES, HELD><<<(unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 256, 0, st>>>(a);
}

// As few lanes a row as hold it, but enough waves.  us at 250 000 x 128 fp32 by 16 lanes 25 (6.4 TB/s), by 64 68; 60 000 x 602 by 16 34, by 64 36;
// 16 384 x 1024 by 64 13.5, by 16 22; 4099 x 4096 by 256 14, by 64 22; 4096 x 602 by 64 4.8, by 16 5.9; 33 rows of 4096 by 256 3.8,
// by 64 7.3.  Rows of 16 bits, eight values a piece, hold less: the instructions of pieces that are not there, or not whole, cost more than
// reading those beyond again (60 000 x 602 by 16 lanes 25, eight pieces held 36; 4099 x 4096 by 64 10.9, by 256 11.2, four held 17;
// 16 384 x 8192 by 256 80, by 64 106).
template <typename X>
void quantize(const QuantizeArgs& a, hipStream_t st) {
  constexpr bool kWide = sizeof(X) == 4;
  const int64_t pieces = ceil_div(a.k, piece_values<X>());
  if (pieces <= 32) launch_quantize<X, 16, 2>(a, st);
  else if (pieces <= 128 && a.m > 8192) launch_quantize<X, 16, kWide ? 8 : 2>(a, st);
  else if (pieces <= (kWide ? 256 : 512) && (pieces <= 128 || a.m > 1024)) launch_quantize<X, 64, kWide ? 4 : 2>(a, st);
  else if (pieces <= 1024) launch_quantize<X, 256, kWide ? 4 : 2>(a, st);
  else launch_quantize<X, 256, kWide ? 8 : 2>(a, st);
}

struct LinearArgs {
  Lines x, w;
  const float* x_scales;
  const float* w_scales;
  const float* bias;
  void* out;
  int64_t m, n;
  int dtype, relu, whole;                      // whole: rows of the output start at multiples of four values
};

// scales: of the tokens from row `from` on.
template <int WN>
struct LinearEpilogue {
  const LinearArgs& a;
  const float* scales;
  int64_t from;
  __device__ __forceinline__ void operator()(const float* strip, int64_t row0, int64_t col0, int lane) const {
    if (a.dtype == F2CGT_DT_F32) put<float>(strip, row0, col0, lane);
    else if (a.dtype == F2CGT_DT_F16) put<_Float16>(strip, row0, col0, lane);
    else put<__bf16>(strip, row0, col0, lane);
  }
  template <typename T>
  __device__ __forceinline__ void put(const float* strip, int64_t row0, int64_t col0, int lane) const {
    typedef T four __attribute__((ext_vector_type(4)));
    constexpr int kAcross = WN / 4, kRows = kWave / kAcross;        // lanes along a row, rows at a time
    static_assert(kWave % kAcross == 0, "whole rows at a time");
    const int c = 4 * (lane % kAcross), r0 = lane / kAcross;
    const int64_t col = col0 + c;
    const int in = a.n - col < 4 ? (int)(a.n - col) : 4, rows = a.m - row0 < 32 ? (int)(a.m - row0) : 32;
    if (in <= 0) return;
    const float least = a.relu ? 0.f : -__builtin_inff();           // (a NaN stays one)
    fltx4 scale, bias = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) scale[e] = a.w_scales[e < in ? col + e : col];
    if (a.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = a.bias[e < in ? col + e : col];
    }
    const float* by = scales + (row0 - from);
    T* out = static_cast<T*>(a.out) + row0 * a.n + col;
    auto values = [&](int r) {
      const intx4 sum = *reinterpret_cast<const intx4*>(strip + r * (WN + 4) + c);
      const float of = by[r < rows ? r : rows - 1];
      fltx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = (float)sum[e] * (of * scale[e]) + bias[e];
        v[e] = v[e] <= least ? least : v[e];
      }
      return v;
    };
    if (a.whole) {
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i) {
        const int r = i * kRows + r0;
        const four v = __builtin_convertvector(values(r), four);
        if (r < rows) *reinterpret_cast<four*>(out + r * a.n) = v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i) {
        const int r = i * kRows + r0;
        const four v = __builtin_convertvector(values(r), four);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r < rows && e < in) out[r * a.n + e] = v[e];
      }
    }
  }
};

// The product of coded rows, a tile per workgroup.  It is bound by matrix instructions: 256 x 256 tiles, whose waves read as many
// clocks of LDS as they multiply, take 509 us for 8192 x 8192 -> 8192 (2.16e15 operations a second) and 950 for 16 384 rows, where the
// card's power holds the clock to 1.9 GHz; 57 % of the clocks then issue one.  128 x 128 tiles read LDS for twice as long as they
// multiply, but there are enough of them for fewer rows: 60 001 x 602 -> 128 in 17 us, 4.1 TB/s of the codes, which is its bound.
template <int BM, int BN, int WM, int WN, int GROUPS, int DEEP>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * GROUPS * kWave) void int8_linear_kernel(LinearArgs a) {
  typedef TileProduct<Int8Op, BM, BN, WM, WN, GROUPS> Tile;
  uint32_t i, j;
  tile_of(place_of(blockIdx.x, gridDim.x), (uint32_t)ceil_div(a.m, BM), (uint32_t)ceil_div(a.n, BN), DEEP, i, j);
  __shared__ __attribute__((aligned(128))) char lds0[Tile::kStage], lds1[Tile::kStage];
  Tile::run({lds0, lds1}, a.x, a.w, (int64_t)i * BM, (int64_t)j * BN, LinearEpilogue<WN>{a, a.x_scales, 0});
}

template <int BM, int BN, int WM, int WN, int GROUPS, int DEEP>
void launch_linear(const LinearArgs& a, hipStream_t st) {
  int8_linear_kernel<BM, BN, WM, WN, GROUPS, DEEP>
      <<<(unsigned)(ceil_div(a.m, BM) * ceil_div(a.n, BN)), (BM / WM) * (BN / WN) * GROUPS * kWave, 0, st>>>(a);
}

// ---- rows of few columns, coded where they are multiplied ------------------------------------------------------
// Floating rows of up to 128 L columns: a workgroup codes 64 of them into LDS (16 lanes a row, as quantize_rows_kernel) while the
// weights of its 128 outputs are copied there, and multiplies.  The codes never go through memory, which is the bound: 250 000 x 100
// -> 128 in fp32 51 us, 228 MB at 4.5 TB/s.
template <typename X, int L>
__global__ __launch_bounds__(256) void int8_rows_kernel(LinearArgs a, int64_t ld) {
  constexpr int V = piece_values<X>(), kHeldPieces = 128 * L / (16 * V), kM = 64, kN = 128;
  constexpr int kStripBytes = 32 * (64 + 4) * 4, kCodes = L * (kM + kN) * kLine;
  __shared__ __attribute__((aligned(128))) char lds[kCodes > 4 * kStripBytes ? kCodes : 4 * kStripBytes];
  __shared__ float s_scale[kM];
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int at = lane & 31, side = lane >> 5;
  const uint32_t tiles = (uint32_t)ceil_div(a.n, kN), place = place_of(blockIdx.x, gridDim.x);
  const int64_t row0 = (int64_t)(place / tiles) * kM, col0 = (int64_t)(place % tiles) * kN, k = a.w.bytes;
  char* lds_w = lds + L * kM * kLine;
  // weights: thread t's pieces lie sixteen rows and more apart; those behind a row's end are the row's first one (the codes are zero)
  const int piece = ((t & 7) ^ (t >> 4 & 7)) << 4;
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int i = 0; i < kN / 32; ++i) {
      const int64_t r = col0 + t / 8 + 32 * i, c = l * kLine + piece;
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(a.w.base + (r < a.n ? r : a.n - 1) * a.w.stride + (c < k ? c : 0)),
          (__attribute__((address_space(3))) void*)(lds_w + l * kN * kLine + (wave * kWave + i * 256) * 16), 16, 0, 0);
    }
  const int turn = lane & 15;
  X v[4][kHeldPieces][V];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t r = row0 + 16 * wave + 4 * p + lane / 16;
    const X* x = reinterpret_cast<const X*>(a.x.base) + (r < a.m ? r : a.m - 1) * ld;
#pragma unroll
    for (int i = 0; i < kHeldPieces; ++i) load_piece<X, V>(x, (turn + 16 * i) * V, k, r >= a.m - 1, v[p][i]);
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kHeldPieces; ++i) most = largest(v[p][i], most);
#pragma unroll
    for (int by = 1; by < 16; by *= 2) most = larger(most, (uint32_t)__shfl_xor((int)most, by));
    const RowCode code(most);
    const int r = 16 * wave + 4 * p + lane / 16;
    if (turn == 0) s_scale[r] = code.scale;
#pragma unroll
    for (int i = 0; i < kHeldPieces; ++i) {
      const int c = (turn + 16 * i) * V;
      Words<V> q(code, v[p][i]);
      if (c >= k) q = Words<V>();
      *reinterpret_cast<Words<V>*>(lds + c / kLine * kM * kLine + piece_at(r, c % kLine / 16) + c % 16) = q;
    }
  }
  wait_copies();                            // (the weights: a barrier alone does not wait for copies into LDS)
  __syncthreads();
  const int wi = 32 * (wave & 1), wj = 64 * (wave >> 1);
  intx16 acc[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[j][e] = 0;
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const intx4 fa = *reinterpret_cast<const intx4*>(lds + l * kM * kLine + piece_at(wi + at, 2 * g + side));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const intx4 fb = *reinterpret_cast<const intx4*>(lds_w + l * kN * kLine + piece_at(wj + 32 * j + at, 2 * g + side));
        acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb, fa, acc[j], 0, 0, 0);
      }
    }
  __syncthreads();
  float* strip = reinterpret_cast<float*>(lds + wave * kStripBytes);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      fltx4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = word_of(acc[j][4 * q + e]);
      *reinterpret_cast<fltx4*>(strip + at * 68 + 32 * j + 8 * q + 4 * side) = o;
    }
  __builtin_amdgcn_wave_barrier();
  LinearEpilogue<64>{a, s_scale, row0}(strip, row0 + wi, col0 + wj, lane);
}

// ---- few tokens -----------------------------------------------------------------------------------------
// Up to 48 tokens: the weights are read once, and that is the time.  A workgroup has NT times 16 outputs; its waves share the
// columns, 64 at a time (a 16 x 16 x 64 instruction takes 64 bytes of each of 16 rows), and add their sums in LDS.  Weights and
// codes go from memory to registers, U instructions' worth at a time.  One token of 4096 -> 4096, 16.8 MB: 5.4 us from its
// code (3.1 TB/s), 7.4 from bf16; that is a launch, the latency of the first loads and a sum over waves.
//
// X other than int8_t: up to 16 floating rows are coded here, in each workgroup again, while the first weights are on
// their way: a launch less.  Waves take the rows in turn, HELD pieces of four columns a lane, and leave the codes in LDS.
struct FewArgs {
  LinearArgs l;
  int64_t ld;                                  // of floating rows, in values
};

constexpr int kHeld = 8;
constexpr int kFusedWaves = 16;
constexpr int kFusedBytes = 40960;             // of codes in LDS

__host__ __device__ constexpr int64_t fused_row(int64_t k) { return ceil_div(k, 64) * 64 + 16; }

template <typename X, int MT, int NT, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void int8_few_kernel(FewArgs f) {
  constexpr bool kCoded = sizeof(X) == 1;
  constexpr int U = 4;
  const LinearArgs& a = f.l;
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int at = lane & 15, part = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), k = a.x.bytes;
  const int blocks = (int)ceil_div(k, 64);
  __shared__ uint32_t s_most[WAVES];
  __shared__ float s_scale[MT * 16];
  __shared__ __attribute__((aligned(16))) int s_sum[WAVES][NT][MT * 16][20];
  extern __shared__ __attribute__((aligned(16))) char s_codes[];        // (floating rows: [m][fused_row(k)])
  const char* w[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t row = n0 + 16 * j + at;
    w[j] = a.w.base + (row < a.n ? row : a.n - 1) * a.w.stride;
  }
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = 16 * i + at < a.m ? 16 * i + at : a.m - 1;
    x[i] = kCoded ? a.x.base + row * a.x.stride : s_codes + row * fused_row(k);
  }
  // Pieces behind a row's end: the row's first one; the token's is made zero.
  intx4 next_w[U][NT], next_x[U][MT];
  auto load_w = [&](int first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t c = 64ll * (first + u * WAVES) + 16 * part;
#pragma unroll
      for (int j = 0; j < NT; ++j) next_w[u][j] = *reinterpret_cast<const intx4*>(w[j] + (c < k ? c : 0));
    }
  };
  auto load_x = [&](int first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t c = 64ll * (first + u * WAVES) + 16 * part;
#pragma unroll
      for (int i = 0; i < MT; ++i) next_x[u][i] = *reinterpret_cast<const intx4*>(x[i] + (c < k ? c : 0));
    }
  };
  if constexpr (kCoded) {
    if (blocks > 0) {
      load_w(wave);
      load_x(wave);
    }
  } else {
    // waves in a row's share: `share`; this one is number `sub` of row `row`
    const int share = WAVES / (int)a.m, row = wave / share, sub = wave - row * share;
    const bool mine = row < a.m;
    const int64_t line = fused_row(k);
    const X* from = reinterpret_cast<const X*>(a.x.base) + (mine ? row : 0) * f.ld;
    X v[kHeld][4];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int64_t c = 4ll * (sub * kWave + lane + i * share * kWave);
      if (i == 0 || 4ll * i * share * kWave < line) load_piece<X, 4>(from, c, k, !mine || row == a.m - 1, v[i]);
      else v[i][0] = v[i][1] = v[i][2] = v[i][3] = (X)0.f;
    }
    __builtin_amdgcn_sched_barrier(0);           // (loads come back in their order: the tokens before the weights)
    if (blocks > 0) load_w(wave);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = largest(v[i], most);
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) most = larger(most, (uint32_t)__shfl_xor((int)most, by));
    if (lane == 0) s_most[wave] = most;
    __syncthreads();
    if (mine) {
      for (int i = 0; i < share; ++i) most = larger(most, s_most[row * share + i]);
      const RowCode code(most);
      if (sub == 0 && lane == 0) s_scale[row] = code.scale;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int64_t c = 4ll * (sub * kWave + lane + i * share * kWave);
        if (c < line) *reinterpret_cast<uint32_t*>(s_codes + row * line + c) = c < k ? code.four((float)v[i][0], (float)v[i][1], (float)v[i][2], (float)v[i][3]) : 0u;
      }
    }
    __syncthreads();
  }
  intx4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = intx4{0, 0, 0, 0};
  for (int first = wave; first < blocks; first += U * WAVES) {
    intx4 now_w[U][NT], now_x[U][MT];
    if (!kCoded) load_x(first);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NT; ++j) now_w[u][j] = next_w[u][j];
#pragma unroll
      for (int i = 0; i < MT; ++i) now_x[u][i] = next_x[u][i];
    }
    if (first + U * WAVES < blocks) {
      load_w(first + U * WAVES);
      if (kCoded) load_x(first + U * WAVES);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t in = k - (64ll * (first + u * WAVES) + 16 * part);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        intx4 p = now_x[u][i];
        if (in < 16) {
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = in <= 4 * e ? 0 : in >= 4 * e + 4 ? p[e] : p[e] & ((1 << (8 * ((int)in - 4 * e))) - 1);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now_w[u][j], p, acc[j][i], 0, 0, 0);
      }
    }
  }
  // a lane has, of token `at`, outputs 4 part to 4 part + 3
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) *reinterpret_cast<intx4*>(&s_sum[wave][j][16 * i + at][4 * part]) = acc[j][i];
  __syncthreads();
  for (int i = t; i < MT * NT * 256; i += WAVES * kWave) {
    const int row = i / (NT * 16), c = i % (NT * 16);
    const int64_t col = n0 + c;
    if (row >= a.m || col >= a.n) continue;
    int sum = 0;
#pragma unroll
    for (int j = 0; j < WAVES; ++j) sum += s_sum[j][c / 16][row][c % 16];
    const float by = kCoded ? a.x_scales[row] : s_scale[row];
    float v = (float)sum * (by * a.w_scales[col]);
    if (a.bias != nullptr) v += a.bias[col];
    if (a.relu && v <= 0.f) v = 0.f;
    store_value(a.out, a.dtype, row * a.n + col, v);
  }
}

// Whether floating rows are coded by the product's own workgroups.  us, so and by two launches: 1 x 4096 -> 4096 7.2 and 9.1,
// 8 x 4096 -> 4096 9.1 and 9.8, 16 x 1000 -> 300 6.1 and 8.1; but 1 x 4096 -> 16384 23 and 18.6 (a thousand workgroups code).
bool fused(int64_t m, int64_t n, int64_t k) {
  if (m < 1 || m > 16 || n >= 8192 || m * fused_row(k) > kFusedBytes) return false;
  return ceil_div(fused_row(k), 4 * kWave * (kFusedWaves / m)) <= kHeld;
}

// Whether rows of few columns are coded where they are multiplied, once for every 128 outputs.  us, so and by two launches:
// 1024 x 128 -> 256 6.3 and 8.6, 20 000 x 100 -> 47 9.1 and 11.1, 250 000 x 100 -> 128 51 and 57, bf16 36 and 62,
// 250 000 x 128 -> 256 84 and 98, 30 000 x 128 -> 512 20 and 23; but 30 000 x 250 -> 512 37 and 29, 100 000 x 200 -> 1024 188 and 140.
// (Without columns there may be no weights to copy.)
bool rows_fused(int64_t m, int64_t n, int64_t k) { return k >= 1 && k <= 256 && n * ceil_div(k, kLine) <= 512 && ceil_div(m, 64) * ceil_div(n, 128) < (1ll << 24); }

template <typename X>
void launch_rows(const FewArgs& f, hipStream_t st) {
  const unsigned grid = (unsigned)(ceil_div(f.l.m, 64) * ceil_div(f.l.n, 128));
  if (f.l.w.bytes <= kLine) int8_rows_kernel<X, 1><<<grid, 256, 0, st>>>(f.l, f.ld);
  else int8_rows_kernel<X, 2><<<grid, 256, 0, st>>>(f.l, f.ld);
}

template <typename X>
void launch_fused(const FewArgs& f, hipStream_t st) {
  int8_few_kernel<X, 1, 1, kFusedWaves><<<(unsigned)ceil_div(f.l.n, 16), kFusedWaves * kWave, (size_t)(f.l.m * fused_row(f.l.x.bytes)), st>>>(f);
}

int64_t code_row(int64_t k) { return ceil_div(k, 16) * 16; }

int check_sizes(const char* what, int64_t m, int64_t n, int64_t k) {
  F2CGT_REQUIRE(m >= 0 && n >= 0 && k >= 0, F2CGT_E_INVALID, "%s: sizes must not be negative", what);
  F2CGT_REQUIRE(m < (1ll << 30) && n < (1ll << 22) && k < (1ll << 17), F2CGT_E_UNSUPPORTED,
                "%s: at most 2^30 - 1 rows, 2^22 - 1 outputs and 2^17 - 1 columns (where 32-bit sums are exact)", what);
  return 0;
}

template <int MT, int NT, int WAVES>
void launch_few(const LinearArgs& a, hipStream_t st) {
  int8_few_kernel<int8_t, MT, NT, WAVES><<<(unsigned)ceil_div(a.n, 16 * NT), WAVES * kWave, 0, st>>>(FewArgs{a, 0});
}

// Which kernel: times in us at rows x columns -> outputs (bf16 results, four sets of weights in turn).
//   few tokens or 64 x 64 tiles: 1 x 4096 -> 4096 5.4 and 12.1, 16 x 4096 -> 4096 6.7 and 12.4, 32 x 4096 -> 4096 8.3 and 13.0,
//     48 x 4096 -> 4096 11.5 and 13.2; but 33 x 4096 -> 16384 24 and 17.5, 32 x 1024 -> 16384 12.9 and 7.5, 64 x 602 -> 128
//     6.1 and 4.8
//   of few tokens 16 or 8 waves: 1 x 4096 -> 4096 5.4 and 6.2, 1 x 128 -> 256 4.2 and 3.7, 24 x 4096 -> 4096 7.5 and 8.7, but
//     48 rows 16.2 and 11.5 (registers); 32 outputs a workgroup or 16: 16 x 2048 -> 16384 8.8 and 10.7, 16 x 4096 -> 4096 8.4 and 7.8
//   64 x 64 tiles by four groups of waves or by two, 64 x 128 or 128 x 128 tiles: 256 x 4096 -> 4096 12.8, 14.3, 20.6, 24.0;
//     33 x 4096 -> 16384 15.8, 15.2, 21.2, 23.4; 490 x 1135 -> 9698 40, 26.7, 20.3, 21.2; 2048 x 2048 -> 2048 31, 20.5, 15.7,
//     17.0; 60001 x 602 -> 128, the last two 18.5 and 17.1; 4099 x 4096 -> 4096 102 and 96
//   (tests/test_gpu_dense_forms.py and test_gpu_int8_linear.py have a shape for each)
//   128 x 128 or 256 x 256: 8192 x 8192 -> 8192 586 and 509, 4099 x 4096 -> 4096 (272 large tiles for 256 CUs) 96 and 124
int linear(const char* what, LinearArgs a, hipStream_t st) {
  if (a.m == 0 || a.n == 0) return 0;
  const int64_t m = a.m, n = a.n, k = a.x.bytes, cus = num_cus();
  if (m <= 16) {
    if (n >= 8192) launch_few<1, 2, 8>(a, st);
    else if (k >= 2048) launch_few<1, 1, 16>(a, st);
    else launch_few<1, 1, 8>(a, st);
    return launch_status(what);
  }
  if (m <= 48 && n <= 4096 && k >= 2048) {
    if (m <= 32) launch_few<2, 1, 16>(a, st);
    else launch_few<3, 1, 8>(a, st);
    return launch_status(what);
  }
  a.whole = n % 4 == 0 && aligned(a.out, 4 * type_size(a.dtype));
  // A few rows behind the last whole 128: where they begin another round of tiles, they go to the kernel for few tokens
  // (4099 x 4096 -> 4096: 96 us in one launch, 75 in two).  A step of a round of tiles is 0.7 us, that kernel reads 4e6 codes a us.
  const int64_t rest = m % 128;
  if (rest > 0 && rest <= 16 && m > 128) {
    auto rounds = [&](int64_t rows) { return ceil_div(ceil_div(rows, 128) * ceil_div(n, 128), cus); };
    if (rounds(m) > rounds(m - rest) && ceil_div(k, kLine) * 0.7 > 4. + n * k / 4e6) {
      LinearArgs tail = a;
      const int64_t done = m - rest;
      tail.x.base += done * a.x.stride;
      tail.x.rows = tail.m = rest;
      tail.x_scales += done;
      tail.out = static_cast<char*>(a.out) + done * n * type_size(a.dtype);
      a.x.rows = a.m = done;
      if (int rc = linear(what, tail, st)) return rc;
      return linear(what, a, st);
    }
  }
  const int64_t large = ceil_div(m, 256) * ceil_div(n, 256), middle = ceil_div(m, 128) * ceil_div(n, 128);
  const int64_t small = ceil_div(m, 64) * ceil_div(n, 128);
  F2CGT_REQUIRE(middle < (1ll << 23), F2CGT_E_UNSUPPORTED, "%s: too many tiles", what);     // (a launch has 2^32 threads at most)
  // a round of large tiles is as long as 3.5 rounds of middle ones
  if (k >= 1024 && large >= cus && 7 * ceil_div(large, cus) * cus <= 2 * middle) launch_linear<256, 256, 128, 64, 1, 4>(a, st);
  else if (2 * middle >= 3 * cus) launch_linear<128, 128, 64, 32, 1, 8>(a, st);
  else if (small >= cus) launch_linear<64, 128, 32, 32, 1, 8>(a, st);
  else if (ceil_div(m, 64) * ceil_div(n, 64) > cus) launch_linear<64, 64, 32, 32, 2, 8>(a, st);
  else launch_linear<64, 64, 32, 32, 4, 8>(a, st);
  return launch_status(what);
}

int check_codes(const char* what, const int8_t* codes, int64_t stride, int64_t k, const char* name) {
  if (k == 0) return 0;
  F2CGT_REQUIRE(codes != nullptr, F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(stride % 16 == 0 && stride >= k && stride < (1ll << 23) && aligned(codes, 16), F2CGT_E_UNSUPPORTED,
                "%s: rows of %s must start at multiples of 16 bytes, less than 2^23 apart, and not overlap", what, name);
  return 0;
}

}  // namespace
}  // namespace f2cgt

using namespace f2cgt;

extern "C" int f2cgt_quantize_rows(const void* x, int dtype, int64_t ld, int8_t* codes, int64_t code_stride, float* scales,
                                   int64_t m, int64_t k, void* stream) {
  const char* what = "quantize_rows";
  if (int rc = check_sizes(what, m, 0, k)) return rc;
  F2CGT_REQUIRE(dense_type(dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 rows only", what);
  F2CGT_REQUIRE(m <= 1 || ld >= k, F2CGT_E_INVALID, "%s: rows overlap", what);
  F2CGT_REQUIRE(code_stride >= k, F2CGT_E_INVALID, "%s: rows of codes overlap", what);
  if (m == 0) return 0;
  F2CGT_REQUIRE(scales && (k == 0 || (x && codes)), F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(aligned(x, type_size(dtype)), F2CGT_E_INVALID, "%s: misaligned rows", what);
  QuantizeArgs a{x, codes, scales, m, k, ld, code_stride};
  hipStream_t st = as_stream(stream);
  if (dtype == F2CGT_DT_F32) quantize<float>(a, st);
  else if (dtype == F2CGT_DT_F16) quantize<_Float16>(a, st);
  else quantize<__bf16>(a, st);
  return launch_status(what);
}

extern "C" int f2cgt_int8_linear(const int8_t* codes, int64_t code_stride, const float* scales, const int8_t* weight,
                                 int64_t weight_stride, const float* weight_scales, const float* bias, void* out, int out_dtype,
                                 int64_t m, int64_t n, int64_t k, int relu, void* stream) {
  const char* what = "int8_linear";
  if (int rc = check_sizes(what, m, n, k)) return rc;
  F2CGT_REQUIRE(dense_type(out_dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 output only", what);
  if (m == 0 || n == 0) return 0;
  F2CGT_REQUIRE(scales && weight_scales && out, F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(aligned(out, type_size(out_dtype)), F2CGT_E_INVALID, "%s: misaligned output", what);
  if (int rc = check_codes(what, codes, code_stride, k, "codes")) return rc;
  if (int rc = check_codes(what, weight, weight_stride, k, "weights")) return rc;
  LinearArgs a{{reinterpret_cast<const char*>(codes), code_stride, m, k}, {reinterpret_cast<const char*>(weight), weight_stride, n, k},
               scales, weight_scales, bias, out, m, n, out_dtype, relu, 0};
  return linear(what, a, as_stream(stream));
}

// The codes of the tokens, then their scales.
extern "C" int64_t f2cgt_quantized_linear_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k < 0 || fused(m, n, k) || rows_fused(m, n, k)) return 0;
  return m * code_row(k) + 4 * m;
}

extern "C" int f2cgt_quantized_linear(const void* x, int dtype, int64_t ld, const int8_t* weight, int64_t weight_stride,
                                      const float* weight_scales, const float* bias, void* out, void* workspace,
                                      int64_t workspace_bytes, int64_t m, int64_t n, int64_t k, int relu, void* stream) {
  const char* what = "quantized_linear";
  if (int rc = check_sizes(what, m, n, k)) return rc;
  F2CGT_REQUIRE(dense_type(dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 rows only", what);
  F2CGT_REQUIRE(m <= 1 || ld >= k, F2CGT_E_INVALID, "%s: rows overlap", what);
  if (m == 0 || n == 0) return 0;
  F2CGT_REQUIRE(weight_scales && out && (k == 0 || x), F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(aligned(out, type_size(dtype)) && aligned(x, type_size(dtype)), F2CGT_E_INVALID, "%s: misaligned rows", what);
  if (int rc = check_codes(what, weight, weight_stride, k, "weights")) return rc;
  const FewArgs f{{{static_cast<const char*>(x), 0, m, k}, {reinterpret_cast<const char*>(weight), weight_stride, n, k}, nullptr,
                   weight_scales, bias, out, m, n, dtype, relu, n % 4 == 0 && aligned(out, 4 * type_size(dtype))}, ld};
  hipStream_t st = as_stream(stream);
  if (fused(m, n, k)) {
    if (dtype == F2CGT_DT_F32) launch_fused<float>(f, st);
    else if (dtype == F2CGT_DT_F16) launch_fused<_Float16>(f, st);
    else launch_fused<__bf16>(f, st);
    return launch_status(what);
  }
  if (rows_fused(m, n, k)) {
    if (dtype == F2CGT_DT_F32) launch_rows<float>(f, st);
    else if (dtype == F2CGT_DT_F16) launch_rows<_Float16>(f, st);
    else launch_rows<__bf16>(f, st);
    return launch_status(what);
  }
  F2CGT_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= f2cgt_quantized_linear_workspace_bytes(m, n, k),
                F2CGT_E_INVALID, "%s: workspace too small or misaligned", what);
  int8_t* codes = static_cast<int8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + m * code_row(k));
  if (int rc = f2cgt_quantize_rows(x, dtype, ld, codes, code_row(k), scales, m, k, stream)) return rc;
  LinearArgs a{{reinterpret_cast<const char*>(codes), code_row(k), m, k}, {reinterpret_cast<const char*>(weight), weight_stride, n, k},
               scales, weight_scales, bias, out, m, n, dtype, relu, 0};
  return linear(what, a, st);
}
