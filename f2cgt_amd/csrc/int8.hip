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

__device__ __forceinline__ float scale_of(float most) { return (most < kLeast ? kLeast : most) * (1.f / 127.f); }

__device__ __forceinline__ int code_of(float x, float inverse) {
  const float q = rintf(x * inverse);
  return q != q ? 0 : (int)fminf(fmaxf(q, -127.f), 127.f);
}

// V neighbours of a row, wherever it starts (memory takes 16 bytes at any address).
template <typename X>
struct Piece {
  static constexpr int kEach = 16 / sizeof(X);
  typedef X Values __attribute__((ext_vector_type(kEach), aligned(sizeof(X))));
  typedef int8_t Codes __attribute__((ext_vector_type(kEach), aligned(1)));
};

template <typename X>
__device__ __forceinline__ void load_piece(const X* row, int64_t c, int64_t k, float (&v)[16 / sizeof(X)]) {
  constexpr int V = 16 / sizeof(X);
  if (c + V <= k) {
    const typename Piece<X>::Values p = *reinterpret_cast<const typename Piece<X>::Values*>(row + c);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)p[e];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c + e < k ? (float)row[c + e] : 0.f;
  }
}

template <int V>
__device__ __forceinline__ float largest(const float (&v)[V], float most) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float o = fabsf(v[e]);
    most = o > most || o != o ? o : most;    // a NaN stays
  }
  return most;
}

// A row per LANES lanes (16, 64, or 256: a workgroup), read once: up to HELD pieces of 16 bytes a lane stay in registers, what is
// beyond them is read again for the codes.
template <typename X, int LANES, int HELD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a) {
  constexpr int V = Piece<X>::kEach;
  const int t = threadIdx.x, lane = t % LANES;
  __shared__ float s_most[4];
  for (int64_t r0 = (int64_t)blockIdx.x * (256 / LANES); r0 < a.m; r0 += (int64_t)gridDim.x * (256 / LANES)) {
    const int64_t r = r0 + t / LANES, rr = r < a.m ? r : a.m - 1;
    const X* x = static_cast<const X*>(a.x) + rr * a.ld;
    float v[HELD][V];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < HELD; ++i) load_piece<X>(x, (int64_t)(lane + i * LANES) * V, a.k, v[i]);
#pragma unroll
    for (int i = 0; i < HELD; ++i) most = largest<V>(v[i], most);
    for (int64_t c = (int64_t)(lane + HELD * LANES) * V; c < a.k; c += LANES * V) {
      float w[V];
      load_piece<X>(x, c, a.k, w);
      most = largest<V>(w, most);
    }
#pragma unroll
    for (int by = 1; by < (LANES < kWave ? LANES : kWave); by *= 2) {
      const float o = __shfl_xor(most, by);
      most = o > most || o != o ? o : most;
    }
    if (LANES > kWave) {
      __syncthreads();                         // (of the row before)
      if (t % kWave == 0) s_most[t / kWave] = most;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float o = s_most[i];
        most = o > most || o != o ? o : most;
      }
    }
    const float scale = scale_of(most), inverse = 1.f / scale;
    if (r >= a.m) continue;
    int8_t* codes = a.codes + r * a.stride;
    auto put = [&](int64_t c, const float (&w)[V]) {
      if (c + V <= a.k) {
        typename Piece<X>::Codes q;
#pragma unroll
        for (int e = 0; e < V; ++e) q[e] = (int8_t)code_of(w[e], inverse);
        *reinterpret_cast<typename Piece<X>::Codes*>(codes + c) = q;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c + e < a.k) codes[c + e] = (int8_t)code_of(w[e], inverse);
      }
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) put((int64_t)(lane + i * LANES) * V, v[i]);
    for (int64_t c = (int64_t)(lane + HELD * LANES) * V; c < a.k; c += LANES * V) {
      float w[V];
      load_piece<X>(x, c, a.k, w);
      put(c, w);
    }
    if (lane == 0) a.scales[r] = scale;
  }
}

template <typename X, int LANES, int HELD>
void launch_quantize(const QuantizeArgs& a, hipStream_t st) {
  const int64_t blocks = ceil_div(a.m, 256 / LANES);
  quantize_rows_kernel<X, LANES, HELD><<<(unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 256, 0, st>>>(a);
}

template <typename X>
void quantize(const QuantizeArgs& a, hipStream_t st) {
  const int64_t pieces = ceil_div(a.k, Piece<X>::kEach);
  const bool spread = a.m <= 2048 && pieces > 64;
  if (!spread && pieces <= 32) launch_quantize<X, 16, 2>(a, st);
  else if (!spread && pieces <= 64) launch_quantize<X, 16, 4>(a, st);
  else if (!spread && pieces <= 256) launch_quantize<X, 64, 4>(a, st);
  else if (!spread && pieces <= 512) launch_quantize<X, 64, 8>(a, st);
  else if (pieces <= 512) launch_quantize<X, 256, 2>(a, st);
  else launch_quantize<X, 256, 8>(a, st);
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

template <int WN>
struct LinearEpilogue {
  const LinearArgs& a;
  __device__ __forceinline__ void operator()(const float* strip, int64_t row0, int64_t col0, int lane) const {
    constexpr int kAcross = WN / 4, kRows = kWave / kAcross;        // lanes along a row, rows at a time
    static_assert(kWave % kAcross == 0, "whole rows at a time");
    const int c = 4 * (lane % kAcross);
    const int64_t col = col0 + c;
    const int in = a.n - col < 4 ? (int)(a.n - col) : 4;
    fltx4 scale = {0.f, 0.f, 0.f, 0.f}, bias = scale;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < in) {
        scale[e] = a.w_scales[col + e];
        if (a.bias != nullptr) bias[e] = a.bias[col + e];
      }
#pragma unroll
    for (int i = 0; i < 32 / kRows; ++i) {
      const int r = i * kRows + lane / kAcross;
      const int64_t row = row0 + r;
      if (row >= a.m || in <= 0) continue;
      const intx4 sum = *reinterpret_cast<const intx4*>(strip + r * (WN + 4) + c);
      const float by = a.x_scales[row];
      fltx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = (float)sum[e] * (by * scale[e]);
        if (a.bias != nullptr) v[e] += bias[e];
        if (a.relu && v[e] <= 0.f) v[e] = 0.f;                      // (a NaN stays one)
      }
      if (a.whole) {
        store_four(a.out, a.dtype, row * a.n + col, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < in) store_value(a.out, a.dtype, row * a.n + col + e, v[e]);
      }
    }
  }
};

template <int BM, int BN, int WM, int WN, int STAGES, int GROUPS, int DEEP>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * GROUPS * kWave) void int8_linear_kernel(LinearArgs a) {
  typedef TileProduct<Int8Op, BM, BN, WM, WN, STAGES, GROUPS> Tile;
  uint32_t i, j;
  tile_of(place_of(blockIdx.x, gridDim.x), (uint32_t)ceil_div(a.m, BM), (uint32_t)ceil_div(a.n, BN), DEEP, i, j);
  __shared__ __attribute__((aligned(128))) char lds0[Tile::kStage], lds1[Tile::kStage];
  if constexpr (STAGES == 2) {
    Tile::run({lds0, lds1}, a.x, a.w, (int64_t)i * BM, (int64_t)j * BN, LinearEpilogue<WN>{a});
  } else {
    __shared__ __attribute__((aligned(128))) char lds2[Tile::kStage], lds3[Tile::kStage];
    Tile::run({lds0, lds1, lds2, lds3}, a.x, a.w, (int64_t)i * BM, (int64_t)j * BN, LinearEpilogue<WN>{a});
  }
}

template <int BM, int BN, int WM, int WN, int STAGES, int GROUPS, int DEEP>
void launch_linear(const LinearArgs& a, hipStream_t st) {
  int8_linear_kernel<BM, BN, WM, WN, STAGES, GROUPS, DEEP>
      <<<(unsigned)(ceil_div(a.m, BM) * ceil_div(a.n, BN)), (BM / WM) * (BN / WN) * GROUPS * kWave, 0, st>>>(a);
}

// ---- few tokens -----------------------------------------------------------------------------------------
// Up to 64 tokens: the weights are read once, and that is the time.  A workgroup has NT times 16 outputs; its waves share the
// columns, 64 at a time (a 16 x 16 x 64 instruction takes 64 bytes of each of 16 rows), and add their sums in LDS.  Weights and
// codes go from memory to registers, U instructions' worth at a time.
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
  __shared__ float s_most[WAVES], s_scale[MT * 16];
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
  if (blocks > 0) load_w(wave);
  if constexpr (kCoded) {
    if (blocks > 0) load_x(wave);
  } else {
    // waves in a row's share: `share`; this one is number `sub` of row `row`
    const int share = WAVES / (int)a.m, row = wave / share, sub = wave - row * share;
    const bool mine = row < a.m;
    const int64_t line = fused_row(k);
    typedef X four __attribute__((ext_vector_type(4), aligned(sizeof(X))));
    const X* from = reinterpret_cast<const X*>(a.x.base) + (mine ? row : 0) * f.ld;
    float v[kHeld][4];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int64_t c = 4ll * (sub * kWave + lane + i * share * kWave);
      if (c + 4 <= k) {
        const four p = *reinterpret_cast<const four*>(from + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = (float)p[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = c + e < k ? (float)from[c + e] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = largest<4>(v[i], most);
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
      const float o = __shfl_xor(most, by);
      most = o > most || o != o ? o : most;
    }
    if (lane == 0) s_most[wave] = most;
    __syncthreads();
    if (mine) {
      for (int i = 0; i < share; ++i) {
        const float o = s_most[row * share + i];
        most = o > most || o != o ? o : most;
      }
      const float scale = scale_of(most), inverse = 1.f / scale;
      if (sub == 0 && lane == 0) s_scale[row] = scale;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int64_t c = 4ll * (sub * kWave + lane + i * share * kWave);
        if (c < line) {
          int word = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) word |= (code_of(v[i][e], inverse) & 255) << (8 * e);
          *reinterpret_cast<int*>(s_codes + row * line + c) = word;       // (zeros behind the row's end)
        }
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

// Whether floating rows are coded by the product's own workgroups.
bool fused(int64_t m, int64_t k) {
  if (m < 1 || m > 16 || m * fused_row(k) > kFusedBytes) return false;
  return ceil_div(fused_row(k), 4 * kWave * (kFusedWaves / m)) <= kHeld;
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
  F2CGT_REQUIRE(ceil_div(m, 64) * ceil_div(n, 64) < (1ll << 24), F2CGT_E_UNSUPPORTED, "%s: too many tiles", what);
  const int64_t large = ceil_div(m, 256) * ceil_div(n, 256), middle = ceil_div(m, 128) * ceil_div(n, 128);
  const int64_t small = ceil_div(m, 64) * ceil_div(n, 128);
  // a round of large tiles is as long as 3.5 rounds of middle ones
  if (k >= 1024 && large >= cus && 7 * ceil_div(large, cus) * cus <= 2 * middle) launch_linear<256, 256, 128, 64, 2, 1, 4>(a, st);
  else if (2 * middle >= 3 * cus) launch_linear<128, 128, 64, 32, 2, 1, 8>(a, st);
  else if (small >= cus) launch_linear<64, 128, 32, 32, 2, 1, 8>(a, st);
  else if (ceil_div(m, 64) * ceil_div(n, 64) > cus) launch_linear<64, 64, 32, 32, 2, 2, 8>(a, st);
  else launch_linear<64, 64, 32, 32, 2, 4, 8>(a, st);
  return launch_status(what);
}

int check_codes(const char* what, const int8_t* codes, int64_t stride, int64_t k, const char* name) {
  if (k == 0) return 0;
  F2CGT_REQUIRE(codes != nullptr, F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(stride % 16 == 0 && stride >= k && aligned(codes, 16), F2CGT_E_UNSUPPORTED,
                "%s: rows of %s must start at multiples of 16 bytes and not overlap", what, name);
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
  if (m <= 0 || n <= 0 || k < 0 || fused(m, k)) return 0;
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
  if (fused(m, k)) {
    const FewArgs f{{{static_cast<const char*>(x), 0, m, k}, {reinterpret_cast<const char*>(weight), weight_stride, n, k}, nullptr,
                     weight_scales, bias, out, m, n, dtype, relu, 0}, ld};
    if (dtype == F2CGT_DT_F32) launch_fused<float>(f, as_stream(stream));
    else if (dtype == F2CGT_DT_F16) launch_fused<_Float16>(f, as_stream(stream));
    else launch_fused<__bf16>(f, as_stream(stream));
    return launch_status(what);
  }
  F2CGT_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= f2cgt_quantized_linear_workspace_bytes(m, n, k),
                F2CGT_E_INVALID, "%s: workspace too small or misaligned", what);
  int8_t* codes = static_cast<int8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + m * code_row(k));
  if (int rc = f2cgt_quantize_rows(x, dtype, ld, codes, code_row(k), scales, m, k, stream)) return rc;
  LinearArgs a{{reinterpret_cast<const char*>(codes), code_row(k), m, k}, {reinterpret_cast<const char*>(weight), weight_stride, n, k},
               scales, weight_scales, bias, out, m, n, dtype, relu, 0};
  return linear(what, a, as_stream(stream));
}
