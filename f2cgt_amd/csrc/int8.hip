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
  int dtype;
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int by = 32; by > 0; by /= 2) {
    const float o = __shfl_xor(v, by);
    v = o > v || o != o ? o : v;             // a NaN stays
  }
  return v;
}

__device__ __forceinline__ int code_of(float x, float inverse) {
  const float q = rintf(x * inverse);
  return q != q ? 0 : (int)fminf(fmaxf(q, -127.f), 127.f);
}

// A wave per row.
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave; r < a.m; r += (int64_t)gridDim.x * 4) {
    const int64_t from = r * a.ld;
    float most = 0.f;
    for (int64_t c = lane; c < a.k; c += kWave) {
      const float v = fabsf(load_value(a.x, a.dtype, from + c));
      most = v > most || v != v ? v : most;
    }
    most = wave_max(most);
    const float scale = (most < kLeast ? kLeast : most) * (1.f / 127.f);
    const float inverse = 1.f / scale;
    for (int64_t c = lane; c < a.k; c += kWave)
      a.codes[r * a.stride + c] = (int8_t)code_of(load_value(a.x, a.dtype, from + c), inverse);
    if (lane == 0) a.scales[r] = scale;
  }
}

struct LinearArgs {
  Lines x, w;
  const float* x_scales;
  const float* w_scales;
  const float* bias;
  void* out;
  int64_t m, n;
  int dtype, relu;
};

template <int WN>
struct LinearEpilogue {
  const LinearArgs& a;
  __device__ __forceinline__ void operator()(const float* strip, int64_t row0, int64_t col0, int lane) const {
    for (int i = lane; i < 32 * WN; i += kWave) {
      const int64_t row = row0 + i / WN, col = col0 + i % WN;
      if (row >= a.m || col >= a.n) continue;
      const int sum = __builtin_bit_cast(int, strip[(i / WN) * (WN + 4) + i % WN]);
      float v = (float)sum * (a.x_scales[row] * a.w_scales[col]);
      if (a.bias != nullptr) v += a.bias[col];
      if (a.relu && v <= 0.f) v = 0.f;       // (a NaN stays one)
      store_value(a.out, a.dtype, row * a.n + col, v);
    }
  }
};

__global__ __launch_bounds__(256) void int8_linear_kernel(LinearArgs a) {
  typedef TileProduct<Int8Op, 64, 64, 32, 32> Tile;
  __shared__ __attribute__((aligned(128))) char lds[Tile::kLds];
  Tile::run(lds, a.x, a.w, (int64_t)blockIdx.x * 64, (int64_t)blockIdx.y * 64, LinearEpilogue<32>{a});
}

int64_t code_row(int64_t k) { return ceil_div(k, 16) * 16; }

int check_sizes(const char* what, int64_t m, int64_t n, int64_t k) {
  F2CGT_REQUIRE(m >= 0 && n >= 0 && k >= 0, F2CGT_E_INVALID, "%s: sizes must not be negative", what);
  F2CGT_REQUIRE(m < (1ll << 30) && n < (1ll << 22) && k < (1ll << 17), F2CGT_E_UNSUPPORTED,
                "%s: at most 2^30 - 1 rows, 2^22 - 1 outputs and 2^17 - 1 columns (where 32-bit sums are exact)", what);
  return 0;
}

int linear(const char* what, const LinearArgs& a, hipStream_t st) {
  if (a.m == 0 || a.n == 0) return 0;
  const dim3 grid((unsigned)ceil_div(a.m, 64), (unsigned)ceil_div(a.n, 64));
  F2CGT_REQUIRE(grid.y <= 65535, F2CGT_E_UNSUPPORTED, "%s: too many tiles", what);
  int8_linear_kernel<<<grid, 256, 0, st>>>(a);
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
  QuantizeArgs a{x, codes, scales, m, k, ld, code_stride, dtype};
  const int64_t blocks = ceil_div(m, 4);
  quantize_rows_kernel<<<(unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 256, 0, as_stream(stream)>>>(a);
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
               scales, weight_scales, bias, out, m, n, out_dtype, relu};
  return linear(what, a, as_stream(stream));
}

// The codes of the tokens, then their scales.
extern "C" int64_t f2cgt_quantized_linear_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k < 0) return 0;
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
  F2CGT_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= f2cgt_quantized_linear_workspace_bytes(m, n, k),
                F2CGT_E_INVALID, "%s: workspace too small or misaligned", what);
  int8_t* codes = static_cast<int8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + m * code_row(k));
  if (int rc = f2cgt_quantize_rows(x, dtype, ld, codes, code_row(k), scales, m, k, stream)) return rc;
  LinearArgs a{{reinterpret_cast<const char*>(codes), code_row(k), m, k}, {reinterpret_cast<const char*>(weight), weight_stride, n, k},
               scales, weight_scales, bias, out, m, n, dtype, relu};
  return linear(what, a, as_stream(stream));
}
