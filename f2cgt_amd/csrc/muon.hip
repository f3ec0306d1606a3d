// An update made orthogonal by Newton-Schulz products, and the optimiser's step around it.
//
//   X = U / (|U|_F + 1e-7), its shorter side as rows;  then `steps` times
//   G = X X^T,  P = a I + b G + c G G,  X = P X
//
// which takes every singular value s of X through s (a + b s^2 + c s^4) and leaves the vectors alone.  What small singular
// values there are grow by a factor a in each step (480 in five), and so does what rounding adds to them: operands of
// eleven bits leave 2 to 4 % of error in updates of low rank, so all operands are two fp16 planes (tile_product.hpp), 22 bits
// and more, with fp32 sums; the result is as near to float64 as fp32 products are, at three fp16 instructions per product.
//
// Planes hold kScale times their number: entries of an n x n matrix of norm one are about 1 / n, too near to the least
// fp16 numbers for a second plane; all numbers stay below 65504 / kScale (the entry points refuse coefficients that would not).
#include "tile_product.hpp"

namespace f2cgt {
namespace {

constexpr float kScale = 8192.f;
constexpr double kMost = 7.5;                  // of the polynomial's values and of what it multiplies
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
  float momentum, keep, size;                  // weights: keep * w - size * o; results: keep 0, size -1
  double* partial;                             // [count][parts]
  int parts;
  char* x;                                     // [count][r] lines of X
  char* xt[2];                                 // [count][l] lines of X^T
  char* g;                                     // [count][r] lines of G
  char* p;                                     // of P
  float a, b, c;
};

// The update's value i: the gradient, or what the momentum makes of it (held: after this step's change).
__device__ __forceinline__ float update_of(const MuonArgs& a, float grad, float held) {
  return a.nesterov ? a.momentum * held + (1.f - a.momentum) * grad : held;
}

// Momenta, and the sum of squares of the updates by parts, in 64 bits (a square of an fp32 number may be none).
__global__ __launch_bounds__(256) void muon_norm_kernel(MuonArgs a) {
  const int64_t count = a.s.rows * a.s.cols, z = blockIdx.y;
  const void* u = a.at.u[z];
  float* held = a.at.held[z];
  double sum = 0.;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float v = load_value(u, a.u_dtype, i);
    if (held != nullptr) {
      const float h = a.momentum * held[i] + (1.f - a.momentum) * v;
      held[i] = h;
      v = update_of(a, v, h);
    }
    sum += (double)v * (double)v;
  }
  __shared__ double s_sum[4];
#pragma unroll
  for (int by = 32; by > 0; by /= 2) sum += __shfl_xor(sum, by);
  if ((threadIdx.x & (kWave - 1)) == 0) s_sum[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.partial[z * a.parts + blockIdx.x] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

__device__ __forceinline__ void put_split(char* row, int64_t c, float v) {
  const _Float16 hi = (_Float16)v;
  const _Float16 lo = (_Float16)(v - (float)hi);
  char* line = row + (c >> 5) * kLine + 2 * (c & 31);
  *reinterpret_cast<_Float16*>(line) = hi;
  *reinterpret_cast<_Float16*>(line + 64) = lo;
}

// The update of length one in planes, both ways round: a 32 x 32 tile of the caller's matrix per workgroup.
__global__ __launch_bounds__(256) void muon_split_kernel(MuonArgs a) {
  __shared__ double s_sum[4];
  __shared__ float s_tile[32][33];
  const int t = threadIdx.x;
  const int64_t z = blockIdx.z;
  double sum = 0.;
  for (int i = t; i < a.parts; i += 256) sum += a.partial[z * a.parts + i];
#pragma unroll
  for (int by = 32; by > 0; by /= 2) sum += __shfl_xor(sum, by);
  if ((t & (kWave - 1)) == 0) s_sum[t / kWave] = sum;
  __syncthreads();
  const double norm = sqrt((s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]));
  const float scale = (float)(kScale / (norm + 1e-7));
  const int64_t row0 = (int64_t)blockIdx.x * 32, col0 = (int64_t)blockIdx.y * 32;
  const void* u = a.at.u[z];
  const float* held = a.at.held[z];
  for (int i = t; i < 1024; i += 256) {
    const int64_t row = row0 + i / 32, col = col0 + i % 32;
    float v = 0.f;
    if (row < a.s.rows && col < a.s.cols) {
      const int64_t at = row * a.s.cols + col;
      v = load_value(u, a.u_dtype, at);
      if (held != nullptr) v = update_of(a, v, held[at]);
      v *= scale;
    }
    s_tile[i / 32][i % 32] = v;
  }
  __syncthreads();
  // the caller's rows are X's, or X^T's
  char* along = a.s.turned ? a.xt[0] + z * a.s.l * a.s.short_line() : a.x + z * a.s.r * a.s.long_line();
  char* across = a.s.turned ? a.x + z * a.s.r * a.s.long_line() : a.xt[0] + z * a.s.l * a.s.short_line();
  const int64_t along_line = a.s.turned ? a.s.short_line() : a.s.long_line();
  const int64_t across_line = a.s.turned ? a.s.long_line() : a.s.short_line();
  for (int i = t; i < 1024; i += 256) {
    if (row0 + i / 32 < a.s.rows) put_split(along + (row0 + i / 32) * along_line, col0 + i % 32, s_tile[i / 32][i % 32]);
    if (col0 + i / 32 < a.s.cols) put_split(across + (col0 + i / 32) * across_line, row0 + i % 32, s_tile[i % 32][i / 32]);
  }
}

// G (square false) from X, or P (square true) from G: the tiles on and below the diagonal, each written on both sides of it.
template <int WN>
struct SymmetricEpilogue {
  const MuonArgs& a;
  char* out;
  const char* g;                               // null for G
  bool mirror;
  __device__ __forceinline__ void operator()(const float* strip, int64_t row0, int64_t col0, int lane) const {
    const int64_t line = a.s.short_line(), r = a.s.r, padded = (r + 31) & ~31ll;
    for (int i = lane; i < 32 * WN; i += kWave) {
      const int64_t row = row0 + i / WN, col = col0 + i % WN;
      if (row < padded && col < padded) {
        float v = strip[(i / WN) * (WN + 4) + i % WN] * (1.f / kScale);
        if (g != nullptr) {
          const int64_t er = row < r ? row : r - 1, ec = col < r ? col : r - 1;
          const char* e = g + er * line + (ec >> 5) * kLine + 2 * (ec & 31);
          const float gv = (float)*reinterpret_cast<const _Float16*>(e) + (float)*reinterpret_cast<const _Float16*>(e + 64);
          v = a.b * gv + a.c * v + (row == col ? a.a * kScale : 0.f);
        }
        if (row >= r || col >= r) v = 0.f;
        if (row < r) put_split(out + row * line, col, v);
        if (mirror && col < r) put_split(out + col * line, row, v);
      }
    }
  }
};

template <bool SQUARE>
__global__ __launch_bounds__(256) void muon_symmetric_kernel(MuonArgs a) {
  typedef TileProduct<SplitOp, 64, 64, 32, 32> Tile;
  __shared__ __attribute__((aligned(128))) char lds[Tile::kLds];
  int i = 0, left = blockIdx.x;                // tile (i, j), j <= i, in the order of rows
  while (left > i) left -= ++i;
  const int64_t z = blockIdx.z, row0 = 64ll * i, col0 = 64ll * left;
  const Shape& s = a.s;
  char* g = a.g + z * s.r * s.short_line();
  char* p = a.p + z * s.r * s.short_line();
  const Lines from = SQUARE ? Lines{g, s.short_line(), s.r, s.short_line()}
                            : Lines{a.x + z * s.r * s.long_line(), s.long_line(), s.r, s.long_line()};
  Tile::run(lds, from, from, row0, col0, SymmetricEpilogue<32>{a, SQUARE ? p : g, SQUARE ? g : nullptr, row0 != col0});
}

// X = P X in planes, both ways round, or the last one into the caller's matrix.
template <int WN>
struct UpdateEpilogue {
  const MuonArgs& a;
  int64_t z;
  char* xt;                                    // null: the last one
  __device__ __forceinline__ void operator()(const float* strip, int64_t row0, int64_t col0, int lane) const {
    const Shape& s = a.s;
    const int64_t padded_r = (s.r + 31) & ~31ll, padded_l = (s.l + 31) & ~31ll;
    for (int i = lane; i < 32 * WN; i += kWave) {
      const int64_t row = row0 + i / WN, col = col0 + i % WN;
      if (row >= padded_r || col >= padded_l) continue;
      float v = strip[(i / WN) * (WN + 4) + i % WN] * (1.f / kScale);
      const bool in = row < s.r && col < s.l;
      if (xt != nullptr) {
        if (!in) v = 0.f;
        if (row < s.r) put_split(a.x + (z * s.r + row) * s.long_line(), col, v);
        if (col < s.l) put_split(xt + (z * s.l + col) * s.short_line(), row, v);
      } else if (in) {
        v *= 1.f / kScale;
        const int64_t at = s.turned ? col * s.cols + row : row * s.cols + col;
        void* w = a.at.out[z];
        if (a.keep != 0.f) v = a.keep * load_value(w, a.out_dtype, at) - a.size * v;
        store_value(w, a.out_dtype, at, v);
      }
    }
  }
};

__global__ __launch_bounds__(256) void muon_update_kernel(MuonArgs a, int from, int last) {
  typedef TileProduct<SplitOp, 64, 64, 32, 32> Tile;
  __shared__ __attribute__((aligned(128))) char lds[Tile::kLds];
  const Shape& s = a.s;
  const int64_t z = blockIdx.z;
  const Lines p{a.p + z * s.r * s.short_line(), s.short_line(), s.r, s.short_line()};
  const Lines x{a.xt[from] + z * s.l * s.short_line(), s.short_line(), s.l, s.short_line()};
  Tile::run(lds, p, x, 64ll * blockIdx.x, 64ll * blockIdx.y, UpdateEpilogue<32>{a, z, last ? nullptr : a.xt[1 - from]});
}

Shape shape_of(int64_t rows, int64_t cols) {
  const int turned = rows > cols;
  return Shape{rows, cols, turned ? cols : rows, turned ? rows : cols, turned};
}

int64_t parts_of(int64_t rows, int64_t cols) {
  const int64_t n = ceil_div(rows * cols, 4096);
  return n < 256 ? n : 256;
}

int64_t whole(int64_t bytes) { return ceil_div(bytes, 256) * 256; }

// Matrices that go through a set of launches together: enough for the chip's workgroups twice, so that the planes of
// those under way are not more than that takes.
int64_t group_of(int64_t count, int64_t rows, int64_t cols) {
  const int64_t tiles = ceil_div(rows, 64) * ceil_div(cols, 64), want = ceil_div(2048, tiles);
  const int64_t most = want < kGroup ? want : kGroup;
  return count < most ? count : most;
}

int64_t workspace_of(int64_t count, int64_t rows, int64_t cols) {
  const Shape s = shape_of(rows, cols);
  const int64_t n = group_of(count, rows, cols);
  return whole(n * parts_of(rows, cols) * 8) + whole(n * s.r * s.long_line()) + 2 * whole(n * s.l * s.short_line()) +
         2 * whole(n * s.r * s.short_line());
}

int check_muon(const char* what, int64_t count, int64_t rows, int64_t cols, int steps, const float* coefficients) {
  F2CGT_REQUIRE(count >= 0 && rows >= 0 && cols >= 0, F2CGT_E_INVALID, "%s: sizes must not be negative", what);
  F2CGT_REQUIRE(rows <= 65536 && cols <= 65536, F2CGT_E_UNSUPPORTED, "%s: at most 65536 rows and columns", what);
  F2CGT_REQUIRE(steps >= 1 && steps <= 100, F2CGT_E_INVALID, "%s: from one to 100 steps", what);
  F2CGT_REQUIRE(coefficients != nullptr, F2CGT_E_INVALID, "%s: null coefficients", what);
  // How far singular values from [0, 1] get, step by step, and what they are multiplied with.
  const double a = coefficients[0], b = coefficients[1], c = coefficients[2];
  double reach = 1.;
  for (int s = 0; s < steps; ++s) {
    double next = 0.;
    for (int i = 0; i <= 4096; ++i) {
      const double x = 1.001 * reach * i / 4096, p = a + b * x * x + c * x * x * x * x;
      F2CGT_REQUIRE(p > -kMost && p < kMost, F2CGT_E_UNSUPPORTED, "%s: these coefficients lead out of the range of the products", what);
      next = fabs(x * p) > next ? fabs(x * p) : next;
    }
    F2CGT_REQUIRE(next < 2.5, F2CGT_E_UNSUPPORTED, "%s: these coefficients lead out of the range of the products", what);
    reach = next;
  }
  return 0;
}

int run_muon(const char* what, MuonArgs a, int64_t count, int64_t rows, int64_t cols, int steps, const float* coefficients,
             void* const* out, const void* const* u, float* const* held, int64_t u_step, void* workspace, hipStream_t st) {
  a.s = shape_of(rows, cols);
  const Shape& s = a.s;
  a.parts = (int)parts_of(rows, cols);
  a.a = coefficients[0]; a.b = coefficients[1]; a.c = coefficients[2];
  const int64_t group = group_of(count, rows, cols);
  char* at = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) { char* p = at; at += whole(bytes); return p; };
  a.partial = reinterpret_cast<double*>(take(group * a.parts * 8));
  a.x = take(group * s.r * s.long_line());
  a.xt[0] = take(group * s.l * s.short_line());
  a.xt[1] = take(group * s.l * s.short_line());
  a.g = take(group * s.r * s.short_line());
  a.p = take(group * s.r * s.short_line());
  for (int64_t first = 0; first < count; first += group) {
    const int64_t n = count - first < group ? count - first : group;
    for (int64_t i = 0; i < n; ++i) {
      a.at.u[i] = u_step ? static_cast<const char*>(u[0]) + (first + i) * u_step * type_size(a.u_dtype) : u[first + i];
      a.at.out[i] = u_step ? static_cast<char*>(out[0]) + (first + i) * u_step * type_size(a.out_dtype) : out[first + i];
      a.at.held[i] = held != nullptr ? held[first + i] : nullptr;
    }
    muon_norm_kernel<<<dim3((unsigned)a.parts, (unsigned)n), 256, 0, st>>>(a);
    muon_split_kernel<<<dim3((unsigned)ceil_div(rows, 32), (unsigned)ceil_div(cols, 32), (unsigned)n), 256, 0, st>>>(a);
    const int64_t tiles = ceil_div(s.r, 64);
    for (int step = 0; step < steps; ++step) {
      const dim3 lower((unsigned)(tiles * (tiles + 1) / 2), 1, (unsigned)n);
      muon_symmetric_kernel<false><<<lower, 256, 0, st>>>(a);
      muon_symmetric_kernel<true><<<lower, 256, 0, st>>>(a);
      muon_update_kernel<<<dim3((unsigned)tiles, (unsigned)ceil_div(s.l, 64), (unsigned)n), 256, 0, st>>>(a, step & 1, step == steps - 1);
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
  if (int rc = check_muon(what, count, rows, cols, steps, coefficients)) return rc;
  F2CGT_REQUIRE(dense_type(dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 only", what);
  if (count == 0 || rows == 0 || cols == 0) return 0;
  F2CGT_REQUIRE(update && out && aligned(update, type_size(dtype)) && aligned(out, type_size(dtype)), F2CGT_E_INVALID,
                "%s: null or misaligned buffer", what);
  F2CGT_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= workspace_of(count, rows, cols), F2CGT_E_INVALID,
                "%s: workspace too small or misaligned", what);
  MuonArgs a{};
  a.u_dtype = a.out_dtype = dtype;
  a.keep = 0.f;
  void* outs[1] = {out};
  const void* ins[1] = {update};
  return run_muon(what, a, count, rows, cols, steps, coefficients, outs, ins, nullptr, rows * cols, workspace, as_stream(stream));
}

extern "C" int f2cgt_muon_step(void* const* weights, int weight_dtype, const void* const* grads, int grad_dtype, float* const* momenta,
                               int64_t count, int64_t rows, int64_t cols, float step_size, float decay, float momentum, int nesterov,
                               int steps, const float* coefficients, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "muon_step";
  if (int rc = check_muon(what, count, rows, cols, steps, coefficients)) return rc;
  F2CGT_REQUIRE(dense_type(weight_dtype) && dense_type(grad_dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 only", what);
  if (count == 0 || rows == 0 || cols == 0) return 0;
  F2CGT_REQUIRE(weights && grads && momenta, F2CGT_E_INVALID, "%s: null list", what);
  for (int64_t i = 0; i < count; ++i)
    F2CGT_REQUIRE(weights[i] && grads[i] && momenta[i] && aligned(weights[i], type_size(weight_dtype)) &&
                      aligned(grads[i], type_size(grad_dtype)) && aligned(momenta[i], 4),
                  F2CGT_E_INVALID, "%s: null or misaligned buffer", what);
  F2CGT_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= workspace_of(count, rows, cols), F2CGT_E_INVALID,
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
  return run_muon(what, a, count, rows, cols, steps, coefficients, weights, grads, momenta, 0, workspace, as_stream(stream));
}
