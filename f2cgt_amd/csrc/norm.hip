// Layer norm of rows, forward and backward.
//
//   mean = sum(x) / d     rstd = 1 / sqrt(sum((x - mean)^2) / d + eps)     n = (x - mean) rstd     out = n w + b
//   u = grad w     dx = rstd (u - sum(u) / d - n sum(u n) / d)     dw = sum over rows of grad n     db = sum over rows of grad
//
// Everything is fp32 until the one rounding of a result.  A row of up to 16384 columns stays in registers from its load to its store, so
// the squares are of differences from the mean (a second pass that costs no memory).  The backward pass takes x or its 8-bit checkpoint;
// with that, n is (decoded x - mean) rstd with the statistics of x itself, as the forward pass kept them.
// dw and db: a workgroup adds the rows that it takes in registers, its sums go to memory, and a second kernel adds those of all
// workgroups; every order is fixed by the sizes.
//
// Memory bounds both.  Where a copy of 4 GB makes 4.8 TB/s: 250 000 x 128 in fp32 forward 46 us (5.6 TB/s of what is read and written;
// with the call 52), 16 384 x 8192 in bf16 backward 150 us (5.4 TB/s), 60 001 x 602 in fp32 from its checkpoint 69 us (4.7 TB/s);
// longer rows, which are read once a pass, 1.1 to 3 TB/s.  Few rows are bound by latency: 1 x 4096 takes 2.4 us, 1024 x 256 backward 3.3
// and 2.4 for the second kernel.
#include "rows.hpp"

namespace f2cgt {
namespace {

struct NormArgs {
  const void* x;
  const void* weight;
  const void* bias;
  void* out;
  float* mean;
  float* rstd;
  int8_t* codes;
  uint8_t* exponents;
  int64_t m, ld, code_stride;
  int d, wide_weight;        // (weight and bias are fp32)
  float eps;
};

struct NormGradArgs {
  const void* grad;
  const void* x;
  const int8_t* codes;
  const uint8_t* exponents;
  const float* mean;
  const float* rstd;
  const void* weight;
  void* dx;
  float* parts;              // [workgroups][2 d]: sums of grad n, then of grad
  int64_t m, ld, grad_ld, code_stride;
  int d, wide_weight;
};

// Which columns a lane holds: pieces lane, lane + LANES, ... of the row.  The last piece of a row whose width is no multiple of V is moved
// back to end with the row; its first `skip` values belong to the piece before, which both hold and only that one adds.
template <int V, int LANES, int C>
struct Columns {
  int at[C], skip[C];
  bool on[C];
  __device__ __forceinline__ Columns(int lane, int d) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int start = (lane + c * LANES) * V;
      on[c] = start < d;
      at[c] = !on[c] ? 0 : start + V > d ? d - V : start;
      skip[c] = on[c] ? start - at[c] : V;
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_weight(const void* weight, int wide, int at, float (&v)[V]) {
  if (wide) load_piece<float, V < 4 ? V : 4>(static_cast<const float*>(weight) + at, *reinterpret_cast<float (*)[V < 4 ? V : 4]>(&v));
  if constexpr (V == 8) {
    if (wide) load_piece<float, 4>(static_cast<const float*>(weight) + at + 4, *reinterpret_cast<float (*)[4]>(&v[4]));
  }
  if (!wide) load_piece<T, V>(static_cast<const T*>(weight) + at, v);
}

// Sums of the waves of a workgroup that share a row: every wave's in LDS, then all of them in one order.  Each call of
// a loop takes the other half of `room`, so one barrier a call is enough.
template <int LANES, int N>
__device__ __forceinline__ void sum_group(float (&v)[N], float* room) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = sum_lanes<(LANES < kWave ? LANES : kWave)>(v[i]);
  if constexpr (LANES > kWave) {
    constexpr int kWaves = LANES / kWave, kSpread = kWaves <= 4 ? 4 : kWaves <= 8 ? 8 : 16;
    const int wave = threadIdx.x / kWave, at = threadIdx.x % kSpread;
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) room[i * kWaves + wave] = v[i];
    __syncthreads();
    // (every lane one wave's sum, then as over lanes)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sum_lanes<kSpread>(at < kWaves ? room[i * kWaves + at] : 0.f);
  }
}

constexpr int block_of(int lanes) { return lanes > kWave ? lanes : 256; }     // (threads of a workgroup)

template <typename T, int V, int LANES, int C, bool PACK>
__global__ __launch_bounds__(block_of(LANES)) void layer_norm_kernel(NormArgs a) {
  constexpr int kRows = block_of(LANES) / LANES, kWaves = LANES > kWave ? LANES / kWave : 1;
  __shared__ float room[2][2][kWaves];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const Columns<V, LANES, C> col(lane, a.d);
  float w[C][V], b[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) { w[c][e] = 1.f; b[c][e] = 0.f; }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (a.weight != nullptr) load_weight<T, V>(a.weight, a.wide_weight, col.at[c], w[c]);
    if (a.bias != nullptr) load_weight<T, V>(a.bias, a.wide_weight, col.at[c], b[c]);
  }
  const float d = (float)a.d;
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.m; base += (int64_t)gridDim.x * kRows) {
    const bool live = base + group < a.m;
    const int64_t row = live ? base + group : a.m - 1;       // (lanes without a row repeat the last one and write nothing)
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    float v[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) load_piece<T, V>(x + col.at[c], v[c]);
    float sum[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] += e >= col.skip[c] ? v[c][e] : 0.f;
    sum_group<LANES>(sum, &room[0][0][0]);
    const float mean = sum[0] / d;
    float squares[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float apart = e >= col.skip[c] ? v[c][e] - mean : 0.f;
        squares[0] += apart * apart;
      }
    sum_group<LANES>(squares, &room[1][0][0]);
    const float rstd = 1.f / sqrtf(squares[0] / d + a.eps);
    T* out = static_cast<T*>(a.out) + row * a.d;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = (v[c][e] - mean) * rstd * w[c][e] + b[c][e];
      if (live && col.on[c]) store_piece<T, V>(out + col.at[c], y);
    }
    if (a.mean != nullptr && live && lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    if constexpr (PACK) {
      constexpr int kShare = kCheckpointGroup / V < LANES ? kCheckpointGroup / V : LANES;      // lanes of a group of columns
#pragma unroll
      for (int c = 0; c < C; ++c) {
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint32_t size = __float_as_uint(v[c][e]) & 0x7FFFFFFFu;
          most = e >= col.skip[c] && size > most ? size : most;
        }
        const uint32_t exponent = exponent_of(most_lanes<kShare>(most));
        if (!live || !col.on[c]) continue;
        int8_t* codes = a.codes + row * a.code_stride + col.at[c];
        if (col.skip[c] == 0 && V > 1) {
          uint32_t packed[(V + 3) / 4] = {};
#pragma unroll
          for (int e = 0; e < V; ++e) packed[e / 4] |= (uint32_t)(code_of(v[c][e], exponent) & 255) << (8 * (e % 4));
#pragma unroll
          for (int e = 0; e < V / 4; ++e) reinterpret_cast<uint32_t*>(codes)[e] = packed[e];       // (rows start at multiples of 16)
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (e >= col.skip[c]) codes[e] = (int8_t)code_of(v[c][e], exponent);
        }
        if (lane % kShare == 0)
          a.exponents[row * ((a.d + kCheckpointGroup - 1) / kCheckpointGroup) + (col.at[c] + col.skip[c]) / kCheckpointGroup] =
              (uint8_t)exponent;
      }
    }
  }
}

// Rows beyond what a workgroup's registers hold: read again for each pass (from the L2, mostly).
template <typename T, bool PACK>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(NormArgs a) {
  __shared__ float room[2][16];
  const float d = (float)a.d;
  const int lane = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    T* out = static_cast<T*>(a.out) + row * a.d;
    float sum[1] = {0.f}, squares[1] = {0.f};
    for (int i = lane; i < a.d; i += 1024) sum[0] += (float)x[i];
    sum_group<1024>(sum, room[0]);
    const float mean = sum[0] / d;
    for (int i = lane; i < a.d; i += 1024) {
      const float apart = (float)x[i] - mean;
      squares[0] += apart * apart;
    }
    sum_group<1024>(squares, room[1]);
    const float rstd = 1.f / sqrtf(squares[0] / d + a.eps);
    const float* wide_w = static_cast<const float*>(a.weight);
    const float* wide_b = static_cast<const float*>(a.bias);
    const int to = PACK ? (a.d + kCheckpointGroup - 1) / kCheckpointGroup * kCheckpointGroup : a.d;   // (whole groups of lanes)
    for (int i = lane; i < to; i += 1024) {
      const bool in = i < a.d;
      const float v = in ? (float)x[i] : 0.f;
      if (in) {
        const float w = a.weight == nullptr ? 1.f : a.wide_weight ? wide_w[i] : (float)static_cast<const T*>(a.weight)[i];
        const float b = a.bias == nullptr ? 0.f : a.wide_weight ? wide_b[i] : (float)static_cast<const T*>(a.bias)[i];
        out[i] = (T)((v - mean) * rstd * w + b);
      }
      if constexpr (PACK) {
        const uint32_t exponent = exponent_of(most_lanes<kCheckpointGroup>(__float_as_uint(v) & 0x7FFFFFFFu));
        if (in) {
          a.codes[row * a.code_stride + i] = (int8_t)code_of(v, exponent);
          if (i % kCheckpointGroup == 0) a.exponents[row * (to / kCheckpointGroup) + i / kCheckpointGroup] = (uint8_t)exponent;
        }
      }
    }
    if (a.mean != nullptr && lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// What a lane holds of a row of the backward pass, as memory has it.
template <typename T, int V, int C, bool PACKED>
struct GradRow {
  typedef typename piece_words<T, V>::type words;
  words g[C], x[PACKED ? 1 : C];
  uint32_t codes[PACKED ? C : 1][(V + 3) / 4], first[PACKED ? C : 1], last[PACKED ? C : 1];
  float mean, rstd;

  template <int LANES>
  __device__ __forceinline__ void load(const NormGradArgs& a, const Columns<V, LANES, C>& col, int64_t row) {
    const T* grad = static_cast<const T*>(a.grad) + row * a.grad_ld;
#pragma unroll
    for (int c = 0; c < C; ++c) g[c] = *reinterpret_cast<const words*>(grad + col.at[c]);
    if constexpr (PACKED) {
      const int8_t* from = a.codes + row * a.code_stride;
      const uint8_t* exponents = a.exponents + row * ((a.d + kCheckpointGroup - 1) / kCheckpointGroup);
      typedef uint32_t word_any __attribute__((aligned(1)));
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if constexpr (V == 1) {
          codes[c][0] = (uint8_t)from[col.at[c]];
        } else {
#pragma unroll
          for (int i = 0; i < V / 4; ++i) codes[c][i] = reinterpret_cast<const word_any*>(from + col.at[c])[i];
        }
        // (a piece that was moved back may lie in two groups)
        first[c] = exponents[col.at[c] / kCheckpointGroup];
        last[c] = exponents[(col.at[c] + V - 1) / kCheckpointGroup];
      }
    } else {
      const T* from = static_cast<const T*>(a.x) + row * a.ld;
#pragma unroll
      for (int c = 0; c < C; ++c) x[c] = *reinterpret_cast<const words*>(from + col.at[c]);
    }
    mean = a.mean[row];
    rstd = a.rstd[row];
  }
  __device__ __forceinline__ void values(int c, int at, float (&v)[V]) const {
    if constexpr (PACKED) {
      const int border = (at + V - 1) / kCheckpointGroup * kCheckpointGroup - at;
      const float step0 = step_of(first[c]), step1 = step_of(last[c]);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = coded_value(codes[c][e / 4], e % 4, e < border ? step0 : step1);
    } else {
      values_of<T, V>(x[c], v);
    }
  }
};

// A row's loads are issued a row ahead: what a workgroup has under way covers the latency of the sums over its lanes (60 001 x 602 from a
// checkpoint 100 us without, 69 with).
template <typename T, int V, int LANES, int C, bool PACKED>
__global__ __launch_bounds__(block_of(LANES)) void layer_norm_grad_kernel(NormGradArgs a) {
  constexpr int kBlock = block_of(LANES), kRows = kBlock / LANES, kWaves = LANES > kWave ? LANES / kWave : 1;
  // a piece's sums of the workgroup's groups of lanes, one piece after the other
  __shared__ float sums[kRows > 1 ? kBlock * 2 * V : 1];
  __shared__ float room[2][2 * kWaves];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const Columns<V, LANES, C> col(lane, a.d);
  // (128 registers hold no second row of sixteen values a lane, nor all of one from a checkpoint: 24 of them lie in scratch in fp32, 3 in 16 bits)
  constexpr bool kAhead = LANES < 1024 || C * V <= 8;
  float w[C][V], dw[C][V], db[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[c][e] = 1.f;
      dw[c][e] = db[c][e] = 0.f;
    }
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (a.weight != nullptr) load_weight<T, V>(a.weight, a.wide_weight, col.at[c], w[c]);
  const float d = (float)a.d;
  const int64_t stride = (int64_t)gridDim.x * kRows, first_row = (int64_t)blockIdx.x * kRows + group;
  auto held = [&](int64_t row) { return row < a.m ? row : a.m - 1; };          // (lanes without a row repeat the last one and write nothing)
  GradRow<T, V, C, PACKED> now, next;
  if (kAhead) next.load(a, col, held(first_row));
  int turn = 0;
  for (int64_t row = first_row; row - group < a.m; row += stride, turn ^= 1) {
    const bool live = row < a.m;
    if constexpr (kAhead) {
      now = next;
      next.load(a, col, held(row + stride));
    } else {
      now.load(a, col, held(row));
    }
    float s[2] = {0.f, 0.f}, g[C][V], n[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      values_of<T, V>(now.g[c], g[c]);
      now.values(c, col.at[c], n[c]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        n[c][e] = (n[c][e] - now.mean) * now.rstd;
        const bool own = e >= col.skip[c];
        const float u = own ? g[c][e] * w[c][e] : 0.f;
        s[0] += u;
        s[1] += own ? u * n[c][e] : 0.f;
        dw[c][e] += live ? g[c][e] * n[c][e] : 0.f;
        db[c][e] += live ? g[c][e] : 0.f;
      }
    }
    sum_group<LANES>(s, room[turn]);
    const float first = s[0] / d, second = s[1] / d;
    T* dx = static_cast<T*>(a.dx) + row * a.d;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = now.rstd * (g[c][e] * w[c][e] - first - n[c][e] * second);
      if (live && col.on[c]) store_piece<T, V>(dx + col.at[c], y);
    }
  }
  if (a.parts == nullptr) return;
  float* parts = a.parts + (int64_t)blockIdx.x * 2 * a.d;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if constexpr (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sums[(e * 2) * kBlock + threadIdx.x] = dw[c][e];
        sums[(e * 2 + 1) * kBlock + threadIdx.x] = db[c][e];
      }
      __syncthreads();
      for (int o = threadIdx.x; o < LANES * 2 * V; o += kBlock) {
        const int l = o % LANES, e = o / LANES / 2, which = o / LANES % 2, start = (l + c * LANES) * V;
        const int at = start + V > a.d ? a.d - V : start;
        if (start >= a.d || e < start - at) continue;
        float sum = 0.f;
#pragma unroll 4
        for (int r = 0; r < kRows; ++r) sum += sums[(e * 2 + which) * kBlock + r * LANES + l];
        parts[which * a.d + at + e] = sum;
      }
    } else if (V > 1 && col.on[c] && col.skip[c] == 0) {
      // (16 bytes at a time: single values of a lane are apart, and 2 x 16053 in bf16 took 21.8 us rather than 10)
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        store_piece<float, 4>(parts + col.at[c] + q, {dw[c][q], dw[c][q + 1], dw[c][q + 2], dw[c][q + 3]});
        store_piece<float, 4>(parts + a.d + col.at[c] + q, {db[c][q], db[c][q + 1], db[c][q + 2], db[c][q + 3]});
      }
    } else if (col.on[c]) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e >= col.skip[c]) {
          parts[col.at[c] + e] = dw[c][e];
          parts[a.d + col.at[c] + e] = db[c][e];
        }
    }
  }
}

// The same of rows beyond what registers hold: dx row by row, dw and db in a kernel that goes down columns.
template <typename T, bool PACKED>
__device__ __forceinline__ float unit_value(const NormGradArgs& a, int64_t row, int i, float mean, float rstd) {
  float x;
  if constexpr (PACKED) {
    const uint8_t* exponents = a.exponents + row * ((a.d + kCheckpointGroup - 1) / kCheckpointGroup);
    x = (float)(int)a.codes[row * a.code_stride + i] * step_of(exponents[i / kCheckpointGroup]);
  } else {
    x = (float)static_cast<const T*>(a.x)[row * a.ld + i];
  }
  return (x - mean) * rstd;
}
template <typename T>
__device__ __forceinline__ float weight_value(const void* weight, int wide, int i) {
  return weight == nullptr ? 1.f : wide ? static_cast<const float*>(weight)[i] : (float)static_cast<const T*>(weight)[i];
}
template <typename T, bool PACKED>
__global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(NormGradArgs a) {
  __shared__ float room[2][32];
  const float d = (float)a.d;
  const int lane = threadIdx.x;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x, turn ^= 1) {
    const T* grad = static_cast<const T*>(a.grad) + row * a.grad_ld;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int i = lane; i < a.d; i += 1024) {
      const float u = (float)grad[i] * weight_value<T>(a.weight, a.wide_weight, i);
      s[0] += u;
      s[1] += u * unit_value<T, PACKED>(a, row, i, mean, rstd);
    }
    sum_group<1024>(s, room[turn]);
    const float first = s[0] / d, second = s[1] / d;
    T* dx = static_cast<T*>(a.dx) + row * a.d;
    for (int i = lane; i < a.d; i += 1024) {
      const float u = (float)grad[i] * weight_value<T>(a.weight, a.wide_weight, i);
      dx[i] = (T)(rstd * (u - first - unit_value<T, PACKED>(a, row, i, mean, rstd) * second));
    }
  }
}
template <typename T, bool PACKED>
__global__ __launch_bounds__(256) void layer_norm_columns_kernel(NormGradArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.d) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const float g = (float)static_cast<const T*>(a.grad)[row * a.grad_ld + i];
    dw += g * unit_value<T, PACKED>(a, row, i, a.mean[row], a.rstd[row]);
    db += g;
  }
  float* parts = a.parts + (int64_t)blockIdx.y * 2 * a.d;
  parts[i] = dw;
  parts[a.d + i] = db;
}

// Sums of the workgroups' sums, 64 columns to a workgroup, sixteen waves with every sixteenth row.
struct JoinArgs {
  const float* parts;
  int rows, columns;         // columns: 2 d
  void* to[2];               // dw, db (either may be null)
  int tag;
};
__global__ __launch_bounds__(1024) void join_sums_kernel(JoinArgs a) {
  __shared__ float room[16][64];
  const int column = blockIdx.x * 64 + threadIdx.x % 64, wave = threadIdx.x / 64;
  float sum = 0.f;
  if (column < a.columns) {
    const float* from = a.parts + column;
    int r = wave;
    for (; r + 7 * 16 < a.rows; r += 8 * 16) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = from[(int64_t)(r + 16 * u) * a.columns];
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += v[u];
    }
    for (; r < a.rows; r += 16) sum += from[(int64_t)r * a.columns];
  }
  room[wave][threadIdx.x % 64] = sum;
  __syncthreads();
  if (wave != 0 || column >= a.columns) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += room[i][threadIdx.x];
  const int half = a.columns / 2, which = column >= half;
  if (a.to[which] == nullptr) return;
  const int at = column - which * half;
  if (a.tag == F2CGT_DT_F32) static_cast<float*>(a.to[which])[at] = sum;
  else if (a.tag == F2CGT_DT_F16) static_cast<_Float16*>(a.to[which])[at] = (_Float16)sum;
  else static_cast<__bf16*>(a.to[which])[at] = (__bf16)sum;
}

// f(piece values, lanes, pieces a lane) for the width d: few lanes to a short row, so that a workgroup has several rows; as many as a row
// has pieces to a long one.  Where those would be a power of two of which many have no piece, three pieces a lane.  Measured, GB/s of
// what is read and written, forward and backward:
//   up to four pieces 4 lanes rather than 8: 1048576 x 16 in fp32 5830 and 5000 against 4400 and 4880;
//   up to 96 32 x 3 rather than 64 x 2: 111476 x 602 in bf16 5470 and 4300 against 4760 and 3530;
//   up to 192 64 x 3 forward (65154 x 1030 in bf16 5250, with 192 lanes 3850, with 256 3270), backward the same in fp32, in 16 bits, where
//   three pieces are 24 values a lane, 192 lanes (3840, with 256 3465);
//   up to 384 and 768 128 x 3 and 256 x 3 forward (32577 x 1030 in fp32 5800 against 4090, 31956 x 2100 in bf16 5020 against 3250), but
//   not backward, where rows and sums of three pieces leave a CU few waves (22369 x 1500 in fp32 3930 against 4820); workgroups of 384
//   and 768 lanes lose to both, since a CU holds two or one;
//   up to 4096 in fp32 1024 x 4 rather than the kernels for long rows: 2048 x 16384 5560 and 4500 against 3290 and 2530 (in 16 bits that
//   would be 32 values a lane, beyond the registers of the backward pass).
template <int N> struct count_of { static constexpr int value = N; };
template <typename T, bool FORWARD, typename F>
bool with_geometry(int64_t d, const F& f) {
  constexpr int V = kPieceOf<T>;
  const int64_t pieces = ceil_div(d, V);
  if (d < V) f(count_of<1>{}, count_of<8>{}, count_of<1>{});
  else if (pieces <= 4) f(count_of<V>{}, count_of<4>{}, count_of<1>{});
  else if (pieces <= 8) f(count_of<V>{}, count_of<8>{}, count_of<1>{});
  else if (pieces <= 16) f(count_of<V>{}, count_of<16>{}, count_of<1>{});
  else if (pieces <= 32) f(count_of<V>{}, count_of<32>{}, count_of<1>{});
  else if (pieces <= 64) f(count_of<V>{}, count_of<64>{}, count_of<1>{});
  else if (pieces <= 96) f(count_of<V>{}, count_of<32>{}, count_of<3>{});
  else if (pieces <= 128) f(count_of<V>{}, count_of<64>{}, count_of<2>{});
  else if (pieces <= 192) {
    if constexpr (V == 4 || FORWARD) f(count_of<V>{}, count_of<64>{}, count_of<3>{});
    else f(count_of<V>{}, count_of<192>{}, count_of<1>{});
  } else if (pieces <= 256) f(count_of<V>{}, count_of<256>{}, count_of<1>{});
  else if (pieces <= 384) {
    if constexpr (FORWARD) f(count_of<V>{}, count_of<128>{}, count_of<3>{});
    else f(count_of<V>{}, count_of<512>{}, count_of<1>{});
  } else if (pieces <= 512) f(count_of<V>{}, count_of<512>{}, count_of<1>{});
  else if (pieces <= 768) {
    if constexpr (FORWARD) f(count_of<V>{}, count_of<256>{}, count_of<3>{});
    else f(count_of<V>{}, count_of<1024>{}, count_of<1>{});
  } else if (pieces <= 1024) f(count_of<V>{}, count_of<1024>{}, count_of<1>{});
  else if (pieces <= 2048) f(count_of<V>{}, count_of<1024>{}, count_of<2>{});
  else if constexpr (V == 4) {
    if (pieces > 4096) return false;
    f(count_of<V>{}, count_of<1024>{}, count_of<4>{});
  } else {
    return false;
  }
  return true;
}

struct BlockOf {
  int64_t block, rows;                     // threads, rows at a time (0: long rows)
};
BlockOf block_for(int64_t d, int size) {
  BlockOf b{0, 0};
  auto count = [&](auto, auto lanes, auto) {
    b.block = block_of(decltype(lanes)::value);
    b.rows = b.block / decltype(lanes)::value;
  };
  if (size == 4) with_geometry<float, false>(d, count);
  else with_geometry<__bf16, false>(d, count);
  return b;
}

// Workgroups of the backward pass: each writes 2 d sums.
int64_t grad_blocks(int64_t m, int64_t d, int size) {
  const BlockOf rows = block_for(d, size);
  if (rows.rows == 0) return m < 64 ? m : 64;         // (rows of the columns' kernel)
  // (as many as are on the chip at once, the same number on each CU: more only write and read more sums, at 16384 x 8192 64 MB of them
  // beside 805)
  const int64_t all = ceil_div(m, rows.rows), most = (int64_t)num_cus() * (1024 / rows.block);
  return all < most ? all : most;
}

int check_rows(const char* what, int64_t m, int64_t d) {
  F2CGT_REQUIRE(m >= 0 && d >= 0, F2CGT_E_INVALID, "%s: sizes must not be negative", what);
  F2CGT_REQUIRE(m < (1ll << 31) && d < (1ll << 24), F2CGT_E_UNSUPPORTED, "%s: at most 2^31 - 1 rows and 2^24 - 1 columns", what);
  F2CGT_REQUIRE(m == 0 || d > 0, F2CGT_E_INVALID, "%s: rows of no columns have no mean", what);
  return 0;
}

}  // namespace
}  // namespace f2cgt

using namespace f2cgt;

namespace {
bool known(int dtype) { return dtype == F2CGT_DT_F32 || dtype == F2CGT_DT_F16 || dtype == F2CGT_DT_BF16; }
int size_of(int dtype) { return dtype == F2CGT_DT_F32 ? 4 : 2; }
}  // namespace

extern "C" int f2cgt_layer_norm(const void* x, int dtype, int64_t ld, const void* weight, const void* bias, int weight_dtype,
                                void* out, float* mean, float* rstd, int8_t* codes, int64_t code_stride, uint8_t* exponents,
                                int64_t m, int64_t d, float eps, void* stream) {
  const char* what = "layer_norm";
  if (int rc = check_rows(what, m, d)) return rc;
  F2CGT_REQUIRE(known(dtype), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 rows only", what);
  F2CGT_REQUIRE((!weight && !bias) || weight_dtype == dtype || weight_dtype == F2CGT_DT_F32, F2CGT_E_UNSUPPORTED,
                "%s: weight and bias must be fp32 or of the rows' type", what);
  F2CGT_REQUIRE(m <= 1 || ld >= d, F2CGT_E_INVALID, "%s: rows overlap", what);
  F2CGT_REQUIRE(eps >= 0.f, F2CGT_E_INVALID, "%s: eps must not be negative", what);
  F2CGT_REQUIRE(!mean == !rstd && !codes == !exponents, F2CGT_E_INVALID, "%s: half of the statistics or of the checkpoint", what);
  F2CGT_REQUIRE(!codes || (code_stride >= d && code_stride % 16 == 0 && aligned(codes, 16)), F2CGT_E_INVALID,
                "%s: rows of codes must start at multiples of 16 bytes and not overlap", what);
  if (m == 0) return 0;
  F2CGT_REQUIRE(x && out, F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(aligned(x, size_of(dtype)) && aligned(out, size_of(dtype)) && aligned(weight, size_of(weight_dtype)) &&
                    aligned(bias, size_of(weight_dtype)), F2CGT_E_INVALID, "%s: misaligned buffer", what);
  const NormArgs a{x, weight, bias, out, mean, rstd, codes, exponents, m, ld, code_stride, (int)d, weight_dtype == F2CGT_DT_F32, eps};
  hipStream_t st = as_stream(stream);
  return with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    auto launch = [&](auto values, auto lanes, auto pieces) {
      constexpr int V = decltype(values)::value, L = decltype(lanes)::value, C = decltype(pieces)::value;
      const int64_t all = ceil_div(m, block_of(L) / L), most = 8 * (int64_t)num_cus() * 256 / block_of(L);
      const dim3 grid((unsigned)(all < most ? all : most)), block(block_of(L));
      if (codes) layer_norm_kernel<T, V, L, C, true><<<grid, block, 0, st>>>(a);
      else layer_norm_kernel<T, V, L, C, false><<<grid, block, 0, st>>>(a);
    };
    if (!with_geometry<T, true>(d, launch)) {
      const dim3 grid((unsigned)(m < 2 * num_cus() ? m : 2 * num_cus()));
      if (codes) layer_norm_long_kernel<T, true><<<grid, dim3(1024), 0, st>>>(a);
      else layer_norm_long_kernel<T, false><<<grid, dim3(1024), 0, st>>>(a);
    }
    return launch_status(what);
  });
}

extern "C" int64_t f2cgt_layer_norm_grad_workspace_bytes(int dtype, int64_t m, int64_t d) {
  if (m <= 0 || d <= 0 || !known(dtype)) return 0;
  return grad_blocks(m, d, size_of(dtype)) * 8 * d;
}

extern "C" int f2cgt_layer_norm_grad(const void* grad, int dtype, int64_t grad_ld, const void* x, int64_t ld, const int8_t* codes,
                                     int64_t code_stride, const uint8_t* exponents, const float* mean, const float* rstd,
                                     const void* weight, int weight_dtype, void* dx, void* dweight, void* dbias, int grad_dtype,
                                     void* workspace, int64_t workspace_bytes, int64_t m, int64_t d, void* stream) {
  const char* what = "layer_norm_grad";
  if (int rc = check_rows(what, m, d)) return rc;
  F2CGT_REQUIRE(known(dtype) && ((!dweight && !dbias) || known(grad_dtype)), F2CGT_E_UNSUPPORTED, "%s: fp32, fp16 or bf16 only", what);
  F2CGT_REQUIRE(!weight || weight_dtype == dtype || weight_dtype == F2CGT_DT_F32, F2CGT_E_UNSUPPORTED,
                "%s: the weight must be fp32 or of the rows' type", what);
  F2CGT_REQUIRE(!x || !codes, F2CGT_E_INVALID, "%s: rows or their checkpoint, not both", what);
  F2CGT_REQUIRE(m <= 1 || (grad_ld >= d && (codes || ld >= d)), F2CGT_E_INVALID, "%s: rows overlap", what);
  F2CGT_REQUIRE(!codes || code_stride >= d, F2CGT_E_INVALID, "%s: rows of codes overlap", what);
  if (d == 0) return 0;
  F2CGT_REQUIRE(m == 0 || (grad && (x || (codes && exponents)) && mean && rstd && dx), F2CGT_E_INVALID, "%s: null buffer", what);
  F2CGT_REQUIRE(aligned(grad, size_of(dtype)) && aligned(x, size_of(dtype)) && aligned(dx, size_of(dtype)) &&
                    aligned(weight, size_of(weight_dtype)) && aligned(dweight, size_of(grad_dtype)) && aligned(dbias, size_of(grad_dtype)),
                F2CGT_E_INVALID, "%s: misaligned buffer", what);
  const bool sums = dweight || dbias;
  const int64_t need = sums ? f2cgt_layer_norm_grad_workspace_bytes(dtype, m, d) : 0;
  F2CGT_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), F2CGT_E_INVALID,
                "%s: workspace too small or misaligned", what);
  float* parts = sums ? static_cast<float*>(workspace) : nullptr;
  const NormGradArgs a{grad, x, codes, exponents, mean, rstd, weight, dx, parts, m, ld, grad_ld, code_stride, (int)d,
                       weight_dtype == F2CGT_DT_F32};
  hipStream_t st = as_stream(stream);
  const int64_t blocks = m == 0 ? 0 : grad_blocks(m, d, size_of(dtype));
  if (m > 0) {
    const int rc = with_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      auto launch = [&](auto values, auto lanes, auto pieces) {
        constexpr int V = decltype(values)::value, L = decltype(lanes)::value, C = decltype(pieces)::value;
        const dim3 grid((unsigned)blocks), block(block_of(L));
        if (codes) layer_norm_grad_kernel<T, V, L, C, true><<<grid, block, 0, st>>>(a);
        else layer_norm_grad_kernel<T, V, L, C, false><<<grid, block, 0, st>>>(a);
      };
      if (!with_geometry<T, false>(d, launch)) {
        const dim3 grid((unsigned)(m < 2 * num_cus() ? m : 2 * num_cus())), columns((unsigned)ceil_div(d, 256), (unsigned)blocks);
        if (codes) layer_norm_grad_long_kernel<T, true><<<grid, dim3(1024), 0, st>>>(a);
        else layer_norm_grad_long_kernel<T, false><<<grid, dim3(1024), 0, st>>>(a);
        if (sums && codes) layer_norm_columns_kernel<T, true><<<columns, dim3(256), 0, st>>>(a);
        else if (sums) layer_norm_columns_kernel<T, false><<<columns, dim3(256), 0, st>>>(a);
      }
      return launch_status(what);
    });
    if (rc) return rc;
  }
  if (!sums) return 0;
  const JoinArgs j{parts, (int)blocks, (int)(2 * d), {dweight, dbias}, grad_dtype};     // (of no rows: zeros)
  join_sums_kernel<<<dim3((unsigned)ceil_div(2 * d, 64)), dim3(1024), 0, st>>>(j);
  return launch_status(what);
}
