// Learnt rows: rows of a table by id, scaled, and the gradient of the table.
//
//   out_i = scale * table[id_i]                     dtable_r = scale * sum over i with id_i = r, in their order, of grad_i
//
// An id outside the table (a place of a padded batch) reads zeros and adds to no row.  The gradient writes every row of the table,
// those without ids as zeros, and adds in the order of the ids' places (a row of more than kLong ids in parts of that order): no
// atomics on values, the same bits each time.
//
// For that the ids are sorted, stable.  Up to kPickMost ids each workgroup, which owns a range of the table's rows, reads all ids,
// keeps those of its range in LDS in their order and sorts them there: one launch.  More are sorted by digits first (a histogram of
// each workgroup's ids, their prefixes, and a scatter that keeps the order, for every digit), and a workgroup finds its range in them.
// Where a row has hundreds of ids, whole runs of kChunk of them are added up beforehand, all over the chip, and a workgroup's waves
// share what is left.
//
// Memory bounds the lookup: 109 074 of 2.4 million rows of 100 in fp32, 87 MB both ways, in 19.5 us.  The gradient of a million ids of
// 250 000 rows of 256 in bf16, 512 MB read and 128 written: digits 45 us, runs 85, sums and zeros 102 to 122 (rows of 512 bytes at
// random places: latency, and few bytes at a time).
#include "rows.hpp"

namespace f2cgt {
namespace {

__host__ __device__ constexpr int bits_of(uint32_t v) {        // of numbers up to v
  int b = 0;
  while (b < 32 && (v >> b) != 0) ++b;
  return b;
}

// An id's row, or `rows` where it has none.
template <typename Idx>
__device__ __forceinline__ uint32_t key_of(Idx id, uint32_t rows) {
  return (uint64_t)(int64_t)id < (uint64_t)rows ? (uint32_t)id : rows;
}

// ---- forward --------------------------------------------------------------------------------------------
struct LookupArgs {
  const void* table;
  const void* index;
  void* out;
  int64_t n, ld;
  uint32_t rows;
  int d, pieces, lanes;      // lanes: of a row, a power of two up to 64
  float scale;
};

template <typename T, int V, typename Idx>
__global__ __launch_bounds__(256) void lookup_kernel(LookupArgs a) {
  constexpr int kUnroll = 4;
  const int per_pass = 256 / a.lanes, sub = threadIdx.x & (a.lanes - 1);
  const int64_t first = (int64_t)blockIdx.x * kUnroll * per_pass + threadIdx.x / a.lanes;
  const T* from[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = first + (int64_t)u * per_pass;
    from[u] = nullptr;
    if (i < a.n) {
      const uint32_t key = key_of(static_cast<const Idx*>(a.index)[i], a.rows);
      if (key < a.rows) from[u] = static_cast<const T*>(a.table) + (int64_t)key * a.ld;
    }
  }
  for (int p = sub; p < a.pieces; p += a.lanes) {
    const int at = p * V + V > a.d ? a.d - V : p * V;        // (the last piece ends with the row)
    float v[kUnroll][V];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[u][e] = 0.f;
      if (from[u] != nullptr) load_piece<T, V>(from[u] + at, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = first + (int64_t)u * per_pass;
      if (i >= a.n) continue;
      if (from[u] != nullptr)
#pragma unroll
        for (int e = 0; e < V; ++e) v[u][e] *= a.scale;
      store_piece<T, V>(static_cast<T*>(a.out) + i * a.d + at, v[u]);
    }
  }
}

// ---- sorting by digits ------------------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortItems = 4, kSortTile = kSortThreads * kSortItems, kSortWaves = kSortThreads / kWave;
constexpr int kMostBits = 10;

struct SortArgs {
  const void* index;         // the first digit's keys are made of these
  const uint2* pairs;        // of the others: (key, place), the last scatter's
  uint2* pairs_out;
  uint32_t* counts;          // [digits][blocks], then [digits] of the totals
  int64_t n;
  uint32_t rows, blocks;
  int shift, bits;
};

// Key and place of the ids as they stand before a digit.
template <typename Idx, bool FIRST>
__device__ __forceinline__ uint2 sort_pair(const SortArgs& a, int64_t i) {
  if constexpr (FIRST) return uint2{key_of(static_cast<const Idx*>(a.index)[i], a.rows), (uint32_t)i};
  else return a.pairs[i];
}

template <typename Idx, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs a) {
  __shared__ uint32_t counts[1 << kMostBits];
  const uint32_t digits = 1u << a.bits;
  for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) counts[d] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int u = 0; u < kSortItems; ++u) {
    const int64_t i = first + u * kSortThreads + threadIdx.x;
    if (i < a.n) atomicAdd(&counts[sort_pair<Idx, FIRST>(a, i).x >> a.shift & (digits - 1)], 1u);
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) a.counts[(int64_t)d * a.blocks + blockIdx.x] = counts[d];
}

// A digit's counts become the sums of those before, its total goes behind them all.  One wave a digit, four workgroups' counts a lane.
__global__ __launch_bounds__(kWave) void sort_prefix_kernel(SortArgs a) {
  uint32_t* row = a.counts + (int64_t)blockIdx.x * a.blocks;
  uint32_t before = 0;
  for (uint32_t b = 0; b < a.blocks; b += 4 * kWave) {
    const uint32_t i = b + 4 * threadIdx.x;
    uint32_t own[4], all = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) own[e] = i + e < a.blocks ? row[i + e] : 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) all += own[e];
    uint32_t upto = all;
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
      const uint32_t left = (uint32_t)__shfl_up((int)upto, by);
      if ((int)threadIdx.x >= by) upto += left;
    }
    uint32_t at = before + upto - all;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e < a.blocks) row[i + e] = at;
      at += own[e];
    }
    before += (uint32_t)__shfl((int)upto, kWave - 1);
  }
  if (threadIdx.x == 0) a.counts[(int64_t)gridDim.x * a.blocks + blockIdx.x] = before;
}

// Lanes of the wave with the same digit as this one, among those that are `on`.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool on) {
  uint64_t same = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const bool set = digit >> b & 1;
    const uint64_t with = __ballot(set);
    same &= set ? with : ~with;
  }
  return same;
}
__device__ __forceinline__ uint32_t below(uint64_t lanes) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}

// Exclusive sums of values[0 .. count) in LDS, by the whole workgroup; `room` holds a word a wave.
template <int THREADS>
__device__ __forceinline__ void prefix_in_lds(uint32_t* values, uint32_t count, uint32_t* room) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  uint32_t before = 0;
  for (uint32_t b = 0; b < count; b += THREADS) {
    const uint32_t i = b + threadIdx.x;
    const uint32_t own = i < count ? values[i] : 0;
    uint32_t upto = own;
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
      const uint32_t left = (uint32_t)__shfl_up((int)upto, by);
      if (lane >= by) upto += left;
    }
    if (lane == kWave - 1) room[wave] = upto;
    __syncthreads();
    uint32_t waves = before, all = 0;
    for (int w = 0; w < THREADS / kWave; ++w) {
      if (w < wave) waves += room[w];
      all += room[w];
    }
    if (i < count) values[i] = waves + upto - own;
    before += all;
    __syncthreads();
  }
}

template <typename Idx, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortArgs a) {
  __shared__ uint32_t base[1 << kMostBits];
  __shared__ uint32_t own[kSortWaves][1 << kMostBits];
  __shared__ uint32_t room[kSortWaves];
  const uint32_t digits = 1u << a.bits;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) {
    base[d] = a.counts[(int64_t)digits * a.blocks + d];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) own[w][d] = 0;
  }
  __syncthreads();
  prefix_in_lds<kSortThreads>(base, digits, room);
  // a wave has a run of the tile: counted, then placed in order
  const int64_t first = (int64_t)blockIdx.x * kSortTile + wave * kWave * kSortItems + lane;
  uint2 pair[kSortItems];
#pragma unroll
  for (int u = 0; u < kSortItems; ++u) {
    const int64_t i = first + u * kWave;
    pair[u] = uint2{0, 0};
    if (i < a.n) {
      pair[u] = sort_pair<Idx, FIRST>(a, i);
      atomicAdd(&own[wave][pair[u].x >> a.shift & (digits - 1)], 1u);
    }
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) {
    uint32_t at = base[d] + a.counts[(int64_t)d * a.blocks + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t count = own[w][d];
      own[w][d] = at;
      at += count;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSortItems; ++u) {
    const int64_t i = first + u * kWave;
    const bool on = i < a.n;
    const uint32_t digit = pair[u].x >> a.shift & (digits - 1);
    const uint64_t same = same_digit(digit, a.bits, on);
    const uint32_t rank = below(same);
    if (on) a.pairs_out[own[wave][digit] + rank] = pair[u];
    __builtin_amdgcn_wave_barrier();
    if (on && rank == 0) own[wave][digit] += (uint32_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- sums over a row's gradients --------------------------------------------------------------------------
// ids of one row whose sum is made beforehand (64 are faster for few ids, but not where a chunk is four waves', and slower for many: the
// million above 293 us)
constexpr int kChunk = 128;
constexpr uint32_t kLong = 64;               // ids of a row above which a workgroup's waves share them

struct SumArgs {
  const void* grad;
  const void* index;
  const uint2* pairs;        // sorted: key, and the place that it had
  float* chunks;             // [n / kChunk][d]: sums of whole runs of one row
  void* out;
  int64_t n, ld;
  uint32_t rows, range;      // range: rows of a workgroup
  int d, pieces, slices;     // slices: parts of 64 pieces of a row, a workgroup each
  int spread;                // waves of a chunk and slice, 1 or 4
  int sparse;                // most rows have no ids: zeros into all of them before anything else
  float scale;
};

__device__ __forceinline__ uint32_t place_in(uint2 pair) { return pair.y; }
__device__ __forceinline__ uint32_t place_in(uint32_t place) { return place; }

// Adds to v the piece at `at` of the gradients of places[first], places[first + 1], ... in order, some on their way at a time.
template <typename T, int V, int kUnroll, typename Place>
__device__ __forceinline__ void add_rows(float (&v)[V], const SumArgs& a, const Place* places, uint32_t first, uint32_t last, int at) {
  typedef typename piece_words<T, V>::type words;
  const T* grad = static_cast<const T*>(a.grad) + at;
  for (uint32_t i = first; i < last; i += kUnroll) {
    words w[kUnroll];
    const uint32_t left = last - i;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (u < left) w[u] = *reinterpret_cast<const words*>(grad + (int64_t)place_in(places[i + u]) * a.ld);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (u >= left) continue;
      float g[V];
      values_of<T, V>(w[u], g);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += g[e];
    }
  }
}
template <int V>
__device__ __forceinline__ void add_chunks(float (&v)[V], const SumArgs& a, uint32_t first, uint32_t last, int at) {
  constexpr int kUnroll = 8;
  for (uint32_t c = first; c < last; c += kUnroll) {
    float w[kUnroll][V];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) w[u][e] = c + u < last ? a.chunks[(int64_t)(c + u) * a.d + at + e] : 0.f;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += w[u][e];
  }
}

// Sums over the groups of `lanes` lanes of a wave, in all of them.  (One group after the other, by way of LDS, a workgroup's 256
// took 23 us.)
template <int V>
__device__ __forceinline__ void sum_shares(float (&v)[V], int lanes) {
  for (int by = lanes; by < kWave; by *= 2)
#pragma unroll
    for (int x = 0; x < V; ++x) v[x] += __shfl_xor(v[x], by);
}

// Where keys of at least `key` begin in the sorted ones from lo to hi, by the 64 lanes of a wave: 64 parts at a time.
__device__ __forceinline__ uint32_t begin_of(const uint2* pairs, uint32_t lo, uint32_t hi, uint32_t key) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  while (lo < hi) {
    const uint32_t step = (hi - lo + kWave - 1) / kWave;
    const uint64_t at = (uint64_t)lo + (uint64_t)lane * step;
    const uint32_t count = (uint32_t)__popcll(__ballot(at < hi && pairs[at < hi ? at : lo].x < key));
    if (count == 0) return lo;
    const uint64_t next = (uint64_t)lo + (uint64_t)count * step;
    lo = lo + (count - 1) * step + 1;
    hi = next < hi ? (uint32_t)next : hi;
  }
  return lo;
}

// Where each row's ids begin among the sorted ones (the last entry: where those outside the table do): a wave looks for the first of
// its 64 rows and the end of the last one, then each lane for its own row in between.  And, in the workgroups behind, sums of the
// chunks that are of one row: a wave a chunk and slice (or four), whose lanes share the chunk where the slice has few pieces.
template <typename T, int V>
__global__ __launch_bounds__(256) void starts_and_chunks_kernel(SumArgs a, uint32_t* starts, uint32_t search_blocks) {
  if (blockIdx.x < search_blocks) {
    const uint32_t r0 = blockIdx.x * 256 + threadIdx.x / kWave * kWave, r = r0 + (threadIdx.x & (kWave - 1));
    if (r0 > a.rows) return;
    uint32_t lo = begin_of(a.pairs, 0, (uint32_t)a.n, r0);
    uint32_t hi = r0 + kWave > a.rows ? (uint32_t)a.n : begin_of(a.pairs, lo, (uint32_t)a.n, r0 + kWave);
    while (lo < hi) {
      const uint32_t middle = lo + (hi - lo) / 2;
      if (a.pairs[middle].x < r) lo = middle + 1;
      else hi = middle;
    }
    if (r <= a.rows) starts[r] = lo;
    return;
  }
  __shared__ uint32_t near[4][kChunk];
  __shared__ float room[4][V][kWave];
  const int wave = threadIdx.x / kWave, quarter = a.spread == 4 ? wave : 0;
  const int64_t item = (int64_t)(blockIdx.x - search_blocks) * (4 / a.spread) + (a.spread == 4 ? 0 : wave);
  const int64_t chunk = item / a.slices;
  const int slice = (int)(item - chunk * a.slices), lane = threadIdx.x & (kWave - 1);
  if (chunk >= a.n / kChunk) return;
  const uint32_t first = (uint32_t)(chunk * kChunk);
  static_assert(kChunk == 2 * kWave, "two places a lane");
  const uint2 mine_low = a.pairs[first + lane], mine_high = a.pairs[first + kWave + lane];
  const uint32_t key = (uint32_t)__builtin_amdgcn_readfirstlane((int)mine_low.x);
  if (key != (uint32_t)__builtin_amdgcn_readlane((int)mine_high.x, kWave - 1) || key >= a.rows) return;
  uint32_t* places = near[wave];               // (within a wave: LDS keeps its order)
  places[lane] = mine_low.y;
  places[kWave + lane] = mine_high.y;
  __builtin_amdgcn_wave_barrier();
  const int here = a.pieces - slice * kWave < kWave ? a.pieces - slice * kWave : kWave;
  int lanes = 1;
  while (lanes < here) lanes *= 2;
  const int shares = kWave / lanes, share = lane / lanes, sub = lane & (lanes - 1);
  const int p = slice * kWave + (sub < here ? sub : here - 1);
  const int at = p * V + V > a.d ? a.d - V : p * V;
  float v[V] = {};
  const uint32_t all = shares * a.spread, mine = quarter * shares + share;      // (up to 256 shares of the 128)
  add_rows<T, V, 8>(v, a, places, kChunk * mine / all, kChunk * (mine + 1) / all, at);
  sum_shares<V>(v, lanes);
  if (a.spread == 4) {                         // (the workgroup has one item: all of it is here)
#pragma unroll
    for (int e = 0; e < V; ++e) room[wave][e][lane] = v[e];
    __syncthreads();
#pragma unroll
    for (int w = 1; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += room[w][e][lane];
    if (wave != 0) return;
  }
  if (share != 0 || sub >= here) return;
  float* to = a.chunks + chunk * a.d + at;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (at + e >= p * V) to[e] = v[e];         // (a piece that was moved back: its own columns)
}

// Zeros into rows of a workgroup's range and slice: those that wanted(row) is true of.
template <typename T, int V, int THREADS, typename Wanted>
__device__ __forceinline__ void zero_rows(const SumArgs& a, uint32_t row0, uint32_t count, int slice, const Wanted& wanted) {
  const int here = a.pieces - slice * kWave < kWave ? a.pieces - slice * kWave : kWave;       // pieces of the slice
  int lanes = 1;
  while (lanes < here) lanes *= 2;
  const int sub = threadIdx.x & (lanes - 1), p = slice * kWave + sub;
  if (sub >= here) return;
  const int at = p * V + V > a.d ? a.d - V : p * V;
  const float zero[V] = {};
  T* out = static_cast<T*>(a.out) + (int64_t)row0 * a.d + at;
  for (uint32_t r = threadIdx.x / lanes; r < count; r += THREADS / lanes) {
    if (!wanted(r)) continue;
    // (a piece that was moved back: its own columns, for those before may hold another slice's sums by now)
    if (at == p * V) store_piece<T, V>(out + (int64_t)r * a.d, zero);
    else
#pragma unroll
      for (int x = 0; x < V; ++x)
        if (at + x >= p * V) out[(int64_t)r * a.d + x] = (T)0.f;
  }
}

// Rows of a workgroup's range that have ids, few and many (in any order: each is a sum of its own).
struct RowLists {
  uint32_t* rows;              // those with up to kLong ids from the front, those with more from the back
  uint32_t* counts;            // of both
};
template <int THREADS>
__device__ __forceinline__ void list_rows(uint32_t count, const uint32_t* start, const RowLists& lists) {
  for (uint32_t r = threadIdx.x; r < count; r += THREADS) {
    const uint32_t ids = start[r + 1] - start[r];
    if (ids > kLong) lists.rows[count - 1 - atomicAdd(&lists.counts[1], 1u)] = r;
    else if (ids > 0) lists.rows[atomicAdd(&lists.counts[0], 1u)] = r;
  }
}

// Their sums: the places of row r's ids lie in order in places[start[r] - skipped .. start[r + 1] - skipped).  `room` holds a piece a lane.
template <typename T, int V, int THREADS, int ROWS, int LONG_UNROLL, typename Place>
__device__ __forceinline__ void sum_range(const SumArgs& a, uint32_t row0, uint32_t count, int slice, const uint32_t* start,
                                          const Place* places, uint32_t skipped, bool chunked, const RowLists& lists, float* room) {
  constexpr int kWaves = THREADS / kWave;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int here = a.pieces - slice * kWave < kWave ? a.pieces - slice * kWave : kWave;       // pieces of the slice
  int lanes = 1;
  while (lanes < here) lanes *= 2;
  const int groups = kWave / lanes, sub = lane & (lanes - 1);
  const int p = slice * kWave + (sub < here ? sub : here - 1);
  const int at = p * V + V > a.d ? a.d - V : p * V;
  const uint32_t few = lists.counts[0], longs = lists.counts[1];
  // Some rows to a group of lanes at a time, whose first two ids are all on their way at once: most rows have no more.
  constexpr int kRows = ROWS, kFirst = 2;
  typedef typename piece_words<T, V>::type words;
  const uint32_t apart = (uint32_t)(kWaves * groups);
  for (uint32_t l0 = (uint32_t)(wave * groups + lane / lanes); l0 < few; l0 += apart * kRows) {
    uint32_t r[kRows], s[kRows], e[kRows];
    words w[kRows][kFirst];
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const uint32_t l = l0 + q * apart;
      r[q] = lists.rows[l < few ? l : few - 1];
      s[q] = start[r[q]] - skipped;
      e[q] = l < few ? start[r[q] + 1] - skipped : s[q];
#pragma unroll
      for (int u = 0; u < kFirst; ++u)          // (the first one twice where there is no second)
        w[q][u] = *reinterpret_cast<const words*>(static_cast<const T*>(a.grad) + at +
                                                  (int64_t)place_in(places[s[q] + u < e[q] ? s[q] + u : s[q]]) * a.ld);
    }
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      float v[V] = {}, g[V];
#pragma unroll
      for (int u = 0; u < kFirst; ++u) {
        values_of<T, V>(w[q][u], g);
#pragma unroll
        for (int x = 0; x < V; ++x) v[x] = s[q] + u < e[q] ? v[x] + g[x] : v[x];
      }
      if (s[q] + kFirst < e[q]) add_rows<T, V, 8>(v, a, places, s[q] + kFirst, e[q], at);
#pragma unroll
      for (int x = 0; x < V; ++x) v[x] *= a.scale;
      if (sub < here && l0 + q * apart < few) store_piece<T, V>(static_cast<T*>(a.out) + (int64_t)(row0 + r[q]) * a.d + at, v);
    }
  }
  // Of a row with many ids each group of lanes has a share, in the groups' order.
  const int shares = kWaves * groups, share = wave * groups + lane / lanes;
  for (uint32_t l = 0; l < longs; ++l) {
    const uint32_t r = lists.rows[count - 1 - l], s = start[r], e = start[r + 1];
    uint32_t c0 = (s + kChunk - 1) / kChunk, c1 = e / kChunk;
    if (!chunked || c0 >= c1) { c0 = 0; c1 = 0; }
    const uint32_t head = c0 < c1 ? c0 * kChunk : e, tail = c0 < c1 ? c1 * kChunk : e;
    auto part = [&](uint32_t from, uint32_t to, int w) { return from + (uint32_t)((uint64_t)(to - from) * w / shares); };
    float v[V] = {};
    add_rows<T, V, LONG_UNROLL>(v, a, places, part(s, head, share) - skipped, part(s, head, share + 1) - skipped, at);
    if (chunked) {
      add_chunks<V>(v, a, part(c0, c1, share), part(c0, c1, share + 1), at);
      add_rows<T, V, LONG_UNROLL>(v, a, places, part(tail, e, share) - skipped, part(tail, e, share + 1) - skipped, at);
    }
    sum_shares<V>(v, lanes);
    __syncthreads();                           // (the row before is done with the room)
    if (lane < lanes)
#pragma unroll
      for (int x = 0; x < V; ++x) room[(wave * V + x) * kWave + lane] = v[x];
    __syncthreads();
    if (wave == 0 && lane < here) {
#pragma unroll
      for (int x = 0; x < V; ++x) v[x] = 0.f;
#pragma unroll 4
      for (int w = 0; w < kWaves; ++w)
#pragma unroll
        for (int x = 0; x < V; ++x) v[x] += room[(w * V + x) * kWave + lane];
#pragma unroll
      for (int x = 0; x < V; ++x) v[x] *= a.scale;
      // (a piece that was moved back leaves the columns of the one before to that: another slice may share the row otherwise)
      T* out = static_cast<T*>(a.out) + (int64_t)(row0 + r) * a.d + at;
      if (at == p * V) store_piece<T, V>(out, v);
      else
#pragma unroll
        for (int x = 0; x < V; ++x)
          if (at + x >= p * V) out[x] = (T)v[x];
    }
  }
}

// From sorted ids.
constexpr uint32_t kRangeSorted = 64;        // rows of a workgroup, at most
constexpr int kSumThreads = 256;
template <typename T, int V>
__global__ __launch_bounds__(kSumThreads) void sorted_sums_kernel(SumArgs a, const uint32_t* starts) {
  constexpr uint32_t kNear = 1024;             // places of the range, brought near where they fit: a round trip less for each row
  __shared__ uint32_t start[kRangeSorted + 1], few[kRangeSorted], counts[2], near[kNear];
  __shared__ float room[kSumThreads * V];
  const uint32_t range = blockIdx.x / a.slices, row0 = range * a.range;
  const int slice = (int)(blockIdx.x - range * a.slices);
  const uint32_t count = a.rows - row0 < a.range ? a.rows - row0 : a.range;
  if (threadIdx.x < 2) counts[threadIdx.x] = 0;
  if (threadIdx.x <= count) start[threadIdx.x] = starts[row0 + threadIdx.x];
  __syncthreads();
  const RowLists lists{few, counts};
  const uint32_t first = start[0], ids = start[count] - first;
  if (ids <= kNear)
    for (uint32_t i = threadIdx.x; i < ids; i += kSumThreads) near[i] = a.pairs[first + i].y;
  list_rows<kSumThreads>(count, start, lists);
  zero_rows<T, V, kSumThreads>(a, row0, count, slice, [&](uint32_t r) { return start[r + 1] == start[r]; });
  __syncthreads();
  if (ids <= kNear) sum_range<T, V, kSumThreads, 4, 8>(a, row0, count, slice, start, near, first, true, lists, room);
  else sum_range<T, V, kSumThreads, 4, 8>(a, row0, count, slice, start, a.pairs, 0, true, lists, room);
}

// From ids as they come: those of the range are kept in their order, then sorted by row.
constexpr int kPickMost = 16384, kPickThreads = 1024, kPickWaves = kPickThreads / kWave, kRangePicked = 1024;

// Where things lie in LDS, in bytes, which is as large as the call's ids and range ask for: two workgroups are to fit a CU.
struct PickRoom {
  uint32_t sorted, own, start, few, all;
  __host__ __device__ PickRoom(uint32_t n, uint32_t range, int values) {
    const uint32_t kept = 4 * n, sums = (uint32_t)(kPickThreads * values * 4);      // (the waves' sums take the place of the kept ids)
    sorted = ((kept > sums ? kept : sums) + 15) / 16 * 16;
    own = sorted + (2 * n + 15) / 16 * 16;
    start = own + kPickWaves * 2 * ((range + 1) / 2 * 2);
    few = start + 4 * (range + 1);
    all = few + 4 * range;
  }
};

template <typename T, int V, typename Idx>
__global__ __launch_bounds__(kPickThreads, 8) void picked_sums_kernel(SumArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ uint32_t room_words[kPickWaves], list_counts[2];
  const PickRoom at_lds((uint32_t)a.n, a.range, V);
  uint32_t* kept = reinterpret_cast<uint32_t*>(lds);                         // place | row in the range << 14, in the places' order
  uint16_t* sorted = reinterpret_cast<uint16_t*>(lds + at_lds.sorted);       // places by row
  uint32_t* start = reinterpret_cast<uint32_t*>(lds + at_lds.start);
  const RowLists lists{reinterpret_cast<uint32_t*>(lds + at_lds.few), list_counts};
  const uint32_t part = blockIdx.x / a.slices, row0 = part * a.range;
  const int slice = (int)(blockIdx.x - part * a.slices);
  const uint32_t count = a.rows - row0 < a.range ? a.rows - row0 : a.range;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const uint32_t each = (a.range + 1) / 2 * 2;
  uint16_t* all_own = reinterpret_cast<uint16_t*>(lds + at_lds.own);         // [waves][each]
  uint16_t* own = all_own + wave * each;
  const Idx* index = static_cast<const Idx*>(a.index);
  if (threadIdx.x < 2) list_counts[threadIdx.x] = 0;
  for (uint32_t r = threadIdx.x; r <= count; r += kPickThreads) start[r] = 0;
  for (uint32_t r = lane; r < each; r += kWave) own[r] = 0;
  // a wave reads a run of the ids: how many of them it keeps, then where
  const uint32_t n = (uint32_t)a.n, run = (n + kPickWaves * kWave - 1) / (kPickWaves * kWave) * kWave;
  const uint32_t first = wave * run, last = first + run < n ? first + run : n;
  constexpr int kMost = kPickMost / kPickThreads;
  Idx raw[kMost];
  uint32_t local[kMost], mine = 0;
#pragma unroll
  for (int u = 0; u < kMost; ++u) {
    const uint32_t i = first + u * kWave + lane;
    raw[u] = -1;
    if (u * kWave < (int)run && i < last) raw[u] = index[i];
  }
  // (their stores are waited for with the ids, in front of the first key: they hide the ids' way and nothing behind it)
  if (a.sparse) zero_rows<T, V, kPickThreads>(a, row0, count, slice, [](uint32_t) { return true; });
#pragma unroll
  for (int u = 0; u < kMost; ++u) {
    const uint32_t key = key_of(raw[u], a.rows), in = key - row0;
    local[u] = key < a.rows && key >= row0 && in < count ? in : ~0u;
  }
#pragma unroll
  for (int u = 0; u < kMost; ++u) mine += (uint32_t)__popcll(__ballot(local[u] != ~0u));
  if (lane == 0) room_words[wave] = mine;
  __syncthreads();
  uint32_t at = 0, all = 0;
  for (int w = 0; w < kPickWaves; ++w) {
    if (w < wave) at += room_words[w];
    all += room_words[w];
  }
#pragma unroll
  for (int u = 0; u < kMost; ++u) {
    const uint64_t with = __ballot(local[u] != ~0u);
    if (local[u] != ~0u) {
      kept[at + below(with)] = (first + u * kWave + lane) | local[u] << 14;
      atomicAdd(&start[local[u]], 1u);
    }
    at += (uint32_t)__popcll(with);
  }
  __syncthreads();
  // the kept ids by row: again a run of them to each wave
  const uint32_t share = (all + kPickWaves * kWave - 1) / (kPickWaves * kWave) * kWave;
  const uint32_t begin = wave * share < all ? wave * share : all, end = begin + share < all ? begin + share : all;
  for (uint32_t i = begin + lane; i < end; i += kWave) {
    // (16-bit counters, two to a word)
    const uint32_t r = kept[i] >> 14;
    atomicAdd(reinterpret_cast<uint32_t*>(own + (r & ~1u)), r & 1 ? 0x10000u : 1u);
  }
  prefix_in_lds<kPickThreads>(start, count + 1, room_words);
  __syncthreads();
  list_rows<kPickThreads>(count, start, lists);
  if (!a.sparse) zero_rows<T, V, kPickThreads>(a, row0, count, slice, [&](uint32_t r) { return start[r + 1] == start[r]; });
  for (uint32_t r = threadIdx.x; r < count; r += kPickThreads) {
    uint32_t before = 0;
    for (int w = 0; w < kPickWaves; ++w) {
      const uint32_t c = all_own[w * each + r];
      all_own[w * each + r] = (uint16_t)before;    // (up to 16384: 16 bits hold it)
      before += c;
    }
  }
  __syncthreads();
  const int bits = bits_of(count - 1);
  for (uint32_t i = begin; i < end; i += kWave) {
    const bool on = i + lane < end;
    const uint32_t word = on ? kept[i + lane] : 0, r = word >> 14;
    const uint64_t same = same_digit(r, bits, on);
    const uint32_t rank = below(same);
    if (on) sorted[start[r] + own[r] + rank] = (uint16_t)(word & (kPickMost - 1));
    __builtin_amdgcn_wave_barrier();
    if (on && rank == 0) own[r] += (uint16_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
  // This wave's zeros are written, before any wave writes sums: said here, whatever was waited for on the way.
  if (a.sparse) __builtin_amdgcn_s_waitcnt(7 << 4 | 15 << 8);
  __syncthreads();
  sum_range<T, V, kPickThreads, 1, 8>(a, row0, count, slice, start, sorted, 0, false, lists, reinterpret_cast<float*>(lds));
}

// Whether ids are picked rather than sorted: up to as many as LDS is laid out for (11264 of 100000 x 128 in fp32 18 us, sorted 39), but not
// thousands of one to three rows, which are a workgroup's each (16384 of one row of 128 113 us, sorted 33; 4000 31 and 31).
bool picks(int64_t n, int64_t rows) { return n <= kPickMost && (n <= 4096 || rows >= 4); }

// Digits of the sort: as few as keys of rows + 1 values need, of one width.
void digits_of(int64_t rows, int& passes, int& bits) {
  const int all = bits_of((uint32_t)rows);
  passes = (int)ceil_div(all, kMostBits);
  bits = (int)ceil_div(all, passes);
}

struct Room {
  int64_t sorted, counts, starts, chunks;    // bytes: pairs twice, counts of the digits, the rows' starts, sums of chunks
  explicit Room(int64_t n, int64_t rows, int64_t d) {
    int passes, bits;
    digits_of(rows, passes, bits);
    sorted = ceil_div(n, 2) * 16 * 2;
    counts = ceil_div((1ll << bits) * (ceil_div(n, kSortTile) + 1), 4) * 16;
    starts = ceil_div(rows + 1, 4) * 16;
    chunks = n / kChunk * d * 4;
  }
};

int check_embedding(const char* what, int64_t n, int64_t rows, int64_t d, int idx_dtype, int dtype) {
  F2CGT_REQUIRE(n >= 0 && rows >= 0 && d >= 0, F2CGT_E_INVALID, "%s: sizes must not be negative", what);
  F2CGT_REQUIRE(idx_dtype == F2CGT_DT_I32 || idx_dtype == F2CGT_DT_I64, F2CGT_E_UNSUPPORTED, "%s: ids must be int32 or int64", what);
  F2CGT_REQUIRE(dtype == F2CGT_DT_F32 || dtype == F2CGT_DT_F16 || dtype == F2CGT_DT_BF16, F2CGT_E_UNSUPPORTED,
                "%s: fp32, fp16 or bf16 rows only", what);
  F2CGT_REQUIRE(n < (1ll << 31) && rows < (1ll << 31) && d < (1ll << 24), F2CGT_E_UNSUPPORTED,
                "%s: at most 2^31 - 1 ids and rows and 2^24 - 1 columns", what);
  return 0;
}

template <typename T, int V>
int launch_lookup(LookupArgs a, int idx_dtype, hipStream_t st) {
  a.pieces = (int)ceil_div(a.d, V);
  a.lanes = a.pieces >= kWave ? kWave : pow2_ceil(a.pieces);
  const int64_t blocks = ceil_div(a.n, 4 * (256 / a.lanes));
  F2CGT_REQUIRE(blocks < (1ll << 24), F2CGT_E_UNSUPPORTED, "embedding: too many ids for a launch");
  const dim3 grid((unsigned)blocks);
  if (idx_dtype == F2CGT_DT_I64) lookup_kernel<T, V, int64_t><<<grid, dim3(256), 0, st>>>(a);
  else lookup_kernel<T, V, int32_t><<<grid, dim3(256), 0, st>>>(a);
  return launch_status("embedding");
}

template <typename T, int V>
int launch_grad(SumArgs a, int idx_dtype, char* workspace, hipStream_t st) {
  const char* what = "embedding_grad";
  a.pieces = (int)ceil_div(a.d, V);
  a.slices = (int)ceil_div(a.pieces, kWave);
  if (picks(a.n, a.rows)) {
    // A workgroup for each CU, since each reads all ids: 16384 ids of 20000 x 128 in fp32 12.3 us, with two for each 19.7, 1000 of them 10.4
    // and 14.0.  Two where zeros are most of it (11264 of 300000 x 128 in fp32, 600 KB a CU, 34.5 us, with one 44.2; of 100000 x 128 with
    // hot ids 21.3 and 22.8, but where LDS has no room for both, 16384 of them, 31.2 and 27.1), and where LDS has no counters for a
    // CU's rows.
    const int64_t cus = num_cus(), one = ceil_div((int64_t)a.rows * a.slices, cus), two = ceil_div((int64_t)a.rows * a.slices, 2 * cus);
    const uint32_t range = (uint32_t)(two > kRangePicked ? kRangePicked : two);
    const bool both = 2 * PickRoom((uint32_t)a.n, range, V).all <= 160 * 1024;
    const bool alone = one <= kRangePicked && (int64_t)a.rows * a.d * (int64_t)sizeof(T) <= cus * (both ? 131072 : 262144);
    a.range = alone ? (uint32_t)one : range;
    const int64_t blocks = ceil_div(a.rows, a.range) * a.slices;
    F2CGT_REQUIRE(blocks < (1ll << 22), F2CGT_E_UNSUPPORTED, "%s: too many rows for a launch", what);
    const uint32_t lds = PickRoom((uint32_t)a.n, a.range, V).all;
    auto kernel = idx_dtype == F2CGT_DT_I64 ? picked_sums_kernel<T, V, int64_t> : picked_sums_kernel<T, V, int32_t>;
    if (lds > 65536) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return fail((int)e, "%s: %s", what, hipGetErrorString(e));
    }
    kernel<<<dim3((unsigned)blocks), dim3(kPickThreads), lds, st>>>(a);
    return launch_status(what);
  }
  const Room room(a.n, a.rows, a.d);
  int passes, bits;
  digits_of(a.rows, passes, bits);
  // fewer rows to a workgroup until there are four for each CU: 40000 ids of 1000 x 128 in fp32 29 us, of 64 rows each 104
  a.range = kRangeSorted;
  while (a.range > 4 && ceil_div((int64_t)a.rows, a.range) * a.slices < 4 * num_cus()) a.range /= 2;
  const int64_t blocks = ceil_div(a.n, kSortTile), sums = ceil_div((int64_t)a.rows, a.range) * a.slices;
  // Four waves to a chunk where the chunks alone are few: 26 906 hot ids of 82 859 x 152 in fp32 62 us, with one 98.
  const int64_t items = a.n / kChunk * a.slices;
  a.spread = items < 16 * num_cus() ? 4 : 1;
  const int64_t chunk_blocks = ceil_div(items * a.spread, 4);
  F2CGT_REQUIRE(sums < (1ll << 23) && chunk_blocks < (1ll << 23), F2CGT_E_UNSUPPORTED, "%s: too many values for a launch", what);
  uint2* pairs = reinterpret_cast<uint2*>(workspace);
  const int64_t each = ceil_div(a.n, 2) * 2;
  SortArgs s{a.index, nullptr, nullptr, reinterpret_cast<uint32_t*>(workspace + room.sorted), a.n, a.rows, (uint32_t)blocks, 0, bits};
  const dim3 grid((unsigned)blocks), digits(1u << bits);
  for (int pass = 0; pass < passes; ++pass) {
    s.shift = pass * bits;
    s.pairs = pairs + (pass & 1 ? 0 : each);
    s.pairs_out = pairs + (pass & 1 ? each : 0);
    if (pass > 0) {
      sort_count_kernel<int32_t, false><<<grid, dim3(kSortThreads), 0, st>>>(s);
      sort_prefix_kernel<<<digits, dim3(kWave), 0, st>>>(s);
      sort_scatter_kernel<int32_t, false><<<grid, dim3(kSortThreads), 0, st>>>(s);
    } else if (idx_dtype == F2CGT_DT_I64) {
      sort_count_kernel<int64_t, true><<<grid, dim3(kSortThreads), 0, st>>>(s);
      sort_prefix_kernel<<<digits, dim3(kWave), 0, st>>>(s);
      sort_scatter_kernel<int64_t, true><<<grid, dim3(kSortThreads), 0, st>>>(s);
    } else {
      sort_count_kernel<int32_t, true><<<grid, dim3(kSortThreads), 0, st>>>(s);
      sort_prefix_kernel<<<digits, dim3(kWave), 0, st>>>(s);
      sort_scatter_kernel<int32_t, true><<<grid, dim3(kSortThreads), 0, st>>>(s);
    }
  }
  a.pairs = s.pairs_out;
  uint32_t* starts = reinterpret_cast<uint32_t*>(workspace + room.sorted + room.counts);
  a.chunks = reinterpret_cast<float*>(workspace + room.sorted + room.counts + room.starts);
  const int64_t search_blocks = ceil_div((int64_t)a.rows + 1, 256);
  starts_and_chunks_kernel<T, V><<<dim3((unsigned)(search_blocks + chunk_blocks)), dim3(256), 0, st>>>(a, starts, (uint32_t)search_blocks);
  sorted_sums_kernel<T, V><<<dim3((unsigned)sums), dim3(kSumThreads), 0, st>>>(a, starts);
  return launch_status(what);
}

}  // namespace
}  // namespace f2cgt

using namespace f2cgt;

extern "C" int f2cgt_embedding(const void* table, int dtype, int64_t ld, const void* index, int idx_dtype, void* out, float scale,
                               int64_t n, int64_t rows, int64_t d, void* stream) {
  const char* what = "embedding";
  if (int rc = check_embedding(what, n, rows, d, idx_dtype, dtype)) return rc;
  F2CGT_REQUIRE(rows <= 1 || ld >= d, F2CGT_E_INVALID, "%s: rows overlap", what);
  if (n == 0 || d == 0) return 0;
  F2CGT_REQUIRE((rows == 0 || table) && index && out, F2CGT_E_INVALID, "%s: null buffer", what);
  const int size = dtype == F2CGT_DT_F32 ? 4 : 2;
  F2CGT_REQUIRE(aligned(table, size) && aligned(out, size) && aligned(index, idx_dtype == F2CGT_DT_I64 ? 8 : 4), F2CGT_E_INVALID,
                "%s: misaligned buffer", what);
  const LookupArgs a{table, index, out, n, ld, (uint32_t)rows, (int)d, 0, 0, scale};
  return with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (d >= kPieceOf<T>) return launch_lookup<T, kPieceOf<T>>(a, idx_dtype, as_stream(stream));
    return launch_lookup<T, 1>(a, idx_dtype, as_stream(stream));
  });
}

extern "C" int64_t f2cgt_embedding_grad_workspace_bytes(int64_t n, int64_t rows, int64_t d) {
  if (rows <= 0 || picks(n, rows) || d <= 0 || n >= (1ll << 31) || rows >= (1ll << 31)) return 0;
  const Room room(n, rows, d);
  return room.sorted + room.counts + room.starts + room.chunks;
}

extern "C" int f2cgt_embedding_grad(const void* grad, int dtype, int64_t ld, const void* index, int idx_dtype, void* dtable,
                                    float scale, void* workspace, int64_t workspace_bytes, int64_t n, int64_t rows, int64_t d,
                                    void* stream) {
  const char* what = "embedding_grad";
  if (int rc = check_embedding(what, n, rows, d, idx_dtype, dtype)) return rc;
  F2CGT_REQUIRE(n <= 1 || ld >= d, F2CGT_E_INVALID, "%s: rows overlap", what);
  if (rows == 0 || d == 0) return 0;
  F2CGT_REQUIRE((n == 0 || (grad && index)) && dtable, F2CGT_E_INVALID, "%s: null buffer", what);
  const int size = dtype == F2CGT_DT_F32 ? 4 : 2;
  F2CGT_REQUIRE(aligned(grad, size) && aligned(dtable, size) && aligned(index, idx_dtype == F2CGT_DT_I64 ? 8 : 4), F2CGT_E_INVALID,
                "%s: misaligned buffer", what);
  const int64_t need = f2cgt_embedding_grad_workspace_bytes(n, rows, d);
  F2CGT_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), F2CGT_E_INVALID,
                "%s: workspace too small or misaligned", what);
  const SumArgs a{grad, index, nullptr, nullptr, dtable, n, ld, (uint32_t)rows, 0, (int)d, 0, 0, 1, rows > n, scale};
  return with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (d >= kPieceOf<T>) return launch_grad<T, kPieceOf<T>>(a, idx_dtype, static_cast<char*>(workspace), as_stream(stream));
    return launch_grad<T, 1>(a, idx_dtype, static_cast<char*>(workspace), as_stream(stream));
  });
}
