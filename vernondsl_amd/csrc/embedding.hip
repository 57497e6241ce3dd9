// Token embedding: the scaled lookup of table rows, and the table's gradient.
//
//   out[i] = scale table[ids[i]],  dtable[v] = scale (sum over the i with ids[i] = v, in ascending i, of dy[i]);
// an id outside [0, vocab) is no row: its output is zero and it adds to no row's gradient.
//
// Both are bound by HBM.  The lookup reads each row where it is and writes the output once (16384 x 4096, bf16 rows
// into f32: 56 us, 6.2 TB/s).  The gradient
// does not add into the table with atomics, whose order would change its bits from run to run: the
// positions are sorted by token (stably, so a token's positions ascend), and then every row of dtable is
// written once, zero or the f32 sum of its terms (16384 positions, 32768 x 4096: sorting 11 us, chunks 8, rows 97 to
// 112 for 588 MB; 300 positions, 5003 x 1001, back to back: 6.2 with uniform ids, 6.8 to 9.2 with ids as frequent as
// words, whose most frequent token's row is the last one done).

#include <algorithm>
#include <type_traits>

#include "rowunit.h"

namespace vdsl {
namespace {

// A value that is the same for all lanes of a wave, as a scalar.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// 2^log_l lanes per output row, KU units of U elements each; blockIdx.y: strips of columns.
template <int TT, int OT, int U, int KU, bool STREAM>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* __restrict__ table, const int32_t* __restrict__ ids,
                                                            void* __restrict__ out, int64_t n, int64_t dim, int64_t vocab,
                                                            float scale, int log_l) {
  const int lanes = 1 << log_l;
  const int64_t i = (block_index() << (8 - log_l)) + (threadIdx.x >> log_l);
  if (i >= n) return;
  const int32_t id = ids[i];
  const bool valid = id >= 0 && id < vocab;
  const int64_t row = valid ? id : 0;
  const int64_t c0 = (static_cast<int64_t>(blockIdx.y) * KU * lanes + (threadIdx.x & (lanes - 1))) * U;
  float v[KU][U];
#pragma unroll
  for (int k = 0; k < KU; ++k) load_whole<TT, U>(table, row * dim + UnitAt<U>(c0 + static_cast<int64_t>(k) * lanes * U, dim).c, v[k]);
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    const UnitAt<U> at(c0 + static_cast<int64_t>(k) * lanes * U, dim);
#pragma unroll
    for (int j = 0; j < U; ++j) v[k][j] = valid ? v[k][j] * scale : 0.0f;
    if (at.any()) store_whole<OT, U, STREAM>(out, i * dim + at.c, v[k]);
  }
}

__global__ __launch_bounds__(256) void embedding_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) p[i] = 0;
}

// ---- positions sorted by token -------------------------------------------------------------------
// Every row's places [x, y) among the sorted positions, none at first.
__device__ __forceinline__ void clear_places(int2* __restrict__ places, int64_t vocab) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t v = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; v < vocab; v += step) places[v] = make_int2(0, 0);
}

// Up to 32768 positions, in tiles of kRankTile.  In a tile position i goes to place #{j : id_j < id_i} + #{j < i : id_j = id_i}.  A block
// ranks 64 positions, one a lane, its 16 waves a share of the ids each.  Ids are compared as unsigned
// numbers, so those that are no row come last.  A second kernel
// adds to an element's rank what the other tiles have before it, a binary search in each.  Us of a gradient of 256
// columns, vocabulary 32768, sorted so and by radix passes: n 4096 20.7, 30.9; 16384 22.1, 31.2; 32768 27.4, 34.3; 65536
// 47.8, 40.3.
constexpr int kRankTile = 1024;

__global__ __launch_bounds__(1024) void embedding_rank_kernel(const int32_t* __restrict__ ids, int n, uint32_t* __restrict__ sorted,
                                                              int32_t* __restrict__ order, int2* __restrict__ places, int64_t vocab) {
  clear_places(places, vocab);
  __shared__ int part[16][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int i0 = static_cast<int>(blockIdx.x) * 64, i = i0 + lane, tile = i0 / kRankTile * kRankTile;
  const uint32_t key = i < n ? static_cast<uint32_t>(ids[i]) : 0;
  constexpr int kShare = kRankTile / 16;
  const int j0 = tile + wave * kShare, j1 = min(j0 + kShare, n);
  int rank = 0;
  if (j0 == i0) {  // the ids at the block's own positions
    for (int j = j0; j < j1; ++j) {
      const uint32_t other = static_cast<uint32_t>(ids[j]);
      rank += other < key || (other == key && j < i);
    }
  } else if (j0 < i0) {  // before them
#pragma unroll 16
    for (int j = j0; j < j1; ++j) rank += static_cast<uint32_t>(ids[j]) <= key;
  } else {
#pragma unroll 16
    for (int j = j0; j < j1; ++j) rank += static_cast<uint32_t>(ids[j]) < key;
  }
  part[wave][lane] = rank;
  __syncthreads();
  if (wave != 0 || i >= n) return;
  rank = tile;
#pragma unroll
  for (int w = 0; w < 16; ++w) rank += part[w][lane];
  sorted[rank] = key;
  order[rank] = i;
}
static_assert(kRankTile / 16 == 64, "a wave's share of the ids is a block's positions, or lies on one side of them");

__global__ __launch_bounds__(1024) void embedding_merge_kernel(const uint32_t* __restrict__ tiles, const int32_t* __restrict__ from, int n,
                                                               uint32_t* __restrict__ sorted, int32_t* __restrict__ order) {
  __shared__ int part[16][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int e0 = static_cast<int>(blockIdx.x) * 64, e = e0 + lane, mine = e0 / kRankTile;
  const uint32_t key = tiles[e < n ? e : n - 1];
  int rank = 0;
  for (int t = wave; t * kRankTile < n; t += 16) {
    if (t == mine) continue;
    // equal tokens of an earlier tile come first
    const uint64_t bound = static_cast<uint64_t>(key) + (t < mine ? 1 : 0);
    int lo = 0, hi = min(kRankTile, n - t * kRankTile);
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (tiles[t * kRankTile + mid] < bound) lo = mid + 1;
      else hi = mid;
    }
    rank += lo;
  }
  part[wave][lane] = rank;
  __syncthreads();
  if (wave != 0 || e >= n) return;
  rank = e - mine * kRankTile;
#pragma unroll
  for (int w = 0; w < 16; ++w) rank += part[w][lane];
  sorted[rank] = key;
  order[rank] = from[e];
}

// Many: a radix sort from the lowest of the tokens' 8-bit digits up, each pass stable.  The positions lie
// in tiles; hist[pass][tile][digit] counts a pass's digits in each tile of its input.  The first pass's
// counts come from a kernel of their own, a later pass's from the pass before, which adds to them where
// it puts a position (whole numbers: their order changes nothing).
constexpr int kDigits = 256;

__device__ __forceinline__ uint32_t token_key(int32_t id, uint32_t vocab) {  // those that are no row last
  return static_cast<uint32_t>(id) < vocab ? static_cast<uint32_t>(id) : vocab;
}

__global__ __launch_bounds__(256) void embedding_count_kernel(const int32_t* __restrict__ ids, int n, uint32_t vocab, int tile,
                                                              int* __restrict__ hist, int passes, int2* __restrict__ places) {
  __shared__ int count[kDigits];
  clear_places(places, vocab);
  count[threadIdx.x] = 0;
  __syncthreads();
  const int i0 = static_cast<int>(blockIdx.x) * tile, i1 = min(i0 + tile, n);
  for (int i = i0 + static_cast<int>(threadIdx.x); i < i1; i += 256) atomicAdd(&count[token_key(ids[i], vocab) & 255u], 1);
  __syncthreads();
  const size_t at = static_cast<size_t>(blockIdx.x) * kDigits + threadIdx.x, pass = static_cast<size_t>(gridDim.x) * kDigits;
  hist[at] = count[threadIdx.x];
  for (int p = 1; p < passes; ++p) hist[p * pass + at] = 0;
}

// One pass, a tile per block, a quarter of it per wave.  keys null: the first pass, which takes the ids.
__global__ __launch_bounds__(256) void embedding_radix_kernel(const int32_t* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                              const int32_t* __restrict__ from, int n, uint32_t vocab, int tile,
                                                              int shift, const int* __restrict__ hist, int* __restrict__ next_hist,
                                                              uint32_t* __restrict__ out_keys, int32_t* __restrict__ out_order) {
  __shared__ int place[4][kDigits];  // the next place of a digit for each wave
  __shared__ int wave_total[4];
  const int b = threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i0 = static_cast<int>(blockIdx.x) * tile, i1 = min(i0 + tile, n);
  const int quarter = tile / 4, w0 = min(i0 + wave * quarter, i1), w1 = min(w0 + quarter, i1);
  int before = 0, total = 0;
#pragma unroll 8
  for (int t = 0; t < static_cast<int>(gridDim.x); ++t) {
    const int c = hist[static_cast<size_t>(t) * kDigits + b];
    total += c;
    before += t < static_cast<int>(blockIdx.x) ? c : 0;
  }
  int scan = total;  // of the digits below: within the wave, then of the waves before
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(scan, d, 64);
    if (lane >= d) scan += up;
  }
  if (lane == 63) wave_total[wave] = scan;
#pragma unroll
  for (int w = 0; w < 4; ++w) place[w][b] = 0;
  __syncthreads();
  int start = scan - total + before;
  for (int w = 0; w < wave; ++w) start += wave_total[w];
  const auto key_at = [&](int i) { return keys ? keys[i] : token_key(ids[i], vocab); };
  for (int i = w0 + lane; i < w1; i += 64) atomicAdd(&place[wave][(key_at(i) >> shift) & 255u], 1);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int c = place[w][b];
    place[w][b] = start;
    start += c;
  }
  __syncthreads();
  volatile int* const mine = place[wave];  // this wave's alone: its LDS accesses keep their order
  for (int c0 = w0; c0 < w1; c0 += 64) {
    const int i = c0 + lane;
    const bool in = i < w1;
    const uint32_t key = in ? key_at(i) : 0;
    const uint32_t digit = (key >> shift) & 255u;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const bool set = (digit >> bit) & 1u;
      const uint64_t ones = __ballot(set);
      same &= set ? ones : ~ones;
    }
    const int below = __popcll(same & ((uint64_t{1} << lane) - 1));
    if (in) {
      const int at = mine[digit] + below;
      if ((same >> lane) >> 1 == 0) mine[digit] = at + 1;  // the last lane of this digit
      out_keys[at] = key;
      out_order[at] = keys ? from[i] : i;
      if (next_hist) atomicAdd(&next_hist[static_cast<size_t>(at / tile) * kDigits + ((key >> (shift + 8)) & 255u)], 1);
    }
  }
}

// ---- the rows' sums ------------------------------------------------------------------------------
// A wave of the following kernels works on one row at a time (several waves share a wide one), so where a
// row is and which positions it sums is the same for all of its lanes and stays in scalar registers.

// The columns of a lane: NV units of U, 2^log_l units apart.
template <int U, int NV>
struct LaneColumns {
  uint32_t c[NV];
  bool any[NV];
  __device__ __forceinline__ LaneColumns(int log_l, int64_t dim) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int64_t unit = ((static_cast<int64_t>(blockIdx.y) * NV + u) << log_l) + (threadIdx.x & ((1 << log_l) - 1));
      const UnitAt<U> at(unit * U, dim);
      c[u] = static_cast<uint32_t>(at.c);
      any[u] = at.any();
    }
  }
};

// A unit as it is loaded, so that the loads in flight take no more registers than they bring.
template <int DT, int U>
struct RawUnit;
template <int DT>
struct RawUnit<DT, 1> {
  float v;
  __device__ __forceinline__ void load(const char* row, uint32_t c) { v = load_elem<DT>(row, c); }
  __device__ __forceinline__ void add_to(float (&acc)[1]) const { acc[0] += v; }
};
template <>
struct RawUnit<VDSL_F32, 4> {
  f32x4 v;
  __device__ __forceinline__ void load(const char* row, uint32_t c) { v = reinterpret_cast<const F32x4At4*>(row + size_t{4} * c)->v; }
  __device__ __forceinline__ void add_to(float (&acc)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += v[j];
  }
};
template <>
struct RawUnit<VDSL_BF16, 4> {
  u32x2 v;
  __device__ __forceinline__ void load(const char* row, uint32_t c) { v = reinterpret_cast<const U32x2At2*>(row + size_t{2} * c)->v; }
  __device__ __forceinline__ void add_to(float (&acc)[4]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      acc[2 * j] += __uint_as_float(v[j] << 16);
      acc[2 * j + 1] += __uint_as_float(v[j] & 0xFFFF0000u);
    }
  }
};

// acc += the E rows index[k] of p, in that order, their loads issued together.
template <int DT, int U, int NV, int E>
__device__ __forceinline__ void add_rows(const void* __restrict__ p, int64_t dim, const LaneColumns<U, NV>& at, float (&acc)[NV][U],
                                         const int* index) {
  RawUnit<DT, U> d[E][NV];
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const char* const row = static_cast<const char*>(p) + index[k] * dim * (DT == VDSL_F32 ? 4 : 2);
#pragma unroll
    for (int u = 0; u < NV; ++u) d[k][u].load(row, at.c[u]);
  }
#pragma unroll
  for (int k = 0; k < E; ++k)
#pragma unroll
    for (int u = 0; u < NV; ++u) d[k][u].add_to(acc[u]);
}

// acc += rows row(e) of p for e in [e0, e1), in order, E at a time; the next E are looked up before these
// are waited for.
template <int DT, int U, int NV, int E, class Row>
__device__ __forceinline__ void add_range(const void* __restrict__ p, int64_t dim, const LaneColumns<U, NV>& at, int e0, int e1,
                                          float (&acc)[NV][U], Row&& row) {
  if (e0 >= e1) return;
  int index[E], next[E];
#pragma unroll
  for (int k = 0; k < E; ++k) index[k] = uniform(row(min(e0 + k, e1 - 1)));
  int e = e0;
  for (; e + E <= e1; e += E) {
#pragma unroll
    for (int k = 0; k < E; ++k) next[k] = uniform(row(min(e + E + k, e1 - 1)));
    add_rows<DT, U, NV, E>(p, dim, at, acc, index);
#pragma unroll
    for (int k = 0; k < E; ++k) index[k] = next[k];
  }
  int left = e1 - e;
  if (E > 4 && left >= 4) {
    add_rows<DT, U, NV, 4>(p, dim, at, acc, index);
    left -= 4;
#pragma unroll
    for (int k = 0; k + 4 < E; ++k) index[k] = index[k + 4];
  }
  if (E > 2 && left >= 2) {
    add_rows<DT, U, NV, 2>(p, dim, at, acc, index);
    left -= 2;
    index[0] = index[2 % E];
  }
  if (left) add_rows<DT, U, NV, 1>(p, dim, at, acc, index);
}

// Rows of this type that fit 8 NV registers, the loads in flight of a lane that shares its CU with many.
template <int DT>
constexpr int kInFlight = DT == VDSL_F32 ? 2 : 4;

// Where the positions are many: each row's places, and the sums of the chunks of sorted places that hold one
// token only (a frequent token's places are then added chunk by chunk, by many blocks).  Blocks below
// `place_blocks` do the former.
template <int DYT, int U, int NV>
__global__ __launch_bounds__(256) void embedding_chunk_kernel(const uint32_t* __restrict__ sorted, const int32_t* __restrict__ order,
                                                              const void* __restrict__ dy, int n, int64_t dim, int64_t vocab,
                                                              int chunk, int log_l, int place_blocks, int2* __restrict__ places,
                                                              float* __restrict__ partials) {
  if (static_cast<int>(blockIdx.x) < place_blocks) {
    const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (blockIdx.y != 0 || e >= n) return;
    const uint32_t token = sorted[e];
    if (token >= vocab) return;
    if (e == 0 || sorted[e - 1] != token) places[token].x = static_cast<int>(e);
    if (e == n - 1 || sorted[e + 1] != token) places[token].y = static_cast<int>(e) + 1;
    return;
  }
  const int k = ((static_cast<int>(blockIdx.x) - place_blocks) << (8 - log_l)) + uniform(threadIdx.x >> log_l);
  const int e0 = k * chunk;
  if (k >= n / chunk) return;
  const uint32_t token = sorted[e0];
  if (token >= vocab || sorted[e0 + chunk - 1] != token) return;
  const LaneColumns<U, NV> at(log_l, dim);
  float acc[NV][U] = {};
  add_range<DYT, U, NV, 2 * kInFlight<DYT>>(dy, dim, at, e0, e0 + chunk, acc, [&](int e) { return order[e]; });
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (at.any[u]) store_whole<VDSL_F32, U>(partials, k * dim + at.c[u], acc[u]);
}

// scale acc as row v of dtable.
template <int U, int NV, bool STREAM>
__device__ __forceinline__ void store_row(float* __restrict__ dtable, int64_t v, int64_t dim, const LaneColumns<U, NV>& at, float scale,
                                          float (&acc)[NV][U]) {
#pragma unroll
  for (int u = 0; u < NV; ++u) {
#pragma unroll
    for (int j = 0; j < U; ++j) acc[u][j] *= scale;
    if (at.any[u]) store_whole<VDSL_F32, U, STREAM>(dtable, v * dim + at.c[u], acc[u]);
  }
}

// dtable rows from the sorted positions: 2^log_l lanes (64 to 256) to a row, each NV units of U columns; blockIdx.y:
// strips of columns.
template <int DYT, int U, int NV, bool STREAM>
__global__ __launch_bounds__(256) void embedding_bwd_kernel(const int32_t* __restrict__ order, const void* __restrict__ dy,
                                                            const int2* __restrict__ places, const float* __restrict__ partials,
                                                            int chunk, float* __restrict__ dtable, int64_t dim, int64_t vocab,
                                                            float scale, int log_l) {
  const int64_t v = (block_index() << (8 - log_l)) + uniform(threadIdx.x >> log_l);
  if (v >= vocab) return;
  const int2 place = places[v];
  int e0 = place.x;
  const int e1 = place.y;
  const LaneColumns<U, NV> at(log_l, dim);
  const auto term = [&](int e) { return order[e]; };
  float acc[NV][U] = {};
  if (e1 - e0 >= 2 * chunk) {  // whole chunks lie inside: the places around them, and their sums between
    const int k0 = (e0 + chunk - 1) / chunk, k1 = e1 / chunk;
    add_range<DYT, U, NV, kInFlight<DYT>>(dy, dim, at, e0, k0 * chunk, acc, term);
    add_range<VDSL_F32, U, NV, 2>(partials, dim, at, k0, k1, acc, [&](int h) { return h; });
    e0 = k1 * chunk;
  }
  add_range<DYT, U, NV, kInFlight<DYT>>(dy, dim, at, e0, e1, acc, term);
  store_row<U, NV, STREAM>(dtable, v, dim, at, scale, acc);
}

// The same of few positions, which need no sort: each row's wave looks through all of them.  Us of uniform ids, so and
// sorted: 300 of 1001 columns, vocabulary 5003 5.8, 11.6; 512 of 64, 32768 8.2, 20.6; 1000 of 1001, 5003 6.4, 13.6; ids as
// frequent as words: 1000 of 1001, 5003 19.1, 23.5, but 2000 34.4, 26.6.  The worst is one token at all positions, whose row one
// wave sums kInFlight rows at a time: 300 of 1001, 5003 56, 31; 1024 of 1001, 5003 223, 49; 1024 of 4096, 32768 429, 116
// (uniform 104.5, 104.9).
constexpr int kFewPositions = 1024;

template <int DYT, int U, int NV>
__global__ __launch_bounds__(256) void embedding_bwd_few_kernel(const int32_t* __restrict__ ids, const void* __restrict__ dy,
                                                                float* __restrict__ dtable, int n, int64_t dim, int64_t vocab,
                                                                float scale, int log_l) {
  __shared__ int32_t tokens[kFewPositions];
  __shared__ uint16_t found[4][kFewPositions];
  for (int e = threadIdx.x; e < (n + 255) / 256 * 256; e += 256) tokens[e] = e < n ? ids[e] : -1;
  __syncthreads();
  const int64_t v = (block_index() << (8 - log_l)) + uniform(threadIdx.x >> log_l);
  if (v >= vocab) return;
  const int lane = threadIdx.x & 63;
  uint16_t* const mine = found[uniform(threadIdx.x >> 6)];
  int count = 0;
  for (int e0 = 0; e0 < n; e0 += 256) {
    bool hit[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) hit[k] = tokens[e0 + 64 * k + lane] == static_cast<int32_t>(v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t hits = __ballot(hit[k]);
      if (hit[k]) mine[count + __popcll(hits & ((uint64_t{1} << lane) - 1))] = static_cast<uint16_t>(e0 + 64 * k + lane);
      count += __popcll(hits);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const LaneColumns<U, NV> at(log_l, dim);
  float acc[NV][U] = {};
  add_range<DYT, U, NV, kInFlight<DYT>>(dy, dim, at, 0, count, acc, [&](int k) { return static_cast<int>(mine[k]); });
  store_row<U, NV, false>(dtable, v, dim, at, scale, acc);
}

// log2 of the lanes that share a row of `units` units: a power of two from 16 to 256.
int lanes_log2(int64_t units) {
  int l = 4;
  while (l < 8 && (int64_t{1} << l) < units) ++l;
  return l;
}

int check_extents(int64_t n, int64_t dim, int64_t vocab) {
  if (n < 0 || dim < 0 || vocab < 0) return fail(VDSL_ERR_INVALID_ARG, "negative shape");
  // positions are ints that may run a tile or a chunk past n, and embedding_chunk_kernel's lanes stay below 2^32
  if (n > 0x7f000000 || vocab > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "embedding: too many tokens or table rows");
  if (dim > 0x1fffffff) return fail(VDSL_ERR_UNSUPPORTED, "embedding: rows too wide");
  return VDSL_OK;
}

}  // namespace
}  // namespace vdsl

using namespace vdsl;

extern "C" int vdsl_op_embedding_fwd(vdsl_queue q, int64_t n, int64_t dim, int64_t vocab, int32_t table_dtype, vdsl_buffer table,
                                     vdsl_buffer ids, float scale, int32_t out_dtype, vdsl_buffer out) {
  VDSL_TRY(enter_queue(q));
  VDSL_TRY(check_extents(n, dim, vocab));
  if (!float_type(table_dtype) || !float_type(out_dtype)) return fail(VDSL_ERR_UNSUPPORTED, "embedding_fwd supports f32 and bf16");
  VDSL_TRY(check_buffer(q, table, nbytes(vocab, dim, dtype_size(table_dtype)), "table", false));
  VDSL_TRY(check_buffer(q, ids, nbytes(n, 4), "ids", false));
  VDSL_TRY(check_buffer(q, out, nbytes(n, dim, dtype_size(out_dtype)), "out", true));
  VDSL_TRY(check_apart("embedding_fwd", {out}, {table, ids}));
  if (n == 0 || dim == 0) return VDSL_OK;
  if (vocab == 0) {  // no id is a row
    hipLaunchKernelGGL(embedding_zero_kernel, dim3(1024), dim3(256), 0, q->stream, static_cast<uint16_t*>(out->ptr),
                       n * dim * static_cast<int64_t>(dtype_size(out_dtype) / 2));
    return check_launch("embedding_zero_kernel");
  }
  const auto go = [&](auto tt, auto ot, auto unit, auto ku, auto stream) {
    constexpr int TT = decltype(tt)::value, OT = decltype(ot)::value, U = decltype(unit)::value, KU = decltype(ku)::value;
    const int64_t units = (dim + U - 1) / U;
    const int l = lanes_log2(units);
    const int64_t bx = (n + (256 >> l) - 1) >> (8 - l), by = (units + (int64_t{KU} << l) - 1) / (int64_t{KU} << l);
    if (by > 65535) return fail(VDSL_ERR_UNSUPPORTED, "embedding_fwd: rows too wide");
    hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, U, KU, decltype(stream)::value>), block_grid(bx, by), dim3(256), 0, q->stream, table->ptr,
                       static_cast<const int32_t*>(ids->ptr), out->ptr, n, dim, vocab, scale, l);
    return check_launch("embedding_fwd_kernel");
  };
  // A lane takes 16 bytes of the wider type, or four times that where its loads' time is the longer then: outputs that
  // pass the caches by.  Us, vocabulary 32768, f32 table and bf16 output, 16 bytes and 64: 4096 x 4096 15.5, 16.0;
  // 16384 x 4096 73.3, 59.4; bf16 table and f32 output: 16384 x 1024 16.2, 18.6; 16384 x 4096 102.6, 70.9.
  const auto pick = [&](auto tt, auto ot) {
    constexpr int U = decltype(tt)::value == VDSL_BF16 && decltype(ot)::value == VDSL_BF16 ? 8 : 4;
    using One = std::integral_constant<int, 1>;
    if (dim < U) return go(tt, ot, One{}, One{}, std::false_type{});
    const bool large = n * dim * static_cast<int64_t>(dtype_size(out_dtype)) >= kStreamBytes;
    if (large) return go(tt, ot, std::integral_constant<int, U>{}, std::integral_constant<int, 16 / U>{}, std::true_type{});
    return go(tt, ot, std::integral_constant<int, U>{}, One{}, std::false_type{});
  };
  using F = std::integral_constant<int, VDSL_F32>;
  using B = std::integral_constant<int, VDSL_BF16>;
  if (table_dtype == VDSL_F32) return out_dtype == VDSL_F32 ? pick(F{}, F{}) : pick(F{}, B{});
  return out_dtype == VDSL_F32 ? pick(B{}, F{}) : pick(B{}, B{});
}

namespace vdsl {
namespace {
// How the gradient of n positions is laid out.
struct GradPlan {
  bool radix;        // the sort: radix passes, or ranks
  int passes, tile;  // of the radix sort
  int64_t tiles;
  int chunk;         // places per chunk; 0: none
  size_t sorted = 0, order = 0, keys2 = 0, order2 = 0, hist = 0, places = 0, partials = 0, bytes = 0;
};

int grad_plan(int64_t n, int64_t vocab, int64_t dim, GradPlan& p) {
  VDSL_TRY(check_extents(n, dim, vocab));
  p.radix = n > 32768;
  p.passes = vocab < 256 ? 1 : vocab < 65536 ? 2 : vocab < (1 << 24) ? 3 : 4;
  p.tile = static_cast<int>(std::max<int64_t>(1024, ((n + 255) / 256 + 1023) / 1024 * 1024));
  p.tiles = (n + p.tile - 1) / p.tile;
  // n / chunk chunks, and up to 2 chunk places of a token outside them.  Us of 512 columns, vocabulary 32768, ids as
  // frequent as words, in chunks of 16, 32, 64, 128: n 4096 26.9, 31.3, 40.3, 51.8; 16384 36.1, 34.6, 42.5, 59.1; 65536
  // 93.6, 73.9, 69.3, 88.5; 262144 297, 201, 164, 152.
  p.chunk = 0;
  if (n > kFewPositions)
    for (p.chunk = 16; int64_t{16} * p.chunk * p.chunk < n;) p.chunk *= 2;
  size_t at = 0;
  bool fits = true;
  const auto take = [&](int64_t a, int64_t b) {
    const size_t from = at, size = nbytes(a, b);
    if (size == kSizeOverflow || __builtin_add_overflow(at, size, &at) || at > kSizeOverflow - 512) fits = false;
    else at = (at + 255) / 256 * 256;
    return from;
  };
  if (p.radix) p.hist = take(p.passes * p.tiles, 4 * kDigits);
  if (p.chunk) {
    p.sorted = take(n, 4);
    p.order = take(n, 4);
    p.keys2 = take(n, 4);
    p.order2 = take(n, 4);
    p.places = take(vocab, 8);
    p.partials = take(n / p.chunk, nbytes(dim, 4) == kSizeOverflow ? -1 : dim * 4);
  }
  p.bytes = at;
  return fits ? VDSL_OK : fail(VDSL_ERR_SHAPE, "embedding_bwd: the workspace's size overflows");
}
}  // namespace
}  // namespace vdsl

extern "C" int vdsl_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t dim, size_t* bytes) {
  if (!bytes) return fail(VDSL_ERR_INVALID_ARG, "bytes is null");
  GradPlan p;
  VDSL_TRY(grad_plan(n, vocab, dim, p));
  *bytes = p.bytes;
  return VDSL_OK;
}

extern "C" int vdsl_op_embedding_bwd(vdsl_queue q, int64_t n, int64_t dim, int64_t vocab, vdsl_buffer ids, int32_t dy_dtype,
                                     vdsl_buffer dy, float scale, vdsl_buffer dtable, vdsl_buffer workspace) {
  VDSL_TRY(enter_queue(q));
  GradPlan p;
  VDSL_TRY(grad_plan(n, vocab, dim, p));
  if (!float_type(dy_dtype)) return fail(VDSL_ERR_UNSUPPORTED, "embedding_bwd supports f32 and bf16");
  VDSL_TRY(check_buffer(q, ids, nbytes(n, 4), "ids", false));
  VDSL_TRY(check_buffer(q, dy, nbytes(n, dim, dtype_size(dy_dtype)), "dy", false));
  VDSL_TRY(check_buffer(q, dtable, nbytes(vocab, dim, 4), "dtable", true));
  if (p.bytes) VDSL_TRY(check_buffer(q, workspace, p.bytes, "workspace", true));
  VDSL_TRY(check_apart("embedding_bwd", {dtable, p.bytes ? workspace : nullptr}, {ids, dy}));
  if (vocab == 0 || dim == 0) return VDSL_OK;
  const hipStream_t s = q->stream;
  // A wave per row of up to 1024 columns (1, 2 or 4 units a lane), 2 or 4 waves for a wider one.
  const int unit = dim < 4 ? 1 : 4;
  const int64_t units = (dim + unit - 1) / unit;
  const int nv = units <= 64 ? 1 : units <= 128 ? 2 : 4;
  const int l = std::max(6, lanes_log2((units + nv - 1) / nv));
  const int64_t strips = (units + (int64_t{nv} << l) - 1) / (int64_t{nv} << l);
  if (strips > 65535) return fail(VDSL_ERR_UNSUPPORTED, "embedding_bwd: rows too wide");
  char* const ws = p.bytes ? static_cast<char*>(workspace->ptr) : nullptr;
  const int32_t* id = static_cast<const int32_t*>(ids->ptr);
  uint32_t* const sorted = reinterpret_cast<uint32_t*>(ws + p.sorted);
  int32_t* const order = reinterpret_cast<int32_t*>(ws + p.order);
  const int count = static_cast<int>(n);
  int2* const places = p.chunk ? reinterpret_cast<int2*>(ws + p.places) : nullptr;
  uint32_t* const keys2 = reinterpret_cast<uint32_t*>(ws + p.keys2);
  int32_t* const order2 = reinterpret_cast<int32_t*>(ws + p.order2);
  if (p.radix) {
    int* const hist = reinterpret_cast<int*>(ws + p.hist);
    const dim3 tiles(static_cast<unsigned>(p.tiles));
    hipLaunchKernelGGL(embedding_count_kernel, tiles, dim3(256), 0, s, id, count, static_cast<uint32_t>(vocab), p.tile, hist, p.passes,
                       places);
    VDSL_TRY(check_launch("embedding_count_kernel"));
    for (int k = 0; k < p.passes; ++k) {  // the last pass ends in sorted and order
      const bool second = (p.passes - 1 - k) & 1, from_second = !second;
      int* const h = hist + static_cast<size_t>(k) * p.tiles * kDigits;
      hipLaunchKernelGGL(embedding_radix_kernel, tiles, dim3(256), 0, s, id, k == 0 ? nullptr : from_second ? keys2 : sorted,
                         from_second ? order2 : order, count, static_cast<uint32_t>(vocab), p.tile, 8 * k, h,
                         k + 1 < p.passes ? h + p.tiles * kDigits : nullptr, second ? keys2 : sorted, second ? order2 : order);
      VDSL_TRY(check_launch("embedding_radix_kernel"));
    }
  } else if (p.chunk) {
    const dim3 blocks(static_cast<unsigned>((n + 63) / 64));
    hipLaunchKernelGGL(embedding_rank_kernel, blocks, dim3(1024), 0, s, id, count, keys2, order2, places,
                       vocab);
    VDSL_TRY(check_launch("embedding_rank_kernel"));
    hipLaunchKernelGGL(embedding_merge_kernel, blocks, dim3(1024), 0, s, keys2, order2, count, sorted, order);
    VDSL_TRY(check_launch("embedding_merge_kernel"));
  }
  float* const partials = reinterpret_cast<float*>(ws + p.partials);
  const auto go = [&](auto dyt, auto u, auto units_a_lane) {
    constexpr int DYT = decltype(dyt)::value, U = decltype(u)::value, NV = decltype(units_a_lane)::value;
    const int64_t rows = 256 >> l;
    const dim3 grid = block_grid((vocab + rows - 1) / rows, strips);
    if (!p.chunk) {
      hipLaunchKernelGGL((embedding_bwd_few_kernel<DYT, U, NV>), grid, dim3(256), 0, s, id, dy->ptr, static_cast<float*>(dtable->ptr), count,
                         dim, vocab, scale, l);
      return check_launch("embedding_bwd_few_kernel");
    }
    const int64_t place_blocks = (n + 255) / 256, chunk_blocks = (n / p.chunk + (256 >> l) - 1) >> (8 - l);
    hipLaunchKernelGGL((embedding_chunk_kernel<DYT, U, NV>), dim3(static_cast<unsigned>(place_blocks + chunk_blocks), static_cast<unsigned>(strips)),
                       dim3(256), 0, s, sorted, order, dy->ptr, count, dim, vocab, p.chunk, l, static_cast<int>(place_blocks), places,
                       partials);
    VDSL_TRY(check_launch("embedding_chunk_kernel"));
    const auto rows_kernel = vocab * dim * 4 >= kStreamBytes
                                 ? embedding_bwd_kernel<DYT, U, NV, true>
                                 : embedding_bwd_kernel<DYT, U, NV, false>;
    hipLaunchKernelGGL(rows_kernel, grid, dim3(256), 0, s, order, dy->ptr, places, partials, p.chunk, static_cast<float*>(dtable->ptr),
                       dim, vocab, scale, l);
    return check_launch("embedding_bwd_kernel");
  };
  const auto pick = [&](auto dyt) {
    using One = std::integral_constant<int, 1>;
    using Four = std::integral_constant<int, 4>;
    if (unit == 1) return go(dyt, One{}, One{});
    return nv == 1 ? go(dyt, Four{}, One{}) : nv == 2 ? go(dyt, Four{}, std::integral_constant<int, 2>{}) : go(dyt, Four{}, Four{});
  };
  if (dy_dtype == VDSL_F32) return pick(std::integral_constant<int, VDSL_F32>{});
  return pick(std::integral_constant<int, VDSL_BF16>{});
}
