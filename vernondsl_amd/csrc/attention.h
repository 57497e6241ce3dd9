// What the attention kernels share: sequences and rows, tiles of keys in LDS, fragments.
//
// Rows.  A sequence's tokens and the `group` heads that share a kv head make its rows: row r is token r / group, head
// r % group of the kv head, so a tile of rows shares every key it reads among tokens and heads alike, a few new
// tokens fill a tile, and a tile's rows see nearly the same keys.  Row tiles do not cross sequences.  Which tile a block has
// follows from `starts` on the device: piece i of the rows (0: those before the first sequence, 1 .. seqs the sequences,
// seqs + 1 those behind the last) has the slots from floor(first row of it / tile) + i on, which leaves each piece as
// many as it needs, so that a grid of floor(all rows / tile) + seqs + 2 slots holds every tile and no pass counts them first.
//
// Products.  Scores are formed transposed, S^T = K Q^T: of a 32 x 32 tile a lane then has one row's scores of 16 keys, so
// the softmax needs one exchange between the wave's halves, and what a lane holds of P^T is its part of the second
// product's operand as it is, once the sum over keys is taken in the order in which the accumulators have them: step e
// of 16 keys takes keys 16 e + 8 (j / 4) + 4 (lane / 32) + j % 4 as its elements j of a lane.  V^T comes in that order
// from transposing LDS reads of 4 neighbouring keys each.
#pragma once

#include "gemm_dma.h"
#include "rowunit.h"

namespace vdsl {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// The largest i in [0, count) with below(i), for a `below` that holds from 0 up to some i; every lane of the wave asks the
// same.  64 places at a time: one round trip for up to 64, two for 4096.
template <class Below>
__device__ __forceinline__ int64_t wave_search(int64_t count, Below&& below) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = count;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
    const uint64_t yes = __ballot(at < hi && below(at));
    const int n = yes ? __popcll(yes) : 1;  // place lo is below
    const int64_t from = lo + (n - 1) * step;
    hi = from + step < hi ? from + step : hi;
    lo = from;
  }
  return lo;
}

struct Sequences {
  const int32_t* starts;
  int64_t n, seqs;
  // Row token i of the seqs + 3 borders of the pieces.
  __device__ __forceinline__ int64_t border(int64_t i) const {
    if (i == 0) return 0;
    if (i > seqs + 1) return n;
    const int64_t s = starts[i - 1];
    return s < 0 ? 0 : s > n ? n : s;
  }
};

// The last piece i with below(i, its first token), which holds for 0, and its first token and the next one's.  Up to 125 sequences
// take one trip to memory: their borders stay with the lanes, two each.
struct Piece {
  int64_t i, token, next;
};
template <class Below>
__device__ __forceinline__ Piece find_piece(const Sequences& s, Below&& below) {
  if (s.seqs <= 125) {
    const int lane = threadIdx.x & 63, count = static_cast<int>(s.seqs) + 2;
    const int first = static_cast<int>(s.border(lane)), second = static_cast<int>(s.border(lane + 64));
    const uint64_t of_first = __ballot(lane < count && below(int64_t{lane}, int64_t{first}));
    const uint64_t of_second = __ballot(lane + 64 < count && below(int64_t{lane} + 64, int64_t{second}));
    const int i = __popcll(of_first) + __popcll(of_second) - 1;
    const auto at = [&](int x) { return x < 64 ? __builtin_amdgcn_readlane(first, x) : __builtin_amdgcn_readlane(second, x - 64); };
    return {i, at(i), at(i + 1)};
  }
  const int64_t i = wave_search(s.seqs + 2, [&](int64_t p) { return below(p, s.border(p)); });
  return {i, s.border(i), s.border(i + 1)};
}

struct RowTile {
  int64_t seq;    // -1: rows of no sequence
  int64_t token;  // the piece's first token
  int len;        // its tokens
  int row;        // the tile's first row in the piece
  bool any;       // whether it has one
};
template <int LOG_TILE>
__device__ __forceinline__ RowTile row_tile(const Sequences& s, int group, int64_t slot) {
  const Piece piece = find_piece(s, [&](int64_t p, int64_t border) { return ((border * group) >> LOG_TILE) + p <= slot; });
  RowTile t;
  t.token = piece.token;
  const int64_t len = piece.next - t.token;
  t.len = len > 0 ? static_cast<int>(len) : 0;
  t.seq = piece.i >= 1 && piece.i <= s.seqs ? piece.i - 1 : -1;
  const int64_t row = (slot - ((t.token * group) >> LOG_TILE) - piece.i) << LOG_TILE;
  t.any = row >= 0 && row < static_cast<int64_t>(t.len) * group;
  t.row = t.any ? static_cast<int>(row) : 0;
  return t;
}
inline int64_t row_slots(int64_t n, int64_t seqs, int64_t group, int log_tile) { return ((n * group) >> log_tile) + seqs + 2; }

// ---- tiles of key rows in LDS ---------------------------------------------------------------------
// DP: a head's columns, a multiple of 32 (those past dim are zeros).  A row takes PITCH bytes in 16-byte chunks, chunk c
// in place c ^ swz(row).  Read as rows, 16 neighbouring rows are read at one chunk together: swz puts them into 16 bank
// groups.  Read as columns, 64 bytes of each of 4 neighbouring rows: swz puts them into the four quarters of the banks.
template <int DP>
struct TileShape {
  static constexpr int PITCH = DP <= 64 ? 128 : 256;
  static constexpr int CPR = PITCH / 16;
  static __device__ __forceinline__ int swz(int row) {
    return PITCH == 256 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  }
};

// The fragment of rows row0 .. + 31, k-step kk (16 columns): element j of lane l is column 16 kk + 8 (l / 32) + j of row
// row0 + l % 32.  row0 is a multiple of 32.
template <int DP>
__device__ __forceinline__ bf16x8 rows_fragment(const char* area, int row0, int kk) {
  using T = TileShape<DP>;
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const bf16x8*>(area + row0 * T::PITCH + (lane & 31) * T::PITCH +
                                          (((2 * kk + (lane >> 5)) ^ T::swz(lane & 31)) << 4));
}
// The fragment of columns col0 .. + 31 over the 16 rows from row0 on: element j of lane l is column col0 + l % 32 of row
// row0 + 8 (j / 4) + 4 (l / 32) + j % 4.  row0 is a multiple of 16, col0 of 32.
template <int DP>
__device__ __forceinline__ bf16x8 cols_fragment(const char* area, int row0, int col0) {
  using T = TileShape<DP>;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int r = 4 * (g >> 1) + (i >> 2);
  const int chunk = (col0 / 8 + 2 * (g & 1) + ((i & 3) >> 1)) ^ T::swz(r);
  const char* const p = area + row0 * T::PITCH + r * T::PITCH + (i & 1) * 8;
  // 8 rows further swz has the other bit 1
  const i16x4_t lo = lds_read_tr16(p + (chunk << 4)), hi = lds_read_tr16(p + 8 * T::PITCH + ((chunk ^ 2) << 4));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 32 rows of this lane's wave as an operand (element j of lane l: column 16 kk + 8 (l / 32) + j of row l % 32), from
// the lane's own row at p.
template <int DP>
__device__ __forceinline__ void load_operand(const uint16_t* p, int dim, bf16x8 (&f)[DP / 16]) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int col = 16 * kk + 8 * ((threadIdx.x & 63) >> 5);
    u32x4 w = {0u, 0u, 0u, 0u};
    if (col < dim) w = *reinterpret_cast<const u32x4*>(p + col);
    f[kk] = __builtin_bit_cast(bf16x8, w);
  }
}

// threadIdx.x where what follows from it is to be formed there and not kept through a loop.
__device__ __forceinline__ int late_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// A wave's copies of ROWS rows of two operands to LDS: from scalar addresses and offsets that a lane keeps.
template <int DP, int ROWS>
struct RowCopies {
  using T = TileShape<DP>;
  static constexpr int C = ROWS * T::PITCH / 1024;  // copies of an operand
  static_assert(C * 1024 == ROWS * T::PITCH, "a wave copies 1 KiB at a time");
  uint32_t a_off[C], b_off[C];  // ~0: a column past the head's
  bool all;                     // a head fills a row of LDS

  static __device__ __forceinline__ int row_of(int u) { return u * (64 / T::CPR) + static_cast<int>(threadIdx.x & 63) / T::CPR; }
  // at_a, at_b: bytes from the operand's first row to row r; row0: the place of that one in its tile.
  template <class AtA, class AtB>
  __device__ __forceinline__ void offsets(int row0, int dim, AtA&& at_a, AtB&& at_b) {
    all = 2 * dim == T::PITCH;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int r = row_of(u), c = static_cast<int>(threadIdx.x & 63) % T::CPR ^ T::swz(row0 + r);
      a_off[u] = c < dim / 8 ? at_a(r) + 16u * static_cast<uint32_t>(c) : ~0u;
      b_off[u] = c < dim / 8 ? at_b(r) + 16u * static_cast<uint32_t>(c) : ~0u;
    }
  }
  // Rows 0 .. last; those behind are zeros.
  __device__ __forceinline__ void copy(const char* a, const char* b, int last, char* to_a, char* to_b) const {
    if (last >= ROWS - 1 && all) {
#pragma unroll
      for (int u = 0; u < C; ++u) {
        lds_copy16(a + a_off[u], to_a + u * 1024);
        lds_copy16(b + b_off[u], to_b + u * 1024);
      }
      return;
    }
    const int lane = late_thread() & 63;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      if (a_off[u] == ~0u) continue;
      if (row_of(u) <= last) {
        lds_copy16(a + a_off[u], to_a + u * 1024);
        lds_copy16(b + b_off[u], to_b + u * 1024);
      } else {
        *reinterpret_cast<u32x4*>(to_a + u * 1024 + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4*>(to_b + u * 1024 + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
      }
    }
  }
};

// The values of lanes l % 32 and l % 32 + 32, in every lane.
__device__ __forceinline__ f32x2_t both_halves(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t lo = r[0], hi = r[1];  // (a bit cast of a vector's element itself takes element 0)
  return f32x2_t{__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ float halves_max(float v) {
  const f32x2_t r = both_halves(v);
  return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float halves_sum(float v) {
  const f32x2_t r = both_halves(v);
  return r[0] + r[1];
}

// Asks the scheduler for READS LDS reads, then MFMAS times a product and PER reads, so that a fragment is read some products
// before the one that takes it (left alone it is read right before, and each product waits for its own).
template <int READS, int MFMAS, int PER>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
  }
}

// Registers 8 e .. 8 e + 7 of a score tile as the operand of a step over its 16 keys.
__device__ __forceinline__ bf16x8 weights_fragment(const f32x16& s, int e) {
  const u32x4 w = {pack_bf16x2(s[8 * e], s[8 * e + 1]), pack_bf16x2(s[8 * e + 2], s[8 * e + 3]),
                   pack_bf16x2(s[8 * e + 4], s[8 * e + 5]), pack_bf16x2(s[8 * e + 6], s[8 * e + 7])};
  return __builtin_bit_cast(bf16x8, w);
}

// What a row does not see has weight 0, and 0 times NaN or infinity would spoil it in the products.  Keys (rows) that are
// not there are zeros in LDS; those of the sequence that only some rows of a tile see are looked through, and from the
// first tile that holds an element that is no finite number on, such tiles are left out and added at the end key by
// key, each lane taking what it sees: by half_dot and add_row.
// Whether 32 rows of a tile hold an element that is no finite number.
template <int DP>
__device__ __forceinline__ bool any_not_finite(const char* area) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  i16x2 above = {0, 0};  // as integers, those from +inf on are the largest signed ones, those from -inf on the largest of all
  u16x2 below = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      const u32x4 w = __builtin_bit_cast(u32x4, cols_fragment<DP>(area, 16 * e, 32 * d));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = w[j];
        above = __builtin_elementwise_max(above, __builtin_bit_cast(i16x2, x));
        below = __builtin_elementwise_max(below, __builtin_bit_cast(u16x2, x));
      }
    }
  return __any(above[0] >= 0x7F80 || above[1] >= 0x7F80 || below[0] >= 0xFF80 || below[1] >= 0xFF80);
}
// Whether a lane of the wave has a value that is no finite number.
__device__ __forceinline__ bool any_not_finite(const f32x16& v) {
  float z = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) z = __builtin_fmaf(v[r], 0.0f, z);
  return __any(z != z);
}
// sum plus the product of 8 bf16 elements each.
__device__ __forceinline__ float dot8(u32x4 x, u32x4 y, float sum) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sum = __builtin_fmaf(__uint_as_float(x[j] << 16), __uint_as_float(y[j] << 16), sum);
    sum = __builtin_fmaf(__uint_as_float(x[j] & 0xFFFF0000u), __uint_as_float(y[j] & 0xFFFF0000u), sum);
  }
  return sum;
}
// This half's share of the product of the lane's row, held as an operand, and the row at p (the same for all lanes).  (The
// scheduling barriers, here and below: this is rare, and loads side by side would take registers from the main loops.)
template <int DP>
__device__ __forceinline__ float half_dot(const bf16x8 (&f)[DP / 16], const uint16_t* p, int dim) {
  float sum = 0.0f;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int col = 16 * kk + 8 * ((threadIdx.x & 63) >> 5);
    if (col >= dim) continue;
    sum = dot8(*reinterpret_cast<const u32x4*>(p + col), __builtin_bit_cast(u32x4, f[kk]), sum);
    __builtin_amdgcn_sched_barrier(0);
  }
  return sum;
}
// acc += w times the row at p, columns 32 d + 8 g + 4 (l / 32) + j.
template <int DP>
__device__ __forceinline__ void add_row(f32x16 (&acc)[DP / 32], float w, const uint16_t* p, int dim) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * d + 8 * g + 4 * ((threadIdx.x & 63) >> 5);
      const u32x2 x = *reinterpret_cast<const u32x2*>(p + min(col, dim - 4));  // columns past dim are not stored
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[d][4 * g + 2 * j] = __builtin_fmaf(w, __uint_as_float(x[j] << 16), acc[d][4 * g + 2 * j]);
        acc[d][4 * g + 2 * j + 1] = __builtin_fmaf(w, __uint_as_float(x[j] & 0xFFFF0000u), acc[d][4 * g + 2 * j + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
}

// The sums of a block's waves by way of LDS, so that whole rows are stored and by code of a few lines (an unrolled store of what a lane
// has reads as many instructions as the main loop, which short calls wait for).  Of its 32 x DP sums (column 32 d + 8 g +
// 4 (l / 32) + j of row l % 32) a wave leaves 4 columns in a place of 528 bytes.  Then 32 * GROUPS rows of `by` times the sums of
// PARTS waves, w, w + GROUPS, ..: at(row) is the element of its column 0, less than 0 for none.
template <int DP>
constexpr int kSumBytes = DP / 4 * 528;
template <int DP, int GROUPS, int PARTS, class At>
__device__ __forceinline__ void store_sums(const f32x16 (&acc)[DP / 32], float by, int dim, int dtype, void* to, char* smem, At&& at) {
  const int thread = late_thread(), lane = thread & 63, wave = thread >> 6;
  __syncthreads();
  char* const mine = smem + wave * kSumBytes<DP> + (lane >> 5) * 528 + (lane & 31) * 16;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(mine + (4 * d + g) * 1056) = f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
  __syncthreads();
#pragma unroll 1
  for (int u = thread; u < 32 * GROUPS * (DP / 8); u += 64 * GROUPS * PARTS) {
    const int row = u / (DP / 8), c = u % (DP / 8);
    const int64_t e = at(row);
    if (8 * c >= dim || e < 0) continue;
    const char* const from = smem + (row >> 5) * kSumBytes<DP> + c * 1056 + (row & 31) * 16;
    float v[8] = {};
#pragma unroll
    for (int o = 0; o < PARTS; ++o) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(from + o * GROUPS * kSumBytes<DP>);
      const f32x4 y = *reinterpret_cast<const f32x4*>(from + o * GROUPS * kSumBytes<DP> + 528);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] += x[j];
        v[4 + j] += y[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= by;
    store_unit<8>(dtype, to, e + 8 * c, v);
  }
}

// Copies 4 bytes a lane straight to LDS, lane l's to l + 4 l.
__device__ __forceinline__ void lds_copy4(const char* g, char* l) { __builtin_amdgcn_global_load_lds(g, (lds_void_t*)l, 4, 0, 0); }

// A wait for all but the last 5 copies, a count that gemm_dma.h has none for.
template <>
__device__ __forceinline__ void dma_wait<5>() { __builtin_amdgcn_s_waitcnt(5 | (0x7 << 4)); }

// r / group for r below 2^31.
struct Divider {
  uint32_t by, mul;
  int shift;
  __device__ __forceinline__ int operator()(int r) const {
    return by == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), mul) >> shift);
  }
};
// With 2^l >= group, mul = ceil(2^(31 + l) / group) < 2^32 gives floor(r mul / 2^(31 + l)) = floor(r / group).
inline Divider divider(int group) {
  int l = 0;
  while ((int64_t{1} << l) < group) ++l;
  return {static_cast<uint32_t>(group), l ? static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + group - 1) / group) : 0u, l - 1};
}

}  // namespace vdsl
