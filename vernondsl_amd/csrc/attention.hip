// Attention forward: over packed sequences, and of new rows over a paged cache; and the append to that cache.
//
// For a row's scores s over the keys it sees: m = max s, p = exp2(c (s - m)), l = sum p, out = sum p v / l, with
// c = scale log2 e; one pass over the keys, tile by tile, with m, l and the unnormalised output carried along and
// rescaled where m grows.  The exponent is one fma, c s - m, whose m = c max s is off by up to 2^-25 of itself: the same factor
// for all of a row's p, which drops out; it stays within f32 for scores up to 2^30.  m may lag behind the maximum by a factor of
// 2^8 in p (bf16 and f32 hold that without loss), so most tiles rescale nothing.  See attention.h for rows, tiles and the order of keys in the products.
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace vdsl {
namespace {

struct AttentionArgs {
  const uint16_t *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  Sequences seqs;
  const int32_t *lengths, *table;  // paged
  void* out;
  float* lse;
  float* parts;  // of splits: the unnormalised outputs, f32 [splits][kv_heads][n * group][dim]
  float2* stats; // and m c and l, [splits][kv_heads][n * group]
  int heads, kv_heads, group, dim, causal, out_dtype;
  float scale;
  int64_t pages;
  int table_cols, page_shift;
  int splits, blocks;
  Divider token_of;
};

constexpr float kLag = 8.0f;  // by how much m may lag, in powers of two

// Keys of one sequence and kv head, copied 16 at a time by one wave: from a scalar address and an offset that a lane keeps.
// Paged: 16 positions lie in one page, whose entry in the table is read as constant memory, by a scalar load, so that no
// copy is waited for with it.
template <int DP, bool PAGED>
struct KeySource {
  using T = TileShape<DP>;
  typedef const __attribute__((address_space(4))) int32_t* ScalarTable;
  static constexpr int C = RowCopies<DP, 16>::C;  // copies for 16 keys, and as many for their values
  const char *k, *v;      // packed: of the sequence's first key; paged: of the caches
  uint32_t k_row, v_row;  // bytes from a key to the next
  RowCopies<DP, 16> copies;
  int keys, head, kv_heads, shift;
  uint32_t pages;
  ScalarTable table;      // the sequence's pages

  __device__ __forceinline__ KeySource(const AttentionArgs& a, const RowTile& t, int sequence_keys, int kv)
      : keys(sequence_keys), head(kv), kv_heads(a.kv_heads), shift(a.page_shift), pages(static_cast<uint32_t>(a.pages)) {
    if constexpr (PAGED) {
      k = reinterpret_cast<const char*>(a.k);
      v = reinterpret_cast<const char*>(a.v);
      k_row = v_row = 2 * a.dim;
      const int seq = __builtin_amdgcn_readfirstlane(static_cast<int>(t.seq < 0 ? 0 : t.seq));
      table = (ScalarTable)(reinterpret_cast<uint64_t>(a.table)) + static_cast<int64_t>(seq) * a.table_cols;
    } else {
      k = reinterpret_cast<const char*>(a.k + t.token * a.k_stride + static_cast<int64_t>(kv) * a.dim);
      v = reinterpret_cast<const char*>(a.v + t.token * a.v_stride + static_cast<int64_t>(kv) * a.dim);
      k_row = static_cast<uint32_t>(2 * a.k_stride);
      v_row = static_cast<uint32_t>(2 * a.v_stride);
    }
    copies.offsets(0, a.dim, [&](int r) { return static_cast<uint32_t>(r) * k_row; }, [&](int r) { return static_cast<uint32_t>(r) * v_row; });
  }
  // The page of keys j .. j + 15 (j the same for all lanes): -1 for none.  (Packed: 0.)
  __device__ __forceinline__ int page(int j) const {
    if (j >= keys) return -1;
    if constexpr (!PAGED) return 0;
    const int e = table[__builtin_amdgcn_readfirstlane(j) >> shift];
    return static_cast<uint32_t>(e) < pages ? e : -1;
  }
  // How many of keys j .. j + 15 hold something, as that many bits.
  __device__ __forceinline__ uint32_t there(int j, int e) const { return e < 0 ? 0u : keys - j >= 16 ? 0xFFFFu : (1u << (keys - j)) - 1u; }
  // Key j's row of the keys or values at `base`, in page e.
  __device__ __forceinline__ const char* row(const char* base, uint32_t bytes, int j, int e) const {
    const int64_t at = PAGED ? ((static_cast<int64_t>(e) * kv_heads + head) << shift) + (j & ((1 << shift) - 1)) : j;
    return base + at * bytes;
  }
  // Keys j .. j + 15 of page e to kt, their values to vt; those that hold nothing are zeros there.
  __device__ __forceinline__ void copy(int j, int e, char* kt, char* vt) const {
    copies.copy(row(k, k_row, j, e), row(v, v_row, j, e), e < 0 ? -1 : keys - 1 - j, kt, vt);
  }
};

// What a block's rows see, and where they are.
struct RowsAt {
  int64_t token;  // of row 0 of the piece
  int rows;       // of the piece
  int keys;       // of its sequence
  int before;     // keys before its first token (negative: its first tokens have none)
  __device__ __forceinline__ int sees(int row, int group, int causal) const {
    const int pos = before + row / group;
    return causal ? min(max(pos + 1, 0), keys) : keys;
  }
};
template <bool PAGED>
__device__ __forceinline__ RowsAt rows_at(const AttentionArgs& a, const RowTile& t) {
  RowsAt r;
  r.token = t.token;
  r.rows = t.len * a.group;
  r.keys = t.len;
  r.before = 0;
  if constexpr (PAGED) {
    if (t.seq >= 0) {
      const int64_t have = a.lengths[t.seq], room = static_cast<int64_t>(a.table_cols) << a.page_shift;
      const int64_t before = have - t.len;
      r.keys = static_cast<int>(have < 0 || a.pages == 0 ? 0 : have < room ? have : room);
      r.before = static_cast<int>(before < -0x7fffffff ? -0x7fffffff : before);
    }
  }
  if (t.seq < 0) r.keys = 0;
  return r;
}

// The state of a wave's 32 rows: this lane has row lane % 32 and, of its outputs, o[d][r] of column
// 32 d + 8 (r / 4) + 4 (lane / 32) + r % 4.
template <int DP>
struct RowState {
  f32x16 o[DP / 32];
  float m, l;  // m in powers of two (times c); l: this half's share

  __device__ __forceinline__ void clear() {
    m = neg_inf();
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = MfmaBf16::zero();
  }
  // s: the rows' scores over KS x 32 keys, those that are not seen -inf; they become p.
  template <int KS>
  __device__ __forceinline__ void weigh(f32x16 (&s)[KS], float scale2) {
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
    top = halves_max(top) * scale2;
    if (__any(top > m + kLag)) {
      const float now = fmaxf(m, top);
      const float by = now == neg_inf() ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= by;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= by;
    }
    const float at = m == neg_inf() ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], scale2, -at));
        sum += s[t][r];
      }
    l += sum;
  }
};

// Hides what a row does not see of a tile of KS x 32 keys.  sees: of the row, less the tile's first key.
template <int KS>
__device__ __forceinline__ void hide(f32x16 (&s)[KS], int sees, uint64_t valid) {
  const int half = 4 * ((threadIdx.x & 63) >> 5);
  const uint64_t mine = valid >> half;
#pragma unroll
  for (int t = 0; t < KS; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = 32 * t + 8 * (r / 4) + r % 4;
      if (!(j < sees - half) || !((mine >> j) & 1)) s[t][r] = neg_inf();
    }
}

// The rows' outputs (or their parts of split `split`) from a wave's state.
template <int DP>
__device__ __forceinline__ void store_rows(const AttentionArgs& a, RowState<DP>& st, const RowsAt& at, int row0, int kv, int split) {
  const int lane = threadIdx.x & 63, row = row0 + (lane & 31);
  const float l = halves_sum(st.l);
  if (row >= at.rows) return;
  const int64_t token = at.token + row / a.group;
  const int head = kv * a.group + row % a.group;
  float by;
  int64_t base;
  if (a.splits > 1) {
    const int64_t place = (static_cast<int64_t>(split) * a.kv_heads + kv) * a.seqs.n * a.group + at.token * a.group + row;
    // scores that are NaN all of them leave m as it was: the join has to see them
    if (lane < 32) a.stats[place] = make_float2(st.m == neg_inf() && l != 0.0f ? l : st.m, l);
    if (l == 0.0f) return;  // not read
    by = 1.0f;
    base = place * a.dim;
  } else {
    if (a.lse && lane < 32)
      a.lse[head * a.seqs.n + token] = l == 0.0f ? neg_inf() : (st.m + __builtin_amdgcn_logf(l)) * kLn2;
    // nothing seen, or scores of -inf (the largest score has p >= 1): 0, also where values are no finite numbers.  (A branch that is
    // not taken: selections at the stores took short calls 0.2 us of code.)
    if (l == 0.0f) st.clear();
    by = l == 0.0f ? 0.0f : 1.0f / l;
    base = (token * a.heads + head) * a.dim;
  }
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * d + 8 * g + 4 * (lane >> 5);
      if (col >= a.dim) continue;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = st.o[d][4 * g + j] * by;
      if (a.splits > 1) store_whole<VDSL_F32, 4>(a.parts, base + col, v);
      else store_unit<4>(a.out_dtype, a.out, base + col, v);
    }
}

// Rows of no sequence, or that see no key: out 0, lse -inf.
__device__ __forceinline__ void store_none(const AttentionArgs& a, const RowsAt& at, int row0, int rows, int kv, int split) {
  rows = min(rows, at.rows - row0);
  if (a.splits > 1) {
    const int64_t place = (static_cast<int64_t>(split) * a.kv_heads + kv) * a.seqs.n * a.group + at.token * a.group + row0;
    for (int r = threadIdx.x; r < rows; r += blockDim.x) a.stats[place + r] = make_float2(neg_inf(), 0.0f);
    return;
  }
  const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int per = a.dim / 4;
  for (int u = threadIdx.x; u < rows * per; u += blockDim.x) {
    const int row = row0 + u / per;
    const int64_t token = at.token + row / a.group;
    const int head = kv * a.group + row % a.group;
    store_unit<4>(a.out_dtype, a.out, (token * a.heads + head) * a.dim + 4 * (u % per), none);
    if (a.lse && u % per == 0) a.lse[head * a.seqs.n + token] = neg_inf();
  }
}

// The block's place: kv head, row slot and split.  Blocks that are dispatched together (to the XCDs in turn) have
// different kv heads, so that an XCD reads few heads' keys where there are 8 or more; the last rows first, which see most of their
// sequence.
struct Place {
  int kv, split;
  int64_t slot;
  __device__ __forceinline__ Place(const AttentionArgs& a) {
    int b = static_cast<int>(blockIdx.x);
    kv = b % a.kv_heads;
    b /= a.kv_heads;
    split = b % a.splits;
    slot = a.blocks - 1 - b / a.splits;
  }
};

// Waves of 32 rows each, sharing tiles of keys through two slots of LDS.  PARTS 1: four waves and tiles of 64 keys, two blocks to a
// CU, so that a SIMD has one wave's exponentials beside another's products.  PARTS 4: two times 32 rows with four waves each, which
// take 32 keys each of a tile of 128 and join what they have at the end.
// What bounds it: the matrix units are busy 54% of the cycles and the vector units 50%, so the two waves of a SIMD are seldom beside
// each other in what they do; LDS is active 26%, without bank conflicts.  64 rows a wave would halve its reads, but leave a SIMD
// one wave: 3020 us where this took 2300.  16384 rows, 32 heads of 128 over 8, causal: 2070 us, 1061 TFLOP/s (the library's product
// of 8192^3: 1360).
template <int DP, bool PAGED, int PARTS>
__global__ __launch_bounds__(PARTS == 1 ? 256 : 512, 2) void attention_rows(AttentionArgs a) {
  static_assert(PARTS == 1 || !PAGED, "a paged cache's keys are split among blocks");
  constexpr int NW = PARTS == 1 ? 4 : 8, GROUPS = NW / PARTS, ROWS = 32 * GROUPS, KT = 16 * NW, KW = KT / PARTS, KS = KW / 32, NS = 2;
  using T = TileShape<DP>;
  constexpr int SLOT = 2 * KT * T::PITCH, SUMS = PARTS == 1 ? 0 : NW * kSumBytes<DP>, AREA = NS * SLOT > SUMS ? NS * SLOT : SUMS;
  __shared__ __attribute__((aligned(1024))) char smem[AREA];
  const Place place(a);
  const RowTile tile = row_tile<GROUPS == 4 ? 7 : 6>(a.seqs, a.group, place.slot);
  if (!tile.any) return;
  const RowsAt at = rows_at<PAGED>(a, tile);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int last_row = min(tile.row + ROWS, at.rows) - 1;
  const int sees_most = at.sees(last_row, a.group, a.causal);
  // the split's share of the block's tiles of keys
  const int tiles = (sees_most + KT - 1) / KT;
  const int share = (tiles + a.splits - 1) / a.splits;
  const int first = place.split * share, end = min(first + share, tiles);
  if (first >= end) {
    store_none(a, at, tile.row, ROWS, place.kv, place.split);
    return;
  }
  const KeySource<DP, PAGED> src(a, tile, at.keys, place.kv);
  if (2 * a.dim < T::PITCH) {  // columns past dim are never copied
    for (int i = threadIdx.x; i < NS * SLOT / 16; i += 64 * NW) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  // Paged: which keys of the tile and of the next one hold something, and the pages of that one.
  uint64_t valid = ~0ull, valid_next = ~0ull;
  int pages[4] = {0, 0, 0, 0};
  const auto look = [&](int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) pages[i] = src.page(t * KT + 16 * i);
  };
  // Tile t to a slot, 16 keys by each wave.
  const auto fetch = [&](int t, int slot) {
    int e = 0;
    valid = valid_next;
    if constexpr (PAGED) {
      valid_next = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        valid_next |= static_cast<uint64_t>(src.there(t * KT + 16 * i, pages[i])) << (16 * i);
        if (wave == i) e = pages[i];
      }
      if (t + 1 < end) look(t + 1);
    } else if (t * KT + 16 * wave >= at.keys) {
      e = -1;
    }
    char* const to = smem + slot * SLOT + wave * 16 * T::PITCH;
    src.copy(t * KT + 16 * wave, e, to, to + KT * T::PITCH);
  };
  if constexpr (PAGED) look(first);
  fetch(first, 0);

  const int part = wave / GROUPS, row0 = tile.row + wave % GROUPS * 32;  // the wave's keys of a tile, its rows
  const bool mine = row0 < at.rows;
  const float scale2 = a.scale * kLog2e;
  const int row = min(row0 + (lane & 31), at.rows - 1), sees = at.sees(row, a.group, a.causal);
  bf16x8 qf[DP / 16];
  load_operand<DP>(a.q + (at.token + row / a.group) * a.q_stride + static_cast<int64_t>(place.kv * a.group + row % a.group) * a.dim, a.dim, qf);
  RowState<DP> st;
  st.clear();
  // of the wave's rows: the fewest and the most keys that one sees
  const int fewest = __builtin_amdgcn_readfirstlane(at.sees(min(row0, at.rows - 1), a.group, a.causal));
  const int most = mine ? at.sees(min(row0 + 32, at.rows) - 1, a.group, a.causal) : 0;
  int slot = 0, t = first;
  // The tile t is there and every wave has left the one before, whose slot the next one goes to.
  const auto enter = [&]() {
    dma_wait<0>();
    dma_barrier();
    if (t + 1 < end) fetch(t + 1, slot ^ 1);
    else valid = valid_next;
  };
  // tiles that all of the wave's rows see all of
#pragma unroll 1
  for (const int whole = min(end, fewest / KT); t < whole; ++t) {
    enter();
    const char* const keys = smem + slot * SLOT + part * KW * T::PITCH;
    const char* const values = keys + KT * T::PITCH;
    slot ^= 1;
    f32x16 s[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) s[k] = MfmaBf16::zero();
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int k = 0; k < KS; ++k) s[k] = MfmaBf16::mma(rows_fragment<DP>(keys, 32 * k, kk), qf[kk], s[k]);
    if constexpr (!PAGED) reads_ahead<6, KS * DP / 16, 1>();  // (paged: 256.0 us with it and without, 1024 rows over 16384 positions)
    if (PAGED && valid != ~0ull) hide(s, KW, valid);
    st.weigh(s, scale2);
#pragma unroll
    for (int e = 0; e < 2 * KS; ++e) {
      const bf16x8 w = weights_fragment(s[e / 2], e % 2);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) st.o[d] = MfmaBf16::mma(cols_fragment<DP>(values, 16 * e, 32 * d), w, st.o[d]);
    }
  }
  // the others, 32 keys at a time
  int left_out = 0x7fffffff;
#pragma unroll 1
  for (; t < end; ++t) {
    enter();
    const char* const keys = smem + slot * SLOT + part * KW * T::PITCH;
    const char* const values = keys + KT * T::PITCH;
    slot ^= 1;
#pragma unroll 1
    for (int k = 0; k < KS; ++k) {
      const int j0 = t * KT + part * KW + 32 * k;
      if (j0 >= most) break;
      f32x16 s[1] = {MfmaBf16::zero()};
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) s[0] = MfmaBf16::mma(rows_fragment<DP>(keys, 32 * k, kk), qf[kk], s[0]);
      hide(s, sees - j0, PAGED ? valid >> (32 * k) : ~0ull);
      st.weigh(s, scale2);
      if (a.causal && (j0 >= left_out || any_not_finite<DP>(values + 32 * k * T::PITCH))) {
        left_out = min(left_out, j0);
        continue;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bf16x8 w = weights_fragment(s[0], e);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) st.o[d] = MfmaBf16::mma(cols_fragment<DP>(values, 32 * k + 16 * e, 32 * d), w, st.o[d]);
      }
    }
  }
#pragma unroll 1
  for (int j = left_out; j < min(most, end * KT); ++j) {
    const int e = src.page(j);
    if (e < 0 || (PARTS > 1 && j % KT / KW != part)) continue;
    const float s = halves_sum(half_dot<DP>(qf, reinterpret_cast<const uint16_t*>(src.row(src.k, src.k_row, j, e)), a.dim));
    if (j >= sees) continue;
    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale2, -(st.m == neg_inf() ? 0.0f : st.m)));
    add_row<DP>(st.o, w, reinterpret_cast<const uint16_t*>(src.row(src.v, src.v_row, j, e)), a.dim);
  }
  if constexpr (PARTS == 1) {
    if (mine) store_rows<DP>(a, st, at, row0, place.kv, place.split);
  } else {
    // the parts joined as attention_join does it
    float2* const stats = reinterpret_cast<float2*>(smem);  // [waves][32]
    const float l = halves_sum(st.l);
    __syncthreads();
    if (lane < 32) stats[32 * wave + lane] = make_float2(st.m, l);
    __syncthreads();
    float m = neg_inf(), sum = 0.0f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) m = fmaxf(m, stats[32 * (wave % GROUPS + p * GROUPS) + (lane & 31)].x);
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const float2 of = stats[32 * (wave % GROUPS + p * GROUPS) + (lane & 31)];
      sum += (of.x == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(of.x - m)) * of.y;
    }
    const float by = sum == 0.0f || st.m == neg_inf() ? sum : __builtin_amdgcn_exp2f(st.m - m) / sum;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[d][i] *= by;
    if (sum == 0.0f) st.clear();  // as in store_rows
    const int row = row0 + (lane & 31);
    if (a.lse && part == 0 && lane < 32 && row < at.rows)
      a.lse[(place.kv * a.group + row % a.group) * a.seqs.n + at.token + row / a.group] = sum == 0.0f ? neg_inf() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
    store_sums<DP, GROUPS, PARTS>(st.o, 1.0f, a.dim, a.out_dtype, a.out, smem, [&](int r) {
      const int x = tile.row + r;
      const int i = a.token_of(x);
      return x < at.rows ? ((at.token + i) * a.heads + place.kv * a.group + x - i * a.group) * a.dim : -1;
    });
  }
}

// Few rows: a block is one wave with 32 rows and a split of the keys, in tiles of 32 through two slots of LDS of its own, so
// that nothing waits for another wave.  What bounds it is the cache's bytes: five such blocks to a CU have up to 80 KiB of them on their
// way, each from a tile's start to its second products (the compiler takes the transposing reads for readers of what the copies
// write, and waits for all of them there).  64 sequences of up to 16384 positions, 32 heads of 128 over 8 (2.7 GB): 460-500 us, 5.4-5.9 TB/s, where blocks of
// attention_rows had 645; a copy of 2 GiB moves 4.9.
template <int DP>
__global__ __launch_bounds__(64, 2) void attention_few(AttentionArgs a) {
  constexpr int KT = 32;
  using T = TileShape<DP>;
  constexpr int SLOT = 2 * KT * T::PITCH;
  __shared__ __attribute__((aligned(1024))) char smem[2 * SLOT];
  const Place place(a);
  const RowTile tile = row_tile<5>(a.seqs, a.group, place.slot);
  if (!tile.any) return;
  const RowsAt at = rows_at<true>(a, tile);
  const int lane = threadIdx.x;
  const int last_row = min(tile.row + 32, at.rows) - 1;
  const int most = at.sees(last_row, a.group, 1), fewest = at.sees(tile.row, a.group, 1);
  const int tiles = (most + KT - 1) / KT;
  const int share = (tiles + a.splits - 1) / a.splits;
  const int first = place.split * share, end = min(first + share, tiles);
  if (first >= end) {
    store_none(a, at, tile.row, 32, place.kv, place.split);
    return;
  }
  if (2 * a.dim < T::PITCH) {  // columns past dim are never copied
    for (int i = lane; i < 2 * SLOT / 16; i += 64) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  const KeySource<DP, true> src(a, tile, most, place.kv);
  int page0 = src.page(first * KT), page1 = src.page(first * KT + 16);
  uint32_t valid = 0u, valid_next = 0u;  // which keys of the tile and of the next one hold something
  const auto fetch = [&](int t, int slot) {
    const int e0 = page0, e1 = page1, j = t * KT;
    if (t + 1 < end) {
      page0 = src.page(j + KT);
      page1 = src.page(j + KT + 16);
    }
    valid = valid_next;
    valid_next = src.there(j, e0) | src.there(j + 16, e1) << 16;
    char* const to = smem + slot * SLOT;
    src.copy(j, e0, to, to + KT * T::PITCH);
    src.copy(j + 16, e1, to + 16 * T::PITCH, to + (KT + 16) * T::PITCH);
  };
  fetch(first, 0);
  const float scale2 = a.scale * kLog2e;
  const int row = min(tile.row + (lane & 31), at.rows - 1), sees = at.sees(row, a.group, 1);
  bf16x8 qf[DP / 16];
  load_operand<DP>(a.q + (at.token + row / a.group) * a.q_stride + static_cast<int64_t>(place.kv * a.group + row % a.group) * a.dim, a.dim, qf);
  RowState<DP> st;
  st.clear();
  int slot = 0, left_out = 0x7fffffff;
#pragma unroll 1
  for (int t = first; t < end; ++t) {
    const char* const keys = smem + slot * SLOT;
    const char* const values = keys + KT * T::PITCH;
    slot ^= 1;
    if (t + 1 < end) {
      fetch(t + 1, slot);
      // these may be on their way, if they are as many as those of a whole tile
      if (valid_next == ~0u) dma_wait<4 * KeySource<DP, true>::C>();
      else dma_wait<0>();
    } else {
      valid = valid_next;
      dma_wait<0>();
    }
    asm volatile("" ::: "memory");
    const int j0 = t * KT;
    f32x16 s[1] = {MfmaBf16::zero()};
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) s[0] = MfmaBf16::mma(rows_fragment<DP>(keys, 0, kk), qf[kk], s[0]);
    if (j0 + KT > fewest || valid != ~0u) hide(s, sees - j0, valid);
    st.weigh(s, scale2);
    // some rows do not see some of these keys
    if (j0 + KT > fewest && fewest < most && (j0 >= left_out || any_not_finite<DP>(values))) {
      left_out = min(left_out, j0);
      continue;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bf16x8 w = weights_fragment(s[0], e);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) st.o[d] = MfmaBf16::mma(cols_fragment<DP>(values, 16 * e, 32 * d), w, st.o[d]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read when the copies after the next one's go to it
  }
#pragma unroll 1
  for (int j = left_out; j < min(most, end * KT); ++j) {
    const int e = src.page(j);
    if (e < 0) continue;
    const float s = halves_sum(half_dot<DP>(qf, reinterpret_cast<const uint16_t*>(src.row(src.k, src.k_row, j, e)), a.dim));
    if (j >= sees) continue;
    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale2, -(st.m == neg_inf() ? 0.0f : st.m)));
    add_row<DP>(st.o, w, reinterpret_cast<const uint16_t*>(src.row(src.v, src.v_row, j, e)), a.dim);
  }
  store_rows<DP>(a, st, at, tile.row, place.kv, place.split);
}

// Joins the splits: with M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.  A block's eight groups of 32 lanes have 8 / SHARES rows,
// each row's groups a share of its splits.  Bounded by the latency of a few rounds of loads: 5 us for 256 rows of 15 splits.
template <int SHARES>
__global__ __launch_bounds__(256) void attention_join(AttentionArgs a) {
  __shared__ float sums[8][5][32];
  const int64_t rows = a.seqs.n * a.group, all = rows * a.kv_heads;
  const int group = threadIdx.x >> 5, lane = threadIdx.x & 31, col = 4 * lane, part = group % SHARES;
  const int64_t r = block_index() * (8 / SHARES) + group / SHARES;
  if (SHARES == 1 && r >= all) return;
  const int64_t row = r < all ? r : all - 1;
  float m = neg_inf();
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, a.stats[s * all + row].x);
#pragma unroll
  for (int i = 16; i >= 1; i >>= 1) m = fmaxf(m, __shfl_xor(m, i, 64));
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
#pragma unroll 4
  for (int s = part; s < a.splits; s += SHARES) {
    const float2 st = a.stats[s * all + row];
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool some = st.x != neg_inf();
    if (some && col < a.dim) load_whole<VDSL_F32, 4>(a.parts, (s * all + row) * a.dim + col, o);
    const float by = some ? __builtin_amdgcn_exp2f(st.x - m) : 0.0f;
    l += by * st.y;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += by * o[j];
  }
  if constexpr (SHARES > 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[group][j][lane] = v[j];
    sums[group][4][lane] = l;
    __syncthreads();
    if (part > 0 || r >= all) return;
#pragma unroll
    for (int g = 1; g < SHARES; ++g) {
      l += sums[group + g][4][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += sums[group + g][j][lane];
    }
  }
  const int kv = static_cast<int>(r / rows);
  const int64_t token = r % rows / a.group;
  const int head = kv * a.group + static_cast<int>(r % rows % a.group);
  const bool none = l == 0.0f;
  if (a.lse && col == 0) a.lse[head * a.seqs.n + token] = none ? neg_inf() : (m + __builtin_amdgcn_logf(l)) * kLn2;
  if (col >= a.dim) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = none ? 0.0f : v[j] / l;
  store_unit<4>(a.out_dtype, a.out, (token * a.heads + head) * a.dim + col, v);
}

// A block per new row: its keys and values of all kv heads into their slots, 16 bytes a lane; a copy at HBM's rate (16384 rows of 8
// heads of 128, 134 MB: 21-30 us, 4.4-6.3 TB/s), of few rows a launch.
__global__ __launch_bounds__(256) void cache_append_rows(AttentionArgs a, uint16_t* __restrict__ k_cache, uint16_t* __restrict__ v_cache) {
  const int64_t row = block_index();
  if (row >= a.seqs.n) return;
  const Piece piece = find_piece(a.seqs, [&](int64_t, int64_t border) { return border <= row; });
  const int64_t i = piece.i;
  if (i < 1 || i > a.seqs.seqs) return;
  const int64_t pos = a.lengths[i - 1] - (piece.next - row);
  if (pos < 0 || pos >= (static_cast<int64_t>(a.table_cols) << a.page_shift)) return;
  const int64_t page = a.table[(i - 1) * a.table_cols + (pos >> a.page_shift)];
  if (page < 0 || page >= a.pages) return;
  const int per = a.dim / 8, slot = static_cast<int>(pos) & ((1 << a.page_shift) - 1);
  for (int u = threadIdx.x; u < 2 * a.kv_heads * per; u += 256) {
    const bool is_v = u >= a.kv_heads * per;
    const int x = is_v ? u - a.kv_heads * per : u;
    const int64_t to = ((((page * a.kv_heads + x / per) << a.page_shift) + slot) * per + x % per) * 8;
    const uint16_t* const from = is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride;
    *reinterpret_cast<u32x4*>((is_v ? v_cache : k_cache) + to) = *reinterpret_cast<const u32x4*>(from + 8 * x);
  }
}

// A launch's blocks of `lanes` lanes: fewer than 2^32 lanes.
constexpr int64_t most_blocks(int64_t lanes) { return 0xffffffff / lanes; }

// `lanes` to a block, tiles of 2^log_tile rows.
template <class Kernel>
int launch_rows(vdsl_queue q, AttentionArgs& a, Kernel kernel, unsigned lanes, int log_tile, const char* name) {
  const int64_t slots = row_slots(a.seqs.n, a.seqs.seqs, a.group, log_tile);
  const int64_t blocks = slots * a.kv_heads * a.splits;
  if (blocks > most_blocks(lanes)) return fail(VDSL_ERR_UNSUPPORTED, "attention: too many rows or sequences");
  a.blocks = static_cast<int>(slots);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(lanes), 0, q->stream, a);
  return check_launch(name);
}
template <bool PAGED, int PARTS>
int launch_rows(vdsl_queue q, AttentionArgs& a) {
  return launch_rows(q, a, a.dim <= 64 ? attention_rows<64, PAGED, PARTS> : a.dim <= 96 ? attention_rows<96, PAGED, PARTS> : attention_rows<128, PAGED, PARTS>,
                     PARTS == 1 ? 256 : 512, PARTS == 4 ? 6 : 7, "attention_rows");
}

}  // namespace

// Checks shared by the attention ops.
int attention_check_shape(const char* op, int64_t n, int64_t seqs, int32_t heads, int32_t kv_heads, int32_t dim) {
  const auto refuse = [&](int status, const char* why) { return fail(status, std::string(op) + why); };
  if (n < 0 || seqs < 0 || heads < 0 || kv_heads < 0 || dim < 0) return refuse(VDSL_ERR_INVALID_ARG, ": negative shape");
  if (heads == 0 || kv_heads == 0 || heads % kv_heads) return refuse(VDSL_ERR_INVALID_ARG, ": kv_heads must divide heads");
  if (dim == 0 || dim % 8 || dim > 128) return refuse(VDSL_ERR_UNSUPPORTED, ": dim must be a multiple of 8 up to 128");
  if (heads > 65535 || n > 0x7f000000 / heads || seqs > 0x3fffffff) return refuse(VDSL_ERR_UNSUPPORTED, ": too many rows");
  return VDSL_OK;
}
int attention_check_scale(const char* op, float scale) {
  if (!(scale >= 0x1p-100f && scale <= 0x1p100f))
    return fail(VDSL_ERR_INVALID_ARG, std::string(op) + ": scale must be between 2^-100 and 2^100");
  return VDSL_OK;
}
// The bytes of a buffer that holds n rows of `heads` heads laid out as h says, and whether h can be used.
int attention_check_heads(const char* op, const char* name, const vdsl_heads& h, int64_t n, int32_t heads, int32_t dim, size_t elem,
                          size_t* bytes) {
  const auto refuse = [&](int status, const char* why) { return fail(status, std::string(op) + ": " + name + why); };
  if (h.first < 0 || h.stride < 0) return refuse(VDSL_ERR_INVALID_ARG, ": negative first or stride");
  const int64_t width = static_cast<int64_t>(heads) * dim;
  if (h.first % 8 || h.stride % 8) return refuse(VDSL_ERR_UNSUPPORTED, ": first and stride must be multiples of 8");
  if (h.stride < width) return refuse(VDSL_ERR_SHAPE, ": stride is less than the heads' columns");
  if (h.stride >= (1 << 24)) return refuse(VDSL_ERR_UNSUPPORTED, ": stride of 2^24 or more");
  if (h.first > (int64_t{1} << 60)) return refuse(VDSL_ERR_SHAPE, ": first is past any buffer");
  *bytes = n == 0 ? 0 : nbytes(h.first + (n - 1) * h.stride + width, static_cast<int64_t>(elem));
  return VDSL_OK;
}

}  // namespace vdsl

using namespace vdsl;

extern "C" int vdsl_op_attention_fwd(vdsl_queue q, const vdsl_attention_params* p, vdsl_buffer qs, vdsl_buffer ks, vdsl_buffer vs,
                                     vdsl_buffer starts, int32_t out_dtype, vdsl_buffer out, vdsl_buffer lse) {
  VDSL_TRY(enter_queue(q));
  if (!p) return fail(VDSL_ERR_INVALID_ARG, "params is null");
  const char* const op = "attention_fwd";
  VDSL_TRY(attention_check_shape(op, p->n, p->seqs, p->heads, p->kv_heads, p->dim));
  VDSL_TRY(attention_check_scale(op, p->scale));
  if (!float_type(out_dtype)) return fail(VDSL_ERR_UNSUPPORTED, "attention_fwd stores f32 and bf16");
  size_t qb, kb, vb;
  VDSL_TRY(attention_check_heads(op, "q", p->q, p->n, p->heads, p->dim, 2, &qb));
  VDSL_TRY(attention_check_heads(op, "k", p->k, p->n, p->kv_heads, p->dim, 2, &kb));
  VDSL_TRY(attention_check_heads(op, "v", p->v, p->n, p->kv_heads, p->dim, 2, &vb));
  VDSL_TRY(check_buffer(q, qs, qb, "q", false));
  VDSL_TRY(check_buffer(q, ks, kb, "k", false));
  VDSL_TRY(check_buffer(q, vs, vb, "v", false));
  VDSL_TRY(check_buffer(q, starts, nbytes(p->seqs + 1, 4), "starts", false));
  VDSL_TRY(check_buffer(q, out, nbytes(p->n, static_cast<int64_t>(p->heads) * p->dim, dtype_size(out_dtype)), "out", true));
  if (lse) VDSL_TRY(check_buffer(q, lse, nbytes(p->n, p->heads, 4), "lse", true));
  VDSL_TRY(check_apart(op, {out, lse}, {qs, ks, vs, starts}));
  if (p->n == 0) return VDSL_OK;
  AttentionArgs a = {};
  a.q = static_cast<const uint16_t*>(qs->ptr) + p->q.first;
  a.k = static_cast<const uint16_t*>(ks->ptr) + p->k.first;
  a.v = static_cast<const uint16_t*>(vs->ptr) + p->v.first;
  a.q_stride = p->q.stride;
  a.k_stride = p->k.stride;
  a.v_stride = p->v.stride;
  a.seqs = {static_cast<const int32_t*>(starts->ptr), p->n, p->seqs};
  a.out = out->ptr;
  a.out_dtype = out_dtype;
  a.lse = lse ? static_cast<float*>(lse->ptr) : nullptr;
  a.heads = p->heads;
  a.kv_heads = p->kv_heads;
  a.group = p->heads / p->kv_heads;
  a.dim = p->dim;
  a.causal = p->causal != 0;
  a.scale = p->scale;
  a.splits = 1;
  a.token_of = divider(a.group);
  // Blocks of 128 rows that are few, walking over many keys one after the other, become blocks of 64 with four parts of the keys.
  // us, heads of 128: 1024 rows of 8 over 8 heads (64 blocks) 26 and 17, 2048 of 8 over 2 (128) 42 and 26, 1024 of 32 over 8 (256)
  // 25.8 and 25.6, 2048 of these (512) 52 and 67; 90 rows of 8 over 2 (6) 8.3 and 8.4.
  // (Many empty sequences can be more blocks than a launch of 512 lanes each takes.)
  if (((p->n * a.group + 127) >> 7) * p->kv_heads <= 192 && row_slots(p->n, p->seqs, a.group, 6) * p->kv_heads <= most_blocks(512))
    return launch_rows<false, 4>(q, a);
  return launch_rows<false, 1>(q, a);
}

namespace vdsl {
namespace {
// How the rows' keys are split.  few: attention_few, where a sequence has up to 32 rows on average.  (One form for a batch, by its
// sizes alone: 63 single tokens over 8192 positions take 376 us and a chunk of 512 rows 97, both in one call 487; that chunk alone among
// 63 empty sequences, with which the average is 8 rows, 190.)
struct PagedPlan {
  bool few;
  int splits;
};
PagedPlan paged_plan(int64_t n, int64_t seqs, int32_t heads, int32_t kv_heads, int64_t positions) {
  const int64_t group = heads / kv_heads, with_rows = std::max<int64_t>(1, std::min(seqs, n));
  PagedPlan plan = {n * group <= 32 * with_rows, 1};
  const int64_t tiles = (n * group / (plan.few ? 32 : 128) + with_rows) * kv_heads;
  const auto split = [&](int64_t blocks, int64_t least) { return std::min<int64_t>({(blocks + tiles - 1) / tiles, positions / least, 256}); };
  // attention_few: two rounds of the blocks the card holds, of 64 positions of the table's room at least, or eight rounds, which
  // sequences of different lengths are better spread over, of 1024.  The lengths are on the device: a table of more room than they take
  // makes empty splits, which cost their blocks and the join: 8 single tokens over 1000 positions 15 us with room for 1008, 21 for
  // 16384, 29 for 131072.  (Two tiles a split at least in the kernel: 19 and 28 there, but 12.3 for 12.1 and 18.5 for 17.5 of
  // sequences of 500.)  us with 2560, 5120 and 10240 blocks of 64 positions at least (32 / 8
  // heads of 128 unless said): 64 sequences of up to 16384 positions 482, 470, 462; 16 of 4096, 8 / 8 heads 37.3, 42.3, 51.2;
  // 8 of 1000 (15 splits) 14.5 all, of 128 positions at least 15.3.  attention_rows: four rounds; 1024 rows over 16384 positions with 512,
  // 1024 and 1536 blocks 266, 257, 257.
  const int64_t fit = most_blocks(plan.few ? 64 : 256) / (row_slots(n, seqs, group, plan.few ? 5 : 7) * kv_heads);  // in a launch
  const int64_t splits = std::min(fit, plan.few ? std::max(split(2560, 64), split(10240, 1024)) : split(1024, 256));
  plan.splits = static_cast<int>(std::max<int64_t>(1, splits));
  return plan;
}
// What a split leaves in the workspace.  A call has as many as its workspace holds, so that one made for the most rows, which may have
// fewer splits, serves any.
size_t split_bytes(int64_t n, int64_t heads, int64_t dim) { return nbytes(n, heads, 8 + 4 * dim); }
int paged_check(const char* op, const vdsl_paged_params* p) {
  if (!p) return fail(VDSL_ERR_INVALID_ARG, "params is null");
  VDSL_TRY(attention_check_shape(op, p->n, p->seqs, p->heads, p->kv_heads, p->dim));
  if (p->pages < 0 || p->table_cols < 0 || p->page <= 0) return fail(VDSL_ERR_INVALID_ARG, std::string(op) + ": negative shape or no page size");
  if ((p->page & (p->page - 1)) || p->page < 16 || p->page > 65536)
    return fail(VDSL_ERR_UNSUPPORTED, std::string(op) + ": page must be a power of two from 16 to 65536");
  if (p->pages > 0x7fffffff || p->table_cols > 0x7fff0000 / p->page)  // a tile further is still below 2^31
    return fail(VDSL_ERR_UNSUPPORTED, std::string(op) + ": more than 2^31 - 2^16 positions a sequence");
  return VDSL_OK;
}
AttentionArgs paged_args(const vdsl_paged_params* p, vdsl_buffer starts, vdsl_buffer lengths, vdsl_buffer table) {
  AttentionArgs a = {};
  a.seqs = {static_cast<const int32_t*>(starts->ptr), p->n, p->seqs};
  a.lengths = static_cast<const int32_t*>(lengths->ptr);
  a.table = static_cast<const int32_t*>(table->ptr);
  a.heads = p->heads;
  a.kv_heads = p->kv_heads;
  a.group = p->heads / p->kv_heads;
  a.dim = p->dim;
  a.causal = 1;
  a.scale = p->scale;
  a.pages = p->pages;
  a.table_cols = static_cast<int>(p->table_cols);
  a.page_shift = __builtin_ctz(static_cast<unsigned>(p->page));
  a.splits = 1;
  return a;
}
size_t cache_bytes(const vdsl_paged_params* p) {
  return nbytes(p->pages, static_cast<int64_t>(p->kv_heads) * p->page, static_cast<int64_t>(p->dim) * 2);
}
}  // namespace
}  // namespace vdsl

extern "C" int vdsl_op_cache_append(vdsl_queue q, const vdsl_paged_params* p, vdsl_buffer ks, vdsl_buffer vs, vdsl_buffer starts,
                                    vdsl_buffer lengths, vdsl_buffer table, vdsl_buffer k_cache, vdsl_buffer v_cache) {
  VDSL_TRY(enter_queue(q));
  const char* const op = "cache_append";
  VDSL_TRY(paged_check(op, p));
  size_t kb, vb;
  VDSL_TRY(attention_check_heads(op, "k", p->k, p->n, p->kv_heads, p->dim, 2, &kb));
  VDSL_TRY(attention_check_heads(op, "v", p->v, p->n, p->kv_heads, p->dim, 2, &vb));
  VDSL_TRY(check_buffer(q, ks, kb, "k", false));
  VDSL_TRY(check_buffer(q, vs, vb, "v", false));
  VDSL_TRY(check_buffer(q, starts, nbytes(p->seqs + 1, 4), "starts", false));
  VDSL_TRY(check_buffer(q, lengths, nbytes(p->seqs, 4), "lengths", false));
  VDSL_TRY(check_buffer(q, table, nbytes(p->seqs, p->table_cols, 4), "table", false));
  VDSL_TRY(check_buffer(q, k_cache, cache_bytes(p), "k_cache", true));
  VDSL_TRY(check_buffer(q, v_cache, cache_bytes(p), "v_cache", true));
  VDSL_TRY(check_apart(op, {k_cache, v_cache}, {ks, vs, starts, lengths, table}));
  if (p->n == 0 || p->seqs == 0) return VDSL_OK;
  AttentionArgs a = paged_args(p, starts, lengths, table);
  a.k = static_cast<const uint16_t*>(ks->ptr) + p->k.first;
  a.v = static_cast<const uint16_t*>(vs->ptr) + p->v.first;
  a.k_stride = p->k.stride;
  a.v_stride = p->v.stride;
  hipLaunchKernelGGL(cache_append_rows, block_grid(p->n), dim3(256), 0, q->stream, a, static_cast<uint16_t*>(k_cache->ptr),
                     static_cast<uint16_t*>(v_cache->ptr));
  return check_launch("cache_append_rows");
}

extern "C" int vdsl_paged_attention_workspace_bytes(int64_t n, int64_t seqs, int32_t heads, int32_t kv_heads, int32_t dim,
                                                    int64_t positions, size_t* bytes) {
  if (!bytes) return fail(VDSL_ERR_INVALID_ARG, "bytes is null");
  VDSL_TRY(attention_check_shape("paged_attention", n, seqs, heads, kv_heads, dim));
  if (positions < 0) return fail(VDSL_ERR_INVALID_ARG, "negative shape");
  const int splits = paged_plan(n, seqs, heads, kv_heads, positions).splits;
  *bytes = splits == 1 ? 0 : splits * split_bytes(n, heads, dim);
  return VDSL_OK;
}

extern "C" int vdsl_op_paged_attention(vdsl_queue q, const vdsl_paged_params* p, vdsl_buffer qs, vdsl_buffer k_cache,
                                       vdsl_buffer v_cache, vdsl_buffer starts, vdsl_buffer lengths, vdsl_buffer table,
                                       int32_t out_dtype, vdsl_buffer out, vdsl_buffer lse, vdsl_buffer workspace) {
  VDSL_TRY(enter_queue(q));
  const char* const op = "paged_attention";
  VDSL_TRY(paged_check(op, p));
  VDSL_TRY(attention_check_scale(op, p->scale));
  if (!float_type(out_dtype)) return fail(VDSL_ERR_UNSUPPORTED, "paged_attention stores f32 and bf16");
  size_t qb;
  VDSL_TRY(attention_check_heads(op, "q", p->q, p->n, p->heads, p->dim, 2, &qb));
  VDSL_TRY(check_buffer(q, qs, qb, "q", false));
  VDSL_TRY(check_buffer(q, k_cache, cache_bytes(p), "k_cache", false));
  VDSL_TRY(check_buffer(q, v_cache, cache_bytes(p), "v_cache", false));
  VDSL_TRY(check_buffer(q, starts, nbytes(p->seqs + 1, 4), "starts", false));
  VDSL_TRY(check_buffer(q, lengths, nbytes(p->seqs, 4), "lengths", false));
  VDSL_TRY(check_buffer(q, table, nbytes(p->seqs, p->table_cols, 4), "table", false));
  VDSL_TRY(check_buffer(q, out, nbytes(p->n, static_cast<int64_t>(p->heads) * p->dim, dtype_size(out_dtype)), "out", true));
  if (lse) VDSL_TRY(check_buffer(q, lse, nbytes(p->n, p->heads, 4), "lse", true));
  PagedPlan plan = paged_plan(p->n, p->seqs, p->heads, p->kv_heads, p->table_cols * p->page);
  if (plan.splits == 1) workspace = nullptr;
  if (workspace) {
    VDSL_TRY(check_buffer(q, workspace, 0, "workspace", true));
    plan.splits = static_cast<int>(std::min<size_t>(plan.splits, workspace->bytes / std::max<size_t>(1, split_bytes(p->n, p->heads, p->dim))));
  }
  if (!workspace || plan.splits == 0) plan.splits = 1;
  VDSL_TRY(check_apart(op, {out, lse, workspace}, {qs, k_cache, v_cache, starts, lengths, table}));
  if (p->n == 0) return VDSL_OK;
  AttentionArgs a = paged_args(p, starts, lengths, table);
  a.q = static_cast<const uint16_t*>(qs->ptr) + p->q.first;
  a.k = static_cast<const uint16_t*>(k_cache->ptr);
  a.v = static_cast<const uint16_t*>(v_cache->ptr);
  a.q_stride = p->q.stride;
  a.out = out->ptr;
  a.out_dtype = out_dtype;
  a.lse = lse ? static_cast<float*>(lse->ptr) : nullptr;
  a.splits = plan.splits;
  if (a.splits > 1) {
    a.parts = static_cast<float*>(workspace->ptr);
    a.stats = reinterpret_cast<float2*>(a.parts + static_cast<int64_t>(a.splits) * p->n * p->heads * p->dim);
  }
  if (plan.few)
    VDSL_TRY(launch_rows(q, a, a.dim <= 64 ? attention_few<64> : a.dim <= 96 ? attention_few<96> : attention_few<128>, 64, 5, "attention_few"));
  else
    VDSL_TRY((launch_rows<true, 1>(q, a)));
  if (a.splits == 1) return VDSL_OK;
  const int shares = a.splits <= 8 ? 1 : a.splits <= 64 ? 4 : 8;
  const auto join = shares == 1 ? attention_join<1> : shares == 4 ? attention_join<4> : attention_join<8>;
  hipLaunchKernelGGL(join, block_grid((p->n * p->heads + 8 / shares - 1) / (8 / shares)), dim3(256), 0, q->stream, a);
  return check_launch("attention_join");
}
