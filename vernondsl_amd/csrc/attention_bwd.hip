// The gradient of attention over packed sequences.  With p = exp2(c s - lse log2 e) formed again from q, k and lse,
// dp = dout v, delta = dout out and ds = p (dp - delta):
//   dq = scale ds k (rows' own sum over keys),   dk = scale ds^T q and dv = p^T dout (keys' own sums over rows and heads)
// The launches: delta of each row; dk and dv, waves holding 32 keys and walking over the rows that see them; what those leave
// (attention_bwd_finish); dq, waves holding their rows and walking over the keys they see.  Where the keys' blocks are
// few, keys and rows have one launch.  Every sum is taken in one order, so nothing is added atomically and the bits are
// the same on every call; the price is that s and dp are formed twice (7 products where 5 would do).  See attention.h for rows,
// tiles and the order of the products' sums.
// 8192 rows of two sequences, 32 heads of 128 over 8, causal, 707 GFLOP by five products: 1005 us, of which rows 30, keys 580 (four
// products, 700 TFLOP/s), what they leave 5, queries 390 (three, 780 TFLOP/s).
#include <algorithm>

#include "attention.h"

namespace vdsl {

int attention_check_shape(const char* op, int64_t n, int64_t seqs, int32_t heads, int32_t kv_heads, int32_t dim);
int attention_check_scale(const char* op, float scale);
int attention_check_heads(const char* op, const char* name, const vdsl_heads& h, int64_t n, int32_t heads, int32_t dim, size_t elem,
                          size_t* bytes);

namespace {

struct GradArgs {
  const uint16_t *q, *k, *v, *dout;  // dout: bf16
  int64_t q_stride, k_stride, v_stride, dout_stride;
  Sequences seqs;
  int* left_out;      // rows, by each wave of the keys' blocks
  float* parts;       // of splits: dk and dv, f32 [splits][2][kv_heads][n][dim]
  int key_log;        // log2 of the keys of a block
  int key_splits;     // of the rows that see them
  const float* rows;  // -lse / scale, then -delta, each [kv_heads][n * group]
  void *dq, *dk, *dv;
  int64_t dq_first, dq_stride, dk_first, dk_stride, dv_first, dv_stride;
  int heads, kv_heads, group, dim, causal, grad_dtype;
  float scale;
  Divider token_of;
  int blocks;      // row slots of attention_bwd_queries
  int key_blocks;  // blocks of keys
};

// The kernel's arguments, read again: what only the end of a kernel takes would hold scalar registers through its main loop, which
// has none to spare.
__device__ __forceinline__ const GradArgs& late_args() {
  typedef const __attribute__((address_space(4))) GradArgs* Args;
  Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const GradArgs*)p;
}

// What a row's scores and dp start from, -lse / scale and -delta, and dout in bf16 where it is f32.  16 lanes a row of one head, 16
// bytes each (8 bytes: 44 us where this takes 30, at 4.5 TB/s).
__global__ __launch_bounds__(256) void attention_bwd_rows(const void* __restrict__ dout, int dout_dtype, const void* __restrict__ out,
                                                          int out_dtype, const float* __restrict__ lse, int64_t n, int heads, int group,
                                                          int dim, float scale, uint16_t* __restrict__ copy, float* __restrict__ rows) {
  const int64_t r = block_index() * 16 + (threadIdx.x >> 4);
  if (r >= n * heads) return;
  const int64_t token = r / heads;
  const int head = static_cast<int>(r % heads), col = 8 * (threadIdx.x & 15);
  float sum = 0.0f;
  if (col < dim) {
    float d[8], o[8];
    if (dout_dtype == VDSL_F32) {
      load_whole<VDSL_F32, 8>(dout, r * dim + col, d);
      store_whole<VDSL_BF16, 8>(copy, r * dim + col, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = bf16_to_f32(f32_to_bf16(d[j]));
    } else {
      load_whole<VDSL_BF16, 8>(dout, r * dim + col, d);
    }
    if (out_dtype == VDSL_F32) load_whole<VDSL_F32, 8>(out, r * dim + col, o);
    else load_whole<VDSL_BF16, 8>(out, r * dim + col, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += d[j] * o[j];
  }
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
  if (col != 0) return;
  const float l = lse[head * n + token];
  float* const to = rows + static_cast<int64_t>(head / group) * n * group + token * group + head % group;
  *to = l == neg_inf() ? neg_inf() : -l / scale;  // no score of such a row has a weight
  to[n * heads] = -sum;
}
__device__ __forceinline__ void store_zeros(int dtype, void* to, int64_t e, int cols) {
  const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = 0; c < cols; c += 4) store_unit<4>(dtype, to, e + c, none);
}

// The tiles of TR rows that see a block's keys, and how many of them a split has.
struct RowShare {
  int first, end, tiles;
  __device__ __forceinline__ RowShare(const GradArgs& a, const RowTile& t, int TR)
      : first(a.causal ? t.row * a.group / TR : 0), end((t.len * a.group + TR - 1) / TR), tiles((end - first + a.key_splits - 1) / a.key_splits) {}
};
// dk and dv: a block has KEYS keys and walks over tiles of rows through a ring of two or three slots of LDS.  Each 32 keys
// have 8 / (KEYS / 32) waves, one for each 32 rows of a tile, which add up their sums at the end.  Two waves share a SIMD.  To
// leave both their registers, wide heads' values are an operand read from LDS (V_LDS).
// Bounded by the eight waves' turns at products and exponentials (a tile of 64 rows takes a block 2 us; its products 0.85 at 2.4 GHz) and
// by the longest block, of the first keys (300 tiles where the mean CU has 272, at 8192 rows of two sequences).  Rows from the last to the first:
// all blocks begin with rows that they all see, and so read the same ones at about the same time (1287 us for the whole
// gradient before, 1165 with it).
template <int DP, int KEYS>
struct KeysShape {
  static constexpr int NW = 8, GROUPS = KEYS / 32, PARTS = NW / GROUPS, TR = 32 * PARTS;
  static constexpr bool V_LDS = DP > 96;
  static constexpr int SUMS = NW * kSumBytes<DP>;
  static constexpr int NS = PARTS == 2 ? 3 : 2, SLOT = 2 * TR * TileShape<DP>::PITCH;
  static constexpr int TILES = NS * SLOT + (V_LDS ? KEYS * TileShape<DP>::PITCH : 0), AREA = TILES > SUMS ? TILES : SUMS;
  static constexpr int BYTES = AREA + NW * NS * 2 * 32 * 4;
};
template <int DP, int KEYS>
__device__ __forceinline__ void keys_block(const GradArgs& a, int b, char* smem) {
  using S = KeysShape<DP, KEYS>;
  constexpr int NW = S::NW, GROUPS = S::GROUPS, PARTS = S::PARTS, TR = S::TR, NS = S::NS, SLOT = S::SLOT;
  constexpr bool V_LDS = S::V_LDS;
  using T = TileShape<DP>;
  constexpr int CR = TR / NW;  // of a tile's rows a wave copies
  using Copies = RowCopies<DP, CR>;
  // what the rows' scores and dp start from, a copy a wave: [NS][2][32] each
  float* const starts = reinterpret_cast<float*>(smem + S::AREA) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * (NS * 64);
  int* const left_out_to = a.left_out + b * NW;
  const int kv = b % a.kv_heads;
  b /= a.kv_heads;
  const int split = b % a.key_splits;
  const RowTile tile = row_tile<KEYS == 128 ? 7 : 6>(a.seqs, 1, b / a.key_splits);
  if (!tile.any) {
    if (threadIdx.x < NW) left_out_to[threadIdx.x] = 0;
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int part = wave / GROUPS;  // of a tile's rows
  const int key0 = tile.row + 32 * (wave % GROUPS), key = key0 + (lane & 31);
  const int64_t head_col = static_cast<int64_t>(kv) * a.dim;
  if (tile.seq < 0) {
    if (lane == 0) left_out_to[wave] = 0;
    if (key < tile.len && half == 0 && part == 0 && split == 0) {
      store_zeros(a.grad_dtype, a.dk, a.dk_first + (tile.token + key) * a.dk_stride + head_col, a.dim);
      store_zeros(a.grad_dtype, a.dv, a.dv_first + (tile.token + key) * a.dv_stride + head_col, a.dim);
    }
    return;
  }
  if (2 * a.dim < T::PITCH) {
    for (int i = threadIdx.x; i < NS * SLOT / 16; i += 512) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  const int rows = tile.len * a.group;
  const RowShare share(a, tile, TR);
  const int first = share.first + split * share.tiles, end = min(first + share.tiles, share.end);
  const char* const qp = reinterpret_cast<const char*>(a.q + tile.token * a.q_stride + head_col * a.group);
  const char* const dp = reinterpret_cast<const char*>(a.dout + tile.token * a.dout_stride + head_col * a.group);
  const float* const sp = a.rows + (static_cast<int64_t>(kv) * a.seqs.n + tile.token) * a.group;
  const int64_t delta_at = a.seqs.n * a.heads;
  // The copies of tile t.  Their offsets are the same for all tiles if a wave's rows are whole tokens.
  Copies copies;
  const auto offsets = [&](int row0, int token0) {
    const auto at = [&](int r, int64_t stride) {
      const int i = a.token_of(row0 + r);
      return 2u * (static_cast<uint32_t>(i - token0) * static_cast<uint32_t>(stride) + static_cast<uint32_t>((row0 + r - i * a.group) * a.dim));
    };
    copies.offsets(CR * wave, a.dim, [&](int r) { return at(r, a.q_stride); }, [&](int r) { return at(r, a.dout_stride); });
  };
  const bool whole_tokens = CR % a.group == 0;
  if (whole_tokens) offsets(0, 0);
  const auto fetch = [&](int t, int slot) {
    const int last = rows - 1 - t * TR, row0 = t * TR + CR * wave, token0 = a.token_of(row0);
    if (!whole_tokens) offsets(row0, token0);
    char* const area = smem + slot * SLOT + CR * wave * T::PITCH;
    copies.copy(qp + 2 * (token0 * a.q_stride), dp + 2 * (token0 * a.dout_stride), last - CR * wave, area, area + TR * T::PITCH);
    float* const to = starts + 64 * slot;
    const int r = 32 * part + (lane & 31);
    if (r <= last) lds_copy4(reinterpret_cast<const char*>(sp + (half ? delta_at : 0) + t * TR + r), reinterpret_cast<char*>(to));
    else to[lane] = 0.0f;  // rows that are not there
  };
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = MfmaBf16::zero();
  const float scale2 = a.scale * kLog2e;
  const int sees_from = a.causal ? key * a.group : 0;  // the key's first row
  // the first row that sees one of the wave's keys, and the first that sees all of them
  const int one_seen = a.causal ? key0 * a.group : 0, all_seen = a.causal ? (key0 + 31) * a.group : 0;
  int left_out = 0;  // rows before this one: attention_bwd_left_out adds them
  // All blocks begin with the last rows, which they all see, and so read the same rows at about the same time.
  if (end > first) fetch(end - 1, 0);
  if (NS == 3 && end - 2 >= first) fetch(end - 2, 1);
  const int64_t token = tile.token + min(key, tile.len - 1);
  bf16x8 kf[DP / 16], vf[DP / 16];
  load_operand<DP>(a.k + token * a.k_stride + head_col, a.dim, kf);
  load_operand<DP>(a.v + token * a.v_stride + head_col, a.dim, vf);
  char* const values = smem + NS * SLOT + wave % GROUPS * 32 * T::PITCH;  // all parts write the same
  if constexpr (V_LDS) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      *reinterpret_cast<bf16x8*>(values + (lane & 31) * T::PITCH + (((2 * kk + half) ^ T::swz(lane & 31)) << 4)) = vf[kk];
  }
  int slot = 0;
#pragma unroll 1
  for (int t = end - 1; t >= first; --t) {
    // Every wave has left the tile before.  Of three slots, the next tile, which is whole, may be on its way, and those issued
    // below until this tile's second products (where the compiler waits for all copies: it takes the transposing reads for readers of
    // what they write).
    if (NS == 3 && t > first) dma_wait<2 * Copies::C + 1>();
    else dma_wait<0>();
    dma_barrier();
    if (t - (NS - 1) >= first) fetch(t - (NS - 1), slot == 0 ? NS - 1 : slot - 1);
    const char* const qs = smem + slot * SLOT + part * 32 * T::PITCH;
    const char* const ds = qs + TR * T::PITCH;
    const float* const x = starts + 64 * slot + 4 * half;
    slot = slot == NS - 1 ? 0 : slot + 1;
    const int r0 = t * TR + 32 * part;
    if (r0 + 32 <= one_seen || r0 >= rows) continue;
    f32x16 s, p;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 s0 = *reinterpret_cast<const f32x4*>(x + 8 * g), p0 = *reinterpret_cast<const f32x4*>(x + 32 + 8 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[4 * g + j] = s0[j];
        p[4 * g + j] = p0[j];
      }
    }
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      s = MfmaBf16::mma(rows_fragment<DP>(qs, 0, kk), kf[kk], s);
      p = MfmaBf16::mma(rows_fragment<DP>(ds, 0, kk), V_LDS ? rows_fragment<DP>(values, 0, kk) : vf[kk], p);
    }
    if constexpr (!V_LDS) reads_ahead<12, DP / 8, 1>();  // the first 8 are of what they start from.  (V_LDS has no registers for it.)
    // a row whose q or dout holds an element that is no finite number has no finite score or dp with any key
    bool leave = false;
    if (r0 < all_seen) leave = left_out > 0 || any_not_finite(s) || any_not_finite(p);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(s[i] * scale2);
      p[i] *= s[i];
    }
    // what does not see the key, and rows that are not there: by selection, since 0 times a key of infinity is NaN
    if (r0 < all_seen || rows < r0 + 32) {
      const int lo = sees_from - r0, count = rows - sees_from;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool in = static_cast<uint32_t>(8 * (i / 4) + 4 * half + i % 4 - lo) < static_cast<uint32_t>(count);
        s[i] = in ? s[i] : 0.0f;
        p[i] = in ? p[i] : 0.0f;
      }
      if (leave) {
        left_out = max(left_out, r0 + 32);
        continue;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bf16x8 wf = weights_fragment(s, e), df = weights_fragment(p, e);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        dv[d] = MfmaBf16::mma(cols_fragment<DP>(ds, 16 * e, 32 * d), wf, dv[d]);
        dk[d] = MfmaBf16::mma(cols_fragment<DP>(qs, 16 * e, 32 * d), df, dk[d]);
      }
    }
    reads_ahead<4, DP / 8, 2>();  // the whole gradient 1046 us without, 1019 with these, 1049 with two more
  }
  if ((late_thread() & 63) == 0) left_out_to[wave] = left_out;
  const GradArgs& z = late_args();
  const bool whole = z.key_splits == 1;
  const int place = static_cast<int>(blockIdx.x), kv_head = place % z.kv_heads, row_split = place / z.kv_heads % z.key_splits;
  const auto store = [&](const f32x16 (&acc)[DP / 32], float by, void* to, int64_t first, int64_t stride, int which) {
    const int64_t e = whole ? first + static_cast<int64_t>(kv_head) * z.dim : ((2 * row_split + which) * z.kv_heads + kv_head) * z.seqs.n * z.dim;
    const int64_t step = whole ? stride : z.dim;
    store_sums<DP, GROUPS, PARTS>(acc, by, z.dim, whole ? z.grad_dtype : static_cast<int>(VDSL_F32), whole ? to : z.parts, smem,
                                  [&](int r) { return tile.row + r < tile.len ? e + (tile.token + tile.row + r) * step : -1; });
  };
  store(dk, z.scale, z.dk, z.dk_first, z.dk_stride, 0);
  store(dv, 1.0f, z.dv, z.dv_first, z.dv_stride, 1);
}

template <int DP>
__global__ __launch_bounds__(512, 2) void attention_bwd_keys(GradArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[KeysShape<DP, 128>::BYTES];
  keys_block<DP, 128>(a, static_cast<int>(blockIdx.x), smem);
}

// What the keys' blocks leave.  Their splits' sums, if they have more than one, in order; then the rows that they left out, added
// row by row to what is stored (so bf16 gradients are rounded once more), each lane taking what its key is seen by, 32 columns of
// the gradients at a time.  (A launch of its own, 3 to 5 us, whose blocks mostly find no such rows: as a part of the keys' kernel it took
// the registers of its loop.)  kSumBlocks: one to four units a lane; fewer wait for one load after the other.
constexpr int kSumBlocks = 16;
__global__ __launch_bounds__(256) void attention_bwd_finish(GradArgs a) {
  const int sums = a.key_splits > 1 ? kSumBlocks : 1;  // blocks that share a tile's sums
  const int block = static_cast<int>(block_index()), place = block / sums, sum_block = block % sums;
  if (place >= a.key_blocks / a.key_splits) return;
  const int kv = place % a.kv_heads, slot = place / a.kv_heads;
  const int64_t split_step = 8 * a.kv_heads;  // from a split's flags to the next one's
  const int* const flags = a.left_out + slot * a.key_splits * split_step + 8 * kv;
  int any = 0;
  for (int s = 0; s < a.key_splits; ++s)
#pragma unroll
    for (int w = 0; w < 8; ++w) any |= flags[s * split_step + w];
  // one block that has them all where rows were left out, which come after the sums
  if (any == 0 ? a.key_splits == 1 : sum_block > 0) return;
  const int lanes = any == 0 ? 256 * sums : 256;
  const RowTile tile = a.key_log == 7 ? row_tile<7>(a.seqs, 1, slot) : row_tile<6>(a.seqs, 1, slot);
  if (!tile.any || tile.seq < 0) return;
  const int64_t head_col = static_cast<int64_t>(kv) * a.dim;
  if (a.key_splits > 1) {
    const int per = a.dim / 4, units = min(1 << a.key_log, tile.len - tile.row) * per;
    const int64_t other = a.kv_heads * a.seqs.n * a.dim;
    for (int u = 256 * sum_block + threadIdx.x; u < 2 * units; u += lanes) {
      const bool is_v = u >= units;
      const int x = is_v ? u - units : u;
      const int64_t token = tile.token + tile.row + x / per;
      const int col = 4 * (x % per);
      const float* from = a.parts + (kv * a.seqs.n + token) * a.dim + col + (is_v ? other : 0);
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int s = 0; s < a.key_splits; ++s, from += 2 * other) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(from);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += v[j];
      }
      if (is_v) store_unit<4>(a.grad_dtype, a.dv, a.dv_first + token * a.dv_stride + head_col + col, sum);
      else store_unit<4>(a.grad_dtype, a.dk, a.dk_first + token * a.dk_stride + head_col + col, sum);
    }
    if (any == 0) return;
    __syncthreads();
  }
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = 1 << (a.key_log - 5), parts = 8 / groups;
  if (wave >= groups) return;
  const int key0 = tile.row + 32 * wave, key = key0 + (lane & 31);
  const int64_t token = tile.token + min(key, tile.len - 1);
  const uint16_t* const kp = a.k + token * a.k_stride + head_col;
  const uint16_t* const vp = a.v + token * a.v_stride + head_col;
  const uint16_t* const qp = a.q + tile.token * a.q_stride + head_col * a.group;
  const uint16_t* const dp = a.dout + tile.token * a.dout_stride + head_col * a.group;
  const float* const sp = a.rows + (static_cast<int64_t>(kv) * a.seqs.n + tile.token) * a.group;
  const float scale2 = a.scale * kLog2e;
  int end = 0;
  for (int s = 0; s < a.key_splits; ++s)
    for (int p = 0; p < parts; ++p) end = max(end, flags[s * split_step + wave + groups * p]);
  end = min(end, tile.len * a.group);
  const int tile_rows = 32 * parts;
  const RowShare share(a, tile, tile_rows);
#pragma unroll 1
  for (int c0 = 0; c0 < a.dim; c0 += 32) {
    f32x16 dk[1] = {MfmaBf16::zero()}, dv[1] = {MfmaBf16::zero()};
#pragma unroll 1
    for (int r = key0 * a.group; r < end; ++r) {
      if (r >= flags[(r / tile_rows - share.first) / share.tiles * split_step + wave + groups * ((r >> 5) & (parts - 1))]) continue;
      const int i = a.token_of(r);
      const int64_t head = static_cast<int64_t>(r - i * a.group) * a.dim;
      const uint16_t* const qr = qp + i * a.q_stride + head;
      const uint16_t* const dr = dp + i * a.dout_stride + head;
      float sr = 0.0f, pr = 0.0f;
#pragma unroll 1
      for (int col = 8 * half; col < a.dim; col += 16) {
        sr = dot8(*reinterpret_cast<const u32x4*>(kp + col), *reinterpret_cast<const u32x4*>(qr + col), sr);
        pr = dot8(*reinterpret_cast<const u32x4*>(vp + col), *reinterpret_cast<const u32x4*>(dr + col), pr);
      }
      sr = halves_sum(sr);
      pr = halves_sum(pr);
      if (r < key * a.group) continue;
      const float w = __builtin_amdgcn_exp2f((sr + sp[r]) * scale2);
      add_row<32>(dv, w, dr + c0, a.dim - c0);
      add_row<32>(dk, w * (pr + sp[a.seqs.n * a.heads + r]), qr + c0, a.dim - c0);
    }
    if (key >= tile.len) continue;
    const auto add = [&](const f32x16& acc, float by, void* to, int64_t e) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = c0 + 8 * g + 4 * half;
        if (c >= a.dim) continue;
        float v[4];
        load_some(a.grad_dtype, to, e + c, 4, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += acc[4 * g + j] * by;
        store_some(a.grad_dtype, to, e + c, 4, v);
      }
    };
    add(dk[0], a.scale, a.dk, a.dk_first + token * a.dk_stride + head_col);
    add(dv[0], 1.0f, a.dv, a.dv_first + token * a.dv_stride + head_col);
  }
}

// dq: a block has 128 rows and walks over tiles of 64 keys.  32 rows have NW / 4 waves, of which each takes its share of a
// tile's keys; they add up their sums at the end.  Bounded as the forward pass is.
template <int DP>
constexpr int kQueriesTiles = 2 * 2 * 64 * TileShape<DP>::PITCH;
template <int DP, int NW>
constexpr int kQueriesBytes = kQueriesTiles<DP> > NW * kSumBytes<DP> ? kQueriesTiles<DP> : NW * kSumBytes<DP>;
template <int DP, int NW>
__device__ __forceinline__ void queries_block(const GradArgs& a, int b, char* smem) {
  constexpr int KT = 64, ROWS = 128, CK = KT / NW, PARTS = NW / 4;
  using T = TileShape<DP>;
  using Copies = RowCopies<DP, CK>;  // of a tile's keys by each wave
  constexpr int SLOT = 2 * KT * T::PITCH;
  const int kv = b % a.kv_heads;
  const RowTile tile = row_tile<7>(a.seqs, a.group, a.blocks - 1 - b / a.kv_heads);
  if (!tile.any) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave >> 2;  // of a tile's keys
  const int rows = tile.len * a.group, row0 = tile.row + 32 * (wave & 3);
  const int64_t head_col = static_cast<int64_t>(kv) * a.dim;
  const auto dq_at = [&tile](const GradArgs& z, int64_t first, int row) {
    const int i = z.token_of(row);
    return first + (tile.token + i) * z.dq_stride + static_cast<int64_t>(row - i * z.group) * z.dim;
  };
  if (tile.seq < 0) {
    for (int row = tile.row + static_cast<int>(threadIdx.x); row < min(tile.row + ROWS, rows); row += 64 * NW)
      store_zeros(a.grad_dtype, a.dq, dq_at(a, a.dq_first + head_col * a.group, row), a.dim);
    return;
  }
  if (2 * a.dim < T::PITCH) {
    for (int i = threadIdx.x; i < 2 * SLOT / 16; i += 64 * NW) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  const auto sees = [&](int row) { return a.causal ? a.token_of(row) + 1 : tile.len; };
  const int end = (sees(min(tile.row + ROWS, rows) - 1) + KT - 1) / KT;
  const char* const kp = reinterpret_cast<const char*>(a.k + tile.token * a.k_stride + head_col);
  const char* const vp = reinterpret_cast<const char*>(a.v + tile.token * a.v_stride + head_col);
  Copies copies;
  copies.offsets(CK * wave, a.dim, [&](int r) { return 2u * static_cast<uint32_t>(r) * static_cast<uint32_t>(a.k_stride); },
                 [&](int r) { return 2u * static_cast<uint32_t>(r) * static_cast<uint32_t>(a.v_stride); });
  const auto fetch = [&](int t, int slot) {
    const int j = t * KT + CK * wave;
    char* const area = smem + slot * SLOT + CK * wave * T::PITCH;
    copies.copy(kp + 2 * (j * a.k_stride), vp + 2 * (j * a.v_stride), tile.len - 1 - j, area, area + KT * T::PITCH);
  };
  fetch(0, 0);
  const bool mine = row0 < rows;
  const int row = min(row0 + (lane & 31), rows - 1), seen = sees(row);
  bf16x8 qf[DP / 16], df[DP / 16];
  {
    const int i = a.token_of(row);
    const int64_t col = head_col * a.group + static_cast<int64_t>(row - i * a.group) * a.dim;
    load_operand<DP>(a.q + (tile.token + i) * a.q_stride + col, a.dim, qf);
    load_operand<DP>(a.dout + (tile.token + i) * a.dout_stride + col, a.dim, df);
  }
  const float* const start = a.rows + (static_cast<int64_t>(kv) * a.seqs.n + tile.token) * a.group + row;
  const float score0 = *start, dp0 = start[a.seqs.n * a.heads];
  f32x16 dq[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dq[d] = MfmaBf16::zero();
  const float scale2 = a.scale * kLog2e;
  const int fewest = sees(min(row0, rows - 1)), most = mine ? sees(min(row0 + 32, rows) - 1) : 0;
  int slot = 0, t = 0, left_out = 0x7fffffff;
  const auto enter = [&]() {
    dma_wait<0>();
    dma_barrier();
    if (t + 1 < end) fetch(t + 1, slot ^ 1);
  };
  // ds of 32 keys; odd: whether to say if a key holds an element that is no finite number, which has no finite score then
  const auto form = [&](const char* ks, bool* odd) {
    f32x16 s = MfmaBf16::zero(), p = MfmaBf16::zero();
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      s = MfmaBf16::mma(rows_fragment<DP>(ks, 0, kk), qf[kk], s);
      p = MfmaBf16::mma(rows_fragment<DP>(ks + KT * T::PITCH, 0, kk), df[kk], p);
    }
    reads_ahead<4, DP / 8, 1>();
    if (odd) *odd = any_not_finite(s);
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f((s[r] + score0) * scale2) * (p[r] + dp0);
    return p;
  };
  const auto add = [&](const char* ks, const f32x16& ds) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bf16x8 w = weights_fragment(ds, e);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) dq[d] = MfmaBf16::mma(cols_fragment<DP>(ks, 16 * e, 32 * d), w, dq[d]);
    }
  };
  // tiles that all of the wave's rows see all of
#pragma unroll 1
  for (const int whole = min(end, fewest / KT); t < whole; ++t) {
    enter();
    const char* const ks = smem + slot * SLOT;
    slot ^= 1;
#pragma unroll 1
    for (int u = part; u < KT / 32; u += PARTS) add(ks + 32 * u * T::PITCH, form(ks + 32 * u * T::PITCH, nullptr));
  }
  // the others
#pragma unroll 1
  for (; t < end; ++t) {
    enter();
    const char* ks = smem + slot * SLOT + part * 32 * T::PITCH;
    slot ^= 1;
#pragma unroll 1
    for (int u = part; u < KT / 32; u += PARTS, ks += PARTS * 32 * T::PITCH) {
      const int j0 = t * KT + 32 * u, hi = seen - j0 - 4 * (lane >> 5);
      if (j0 >= most) break;
      bool odd;
      f32x16 p = form(ks, &odd);
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = 8 * (r / 4) + r % 4 < hi ? p[r] : 0.0f;
      // some rows do not see some of these keys
      if (a.causal && (j0 >= left_out || odd)) left_out = min(left_out, j0);
      else add(ks, p);
    }
  }
#pragma unroll 1
  for (int j = left_out; j < most; ++j) {
    if (PARTS == 2 && ((j >> 5) & 1) != part) continue;
    const uint16_t* const kr = reinterpret_cast<const uint16_t*>(kp) + j * a.k_stride;
    const uint16_t* const vr = reinterpret_cast<const uint16_t*>(vp) + j * a.v_stride;
    const float s = halves_sum(half_dot<DP>(qf, kr, a.dim)), p = halves_sum(half_dot<DP>(df, vr, a.dim));
    if (j >= seen) continue;
    add_row<DP>(dq, __builtin_amdgcn_exp2f((s + score0) * scale2) * (p + dp0), kr, a.dim);
  }
  const GradArgs& z = late_args();
  const int64_t first = z.dq_first + static_cast<int64_t>((static_cast<int>(blockIdx.x) - (PARTS == 2 ? z.key_blocks : 0)) % z.kv_heads) * z.group * z.dim;
  store_sums<DP, 4, PARTS>(dq, z.scale, z.dim, z.grad_dtype, z.dq, smem,
                           [&](int r) { return tile.row + r < rows ? dq_at(z, first, tile.row + r) : -1; });
}
template <int DP>
__global__ __launch_bounds__(256, 2) void attention_bwd_queries(GradArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[kQueriesBytes<DP, 4>];
  queries_block<DP, 4>(a, static_cast<int>(blockIdx.x), smem);
}

// Both in one launch, side by side: the keys' blocks first, which are the longer ones.  293 rows of 6 heads of 80 over 2: 27 us in two
// launches, 18 in one.
template <int DP>
__global__ __launch_bounds__(512, 2) void attention_bwd_both(GradArgs a) {
  constexpr int BYTES = KeysShape<DP, 64>::BYTES;
  static_assert(BYTES >= kQueriesBytes<DP, 8>, "one area for either");
  __shared__ __attribute__((aligned(1024))) char smem[BYTES];
  const int b = static_cast<int>(blockIdx.x);
  if (b < a.key_blocks) keys_block<DP, 64>(a, b, smem);
  else queries_block<DP, 8>(a, b - a.key_blocks, smem);
}

// 128 keys a block, or 64 in twice the blocks, each half as long, where 128 would leave CUs idle (full attention) or wait for the
// blocks of the first keys, which the most rows see (causal).  Whole gradients, 32 heads of 128 over 8: causal, one sequence of 1024
// rows 164 us by 128 keys and 66 by 64 with the queries in the same launch, 2048: 309 and 158, 4096: 684 and 534, 8192: 1820
// and (a launch each) 2040; full, 4096: 893 and 1042.
int key_tile_log(int64_t n, int64_t kv_heads, bool causal) {
  return ((n + 127) >> 7) * kv_heads <= (causal ? 256 : 128) ? 6 : 7;
}
// Splits of the rows that see a block's 64 keys, where those blocks are few: so many that the longest block (a tile of 128 rows takes it
// about 2 us, and its start and end as long as five) times the rounds of the card's 256 CUs is least.  us with 1 split, as many as
// make 256 blocks, and these: 1000 rows, 8 heads of 128 over 2 74, 52, 38; 2048 136, 74, 74; 1024 over 8 each 34, 55, 34; 8192, 8
// over 1 986, 554, 554; 32 over 8: 512 47, 44, 44, 1024 78, 66, 66.
constexpr int64_t kMostKeySplits = 8;
constexpr int64_t kMostBlocks = 0x3fffff;  // of keys, and of rows: both in one launch of 512 lanes each are fewer than 2^32 lanes
int key_splits(int64_t n, int64_t seqs, int64_t heads, int64_t kv_heads) {
  const int64_t with_rows = std::max<int64_t>(1, std::min(seqs, n)), tiles = n * (heads / kv_heads) / 128 / with_rows;
  const int64_t most = std::min({256 / std::max<int64_t>(1, ((n + 63) >> 6) * kv_heads), tiles, kMostKeySplits,
                                 kMostBlocks / (row_slots(n, seqs, 1, 6) * kv_heads)});
  int64_t best = 1, least = INT64_MAX;
  for (int64_t s = 1; s <= most; ++s) {
    const int64_t blocks = (row_slots(n, seqs, 1, 6) * s + row_slots(n, seqs, heads / kv_heads, 7)) * kv_heads;
    const int64_t takes = (blocks + 255) / 256 * (5 * s + tiles) * 840 / s;  // 840: a multiple of 1 .. kMostKeySplits
    if (takes < least) best = s, least = takes;
  }
  return static_cast<int>(best);
}

// Whether two of the gradients, as columns of one buffer, have no element in common.
bool apart(const vdsl_heads& x, int64_t x_width, const vdsl_heads& y, int64_t y_width) {
  if (x.stride != y.stride) return false;
  if (x.first + x_width > x.stride || y.first + y_width > y.stride) return false;
  return x.first + x_width <= y.first || y.first + y_width <= x.first;
}

}  // namespace
}  // namespace vdsl

using namespace vdsl;

// What the rows' scores and dp start from, what the keys' blocks left out, a copy of dout in bf16, splits' sums.
extern "C" int vdsl_attention_bwd_workspace_bytes(int64_t n, int64_t seqs, int32_t heads, int32_t kv_heads, int32_t dim, size_t* bytes) {
  if (!bytes) return fail(VDSL_ERR_INVALID_ARG, "bytes is null");
  VDSL_TRY(attention_check_shape("attention_bwd", n, seqs, heads, kv_heads, dim));
  // The most that a call of up to so many rows and sequences takes, so that a batch of fewer rows, which may be split more, fits too:
  // key_splits gives s splits to 256 / (kv_heads * s) tiles of 64 keys at most, and to 128 * s of a sequence's rows at least.
  int64_t slots = row_slots(n, seqs, 1, 6), split_rows = 0;
  for (int64_t s = 2; s <= kMostKeySplits; ++s) {
    const int64_t with = std::min(n, 256 / (kv_heads * s) * 64);
    if (with * (heads / kv_heads) / 128 < s) continue;
    slots = std::max(slots, row_slots(with, seqs, 1, 6) * s);
    split_rows = std::max(split_rows, with * s);
  }
  // a multiple of 16 bytes before the copy
  const size_t flags = nbytes(slots, kv_heads, 32), rows = nbytes(n, heads, 8 + 2 * static_cast<int64_t>(dim));
  const size_t parts = nbytes(split_rows, static_cast<int64_t>(kv_heads) * dim, 8);
  if (flags == kSizeOverflow || rows == kSizeOverflow || parts == kSizeOverflow || rows + flags + 32 < rows || rows + flags + 32 + parts < parts)
    return fail(VDSL_ERR_SHAPE, "attention_bwd workspace size overflows");
  *bytes = rows + flags + parts + 32;
  return VDSL_OK;
}

extern "C" int vdsl_op_attention_bwd(vdsl_queue q, const vdsl_attention_params* p, int32_t dout_dtype, vdsl_buffer dout, vdsl_buffer qs,
                                     vdsl_buffer ks, vdsl_buffer vs, vdsl_buffer starts, int32_t out_dtype, vdsl_buffer out,
                                     vdsl_buffer lse, int32_t grad_dtype, vdsl_buffer dq, vdsl_buffer dk, vdsl_buffer dv,
                                     vdsl_buffer workspace) {
  VDSL_TRY(enter_queue(q));
  if (!p) return fail(VDSL_ERR_INVALID_ARG, "params is null");
  const char* const op = "attention_bwd";
  VDSL_TRY(attention_check_shape(op, p->n, p->seqs, p->heads, p->kv_heads, p->dim));
  VDSL_TRY(attention_check_scale(op, p->scale));
  if (!float_type(dout_dtype) || !float_type(out_dtype) || !float_type(grad_dtype))
    return fail(VDSL_ERR_UNSUPPORTED, "attention_bwd supports f32 and bf16");
  const size_t elem = dtype_size(grad_dtype);
  size_t qb, kb, vb, dqb, dkb, dvb, need;
  VDSL_TRY(attention_check_heads(op, "q", p->q, p->n, p->heads, p->dim, 2, &qb));
  VDSL_TRY(attention_check_heads(op, "k", p->k, p->n, p->kv_heads, p->dim, 2, &kb));
  VDSL_TRY(attention_check_heads(op, "v", p->v, p->n, p->kv_heads, p->dim, 2, &vb));
  VDSL_TRY(attention_check_heads(op, "dq", p->dq, p->n, p->heads, p->dim, elem, &dqb));
  VDSL_TRY(attention_check_heads(op, "dk", p->dk, p->n, p->kv_heads, p->dim, elem, &dkb));
  VDSL_TRY(attention_check_heads(op, "dv", p->dv, p->n, p->kv_heads, p->dim, elem, &dvb));
  const int64_t width = static_cast<int64_t>(p->heads) * p->dim, kv_width = static_cast<int64_t>(p->kv_heads) * p->dim;
  VDSL_TRY(check_buffer(q, dout, nbytes(p->n, width, dtype_size(dout_dtype)), "dout", false));
  VDSL_TRY(check_buffer(q, qs, qb, "q", false));
  VDSL_TRY(check_buffer(q, ks, kb, "k", false));
  VDSL_TRY(check_buffer(q, vs, vb, "v", false));
  VDSL_TRY(check_buffer(q, starts, nbytes(p->seqs + 1, 4), "starts", false));
  VDSL_TRY(check_buffer(q, out, nbytes(p->n, width, dtype_size(out_dtype)), "out", false));
  VDSL_TRY(check_buffer(q, lse, nbytes(p->n, p->heads, 4), "lse", false));
  VDSL_TRY(check_buffer(q, dq, dqb, "dq", true));
  VDSL_TRY(check_buffer(q, dk, dkb, "dk", true));
  VDSL_TRY(check_buffer(q, dv, dvb, "dv", true));
  VDSL_TRY(vdsl_attention_bwd_workspace_bytes(p->n, p->seqs, p->heads, p->kv_heads, p->dim, &need));
  VDSL_TRY(check_buffer(q, workspace, need, "workspace", true));
  for (const vdsl_buffer w : {dq, dk, dv}) VDSL_TRY(check_apart(op, {w, workspace}, {dout, qs, ks, vs, starts, out, lse}));
  if ((dq == dk && !apart(p->dq, width, p->dk, kv_width)) || (dq == dv && !apart(p->dq, width, p->dv, kv_width)) ||
      (dk == dv && !apart(p->dk, kv_width, p->dv, kv_width)))
    return fail(VDSL_ERR_INVALID_ARG, "attention_bwd: gradients in one buffer must be disjoint columns of one stride");
  if (p->n == 0) return VDSL_OK;
  const int group = p->heads / p->kv_heads;
  float* const rows = static_cast<float*>(workspace->ptr);
  const int key_log = key_tile_log(p->n, p->kv_heads, p->causal != 0);
  const int splits = key_log == 6 ? key_splits(p->n, p->seqs, p->heads, p->kv_heads) : 1;
  const int64_t key_slots = row_slots(p->n, p->seqs, 1, key_log), query_slots = row_slots(p->n, p->seqs, group, 7);
  if (std::max(key_slots * splits, query_slots) * p->kv_heads > kMostBlocks)
    return fail(VDSL_ERR_UNSUPPORTED, "attention_bwd: too many rows or sequences");
  const int64_t flags_at = 2 * p->n * p->heads, copy_at = (flags_at + 8 * key_slots * splits * p->kv_heads + 3) & ~int64_t{3};
  uint16_t* const copy = dout_dtype == VDSL_F32 ? reinterpret_cast<uint16_t*>(rows + copy_at) : nullptr;
  GradArgs a = {};
  a.q = static_cast<const uint16_t*>(qs->ptr) + p->q.first;
  a.k = static_cast<const uint16_t*>(ks->ptr) + p->k.first;
  a.v = static_cast<const uint16_t*>(vs->ptr) + p->v.first;
  a.dout = copy ? copy : static_cast<const uint16_t*>(dout->ptr);
  a.q_stride = p->q.stride;
  a.k_stride = p->k.stride;
  a.v_stride = p->v.stride;
  a.dout_stride = width;
  a.seqs = {static_cast<const int32_t*>(starts->ptr), p->n, p->seqs};
  a.rows = rows;
  a.key_log = key_log;
  a.key_splits = splits;
  a.parts = rows + ((copy_at + (copy ? p->n * width / 2 : 0) + 3) & ~int64_t{3});
  a.left_out = reinterpret_cast<int*>(rows + flags_at);
  a.dq = dq->ptr;
  a.dk = dk->ptr;
  a.dv = dv->ptr;
  a.dq_first = p->dq.first;
  a.dq_stride = p->dq.stride;
  a.dk_first = p->dk.first;
  a.dk_stride = p->dk.stride;
  a.dv_first = p->dv.first;
  a.dv_stride = p->dv.stride;
  a.heads = p->heads;
  a.kv_heads = p->kv_heads;
  a.group = group;
  a.dim = p->dim;
  a.causal = p->causal != 0;
  a.grad_dtype = grad_dtype;
  a.scale = p->scale;
  a.token_of = divider(group);
  hipLaunchKernelGGL(attention_bwd_rows, block_grid((p->n * p->heads + 15) / 16), dim3(256), 0, q->stream, dout->ptr, dout_dtype,
                     out->ptr, out_dtype, static_cast<const float*>(lse->ptr), p->n, p->heads, group, p->dim, p->scale, copy, rows);
  VDSL_TRY(check_launch("attention_bwd_rows"));
  const auto go = [&](auto kernel, unsigned lanes, int64_t blocks, const char* name) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(lanes), 0, q->stream, a);
    return check_launch(name);
  };
  const int64_t tiles = key_slots * p->kv_heads, key_blocks = tiles * splits, query_blocks = query_slots * p->kv_heads;
  const auto pick = [&](auto of64, auto of96, auto of128) { return p->dim <= 64 ? of64 : p->dim <= 96 ? of96 : of128; };
  const auto finish = [&]() -> int {
    if (!p->causal && splits == 1) return VDSL_OK;
    hipLaunchKernelGGL(attention_bwd_finish, block_grid(splits > 1 ? kSumBlocks * tiles : tiles), dim3(256), 0, q->stream, a);
    return check_launch("attention_bwd_finish");
  };
  a.blocks = static_cast<int>(query_slots);
  a.key_blocks = static_cast<int>(key_blocks);
  if (key_log == 6) {
    VDSL_TRY(go(pick(attention_bwd_both<64>, attention_bwd_both<96>, attention_bwd_both<128>), 512, key_blocks + query_blocks, "attention_bwd_both"));
    return finish();
  }
  VDSL_TRY(go(pick(attention_bwd_keys<64>, attention_bwd_keys<96>, attention_bwd_keys<128>), 512, key_blocks, "attention_bwd_keys"));
  VDSL_TRY(finish());
  return go(pick(attention_bwd_queries<64>, attention_bwd_queries<96>, attention_bwd_queries<128>), 256, query_blocks, "attention_bwd_queries");
}
