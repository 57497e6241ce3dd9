// The gradient of attention over packed sequences.  With p = exp2(c s - lse log2 e) formed again from q, k and lse,
// dp = dout v, delta = dout out and ds = p (dp - delta):
//   dq = scale ds k (rows' own sum over keys),   dk = scale ds^T q and dv = p^T dout (keys' own sums over rows and heads)
// The launches: delta of each row; dk and dv, a wave holding 32 keys and walking over the rows that see them; dq, a
// wave holding its rows and walking over the keys they see.  Each sum belongs to one wave and is taken in one order, so
// nothing is added atomically and the bits are the same on every call; the price is that s and dp are formed twice (7
// products where 5 would do).  See attention.h for rows, tiles and the order of the products' sums.
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
  int* left_out;      // by the waves of attention_bwd_keys
  int key_log;        // log2 of the keys of one of its blocks
  const float* rows;  // -lse / scale, then -delta, each [kv_heads][n * group]
  void *dq, *dk, *dv;
  int64_t dq_first, dq_stride, dk_first, dk_stride, dv_first, dv_stride;
  int heads, kv_heads, group, dim, causal, grad_dtype;
  float scale;
  Divider token_of;
  int blocks;
};

// What a row's scores and dp start from, -lse / scale and -delta, and dout in bf16 where it is f32.  16 lanes a row of one head.
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

// acc (columns x rows: this lane has columns 32 d + 8 g + 4 (l / 32) + j of its own row) times `by` to element e of `to`.
template <int DP>
__device__ __forceinline__ void store_gradient(const f32x16 (&acc)[DP / 32], float by, int dtype, void* to, int64_t e, int dim) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * d + 8 * g + 4 * ((threadIdx.x & 63) >> 5);
      if (col >= dim) continue;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = acc[d][4 * g + j] * by;
      store_unit<4>(dtype, to, e + col, v);
    }
}
__device__ __forceinline__ void store_zeros(int dtype, void* to, int64_t e, int cols) {
  const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = 0; c < cols; c += 4) store_unit<4>(dtype, to, e + c, none);
}

// dk and dv: a block has KEYS keys and walks over tiles of rows through a ring of two or three slots of LDS.  Each 32 keys
// have 8 / (KEYS / 32) waves, one for each 32 rows of a tile, which add up their sums at the end.  Two waves share a SIMD,
// and one has priority there, so that its exponentials come beside the other's products.  To leave both their
// registers, wide heads' values are an operand read from LDS (V_LDS).
template <int DP, int KEYS>
__global__ __launch_bounds__(512, 2) void attention_bwd_keys(GradArgs a) {
  constexpr int NW = 8, GROUPS = KEYS / 32, PARTS = NW / GROUPS, TR = 32 * PARTS;
  constexpr bool V_LDS = DP > 96;
  using T = TileShape<DP>;
  constexpr int CR = TR / NW;  // of a tile's rows a wave copies
  using Copies = RowCopies<DP, CR>;
  constexpr int SUMS = (NW - GROUPS) * 32 * DP * 4;  // one gradient's sums of all but the first parts
  constexpr int NS = PARTS == 2 ? 3 : 2, SLOT = 2 * TR * T::PITCH, AREA = NS * SLOT + (V_LDS ? KEYS * T::PITCH : 0);
  __shared__ __attribute__((aligned(1024))) char smem[AREA > SUMS ? AREA : SUMS];
  __shared__ __attribute__((aligned(16))) float starts[NW][NS][2][32];  // what the rows' scores and dp start from, a copy a wave
  int b = static_cast<int>(blockIdx.x);
  const int kv = b % a.kv_heads;
  const RowTile tile = row_tile<KEYS == 128 ? 7 : 6>(a.seqs, 1, b / a.kv_heads);
  if (!tile.any) {
    if (threadIdx.x < NW) a.left_out[blockIdx.x * NW + threadIdx.x] = 0;
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int part = wave / GROUPS;  // of a tile's rows
  const int key0 = tile.row + 32 * (wave % GROUPS), key = key0 + (lane & 31);
  const int64_t head_col = static_cast<int64_t>(kv) * a.dim;
  if (tile.seq < 0) {
    if (lane == 0) a.left_out[blockIdx.x * NW + wave] = 0;
    if (key < tile.len && half == 0 && part == 0) {
      store_zeros(a.grad_dtype, a.dk, a.dk_first + (tile.token + key) * a.dk_stride + head_col, a.dim);
      store_zeros(a.grad_dtype, a.dv, a.dv_first + (tile.token + key) * a.dv_stride + head_col, a.dim);
    }
    return;
  }
  if (2 * a.dim < T::PITCH) {
    for (int i = threadIdx.x; i < NS * SLOT / 16; i += 512) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
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
  const int rows = tile.len * a.group;
  const int first = a.causal ? tile.row * a.group / TR : 0, end = (rows + TR - 1) / TR;
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
    float* const to = starts[wave][slot][0];
    const int r = 32 * part + (lane & 31);
    // rows that are not there: no weight
    if (r <= last) lds_copy4(reinterpret_cast<const char*>(sp + (half ? delta_at : 0) + t * TR + r), reinterpret_cast<char*>(to));
    else to[lane] = half ? 0.0f : -3e38f;
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
  fetch(end - 1, 0);
  if (NS == 3 && end - 2 >= first) fetch(end - 2, 1);
  int slot = 0;
  if (wave < 4) __builtin_amdgcn_s_setprio(1);
#pragma unroll 1
  for (int t = end - 1; t >= first; --t) {
    // Every wave has left the tile before.  Of three slots, the next tile, which is whole, may be on its way.
    if (NS == 3 && t > first) dma_wait<2 * Copies::C + 1>();
    else dma_wait<0>();
    dma_barrier();
    if (t - (NS - 1) >= first) fetch(t - (NS - 1), slot == 0 ? NS - 1 : slot - 1);
    const char* const qs = smem + slot * SLOT + part * 32 * T::PITCH;
    const char* const ds = qs + TR * T::PITCH;
    const float* const x = starts[wave][slot][0] + 4 * half;
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
    if constexpr (V_LDS) reads_ahead<14, DP / 8, 2>();  // the first 8 are of what they start from
    else reads_ahead<12, DP / 8, 1>();
    // a row whose q or dout holds an element that is no finite number has no finite score or dp with any key
    bool leave = false;
    if (r0 < all_seen) leave = left_out > 0 || any_not_finite(s) || any_not_finite(p);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(s[i] * scale2);
      p[i] *= s[i];
    }
    if (r0 < all_seen) {
      const int lo = sees_from - r0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool in = 8 * (i / 4) + 4 * half + i % 4 >= lo;
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
  }
  __builtin_amdgcn_s_setprio(0);
  if (lane == 0) a.left_out[blockIdx.x * NW + wave] = left_out;
  // the other parts' sums by way of LDS, one gradient after the other
  float* const sums = reinterpret_cast<float*>(smem) + lane * 4;
  const auto join = [&](f32x16 (&acc)[DP / 32]) {
    __syncthreads();
    if (part != 0) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(sums + (wave - GROUPS) * DP * 32 + (4 * d + g) * 256) = f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
    }
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int o = 0; o < PARTS - 1; ++o)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(sums + (wave + o * GROUPS) * DP * 32 + (4 * d + g) * 256);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[d][4 * g + j] += v[j];
          }
    }
  };
  join(dk);
  join(dv);
  if (part == 0 && key < tile.len) {
    store_gradient<DP>(dk, a.scale, a.grad_dtype, a.dk, a.dk_first + token * a.dk_stride + head_col, a.dim);
    store_gradient<DP>(dv, 1.0f, a.grad_dtype, a.dv, a.dv_first + token * a.dv_stride + head_col, a.dim);
  }
}

// The rows that a block of attention_bwd_keys left out, added to what it stored (so of bf16 gradients rounded once more): row by
// row, each lane taking what its key is seen by.  (A launch of its own, whose blocks mostly find nothing: as a part of
// that kernel it took the registers of its loop.)
template <int DP>
__global__ __launch_bounds__(256) void attention_bwd_left_out(GradArgs a) {
  const int place = static_cast<int>(blockIdx.x);
  const int* const flags = a.left_out + 8 * place;
  int any = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) any |= flags[w];
  if (any == 0) return;
  const int kv = place % a.kv_heads;
  const RowTile tile = a.key_log == 7 ? row_tile<7>(a.seqs, 1, place / a.kv_heads) : row_tile<6>(a.seqs, 1, place / a.kv_heads);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = 1 << (a.key_log - 5), parts = 8 / groups;
  if (wave >= groups) return;
  const int key0 = tile.row + 32 * wave, key = key0 + (lane & 31);
  const int64_t head_col = static_cast<int64_t>(kv) * a.dim, token = tile.token + min(key, tile.len - 1);
  bf16x8 kf[DP / 16], vf[DP / 16];
  load_operand<DP>(a.k + token * a.k_stride + head_col, a.dim, kf);
  load_operand<DP>(a.v + token * a.v_stride + head_col, a.dim, vf);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = MfmaBf16::zero();
  const uint16_t* const qp = a.q + tile.token * a.q_stride + head_col * a.group;
  const uint16_t* const dp = a.dout + tile.token * a.dout_stride + head_col * a.group;
  const float* const sp = a.rows + (static_cast<int64_t>(kv) * a.seqs.n + tile.token) * a.group;
  const float scale2 = a.scale * kLog2e;
  int end = 0;
  for (int p = 0; p < parts; ++p) end = max(end, flags[wave + groups * p]);
  end = min(end, tile.len * a.group);
#pragma unroll 1
  for (int r = key0 * a.group; r < end; ++r) {
    if (r >= flags[wave + groups * ((r >> 5) & (parts - 1))]) continue;
    const int i = a.token_of(r);
    const int64_t col = static_cast<int64_t>(r - i * a.group) * a.dim;
    const uint16_t* const qr = qp + i * a.q_stride + col;
    const uint16_t* const dr = dp + i * a.dout_stride + col;
    const float sr = halves_sum(half_dot<DP>(kf, qr, a.dim)), pr = halves_sum(half_dot<DP>(vf, dr, a.dim));
    if (r < key * a.group) continue;
    const float w = __builtin_amdgcn_exp2f((sr + sp[r]) * scale2);
    add_row<DP>(dv, w, dr, a.dim);
    add_row<DP>(dk, w * (pr + sp[a.seqs.n * a.heads + r]), qr, a.dim);
  }
  if (key >= tile.len) return;
  const auto add = [&](const f32x16 (&acc)[DP / 32], float by, void* to, int64_t e) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * d + 8 * g + 4 * (lane >> 5);
        if (c >= a.dim) continue;
        float v[4];
        load_some(a.grad_dtype, to, e + c, 4, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += acc[d][4 * g + j] * by;
        store_some(a.grad_dtype, to, e + c, 4, v);
      }
  };
  add(dk, a.scale, a.dk, a.dk_first + token * a.dk_stride + head_col);
  add(dv, 1.0f, a.dv, a.dv_first + token * a.dv_stride + head_col);
}

// dq: four waves of 32 rows each, walking over tiles of 64 keys.
template <int DP>
__global__ __launch_bounds__(256, 2) void attention_bwd_queries(GradArgs a) {
  constexpr int KT = 64, ROWS = 128;
  using T = TileShape<DP>;
  using Copies = RowCopies<DP, 16>;  // of a tile's keys by each wave
  constexpr int SLOT = 2 * KT * T::PITCH;
  __shared__ __attribute__((aligned(1024))) char smem[2 * SLOT];
  int b = static_cast<int>(blockIdx.x);
  const int kv = b % a.kv_heads;
  const RowTile tile = row_tile<7>(a.seqs, a.group, a.blocks - 1 - b / a.kv_heads);
  if (!tile.any) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = tile.len * a.group, row0 = tile.row + 32 * wave;
  const int64_t head_col = static_cast<int64_t>(kv) * a.dim;
  const auto dq_at = [&](int row) {
    const int i = a.token_of(row);
    return a.dq_first + (tile.token + i) * a.dq_stride + head_col * a.group + static_cast<int64_t>(row - i * a.group) * a.dim;
  };
  if (tile.seq < 0) {
    for (int row = tile.row + static_cast<int>(threadIdx.x); row < min(tile.row + ROWS, rows); row += 256)
      store_zeros(a.grad_dtype, a.dq, dq_at(row), a.dim);
    return;
  }
  if (2 * a.dim < T::PITCH) {
    for (int i = threadIdx.x; i < 2 * SLOT / 16; i += 256) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  const auto sees = [&](int row) { return a.causal ? a.token_of(row) + 1 : tile.len; };
  const int end = (sees(min(tile.row + ROWS, rows) - 1) + KT - 1) / KT;
  const char* const kp = reinterpret_cast<const char*>(a.k + tile.token * a.k_stride + head_col);
  const char* const vp = reinterpret_cast<const char*>(a.v + tile.token * a.v_stride + head_col);
  Copies copies;
  copies.offsets(0, a.dim, [&](int r) { return 2u * static_cast<uint32_t>(r) * static_cast<uint32_t>(a.k_stride); },
                 [&](int r) { return 2u * static_cast<uint32_t>(r) * static_cast<uint32_t>(a.v_stride); });
  const auto fetch = [&](int t, int slot) {
    const int j = t * KT + 16 * wave;
    char* const area = smem + slot * SLOT + 16 * wave * T::PITCH;
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
    for (int u = 0; u < KT / 32; ++u) add(ks + 32 * u * T::PITCH, form(ks + 32 * u * T::PITCH, nullptr));
  }
  // the others
#pragma unroll 1
  for (; t < end; ++t) {
    enter();
    const char* ks = smem + slot * SLOT;
    slot ^= 1;
#pragma unroll 1
    for (int u = 0; u < KT / 32; ++u, ks += 32 * T::PITCH) {
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
    const uint16_t* const kr = reinterpret_cast<const uint16_t*>(kp) + j * a.k_stride;
    const uint16_t* const vr = reinterpret_cast<const uint16_t*>(vp) + j * a.v_stride;
    const float s = halves_sum(half_dot<DP>(qf, kr, a.dim)), p = halves_sum(half_dot<DP>(df, vr, a.dim));
    if (j >= seen) continue;
    add_row<DP>(dq, __builtin_amdgcn_exp2f((s + score0) * scale2) * (p + dp0), kr, a.dim);
  }
  if (row0 + (lane & 31) < rows) store_gradient<DP>(dq, a.scale, a.grad_dtype, a.dq, dq_at(row), a.dim);
}

// 128 keys a block, or 64 in twice the blocks, each half as long, where 128 would leave CUs idle (full attention) or wait for the
// blocks of the first keys, which the most rows see (causal).  32 heads of 128 over 8: causal, one sequence of 1024 rows 164 us by
// 128 keys and 124 by 64, 2048: 309 and 238, 4096: 684 and 571, 8192: 1820 and 2040; full, 4096: 893 and 1042.
int key_tile_log(int64_t n, int64_t kv_heads, bool causal) {
  return ((n + 127) >> 7) * kv_heads <= (causal ? 256 : 128) ? 6 : 7;
}

bool float_type(int32_t t) { return t == VDSL_F32 || t == VDSL_BF16; }

// Whether two of the gradients, as columns of one buffer, have no element in common.
bool apart(const vdsl_heads& x, int64_t x_width, const vdsl_heads& y, int64_t y_width) {
  if (x.stride != y.stride) return false;
  if (x.first + x_width > x.stride || y.first + y_width > y.stride) return false;
  return x.first + x_width <= y.first || y.first + y_width <= x.first;
}

}  // namespace
}  // namespace vdsl

using namespace vdsl;

// What the rows' scores and dp start from, what attention_bwd_keys left out, a copy of dout in bf16.
extern "C" int vdsl_attention_bwd_workspace_bytes(int64_t n, int64_t seqs, int32_t heads, int32_t kv_heads, int32_t dim, size_t* bytes) {
  if (!bytes) return fail(VDSL_ERR_INVALID_ARG, "bytes is null");
  VDSL_TRY(attention_check_shape("attention_bwd", n, seqs, heads, kv_heads, dim));
  // a multiple of 16 bytes before the copy
  const size_t flags = nbytes(row_slots(n, seqs, 1, 6), kv_heads, 32), rows = nbytes(n, heads, 8 + 2 * static_cast<int64_t>(dim));
  if (flags == kSizeOverflow || rows == kSizeOverflow || rows + flags + 16 < rows)
    return fail(VDSL_ERR_SHAPE, "attention_bwd workspace size overflows");
  *bytes = rows + flags + 16;
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
  const int64_t key_slots = row_slots(p->n, p->seqs, 1, key_log), query_slots = row_slots(p->n, p->seqs, group, 7);
  if (std::max(key_slots, query_slots) * p->kv_heads > 0x3fffff) return fail(VDSL_ERR_UNSUPPORTED, "attention_bwd: too many rows");
  const int64_t flags_at = 2 * p->n * p->heads, copy_at = (flags_at + 8 * key_slots * p->kv_heads + 3) & ~int64_t{3};
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
  const auto go = [&](auto kernel, unsigned lanes, int64_t slots, const char* name) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(slots * p->kv_heads)), dim3(lanes), 0, q->stream, a);
    return check_launch(name);
  };
  a.blocks = static_cast<int>(query_slots);
  const auto keys = a.key_log == 7 ? (p->dim <= 64 ? attention_bwd_keys<64, 128> : p->dim <= 96 ? attention_bwd_keys<96, 128> : attention_bwd_keys<128, 128>)
                                   : (p->dim <= 64 ? attention_bwd_keys<64, 64> : p->dim <= 96 ? attention_bwd_keys<96, 64> : attention_bwd_keys<128, 64>);
  const auto queries = p->dim <= 64 ? attention_bwd_queries<64> : p->dim <= 96 ? attention_bwd_queries<96> : attention_bwd_queries<128>;
  const auto rest = p->dim <= 64 ? attention_bwd_left_out<64> : p->dim <= 96 ? attention_bwd_left_out<96> : attention_bwd_left_out<128>;
  VDSL_TRY(go(keys, 512, key_slots, "attention_bwd_keys"));
  if (p->causal) VDSL_TRY(go(rest, 256, key_slots, "attention_bwd_left_out"));
  return go(queries, 256, query_slots, "attention_bwd_queries");
}
