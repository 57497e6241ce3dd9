// The output layer of a model over a vocabulary with its softmax cross entropy, loss and gradients,
// in pieces of the vocabulary.
//
//   z = x w^T (x bf16 [n][dim], w bf16 [vocab][dim]),  lse_i = log sum_v exp z_iv,
//   loss = mean over the rows that count of lse_i - z_i,label_i  (a row whose label is outside [0, vocab)
//   does not count: no loss, no gradient; the mean over no row is 0),
//   G_iv = exp(z_iv - lse_i) - [v = label_i],  dx = G w / count,  dw = G^T x / count.
//
// The logits are never held as such.  A block forms a tile of them in its accumulators, in f32 and in
// units of log2 (z log2 e), and leaves the maximum and the sum of 2^(z - maximum) of each row over each
// group of columns, from which lse follows.  The gradient needs all of z once lse is known: the last piece
// of the vocabulary leaves 16-bit codes of z for that, the others form their logits again.  A code is the
// distance below its group's maximum in steps of 32 / 65535 octaves, so exp of it is off by at most 1.7e-4
// relative (1e-4 root mean square) wherever it is more than 2^-32 of that maximum (below, it counts as 0), a
// sixteenth of what the rounding of G to bf16 moves it by: a bf16 code
// would double that rounding.  G is rounded to bf16 as every gradient between ops is, and before its
// division by count: the label's entry then lies in [-1, 0), where a rounding is at most 2^-9 of 1.  That entry's
// rounding is nearly all of the gradients' error: 0.9e-3 to 1.5e-3 of their norm in f32 (16 to 8192 rows), 1.9e-3 to
// 2.2e-3 once rounded to bf16, of which that last rounding alone is 1.7e-3.
// Where the vocabulary is one piece that is 6 n vocab dim operations, else up to 8 n vocab dim.
//
// 8192 x 4096, vocabulary 32768, in one piece: logits 1600 to 1720 us on the power-limited card (76% of the cycles in
// MFMAs, at 1.6 GHz), the rows' pass 188 (537 MB of codes in, as much of G out), dx 1490 to 1580, dw 1560 to 1670.
// Gradients in f32 take 1.6% more of a call; pieces of 8192 columns 25% (6170 us for 4950) at half of the workspace.
// 300 x 1000, 5003: 38 in four launches, 67 in three pieces and eight.  16 x 512, 5003: logits 5.5, rows 4.5,
// both gradients 7.5, joining dx's splits 4.

#include <algorithm>

#include "gemm_ring.h"
#include "gemm_wide.h"
#include "rowunit.h"

namespace vdsl {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kCodeOctaves = 32.0f;
constexpr uint32_t kCodeZero = 65535;  // 2^-32 of the group's maximum or less

enum { kLogitStats = 0, kLogitCodes = 1, kLogitGrad = 2 };

// Two codes from two distances below the group's maximum as shares of kCodeOctaves (a NaN: 0, its row is one).
__device__ __forceinline__ uint32_t codes_of(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(a, b));
}

struct LogitArgs {
  const uint16_t* x;       // [n][dim]
  const uint16_t* w;       // the piece's rows, [cols][dim]
  const int32_t* labels;   // [n]
  float2* stats;           // [n][groups]: maximum and sum of 2^(z - maximum) of each group of columns
  float* zlabel;           // [n]: the label's logit, in octaves
  uint16_t* g;             // [n][ldg]: codes, or G
  const float* lse;        // [n], in octaves
  int n, cols, dim, vocab;
  int v0;                  // the piece's first column
  int group0, groups;      // its first group, and all groups
  int64_t ldg;
  int g0;                  // the first of the columns whose codes are wanted, G's first
};

// What a wave does with its tile of logits, 32 FM columns of the vocabulary (one group) from c0 on by 32 FN
// tokens from row0 on.  The vocabulary is C's row side, so a lane has a token's logits of half of the columns:
// the token's maximum and sum need one exchange with the lane of the other half, and four neighbours (eight
// after another exchange) are stored together.  value(i, j, r): the accumulator's element; EDGE: some of the
// columns are not there.  MODE kLogitStats: stats and zlabel; kLogitCodes: also the codes; kLogitGrad: G from lse.
template <int FM, int FN, int MODE, bool EDGE, class Value>
__device__ __forceinline__ void logits_epilogue(const LogitArgs& p, int c0, int row0, Value&& value) {
  const int half = (threadIdx.x & 63) >> 5;
  const int group = p.group0 + c0 / (32 * FM);
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    __builtin_amdgcn_sched_barrier(0);
    const int row = row0 + 32 * j + static_cast<int>(threadIdx.x & 31);
    const bool in = row < p.n;
    const int label = in ? p.labels[row] : -1;
    const bool counts = label >= 0 && label < p.vocab;
    const int at = label - p.v0 - c0;  // among the wave's columns
    const bool here = counts && at >= 0 && at < 32 * FM && at % 8 / 4 == half;
    const bool any_label = __any(here);
    float z[FM][16];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        z[i][r] = value(i, j, r);
        if (EDGE && c0 + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3) >= p.cols) z[i][r] = -INFINITY;
      }
    float base;  // exp2's argument is z log2 e - base
    if constexpr (MODE == kLogitGrad) {
      base = in ? p.lse[row] : 0.0f;
    } else {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, z[i][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * kLog2e;
      base = top == -INFINITY ? 0.0f : top;  // a group of -inf only: a sum of 0
      float s[4] = {};
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(z[i][r], kLog2e, -base));
      float sum = (s[0] + s[1]) + (s[2] + s[3]);
      sum += __shfl_xor(sum, 32, 64);
      if (in && half == 0) p.stats[static_cast<int64_t>(row) * p.groups + group] = make_float2(top, sum);
      if (any_label) {
        float zl = 0.0f;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) zl = at == 32 * i + 8 * (r >> 2) + 4 * half + (r & 3) ? z[i][r] : zl;
        if (here) p.zlabel[row] = zl * kLog2e;
      }
    }
    if constexpr (MODE != kLogitStats) {
      uint16_t* const out = p.g + row * p.ldg + (c0 - p.g0) + 8 * half;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        if constexpr (MODE == kLogitCodes) {
#pragma unroll
          for (int r = 0; r < 16; ++r) z[i][r] = __builtin_fmaf(z[i][r], -kLog2e / kCodeOctaves, base * (1.0f / kCodeOctaves));
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) z[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i][r], kLog2e, -base));
          if (any_label) {
#pragma unroll
            for (int r = 0; r < 16; ++r) z[i][r] -= here && at == 32 * i + 8 * (r >> 2) + 4 * half + (r & 3) ? 1.0f : 0.0f;
          }
        }
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          uint32_t word[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float a = z[i][4 * q + 2 * h], b = z[i][4 * q + 2 * h + 1];
            word[h] = MODE == kLogitCodes ? codes_of(a, b) : pack_bf16x2(counts ? a : 0.0f, counts ? b : 0.0f);
          }
          const u32x4 eight = wide_exchange(word[0], word[1], word[2], word[3]);
          if (in && (!EDGE || c0 - p.g0 + 32 * i + 8 * (q + half) < p.ldg)) *reinterpret_cast<u32x4*>(out + 32 * i + 8 * q) = eight;
        }
      }
    }
  }
}

template <int FM, int FN, int MODE, class Value>
__device__ __forceinline__ void logits_tile(const LogitArgs& p, int c0, int row0, Value&& value) {
  if (c0 >= p.cols) return;
  if (MODE == kLogitCodes && c0 < p.g0) {  // a column of a piece whose logits are formed again
    logits_epilogue<FM, FN, kLogitStats, false>(p, c0, row0, value);  // whole: pieces are multiples of 256
    return;
  }
  if (c0 + 32 * FM <= p.cols) logits_epilogue<FM, FN, MODE, false>(p, c0, row0, value);
  else logits_epilogue<FM, FN, MODE, true>(p, c0, row0, value);
}

template <int MODE>
__global__ __launch_bounds__(WideCfg::NT, 1) void xent_logits_wide(LogitArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[WideCfg::LDS_BYTES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  wide_gemm<false, false>(p.w, p.x, p.cols, p.n, p.dim, p.dim, p.dim, false, smem, [&](const f32x16 (&acc)[4][4], int m0, int n0) {
    logits_tile<4, 4, MODE>(p, m0 + 128 * (wave >> 1), n0 + 128 * (wave & 1),
                            [&](int i, int j, int r) { return wide_value(acc[i][j][r]); });
  });
}

// inv: the gradients' factor, grad_scale over the number of rows that count, and that number's bits (1 if none does).
// area: LDS (the block's only array: with a second one the compiler waits for every copy before each read of the first).
__device__ __forceinline__ void count_rows(const int32_t* __restrict__ labels, int n, int vocab, float grad_scale, float* inv, char* area) {
  int* const part = reinterpret_cast<int*>(area);
  int k = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += blockDim.x) k += labels[i] >= 0 && labels[i] < vocab;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) k += __shfl_xor(k, m, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = k;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (unsigned w = 1; w < blockDim.x / 64; ++w) k += part[w];
  inv[0] = static_cast<float>(static_cast<double>(grad_scale) / (k > 0 ? k : 1));
  inv[1] = __int_as_float(k > 0 ? k : 1);
}

// The smaller tiles, of gemm_ring.h.  Stages in the ring: as many as leave two blocks a CU.
template <int BM_, int BN_, int NS>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, NT = 256;
  template <bool AKM, bool BKM>
  using Loop = RingConfig<BM_, BN_, 2, 2, NS, AKM, BKM>;
  static int64_t tiles(int64_t m, int64_t n) { return ((m + BM - 1) / BM) * ((n + BN - 1) / BN); }
};
using Tile64 = Tile<64, 64, 5>;
using Tile128x64 = Tile<128, 64, 3>;

// The logits on smaller tiles.  The launch has a block more than tiles: the last one counts the rows.
template <class Cfg, int MODE>
__global__ __launch_bounds__(Cfg::NT) void xent_logits_small(LogitArgs p, float grad_scale, float* inv) {
  __shared__ __attribute__((aligned(1024))) char smem[Cfg::LDS_BYTES];
  const int tiles_m = (p.cols + Cfg::BM - 1) / Cfg::BM, tiles_n = (p.n + Cfg::BN - 1) / Cfg::BN, tiles = tiles_m * tiles_n;
  const int64_t block = block_index();
  if (block >= tiles) {
    if (block == tiles) count_rows(p.labels, p.n, p.vocab, grad_scale, inv, smem);
    return;
  }
  int tm, tn;
  tile_coords(xcd_remap(static_cast<int>(block), tiles), tiles_m, tiles_n, tm, tn);
  f32x16 acc[Cfg::FM][Cfg::FN];
  ring_mainloop<Cfg>(p.w, p.x, p.cols, p.n, 0, p.dim, tm * Cfg::BM, tn * Cfg::BN, smem, acc, p.dim, p.dim);
  const int wave = threadIdx.x >> 6;
  logits_tile<Cfg::FM, Cfg::FN, MODE>(p, tm * Cfg::BM + wave / Cfg::WGN * Cfg::WTM, tn * Cfg::BN + wave % Cfg::WGN * Cfg::WTN,
                                      [&](int i, int j, int r) { return acc[i][j][r]; });
}

__device__ __forceinline__ float block_sum_256(float v, float* area) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) area[threadIdx.x >> 6] = v;
  __syncthreads();
  return (area[0] + area[1]) + (area[2] + area[3]);
}
__device__ __forceinline__ float block_max_256(float v, float* area) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) area[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(area[0], area[1]), fmaxf(area[2], area[3]));
}

// Rows of x and w of `dim` elements copied in rows of `ld` (a multiple of 8), zeros behind them; a wave per row.  For
// dims that are no whole units, which neither the copies to LDS nor the 256 x 256 tiles take: a main loop that takes
// any (loads to registers, element-wise edges) needed 13653 us for 8192 x 4093, 32768, this and the others 5029; 300 x
// 1001, 5003 57 and 46.
__global__ __launch_bounds__(256) void xent_layout_kernel(const uint16_t* __restrict__ x, int64_t n, const uint16_t* __restrict__ w,
                                                          int64_t vocab, int64_t dim, uint16_t* __restrict__ x_out,
                                                          uint16_t* __restrict__ w_out, int64_t ld) {
  int64_t row = block_index() * 4 + (threadIdx.x >> 6);
  if (row >= n + vocab) return;
  const bool of_x = row < n;
  if (!of_x) row -= n;
  const uint16_t* const from = (of_x ? x : w) + row * dim;
  uint16_t* const to = (of_x ? x_out : w_out) + row * ld;
#pragma unroll 4
  for (int64_t c = 8 * static_cast<int64_t>(threadIdx.x & 63); c < ld; c += 512) {
    // whole units, the row's last moved back to its end (dim >= 8) and shifted into place
    const UnitAt<8> at(c, dim);
    u32x4 v = reinterpret_cast<const U32x4At2*>(from + at.c)->v;
    if (at.skip) {
      uint16_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = static_cast<uint16_t>(v[j / 2] >> (16 * (j & 1)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t word = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pick = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) pick = k == 2 * j + h + at.skip ? e[k] : pick;
          word |= pick << (16 * h);
        }
        v[j] = word;
      }
    }
    *reinterpret_cast<u32x4*>(to + c) = v;
  }
}

struct RowArgs {
  const int32_t* labels;
  const float2* stats;
  const float* zlabel;
  float* lse_octaves;
  float* lse;       // may be null
  float* row_loss;  // of the workspace
  float* row_loss_out;  // may be null
  uint16_t* g;      // codes in, G out, [n][ldg]; null: none
  int n, cols, vocab, v0, group0, groups, group_cols;
  int64_t ldg, g_rows;
};

// A block per row: lse and the row's loss from the groups' maxima and sums, then G from the codes.  Rows of G
// past n are zeros.  Bound by HBM where there are codes: 5.7 TB/s at 8192 x 32768.
__global__ __launch_bounds__(256) void xent_rows_kernel(RowArgs p) {
  __shared__ float area[2][4];
  const int64_t row = block_index();
  if (row >= p.n) {
    if (row >= p.g_rows) return;
    u32x4* const g = reinterpret_cast<u32x4*>(p.g + row * p.ldg);
    for (int c = 8 * static_cast<int>(threadIdx.x); c < p.ldg; c += 2048) g[c / 8] = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  const float2* const st = p.stats + row * p.groups;
  constexpr int kAhead = 4;  // of this lane's units of 8 codes, loaded before lse is known
  const u32x4* const codes = reinterpret_cast<const u32x4*>(p.g + row * p.ldg);
  u32x4 ahead[kAhead];
  if (p.g) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = 8 * static_cast<int>(threadIdx.x) + 2048 * k;
      ahead[k] = codes[(c < p.ldg ? c : 0) / 8];
    }
  }
  float top = -INFINITY;
  for (int t = threadIdx.x; t < p.groups; t += 256) top = fmaxf(top, st[t].x);
  top = block_max_256(top, area[0]);
  const float base = top == -INFINITY ? 0.0f : top;
  float s = 0.0f;
  for (int t = threadIdx.x; t < p.groups; t += 256) s += st[t].y * __builtin_amdgcn_exp2f(st[t].x - base);
  s = block_sum_256(s, area[1]);
  const float lse = top + log2f(s);
  const int label = p.labels[row];
  const bool counts = label >= 0 && label < p.vocab;
  const float zl = counts ? p.zlabel[row] : 0.0f;
  if (threadIdx.x == 0) {
    const float loss = counts ? (lse - zl) * kLn2 : 0.0f;
    p.lse_octaves[row] = lse;
    p.row_loss[row] = loss;
    if (p.lse) p.lse[row] = lse * kLn2;
    if (p.row_loss_out) p.row_loss_out[row] = loss;
  }
  if (!p.g) return;
  u32x4* const g = reinterpret_cast<u32x4*>(p.g + row * p.ldg);
  const auto to_gradient = [&](int c, u32x4 two) {
    if (c >= p.ldg) return;
    if (counts) {
      const bool none = !(lse > -INFINITY);  // a NaN in the row, or nothing above -inf: NaN in all of its gradient
      const float below = st[p.group0 + (c < p.cols ? c : p.cols - 1) / p.group_cols].x - lse;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t u = h ? two[k] >> 16 : two[k] & 0xFFFFu;
          const int col = c + 2 * k + h;
          v[h] = u != kCodeZero ? __builtin_amdgcn_exp2f(__builtin_fmaf(static_cast<float>(u), -kCodeOctaves / 65535.0f, below)) : 0.0f;
          if (none) v[h] = NAN;
          if (p.v0 + col == label) v[h] = __builtin_amdgcn_exp2f(zl - lse) - 1.0f;
          if (col >= p.cols) v[h] = 0.0f;
        }
        two[k] = pack_bf16x2(v[0], v[1]);
      }
    } else {
      two = u32x4{0u, 0u, 0u, 0u};
    }
    g[c / 8] = two;
  };
  const int c0 = 8 * static_cast<int>(threadIdx.x);
#pragma unroll
  for (int k = 0; k < kAhead; ++k) to_gradient(c0 + 2048 * k, ahead[k]);
  for (int c = c0 + 2048 * kAhead; c < p.ldg; c += 2048 * kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) ahead[k] = codes[(c + 2048 * k < p.ldg ? c + 2048 * k : 0) / 8];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) to_gradient(c + 2048 * k, ahead[k]);
  }
}

// One block: loss = the rows' losses over the number of rows that count, and grad_scale over that number.
__global__ __launch_bounds__(1024) void xent_mean_kernel(const float* __restrict__ row_loss, const int32_t* __restrict__ labels,
                                                         int64_t n, int vocab, float grad_scale, float* __restrict__ loss,
                                                         float* __restrict__ inv) {
  __shared__ double sums[16];
  __shared__ int64_t counts[16];
  double s = 0.0;
  int64_t k = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    s += row_loss[i];
    k += labels[i] >= 0 && labels[i] < vocab;
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    s += __shfl_xor(s, m, 64);
    k += __shfl_xor(k, m, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6] = s;
    counts[threadIdx.x >> 6] = k;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) {
    s += sums[w];
    k += counts[w];
  }
  const double c = k > 0 ? static_cast<double>(k) : 1.0;
  loss[0] = static_cast<float>(s / c);
  inv[0] = static_cast<float>(static_cast<double>(grad_scale) / c);
  inv[1] = __int_as_float(static_cast<int>(c));
}

__global__ __launch_bounds__(256) void xent_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) p[i] = 0;
}

// Eight bf16 values, of which the first n (or all) are stored.
__device__ __forceinline__ void store_eight(uint16_t* to, u32x4 v, int n) {
  if (n >= 8) {
    reinterpret_cast<U32x4At2*>(to)->v = v;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) to[j] = static_cast<uint16_t>(v[j / 2] >> (16 * (j & 1)));
  }
}

// A gradient's product, transposed: out[n][m] = inv sum_k A(m, k) B(n, k), A K-major, so that a lane has
// neighbouring elements of a row of out.  k may be split, and there may be pieces: then the products go to
// sum, [split][n][m] in f32, and a last kernel adds the splits.
struct GradArgs {
  const uint16_t *a, *b;
  int m, n, k;
  int64_t lda, ldb;
  float* sum;          // null: this product is all of it
  bool first;          // of the pieces: sum holds nothing yet
  int splits;
  const float* inv;    // the factor of the result
  void* out;           // [n][m] of out_dt
  int out_dt;
};

template <class Cfg>
__device__ __forceinline__ void grad_tile(const GradArgs& p, int block, char* smem) {
  const int tiles_m = (p.m + Cfg::BM - 1) / Cfg::BM, tiles_n = (p.n + Cfg::BN - 1) / Cfg::BN, tiles = tiles_m * tiles_n;
  const int split = block / tiles;
  int tm, tn;
  tile_coords(block - split * tiles, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * Cfg::BM, n0 = tn * Cfg::BN;
  const int stages = (p.k + 63) / 64;
  const int kb = 64 * static_cast<int>(static_cast<int64_t>(stages) * split / p.splits);
  const int ke = min(p.k, 64 * static_cast<int>(static_cast<int64_t>(stages) * (split + 1) / p.splits));
  f32x16 acc[Cfg::FM][Cfg::FN];
  if (kb < ke) {  // block-uniform
    ring_mainloop<Cfg>(p.a, p.b, p.m, p.n, kb, ke, m0, n0, smem, acc, p.lda, p.ldb);
  } else {
#pragma unroll
    for (int i = 0; i < Cfg::FM; ++i)
#pragma unroll
      for (int j = 0; j < Cfg::FN; ++j) acc[i][j] = MfmaBf16::zero();
  }
  const int half = (threadIdx.x & 63) >> 5, wave = threadIdx.x >> 6;
  const float inv = p.inv[0];
  float* const sum = p.sum ? p.sum + static_cast<int64_t>(split) * p.n * p.m : nullptr;
#pragma unroll
  for (int j = 0; j < Cfg::FN; ++j) {
    const int row = n0 + wave % Cfg::WGN * Cfg::WTN + 32 * j + static_cast<int>(threadIdx.x & 31);
    const int col0 = m0 + wave / Cfg::WGN * Cfg::WTM;
    if (!sum && p.out_dt == VDSL_BF16) {  // the lane of the other half has the row's next four
      uint16_t* const out = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(row) * p.m;
#pragma unroll
      for (int i = 0; i < Cfg::FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          uint32_t word[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) word[h] = pack_bf16x2(acc[i][j][4 * q + 2 * h] * inv, acc[i][j][4 * q + 2 * h + 1] * inv);
          const u32x4 eight = wide_exchange(word[0], word[1], word[2], word[3]);
          const int col = col0 + 32 * i + 8 * (q + half);
          if (row < p.n && col < p.m) store_eight(out + col, eight, p.m - col);
        }
      continue;
    }
    if (row >= p.n) continue;
#pragma unroll
    for (int i = 0; i < Cfg::FM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = col0 + 32 * i + 8 * q + 4 * half;
        const int64_t o = static_cast<int64_t>(row) * p.m + col;
        float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        if (sum) {
          if (!p.first) {
            float before[4];
            load_some(VDSL_F32, sum, o, p.m - col, before);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += before[e];
          }
          store_some(VDSL_F32, sum, o, p.m - col, v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= inv;
          store_some(p.out_dt, p.out, o, p.m - col, v);
        }
      }
  }
}

__device__ __forceinline__ void mean_loss(const float* __restrict__ row_loss, int64_t n, const float* __restrict__ inv,
                                          float* __restrict__ loss, char* area) {
  double* const sums = reinterpret_cast<double*>(area);
  double s = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) s += row_loss[i];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (unsigned w = 1; w < blockDim.x / 64; ++w) s += sums[w];
  loss[0] = static_cast<float>(s / __float_as_int(inv[1]));
}

// Both gradients of a piece in one launch, dx's blocks first (they have the longer sums); loss, if not null:
// one more block, which forms the mean loss.
template <class T>
__global__ __launch_bounds__(T::NT) void xent_grads_small(GradArgs dx, GradArgs dw, int64_t dx_blocks, int64_t dw_blocks,
                                                            const float* row_loss, float* loss) {
  using ForDx = typename T::template Loop<true, false>;
  using ForDw = typename T::template Loop<true, true>;
  __shared__ __attribute__((aligned(1024))) char smem[ForDx::LDS_BYTES > ForDw::LDS_BYTES ? ForDx::LDS_BYTES : ForDw::LDS_BYTES];
  const int64_t block = block_index();
  if (block < dx_blocks) grad_tile<ForDx>(dx, static_cast<int>(block), smem);
  else if (block < dx_blocks + dw_blocks) grad_tile<ForDw>(dw, static_cast<int>(block - dx_blocks), smem);
  else if (loss && block == dx_blocks + dw_blocks) mean_loss(row_loss, dx.n, dx.inv, loss, smem);
}

// out = inv times the sum of the splits, four elements a lane, of one or two gradients.
struct Join {
  const float* sum;
  int splits, out_dt;
  int64_t n;  // elements, 0: nothing to do
  void* out;
};
__global__ __launch_bounds__(64) void xent_join_kernel(Join dx, Join dw, int64_t dx_blocks, const float* __restrict__ inv) {
  int64_t block = block_index();
  const Join p = block < dx_blocks ? dx : dw;
  if (block >= dx_blocks) block -= dx_blocks;
  const int64_t e = (block * 64 + threadIdx.x) * 4;
  if (e >= p.n) return;
  float s[4] = {};
#pragma unroll 8
  for (int k = 0; k < p.splits; ++k) {
    float v[4];
    load_some(VDSL_F32, p.sum, k * p.n + e, p.n - e, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += v[j];
  }
  const float f = inv[0];
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] *= f;
  store_some(p.out_dt, p.out, e, p.n - e, s);
}

// The gradients' products on tiles of gemm_wide.h: out[n][m] from A(m, k) and B(n, k), so that a lane has
// neighbouring elements of a row of out.
struct WideGradArgs {
  const uint16_t *a, *b;
  int m, n, k;         // m, n: of out
  int n_alloc;         // of B, where it is K-major: columns that are allocated (of A: lda)
  int64_t lda, ldb;
  float* sum;          // [splits][n][m] f32, the pieces' sum
  int held;            // splits of sum that hold something already
  bool last;           // of the pieces: the result is whole (never with splits)
  int splits;          // of k, blockIdx.y's: no more than k has stages
  const float* inv;
  void* out;
  int out_dt;
};

// Four elements from e on, of which the first n (or all) are the row's, to sum or to out.
__device__ __forceinline__ void store_sum(const WideGradArgs& p, float* sum, float inv, int64_t e, int n, float (&v)[4]) {
  if (static_cast<int>(blockIdx.y) < p.held) {
    float before[4];
    load_some(VDSL_F32, sum, e, n, before);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += before[j];
  }
  if (!p.last) {
    store_some(VDSL_F32, sum, e, n, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] *= inv;
  store_some(p.out_dt, p.out, e, n, v);
}

// WHOLE: the product is all of the sum, rounded to bf16; otherwise any of the forms.
template <bool BKM, bool WHOLE>
__global__ __launch_bounds__(WideCfg::NT, 1) void xent_grad_wide(WideGradArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[WideCfg::LDS_BYTES];
  const int half = (threadIdx.x & 63) >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inv = p.inv[0];
  const int64_t stages = (p.k + 63) / 64;
  const int kb = 64 * static_cast<int>(stages * blockIdx.y / p.splits);
  const int ke = min(p.k, 64 * static_cast<int>(stages * (blockIdx.y + 1) / p.splits));
  const uint16_t *const a = p.a + kb * p.lda, *const b = p.b + (BKM ? kb * p.ldb : kb);
  float* const sum = p.sum + static_cast<int64_t>(blockIdx.y) * p.n * p.m;
  const int cols = BKM ? p.n_alloc : p.n;
  wide_gemm<true, BKM>(a, b, static_cast<int>(p.lda), cols, ke - kb, p.lda, p.ldb, BKM, smem, [&](const f32x16 (&acc)[4][4], int m0, int n0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = n0 + 128 * (wave & 1) + 32 * j + static_cast<int>(threadIdx.x & 31);
      const int c0 = m0 + 128 * (wave >> 1);
      const int64_t out = static_cast<int64_t>(row) * p.m + c0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        float v[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = wide_value(acc[i][j][r]);
        if constexpr (WHOLE) {
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            uint32_t word[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) word[h] = pack_bf16x2(v[4 * q + 2 * h] * inv, v[4 * q + 2 * h + 1] * inv);
            const u32x4 eight = wide_exchange(word[0], word[1], word[2], word[3]);
            const int c = 32 * i + 8 * (q + half);
            if (row < p.n && c0 + c < p.m) store_eight(static_cast<uint16_t*>(p.out) + out + c, eight, p.m - c0 - c);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c = 32 * i + 8 * q + 4 * half;
            if (row >= p.n || c0 + c >= p.m) continue;
            float four[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            store_sum(p, sum, inv, out + c, p.m - c0 - c, four);
          }
        }
      }
    }
  });
}

// ---- host ----------------------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

enum Tiling { kTiles64, kTiles128x64, kTilesWide };

// go(tile) for one of the smaller tiles.
template <class Go>
int on_tile(Tiling t, Go&& go) {
  return t == kTiles64 ? go(Tile64{}) : go(Tile128x64{});
}

// Whether a gradient takes 3 2^32 products or more.
bool many_products(int64_t n, int64_t cols, int64_t dim) { return n * cols >= ceil_div(int64_t{3} << 32, dim); }

// Whether products may take gemm_wide.h's tiles: whole stages of dim, or so many products that laying out the rows
// in whole stages is worth it; offsets of 256 rows that fit 32 bits.
bool wide_fits(int64_t n, int64_t cols, int64_t dim) {
  const bool whole = dim % 64 == 0 || (many_products(n, cols, dim) && 4 * dim >= 3 * (ceil_div(dim, 64) * 64));
  return whole && dim < (1 << 22) && cols < (1 << 22);
}

// How many 128 x 64 tiles an m x n product has.
int64_t small_tiles(int64_t m, int64_t n) { return ceil_div(m, 128) * ceil_div(n, 64); }

// The logits' tiles.  256 x 256 where they use half of the card or more: a CU takes about 1 us for a stage of such a
// tile on a card that is half idle (1.6 at full power), 0.42 for one of 128 x 64, an eighth of that.  Us of a loss,
// 256 x 256 and 128 x 64: 2048 rows of 512, 8192 columns (the card full) 26.5, 34.5; 2048 x 1024, 5003 (61%) 33.6,
// 37.5; 1024 x 1024, 8192 (half) 30.7, 30.0; 512 x 4096, 8192 (a quarter) 73, 43.5.
// 64 x 64 where the others leave half of the CUs without one (64 x 64 and 128 x 64): 64 x 1000, 5003 (40 tiles)
// 12.5, 14.5; 128 x 512, 8192 (128) 11.1, 11.9; 300 x 1000, 5003 (200) 16.8, 15.7; 1 x 4096, 32768 (256) 45.5, 43.3.
Tiling logit_tiles(int64_t n, int64_t cols, int64_t dim) {
  const int64_t rounds = ceil_div(ceil_div(n, 256) * ceil_div(cols, 256), 256);
  if (wide_fits(n, cols, dim) && 2 * n * cols > rounds * 256 * 256 * 256) return kTilesWide;
  return small_tiles(cols, n) <= 128 ? kTiles64 : kTiles128x64;
}

// The gradients' tiles, of both products.  256 x 256 from 3 2^32 products of a gradient on: they are two launches,
// join f32 sums where they leave CUs idle and count the rows apart, 40 us.  Us of a call, 256 x 256 and 128 x 64:
// 128 rows of 4096, 32768 columns 252, 272; 1024 x 2048, 8192 149, 152; 1024 x 1024, 12288 (the bound) 126, 131;
// 2048 x 1024, 5003 131, 113; 300 x 1024, 32768 146, 137; 64 x 1024, 32768 92, 72.
// 64 x 64 where two blocks to a CU have two stages of the others each or fewer (64 x 64 and 128 x 64): 16 x 512, 5003
// 20.3, 22.6; 512 x 256, 1000 17.4, 18.7; 64 x 1000, 5003 28.9, 27.1; 300 x 512, 8192 40.9, 37.3.
Tiling grad_tiles(int64_t n, int64_t cols, int64_t dim) {
  if (wide_fits(n, cols, dim) && many_products(n, cols, dim)) return kTilesWide;
  const int64_t stages = small_tiles(dim, n) * ceil_div(cols, 64) + small_tiles(dim, cols) * ceil_div(n, 64);
  return stages <= 1024 ? kTiles64 : kTiles128x64;
}
int64_t rows_of(Tiling t) { return t == kTiles64 ? 64 : 128; }

// How a call is laid out: the pieces, the tiles and the workspace.
struct Plan {
  int64_t piece = 0, pieces = 0;  // columns of a piece (the last may have fewer)
  Tiling logits = kTiles64, again = kTiles64, grads = kTiles64;  // of all logits, of a piece's formed again, of the gradients
  int64_t group_cols = 0, groups = 0;
  int64_t g_rows = 0, ldg = 0;    // of G; its rows past n are zeros
  int64_t ld = 0;                 // of x and w: dim, or that of their copies in whole units (stages, for 256 x 256 tiles)
  int splits = 1, dw_splits = 1;  // of the sums over a piece's columns for dx, over the rows for dw
  int last_splits = 1;            // of dx's that the last piece fills: it may be a few columns of many pieces' remainder
  bool sum = false;               // whether dx is formed by way of f32 sums (dw: where it has splits)
  size_t at_stats = 0, at_zlabel = 0, at_lse = 0, at_row_loss = 0, at_inv = 0, at_g = 0, at_sum = 0, at_dw_sum = 0, at_x = 0, at_w = 0, bytes = 0;
};

// The splits of the k of an m x n product on 256 x 256 tiles: as many as make its time least, rounds of a block on
// each CU times their stages (1.6 us each) and what writing and adding the f32 sums takes (at 5 TB/s, and a launch).
// Us of a call so and without splits: 2048 x 1024, 32768 428, 803; 8192 x 512, 32768 1023, 1347; 8192 x 1024, 32768 1575,
// 1751; 2048 x 4096, 32768 1194, 1351; 4096 x 4096, 8192 (none taken) 570, with two 737.
int wide_splits(int64_t n, int64_t m, int64_t k) {
  const int64_t tiles = ceil_div(n, 256) * ceil_div(m, 256), stages = ceil_div(k, 64);
  int best = 1;
  double least = 0.0;
  for (int s = 1; s <= 16 && stages >= 4 * s; ++s) {
    const double us = 1.6 * static_cast<double>(ceil_div(tiles * s, 256) * ceil_div(stages, s)) +
                      (s > 1 ? 6.0 + static_cast<double>(n) * static_cast<double>(m) * 8.0 * s / 5e6 : 0.0);
    if (s > 1 && us >= least) continue;
    best = s;
    least = us;
  }
  return best;
}

constexpr int64_t kPieceBytes = int64_t{1} << 30;  // of codes, where the caller leaves the piece to the library
// ... and of any piece at least, since smaller ones spare less than the f32 sums of dx that pieces need and cost three
// launches each: 300 x 1000, vocabulary 5003, whole 39 us, in three pieces 67; 8 x 1168, 28960 71, in 15 242.
constexpr int64_t kPieceLeastBytes = int64_t{4} << 20;
constexpr int64_t kPieceMost = int64_t{1} << 24;   // columns: the offsets of 64 rows of G fit 32 bits

int make_plan(int64_t n, int64_t vocab, int64_t dim, int64_t piece, bool backward, Plan& p) {
  if (n < 0 || vocab < 0 || dim < 0 || piece < 0) return fail(VDSL_ERR_INVALID_ARG, "linear_xent: negative extent");
  if (vocab == 0) return fail(VDSL_ERR_INVALID_ARG, "linear_xent: the vocabulary is empty");
  if (dim < 8) return fail(VDSL_ERR_UNSUPPORTED, "linear_xent: dim must be at least 8");
  if (n > 0x7fffff00 || vocab > 0x7fffff00 || dim > 0x7fff00) return fail(VDSL_ERR_UNSUPPORTED, "linear_xent: extents too large");
  if (piece == 0) piece = std::max<int64_t>(256, kPieceBytes / 2 / std::max<int64_t>(n, 1));
  piece = std::max(piece, kPieceLeastBytes / 2 / std::max<int64_t>(n, 1));
  piece = backward ? std::min({piece, vocab, kPieceMost}) : vocab;
  p.pieces = ceil_div(vocab, std::min(vocab, ceil_div(piece, 256) * 256));
  p.piece = p.pieces == 1 ? vocab : ceil_div(ceil_div(vocab, p.pieces), 256) * 256;
  p.pieces = ceil_div(vocab, p.piece);
  p.logits = logit_tiles(n, vocab, dim);
  if (backward) {
    p.again = logit_tiles(n, p.piece, dim);
    p.grads = grad_tiles(n, p.piece, dim);
  }
  const bool wide = p.logits == kTilesWide || p.again == kTilesWide || p.grads == kTilesWide;
  p.ld = wide ? ceil_div(dim, 64) * 64 : ceil_div(dim, 8) * 8;
  p.group_cols = p.logits == kTilesWide ? 128 : rows_of(p.logits) / 2;
  p.groups = ceil_div(vocab, p.group_cols);  // pieces are whole groups
  const int64_t unit = p.grads == kTilesWide ? 256 : 8;
  p.ldg = ceil_div(p.piece, unit) * unit;
  p.g_rows = p.grads == kTilesWide ? ceil_div(n, 64) * 64 : n;
  if (backward && p.grads == kTilesWide) {
    p.splits = wide_splits(n, dim, p.piece);
    p.dw_splits = wide_splits(p.piece, dim, n);
    p.last_splits = static_cast<int>(std::min<int64_t>(p.splits, ceil_div(vocab - (p.pieces - 1) * p.piece, 64)));
  } else if (backward) {
    // One launch: splits of as many stages as two blocks a CU come to, but of 12 or more, since each split's sums are
    // written and read again (us with 12 and with 5: 16 x 512, 5003 20.3, 22.3; 300 x 1000, 5003 37.6, 39.6; 128 x 512,
    // 8192 27.8, 33.6).
    const auto tiles = [&](int64_t rows) { return ceil_div(dim, rows_of(p.grads)) * ceil_div(rows, 64); };
    const int64_t x_stages = ceil_div(p.piece, 64), w_stages = ceil_div(n, 64);
    const int64_t share = std::max<int64_t>(12, ceil_div(tiles(n) * x_stages + tiles(p.piece) * w_stages, 512));
    p.splits = p.last_splits = static_cast<int>(std::clamp<int64_t>(ceil_div(x_stages, share), 1, 64));  // (any may be empty)
    p.dw_splits = static_cast<int>(std::clamp<int64_t>(ceil_div(w_stages, share), 1, 64));
  }
  p.sum = p.pieces > 1 || p.splits > 1;  // (forward: one piece, no splits)
  size_t at = 0;
  bool fits = true;
  const auto take = [&](int64_t a, int64_t b, int64_t c) {
    const size_t from = at, size = nbytes(a, b, c);
    if (size == kSizeOverflow || __builtin_add_overflow(at, size, &at) || at > kSizeOverflow - 512) fits = false;
    else at = (at + 255) / 256 * 256;
    return from;
  };
  p.at_stats = take(n, p.groups, 8);
  p.at_zlabel = take(n, 4, 1);
  p.at_lse = take(n, 4, 1);
  p.at_row_loss = take(n, 4, 1);
  p.at_inv = take(2, 4, 1);
  if (p.ld != dim) {
    p.at_x = take(n, p.ld, 2);
    p.at_w = take(vocab, p.ld, 2);
  }
  if (backward) {
    p.at_g = take(p.g_rows, p.ldg, 2);
    if (p.sum) p.at_sum = take(n, dim, 4 * p.splits);
    if (p.dw_splits > 1) p.at_dw_sum = take(p.piece, dim, 4 * p.dw_splits);
  }
  p.bytes = at;
  return fits ? VDSL_OK : fail(VDSL_ERR_SHAPE, "linear_xent: the workspace's size overflows");
}

template <class Cfg, int MODE>
int launch_logits_small(const LogitArgs& a, float grad_scale, float* inv, hipStream_t s) {
  const int64_t tiles = ceil_div(a.cols, Cfg::BM) * ceil_div(a.n, Cfg::BN);
  if (tiles >= 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "linear_xent: too many tiles");
  hipLaunchKernelGGL((xent_logits_small<Cfg, MODE>), block_grid(tiles + 1), dim3(Cfg::NT), 0, s, a, grad_scale, inv);
  return check_launch("xent_logits_small");
}

template <int MODE>
int launch_logits(const LogitArgs& a, Tiling tiling, float grad_scale, float* inv, hipStream_t s) {
  if (tiling != kTilesWide) {
    return on_tile(tiling, [&](auto tile) {
      return launch_logits_small<typename decltype(tile)::template Loop<false, false>, MODE>(a, grad_scale, inv, s);
    });
  }
  hipLaunchKernelGGL(xent_logits_wide<MODE>, dim3(wide_blocks(ceil_div(a.n, 256) * ceil_div(a.cols, 256))), dim3(WideCfg::NT), 0, s, a);
  return check_launch("xent_logits_wide");
}

template <class T>
int launch_grads_small(const GradArgs& dx, const GradArgs& dw, const float* row_loss, float* loss, hipStream_t s) {
  const int64_t x = T::tiles(dx.m, dx.n) * dx.splits, w = T::tiles(dw.m, dw.n) * dw.splits;
  if (x > 0x7fffffff || w > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "linear_xent: too many tiles");
  const dim3 grid = block_grid(x + w + (loss ? 1 : 0));
  hipLaunchKernelGGL(xent_grads_small<T>, grid, dim3(T::NT), 0, s, dx, dw, x, w, row_loss, loss);
  return check_launch("xent_grads_small");
}

template <bool BKM>
int launch_grad_wide(const WideGradArgs& a, int64_t n, hipStream_t s) {
  const dim3 grid(wide_blocks(ceil_div(a.m, 256) * ceil_div(n, 256)), static_cast<unsigned>(a.splits));
  if (a.held == 0 && a.last && a.out_dt == VDSL_BF16)
    hipLaunchKernelGGL((xent_grad_wide<BKM, true>), grid, dim3(WideCfg::NT), 0, s, a);
  else
    hipLaunchKernelGGL((xent_grad_wide<BKM, false>), grid, dim3(WideCfg::NT), 0, s, a);
  return check_launch("xent_grad_wide");
}

int run_xent(vdsl_queue q, int64_t n, int64_t dim, int64_t vocab, vdsl_buffer x, vdsl_buffer w, vdsl_buffer labels, int64_t piece,
             vdsl_buffer loss, vdsl_buffer row_loss, vdsl_buffer lse, bool backward, float grad_scale, int32_t dx_dtype,
             vdsl_buffer dx, int32_t dw_dtype, vdsl_buffer dw, vdsl_buffer workspace) {
  VDSL_TRY(enter_queue(q));
  Plan plan;
  VDSL_TRY(make_plan(n, vocab, dim, piece, backward, plan));
  const auto float_type = [](int32_t t) { return t == VDSL_F32 || t == VDSL_BF16; };
  if (backward && (!float_type(dx_dtype) || !float_type(dw_dtype)))
    return fail(VDSL_ERR_UNSUPPORTED, "linear_xent_fwd_bwd stores f32 and bf16 gradients");
  VDSL_TRY(check_buffer(q, x, nbytes(n, dim, 2), "x", false));
  VDSL_TRY(check_buffer(q, w, nbytes(vocab, dim, 2), "w", false));
  VDSL_TRY(check_buffer(q, labels, nbytes(n, 4), "labels", false));
  VDSL_TRY(check_buffer(q, loss, 4, "loss", true));
  if (row_loss) VDSL_TRY(check_buffer(q, row_loss, nbytes(n, 4), "row_loss", true));
  if (lse) VDSL_TRY(check_buffer(q, lse, nbytes(n, 4), "lse", true));
  if (backward) {
    VDSL_TRY(check_buffer(q, dx, nbytes(n, dim, dtype_size(dx_dtype)), "dx", true));
    VDSL_TRY(check_buffer(q, dw, nbytes(vocab, dim, dtype_size(dw_dtype)), "dw", true));
  }
  VDSL_TRY(check_buffer(q, workspace, plan.bytes, "workspace", true));
  VDSL_TRY(check_apart("linear_xent", {loss, row_loss, lse, dx, dw, workspace}, {x, w, labels}));
  const hipStream_t s = q->stream;
  char* const ws = static_cast<char*>(workspace->ptr);
  const int32_t* lab = static_cast<const int32_t*>(labels->ptr);
  float* const inv = reinterpret_cast<float*>(ws + plan.at_inv);
  float* const each = reinterpret_cast<float*>(ws + plan.at_row_loss);
  float* const loss_out = static_cast<float*>(loss->ptr);
  uint16_t* const g = backward ? reinterpret_cast<uint16_t*>(ws + plan.at_g) : nullptr;
  const int64_t last_piece = (plan.pieces - 1) * plan.piece;
  LogitArgs la{};
  la.x = static_cast<const uint16_t*>(x->ptr);
  const uint16_t* w_rows = static_cast<const uint16_t*>(w->ptr);
  la.labels = lab;
  la.stats = reinterpret_cast<float2*>(ws + plan.at_stats);
  la.zlabel = reinterpret_cast<float*>(ws + plan.at_zlabel);
  la.g = g;
  la.lse = reinterpret_cast<const float*>(ws + plan.at_lse);
  la.n = static_cast<int>(n);
  la.cols = la.vocab = static_cast<int>(vocab);
  la.dim = static_cast<int>(plan.ld);
  la.groups = static_cast<int>(plan.groups);
  la.ldg = plan.ldg;
  la.g0 = static_cast<int>(last_piece);
  if (n > 0 && plan.ld != dim) {
    uint16_t* const x_copy = reinterpret_cast<uint16_t*>(ws + plan.at_x);
    uint16_t* const w_copy = reinterpret_cast<uint16_t*>(ws + plan.at_w);
    hipLaunchKernelGGL(xent_layout_kernel, block_grid(ceil_div(n + vocab, 4)), dim3(256), 0, s, la.x, n, w_rows, vocab, dim, x_copy, w_copy,
                       plan.ld);
    VDSL_TRY(check_launch("xent_layout_kernel"));
    la.x = x_copy;
    w_rows = w_copy;
  }
  la.w = w_rows;
  if (n > 0) {
    if (backward) VDSL_TRY(launch_logits<kLogitCodes>(la, plan.logits, grad_scale, inv, s));
    else VDSL_TRY(launch_logits<kLogitStats>(la, plan.logits, grad_scale, inv, s));
    RowArgs ra{};
    ra.labels = lab;
    ra.stats = la.stats;
    ra.zlabel = la.zlabel;
    ra.lse_octaves = reinterpret_cast<float*>(ws + plan.at_lse);
    ra.lse = lse ? static_cast<float*>(lse->ptr) : nullptr;
    ra.row_loss = each;
    ra.row_loss_out = row_loss ? static_cast<float*>(row_loss->ptr) : nullptr;
    ra.g = g;
    ra.n = la.n;
    ra.cols = static_cast<int>(vocab - last_piece);
    ra.vocab = la.vocab;
    ra.v0 = static_cast<int>(last_piece);
    ra.group0 = static_cast<int>(last_piece / plan.group_cols);
    ra.groups = la.groups;
    ra.group_cols = static_cast<int>(plan.group_cols);
    ra.ldg = plan.ldg;
    ra.g_rows = backward ? plan.g_rows : n;
    hipLaunchKernelGGL(xent_rows_kernel, block_grid(ra.g_rows), dim3(256), 0, s, ra);
    VDSL_TRY(check_launch("xent_rows_kernel"));
  }
  // (the smaller tiles' launches have blocks for the loss and for the factor of the gradients)
  const bool mean_apart = !backward || n == 0 || plan.logits == kTilesWide || plan.grads == kTilesWide;
  if (mean_apart) {
    hipLaunchKernelGGL(xent_mean_kernel, dim3(1), dim3(1024), 0, s, each, lab, n, la.vocab, grad_scale, loss_out, inv);
    VDSL_TRY(check_launch("xent_mean_kernel"));
  }
  if (!backward) return VDSL_OK;
  if (n == 0) {
    hipLaunchKernelGGL(xent_zero_kernel, dim3(2048), dim3(256), 0, s, static_cast<uint16_t*>(dw->ptr),
                       vocab * dim * static_cast<int64_t>(dtype_size(dw_dtype) / 2));
    return check_launch("xent_zero_kernel");
  }
  float* const sum = plan.sum ? reinterpret_cast<float*>(ws + plan.at_sum) : nullptr;
  float* const dw_sum = plan.dw_splits > 1 ? reinterpret_cast<float*>(ws + plan.at_dw_sum) : nullptr;
  la.g0 = 0;
  const int out_cols = static_cast<int>(dim);
  // The piece whose codes are held comes first, then those whose logits are formed again.
  for (int64_t t = 0; t < plan.pieces; ++t) {
    const int64_t v0 = last_piece - t * plan.piece;
    la.w = w_rows + v0 * plan.ld;
    la.v0 = static_cast<int>(v0);
    la.cols = static_cast<int>(std::min(plan.piece, vocab - v0));
    const bool last = t == plan.pieces - 1;
    if (t > 0) VDSL_TRY(launch_logits<kLogitGrad>(la, plan.again, grad_scale, inv, s));
    void* const dw_piece = static_cast<char*>(dw->ptr) + v0 * dim * static_cast<int64_t>(dtype_size(dw_dtype));
    if (plan.grads == kTilesWide) {
      // the last piece comes first and may not fill the splits; those it leaves start with the next piece
      const int splits = t == 0 ? plan.last_splits : plan.splits, held = t == 0 ? 0 : t == 1 ? plan.last_splits : plan.splits;
      const WideGradArgs for_dx{la.w, g, out_cols, la.n, la.cols, 0, plan.ld, plan.ldg, sum, held, last && plan.splits == 1,
                                splits, inv, dx->ptr, dx_dtype};
      VDSL_TRY(launch_grad_wide<false>(for_dx, n, s));
      const WideGradArgs for_dw{la.x, g, out_cols, la.cols, la.n, static_cast<int>(plan.ldg), plan.ld, plan.ldg, dw_sum, 0, !dw_sum,
                                plan.dw_splits, inv, dw_piece, dw_dtype};
      VDSL_TRY(launch_grad_wide<true>(for_dw, plan.ldg, s));
    } else {
      const GradArgs for_dx{la.w, g, out_cols, la.n, la.cols, plan.ld, plan.ldg, sum, t == 0, plan.splits, inv, dx->ptr, dx_dtype};
      const GradArgs for_dw{la.x, g, out_cols, la.cols, la.n, plan.ld, plan.ldg, dw_sum, true, plan.dw_splits, inv, dw_piece, dw_dtype};
      float* const mean = t == 0 && !mean_apart ? loss_out : nullptr;
      VDSL_TRY(on_tile(plan.grads, [&](auto tile) { return launch_grads_small<decltype(tile)>(for_dx, for_dw, each, mean, s); }));
    }
    // a wide dx without splits is whole with its last piece
    const bool join_dx = last && sum && (plan.grads != kTilesWide || plan.splits > 1);
    if (!join_dx && !dw_sum) continue;
    const Join for_x{sum, plan.splits, dx_dtype, join_dx ? n * dim : 0, dx->ptr};
    const Join for_w{dw_sum, plan.dw_splits, dw_dtype, dw_sum ? la.cols * dim : 0, dw_piece};
    const int64_t x_blocks = ceil_div(for_x.n, 256);
    hipLaunchKernelGGL(xent_join_kernel, block_grid(x_blocks + ceil_div(for_w.n, 256)), dim3(64), 0, s, for_x, for_w, x_blocks, inv);
    VDSL_TRY(check_launch("xent_join_kernel"));
  }
  return VDSL_OK;
}

}  // namespace
}  // namespace vdsl

using namespace vdsl;

extern "C" int vdsl_linear_xent_workspace_bytes(int64_t n, int64_t vocab, int64_t dim, int64_t piece, int32_t backward, size_t* bytes) {
  if (!bytes) return fail(VDSL_ERR_INVALID_ARG, "bytes is null");
  Plan plan;
  VDSL_TRY(make_plan(n, vocab, dim, piece, backward != 0, plan));
  *bytes = plan.bytes;
  return VDSL_OK;
}

extern "C" int vdsl_debug_linear_xent_plan(int64_t n, int64_t vocab, int64_t dim, int64_t piece, int64_t* plan) {
  if (!plan) return fail(VDSL_ERR_INVALID_ARG, "plan is null");
  Plan p;
  VDSL_TRY(make_plan(n, vocab, dim, piece, true, p));
  const int64_t values[7] = {p.pieces, p.piece, vocab - (p.pieces - 1) * p.piece, p.grads, p.splits, p.last_splits, p.dw_splits};
  std::copy(values, values + 7, plan);
  return VDSL_OK;
}

extern "C" int vdsl_op_linear_xent_fwd(vdsl_queue q, int64_t n, int64_t dim, int64_t vocab, vdsl_buffer x, vdsl_buffer w,
                                       vdsl_buffer labels, vdsl_buffer loss, vdsl_buffer row_loss, vdsl_buffer lse,
                                       vdsl_buffer workspace) {
  return run_xent(q, n, dim, vocab, x, w, labels, 0, loss, row_loss, lse, false, 1.0f, VDSL_F32, nullptr, VDSL_F32, nullptr, workspace);
}

extern "C" int vdsl_op_linear_xent_fwd_bwd(vdsl_queue q, int64_t n, int64_t dim, int64_t vocab, vdsl_buffer x, vdsl_buffer w,
                                           vdsl_buffer labels, int64_t piece, float grad_scale, vdsl_buffer loss, vdsl_buffer row_loss,
                                           vdsl_buffer lse, int32_t dx_dtype, vdsl_buffer dx, int32_t dw_dtype, vdsl_buffer dw,
                                           vdsl_buffer workspace) {
  return run_xent(q, n, dim, vocab, x, w, labels, piece, loss, row_loss, lse, true, grad_scale, dx_dtype, dx, dw_dtype, dw, workspace);
}
