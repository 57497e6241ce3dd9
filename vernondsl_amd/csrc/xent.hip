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
// division by count: the label's entry then lies in [-1, 0), where a rounding is at most 2^-9 of 1.
// Where the vocabulary is one piece that is 6 n vocab dim operations, else up to 8 n vocab dim.

#include <algorithm>
#include <type_traits>

#include "gemm_any.h"
#include "gemm_wide.h"

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

// Butterflies over the 32 lanes that hold a row of an accumulator.
__device__ __forceinline__ float half_max(float v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
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
};

// MODE kLogitStats: stats and zlabel; kLogitCodes: also the codes; kLogitGrad: G from lse.
template <class Cfg, int MODE>
__device__ __forceinline__ void logits_epilogue(const LogitArgs& p, const f32x16 (&acc)[Cfg::FM][Cfg::FN], int m0, int n0) {
  const int lane = threadIdx.x & 63;
  const int wcol = acc_col<Cfg>(n0, 0) - (lane & 31);  // the wave's first column: a group is a wave's columns
  const int group = p.group0 + wcol / Cfg::WTN;
#pragma unroll
  for (int i = 0; i < Cfg::FM; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = acc_row<Cfg>(m0, i, r);
      const bool in = row < p.n;
      const int label = in ? p.labels[row] : -1;
      const bool counts = label >= 0 && label < p.vocab;
      float v[Cfg::FN];
#pragma unroll
      for (int j = 0; j < Cfg::FN; ++j) v[j] = acc_col<Cfg>(n0, j) < p.cols ? acc[i][j][r] * kLog2e : -INFINITY;
      if constexpr (MODE == kLogitGrad) {
        const float lse = in ? p.lse[row] : 0.0f;
#pragma unroll
        for (int j = 0; j < Cfg::FN; ++j) {
          const int col = acc_col<Cfg>(n0, j);
          float g = __builtin_amdgcn_exp2f(v[j] - lse);
          if (p.v0 + col == label) g -= 1.0f;
          if (!counts || col >= p.cols) g = 0.0f;
          if (in && col < p.ldg) p.g[row * p.ldg + col] = f32_to_bf16(g);
        }
      } else {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < Cfg::FN; ++j) top = fmaxf(top, v[j]);
        top = half_max(top);
        const float base = top == -INFINITY ? 0.0f : top;  // a group of -inf only: a sum of 0
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < Cfg::FN; ++j) s += __builtin_amdgcn_exp2f(v[j] - base);
        s = half_sum(s);
        if (in && wcol < p.cols && (lane & 31) == 0) p.stats[static_cast<int64_t>(row) * p.groups + group] = make_float2(top, s);
#pragma unroll
        for (int j = 0; j < Cfg::FN; ++j) {
          const int col = acc_col<Cfg>(n0, j);
          if (counts && col < p.cols && p.v0 + col == label) p.zlabel[row] = v[j];
          if constexpr (MODE == kLogitCodes)
            if (in && col < p.cols) p.g[row * p.ldg + col] = static_cast<uint16_t>(codes_of((base - v[j]) * (1.0f / kCodeOctaves), 0.0f));
        }
      }
    }
}

template <class Cfg, int MODE>
__global__ __launch_bounds__(Cfg::NT) void xent_logits_any(LogitArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[Cfg::LDS_BYTES];
  const int tiles_m = (p.n + Cfg::BM - 1) / Cfg::BM, tiles_n = (p.cols + Cfg::BN - 1) / Cfg::BN;
  int tm, tn;
  tile_coords(xcd_remap(blockIdx.x, gridDim.x), tiles_m, tiles_n, tm, tn);
  f32x16 acc[Cfg::FM][Cfg::FN];
  any_mainloop<Cfg>(p.x, p.w, p.n, p.cols, p.dim, tm * Cfg::BM, tn * Cfg::BN, smem, acc);
  logits_epilogue<Cfg, MODE>(p, acc, tm * Cfg::BM, tn * Cfg::BN);
}

// The same for tiles of gemm_wide.h, the vocabulary as C's rows: a lane has a token's logits of half of 128
// columns, so the token's maximum and sum over them need one exchange with the lane of the other half, and
// 16-byte stores leave the codes or G.  A group is 128 columns.
template <int MODE, bool EDGE>
__device__ __forceinline__ void logits_epilogue_wide(const LogitArgs& p, const f32x16 (&acc)[4][4], int c0, int row0) {
  const int half = (threadIdx.x & 63) >> 5;
  const int group = p.group0 + c0 / 128;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    __builtin_amdgcn_sched_barrier(0);
    const int row = row0 + 32 * j + static_cast<int>(threadIdx.x & 31);
    const bool in = row < p.n;
    const int label = in ? p.labels[row] : -1;
    const bool counts = label >= 0 && label < p.vocab;
    const int at = label - p.v0 - c0;  // among the wave's columns
    const bool here = counts && at >= 0 && at < 128 && at % 8 / 4 == half;
    const bool any_label = __any(here);
    float z[4][16];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        z[i][r] = wide_value(acc[i][j][r]);
        if (EDGE && c0 + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3) >= p.cols) z[i][r] = -INFINITY;
      }
    float base;  // exp2's argument is z log2 e - base
    if constexpr (MODE == kLogitGrad) {
      base = in ? p.lse[row] : 0.0f;
    } else {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, z[i][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * kLog2e;
      base = top == -INFINITY ? 0.0f : top;
      float s[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(z[i][r], kLog2e, -base));
      float sum = (s[0] + s[1]) + (s[2] + s[3]);
      sum += __shfl_xor(sum, 32, 64);
      if (in && half == 0) p.stats[static_cast<int64_t>(row) * p.groups + group] = make_float2(top, sum);
      if (any_label) {
        float zl = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) zl = at == 32 * i + 8 * (r >> 2) + 4 * half + (r & 3) ? z[i][r] : zl;
        if (here) p.zlabel[row] = zl * kLog2e;
      }
    }
    if constexpr (MODE != kLogitStats) {
      uint16_t* const out = p.g + row * p.ldg + c0 + 8 * half;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
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
          if (in && (!EDGE || c0 + 32 * i + 8 * (q + half) < p.ldg)) *reinterpret_cast<u32x4*>(out + 32 * i + 8 * q) = eight;
        }
      }
    }
  }
}

template <int MODE>
__global__ __launch_bounds__(WideCfg::NT, 1) void xent_logits_wide(LogitArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[WideCfg::LDS_BYTES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  wide_gemm<false, false>(p.w, p.x, p.cols, p.n, p.dim, p.dim, p.dim, false, smem, [&](const f32x16 (&acc)[4][4], int m0, int n0) {
    const int c0 = m0 + 128 * (wave >> 1), row0 = n0 + 128 * (wave & 1);  // of the wave
    if (c0 + 128 <= p.cols) logits_epilogue_wide<MODE, false>(p, acc, c0, row0);
    else if (c0 < p.cols) logits_epilogue_wide<MODE, true>(p, acc, c0, row0);
  });
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
  int64_t ldg;
};

// A block per row: lse and the row's loss from the groups' maxima and sums, then G from the codes.  Rows of G
// past n are zeros.
__global__ __launch_bounds__(256) void xent_rows_kernel(RowArgs p) {
  __shared__ float area[2][4];
  const int64_t row = blockIdx.x;
  if (row >= p.n) {
    u32x4* const g = reinterpret_cast<u32x4*>(p.g + row * p.ldg);
    for (int c = 8 * static_cast<int>(threadIdx.x); c < p.ldg; c += 2048) g[c / 8] = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  const float2* const st = p.stats + row * p.groups;
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
  for (int c = 8 * static_cast<int>(threadIdx.x); c < p.ldg; c += 2048) {
    u32x4 two = g[c / 8];
    if (counts) {
      const float below = st[p.group0 + (c < p.cols ? c : p.cols - 1) / p.group_cols].x - lse;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t u = h ? two[k] >> 16 : two[k] & 0xFFFFu;
          const int col = c + 2 * k + h;
          v[h] = u != kCodeZero ? __builtin_amdgcn_exp2f(__builtin_fmaf(static_cast<float>(u), -kCodeOctaves / 65535.0f, below)) : 0.0f;
          if (!(lse == lse)) v[h] = lse;  // NaN in the row: in all of its gradient
          if (p.v0 + col == label) v[h] = __builtin_amdgcn_exp2f(zl - lse) - 1.0f;
          if (col >= p.cols) v[h] = 0.0f;
        }
        two[k] = pack_bf16x2(v[0], v[1]);
      }
    } else {
      two = u32x4{0u, 0u, 0u, 0u};
    }
    g[c / 8] = two;
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
}

__global__ __launch_bounds__(256) void xent_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) p[i] = 0;
}

struct GradArgs {
  const uint16_t *a, *b;
  int m, n, k;
  int64_t lda, ldb;    // negative: dense
  float* sum;          // [m][n] f32, the pieces' sum; null: this product is all of it
  bool first, last;    // of the pieces: sum holds nothing yet; the result is whole
  const float* inv;    // the factor of the result
  void* out;           // [m][n] of out_dt
  int out_dt;
};

template <class Cfg>
__device__ __forceinline__ void grad_epilogue(const GradArgs& p, const f32x16 (&acc)[Cfg::FM][Cfg::FN], int m0, int n0) {
  const float inv = p.inv[0];
#pragma unroll
  for (int i = 0; i < Cfg::FM; ++i)
#pragma unroll
    for (int j = 0; j < Cfg::FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = acc_row<Cfg>(m0, i, r), col = acc_col<Cfg>(n0, j);
        if (row >= p.m || col >= p.n) continue;
        const int64_t o = static_cast<int64_t>(row) * p.n + col;
        float v = acc[i][j][r];
        if (!p.first) v += p.sum[o];
        if (!p.last) {
          p.sum[o] = v;
        } else {
          v *= inv;
          if (p.out_dt == VDSL_F32) static_cast<float*>(p.out)[o] = v;
          else static_cast<uint16_t*>(p.out)[o] = f32_to_bf16(v);
        }
      }
}

template <class Cfg>
__global__ __launch_bounds__(Cfg::NT) void xent_grad_any(GradArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[Cfg::LDS_BYTES];
  const int tiles_m = (p.m + Cfg::BM - 1) / Cfg::BM, tiles_n = (p.n + Cfg::BN - 1) / Cfg::BN;
  int tm, tn;
  tile_coords(xcd_remap(blockIdx.x, gridDim.x), tiles_m, tiles_n, tm, tn);
  f32x16 acc[Cfg::FM][Cfg::FN];
  any_mainloop<Cfg>(p.a, p.b, p.m, p.n, p.k, tm * Cfg::BM, tn * Cfg::BN, smem, acc, p.lda, p.ldb);
  grad_epilogue<Cfg>(p, acc, tm * Cfg::BM, tn * Cfg::BN);
}

// The gradients' products on tiles of gemm_wide.h: out[n][m] from A(m, k) and B(n, k), so that a lane has
// neighbouring elements of a row of out.
struct WideGradArgs {
  const uint16_t *a, *b;
  int m, n, k;         // m, n: of out
  int n_alloc;         // of B, where it is K-major: columns that are allocated
  int64_t lda, ldb;
  float* sum;          // as GradArgs, [n][m]
  bool first, last;
  const float* inv;
  void* out;
  int out_dt;
};

// WHOLE: the product is all of the sum, rounded to bf16; otherwise any of the forms.
template <bool BKM, bool WHOLE>
__global__ __launch_bounds__(WideCfg::NT, 1) void xent_grad_wide(WideGradArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[WideCfg::LDS_BYTES];
  const int half = (threadIdx.x & 63) >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inv = p.inv[0];
  wide_gemm<true, BKM>(p.a, p.b, p.m, BKM ? p.n_alloc : p.n, p.k, p.lda, p.ldb, BKM, smem, [&](const f32x16 (&acc)[4][4], int m0, int n0) {
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
            if (row < p.n && c0 + c < p.m) *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.out) + out + c) = eight;
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c = 32 * i + 8 * q + 4 * half;
            if (row >= p.n || c0 + c >= p.m) continue;
            f32x4 s = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            if (!p.first) s += *reinterpret_cast<const f32x4*>(p.sum + out + c);
            if (!p.last)
              *reinterpret_cast<f32x4*>(p.sum + out + c) = s;
            else if (p.out_dt == VDSL_F32)
              *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + out + c) = s * inv;
            else
              *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + out + c) =
                  make_uint2(pack_bf16x2(s[0] * inv, s[1] * inv), pack_bf16x2(s[2] * inv, s[3] * inv));
          }
        }
      }
    }
  });
}

// ---- host ----------------------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether a product takes tiles of 128 x 128 or of 64 x 64.
bool big_tiles(int64_t m, int64_t n) { return ceil_div(m, 64) * ceil_div(n, 64) >= 1024; }

// Whether the products take gemm_wide.h's tiles: whole stages of dim, offsets of 256 rows that fit 32 bits, and
// tiles for the card's 256 CUs.
bool wide_runs(int64_t n, int64_t cols, int64_t dim) {
  return dim % 64 == 0 && dim < (1 << 22) && cols < (1 << 22) && ceil_div(n, 256) * ceil_div(cols, 256) >= 192;
}

// How a call is laid out: the pieces and the workspace.
struct Plan {
  int64_t piece = 0, pieces = 0;      // columns of a piece (the last may have fewer)
  bool wide = false;                  // gemm_wide.h's tiles, else gemm_any.h's
  int64_t group_cols = 0, groups = 0;
  int64_t g_rows = 0;                 // rows of G, those past n zeros
  int64_t ldg = 0;
  size_t stats = 0, zlabel = 0, lse = 0, row_loss = 0, inv = 0, g = 0, sum = 0, bytes = 0;
};

constexpr int64_t kPieceBytes = int64_t{1} << 30;  // of codes, where the caller leaves the piece to the library

int make_plan(int64_t n, int64_t vocab, int64_t dim, int64_t piece, bool backward, Plan& p) {
  if (n < 0 || vocab < 0 || dim < 0 || piece < 0) return fail(VDSL_ERR_INVALID_ARG, "linear_xent: negative extent");
  if (vocab == 0) return fail(VDSL_ERR_INVALID_ARG, "linear_xent: the vocabulary is empty");
  if (dim < 8) return fail(VDSL_ERR_UNSUPPORTED, "linear_xent: dim must be at least 8");
  if (n > 0x7fffff00 || vocab > 0x7fffff00 || dim > 0x3fffff00) return fail(VDSL_ERR_UNSUPPORTED, "linear_xent: extents too large");
  if (!backward) piece = vocab;
  else if (piece == 0) piece = std::max<int64_t>(256, kPieceBytes / 2 / std::max<int64_t>(n, 1));
  p.pieces = ceil_div(vocab, std::min(vocab, ceil_div(piece, 256) * 256));
  p.piece = p.pieces == 1 ? vocab : ceil_div(ceil_div(vocab, p.pieces), 256) * 256;
  p.pieces = ceil_div(vocab, p.piece);
  p.wide = wide_runs(n, p.piece, dim);
  p.group_cols = p.wide ? 128 : big_tiles(n, p.piece) ? 64 : 32;
  p.groups = (p.pieces - 1) * ceil_div(p.piece, p.group_cols) + ceil_div(vocab - (p.pieces - 1) * p.piece, p.group_cols);
  p.ldg = ceil_div(p.piece, p.wide ? 256 : 8) * (p.wide ? 256 : 8);
  p.g_rows = p.wide ? ceil_div(n, 64) * 64 : n;
  size_t at = 0;
  bool fits = true;
  const auto take = [&](int64_t a, int64_t b) {
    const size_t from = at, size = nbytes(a, b);
    if (size == kSizeOverflow || __builtin_add_overflow(at, size, &at) || at > kSizeOverflow - 512) fits = false;
    else at = (at + 255) / 256 * 256;
    return from;
  };
  p.stats = take(n, p.groups * 8);
  p.zlabel = take(n, 4);
  p.lse = take(n, 4);
  p.row_loss = take(n, 4);
  p.inv = take(1, 4);
  if (backward) {
    p.g = take(p.g_rows, p.ldg * 2);
    if (p.pieces > 1) p.sum = take(n, dim * 4);
  }
  p.bytes = at;
  return fits ? VDSL_OK : fail(VDSL_ERR_SHAPE, "linear_xent: the workspace's size overflows");
}

template <class Go>
int with_tiles(int64_t m, int64_t n, bool big, const char* name, Go&& go) {
  const int64_t b = big ? 128 : 64, tiles = ceil_div(m, b) * ceil_div(n, b);
  if (tiles > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, std::string(name) + ": too many tiles");
  go(static_cast<unsigned>(tiles));
  return check_launch(name);
}

template <int MODE>
int launch_logits(const LogitArgs& a, const Plan& plan, hipStream_t s) {
  if (plan.wide) {
    const unsigned blocks = wide_blocks(ceil_div(a.n, 256) * ceil_div(a.cols, 256));
    hipLaunchKernelGGL(xent_logits_wide<MODE>, dim3(blocks), dim3(WideCfg::NT), 0, s, a);
    return check_launch("xent_logits_wide");
  }
  const bool big = plan.group_cols == 64;
  using Big = AnyConfig<128, 128, 2, 2, false, false>;
  using Small = AnyConfig<64, 64, 2, 2, false, false>;
  return with_tiles(a.n, a.cols, big, "xent_logits_any", [&](unsigned tiles) {
    if (big) hipLaunchKernelGGL((xent_logits_any<Big, MODE>), dim3(tiles), dim3(Big::NT), 0, s, a);
    else hipLaunchKernelGGL((xent_logits_any<Small, MODE>), dim3(tiles), dim3(Small::NT), 0, s, a);
  });
}

template <bool AKM, bool BKM>
int launch_grad(const GradArgs& a, hipStream_t s) {
  using Big = AnyConfig<128, 128, 2, 2, AKM, BKM>;
  using Small = AnyConfig<64, 64, 2, 2, AKM, BKM>;
  const bool big = big_tiles(a.m, a.n);
  return with_tiles(a.m, a.n, big, "xent_grad_any", [&](unsigned tiles) {
    if (big) hipLaunchKernelGGL(xent_grad_any<Big>, dim3(tiles), dim3(Big::NT), 0, s, a);
    else hipLaunchKernelGGL(xent_grad_any<Small>, dim3(tiles), dim3(Small::NT), 0, s, a);
  });
}

template <bool BKM>
int launch_grad_wide(const WideGradArgs& a, int64_t n, hipStream_t s) {
  const unsigned blocks = wide_blocks(ceil_div(a.m, 256) * ceil_div(n, 256));
  if (a.first && a.last && a.out_dt == VDSL_BF16)
    hipLaunchKernelGGL((xent_grad_wide<BKM, true>), dim3(blocks), dim3(WideCfg::NT), 0, s, a);
  else
    hipLaunchKernelGGL((xent_grad_wide<BKM, false>), dim3(blocks), dim3(WideCfg::NT), 0, s, a);
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
    if (dx == x || dx == w || dw == x || dw == w) return fail(VDSL_ERR_INVALID_ARG, "linear_xent_fwd_bwd: a gradient must not overwrite x or w");
  }
  VDSL_TRY(check_buffer(q, workspace, plan.bytes, "workspace", true));
  const hipStream_t s = q->stream;
  char* const ws = static_cast<char*>(workspace->ptr);
  const int32_t* lab = static_cast<const int32_t*>(labels->ptr);
  float* const inv = reinterpret_cast<float*>(ws + plan.inv);
  float* const each = reinterpret_cast<float*>(ws + plan.row_loss);
  uint16_t* const g = backward ? reinterpret_cast<uint16_t*>(ws + plan.g) : nullptr;
  LogitArgs la{};
  la.x = static_cast<const uint16_t*>(x->ptr);
  la.labels = lab;
  la.stats = reinterpret_cast<float2*>(ws + plan.stats);
  la.zlabel = reinterpret_cast<float*>(ws + plan.zlabel);
  la.g = g;
  la.lse = reinterpret_cast<const float*>(ws + plan.lse);
  la.n = static_cast<int>(n);
  la.dim = static_cast<int>(dim);
  la.vocab = static_cast<int>(vocab);
  la.groups = static_cast<int>(plan.groups);
  la.ldg = plan.ldg;
  const auto set_piece = [&](int64_t k) {
    const int64_t v0 = k * plan.piece;
    la.w = static_cast<const uint16_t*>(w->ptr) + v0 * dim;
    la.v0 = static_cast<int>(v0);
    la.cols = static_cast<int>(std::min(plan.piece, vocab - v0));
    la.group0 = static_cast<int>(k * ceil_div(plan.piece, plan.group_cols));
  };
  if (n > 0) {
    for (int64_t k = 0; k < plan.pieces; ++k) {
      set_piece(k);
      if (backward && k == plan.pieces - 1) VDSL_TRY(launch_logits<kLogitCodes>(la, plan, s));
      else VDSL_TRY(launch_logits<kLogitStats>(la, plan, s));
    }
    RowArgs ra{};
    ra.labels = lab;
    ra.stats = la.stats;
    ra.zlabel = la.zlabel;
    ra.lse_octaves = reinterpret_cast<float*>(ws + plan.lse);
    ra.lse = lse ? static_cast<float*>(lse->ptr) : nullptr;
    ra.row_loss = each;
    ra.row_loss_out = row_loss ? static_cast<float*>(row_loss->ptr) : nullptr;
    ra.g = g;
    ra.n = la.n;
    ra.cols = la.cols;
    ra.vocab = la.vocab;
    ra.v0 = la.v0;
    ra.group0 = la.group0;
    ra.groups = la.groups;
    ra.group_cols = static_cast<int>(plan.group_cols);
    ra.ldg = plan.ldg;
    hipLaunchKernelGGL(xent_rows_kernel, dim3(static_cast<unsigned>(backward ? plan.g_rows : n)), dim3(256), 0, s, ra);
    VDSL_TRY(check_launch("xent_rows_kernel"));
  }
  hipLaunchKernelGGL(xent_mean_kernel, dim3(1), dim3(1024), 0, s, each, lab, n, static_cast<int>(vocab), grad_scale,
                     static_cast<float*>(loss->ptr), inv);
  VDSL_TRY(check_launch("xent_mean_kernel"));
  if (!backward) return VDSL_OK;
  if (n == 0) {
    hipLaunchKernelGGL(xent_zero_kernel, dim3(2048), dim3(256), 0, s, static_cast<uint16_t*>(dw->ptr),
                       vocab * dim * static_cast<int64_t>(dtype_size(dw_dtype) / 2));
    return check_launch("xent_zero_kernel");
  }
  // The piece whose codes are held comes first, then those whose logits are formed again.
  for (int64_t t = 0; t < plan.pieces; ++t) {
    const int64_t k = plan.pieces - 1 - t;
    set_piece(k);
    if (t > 0) VDSL_TRY(launch_logits<kLogitGrad>(la, plan, s));
    float* const sum = plan.pieces > 1 ? reinterpret_cast<float*>(ws + plan.sum) : nullptr;
    void* const dw_piece = static_cast<char*>(dw->ptr) + static_cast<int64_t>(la.v0) * dim * static_cast<int64_t>(dtype_size(dw_dtype));
    if (plan.wide) {
      // dx^T = w^T G^T over the piece, dw^T = x^T G
      WideGradArgs x_args{la.w, g,        la.dim, la.n,        la.cols, 0,       dim,       plan.ldg, sum,
                          t == 0, t == plan.pieces - 1, inv, dx->ptr, dx_dtype};
      VDSL_TRY(launch_grad_wide<false>(x_args, n, s));
      WideGradArgs w_args{la.x, g, la.dim, la.cols, la.n, static_cast<int>(plan.ldg), dim, plan.ldg, nullptr, true, true, inv,
                          dw_piece, dw_dtype};
      VDSL_TRY(launch_grad_wide<true>(w_args, plan.ldg, s));
      continue;
    }
    GradArgs ga{};
    ga.inv = inv;
    ga.a = g;  // dx += G w
    ga.lda = plan.ldg;
    ga.b = la.w;
    ga.ldb = -1;
    ga.m = la.n;
    ga.n = la.dim;
    ga.k = la.cols;
    ga.first = t == 0;
    ga.last = t == plan.pieces - 1;
    ga.sum = sum;
    ga.out = dx->ptr;
    ga.out_dt = dx_dtype;
    VDSL_TRY((launch_grad<false, true>(ga, s)));
    ga.a = g;  // dw of the piece = G^T x
    ga.lda = plan.ldg;
    ga.b = la.x;
    ga.ldb = -1;
    ga.m = la.cols;
    ga.n = la.dim;
    ga.k = la.n;
    ga.first = ga.last = true;
    ga.sum = nullptr;
    ga.out = dw_piece;
    ga.out_dt = dw_dtype;
    VDSL_TRY((launch_grad<true, true>(ga, s)));
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
