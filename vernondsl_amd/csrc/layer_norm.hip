// Layer norm over the rows of a [rows][cols] tensor, and its backward pass with the reductions of the
// gain's and the offset's gradients.
//
//   mean = sum_j x_j / cols,  rstd = 1 / sqrt(sum_j (x_j - mean)^2 / cols + eps),  h_j = (x_j - mean) rstd,
//   y_j = h_j gamma_j + beta_j;
//   with g_j = dy_j gamma_j:  dx_j = rstd (g_j - mean(g) - h_j mean(g h)),
//   dgamma_j = sum over rows of dy_j h_j,  dbeta_j = sum over rows of dy_j.
//
// All of it in f32, the outputs rounded once to their types.  Both passes are bound by HBM: x (and dy) are
// read once and held in registers as units of U consecutive elements, y (dx) is written once: 16384 x 4096 f32 to
// bf16 70 us (5.8 TB/s), bf16 to bf16 42 (6.4); the backward pass in bf16 78 (5.2, 4.9 of it the second kernel);
// 300 x 1001 in f32, backward, 6.  A wave
// holds a row of up to 1024 columns, 256 lanes one of up to 4096, 1024 lanes one of up to 16384.  Wider rows have no
// place in a block's registers (1024 lanes have 128 each, and a row takes 16 and more for x, as many for the next row,
// gamma and beta), so they are read again for each step: 4096 x 16500 in bf16 103 us where 16384 columns take 49, the
// backward pass with all gradients 274.  A block walks over rows and loads the next
// row before it works on the present one, so gamma, beta and, in the backward pass, the sums for dgamma
// and dbeta stay in its lanes' registers.  Those sums go to a workspace, one row of it per block, and a
// second kernel adds the blocks' rows in a fixed order: no atomics, the same bits every time.  Of few rows,
// other blocks of the same launch form them.

#include <algorithm>
#include <type_traits>

#include "rowunit.h"

namespace vdsl {
namespace {

// Sum of v over the TPR lanes that share a row.  Lanes of several waves meet in LDS; `parity` selects
// one of two areas so that one barrier a call is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], int parity) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum_rows(v[k]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    __shared__ float part[2][K][W];
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) part[parity][k][threadIdx.x >> 6] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += part[parity][k][w];
      v[k] = s;
    }
  }
}

// The largest number of columns that TPR lanes hold in NV units of U elements each.
template <int TPR, int U, int NV>
struct RowShape {
  static constexpr int kLanes = TPR, kUnit = U, kUnits = NV;
  static constexpr int kRows = TPR < 256 ? 256 / TPR : 1;       // rows a block holds at a time
  static constexpr int kThreads = TPR < 256 ? 256 : TPR;
  static constexpr int64_t kCols = int64_t{TPR} * U * NV;
};

// gamma or beta for this lane's columns; `none` where there is none.
template <class S>
__device__ __forceinline__ void load_params(const void* __restrict__ p, int dt, int64_t cols, int t, float none,
                                            float (&v)[S::kUnits][S::kUnit]) {
#pragma unroll
  for (int k = 0; k < S::kUnits; ++k) {
    const UnitAt<S::kUnit> at((int64_t{k} * S::kLanes + t) * S::kUnit, cols);
    if (p && dt == VDSL_F32) {
      load_whole<VDSL_F32, S::kUnit>(p, at.c, v[k]);
    } else if (p) {
      load_whole<VDSL_BF16, S::kUnit>(p, at.c, v[k]);
    } else {
#pragma unroll
      for (int j = 0; j < S::kUnit; ++j) v[k][j] = none;
    }
  }
}

template <class S, int DT>
__device__ __forceinline__ void load_row(const void* __restrict__ p, int64_t row, int64_t cols, int t,
                                         float (&v)[S::kUnits][S::kUnit]) {
#pragma unroll
  for (int k = 0; k < S::kUnits; ++k) {
    const UnitAt<S::kUnit> at((int64_t{k} * S::kLanes + t) * S::kUnit, cols);
    load_whole<DT, S::kUnit>(p, row * cols + at.c, v[k]);
  }
}

template <class S, int XT, bool STREAM>
__global__ __launch_bounds__(S::kThreads) void layer_norm_fwd_rows(const void* x, const void* __restrict__ gamma,
                                                                   const void* __restrict__ beta, int param_dt, void* y, int y_dt,
                                                                   float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                                   int64_t rows, int64_t cols, float eps) {
  constexpr int U = S::kUnit, NV = S::kUnits;
  const int t = threadIdx.x % S::kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * S::kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * S::kRows + threadIdx.x / S::kLanes;
  if (S::kRows > 1 && row >= rows) return;  // a wave of its own: no barrier is ahead
  float ga[NV][U], be[NV][U], next[NV][U];
  load_row<S, XT>(x, row, cols, t, next);
  load_params<S>(gamma, param_dt, cols, t, 1.0f, ga);
  load_params<S>(beta, param_dt, cols, t, 0.0f, be);
  const float inv_cols = 1.0f / static_cast<float>(cols);
  for (; row < rows; row += step) {
    float v[NV][U];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < U; ++j) v[k][j] = next[k][j];
    if (row + step < rows) load_row<S, XT>(x, row + step, cols, t, next);
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const UnitAt<U> at((int64_t{k} * S::kLanes + t) * U, cols);
#pragma unroll
      for (int j = 0; j < U; ++j) s[0] += j >= at.skip ? v[k][j] : 0.0f;
    }
    row_sums<S::kLanes>(s, 0);
    const float mean = s[0] * inv_cols;
    // the sum of squares about the mean: no cancellation, however large the mean
    float q[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const UnitAt<U> at((int64_t{k} * S::kLanes + t) * U, cols);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        v[k][j] -= mean;
        q[0] += j >= at.skip ? v[k][j] * v[k][j] : 0.0f;
      }
    }
    row_sums<S::kLanes>(q, 1);
    const float rstd = 1.0f / sqrtf(q[0] * inv_cols + eps);
    if (t == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const UnitAt<U> at((int64_t{k} * S::kLanes + t) * U, cols);
      float o[U];
#pragma unroll
      for (int j = 0; j < U; ++j) o[j] = v[k][j] * rstd * ga[k][j] + be[k][j];
      if (at.any()) store_unit<U, STREAM>(y_dt, y, row * cols + at.c, o);
    }
  }
}

// Rows wider than any RowShape: a block per row, which reads it for the mean, for the variance and to
// write y.
__global__ __launch_bounds__(1024) void layer_norm_fwd_stream(const void* x, int x_dt, const void* __restrict__ gamma,
                                                              const void* __restrict__ beta, int param_dt, void* y, int y_dt,
                                                              float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                              int64_t rows, int64_t cols, float eps) {
  const int64_t row = block_index(), base = row * cols;
  if (row >= rows) return;
  float s[1] = {0.0f};
  for (int64_t c = 4 * threadIdx.x; c < cols; c += 4096) {
    float v[4];
    load_some(x_dt, x, base + c, cols - c, v);
    s[0] += (v[0] + v[1]) + (v[2] + v[3]);
  }
  row_sums<1024>(s, 0);
  const float inv_cols = 1.0f / static_cast<float>(cols), mean = s[0] * inv_cols;
  float q[1] = {0.0f};
  for (int64_t c = 4 * threadIdx.x; c < cols; c += 4096) {
    float v[4];
    load_some(x_dt, x, base + c, cols - c, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = c + j < cols ? v[j] - mean : 0.0f;
      q[0] += d * d;
    }
  }
  row_sums<1024>(q, 1);
  const float rstd = 1.0f / sqrtf(q[0] * inv_cols + eps);
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[row] = mean;
    if (rstd_out) rstd_out[row] = rstd;
  }
  for (int64_t c = 4 * threadIdx.x; c < cols; c += 4096) {
    float v[4], ga[4] = {1.0f, 1.0f, 1.0f, 1.0f}, be[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    load_some(x_dt, x, base + c, cols - c, v);
    if (gamma) load_some(param_dt, gamma, c, cols - c, ga);
    if (beta) load_some(param_dt, beta, c, cols - c, be);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (v[j] - mean) * rstd * ga[j] + be[j];
    store_some(y_dt, y, base + c, cols - c, v);
  }
}

// dgamma and dbeta of 16 columns from c0 on by one block: a sixteenth of its lanes to a column, their shares of the rows
// added in f64 in order.
template <int THREADS, int XT, int DYT>
__device__ __forceinline__ void column_sums(const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ mean,
                                            const float* __restrict__ rstd, int64_t rows, int64_t cols, int64_t c0,
                                            float* __restrict__ dgamma, float* __restrict__ dbeta) {
  constexpr int SLOTS = THREADS / 16;
  __shared__ float part[SLOTS][2][16];
  const int column = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const int64_t c = c0 + column < cols ? c0 + column : cols - 1;
  float g = 0.0f, b = 0.0f;
#pragma unroll 8
  for (int64_t row = slot; row < rows; row += SLOTS) {
    const float d = load_elem<DYT>(dy, row * cols + c), h = (load_elem<XT>(x, row * cols + c) - mean[row]) * rstd[row];
    g += d * h;
    b += d;
  }
  part[slot][0][column] = g;
  part[slot][1][column] = b;
  __syncthreads();
  if (threadIdx.x >= 32 || c0 + column >= cols) return;
  double s = 0.0;
#pragma unroll 8
  for (int k = 0; k < SLOTS; ++k) s += part[k][slot][column];
  float* const out = slot ? dbeta : dgamma;
  if (out) out[c] = static_cast<float>(s);
}

// partials: [row_blocks][2][cols], a block's sums for dgamma and dbeta over its rows (waves of one block
// that hold rows of their own meet in LDS, in the order of the waves); null where neither is wanted.  FEW: no partials, but
// blocks past row_blocks that form dgamma and dbeta.
template <class S, int XT, int DYT, bool STREAM, bool FEW>
__global__ __launch_bounds__(S::kThreads) void layer_norm_bwd_rows(const void* dy, const void* __restrict__ x,
                                                                   const void* __restrict__ gamma, int param_dt,
                                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                   void* dx, int dx_dt, float* __restrict__ partials, int64_t rows,
                                                                   int64_t cols, int row_blocks, float* __restrict__ dgamma,
                                                                   float* __restrict__ dbeta) {
  if constexpr (FEW) {
    if (static_cast<int>(blockIdx.x) >= row_blocks) {
      const int64_t c0 = int64_t{16} * (static_cast<int>(blockIdx.x) - row_blocks);
      column_sums<S::kThreads, XT, DYT>(dy, x, mean, rstd, rows, cols, c0, dgamma, dbeta);
      return;
    }
  }
  constexpr int U = S::kUnit, NV = S::kUnits;
  const int t = threadIdx.x % S::kLanes, slot = threadIdx.x / S::kLanes;
  const int64_t step = static_cast<int64_t>(row_blocks) * S::kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * S::kRows + slot;
  constexpr bool AHEAD = NV * U * S::kThreads < 16384;  // 1024 lanes of 16 columns have no registers for another row, or gamma
  float ga[NV][U], dg[NV][U], db[NV][U], nx[NV][U], ny[NV][U];
  float nmean = 0.0f, nrstd = 0.0f;
  const auto load = [&](int64_t at) {
    load_row<S, XT>(x, at, cols, t, nx);
    load_row<S, DYT>(dy, at, cols, t, ny);
    nmean = mean[at];
    nrstd = rstd[at];
  };
  if (AHEAD && row < rows) load(row);
  if (AHEAD) load_params<S>(gamma, param_dt, cols, t, 1.0f, ga);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < U; ++j) dg[k][j] = db[k][j] = 0.0f;
  const float inv_cols = 1.0f / static_cast<float>(cols);
  int parity = 0;
  for (; row < rows; row += step) {
    if (!AHEAD) {
      asm volatile("" ::: "memory");  // gamma again for each row, not kept through the loop
      load(row);
      load_params<S>(gamma, param_dt, cols, t, 1.0f, ga);
    }
    float h[NV][U], d[NV][U];
    const float r = nrstd;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        h[k][j] = (nx[k][j] - nmean) * r;
        d[k][j] = ny[k][j];
      }
    }
    if (AHEAD && row + step < rows) load(row + step);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const UnitAt<U> at((int64_t{k} * S::kLanes + t) * U, cols);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (!FEW) {
          dg[k][j] += d[k][j] * h[k][j];
          db[k][j] += d[k][j];
        }
        d[k][j] *= ga[k][j];
        s[0] += j >= at.skip ? d[k][j] : 0.0f;
        s[1] += j >= at.skip ? d[k][j] * h[k][j] : 0.0f;
      }
    }
    row_sums<S::kLanes>(s, parity);
    parity ^= 1;
    const float m1 = s[0] * inv_cols, m2 = s[1] * inv_cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const UnitAt<U> at((int64_t{k} * S::kLanes + t) * U, cols);
      float o[U];
#pragma unroll
      for (int j = 0; j < U; ++j) o[j] = r * ((d[k][j] - m1) - h[k][j] * m2);
      if (at.any()) store_unit<U, STREAM>(dx_dt, dx, row * cols + at.c, o);
    }
  }
  if (FEW || !partials) return;
  if constexpr (S::kRows > 1) {
    __shared__ float sums[S::kRows - 1][2][S::kCols];
    if (slot > 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < U; ++j) {
          sums[slot - 1][0][(k * U + j) * S::kLanes + t] = dg[k][j];
          sums[slot - 1][1][(k * U + j) * S::kLanes + t] = db[k][j];
        }
    }
    __syncthreads();
    if (slot > 0) return;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int w = 0; w < S::kRows - 1; ++w) {
          dg[k][j] += sums[w][0][(k * U + j) * S::kLanes + t];
          db[k][j] += sums[w][1][(k * U + j) * S::kLanes + t];
        }
  }
  float* const out = partials + static_cast<int64_t>(blockIdx.x) * 2 * cols;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const UnitAt<U> at((int64_t{k} * S::kLanes + t) * U, cols);
    if (!at.any()) continue;
    store_whole<VDSL_F32, U>(out, at.c, dg[k]);
    store_whole<VDSL_F32, U>(out, cols + at.c, db[k]);
  }
}

__global__ __launch_bounds__(1024) void layer_norm_bwd_stream(const void* dy, int dy_dt, const void* __restrict__ x, int x_dt,
                                                              const void* __restrict__ gamma, int param_dt,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              void* dx, int dx_dt, int64_t rows, int64_t cols) {
  const int64_t row = block_index(), base = row * cols;
  if (row >= rows) return;
  const float m = mean[row], r = rstd[row];
  float s[2] = {0.0f, 0.0f};
  float m1 = 0.0f, m2 = 0.0f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t c = 4 * threadIdx.x; c < cols; c += 4096) {
      float h[4], d[4], ga[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      load_some(x_dt, x, base + c, cols - c, h);
      load_some(dy_dt, dy, base + c, cols - c, d);
      if (gamma) load_some(param_dt, gamma, c, cols - c, ga);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = c + j < cols ? (h[j] - m) * r : 0.0f;
        d[j] *= ga[j];
        s[0] += d[j];
        s[1] += d[j] * h[j];
        h[j] = r * ((d[j] - m1) - h[j] * m2);
      }
      if (pass) store_some(dx_dt, dx, base + c, cols - c, h);
    }
    if (pass) return;
    row_sums<1024>(s, 0);
    m1 = s[0] / static_cast<float>(cols);
    m2 = s[1] / static_cast<float>(cols);
  }
}

// The sums for dgamma and dbeta of such rows: block (x, y) takes 1024 columns and every gridDim.y-th row.  The wider the
// rows, the fewer blocks share them (from 2^18 columns on one takes all), so f32 sums of 64 rows are added up in f64
// (at the speed of one f32 sum: 16384 x 20000 in bf16 1311 us and 1294, 512 x 300000 882 and 869).
// Runs before layer_norm_bwd_stream, which may overwrite dy.
__global__ __launch_bounds__(256) void layer_norm_bwd_columns(const void* __restrict__ dy, int dy_dt, const void* __restrict__ x,
                                                              int x_dt, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, float* __restrict__ partials,
                                                              int64_t rows, int64_t cols) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 1024 + 4 * threadIdx.x;
  if (c >= cols) return;
  double gs[4] = {0.0, 0.0, 0.0, 0.0}, bs[4] = {0.0, 0.0, 0.0, 0.0};
  for (int64_t row = blockIdx.y; row < rows;) {
    float dg[4] = {0.0f, 0.0f, 0.0f, 0.0f}, db[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < 64 && row < rows; ++k, row += gridDim.y) {
      float h[4], d[4];
      load_some(x_dt, x, row * cols + c, cols - c, h);
      load_some(dy_dt, dy, row * cols + c, cols - c, d);
      const float m = mean[row], r = rstd[row];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dg[j] += d[j] * ((h[j] - m) * r);
        db[j] += d[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      gs[j] += dg[j];
      bs[j] += db[j];
    }
  }
  float dg[4], db[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    dg[j] = static_cast<float>(gs[j]);
    db[j] = static_cast<float>(bs[j]);
  }
  float* const out = partials + static_cast<int64_t>(blockIdx.y) * 2 * cols;
  store_some(VDSL_F32, out, c, cols - c, dg);
  store_some(VDSL_F32, out, cols + c, cols - c, db);
}

// dgamma and dbeta: the column sums of the n partial rows, each wave of a block a share of them, added in
// f64 in the order of the rows and then of the waves.  Column i of the [2 cols] of a partial row is
// dgamma's i-th or dbeta's (i - cols)-th.
__global__ __launch_bounds__(1024) void layer_norm_bwd_finish(const float* __restrict__ partials, int64_t n, int64_t cols,
                                                              float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ double part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = block_index() * 64 + lane;
  double s = 0.0;
  if (i < 2 * cols) {
#pragma unroll 8
    for (int64_t b = wave; b < n; b += 16) s += partials[b * 2 * cols + i];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || i >= 2 * cols) return;
  s = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += part[w][lane];
  if (i < cols) {
    if (dgamma) dgamma[i] = static_cast<float>(s);
  } else if (dbeta) {
    dbeta[i - cols] = static_cast<float>(s);
  }
}

// Calls go(RowShape) for rows of `cols` columns in units of U, or wide() where no shape holds one.
template <int U, class Go, class Wide>
int row_shape(int64_t cols, Go&& go, Wide&& wide) {
  if (cols < U) return go(RowShape<64, 1, 1>{});
  if (cols <= 64 * U) return go(RowShape<64, U, 1>{});
  if (cols <= 512) return go(RowShape<64, U, 512 / 64 / U>{});
  if (cols <= 1024) return go(RowShape<64, U, 1024 / 64 / U>{});
  if (cols <= 2048) return go(RowShape<256, U, 2048 / 256 / U>{});
  if (cols <= 4096) return go(RowShape<256, U, 4096 / 256 / U>{});
  if (cols <= 8192) return go(RowShape<1024, U, 8192 / 1024 / U>{});
  if (cols <= 16384) return go(RowShape<1024, U, 16384 / 1024 / U>{});
  return wide();
}

// Whether dgamma and dbeta are formed by blocks of their own of the one launch, which read x and dy again, instead of by
// way of partial rows and a second launch.  Us so and by partial rows, bf16: 8 x 4096 5.9, 8.6; 300 x 1001 5.8, 8.1; 1000 x
// 1024 5.9, 9.5; 256 x 8192 11.6, 15.0; 512 x 4096 7.6, 12.4; 1000 x 4096 18.6, 14.6; 512 x 16384 36.4, 23.8.
bool few_rows(int64_t rows, int64_t cols) { return rows <= 1024 && cols <= 16384 && rows * cols <= int64_t{1} << 21; }

// Blocks of the backward pass, each of which leaves a partial row: so many that a CU has 24 to 48 KiB of rows on their
// way (us of 256, 512 and 1024, rows of bf16: 65536 x 256 51.2, 35.5, 29.4; 32768 x 2048 168, 107, 81.5;
// 16384 x 4096 113, 78.0, 94.2; 8192 x 8192 86.1, 90.9, 101; of f32: 16384 x 4096 147, 161, 164; x of f32 and dy of
// bf16: 16384 x 4096 129, 102), but of four rows
// or more where there are more than 256 (2048 x 2048, bf16, in 1024 and in 512 blocks 18.8, 14.3; 512 x 8192 in 512 and
// in 256 22.7, 17.6).
// together: the rows a block holds at a time; bytes: of a row of x and one of dy.
int64_t bwd_blocks(int64_t rows, int64_t together, int64_t bytes) {
  const int64_t most = together * bytes <= 8192 ? 1024 : together * bytes <= 24576 ? 512 : 256;
  const int64_t blocks = (rows + together - 1) / together;
  return blocks <= 256 ? blocks : std::min(most, std::max<int64_t>(256, blocks / 4));
}
int64_t bwd_most_blocks(int64_t rows, int64_t cols) { return bwd_blocks(rows, cols <= 1024 ? 4 : 1, 4 * std::min<int64_t>(cols, 1 << 24)); }

bool float_type(int32_t t) { return t == VDSL_F32 || t == VDSL_BF16; }

}  // namespace
}  // namespace vdsl

using namespace vdsl;

extern "C" int vdsl_op_layer_norm_fwd(vdsl_queue q, int64_t rows, int64_t cols, int32_t x_dtype, vdsl_buffer x,
                                      int32_t param_dtype, vdsl_buffer gamma, vdsl_buffer beta, float eps, int32_t y_dtype,
                                      vdsl_buffer y, vdsl_buffer mean, vdsl_buffer rstd) {
  VDSL_TRY(enter_queue(q));
  if (rows < 0 || cols < 0) return fail(VDSL_ERR_INVALID_ARG, "negative shape");
  if (!(eps >= 0.0f)) return fail(VDSL_ERR_INVALID_ARG, "layer_norm: eps must not be negative");
  if (!float_type(x_dtype) || !float_type(param_dtype) || !float_type(y_dtype))
    return fail(VDSL_ERR_UNSUPPORTED, "layer_norm_fwd supports f32 and bf16");
  VDSL_TRY(check_buffer(q, x, nbytes(rows, cols, dtype_size(x_dtype)), "x", false));
  if (gamma) VDSL_TRY(check_buffer(q, gamma, nbytes(cols, dtype_size(param_dtype)), "gamma", false));
  if (beta) VDSL_TRY(check_buffer(q, beta, nbytes(cols, dtype_size(param_dtype)), "beta", false));
  VDSL_TRY(check_buffer(q, y, nbytes(rows, cols, dtype_size(y_dtype)), "y", true));
  if (mean) VDSL_TRY(check_buffer(q, mean, nbytes(rows, 4), "mean", true));
  if (rstd) VDSL_TRY(check_buffer(q, rstd, nbytes(rows, 4), "rstd", true));
  if (x == y && x_dtype != y_dtype) return fail(VDSL_ERR_INVALID_ARG, "in-place layer_norm_fwd needs one dtype");
  VDSL_TRY(check_apart("layer_norm_fwd", {y, mean, rstd}, {gamma, beta}));
  VDSL_TRY(check_apart("layer_norm_fwd", {mean, rstd}, {x}));
  if (rows == 0 || cols == 0) return VDSL_OK;
  if (rows > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "layer_norm_fwd: too many rows");
  const void* g = gamma ? gamma->ptr : nullptr;
  const void* b = beta ? beta->ptr : nullptr;
  float* mo = mean ? static_cast<float*>(mean->ptr) : nullptr;
  float* ro = rstd ? static_cast<float*>(rstd->ptr) : nullptr;
  const auto rows_kernel = [&](auto shape, auto xt) {
    using S = decltype(shape);
    constexpr int XT = decltype(xt)::value;
    const int64_t blocks = std::min<int64_t>((rows + S::kRows - 1) / S::kRows, 512 * 2048 / S::kThreads);
    const bool stream = rows * cols * static_cast<int64_t>(dtype_size(y_dtype)) >= kStreamBytes;
    const auto kernel = stream ? layer_norm_fwd_rows<S, XT, true> : layer_norm_fwd_rows<S, XT, false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(S::kThreads), 0, q->stream, x->ptr,
                       g, b, param_dtype, y->ptr, y_dtype, mo, ro, rows, cols, eps);
    return check_launch("layer_norm_fwd_rows");
  };
  const auto wide = [&] {
    hipLaunchKernelGGL(layer_norm_fwd_stream, block_grid(rows), dim3(1024), 0, q->stream, x->ptr, x_dtype, g, b,
                       param_dtype, y->ptr, y_dtype, mo, ro, rows, cols, eps);
    return check_launch("layer_norm_fwd_stream");
  };
  using F = std::integral_constant<int, VDSL_F32>;
  using B = std::integral_constant<int, VDSL_BF16>;
  if (x_dtype == VDSL_F32) return row_shape<4>(cols, [&](auto s) { return rows_kernel(s, F{}); }, wide);
  if (y_dtype == VDSL_F32) return row_shape<4>(cols, [&](auto s) { return rows_kernel(s, B{}); }, wide);
  return row_shape<8>(cols, [&](auto s) { return rows_kernel(s, B{}); }, wide);
}

extern "C" int vdsl_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols, size_t* bytes) {
  if (!bytes) return fail(VDSL_ERR_INVALID_ARG, "bytes is null");
  if (rows < 0 || cols < 0) return fail(VDSL_ERR_INVALID_ARG, "negative shape");
  const size_t n = nbytes(bwd_most_blocks(rows, std::max<int64_t>(cols, 1)), cols, 8);
  if (n == kSizeOverflow) return fail(VDSL_ERR_SHAPE, "layer_norm_bwd workspace size overflows");
  *bytes = n;
  return VDSL_OK;
}

extern "C" int vdsl_op_layer_norm_bwd(vdsl_queue q, int64_t rows, int64_t cols, int32_t dy_dtype, vdsl_buffer dy, int32_t x_dtype,
                                      vdsl_buffer x, int32_t param_dtype, vdsl_buffer gamma, vdsl_buffer mean, vdsl_buffer rstd,
                                      int32_t dx_dtype, vdsl_buffer dx, vdsl_buffer dgamma, vdsl_buffer dbeta,
                                      vdsl_buffer workspace) {
  VDSL_TRY(enter_queue(q));
  if (rows < 0 || cols < 0) return fail(VDSL_ERR_INVALID_ARG, "negative shape");
  if (!float_type(dy_dtype) || !float_type(x_dtype) || !float_type(param_dtype) || !float_type(dx_dtype))
    return fail(VDSL_ERR_UNSUPPORTED, "layer_norm_bwd supports f32 and bf16");
  VDSL_TRY(check_buffer(q, dy, nbytes(rows, cols, dtype_size(dy_dtype)), "dy", false));
  VDSL_TRY(check_buffer(q, x, nbytes(rows, cols, dtype_size(x_dtype)), "x", false));
  if (gamma) VDSL_TRY(check_buffer(q, gamma, nbytes(cols, dtype_size(param_dtype)), "gamma", false));
  VDSL_TRY(check_buffer(q, mean, nbytes(rows, 4), "mean", false));
  VDSL_TRY(check_buffer(q, rstd, nbytes(rows, 4), "rstd", false));
  VDSL_TRY(check_buffer(q, dx, nbytes(rows, cols, dtype_size(dx_dtype)), "dx", true));
  const bool params = dgamma || dbeta;
  if (dgamma) VDSL_TRY(check_buffer(q, dgamma, nbytes(cols, 4), "dgamma", true));
  if (dbeta) VDSL_TRY(check_buffer(q, dbeta, nbytes(cols, 4), "dbeta", true));
  if (dx == dy && dx_dtype != dy_dtype) return fail(VDSL_ERR_INVALID_ARG, "in-place layer_norm_bwd needs one dtype");
  if (cols == 0) return VDSL_OK;
  if (rows > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "layer_norm_bwd: too many rows");
  int64_t partial_rows = 0;
  size_t need = 0;
  if (params) {
    VDSL_TRY(vdsl_layer_norm_bwd_workspace_bytes(rows, cols, &need));
    if (need) VDSL_TRY(check_buffer(q, workspace, need, "workspace", true));
  }
  const vdsl_buffer used = need ? workspace : nullptr;
  VDSL_TRY(check_apart("layer_norm_bwd", {dx, dgamma, dbeta, used}, {x, gamma, mean, rstd}));
  VDSL_TRY(check_apart("layer_norm_bwd", {dgamma, dbeta, used}, {dy}));  // dx may be dy
  float* part = params && rows ? static_cast<float*>(workspace->ptr) : nullptr;
  const void* g = gamma ? gamma->ptr : nullptr;
  float* const dgp = dgamma ? static_cast<float*>(dgamma->ptr) : nullptr;
  float* const dbp = dbeta ? static_cast<float*>(dbeta->ptr) : nullptr;
  const bool few = params && few_rows(rows, cols) && dx != dy;  // dy is read beside the writing of dx
  const float* mi = static_cast<const float*>(mean->ptr);
  const float* ri = static_cast<const float*>(rstd->ptr);
  const auto rows_kernel = [&](auto shape, auto xt, auto dyt) {
    using S = decltype(shape);
    constexpr int XT = decltype(xt)::value, DYT = decltype(dyt)::value;
    const int64_t blocks = bwd_blocks(rows, S::kRows, cols * static_cast<int64_t>(dtype_size(x_dtype) + dtype_size(dy_dtype)));
    partial_rows = blocks;
    if (few) {
      const int64_t all = (rows + S::kRows - 1) / S::kRows;
      hipLaunchKernelGGL((layer_norm_bwd_rows<S, XT, DYT, false, true>), dim3(static_cast<unsigned>(all + (cols + 15) / 16)),
                         dim3(S::kThreads), 0, q->stream, dy->ptr, x->ptr, g, param_dtype, mi, ri, dx->ptr, dx_dtype, nullptr, rows, cols,
                         static_cast<int>(all), dgp, dbp);
      return check_launch("layer_norm_bwd_rows");
    }
    const bool stream = rows * cols * static_cast<int64_t>(dtype_size(dx_dtype)) >= kStreamBytes;
    const auto kernel = stream ? layer_norm_bwd_rows<S, XT, DYT, true, false> : layer_norm_bwd_rows<S, XT, DYT, false, false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(S::kThreads), 0, q->stream,
                       dy->ptr, x->ptr, g, param_dtype, mi, ri, dx->ptr, dx_dtype, part, rows, cols, static_cast<int>(blocks), nullptr,
                       nullptr);
    return check_launch("layer_norm_bwd_rows");
  };
  const auto wide = [&] {
    if (params) {
      const int64_t strips = (cols + 1023) / 1024;
      partial_rows = std::min<int64_t>(bwd_most_blocks(rows, cols), std::max<int64_t>(1, 512 / strips));
      hipLaunchKernelGGL(layer_norm_bwd_columns, dim3(static_cast<unsigned>(strips), static_cast<unsigned>(partial_rows)), dim3(256),
                         0, q->stream, dy->ptr, dy_dtype, x->ptr, x_dtype, mi, ri, part, rows, cols);
      VDSL_TRY(check_launch("layer_norm_bwd_columns"));
    }
    hipLaunchKernelGGL(layer_norm_bwd_stream, block_grid(rows), dim3(1024), 0, q->stream, dy->ptr, dy_dtype, x->ptr,
                       x_dtype, g, param_dtype, mi, ri, dx->ptr, dx_dtype, rows, cols);
    return check_launch("layer_norm_bwd_stream");
  };
  using F = std::integral_constant<int, VDSL_F32>;
  using B = std::integral_constant<int, VDSL_BF16>;
  if (rows > 0) {
    int st;
    if (x_dtype == VDSL_F32 && dy_dtype == VDSL_F32) st = row_shape<4>(cols, [&](auto s) { return rows_kernel(s, F{}, F{}); }, wide);
    else if (x_dtype == VDSL_F32) st = row_shape<4>(cols, [&](auto s) { return rows_kernel(s, F{}, B{}); }, wide);
    else if (dy_dtype == VDSL_F32) st = row_shape<4>(cols, [&](auto s) { return rows_kernel(s, B{}, F{}); }, wide);
    else if (dx_dtype == VDSL_F32) st = row_shape<4>(cols, [&](auto s) { return rows_kernel(s, B{}, B{}); }, wide);
    else st = row_shape<8>(cols, [&](auto s) { return rows_kernel(s, B{}, B{}); }, wide);
    VDSL_TRY(st);
  }
  if (!params || (few && rows > 0)) return VDSL_OK;
  const int64_t blocks = (2 * cols + 63) / 64;
  if (blocks > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "layer_norm_bwd: too many columns");
  hipLaunchKernelGGL(layer_norm_bwd_finish, block_grid(blocks), dim3(1024), 0, q->stream, part, partial_rows, cols, dgp, dbp);
  return check_launch("layer_norm_bwd_finish");
}
