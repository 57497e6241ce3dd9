// Rotary positions: pair (a, b) of a head at position p becomes m (a cos t - b sin t, a sin t + b cos t), t = 2 pi p f
// (-t for the gradient, which is the inverse rotation).  Pairs are columns (i, i + pairs) or (2 i, 2 i + 1) of the first
// 2 * pairs columns of a head; everything else of a row is handed on.
//
// A block has one row.  Its angles depend on the pair alone, so they are made once a row and shared through LDS by all
// heads (one sine and cosine per row and pair, whatever the number of heads); the rest is a copy at memory rate, which bounds
// it: 16384 rows of 48 heads of 128, of which 40 turn, f32 to bf16 (604 MB) take 107 us, 5.6 TB/s; 8 rows a launch.  Pairs and widths
// that are no multiples of 4 move single elements: 48 heads of 126 in bf16, 63 pairs each, 3.7 TB/s where heads of 128 have 5.6.  The turns
// p f are formed in f64: at p = 2^20 a product in f32 would hold its fraction to 2^-4 only.  They leave as a
// fraction of a turn in [-1/2, 1/2], of which f32 sine and cosine are good to their last place.
#include <algorithm>
#include <cmath>

#include "rowunit.h"

namespace vdsl {
namespace {

struct RopeArgs {
  const void* x;
  void* y;
  const int32_t* positions;
  const float* freqs;
  int64_t rows, width, first;
  int heads, dim, pairs, interleaved;
  float sign, magnitude;
  bool copy;  // whether the columns that do not turn are to be written (not in place)
};

// Units of U pairs, and of U columns that stay: U divides the pairs and every run of the others.
template <int XT, int YT, int U>
__global__ __launch_bounds__(256) void rope_rows(RopeArgs p) {
  extern __shared__ float2 turn[];  // of the row's pairs: magnitude cos t, magnitude sin t
  const int64_t row = block_index();
  if (row >= p.rows) return;
  const int64_t base = row * p.width;
  if (p.heads > 0) {
    const double at = static_cast<double>(p.positions[row]);
    for (int i = threadIdx.x; i < p.pairs; i += 256) {
      double t = at * (static_cast<double>(p.freqs[i]) + static_cast<double>(p.freqs[p.pairs + i]));
      t -= rint(t);
      float s, c;
      sincospif(2.0f * static_cast<float>(t), &s, &c);
      turn[i] = make_float2(p.magnitude * c, p.sign * p.magnitude * s);
    }
    __syncthreads();
    const int per = p.pairs / U;  // units of a head
    int h = threadIdx.x / per, i = threadIdx.x % per;
    const int dh = 256 / per, di = 256 % per;
    while (h < p.heads) {
      const int64_t e = base + p.first + static_cast<int64_t>(h) * p.dim + (p.interleaved ? 2 * U * i : U * i);
      const int64_t e2 = e + (p.interleaved ? U : p.pairs);
      float a[U], b[U];
      load_whole<XT, U>(p.x, e, a);
      load_whole<XT, U>(p.x, e2, b);
      if constexpr (U > 1) {
        if (p.interleaved) {
          float lo[U], hi[U];
#pragma unroll
          for (int j = 0; j < U; j += 2) {
            const float2 w = turn[U * i + j / 2], z = turn[U * i + U / 2 + j / 2];
            lo[j] = a[j] * w.x - a[j + 1] * w.y;
            lo[j + 1] = a[j] * w.y + a[j + 1] * w.x;
            hi[j] = b[j] * z.x - b[j + 1] * z.y;
            hi[j + 1] = b[j] * z.y + b[j + 1] * z.x;
          }
          store_whole<YT, U>(p.y, e, lo);
          store_whole<YT, U>(p.y, e2, hi);
        }
      }
      if (U == 1 || !p.interleaved) {
        float lo[U], hi[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const float2 w = turn[U * i + j];
          lo[j] = a[j] * w.x - b[j] * w.y;
          hi[j] = a[j] * w.y + b[j] * w.x;
        }
        store_whole<YT, U>(p.y, e, lo);
        store_whole<YT, U>(p.y, e2, hi);
      }
      h += dh;
      i += di;
      if (i >= per) {
        i -= per;
        ++h;
      }
    }
  }
  if (!p.copy) return;
  // the columns that stay: before the heads, the end of each head, behind the heads
  const int64_t end = p.first + static_cast<int64_t>(p.heads) * p.dim;
  const int stay = p.dim - 2 * p.pairs;
  const auto hand_on = [&](int64_t c) {
    float v[U];
    load_whole<XT, U>(p.x, base + c, v);
    store_whole<YT, U>(p.y, base + c, v);
  };
  for (int64_t c = static_cast<int64_t>(U) * threadIdx.x; c < p.first; c += 256 * U) hand_on(c);
  for (int64_t c = end + static_cast<int64_t>(U) * threadIdx.x; c < p.width; c += 256 * U) hand_on(c);
  if (stay > 0) {
    const int units = stay / U;
    int k = threadIdx.x / units, u = threadIdx.x % units;
    while (k < p.heads) {
      hand_on(p.first + static_cast<int64_t>(k) * p.dim + 2 * p.pairs + U * u);
      k += 256 / units;
      u += 256 % units;
      if (u >= units) {
        u -= units;
        ++k;
      }
    }
  }
}

}  // namespace
}  // namespace vdsl

using namespace vdsl;

extern "C" int vdsl_op_rope(vdsl_queue q, const vdsl_rope_params* p, int32_t x_dtype, vdsl_buffer x, vdsl_buffer positions,
                            vdsl_buffer freqs, int32_t y_dtype, vdsl_buffer y) {
  VDSL_TRY(enter_queue(q));
  if (!p) return fail(VDSL_ERR_INVALID_ARG, "params is null");
  if (p->rows < 0 || p->width < 0 || p->first < 0 || p->heads < 0 || p->dim < 0 || p->pairs < 0)
    return fail(VDSL_ERR_INVALID_ARG, "negative shape");
  if (!float_type(x_dtype) || !float_type(y_dtype)) return fail(VDSL_ERR_UNSUPPORTED, "rope supports f32 and bf16");
  if (!std::isfinite(p->magnitude)) return fail(VDSL_ERR_INVALID_ARG, "rope: magnitude must be finite");
  if (p->pairs > p->dim / 2) return fail(VDSL_ERR_SHAPE, "rope: 2 * pairs columns do not fit a head");
  if (p->first > p->width || static_cast<int64_t>(p->heads) * p->dim > p->width - p->first)
    return fail(VDSL_ERR_SHAPE, "rope: the heads do not fit a row");
  VDSL_TRY(check_buffer(q, x, nbytes(p->rows, p->width, dtype_size(x_dtype)), "x", false));
  VDSL_TRY(check_buffer(q, positions, nbytes(p->rows, 4), "positions", false));
  VDSL_TRY(check_buffer(q, freqs, nbytes(p->pairs, 8), "freqs", false));
  VDSL_TRY(check_buffer(q, y, nbytes(p->rows, p->width, dtype_size(y_dtype)), "y", true));
  if (x == y && x_dtype != y_dtype) return fail(VDSL_ERR_INVALID_ARG, "in-place rope needs one dtype");
  VDSL_TRY(check_apart("rope", {y}, {positions, freqs}));
  if (p->rows == 0 || p->width == 0) return VDSL_OK;
  if (p->rows > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "rope: too many rows");
  if (p->pairs > 4096) return fail(VDSL_ERR_UNSUPPORTED, "rope: more than 4096 pairs");
  // without a pair everything stays: as no heads at all
  const bool any = p->heads > 0 && p->pairs > 0;
  const RopeArgs args = {x->ptr, y->ptr, static_cast<const int32_t*>(positions->ptr), static_cast<const float*>(freqs->ptr),
                         p->rows, p->width, any ? p->first : 0, any ? p->heads : 0, any ? p->dim : 0, any ? p->pairs : 0,
                         p->interleaved != 0, p->inverse ? -1.0f : 1.0f, p->magnitude, x != y};
  if (!any && x == y) return VDSL_OK;
  const auto fits = [&](int u) { return args.pairs % u == 0 && args.dim % u == 0 && args.first % u == 0 && p->width % u == 0; };
  const auto run = [&](auto xt, auto yt) {
    constexpr int XT = decltype(xt)::value, YT = decltype(yt)::value;
    const auto kernel = fits(8) ? rope_rows<XT, YT, 8> : fits(4) ? rope_rows<XT, YT, 4> : rope_rows<XT, YT, 1>;
    hipLaunchKernelGGL(kernel, block_grid(p->rows), dim3(256), sizeof(float2) * static_cast<size_t>(args.pairs), q->stream, args);
    return check_launch("rope_rows");
  };
  using F = std::integral_constant<int, VDSL_F32>;
  using B = std::integral_constant<int, VDSL_BF16>;
  if (x_dtype == VDSL_F32) return y_dtype == VDSL_F32 ? run(F{}, F{}) : run(F{}, B{});
  return y_dtype == VDSL_F32 ? run(B{}, F{}) : run(B{}, B{});
}
