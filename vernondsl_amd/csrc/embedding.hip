// Token embedding: the scaled lookup of table rows, and the table's gradient.
//
//   out[i] = scale table[ids[i]],  dtable[v] = scale (sum over the i with ids[i] = v, in ascending i, of dy[i]);
// an id outside [0, vocab) is no row: its output is zero and it adds to no row's gradient.
//
// Both are bound by HBM.  The lookup reads each row where it is and writes the output once.  The gradient
// does not add into the table with atomics, whose order would change its bits from run to run: the
// positions are sorted by token (stably, so a token's positions ascend), and then every row of dtable is
// written once, zero or the f32 sum of its terms.

#include <algorithm>
#include <type_traits>

#include "rowunit.h"

namespace vdsl {
namespace {

// L lanes per output row (a power of two), KU units of U elements each; blockIdx.y: strips of L KU units.
template <int TT, int OT, int U, int KU>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* __restrict__ table, const int32_t* __restrict__ ids,
                                                            void* __restrict__ out, int64_t n, int64_t dim, int64_t vocab,
                                                            float scale, int log_l) {
  const int lanes = 1 << log_l;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) << (8 - log_l)) + (threadIdx.x >> log_l);
  if (i >= n) return;
  const int32_t id = ids[i];
  const bool valid = id >= 0 && id < vocab;
  const int64_t c0 = (static_cast<int64_t>(blockIdx.y) * KU * lanes + (threadIdx.x & (lanes - 1))) * U;
  float v[KU][U];
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    const int64_t c = c0 + static_cast<int64_t>(k) * lanes * U;
    load_unit<TT, U>(table, static_cast<int64_t>(id) * dim + c, valid ? dim - c : 0, v[k]);
  }
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    const int64_t c = c0 + static_cast<int64_t>(k) * lanes * U;
#pragma unroll
    for (int j = 0; j < U; ++j) v[k][j] = valid ? v[k][j] * scale : 0.0f;
    store_unit<OT, U>(out, i * dim + c, dim - c, v[k]);
  }
}

// The positions sorted by token: position i goes to place #{j : id_j < id_i} + #{j < i : id_j = id_i}.
// A block ranks 64 positions, one a lane, its 16 waves a share of all ids each.  Ids are compared as
// unsigned numbers, so those that are no row come last.
__global__ __launch_bounds__(1024) void embedding_rank_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                              uint32_t* __restrict__ sorted, int32_t* __restrict__ order) {
  __shared__ int part[16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  const uint32_t key = i < n ? static_cast<uint32_t>(ids[i]) : 0;
  const int64_t share = (n + 15) / 16, j0 = wave * share, j1 = j0 + share < n ? j0 + share : n;
  int rank = 0;
  for (int64_t j = j0; j < j1; ++j) {
    const uint32_t other = static_cast<uint32_t>(ids[j]);
    rank += other < key || (other == key && j < i);
  }
  part[wave][lane] = rank;
  __syncthreads();
  if (wave != 0 || i >= n) return;
  rank = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) rank += part[w][lane];
  sorted[rank] = key;
  order[rank] = static_cast<int32_t>(i);
}

// dtable rows: a block takes 2^(8 - log_l) R consecutive rows, 2^log_l lanes to a row, each NV units of 4
// columns; blockIdx.y: strips of columns.  The rows' shares of the sorted positions come from binary searches.
constexpr int kRowsPerSlot = 4;

template <int DYT, int NV>
__global__ __launch_bounds__(256) void embedding_bwd_kernel(const uint32_t* __restrict__ sorted, const int32_t* __restrict__ order,
                                                            const void* __restrict__ dy, float* __restrict__ dtable, int64_t n,
                                                            int64_t dim, int64_t vocab, float scale, int log_l) {
  __shared__ int first[256 + 1];
  const int slots = 256 >> log_l, lanes = 1 << log_l, rows = slots * kRowsPerSlot;
  const int64_t v0 = static_cast<int64_t>(blockIdx.x) * rows;
  for (int r = threadIdx.x; r <= rows; r += 256) {  // the first place whose token is not below row v0 + r
    const uint64_t v = static_cast<uint64_t>(v0 + r < vocab ? v0 + r : vocab);
    int lo = 0, hi = static_cast<int>(n);
    while (lo < hi) {
      const int mid = lo + ((hi - lo) >> 1);
      if (sorted[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    first[r] = lo;
  }
  __syncthreads();
  const int64_t c0 = (static_cast<int64_t>(blockIdx.y) * NV * lanes + (threadIdx.x & (lanes - 1))) * 4;
  for (int k = 0; k < kRowsPerSlot; ++k) {
    const int r = k * slots + static_cast<int>(threadIdx.x >> log_l);
    const int64_t v = v0 + r;
    if (v >= vocab) return;
    float acc[NV][4];
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[u][j] = 0.0f;
    for (int e = first[r]; e < first[r + 1]; ++e) {
      const int64_t i = order[e];
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int64_t c = c0 + static_cast<int64_t>(u) * lanes * 4;
        float d[4];
        load_unit<DYT, 4>(dy, i * dim + c, dim - c, d);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[u][j] += d[j];
      }
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int64_t c = c0 + static_cast<int64_t>(u) * lanes * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[u][j] *= scale;
      store_unit<VDSL_F32, 4>(dtable, v * dim + c, dim - c, acc[u]);
    }
  }
}

bool float_type(int32_t t) { return t == VDSL_F32 || t == VDSL_BF16; }

// log2 of the lanes that share a row of `units` units: a power of two from 16 to 256.
int lanes_log2(int64_t units) {
  int l = 4;
  while (l < 8 && (int64_t{1} << l) < units) ++l;
  return l;
}

int check_extents(int64_t n, int64_t dim, int64_t vocab) {
  if (n < 0 || dim < 0 || vocab < 0) return fail(VDSL_ERR_INVALID_ARG, "negative shape");
  if (n > 0x7fffffff || vocab > 0x7fffffff) return fail(VDSL_ERR_UNSUPPORTED, "embedding: too many tokens or table rows");
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
  if (out == table) return fail(VDSL_ERR_INVALID_ARG, "embedding_fwd: out must not be the table");
  if (n == 0 || dim == 0) return VDSL_OK;
  const auto go = [&](auto tt, auto ot, auto unit, auto ku) {
    constexpr int TT = decltype(tt)::value, OT = decltype(ot)::value, U = decltype(unit)::value, KU = decltype(ku)::value;
    const int64_t units = (dim + U - 1) / U;
    const int l = lanes_log2(units);
    const int64_t bx = (n + (256 >> l) - 1) >> (8 - l), by = (units + (int64_t{KU} << l) - 1) / (int64_t{KU} << l);
    if (by > 65535) return fail(VDSL_ERR_UNSUPPORTED, "embedding_fwd: rows too wide");
    hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, U, KU>), dim3(static_cast<unsigned>(bx), static_cast<unsigned>(by)), dim3(256), 0,
                       q->stream, table->ptr, static_cast<const int32_t*>(ids->ptr), out->ptr, n, dim, vocab, scale, l);
    return check_launch("embedding_fwd_kernel");
  };
  using F = std::integral_constant<int, VDSL_F32>;
  using B = std::integral_constant<int, VDSL_BF16>;
  using K = std::integral_constant<int, 1>;
  using U4 = std::integral_constant<int, 4>;
  using U8 = std::integral_constant<int, 8>;
  if (table_dtype == VDSL_F32 && out_dtype == VDSL_F32) return go(F{}, F{}, U4{}, K{});
  if (table_dtype == VDSL_F32) return go(F{}, B{}, U4{}, K{});
  if (out_dtype == VDSL_F32) return go(B{}, F{}, U4{}, K{});
  return go(B{}, B{}, U8{}, K{});
}

extern "C" int vdsl_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t dim, size_t* bytes) {
  if (!bytes) return fail(VDSL_ERR_INVALID_ARG, "bytes is null");
  VDSL_TRY(check_extents(n, dim, vocab));
  *bytes = static_cast<size_t>(n) * 8;
  return VDSL_OK;
}

extern "C" int vdsl_op_embedding_bwd(vdsl_queue q, int64_t n, int64_t dim, int64_t vocab, vdsl_buffer ids, int32_t dy_dtype,
                                     vdsl_buffer dy, float scale, vdsl_buffer dtable, vdsl_buffer workspace) {
  VDSL_TRY(enter_queue(q));
  VDSL_TRY(check_extents(n, dim, vocab));
  if (!float_type(dy_dtype)) return fail(VDSL_ERR_UNSUPPORTED, "embedding_bwd supports f32 and bf16");
  VDSL_TRY(check_buffer(q, ids, nbytes(n, 4), "ids", false));
  VDSL_TRY(check_buffer(q, dy, nbytes(n, dim, dtype_size(dy_dtype)), "dy", false));
  VDSL_TRY(check_buffer(q, dtable, nbytes(vocab, dim, 4), "dtable", true));
  size_t need = 0;
  VDSL_TRY(vdsl_embedding_bwd_workspace_bytes(n, vocab, dim, &need));
  if (need) VDSL_TRY(check_buffer(q, workspace, need, "workspace", true));
  if (vocab == 0 || dim == 0) return VDSL_OK;
  uint32_t* sorted = n ? static_cast<uint32_t*>(workspace->ptr) : nullptr;
  int32_t* order = reinterpret_cast<int32_t*>(sorted) + n;
  if (n) {
    hipLaunchKernelGGL(embedding_rank_kernel, dim3(static_cast<unsigned>((n + 63) / 64)), dim3(1024), 0, q->stream,
                       static_cast<const int32_t*>(ids->ptr), n, sorted, order);
    VDSL_TRY(check_launch("embedding_rank_kernel"));
  }
  constexpr int NV = 4;
  const int64_t units = (dim + 3) / 4;
  const int l = lanes_log2((units + NV - 1) / NV);
  const int64_t rows = int64_t{256 >> l} * kRowsPerSlot;
  const int64_t by = (units + (int64_t{NV} << l) - 1) / (int64_t{NV} << l);
  if (by > 65535) return fail(VDSL_ERR_UNSUPPORTED, "embedding_bwd: rows too wide");
  const dim3 grid(static_cast<unsigned>((vocab + rows - 1) / rows), static_cast<unsigned>(by));
  if (dy_dtype == VDSL_F32)
    hipLaunchKernelGGL((embedding_bwd_kernel<VDSL_F32, NV>), grid, dim3(256), 0, q->stream, sorted, order, dy->ptr,
                       static_cast<float*>(dtable->ptr), n, dim, vocab, scale, l);
  else
    hipLaunchKernelGGL((embedding_bwd_kernel<VDSL_BF16, NV>), grid, dim3(256), 0, q->stream, sorted, order, dy->ptr,
                       static_cast<float*>(dtable->ptr), n, dim, vocab, scale, l);
  return check_launch("embedding_bwd_kernel");
}
