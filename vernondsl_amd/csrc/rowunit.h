// Units of consecutive elements of a dense row, for kernels that give a lane several units of a row of
// any length (F32 or BF16 memory, f32 registers), and grids of any number of blocks.  A row of an odd number of elements starts anywhere,
// so the vector accesses ask for no more than the element's alignment.
#pragma once

#include "common.h"

namespace vdsl {

// (At: the vector with the struct's alignment, for a builtin that takes its address: a member's address would promise
// the vector's own.)
struct __attribute__((packed, aligned(2))) U32x4At2 {
  u32x4 v;
  typedef u32x4 At __attribute__((aligned(2)));
};
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(2))) U32x2At2 {
  u32x2 v;
  typedef u32x2 At __attribute__((aligned(2)));
};
struct __attribute__((packed, aligned(4))) F32x4At4 {
  f32x4 v;
  typedef f32x4 At __attribute__((aligned(4)));
};

// A grid of `blocks` blocks of up to 1024 lanes (times y): a launch takes fewer than 2^32 lanes along x, so x holds
// 2^21 blocks and z what that leaves.  The last of z may hold more: a kernel returns from those past its own.
inline dim3 block_grid(int64_t blocks, int64_t y = 1) {
  const int64_t x = blocks < (1 << 21) ? blocks : (1 << 21);
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>(y), static_cast<unsigned>((blocks + x - 1) / x));
}
__device__ __forceinline__ int64_t block_index() { return static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x; }

template <int DT>
__device__ __forceinline__ float load_elem(const void* __restrict__ p, int64_t i) {
  if constexpr (DT == VDSL_F32) return static_cast<const float*>(p)[i];
  else return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// Elements [e, e + U) of p, U 1, 4 or 8, and their store, rounded once to p's type.
template <int DT, int U>
__device__ __forceinline__ void load_whole(const void* __restrict__ p, int64_t e, float (&v)[U]) {
  if constexpr (U == 1) {
    v[0] = load_elem<DT>(p, e);
  } else if constexpr (DT == VDSL_F32) {
#pragma unroll
    for (int h = 0; h < U / 4; ++h) {
      const f32x4 x = reinterpret_cast<const F32x4At4*>(static_cast<const float*>(p) + e + 4 * h)->v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * h + j] = x[j];
    }
  } else if constexpr (U == 8) {
    const u32x4 x = reinterpret_cast<const U32x4At2*>(static_cast<const uint16_t*>(p) + e)->v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(x[j] << 16);
      v[2 * j + 1] = __uint_as_float(x[j] & 0xFFFF0000u);
    }
  } else {
    const u32x2 x = reinterpret_cast<const U32x2At2*>(static_cast<const uint16_t*>(p) + e)->v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v[2 * j] = __uint_as_float(x[j] << 16);
      v[2 * j + 1] = __uint_as_float(x[j] & 0xFFFF0000u);
    }
  }
}
// Outputs of this many bytes or more pass the caches by: they would drive out what else is there, and whoever reads
// them next finds little of them.  us of an embedding's lookup and the layer norm that reads it, rows of 4096 in bf16,
// stores kept and passed by: 64 MiB 44.5, 47.5; 128 MiB 91.7, 88.5; of layer norm's gradient and one that reads it
// 64.0, 73.5; 129.6, 125.8.
constexpr int64_t kStreamBytes = int64_t{96} << 20;

// STREAM is the kernels' parameter, since of a plain and a passing store in two branches the compiler makes one plain one.
template <bool STREAM, class Unit>
__device__ __forceinline__ void store_at(Unit* to, typename Unit::At v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<typename Unit::At*>(to));
  else to->v = v;
}
template <int DT, int U, bool STREAM = false>
__device__ __forceinline__ void store_whole(void* __restrict__ p, int64_t e, const float (&v)[U]) {
  if constexpr (U == 1) {
    if constexpr (DT == VDSL_F32) static_cast<float*>(p)[e] = v[0];
    else static_cast<uint16_t*>(p)[e] = f32_to_bf16(v[0]);
  } else if constexpr (DT == VDSL_F32) {
#pragma unroll
    for (int h = 0; h < U / 4; ++h) {
      const f32x4 x = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
      store_at<STREAM>(reinterpret_cast<F32x4At4*>(static_cast<float*>(p) + e + 4 * h), x);
    }
  } else if constexpr (U == 8) {
    const u32x4 x = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    store_at<STREAM>(reinterpret_cast<U32x4At2*>(static_cast<uint16_t*>(p) + e), x);
  } else {
    const u32x2 x = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    store_at<STREAM>(reinterpret_cast<U32x2At2*>(static_cast<uint16_t*>(p) + e), x);
  }
}
template <int U, bool STREAM = false>
__device__ __forceinline__ void store_unit(int dt, void* __restrict__ p, int64_t e, const float (&v)[U]) {
  if (dt == VDSL_F32) store_whole<VDSL_F32, U, STREAM>(p, e, v);
  else store_whole<VDSL_BF16, U, STREAM>(p, e, v);
}

// A lane's unit of U columns from column c on, in a row of at least U: a unit that would pass the row's end
// is moved back to end there, so every access is whole and no load has a branch around it (which would
// wait for that load before the next is issued).  Its first `skip` elements belong to the unit before
// (all of them for a unit past the end): a sum leaves them out; a store may repeat them, its lane having
// computed the same values.
template <int U>
struct UnitAt {
  int64_t c;
  int skip;
  __device__ __forceinline__ UnitAt(int64_t col, int64_t cols) {
    const int64_t over = col + U - cols;
    c = over > 0 ? cols - U : col;
    skip = over <= 0 ? 0 : over < U ? static_cast<int>(over) : U;
  }
  __device__ __forceinline__ bool any() const { return skip < U; }
};

// For accesses that are few: elements [e, e + 4) of p, of type dt (the same for every lane), those from the
// n-th on as 0 and never read (n may be zero or negative); and the store of the first n of v.
__device__ __forceinline__ void load_some(int dt, const void* __restrict__ p, int64_t e, int64_t n, float (&v)[4]) {
  if (n >= 4) {
    if (dt == VDSL_F32) load_whole<VDSL_F32, 4>(p, e, v);
    else load_whole<VDSL_BF16, 4>(p, e, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? (dt == VDSL_F32 ? load_elem<VDSL_F32>(p, e + j) : load_elem<VDSL_BF16>(p, e + j)) : 0.0f;
  }
}
__device__ __forceinline__ void store_some(int dt, void* __restrict__ p, int64_t e, int64_t n, const float (&v)[4]) {
  if (n >= 4) {
    store_unit<4>(dt, p, e, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < n) {
        if (dt == VDSL_F32) static_cast<float*>(p)[e + j] = v[j];
        else static_cast<uint16_t*>(p)[e + j] = f32_to_bf16(v[j]);
      }
    }
  }
}

// A wave's sum through DPP, every lane getting it: a butterfly inside each row of 16 lanes, then the
// four rows' values as scalars.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float wave_sum_rows(float v) {
  v = dpp_add<0xB1>(v);   // quad_perm [1,0,3,2]
  v = dpp_add<0x4E>(v);   // quad_perm [2,3,0,1]
  v = dpp_add<0x141>(v);  // row_half_mirror
  v = dpp_add<0x140>(v);  // row_mirror
  const int b = __builtin_bit_cast(int, v);
  const auto at = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, lane)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

}  // namespace vdsl
