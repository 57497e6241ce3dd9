// Units of consecutive elements of a dense row, for kernels that give a lane several units of a row of
// any length: F32 or BF16 memory, f32 registers.  A row of an odd number of elements starts anywhere,
// so the vector accesses ask for no more than the element's alignment.
#pragma once

#include "common.h"

namespace vdsl {

struct __attribute__((packed, aligned(2))) U32x4At2 {
  u32x4 v;
};
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(2))) U32x2At2 {
  u32x2 v;
};
struct __attribute__((packed, aligned(4))) F32x4At4 {
  f32x4 v;
};

template <int DT>
__device__ __forceinline__ float load_elem(const void* __restrict__ p, int64_t i) {
  if constexpr (DT == VDSL_F32) return static_cast<const float*>(p)[i];
  else return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// Elements [e, e + U) of p, those from the n-th on as 0 and never read (n may be zero or negative).
template <int DT, int U>
__device__ __forceinline__ void load_unit(const void* __restrict__ p, int64_t e, int64_t n, float (&v)[U]) {
  static_assert(U == 4 || U == 8, "units of 4 or 8 elements");
  if (n >= U) {
    if constexpr (DT == VDSL_F32) {
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
  } else {
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] = j < n ? load_elem<DT>(p, e + j) : 0.0f;
  }
}

// The first n of v (at most U) to elements [e, e + n) of p, rounded once to its type.
template <int DT, int U>
__device__ __forceinline__ void store_unit(void* __restrict__ p, int64_t e, int64_t n, const float (&v)[U]) {
  if (n >= U) {
    if constexpr (DT == VDSL_F32) {
#pragma unroll
      for (int h = 0; h < U / 4; ++h) {
        const f32x4 x = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
        reinterpret_cast<F32x4At4*>(static_cast<float*>(p) + e + 4 * h)->v = x;
      }
    } else if constexpr (U == 8) {
      const u32x4 x = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
      reinterpret_cast<U32x4At2*>(static_cast<uint16_t*>(p) + e)->v = x;
    } else {
      const u32x2 x = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      reinterpret_cast<U32x2At2*>(static_cast<uint16_t*>(p) + e)->v = x;
    }
  } else {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (j < n) {
        if constexpr (DT == VDSL_F32) static_cast<float*>(p)[e + j] = v[j];
        else static_cast<uint16_t*>(p)[e + j] = f32_to_bf16(v[j]);
      }
    }
  }
}

// The same with the type as an argument that every lane shares.
template <int U>
__device__ __forceinline__ void load_unit(int dt, const void* __restrict__ p, int64_t e, int64_t n, float (&v)[U]) {
  if (dt == VDSL_F32) load_unit<VDSL_F32, U>(p, e, n, v);
  else load_unit<VDSL_BF16, U>(p, e, n, v);
}
template <int U>
__device__ __forceinline__ void store_unit(int dt, void* __restrict__ p, int64_t e, int64_t n, const float (&v)[U]) {
  if (dt == VDSL_F32) store_unit<VDSL_F32, U>(p, e, n, v);
  else store_unit<VDSL_BF16, U>(p, e, n, v);
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
