// Direct-to-LDS bf16 MFMA main loop for gfx950 on small tiles: C[m][n] = sum_k A(m, k) B(n, k) for K values
// [kb, ke), each operand row-major ([rows][K]) or K-major ([K][rows]), rows of whole 16-byte units.
//
// For launches that give a CU one or two small blocks: what a stage costs is then the latency of its loads over
// the stages in flight, so a ring of NS stages of 64 K values is filled by copies that take no registers (loads
// into registers were sunk behind the stage's MFMAs or waited for all together, 0.8 us a stage; a tile of 128 x 64
// takes 0.42 us of a CU so, two blocks to a CU).  Per stage: wait
// for this wave's copies of it, barrier, issue those of the stage NS - 1 further into the slot that every wave has
// left, compute.
//
// LDS: row-major as gemm_wide.h's, rows of 128 bytes.  K-major: 64 rows of 2 ROWS bytes; a transposing read
// takes 64 bytes of each of 4 neighbouring rows at a time, which ring_swz puts into the four quarters of the banks.
//
// Edges: rows past M or N repeat the last one (row-major) or the last 8 allocated columns (K-major): they reach no
// stored output.  In a last stage that is not whole the lanes past ke write zeros instead of copying.
#pragma once

#include "gemm_dma.h"

namespace vdsl {

template <int BM_, int BN_, int WGM_, int WGN_, int NS_, bool AKM_, bool BKM_>
struct RingConfig {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, NS = NS_;
  static constexpr bool AKM = AKM_, BKM = BKM_;
  static constexpr int NW = WGM * WGN, NT = 64 * NW, BK = 64;
  static constexpr int WTM = BM / WGM, WTN = BN / WGN, FM = WTM / 32, FN = WTN / 32;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES, LDS_BYTES = NS * STAGE;
  static constexpr int CA = BM / 8 / NW, CB = BN / 8 / NW;  // 1 KiB copies per wave and stage
  static_assert(CA * NW * 8 == BM && CB * NW * 8 == BN, "copies must split evenly over the waves");
};

// K-major rows of RB bytes: the XOR of row k's 16-byte chunk index (its bits 2 and 3, whole 64-byte windows).
template <int RB>
__device__ __forceinline__ int ring_swz(int k) {
  return RB >= 256 ? (k & 3) << 2 : RB == 128 ? ((k >> 1) & 1) << 2 : 0;
}

// One operand's copies: C blocks of 1 KiB per wave and stage.
template <bool KM, int ROWS, int NW, int C>
struct RingOperand {
  static constexpr int RB = KM ? 2 * ROWS : 128;  // bytes of an LDS row
  const char* base;  // of stage 0
  size_t step;       // bytes from a stage to the next
  uint32_t off[C];
  int k_of[C];       // the lane's first K value within a stage

  __device__ __forceinline__ RingOperand(const uint16_t* p, int rows, int r0, int64_t ld, int kb) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int CPR = RB / 16;  // chunks per LDS row
    base = reinterpret_cast<const char*>(p) + 2 * (KM ? static_cast<size_t>(kb) * ld + r0 : static_cast<size_t>(r0) * ld + kb);
    step = KM ? static_cast<size_t>(ld) * 128 : 128;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int row = (wave * C + u) * (64 / CPR) + lane / CPR, slot = lane % CPR;
      if constexpr (KM) {
        k_of[u] = row;
        const int col = min(8 * (slot ^ ring_swz<RB>(row)), static_cast<int>(ld) - 8 - r0);
        off[u] = 2 * (static_cast<uint32_t>(row) * static_cast<uint32_t>(ld) + static_cast<uint32_t>(col));
      } else {
        const int c = slot ^ ((row >> 1) & 7);
        k_of[u] = 8 * c;
        off[u] = 2 * static_cast<uint32_t>(min(row, rows - 1 - r0)) * static_cast<uint32_t>(ld) + 16 * c;
      }
    }
  }
  // Stage t, of which `left` K values (64 or fewer) are there, to the operand's area of its slot.
  __device__ __forceinline__ void copy(int t, int left, char* area) const {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const char* const from = base + t * step;
    char* const to = area + wave * C * 1024;
    if (left >= 64) {
#pragma unroll
      for (int u = 0; u < C; ++u) lds_copy16(from + off[u], to + u * 1024);
    } else {
#pragma unroll
      for (int u = 0; u < C; ++u) {
        if (k_of[u] < left) lds_copy16(from + off[u], to + u * 1024);
        else *reinterpret_cast<u32x4*>(to + u * 1024 + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
      }
    }
  }
};

// Fragment f of k-step kk of a stage's operand area for this lane: rows row0 + 32 f + l % 32.
template <bool KM, int ROWS>
__device__ __forceinline__ bf16x8 ring_fragment(const char* area, int row0, int f, int kk) {
  const int lane = threadIdx.x & 63;
  if constexpr (KM) {
    constexpr int RB = 2 * ROWS;
    const int g = lane >> 4, i = lane & 15;
    const int n = row0 + 32 * f + 16 * (g & 1) + 4 * (i & 3), k = 16 * kk + 8 * (g >> 1) + (i >> 2);
    // k and k + 4 have the same swizzle: it looks at k's bits 0 and 1
    const char* const p = area + k * RB + (((n >> 3) ^ ring_swz<RB>(k)) << 4) + ((n >> 2) & 1) * 8;
    const i16x4_t lo = lds_read_tr16(p), hi = lds_read_tr16(p + 4 * RB);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const int row = row0 + (lane & 31);
    return *reinterpret_cast<const bf16x8*>(area + row * 128 + 4096 * f + (((2 * kk + (lane >> 5)) ^ ((row >> 1) & 7)) << 4));
  }
}

// kb a multiple of 64, ke one or K; K-major: ld columns are allocated in every row.
template <class Cfg>
__device__ __forceinline__ void ring_mainloop(const uint16_t* __restrict__ A, const uint16_t* __restrict__ B, int M, int N, int kb, int ke,
                                              int m0, int n0, char* smem, f32x16 (&acc)[Cfg::FM][Cfg::FN], int64_t lda, int64_t ldb) {
  constexpr int NS = Cfg::NS;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / Cfg::WGN * Cfg::WTM, wc = wave % Cfg::WGN * Cfg::WTN;
#pragma unroll
  for (int i = 0; i < Cfg::FM; ++i)
#pragma unroll
    for (int j = 0; j < Cfg::FN; ++j) acc[i][j] = MfmaBf16::zero();
  const RingOperand<Cfg::AKM, Cfg::BM, Cfg::NW, Cfg::CA> a(A, M, m0, lda, kb);
  const RingOperand<Cfg::BKM, Cfg::BN, Cfg::NW, Cfg::CB> b(B, N, n0, ldb, kb);
  const int nk = (ke - kb + 63) / 64;
  const auto copy = [&](int t, int slot) {
    const int left = ke - kb - 64 * t;
    a.copy(t, left, smem + slot * Cfg::STAGE);
    b.copy(t, left, smem + slot * Cfg::STAGE + Cfg::A_BYTES);
  };
  // A stage's fragments are all read before its first MFMA: left alone, the compiler reads and waits for each k-step's.
  bf16x8 fa[4][Cfg::FM], fb[4][Cfg::FN];
  const auto read = [&](int slot) {
    const char* const stage = smem + slot * Cfg::STAGE;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
      for (int i = 0; i < Cfg::FM; ++i) fa[kk][i] = ring_fragment<Cfg::AKM, Cfg::BM>(stage, wr, i, kk);
#pragma unroll
      for (int j = 0; j < Cfg::FN; ++j) fb[kk][j] = ring_fragment<Cfg::BKM, Cfg::BN>(stage + Cfg::A_BYTES, wc, j, kk);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto multiply = [&]() {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int i = 0; i < Cfg::FM; ++i)
#pragma unroll
        for (int j = 0; j < Cfg::FN; ++j) acc[i][j] = MfmaBf16::mma(fa[kk][i], fb[kk][j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto on = [&](int slot) { return slot + 1 == NS ? 0 : slot + 1; };
#pragma unroll
  for (int t = 0; t < NS - 1; ++t)
    if (t < nk) copy(t, t);
  int t = 0, slot = 0, free_slot = NS - 1;
  for (; t + NS - 1 < nk; ++t) {
    dma_wait<(NS - 2) * (Cfg::CA + Cfg::CB)>();
    dma_barrier();
    read(slot);
    copy(t + NS - 1, free_slot);
    __builtin_amdgcn_sched_barrier(0);
    multiply();
    free_slot = slot;
    slot = on(slot);
  }
  dma_wait<0>();
  dma_barrier();
  for (; t < nk; ++t) {
    read(slot);
    multiply();
    slot = on(slot);
  }
}

}  // namespace vdsl
