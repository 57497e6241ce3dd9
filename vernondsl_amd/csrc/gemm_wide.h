// bf16 MFMA main loop for gfx950 over tiles of 256 x 256 in four waves of 128 x 128:
// C[m][n] = sum_k A(m, k) B(n, k), each operand row-major ([rows][K]) or K-major ([K][rows]).
//
// Why four waves: a wave of 128 x 128 reads 8 fragments for 16 MFMAs, one of 128 x 64 (gemm_dma.h's eight
// waves a tile) 6 for 8.  Per 16 K values a CU then reads 32 KiB of LDS and writes 16 for 512 cycles of
// MFMAs instead of 48 and 16.  The price is
// one wave to a SIMD: nothing else runs while it waits, so every fragment read and copy is placed between
// two MFMAs by hand (sched_barrier), and the accumulators take all 256 accumulation registers.
//
// Why 64 K values per stage: copies of 64-byte pieces of a row (32 K values) are what bounds the loop then
// (8192 x 32768 x 4096: 1090 TFLOP/s, 1400 without the copies); 128-byte pieces take half the requests.
//
// LDS: a ring of five slots of 32 KiB, an operand's stage each: A(0), B(0), A(1), B(1), A(2), ...
// Row-major: 256 rows of 128 bytes, a row's 16-byte chunk c in place c ^ (row / 2 % 8), so the 16 rows that
// are read together lie in 16 bank groups.  K-major: 64 rows of 512 bytes as in gemm_dma.h, read by
// ds_read_b64_tr_b16.  Copies go straight to LDS, 8 of a wave for each slot.  Stage t, four k-steps of 16 MFMAs:
//   k-steps 0 to 2: the MFMAs, the fragments of the next k-step, copies
//   k-step 3: 4 MFMAs; wait for this wave's copies of stage t + 1; barrier; the other MFMAs, with the first
//             fragments of t + 1 and copies
// From that barrier to the next, B(t + 2) goes to the slot of A(t) and then A(t + 3) to that of B(t), whose last
// fragments every wave has read by then.  The wait leaves A(t + 2) in flight: the copies never drain, and
// have half a stage or more to land.  The stages of a block's next tile follow those of the present one in
// the ring, so its first copies are in flight during the epilogue.
//
// 8192 x 4096 x 32768 (B row-major, A K-major), us on one card: eight waves with 64-byte stages 1821; these
// tiles with 32-value stages 1814, with two slots of both operands that drain at each barrier 1750, with the
// ring 1597 (the MFMA units busy 82% of the cycles at the 1.64 GHz that the power limit leaves).
//
// Edges: rows past M or N repeat the last one (row-major) or the last 8 columns (K-major): they reach no
// stored output.  K is taken in whole stages: a row-major operand holds them whole (K a multiple of 64, or
// zeros past K); a K-major one repeats its last row past K, which the other operand's zeros cancel.
#pragma once

#include "gemm_dma.h"

namespace vdsl {

struct WideCfg {
  static constexpr int BM = 256, BN = 256, WGM = 2, WGN = 2, NT = 256, NW = 4;
  static constexpr int WTM = 128, WTN = 128, FM = 4, FN = 4;
  static constexpr int BK = 64, SLOT = 32768, LDS_BYTES = 5 * SLOT;
};

// A scalar base plus a 32-bit offset per lane: the form that needs no vector address arithmetic.
__device__ __forceinline__ void wide_copy16(const char* base, uint32_t off, char* l) {
  __builtin_amdgcn_global_load_lds(base + off, (lds_void_t*)l, 16, 0, 0);
}

// The tiles of one block of a persistent launch: place p of all tiles for p = blockIdx.x, + gridDim.x, ...
// Places congruent mod 8 run on one XCD; each XCD gets a contiguous share of the tiles, walked in
// tile_coords' order, so the 32 tiles it works on at a time cover 8 tile rows x 4 tile columns.
struct WideWalk {
  int tiles_m, tiles_n, share, place;
  __device__ __forceinline__ WideWalk(int M, int N)
      : tiles_m((M + 255) / 256), tiles_n((N + 255) / 256), share((tiles_m * tiles_n + 7) / 8), place(blockIdx.x) {
    settle();
  }
  __device__ __forceinline__ int tile() const { return place % 8 * share + place / 8; }
  __device__ __forceinline__ bool valid() const { return place < 8 * share; }
  __device__ __forceinline__ void settle() {
    while (valid() && tile() >= tiles_m * tiles_n) place += gridDim.x;
  }
  __device__ __forceinline__ void next() {
    place += gridDim.x;
    settle();
  }
  __device__ __forceinline__ void origin(int& m0, int& n0) const {
    int tm, tn;
    tile_coords(tile(), tiles_m, tiles_n, tm, tn);
    m0 = tm * 256;
    n0 = tn * 256;
  }
};
inline unsigned wide_blocks(int64_t tiles) { return static_cast<unsigned>(tiles < 256 ? (tiles + 7) / 8 * 8 : 256); }

// A wave's copies of an operand, 8 blocks of 1 KiB per stage: all stages of a tile, then those of the
// block's next tile, so the copies run on through the end of a tile.
template <bool IS_A, bool KM>
struct WideSource {
  const uint16_t* p;
  int rows, stages, left;
  int64_t ld;          // elements between stored rows
  WideWalk walk;
  int at, r0;          // the stage, and the tile's first row
  int event;           // the stage before which something other than the base changes
  const char* base;    // of the stage's first K value
  size_t step;         // bytes from a stage to the next
  uint32_t off[8];     // of this lane

  // all_rows: M or N; K: all K values; whole: its last stage is there whole.
  __device__ __forceinline__ WideSource(const uint16_t* p_, int all_rows, int64_t ld_, int K, bool whole, const WideWalk& w)
      : p(p_), rows(all_rows), stages((K + 63) / 64), left(!KM || whole ? 64 : K - 64 * (stages - 1)), ld(ld_), walk(w),
        step(KM ? static_cast<size_t>(ld_) * 128 : 128) {
    tile();
  }
  __device__ __forceinline__ void tile() {
    int m0, n0;
    walk.origin(m0, n0);
    at = 0;
    r0 = IS_A ? m0 : n0;
    base = reinterpret_cast<const char*>(p) + (KM ? 2 * static_cast<size_t>(r0) : 2 * static_cast<size_t>(r0) * ld);
    offsets(stages == 1 ? left : 64);
    event = left < 64 && stages > 1 ? stages - 1 : stages;
  }
  // In a stage of which `there` K values are there (K-major).
  __device__ __forceinline__ void offsets(int there) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if constexpr (KM) {
        const int k = 2 * (8 * wave + u) + (lane >> 5);
        const int col = min(8 * ((lane & 31) ^ kn_swz(k)), rows - 8 - r0);
        off[u] = static_cast<uint32_t>(min(k, there - 1)) * static_cast<uint32_t>(ld) * 2 + 2 * static_cast<uint32_t>(col);
      } else {
        const int r = 8 * (8 * wave + u) + (lane >> 3);
        const int c = (lane & 7) ^ ((r >> 1) & 7);
        off[u] = static_cast<uint32_t>(min(r, rows - 1 - r0)) * static_cast<uint32_t>(ld) * 2 + 16 * c;
      }
    }
  }
  // On to the next stage; the last one of all is repeated (never read), so that the number of copies in
  // flight stays what the waits count on.
  __device__ __forceinline__ void next() {
    base += step;
    if (__builtin_expect(++at == event, 0)) {
      if (at < stages) {
        offsets(left);
        event = stages;
        return;
      }
      WideWalk w = walk;
      w.next();
      if (w.valid()) {
        walk = w;
        tile();
      } else {
        base -= step;
        --at;
      }
    }
  }
};

// Where a lane's fragments of an operand lie: row-major, the first fragment of each k-step (fragment f is
// 4096 f further); K-major, the two halves of each fragment (a k-step is 8192 further).
template <bool KM>
struct WideFragments {
  static constexpr int kAt = KM ? 8 : 4, kReads = KM ? 2 : 1;  // LDS reads per fragment
  int at[kAt];
  __device__ __forceinline__ WideFragments(int area, int row0) {  // the wave's first row within the tile
    const int lane = threadIdx.x & 63;
    if constexpr (KM) {
      const int g = lane >> 4, i = lane & 15;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int k = 8 * (g >> 1) + 4 * r + (i >> 2);
          const int n = row0 + 32 * f + 16 * (g & 1) + 4 * (i & 3);
          at[2 * f + r] = area + k * 512 + (((n >> 3) ^ kn_swz(k)) << 4) + ((n >> 2) & 1) * 8;
        }
    } else {
      const int row = row0 + (lane & 31);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) at[kk] = area + row * 128 + (((2 * kk + (lane >> 5)) ^ ((row >> 1) & 7)) << 4);
    }
  }
  __device__ __forceinline__ void move(int bytes) {
#pragma unroll
    for (int i = 0; i < kAt; ++i) at[i] += bytes;
  }
  // Read r of fragment f of k-step kk into v.
  __device__ __forceinline__ void read(bf16x8& v, i16x4_t& lo, const char* smem, int f, int kk, int r) const {
    if constexpr (KM) {
      if (r == 0) {
        lo = lds_read_tr16(smem + at[2 * f] + 8192 * kk);
      } else {
        const i16x4_t hi = lds_read_tr16(smem + at[2 * f + 1] + 8192 * kk);
        v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    } else {
      v = *reinterpret_cast<const bf16x8*>(smem + at[kk] + 4096 * f);
    }
  }
};

// All tiles of this block: epilogue(acc, m0, n0) for each.  A(m, k) with lda elements between stored rows, B
// likewise; a K-major operand's M or N a multiple of 8 (of what is allocated).  b_whole: B is K-major, its last stage
// is allocated whole and holds zeros past K.  K > 0: the copies run
// ahead of the loop and repeat its last stage, which has to be there.  smem: WideCfg's bytes.
template <bool AKM, bool BKM, class Epilogue>
__device__ __forceinline__ void wide_gemm(const uint16_t* __restrict__ A, const uint16_t* __restrict__ B, int M, int N, int K,
                                          int64_t lda, int64_t ldb, bool b_whole, char* smem, Epilogue&& epilogue) {
  constexpr int SLOT = WideCfg::SLOT;
  WideWalk walk(M, N);
  if (!walk.valid()) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  WideSource<true, AKM> sa(A, M, lda, K, false, walk);
  WideSource<false, BKM> sb(B, N, ldb, K, b_whole, walk);
  WideFragments<AKM> fa(0, 128 * (wave >> 1));
  WideFragments<BKM> fb(SLOT, 128 * (wave & 1));
  const int nk = (K + 63) / 64;
  char* const dst = smem + wave * 8192;
  const auto copy_a = [&](int slot, int u) { wide_copy16(sa.base, sa.off[u], dst + slot + u * 1024); };
  const auto copy_b = [&](int slot, int u) { wide_copy16(sb.base, sb.off[u], dst + slot + u * 1024); };
  const auto on = [&](int slot) { return slot >= 3 * SLOT ? slot - 3 * SLOT : slot + 2 * SLOT; };  // to the next stage's
#pragma unroll
  for (int u = 0; u < 8; ++u) copy_a(0, u);
  sa.next();
#pragma unroll
  for (int u = 0; u < 8; ++u) copy_b(SLOT, u);
  sb.next();
#pragma unroll
  for (int u = 0; u < 8; ++u) copy_a(2 * SLOT, u);
  sa.next();
#pragma unroll
  for (int u = 0; u < 6; ++u) copy_b(3 * SLOT, u);
  dma_wait<12>();
  dma_barrier();

  bf16x8 af[2][4], bf[2][4];
  i16x4_t lo_a, lo_b;
  // The n-th read of a k-step's fragments: B's, then A's, in the order in which they are needed.
  constexpr int RB = 4 * WideFragments<BKM>::kReads, RA = 4 * WideFragments<AKM>::kReads;
  const auto read_nth = [&](int n, int set, int kk) {
    if (n < RB) fb.read(bf[set][n / fb.kReads], lo_b, smem, n / fb.kReads, kk, n % fb.kReads);
    else if (n < RB + RA) fa.read(af[set][(n - RB) / fa.kReads], lo_a, smem, (n - RB) / fa.kReads, kk, (n - RB) % fa.kReads);
  };
#pragma unroll
  for (int n = 0; n < RB + RA; ++n) read_nth(n, 0, 0);
  int slot_a = 0, slot_b = SLOT;                // of stage kt
  int before_a = 3 * SLOT, before_b = 4 * SLOT;  // of the one before it
  for (; walk.valid(); walk.next()) {
    f32x16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = MfmaBf16::zero();
    for (int kt = 0; kt < nk; ++kt) {
      const int next_a = on(slot_a), next_b = on(slot_b);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int cur = kk & 1;
#pragma unroll
        for (int m = 0; m < 16; ++m) {
          acc[m / 4][m % 4] = MfmaBf16::mma(af[cur][m / 4], bf[cur][m % 4], acc[m / 4][m % 4]);
          __builtin_amdgcn_sched_barrier(0);
          if (kk < 3) {
            if (RA + RB > 8 || m < 8) read_nth(m, cur ^ 1, kk + 1);
            const int n = 16 * kk + m;
            if (n == 1) copy_b(before_a, 6);  // B(kt + 1)'s last
            if (n == 3) {
              copy_b(before_a, 7);
              sb.next();
            }
            if (n >= 7 && n % 4 == 3 && (n - 7) / 4 < 8) copy_a(before_b, (n - 7) / 4);  // A(kt + 2)
            if (n == 36) sa.next();
          } else {
            if (m == 3) {
              fa.move(next_a - slot_a);
              fb.move(next_b - slot_b);
              dma_wait<8>();
              dma_barrier();
              __builtin_amdgcn_sched_barrier(0);
            }
            if (m >= 3) {
              constexpr int per = (RA + RB + 9) / 10;  // reads after an MFMA
#pragma unroll
              for (int r = 0; r < per; ++r) read_nth((m - 3) * per + r, cur ^ 1, 0);
            }
            if (m >= 5 && m % 2 == 1) copy_b(slot_a, (m - 5) / 2);  // B(kt + 2)'s first 6
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      before_a = slot_a;
      before_b = slot_b;
      slot_a = next_a;
      slot_b = next_b;
    }
    int m0, n0;
    walk.origin(m0, n0);
    // the last MFMAs' results are in their registers after 18 wait states at most
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15");
    __builtin_amdgcn_sched_barrier(0);
    epilogue(acc, m0, n0);
    __builtin_amdgcn_sched_barrier(0);
  }
  dma_wait<0>();  // the copies past the end, before the block's LDS is freed
}

// An accumulator's value.  The accumulators fill the accumulation registers, and the compiler copies all of them
// to others before an epilogue's first use, spilling most: read one by one here.  wide_gemm has waited for
// the MFMAs before it calls the epilogue.
__device__ __forceinline__ float wide_value(float acc) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(acc));
  return v;
}

// The accumulators of a wave with C stored transposed, [N][M]: a lane has, of columns n0 + 32 j + lane % 32,
// the rows m0 + 32 i + 8 q + 4 (lane / 32) + e in acc[i][j][4 q + e] (m0, n0 the wave's own).  Four of
// them are neighbours in C; the lanes of the two halves exchange theirs, so that each holds eight.
//   lo, hi: this lane's packed words of q = 2 p and of q = 2 p + 1 (two 16-bit values a word); the eight
//   values of rows 8 (2 p + lane / 32) .. + 7 come back in order.
__device__ __forceinline__ u32x4 wide_exchange(uint32_t lo0, uint32_t lo1, uint32_t hi0, uint32_t hi1) {
  const auto a = __builtin_amdgcn_permlane32_swap(lo0, hi0, false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(lo1, hi1, false, false);
  return u32x4{a[0], b[0], a[1], b[1]};
}

}  // namespace vdsl
