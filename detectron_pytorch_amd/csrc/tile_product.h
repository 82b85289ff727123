// tile_product.h -- C[M, N] = sum_k A[m, k] B[n, k] of one workgroup's BM x BN tile on the matrix cores of gfx950, the loop that
// the classifier loss and the orthogonalised update share.  What is done with the tile is the caller's epilogue.
//
// Operands are 16-bit (fp16 or bf16) in one of two orders, chosen per operand, so that no product needs a transposed copy:
//   rows of k   element (row, k) at row * ld + k          fragments come by ds_read_b128
//   k-major     element (row, k) at k * ld + row          fragments come by ds_read_b64_tr_b16, which transposes on the way
// A split operand stands for a 32-bit one as hi + lo, two fp16 numbers of 11 bits each: every 32 elements of the contiguous
// axis are stored as 32 hi, then 32 lo, and the product is hi hi + hi lo + lo hi (the dropped lo lo is below 2^-22 of
// the term).  Three matrix instructions per 22-bit product run at 1/3 of the fp16 rate, more than five times the rate of
// the fp32 matrix instruction, and the accuracy is that of a float32 product (the accumulators are float32 in both).
//
// Staging: 16 bytes per lane go from memory straight to LDS (buffer_load_dwordx4 ... lds) into STAGES buffers of
// (BM + BN) * 128 bytes; the next STAGES - 1 stages are in flight while the waves multiply one, with one barrier per
// stage.  The DMA writes lanes in order, so the swizzle that keeps fragment reads free of bank conflicts is applied to the lanes' source
// addresses.  The buffer descriptor ends with the operand: what lies behind it reads as zero.
// The caller pads k with zeros to kStep in rows-of-k operands; a k-major operand ends after its last k by the descriptor.
#pragma once

#include "lds_dma.h"

namespace mi {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using lds_bytes = __attribute__((address_space(3))) char*;

template <bool BF16>
__device__ __forceinline__ f32x4 mfma_16x16x32(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One operand as the product sees it.  `rows`: its extent in the tile's direction; `k`: its extent in k (padded to kStep for
// rows of k).  Both count elements; `ld` and the base count 16-bit words (a split element takes two).
struct Operand {
  const uint16_t* base;
  long long ld;
  int rows, k;
};

template <int ROWS, int WAVES, bool SPLIT, bool KMAJOR>
struct Loader {
  static constexpr int kPieces = ROWS * 128 / 1024;  // 1 KB DMA pieces of a stage
  static constexpr int kPer = kPieces / WAVES;
  static_assert(kPieces % WAVES == 0, "every wave issues the same number of pieces");
  static constexpr int kWords = SPLIT ? 2 : 1;
  static constexpr int kStep = SPLIT ? 32 : 64;
  static constexpr int kRowBytes = ROWS * kWords * 2;  // k-major: bytes of one k in LDS
  unsigned voff[kPer];
  uintptr_t at;      // stage's first byte
  long long left;    // bytes of the operand from `at` on
  long long advance;

  // XOR of a k-major row's 32-byte units: the 16 rows that a fragment read touches at once fall into all banks evenly
  static __device__ __forceinline__ unsigned twist(unsigned k) {
    if constexpr (kRowBytes == 128) return ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
    return (k & 3) | (((k >> 3) & 1) << 2);
  }

  __device__ __forceinline__ void init(const Operand& o, int row0, int step0, int wave, int lane) {
    if constexpr (!KMAJOR) {
      const int last = o.rows - 1 - row0;  // rows behind the operand repeat its last one
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int row = (wave * kPer + j) * 8 + (lane >> 3);
        voff[j] = (unsigned)min(row, last) * (unsigned)(o.ld * 2) + (unsigned)(((lane & 7) ^ (lane >> 3)) * 16);
      }
      at = reinterpret_cast<uintptr_t>(o.base + (long long)row0 * o.ld);
      left = ((long long)last * o.ld + (long long)o.k * kWords) * 2;
      advance = 128;
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const unsigned byte = (unsigned)(wave * kPer + j) * 1024u + (unsigned)lane * 16u;
        const unsigned k = byte / kRowBytes, pos = byte % kRowBytes / 16u;
        voff[j] = k * (unsigned)(o.ld * 2) + ((((pos >> 1) ^ twist(k)) << 1) | (pos & 1)) * 16u;
      }
      at = reinterpret_cast<uintptr_t>(o.base + (long long)row0 * kWords);
      // a row is read to the end of a whole DMA lane (8 words), a split one to the end of its block of 32 hi, 32 lo
      const int rows = SPLIT ? (o.rows + 31) & ~31 : (o.rows + 7) & ~7;
      left = ((long long)(o.k - 1) * o.ld + (long long)(rows - row0) * kWords) * 2;
      advance = (long long)kStep * o.ld * 2;
    }
    at += advance * step0;
    left -= advance * step0;
  }

  __device__ __forceinline__ void issue(unsigned lds, int wave) {
    const long long l = left < 0 ? 0 : left;
    const srd_t srd = make_srd(reinterpret_cast<const void*>(at), l > 0xffffffffLL ? 0xffffffffu : (unsigned)l);
#pragma unroll
    for (int j = 0; j < kPer; ++j) dma_dwordx4(srd, lds + (unsigned)(wave * kPer + j) * 1024u, voff[j], 0u);
    at += advance;
    left -= advance;
  }
};

// WR x WC waves share the tile; each holds FM x FN fragments of 16 x 16.  acc[i][j][r] of lane l is the element
// (row i * 16 + (l & 15), column j * 16 + (l >> 4) * 4 + r) of the wave's part: four consecutive columns per lane.
template <int BM_, int BN_, int WR_, int WC_, int STAGES_, bool SPLIT_, bool BF16_, bool AKM, bool BKM>
struct TileProduct {
  static constexpr int BM = BM_, BN = BN_, WR = WR_, WC = WC_;
  static constexpr bool SPLIT = SPLIT_, BF16 = BF16_;
  static constexpr int kWaves = WR * WC, kThreads = kWaves * 64;
  static constexpr int kStep = SPLIT ? 32 : 64;
  static constexpr int FM = BM / WR / 16, FN = BN / WC / 16;
  static constexpr unsigned kABytes = BM * 128, kStage = (BM + BN) * 128;
  static constexpr int STAGES = STAGES_;
  static constexpr unsigned kLds = STAGES * kStage;
  using LoadA = Loader<BM, kWaves, SPLIT, AKM>;
  using LoadB = Loader<BN, kWaves, SPLIT, BKM>;

  template <class L, bool KMAJOR>
  static __device__ __forceinline__ s16x8 fragment(lds_bytes tile, int row, int kk, int lo, int lane) {
    if constexpr (!KMAJOR) {
      const int chunk = (SPLIT ? lo * 4 : kk * 4) + (lane >> 4);
      return *reinterpret_cast<__attribute__((address_space(3))) const s16x8*>(
          tile + (row + (lane & 15)) * 128 + ((chunk ^ (lane & 7)) << 4));
    } else {
      const int i = lane & 15, k = kk * 32 + (lane >> 4) * 8 + (i >> 2);
      const int unit = SPLIT ? (row >> 5) * 4 + lo * 2 + ((row >> 4) & 1) : row >> 4;
      lds_bytes p = tile + k * L::kRowBytes + ((unit ^ L::twist(k)) << 5) + (i & 3) * 8;
      // rows k + 4 .. k + 7 of the same lane: the twist looks at bits 0, 1 (or 1) and 3 of k only; bit 2 is h
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(p));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<__attribute__((address_space(3))) s16x4*>(p + 4 * L::kRowBytes));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }

  // the tile's sum over `steps` stages from stage `step0` on; ends with all waves past their last read of LDS
  static __device__ __forceinline__ void run(f32x4 (&acc)[FM][FN], const Operand& a, const Operand& b, int row0, int col0,
                                             int step0, int steps, lds_bytes lds) {
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const unsigned base = (unsigned)(uintptr_t)lds;
    LoadA la;
    LoadB lb;
    la.init(a, row0, step0, wave, lane);
    lb.init(b, col0, step0, wave, lane);
    const int wm = wave / WC * (BM / WR), wn = wave % WC * (BN / WC);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int kAhead = (STAGES - 2) * (LoadA::kPer + LoadB::kPer);  // DMA of younger stages that may stay in flight
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (s < steps) {
        la.issue(base + s * kStage, wave);
        lb.issue(base + s * kStage + kABytes, wave);
      }
    int slot = 0;
    for (int s = 0; s < steps; ++s) {
      // this stage has landed, and this wave's reads of the last one have returned: its LDS may be overwritten
      if (kAhead > 0 && s + STAGES - 2 < steps)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kAhead) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s + STAGES - 1 < steps) {
        const unsigned next = base + (unsigned)(slot == 0 ? STAGES - 1 : slot - 1) * kStage;
        la.issue(next, wave);
        lb.issue(next + kABytes, wave);
      }
      const lds_bytes ta = lds + slot * kStage, tb = ta + kABytes;
      slot = slot == STAGES - 1 ? 0 : slot + 1;
      if constexpr (SPLIT) {
        s16x8 ah[FM], al[FM], bh[FN], bl[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) ah[i] = fragment<LoadA, AKM>(ta, wm + i * 16, 0, 0, lane);
#pragma unroll
        for (int j = 0; j < FN; ++j) bh[j] = fragment<LoadB, BKM>(tb, wn + j * 16, 0, 0, lane);
#pragma unroll
        for (int j = 0; j < FN; ++j) bl[j] = fragment<LoadB, BKM>(tb, wn + j * 16, 0, 1, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i) al[i] = fragment<LoadA, AKM>(ta, wm + i * 16, 0, 1, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma_16x16x32<BF16>(bh[j], ah[i], acc[i][j]);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma_16x16x32<BF16>(bl[j], ah[i], acc[i][j]);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma_16x16x32<BF16>(bh[j], al[i], acc[i][j]);
      } else {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          s16x8 af[FM], bf[FN];
#pragma unroll
          for (int i = 0; i < FM; ++i) af[i] = fragment<LoadA, AKM>(ta, wm + i * 16, kk, 0, lane);
#pragma unroll
          for (int j = 0; j < FN; ++j) bf[j] = fragment<LoadB, BKM>(tb, wn + j * 16, kk, 0, lane);
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mfma_16x16x32<BF16>(bf[j], af[i], acc[i][j]);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // this lane's first row and column inside the tile
  static __device__ __forceinline__ int lane_row() {
    const int wave = uniform((int)(threadIdx.x >> 6));
    return wave / WC * (BM / WR) + (threadIdx.x & 15);
  }
  static __device__ __forceinline__ int lane_col() {
    const int wave = uniform((int)(threadIdx.x >> 6));
    return wave % WC * (BN / WC) + ((threadIdx.x >> 4) & 3) * 4;
  }
};

// Workgroup -> tile.  Consecutive workgroups go to the 8 XCDs in turn: each XCD gets one contiguous run of the tile order,
// which walks bands of `band` tile rows column by column, so that the tiles an XCD works on at a time share
// rows of A and columns of B in its L2.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int band, int& tm, int& tn) {
  const int total = tiles_m * tiles_n, q = total >> 3, r = total & 7, xcd = id & 7, pos = id >> 3;
  const int t = xcd * q + min(xcd, r) + pos;
  const int per = band * tiles_n, b = t / per, in = t - b * per;
  const int high = min(band, tiles_m - b * band);
  tn = in / high;
  tm = b * band + in - tn * high;
}

}  // namespace
}  // namespace mi
