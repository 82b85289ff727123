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
// (BM + BN) * 128 bytes (64 k a stage, split 32), with one barrier per stage.  Fragments are read half a stage ahead of their
// products, so a stage's buffer is free, and the stage STAGES later on its way into it, while its second half is still being
// multiplied.  The DMA writes lanes in order, so the swizzle that keeps fragment reads free of bank conflicts is applied to the lanes' source
// addresses.  The buffer descriptor ends with the operand: what lies behind it reads as zero.
// The caller pads k with zeros to kStep in rows-of-k operands; a k-major operand ends after its last k by the descriptor.
#pragma once

#include "common.h"
#include "lds_dma.h"

namespace mi {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using lds_bytes = __attribute__((address_space(3))) char*;

// The 32 x 32 x 16 form: one wave per SIMD keeps the matrix cores busy with it (2.46 PFLOP/s over the chip on zeros), where the
// 16 x 16 x 32 form reaches 1.45-1.58 with one wave per SIMD and 2.27 with two.
template <bool BF16>
__device__ __forceinline__ f32x16 mfma_32x32x16(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
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
  static constexpr int kStep = 64 / kWords;
  static constexpr int kRowBytes = ROWS * kWords * 2;  // k-major: bytes of one k in LDS
  unsigned voff[kPer];
  uintptr_t at;      // stage's first byte
  long long left;    // bytes of the operand from `at` on
  long long advance;

  // XOR of a row's chunks: the rows that a fragment read touches at once fall into all banks evenly
  static __device__ __forceinline__ int shuffle(int row) { return (row >> 1) & 7; }
  // XOR of a k-major row's 32-byte units: the 16 rows that a fragment read touches at once fall into all banks evenly
  static __device__ __forceinline__ unsigned twist(unsigned k) {
    if constexpr (kRowBytes == 128) return (((k >> 1) & 1) << 1) | ((k >> 3) & 1);
    return ((k & 3) << 1) | ((k >> 3) & 1);
  }

  __device__ __forceinline__ void init(const Operand& o, int row0, int step0, int wave, int lane) {
    if constexpr (!KMAJOR) {
      const int last = o.rows - 1 - row0;  // rows behind the operand repeat its last one
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int row = (wave * kPer + j) * 8 + (lane >> 3);
        voff[j] = (unsigned)min(row, last) * (unsigned)(o.ld * 2) + (unsigned)(((lane & 7) ^ shuffle(row)) * 16);
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

  // The descriptor of the stage that is due, empty for stages behind the last one: their pieces read nothing.
  __device__ __forceinline__ srd_t begin(bool any) {
    const long long l = !any || left < 0 ? 0 : left;
    const srd_t srd = make_srd(reinterpret_cast<const void*>(at), l > 0xffffffffLL ? 0xffffffffu : (unsigned)l);
    at += advance;
    left -= advance;
    return srd;
  }
  __device__ __forceinline__ void piece(const srd_t& srd, unsigned lds, int wave, int j) {
    dma_dwordx4(srd, lds + (unsigned)(wave * kPer + j) * 1024u, voff[j], 0u);
  }
};

// WR x WC waves share the tile; each holds FM x FN fragments of 32 x 32.  acc[i][j][4 g + r] of lane l is the element
// (row i * 32 + (l & 31), column j * 32 + g * 8 + (l >> 5) * 4 + r) of the wave's part: four consecutive columns per lane and g.
template <int BM_, int BN_, int WR_, int WC_, int STAGES_, bool SPLIT_, bool BF16_, bool AKM, bool BKM>
struct TileProduct {
  static constexpr int BM = BM_, BN = BN_, WR = WR_, WC = WC_;
  static constexpr bool SPLIT = SPLIT_, BF16 = BF16_;
  static constexpr int kWaves = WR * WC, kThreads = kWaves * 64;
  static constexpr int kStep = SPLIT ? 32 : 64;
  static constexpr int FM = BM / WR / 32, FN = BN / WC / 32;
  static constexpr unsigned kABytes = BM * 128, kStage = (BM + BN) * 128;
  static constexpr int STAGES = STAGES_;
  static constexpr unsigned kLds = STAGES * kStage;
  using LoadA = Loader<BM, kWaves, SPLIT, AKM>;
  using LoadB = Loader<BN, kWaves, SPLIT, BKM>;

  // rows row .. row + 31, k from 16 kk on (split: of the hi or the lo words); lane l holds row l & 31, k (l >> 5) * 8 .. + 7
  template <class L, bool KMAJOR>
  static __device__ __forceinline__ s16x8 fragment(lds_bytes tile, int row, int kk, int lo, int lane) {
    if constexpr (!KMAJOR) {
      const int chunk = lo * 4 + kk * 2 + (lane >> 5);
      return *reinterpret_cast<__attribute__((address_space(3))) const s16x8*>(
          tile + (row + (lane & 31)) * 128 + ((chunk ^ L::shuffle(lane & 31)) << 4));
    } else {
      const int i = lane & 15, k = kk * 16 + (lane >> 5) * 8 + (i >> 2), col = row + (lane & 16);
      const int unit = SPLIT ? (col >> 5) * 4 + lo * 2 + ((col >> 4) & 1) : col >> 4;
      lds_bytes p = tile + k * L::kRowBytes + ((unit ^ L::twist(k)) << 5) + (i & 3) * 8;
      // rows k .. k + 3, then k + 4 .. k + 7 of the same lane: the twist does not look at bit 2 of k
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(p));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<__attribute__((address_space(3))) s16x4*>(p + 4 * L::kRowBytes));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }

  // Fragments of a stage in two halves.  Plain: k 0..31 and k 32..63.  Split: the hi words, then the lo words.
  struct Fragments {
    s16x8 a[2][FM], b[2][FN];
  };
  static constexpr int kLoads = 2 * (FM + FN);                // fragments of a half
  static constexpr int kProducts = 2 * FM * FN;               // matrix instructions of a half
  static constexpr int kPieces = LoadA::kPer + LoadB::kPer;   // DMA pieces of a stage that a wave issues

  struct Place {  // of this wave in the tile
    int wm, wn, lane;
  };
  static __device__ __forceinline__ void load_a(Fragments& f, int k, int i, lds_bytes stage, int half, const Place& w) {
    f.a[k][i] = fragment<LoadA, AKM>(stage, w.wm + i * 32, SPLIT ? k : half * 2 + k, SPLIT ? half : 0, w.lane);
  }
  static __device__ __forceinline__ void load_b(Fragments& f, int k, int j, lds_bytes stage, int half, const Place& w) {
    f.b[k][j] = fragment<LoadB, BKM>(stage + kABytes, w.wn + j * 32, SPLIT ? k : half * 2 + k, SPLIT ? half : 0, w.lane);
  }
  // the half's n-th fragment, in the order in which products need them
  static __device__ __forceinline__ void load(Fragments& f, int n, lds_bytes stage, int half, const Place& w) {
    const int k = n / (FM + FN), m = n % (FM + FN);
    if (m < FN)
      load_b(f, k, m, stage, half, w);
    else
      load_a(f, k, m - FN, stage, half, w);
  }

  // One half's products; behind the n-th of them `between(n)` issues memory instructions.  A wave issues in order, and LDS reads and
  // DMA pieces queue: in one bunch they would hold up the products behind them (64 KB of pieces take as long to issue
  // as half a stage's products), one at a time they pass beside them.
  template <class F>
  static __device__ __forceinline__ void multiply(f32x16 (&acc)[FM][FN], const s16x8 (&a)[2][FM], const s16x8 (&b)[2][FN],
                                                  F between) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          acc[i][j] = mfma_32x32x16<BF16>(b[k][j], a[k][i], acc[i][j]);
          between((k * FN + j) * FM + i);
        }
  }
  static __device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

  // Behind product n, its share of LOADS fragment loads and PIECES DMA pieces, one of each in turn.
  template <int LOADS, int PIECES, class L, class S>
  static __device__ __forceinline__ void deal(int n, L load_one, S piece_one) {
    constexpr int ops = LOADS + PIECES, each = (ops + kProducts - 1) / kProducts, both = LOADS < PIECES ? LOADS : PIECES;
#pragma unroll
    for (int e = 0; e < each; ++e) {
      const int op = n * each + e;
      if (op >= ops) continue;
      if (op < 2 * both) {
        if (op % 2 == 0)
          piece_one(op / 2);
        else
          load_one(op / 2);
      } else if (PIECES > LOADS) {
        piece_one(op - both);
      } else {
        load_one(op - both);
      }
    }
    if (n * each < ops) pin();
  }

  // the tile's sum over `steps` stages from stage `step0` on
  static __device__ __forceinline__ void run(f32x16 (&acc)[FM][FN], const Operand& a, const Operand& b, int row0, int col0,
                                             int step0, int steps, lds_bytes lds) {
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const unsigned base = (unsigned)(uintptr_t)lds;
    const Place w = {wave / WC * (BM / WR), wave % WC * (BN / WC), lane};
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};
    LoadA la;
    LoadB lb;
    la.init(a, row0, step0, wave, lane);
    lb.init(b, col0, step0, wave, lane);
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      const srd_t sa = la.begin(s < steps), sb = lb.begin(s < steps);
#pragma unroll
      for (int j = 0; j < LoadA::kPer; ++j) la.piece(sa, base + s * kStage, wave, j);
#pragma unroll
      for (int j = 0; j < LoadB::kPer; ++j) lb.piece(sb, base + s * kStage + kABytes, wave, j);
    }
    Fragments now, rest;
    wait_for_stage<(STAGES - 1) * kPieces>();
#pragma unroll
    for (int n = 0; n < kLoads; ++n) load(now, n, lds, 0, w);
    int slot = 0;
    for (int s = 0; s < steps; ++s) {
      const lds_bytes here = lds + slot * kStage;
      const unsigned freed = base + slot * kStage;
      slot = slot == STAGES - 1 ? 0 : slot + 1;
      const lds_bytes next = lds + slot * kStage;  // behind the last stage: a buffer that is read and not used
      asm volatile("" ::: "memory");
      multiply(acc, now.a, now.b, [&](int n) {  // under it, the other half's fragments
        constexpr int every = kProducts / kLoads > 1 ? kProducts / kLoads : 1, each = (kLoads + kProducts - 1) / kProducts;
        if (n % every == 0) {
#pragma unroll
          for (int e = 0; e < each; ++e)
            if (n / every * each + e < kLoads) load(rest, n / every * each + e, here, 1, w);
          pin();
        }
      });
      // the next stage has landed, and every wave has this one's fragments in registers: its LDS may be overwritten
      wait_for_stage<(STAGES - 2) * kPieces>();
      const srd_t sa = la.begin(s + STAGES < steps), sb = lb.begin(s + STAGES < steps);
      const auto stage = [&](int n) {  // the n-th DMA piece of the stage that takes this one's place
        if (n < LoadA::kPer)
          la.piece(sa, freed, wave, n);
        else if (n < kPieces)
          lb.piece(sb, freed + kABytes, wave, n - LoadA::kPer);
      };
      if constexpr (SPLIT) {
        multiply(acc, now.a, rest.b, [&](int n) {
          constexpr int each = (kPieces + kProducts - 1) / kProducts;
#pragma unroll
          for (int e = 0; e < each; ++e) stage(n * each + e);
          if (n * each < kPieces) pin();
        });
        asm volatile("" ::: "memory");
        multiply(acc, rest.a, now.b, [&](int n) {  // now.a is free, now.b[k][j] after its last product
          const int k = n / (FM * FN), j = n / FM % FN, i = n % FM;
          if (j == 0) load_a(now, k, i, next, 0, w);
          if (i == FM - 1) load_b(now, k, j, next, 0, w);
          pin();
        });
      } else {
        multiply(acc, rest.a, rest.b, [&](int n) {
          deal<kLoads, kPieces>(n, [&](int m) { load(now, m, next, 0, w); }, stage);
        });
      }
    }
    // a workgroup may not end, nor its LDS be used otherwise, while pieces are in flight
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }

  // Waits until at most `YOUNGER` of this wave's DMA pieces are in flight and its LDS reads have returned, then for the other waves.
  template <int YOUNGER>
  static __device__ __forceinline__ void wait_for_stage() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(YOUNGER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // Hands the wave's part of the tile out in the order of memory: four columns of a row a lane, lanes along the row.  As it lies in
  // the registers, a store would touch 32 rows with 16 or 32 bytes each; through LDS (a strip of 32 rows at a time, a
  // region per wave) it writes whole rows of the part.  `by_row(row, col, v, old)` gets them; `old` is what `before` returned for the
  // place: a strip's are all asked for before the first of its stores, behind which the compiler would not move them.  With COLUMNS
  // `by_row` returns what it made of v, and `by_column(row, col, v)` gets four rows of a column of that a lane, lanes along the
  // column, for a result that is also stored transposed.
  // Lanes read there what other lanes of their wave wrote: LDS takes a wave's operations in order, lanes_meet() keeps the compiler to it.
  static __device__ __forceinline__ void lanes_meet() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
  }
  static constexpr int kPitch = FN * 32 + 4;
  static_assert(kWaves * 32 * kPitch * 4 <= kLds, "the strips fit where the stages were");
  template <bool COLUMNS, class B, class R, class C>
  static __device__ __forceinline__ void hand_out(const f32x16 (&acc)[FM][FN], lds_bytes lds, B before, R by_row, C by_column) {
    using quad_at = __attribute__((address_space(3))) f32x4*;
    using float_at = __attribute__((address_space(3))) const float*;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const lds_bytes mine = lds + wave * (32 * kPitch * 4);
    const int row0 = wave / WC * (BM / WR), col0 = wave % WC * (BN / WC);
    __syncthreads();  // the other waves are through with the stages
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<quad_at>(mine + ((lane & 31) * kPitch + j * 32 + g * 8 + (lane >> 5) * 4) * 4) = quad(acc[i][j], g);
      lanes_meet();
      constexpr int kQuads = FN * 8, kRows = 64 / kQuads;
      const int r = lane / kQuads, c = lane % kQuads * 4, rc = (lane & 7) * 4, cc = lane >> 3;
      f32x4 old[32 / kRows];
#pragma unroll
      for (int n = 0; n < 32 / kRows; ++n) old[n] = before(row0 + i * 32 + n * kRows + r, col0 + c);
#pragma unroll
      for (int n = 0; n < 32 / kRows; ++n) {
        const quad_at p = reinterpret_cast<quad_at>(mine + ((n * kRows + r) * kPitch + c) * 4);
        if constexpr (COLUMNS)
          *p = by_row(row0 + i * 32 + n * kRows + r, col0 + c, *p, old[n]);
        else
          by_row(row0 + i * 32 + n * kRows + r, col0 + c, *p, old[n]);
      }
      lanes_meet();
      if constexpr (COLUMNS) {
#pragma unroll
        for (int n = 0; n < FN * 4; ++n) {
          const float_at p = reinterpret_cast<float_at>(mine + (rc * kPitch + n * 8 + cc) * 4);
          by_column(row0 + i * 32 + rc, col0 + n * 8 + cc, f32x4{p[0], p[kPitch], p[2 * kPitch], p[3 * kPitch]});
        }
        lanes_meet();
      }
    }
  }

  struct Nothing {  // for results that are only written
    __device__ __forceinline__ f32x4 operator()(int, int) const { return f32x4{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ void operator()(int, int, f32x4) const {}
  };
  template <class R>
  static __device__ __forceinline__ void hand_out(const f32x16 (&acc)[FM][FN], lds_bytes lds, R by_row) {
    hand_out<false>(acc, lds, Nothing{}, [&](int r, int c, f32x4 v, f32x4) { by_row(r, c, v); }, Nothing{});
  }

  // columns 8 g .. 8 g + 3 from the lane's column of fragment j on
  static __device__ __forceinline__ f32x4 quad(const f32x16& v, int g) {
    return f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
  }
  // this lane's first row and column inside the tile
  static __device__ __forceinline__ int lane_row() {
    const int wave = uniform((int)(threadIdx.x >> 6));
    return wave / WC * (BM / WR) + (threadIdx.x & 31);
  }
  static __device__ __forceinline__ int lane_col() {
    const int wave = uniform((int)(threadIdx.x >> 6));
    return wave % WC * (BN / WC) + ((threadIdx.x >> 5) & 1) * 4;
  }
};

// Consecutive workgroups go to the 8 XCDs in turn.  Workgroup -> place in an order of which each XCD gets one contiguous run.
__device__ __forceinline__ int run_of_xcd(int id, int total) {
  const int q = total >> 3, r = total & 7, xcd = id & 7;
  return xcd * q + min(xcd, r) + (id >> 3);
}
// The t-th tile of an order that walks bands of `band` tile rows column by column, so that tiles that are near in it share rows of A and
// columns of B: those an XCD works on at a time, in its L2.
__device__ __forceinline__ void tile_in_bands(int t, int tiles_m, int tiles_n, int band, int& tm, int& tn) {
  const int per = band * tiles_n, b = t / per, in = t - b * per;
  const int high = min(band, tiles_m - b * band);
  tn = in / high;
  tm = b * band + in - tn * high;
}
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int band, int& tm, int& tn) {
  tile_in_bands(run_of_xcd(id, tiles_m * tiles_n), tiles_m, tiles_n, band, tm, tn);
}
// The same order of the tiles on and above the diagonal of n x n.
__device__ __forceinline__ void tile_in_triangle(int t, int n, int band, int& tm, int& tn) {
  int first = 0;  // tile row the band begins with; its columns begin there too
  for (;; first += band) {
    const int high = min(band, n - first), wide = n - first, corner = high * (high + 1) / 2;
    const int all = corner + (wide - high) * high;
    if (t >= all) {
      t -= all;
      continue;
    }
    if (t >= corner) {
      t -= corner;
      tn = first + high + t / high;
      tm = first + t % high;
    } else {
      int c = 0;
      while (t > c) t -= ++c;
      tn = first + c;
      tm = first + t;
    }
    return;
  }
}

template <bool SPLIT, bool BF16, bool AKM, bool BKM>
using Tile256 = TileProduct<256, 256, 2, 2, 2, SPLIT, BF16, AKM, BKM>;
template <bool SPLIT, bool BF16, bool AKM, bool BKM>
using Tile128 = TileProduct<128, 128, 2, 2, 2, SPLIT, BF16, AKM, BKM>;
template <bool SPLIT, bool BF16, bool AKM, bool BKM>
using Tile64 = TileProduct<64, 64, 2, 2, 4, SPLIT, BF16, AKM, BKM>;
// For launches of 128 tiles that leave compute units empty: a tile there has no neighbour that works while it waits, so it brings
// two waves per SIMD itself, and a third stage (96 KB) against the latency of memory (136 tiles of k = 2048 in float32: 36.5 us, with
// four waves and two stages 40; where all are taken, 4096 x 4096 x 2048, it is the slower one, 186 against 168).
template <bool SPLIT, bool BF16, bool AKM, bool BKM>
using Lone128 = TileProduct<128, 128, 2, 4, 3, SPLIT, BF16, AKM, BKM>;
// waves per SIMD that a kernel with this tile is compiled for
template <class P>
constexpr int kWavesPerSimd = P::BM == 256 ? 1 : 2;

// What a launch takes, in us: a stage of a tile where it shares its compute unit with nothing (`alone`) and where all places are taken
// (`full`; one 256 tile fits a compute unit, two of the others do), and what is around a tile's stages.  Measured on products
// from one tile up to 8192 x 8192; in float32 terms the tiles of 256, 128 and 64 reach 450, 420 and 280 TFLOP/s
// there, in bf16 1190, 1060 and 570, and 1024 x 1204 x 1024 in bf16 takes 26, 11 and 9 us.
struct TileTime {
  float alone, full, around;
};
inline TileTime tile_time(int tile, bool split) {
  return tile == 256   ? (split ? TileTime{1.7f, 2.4f, 8.f} : TileTime{1.1f, 1.8f, 8.f})
         : tile == 128 ? (split ? TileTime{0.58f, 1.28f, 3.f} : TileTime{0.61f, 1.09f, 3.f})
                       : (split ? TileTime{0.31f, 0.51f, 2.f} : TileTime{0.29f, 0.51f, 2.f});
}
inline long long tile_places(int tile) { return (long long)compute_units() * (tile == 256 ? 1 : 2); }
inline float launch_us(int tile, bool split, long long tiles, float steps) {
  const TileTime t = tile_time(tile, split);
  const long long places = tile_places(tile), rounds = tiles / places, rest = tiles % places;
  const float last = rest == 0 ? 0.f : t.around + steps * (rest <= places / 2 ? t.alone : t.full);
  return rounds * (t.around + steps * t.full) + last;
}
// The tile side with the least estimated time for a launch with that many tiles of 256, 128 and 64.
inline int choose_tile(long long t256, long long t128, long long t64, float steps, bool split) {
  const float a = launch_us(256, split, t256, steps), b = launch_us(128, split, t128, steps), c = launch_us(64, split, t64, steps);
  return a <= b && a <= c ? 256 : b <= c ? 128 : 64;
}

}  // namespace
}  // namespace mi
