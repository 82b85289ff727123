// linear_cross_entropy.hip -- softmax cross entropy of a linear classifier, forward and backward, without the logits in memory.
//
// Mathematics, for rows x_i (features), classes w_v with bias b_v, and labels y_i:
//   z_iv = x_i . w_v + b_v,   lse_i = log sum_v exp z_iv,   l_i = lse_i - z_i,y_i
//   q_iv = exp(z_iv - lse_i) - [v = y_i],   dx_i = g_i sum_v q_iv w_v,   dw_v = sum_i g_i q_iv x_i,   db_v = sum_i g_i q_iv
// The [rows, classes] logits are formed tile by tile on the matrix cores (tile_product.h) and die in registers: the forward
// keeps, per row and strip of columns, the running maximum and the sum of exponentials, and a second kernel joins the
// strips.  The backward forms the same tiles again, piece of the vocabulary by piece, turns them into q (16 bits or 2 x 16, up to 256 MB
// of it at a time: make_pieces) and multiplies q by the weights and by the features.
//
// Work: 2 R V D operations forward, 6 R V D backward (one third of it the logits' second time).  Bound by the matrix cores
// wherever R and V fill the chip: at 8192 x 4096 and 50021 classes in bf16 the forward's logits take 2.73 ms (1230 TFLOP/s), the
// backward's with q 3.20 ms, both gradients 5.67 ms (1183 TFLOP/s), these in four pieces.  By launches and the latency of a K loop where they do
// not: 1024 x 1024 and 81 classes in float32 take 59 us in seven launches.
//
// Types.  16-bit features and weights are multiplied as they are, in place.  float32 ones are laid out as hi + lo fp16 under one
// power-of-two scale per tensor (its largest finite magnitude lands in [2^14, 2^15), so hi + lo carry 22 bits for
// everything within 2^18 of it and lose one bit per halving below).  Maximum, sum, lse, loss and all accumulators are float32;
// the sum over rows is fp64.
// q is stored times 2^14 in 16 bits: in the features' type, for float32 as hi + lo fp16.  Against that, elements of q near 1 (a row's own
// class) keep 8, 11 or 22 bits, as many as the type of the gradients holds; in fp16 and float32 the smallest step is 2^-38, so a
// probability keeps all its bits down to 2^-28 (float32: 2^-17, one bit less per halving below) and is zero below 2^-39.  A gradient
// element whose terms are all that small, a class that no row is near, is off by as much: in float32 by 1e-5 of itself where its
// probabilities are 2^-28.  Gradients of single rows are kept apart from q as powers of two, so dx has these bits in every row; in dw
// rows are summed, and there a row's part is rounded at 2^-38 of the largest row gradient (weigh_rows).
//
// Rows with the ignored label are laid out as zeros, whatever they hold, and get q = 0.  A label that is neither ignored nor
// a class makes its row's loss and gradient NaN.
#include "common.h"
#include "tile_product.h"

#include <climits>
#include <cmath>

namespace mi {
namespace {

constexpr int kPad = 64;              // rows and classes of the operands' k axes are padded to this
constexpr int kMaxParts = 1024;       // workgroups of the maximum's pass
constexpr int kQExponent = 14;        // q is stored times 2^14: fp16 keeps probabilities down to 2^-38
constexpr float kQScale = 1 << kQExponent;
constexpr int kIgnored = -1, kOutside = -2;
constexpr int kIsNaN = 1 << 30;       // mark of a predicted class whose logit is NaN
constexpr int kNoClass = kIsNaN - 1;
constexpr int kElsewhere = 1 << 28;   // a row's largest logit is not among this lane's columns
constexpr float kLargest = 3.402823466e38f;
// What a call may hold, so that it stays below the logits that it does without (make_pieces)
constexpr size_t kMB = size_t(1) << 20;
constexpr size_t kWeightBytes = 128 * kMB;  // laid-out weights: up to this they are kept from the forward to the backward, more of
                                            // them are laid out in pieces of this, in either pass
constexpr size_t kQBytes = 64 * kMB, kMostQBytes = 256 * kMB;  // q of a piece: half of the float32 logits between these
constexpr size_t kSliceBytes = 32 * kMB;    // sums of the slices of one product, where it has several

__device__ __forceinline__ float to_float(uint16_t v, bool bf16) {
  return bf16 ? __uint_as_float((unsigned)v << 16) : (float)__builtin_bit_cast(_Float16, v);
}
template <int T>
__device__ __forceinline__ float load_as_float(const void* p, long long i) {
  if constexpr (T == MI_TYPE_F32)
    return static_cast<const float*>(p)[i];
  else
    return to_float(static_cast<const uint16_t*>(p)[i], T == MI_TYPE_BF16);
}
__device__ __forceinline__ uint16_t half_bits(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ uint16_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
template <int T>
__device__ __forceinline__ uint16_t round16(float v) {
  if constexpr (T == MI_TYPE_BF16)
    return bf16_bits(v);
  else
    return half_bits(v);
}
template <int T>
__device__ __forceinline__ void store_from_float(void* p, long long i, float v) {
  if constexpr (T == MI_TYPE_F32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = round16<T>(v);
}

// What a forward keeps for its backward and what both work with, all inside the caller's two buffers.
struct Plan {
  int rows, dim, classes;
  int rows_p, dim_p;        // padded to kPad
  bool split, copy_w;       // float32; weights laid out anew (float32, or 16-bit ones that the product cannot take in place)
  bool keep_w;              // the whole of them lies in `saved`; otherwise a piece at a time in the workspace, in both passes
  long long ld;             // words between rows of a laid-out operand
  size_t x_at, lab_at, lse_at, scalars_at, w_at, saved_bytes;
};

size_t up(size_t v) { return (v + 255) & ~size_t(255); }

Plan make_plan(int rows, int dim, int classes, int dtype, bool w_in_place) {
  Plan p;
  p.rows = rows, p.dim = dim, p.classes = classes;
  p.rows_p = (rows + kPad - 1) / kPad * kPad;
  p.dim_p = (dim + kPad - 1) / kPad * kPad;
  p.split = dtype == MI_TYPE_F32;
  p.copy_w = p.split || !w_in_place;
  p.ld = (long long)p.dim_p * (p.split ? 2 : 1);
  // 16-bit weights of padded dim that lie off 16 bytes are kept whatever their size: the workspace's size does not know where they lie
  p.keep_w = p.copy_w && ((size_t)classes * p.ld * 2 <= kWeightBytes || (!p.split && dim % kPad == 0));
  size_t at = 0;
  p.x_at = at, at = up(at + (size_t)p.rows_p * p.ld * 2);
  p.lab_at = at, at = up(at + (size_t)p.rows_p * 4);
  p.lse_at = at, at = up(at + (size_t)p.rows_p * 4);
  p.scalars_at = at, at = up(at + 64);
  // the weights come last: a backward whose weight lies on another alignment than the forward's finds the rest where it was left
  p.w_at = at, at = up(at + (p.keep_w ? (size_t)classes * p.ld * 2 : 0));
  p.saved_bytes = at;
  return p;
}

struct Scalars {        // at scalars_at
  int ex, ew;   // features and weights are their stored forms times 2^ex and 2^ew
  float count;  // rows that count, at least 1
  int done;     // workgroups of the join that are through
};
struct Sum {
  double loss;
  int rows;
};

// ---- laying out --------------------------------------------------------------------------------------------------------

// 14 - floor(log2 m); 0 for zero and for what is no number
__device__ __forceinline__ int exponent_of(float m) {
  if (!(m > 0.f) || m > kLargest) return 0;
  return min(max(14 - ilogbf(m), -120), 120);
}

// Four float32 from `p`: one load where the row starts on 16 bytes (`aligned`), else one each; zeros behind `left` elements.
__device__ __forceinline__ f32x4 four(const float* p, int left, bool aligned) {
  if (aligned && left >= 4) return *reinterpret_cast<const f32x4*>(p);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) v[e] = p[e];
  return v;
}

// Largest finite magnitude of the features that count (blocks below `x_blocks`) and of the weights (the others): one value per
// block.  A wave takes a row at a time.
template <class LABEL>
__global__ __launch_bounds__(256) void largest(const float* x, long long x_stride, const float* w, long long w_stride,
                                               const LABEL* labels, long long ignore, int rows, int classes, int dim,
                                               int x_blocks, float* parts) {
  const bool is_x = (int)blockIdx.x < x_blocks;
  const float* src = is_x ? x : w;
  const long long stride = is_x ? x_stride : w_stride;
  const int n = is_x ? rows : classes, blocks = is_x ? x_blocks : gridDim.x - x_blocks;
  const int b = is_x ? blockIdx.x : blockIdx.x - x_blocks;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const bool aligned = reinterpret_cast<uintptr_t>(src) % 16 == 0 && stride % 4 == 0;
  float m = 0.f;
  for (int r = b * 4 + wave; r < n; r += blocks * 4) {
    if (is_x && (long long)labels[r] == ignore) continue;
    const float* p = src + (long long)r * stride;
#pragma unroll 4
    for (int c = lane * 4; c < dim; c += 256) {
      const f32x4 v = four(p + c, dim - c, aligned);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = fabsf(v[e]);
        m = a <= kLargest ? fmaxf(m, a) : m;
      }
    }
  }
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  __shared__ float s[4];
  if (lane == 0) s[wave] = m;
  __syncthreads();
  if (threadIdx.x == 0) parts[blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

// One row in the product's form by one wave, a lane eight elements at a time.
template <bool SPLIT>
__device__ __forceinline__ void lay_out_row(const char* src, uint16_t* to, int dim, int dim_p, bool zero, float scale, int lane) {
  const bool aligned = reinterpret_cast<uintptr_t>(src) % 16 == 0;
#pragma unroll 2
  for (int c = lane * 8; c < dim_p; c += 512) {
    s16x8 hi = {0, 0, 0, 0, 0, 0, 0, 0}, lo = hi;
    if constexpr (SPLIT) {
      if (!zero) {
        const float* p = reinterpret_cast<const float*>(src) + c;
        const f32x4 v0 = four(p, dim - c, aligned), v1 = four(p + 4, dim - c - 4, aligned);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = (e < 4 ? v0[e & 3] : v1[e & 3]) * scale;
          const _Float16 h = (_Float16)v;
          hi[e] = __builtin_bit_cast(short, h);
          lo[e] = (short)half_bits(v - (float)h);
        }
      }
      uint16_t* at = to + (c >> 5) * 64 + (c & 31);
      *reinterpret_cast<s16x8*>(at) = hi;
      *reinterpret_cast<s16x8*>(at + 32) = lo;
    } else {
      const short* p = reinterpret_cast<const short*>(src) + c;
      if (!zero && aligned && c + 8 <= dim) {
        hi = *reinterpret_cast<const s16x8*>(p);
      } else if (!zero) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < dim) hi[e] = p[e];
      }
      *reinterpret_cast<s16x8*>(to + c) = hi;
    }
  }
}

// Features (rows_p rows; ignored ones and the padding are zeros), weights and labels in the product's form.  A wave takes one
// row at a time, a lane eight elements of it.  Bound by memory: 8192 x 4096 bf16 features in 25 us (5.3 TB/s).
template <int T, class LABEL>
__global__ __launch_bounds__(256) void lay_out(const void* x, long long x_stride, const void* w, long long w_stride,
                                               const LABEL* labels, long long ignore, int rows, int rows_p, int classes,
                                               int dim, int dim_p, uint16_t* xo, uint16_t* wo, int* lab, const float* parts,
                                               int x_parts, int w_parts, Scalars* sc) {
  constexpr bool split = T == MI_TYPE_F32;
  __shared__ int scales[2];  // their exponents
  if constexpr (split) {
    __shared__ float s[2][4];
    float mx = 0.f, mw = 0.f;
    for (int i = threadIdx.x; i < x_parts; i += 256) mx = fmaxf(mx, parts[i]);
    for (int i = threadIdx.x; i < w_parts; i += 256) mw = fmaxf(mw, parts[x_parts + i]);
    for (int d = 32; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d)), mw = fmaxf(mw, __shfl_xor(mw, d));
    if ((threadIdx.x & 63) == 0) s[0][threadIdx.x >> 6] = mx, s[1][threadIdx.x >> 6] = mw;
    __syncthreads();
    if (threadIdx.x < 2) {
      const float* v = s[threadIdx.x];
      scales[threadIdx.x] = exponent_of(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    sc->ex = split ? -scales[0] : 0, sc->ew = split ? -scales[1] : 0;
    sc->done = 0;
  }
  for (int i = blockIdx.x * 256 + threadIdx.x; i < rows_p; i += gridDim.x * 256) {
    const long long y = i < rows ? (long long)labels[i] : ignore;
    lab[i] = y == ignore ? kIgnored : (y >= 0 && y < classes) ? (int)y : kOutside;
  }
  const int total = rows_p + (wo != nullptr ? classes : 0);
  const int lane = threadIdx.x & 63, bytes = split ? 4 : 2;
  for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < total; r += gridDim.x * 4) {
    const bool is_x = r < rows_p;
    const int row = is_x ? r : r - rows_p;
    const bool zero = is_x && (row >= rows || (long long)labels[row] == ignore);
    const char* src = static_cast<const char*>(is_x ? x : w) + (long long)row * (is_x ? x_stride : w_stride) * bytes;
    lay_out_row<split>(src, (is_x ? xo : wo) + (long long)row * dim_p * (split ? 2 : 1), dim, dim_p, zero,
                       split ? ldexpf(1.f, scales[is_x ? 0 : 1]) : 1.f, lane);
  }
}

// A piece of the weights, under the scale that `lay_out` found.
template <int T>
__global__ __launch_bounds__(256) void lay_out_weights(const void* w, long long w_stride, int classes, int dim, int dim_p, uint16_t* wo,
                                                       const Scalars* sc) {
  constexpr bool split = T == MI_TYPE_F32;
  const float scale = split ? ldexpf(1.f, -sc->ew) : 1.f;
  for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < classes; r += gridDim.x * 4)
    lay_out_row<split>(static_cast<const char*>(w) + (long long)r * w_stride * (split ? 4 : 2),
                       wo + (long long)r * dim_p * (split ? 2 : 1), dim, dim_p, false, scale, threadIdx.x & 63);
}

// ---- forward -------------------------------------------------------------------------------------------------------------

struct Best {  // largest logit of a row and its lowest class; a NaN is the largest of all
  float v;
  int at;
};
__device__ __forceinline__ bool beats(const Best& a, const Best& b) {
  const bool na = a.v != a.v, nb = b.v != b.v;
  if (na != nb) return na;
  if (na || a.v == b.v) return a.at < b.at;
  return a.v > b.v;
}

// A lane's e-th of the 16 columns of a fragment
__device__ __forceinline__ constexpr int column(int e) { return (e >> 2) * 8 + (e & 3); }

// The lane's biases; columns behind the last class get -inf, which takes them out of maximum, sum and gradient.
template <class P, int T>
__device__ __forceinline__ void load_bias(float (&b)[P::FN][16], const void* bias, int class0, int col0, int classes) {
#pragma unroll
  for (int j = 0; j < P::FN; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int col = col0 + j * 32 + column(e);
      b[j][e] = col >= classes ? -INFINITY : bias != nullptr ? load_as_float<T>(bias, class0 + col) : 0.f;
    }
}

// One tile of logits -> per row and strip of columns (one strip per wave column) the maximum and the sum of exp(z - max).  Strips are
// as wide as a wave's part of the tile, so no wave waits for another; they cost 8 bytes a row for 32 to 128 logits.
template <class P, int T, bool PRED>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void logits_forward(Operand x, Operand w, const void* bias,
                                                                                const int* lab, const Scalars* sc, int rows,
                                                                                int rows_p, int class0, int classes, int tiles_m,
                                                                                int tiles_n, int steps, float2* part, int* best,
                                                                                float* target) {
  extern __shared__ char smem[];
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
  f32x16 acc[P::FM][P::FN];
  P::run(acc, x, w, tm * P::BM, tn * P::BN, 0, steps, (lds_bytes)smem);
  const int row0 = tm * P::BM + P::lane_row(), col0 = tn * P::BN + P::lane_col();
  const int scale = P::SPLIT ? sc->ex + sc->ew : 0;  // one step: neither factor's own scale may leave the range of a float
  float b[P::FN][16];
  load_bias<P, T>(b, bias, class0, col0, classes);
  const int strip = tn * P::WC + uniform((int)(threadIdx.x >> 6)) % P::WC;
#pragma unroll
  for (int i = 0; i < P::FM; ++i) {
    const int row = row0 + i * 32;
    const int y = row < rows ? lab[row] : kIgnored;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[i][j][e] = (P::SPLIT ? ldexpf(acc[i][j][e], scale) : acc[i][j][e]) + b[j][e];
        m = fmaxf(m, acc[i][j][e]);
      }
    const int in = y - class0 - col0;  // the label's class among the wave's columns, from the lane's first one on
    if (__any(in >= 0 && in < P::FN * 32)) {
#pragma unroll
      for (int j = 0; j < P::FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (in == j * 32 + column(e)) target[row] = acc[i][j][e];
    }
    m = fmaxf(m, __shfl_xor(m, 32));
    const float from = m == -INFINITY ? 0.f : m;  // a strip of classes that are all masked sums to zero
    float s = 0.f;
    int at = kElsewhere;  // from the last column down, so that the lowest one of the largest logit stays
#pragma unroll
    for (int j = P::FN - 1; j >= 0; --j)
#pragma unroll
      for (int e = 15; e >= 0; --e) {
        if constexpr (PRED) at = acc[i][j][e] == m ? j * 32 + column(e) : at;
        s += __expf(acc[i][j][e] - from);
      }
    s += __shfl_xor(s, 32);
    const bool writes = row < rows && (threadIdx.x & 32) == 0;
    if (writes) part[(long long)strip * rows_p + row] = make_float2(m, s);
    if constexpr (PRED) {
      at += class0 + col0;
      if (__any(s != s)) {  // the first NaN, where the row has one
        int first = kNoClass, inside = classes - col0;
        asm volatile("" : "+v"(inside));  // compared here only: kept for all rows, 64 results would fill the scalar registers
#pragma unroll
        for (int j = P::FN - 1; j >= 0; --j)
#pragma unroll
          for (int e = 15; e >= 0; --e)
            first = j * 32 + column(e) < inside && acc[i][j][e] != acc[i][j][e] ? class0 + col0 + j * 32 + column(e) : first;
        const int other = min(first, __shfl_xor(first, 32));
        if (other != kNoClass) at = other | kIsNaN;
      }
      at = min(at, __shfl_xor(at, 32));
      if (writes) best[(long long)strip * rows_p + row] = at;
    }
  }
}

// Joins the strips of 16 rows, 16 threads a row with eight strips on their way at a time; the workgroup that comes last sums the rows'
// losses in their order.  Bound by latency: 171 strips of 2000 rows with classes 9.1 us (two to four at a time 12.2).
__global__ __launch_bounds__(256) void join_strips(const float2* part, const int* best, int strips, const int* lab, int rows,
                                                   int rows_p, const float* target, float* lse, float* losses, int64_t* pred,
                                                   int mean, float* loss, Sum* sums, Scalars* sc) {
  __shared__ float2 s[4][16];
  __shared__ Best sb[4][16];
  __shared__ Sum total[16];
  __shared__ int last;
  const int r = threadIdx.x & 15, p0 = threadIdx.x >> 4, row = blockIdx.x * 16 + r;
  const auto merge = [](float2& a, float2 v) {
    const float n = fmaxf(a.x, v.x), from = n == -INFINITY ? 0.f : n;
    a = make_float2(n, a.y * __expf(a.x - from) + v.y * __expf(v.x - from));
  };
  float2 a = make_float2(-INFINITY, 0.f);
  Best b = {-INFINITY, kNoClass};
  if (row < rows) {
    constexpr int kTogether = 8;
    for (int from = p0; from < strips; from += 16 * kTogether) {
      float2 v[kTogether];
      int at[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        const int p = from + 16 * u;
        v[u] = p < strips ? part[(long long)p * rows_p + row] : make_float2(-INFINITY, 0.f);
        at[u] = best != nullptr && p < strips ? best[(long long)p * rows_p + row] : kNoClass;
      }
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        if (from + 16 * u >= strips) continue;
        merge(a, v[u]);
        const Best o = {at[u] & kIsNaN ? NAN : v[u].x, at[u] & ~kIsNaN};
        if (beats(o, b)) b = o;
      }
    }
  }
  // a wave's four threads of a row, then the four waves
#pragma unroll
  for (int d = 16; d < 64; d <<= 1) {
    const float2 v = make_float2(__shfl_xor(a.x, d), __shfl_xor(a.y, d));
    const Best o = {__shfl_xor(b.v, d), __shfl_xor(b.at, d)};
    merge(a, v);
    if (beats(o, b)) b = o;
  }
  if ((threadIdx.x & 48) == 0) s[threadIdx.x >> 6][r] = a, sb[threadIdx.x >> 6][r] = b;
  __syncthreads();
  if (p0 == 0) {
#pragma unroll
    for (int p = 1; p < 4; ++p) {
      merge(a, s[p][r]);
      if (beats(sb[p][r], b)) b = sb[p][r];
    }
    float mine = 0.f;
    int y = kIgnored;
    if (row < rows_p) {
      y = lab[row];
      const float l = y == kOutside ? NAN : a.x + logf(a.y);
      lse[row] = y == kIgnored ? INFINITY : l;  // exp(z - inf) = 0: an ignored row has no gradient
      if (row < rows) {
        if (y != kIgnored) mine = y == kOutside ? NAN : l - target[row];
        if (losses != nullptr) losses[row] = mine;
        if (pred != nullptr) pred[row] = y == kIgnored ? -1 : b.at;
      }
    }
    total[r] = {(double)mine, y != kIgnored};
  }
  if (loss == nullptr) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    Sum t = total[0];
    for (int i = 1; i < 16; ++i) t.loss += total[i].loss, t.rows += total[i].rows;
    __hip_atomic_store(&sums[blockIdx.x].loss, t.loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&sums[blockIdx.x].rows, t.rows, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(&sc->done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  Sum t = {0.0, 0};
  for (int i = threadIdx.x; i < (int)gridDim.x; i += 256) {
    t.loss += __hip_atomic_load(&sums[i].loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    t.rows += __hip_atomic_load(&sums[i].rows, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  for (int d = 32; d; d >>= 1) t.loss += __shfl_xor(t.loss, d), t.rows += __shfl_xor(t.rows, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) total[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 4; ++i) t.loss += total[i].loss, t.rows += total[i].rows;
  const int count = max(t.rows, 1);
  sc->count = (float)count;
  *loss = (float)(mean ? t.loss / (double)count : t.loss);
}

// ---- backward ------------------------------------------------------------------------------------------------------------

// A single row's gradient as m 2^(E + log2 w): E is the largest exponent of all rows, m in [1, 2), w a power of two up to 1 (0: the row's
// gradient is below 2^-149 of the largest).  q holds m only, so that a row of small gradient keeps its bits; dx gets w when its sums are done.
struct RowFactor {
  float m, w;
};
// What the finished sums are multiplied with.  A common gradient stays out of q.
struct Factor {
  const float* grad;  // of the loss; NULL: the rows' factors are in use
  const Scalars* sc;
  const RowFactor* rows;
  const int* exponent;  // E
  int mean;
  const int* lab;
};
// It and the operands' scales, as one number in [1, 2) and a power of two: their product alone may be no float where the result is one.
struct Undo {
  float m;
  int e;
  __device__ __forceinline__ float operator()(float v) const { return ldexpf(v * m, e); }
};
__device__ __forceinline__ Undo undo(const Factor& f, int e) {
  e -= kQExponent;
  if (f.grad == nullptr) return {1.f, e + *f.exponent};
  const float v = f.mean ? *f.grad / f.sc->count : *f.grad;
  if (!(fabsf(v) > 0.f && fabsf(v) <= kLargest)) return {v, 0};
  const int k = ilogbf(v);
  return {ldexpf(v, -k), k + e};
}

__global__ __launch_bounds__(1024) void row_factors(const float* grad, const int* lab, int rows, int rows_p, RowFactor* factors,
                                                    int* exponent) {
  const auto counts = [](float v) { return fabsf(v) > 0.f && fabsf(v) <= kLargest; };
  int most = INT_MIN;
  for (int i = threadIdx.x; i < rows; i += 1024)
    if (lab[i] != kIgnored && counts(grad[i])) most = max(most, ilogbf(grad[i]));
  for (int d = 32; d; d >>= 1) most = max(most, __shfl_xor(most, d));
  __shared__ int sm[16];
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = most;
  __syncthreads();
  for (int i = 0; i < 16; ++i) most = max(most, sm[i]);
  if (most == INT_MIN) most = 0;
  for (int i = threadIdx.x; i < rows_p; i += 1024) {
    RowFactor f = {0.f, 1.f};  // a row that does not count: zeros in q
    if (i < rows && lab[i] != kIgnored) {
      const float g = grad[i];
      const int e = counts(g) ? ilogbf(g) : most;
      f = {counts(g) ? ldexpf(g, -e) : g, ldexpf(1.f, e - most)};
    }
    factors[i] = f;
  }
  if (threadIdx.x == 0) *exponent = most;
}

// q times its rows' w, for q' x: there the rows are summed, and only their ratios count.  What falls below 2^-38 of the largest row's
// gradient is lost.  A wave takes a row; rows of the largest exponent stay as they are.
template <int T>
__global__ __launch_bounds__(256) void weigh_rows(const RowFactor* factors, int rows_p, int classes_p, uint16_t* q) {
  constexpr int words = T == MI_TYPE_F32 ? 2 : 1;
  for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows_p; r += gridDim.x * 4) {
    const float w = factors[r].w;
    if (w == 1.f) continue;
    uint16_t* row = q + (long long)r * classes_p * words;
    for (int c = (threadIdx.x & 63) * 8; c < classes_p; c += 512) {
      if constexpr (T == MI_TYPE_F32) {
        s16x8 *hi = reinterpret_cast<s16x8*>(row + (c >> 5) * 64 + (c & 31)), *lo = hi + 4;
        s16x8 h = *hi, l = *lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = (to_float((uint16_t)h[e], false) + to_float((uint16_t)l[e], false)) * w;
          const _Float16 f = (_Float16)v;
          h[e] = __builtin_bit_cast(short, f);
          l[e] = (short)half_bits(v - (float)f);
        }
        *hi = h, *lo = l;
      } else {
        s16x8* at = reinterpret_cast<s16x8*>(row + c);
        s16x8 h = *at;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = (short)round16<T>(to_float((uint16_t)h[e], T == MI_TYPE_BF16) * w);
        *at = h;
      }
    }
  }
}

// One tile of logits, again -> q times its row's m (`whole`: and w); column sums for the bias gradient, one strip per wave row.  Forming the
// logits a second time costs 2 R V D operations; keeping them would cost 8 R V bytes of traffic and 4 R V of memory.
template <class P, int T>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void logits_backward(Operand x, Operand w, const void* bias,
                                                                                 const int* lab, const float* lse,
                                                                                 const RowFactor* factors, int whole,
                                                                                 const Scalars* sc, int rows_p, int class0,
                                                                                 int classes, int classes_p, int tiles_m, int tiles_n,
                                                                                 int steps, uint16_t* q, float* sums) {
  extern __shared__ char smem[];
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
  f32x16 acc[P::FM][P::FN];
  P::run(acc, x, w, tm * P::BM, tn * P::BN, 0, steps, (lds_bytes)smem);
  const int row0 = tm * P::BM + P::lane_row(), col0 = tn * P::BN + P::lane_col();
  const int scale = P::SPLIT ? sc->ex + sc->ew : 0;  // one step: neither factor's own scale may leave the range of a float
  const long long ld = (long long)classes_p * (P::SPLIT ? 2 : 1);
  float b[P::FN][16], sum[P::FN][16];
  load_bias<P, T>(b, bias, class0, col0, classes);
#pragma unroll
  for (int j = 0; j < P::FN; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[j][e] = 0.f;
#pragma unroll
  for (int i = 0; i < P::FM; ++i) {
    const int row = row0 + i * 32;
    const bool in = row < rows_p;
    const int label = in ? lab[row] : kIgnored, y = label - class0 - col0;
    const bool ignored = label == kIgnored;
    const float l = in ? lse[row] : INFINITY;
    RowFactor g = {1.f, 1.f};
    if (factors != nullptr) {
      g = in ? factors[row] : RowFactor{0.f, 1.f};
      if (whole) g = {g.m * g.w, 1.f};
    }
    const float f = g.m * kQScale;
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        acc[i][j][e] = __expf((P::SPLIT ? ldexpf(acc[i][j][e], scale) : acc[i][j][e]) + b[j][e] - l) * f;
    if (__any(ignored)) {  // rows that do not count, also beside a bias or weight that is no number
#pragma unroll
      for (int j = 0; j < P::FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = ignored ? 0.f : acc[i][j][e];
    }
    if (__any(y >= 0 && y < P::FN * 32)) {
#pragma unroll
      for (int j = 0; j < P::FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] -= y == j * 32 + column(e) ? f : 0.f;
    }
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[j][e] = fmaf(acc[i][j][e], g.w, sum[j][e]);
  }
  P::hand_out(acc, (lds_bytes)smem, [&](int r, int c, f32x4 v) {
    const int row = tm * P::BM + r, col = tn * P::BN + c;
    if (row >= rows_p || col >= classes_p) return;
    s16x4 hi, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (P::SPLIT) {
        const _Float16 h = (_Float16)v[k];
        hi[k] = __builtin_bit_cast(short, h);
        lo[k] = (short)half_bits(v[k] - (float)h);
      } else {
        hi[k] = (short)round16<T>(v[k]);
      }
    }
    if constexpr (P::SPLIT) {
      uint16_t* at = q + row * ld + (col >> 5) * 64 + (col & 31);
      *reinterpret_cast<s16x4*>(at) = hi;
      *reinterpret_cast<s16x4*>(at + 32) = lo;
    } else {
      *reinterpret_cast<s16x4*>(q + row * ld + col) = hi;
    }
  });
  if (sums == nullptr) return;
  const int strip = tm * P::WR + uniform((int)(threadIdx.x >> 6)) / P::WC;
#pragma unroll
  for (int j = 0; j < P::FN; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float v = sum[j][e];
      for (int d = 1; d < 32; d <<= 1) v += __shfl_xor(v, d);
      const int col = col0 + j * 32 + column(e);
      if ((threadIdx.x & 31) == 0 && col < classes) sums[(long long)strip * classes_p + col] = v;
    }
}

// One of the two products q W and q' x.  With one slice of the k axis the result goes out rounded; otherwise the slices'
// float32 sums are kept (and added to those of the pieces before) and joined by join_slices in their order.
struct Gradient {
  Operand a, b;
  int rows, cols, tiles_m, tiles_n, steps, per_slice;
  void* out;
  float* slices;
  int add;
};
struct BiasGradient {
  const float* sums;
  int strips, classes, classes_p;
  void* out;
};

template <class P, int T, bool OF_WEIGHT>
__device__ __forceinline__ void gradient_tile(const Gradient& g, int id, const Factor& factor, lds_bytes lds) {
  const int tiles = g.tiles_m * g.tiles_n, slice = id / tiles;
  int tm, tn;
  tile_of(id - slice * tiles, g.tiles_m, g.tiles_n, 4, tm, tn);
  f32x16 acc[P::FM][P::FN];
  const int step0 = slice * g.per_slice;
  P::run(acc, g.a, g.b, tm * P::BM, tn * P::BN, step0, min(g.per_slice, g.steps - step0), lds);
  const Undo scaled = undo(factor, P::SPLIT ? (OF_WEIGHT ? factor.sc->ex : factor.sc->ew) : 0);
  const bool whole = (g.cols & 3) == 0;  // then every four columns of a lane are inside or outside together, and aligned
  P::hand_out(acc, lds, [&](int r0, int c0, f32x4 v) {
    const int row = tm * P::BM + r0, col = tn * P::BN + c0;
    if (row >= g.rows || col >= g.cols) return;
    if (!OF_WEIGHT && factor.rows != nullptr) v *= factor.rows[row].w;
    if (!OF_WEIGHT && factor.lab[row] == kIgnored) v = f32x4{0.f, 0.f, 0.f, 0.f};  // q is 0 there, but 0 times a weight may be NaN
    if (g.slices != nullptr) {
      float* at = g.slices + ((long long)slice * g.rows + row) * g.cols + col;
      if (whole) {
        if (g.add) v += *reinterpret_cast<const f32x4*>(at);
        *reinterpret_cast<f32x4*>(at) = v;
      } else {
        for (int r = 0; r < 4; ++r)
          if (col + r < g.cols) at[r] = g.add ? at[r] + v[r] : v[r];
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = scaled(v[r]);
    const long long at = (long long)row * g.cols + col;
    if (whole && T == MI_TYPE_F32) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(g.out) + at) = v;
    } else if (whole) {
      s16x4 h;
      for (int r = 0; r < 4; ++r) h[r] = (short)round16<T>(v[r]);
      *reinterpret_cast<s16x4*>(static_cast<uint16_t*>(g.out) + at) = h;
    } else {
      for (int r = 0; r < 4; ++r)
        if (col + r < g.cols) store_from_float<T>(g.out, at + r, v[r]);
    }
  });
}

// All gradients of a piece in one launch: the tiles of q W, those of q' x, and the bias' columns, 64 a workgroup.  Where each
// product alone would leave compute units empty, they fill up together (1024 x 1024 and 1204 classes in float32: 31 us).  With a gradient
// per row they go out in two, q being weighed in between.
template <class PX, class PW, int T>
__global__ __launch_bounds__(PX::kThreads, kWavesPerSimd<PX>) void gradients(Gradient x, Gradient w, BiasGradient bias, int x_blocks,
                                                                             int w_blocks, Factor factor) {
  extern __shared__ char smem[];
  const int id = blockIdx.x;
  if (id < x_blocks) {
    gradient_tile<PX, T, false>(x, id, factor, (lds_bytes)smem);
  } else if (id < x_blocks + w_blocks) {
    gradient_tile<PW, T, true>(w, id - x_blocks, factor, (lds_bytes)smem);
  } else {
    float* part = reinterpret_cast<float*>(smem);
    const int c = (id - x_blocks - w_blocks) * 64 + (threadIdx.x & 63), at = threadIdx.x >> 6;
    float v = 0.f;
    if (c < bias.classes)
#pragma unroll 8
      for (int s = at; s < bias.strips; s += PX::kThreads / 64) v += bias.sums[(long long)s * bias.classes_p + c];
    part[threadIdx.x] = v;
    __syncthreads();
    if (at != 0 || c >= bias.classes) return;
    for (int s = 1; s < PX::kThreads / 64; ++s) v += part[s * 64 + threadIdx.x];
    store_from_float<T>(bias.out, c, undo(factor, 0)(v));
  }
}

// Sums the slices of up to two gradients, four elements a thread.
struct Joined {
  const float* slices;
  int n;
  long long count;
  void* out;
};
template <int T>
__global__ __launch_bounds__(256) void join_slices(Joined x, Joined w, int x_blocks, Factor factor) {
  const bool is_x = (int)blockIdx.x < x_blocks;
  const Joined& j = is_x ? x : w;
  const int block = is_x ? blockIdx.x : blockIdx.x - x_blocks, blocks = is_x ? x_blocks : gridDim.x - x_blocks;
  const Undo scaled = undo(factor, T == MI_TYPE_F32 ? (is_x ? factor.sc->ew : factor.sc->ex) : 0);
  const bool whole = (j.count & 3) == 0;
  for (long long i = (block * 256LL + threadIdx.x) * 4; i < j.count; i += blocks * 1024LL) {
    const int left = j.count - i < 4 ? (int)(j.count - i) : 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < j.n; ++s) v += four(j.slices + s * j.count + i, left, whole);
    for (int r = 0; r < left; ++r) store_from_float<T>(j.out, i + r, scaled(v[r]));
  }
}

// ---- launching -----------------------------------------------------------------------------------------------------------

// The tile of a product whose k axis stays whole.
int tile_for(long long m, long long n, int k, bool split) {
  const auto tiles = [&](int t) { return (long long)ceil_div(m, t) * ceil_div(n, t); };
  return choose_tile(tiles(256), tiles(128), tiles(64), (float)k / (split ? 32 : 64), split);
}

// Tile of both gradients' products and the slices of their k axes: the least estimated time.  A slice is at least 8 stages long;
// a join costs a launch and its slices' way to memory and back (8 bytes an element at 4 TB/s), and slices stay within kSliceBytes.
struct Cut {
  int tile, x, w;
  float us;
};
Cut cut_for(const Plan& p, int width, bool x_joined) {
  const int step = p.split ? 32 : 64;
  const long long xs = width / step, ws = p.rows_p / step;
  Cut best = {64, 1, 1, INFINITY};
  for (int tile : {256, 128, 64}) {
    const long long xt = (long long)ceil_div(p.rows, tile) * ceil_div(p.dim, tile), wt = (long long)ceil_div(width, tile) * ceil_div(p.dim, tile);
    const TileTime t = tile_time(tile, p.split);
    const long long places = tile_places(tile);
    const long long x_bytes = 4LL * p.rows * p.dim, w_bytes = 4LL * width * p.dim, most = kSliceBytes;
    for (long long a = 1; a == 1 || (a <= 64 && xs / a >= 8 && a * x_bytes <= most); a *= 2)
      for (long long b = 1; b == 1 || (b <= 64 && ws / b >= 8 && b * w_bytes <= most); b *= 2) {
        const long long blocks = xt * a + wt * b, longest = xs / a > ws / b ? xs / a : ws / b;
        float us = t.around + longest * t.alone;
        if (blocks > places / 2) {  // the longest tile may begin when the others are half through
          const float busy = (float)(xt * xs + wt * ws) / places * t.full + (float)blocks / places * t.around + 0.5f * longest * t.full;
          us = us > busy ? us : busy;
        }
        const bool xj = x_joined || a > 1, wj = b > 1;
        if (xj || wj) us += 4.f;
        if (xj) us += 2e-6f * p.rows * p.dim * (a + 1);
        if (wj) us += 2e-6f * width * p.dim * (b + 1);
        if (us < best.us) best = {tile, (int)a, (int)b, us};
      }
  }
  return best;
}

struct Pieces {
  int n, width;  // of the vocabulary; width is a multiple of kPad
  Cut cut;
  bool x_joined;
  size_t q_at, sums_at, factors_at, x_at, w_at, weights_at, bytes;
};

// Classes of one piece of laid-out weights.
int weights_width(const Plan& p) {
  const long long most = (long long)(kWeightBytes / ((size_t)p.ld * 2)) / kPad * kPad;
  return most < kPad ? kPad : most < p.classes ? (int)most : ceil_div(p.classes, kPad) * kPad;
}
// Whether they come in pieces; the same for weights that turn out to be read in place.
bool weights_in_pieces(const Plan& p) {
  return (size_t)p.classes * p.ld * 2 > kWeightBytes && (p.split || p.dim % kPad != 0);
}

// The backward's workspace.  q of a piece takes at most half of what float32 logits of all classes would, and at most 256 MB (64 MB
// where half is less: smaller pieces would leave compute units empty); beside it lie at most an eighth of that in sums for the
// bias, 32 MB in slices of each product, dx in float32 where there are several pieces, and 128 MB of weights that are not kept (or 64
// of them).  Several pieces cost the adding up of dx and a launch's last, half-empty round each: 8192 x 4096 and 50021 classes in
// bf16 take 11.1 to 11.4 ms, 0.5 to 2 % more than in one piece of 0.82 GB; pieces of 55 MB cost 8192 x 1024 and 10000 classes 12 %, weights laid out
// twice 512 x 4096 and 50000 classes in float32 15 %.  Of the widths that are allowed, the one with the least estimated time.
Pieces make_pieces(const Plan& p) {
  Pieces c;
  const size_t words = p.split ? 2 : 1, logits = (size_t)p.rows_p * p.classes * 4;
  const size_t room = logits / 2 < kQBytes ? kQBytes : logits / 2 > kMostQBytes ? kMostQBytes : logits / 2;
  const long long all = ceil_div(p.classes, kPad) * kPad;
  long long most = (long long)(room / ((size_t)p.rows_p * words * 2)) / kPad * kPad;
  // nothing is gained where dx in float32, which several pieces need, is as large as what they save
  if ((size_t)p.rows_p * all * words * 2 <= room + (size_t)p.rows * p.dim * 4) most = all;
  if (weights_in_pieces(p) && most > weights_width(p)) most = weights_width(p);
  if (most < kPad) most = kPad;
  if (most >= p.classes) {
    c.width = (int)all;
    c.cut = cut_for(p, c.width, false);
  } else {
    const int fewest = ceil_div(p.classes, most);
    float least = INFINITY;
    for (int k = 0; k < 8; ++k) {  // equal pieces, and widths of whole tiles with what is left over
      const long long unit = most >= 1024 ? 256 : kPad, some = (most - most * (k - 4) / 8) / unit * unit;
      const long long width = k < 4 ? (long long)ceil_div(ceil_div(p.classes, fewest + k), kPad) * kPad : some < unit ? unit : some;
      const long long whole = p.classes / width, rest = p.classes - whole * width;
      const Cut cut = cut_for(p, (int)width, true);
      float us = 0.f;
      for (const long long n : {width, rest}) {
        if (n == 0) continue;
        const int tile = tile_for(p.rows_p, n, p.dim_p, p.split);
        const float steps = (float)p.dim_p / (p.split ? 32 : 64);
        const float one = launch_us(tile, p.split, (long long)ceil_div(p.rows_p, tile) * ceil_div(n, tile), steps) + 8.f +
                          (n == width ? cut.us : cut_for(p, ceil_div(n, kPad) * kPad, true).us);
        us += n == width ? one * whole : one;
      }
      if (us < least) least = us, c.width = (int)width, c.cut = cut;
    }
  }
  c.n = ceil_div(p.classes, c.width);
  c.x_joined = c.n > 1 || c.cut.x > 1;
  size_t at = 0;
  c.q_at = at, at = up(at + (size_t)p.rows_p * c.width * words * 2);
  c.sums_at = at, at = up(at + (size_t)(ceil_div(p.rows_p, 64) * 2) * c.width * 4);
  c.factors_at = at, at = up(at + (size_t)(p.rows_p + 1) * sizeof(RowFactor));  // E behind them
  c.x_at = at, at = up(at + (c.x_joined ? (size_t)c.cut.x * p.rows * p.dim * 4 : 0));
  c.w_at = at, at = up(at + (c.cut.w > 1 ? (size_t)c.cut.w * c.width * p.dim * 4 : 0));
  c.weights_at = at, at = up(at + (weights_in_pieces(p) ? (size_t)c.width * p.ld * 2 : 0));
  c.bytes = at;
  return c;
}

struct ForwardRoom {
  int width, tile, strips;  // classes, tile side and strips of a piece (of the weights where these are laid out in pieces)
  size_t parts_at, best_at, target_at, sums_at, max_at, weights_at, bytes;
};
ForwardRoom make_room(const Plan& p, bool with_pred) {
  ForwardRoom f;
  f.width = weights_in_pieces(p) ? weights_width(p) : p.classes;
  f.tile = tile_for(p.rows, f.width, p.dim_p, p.split);
  f.strips = ceil_div(f.width, f.tile) * 2;
  const size_t strips = (size_t)f.strips * ceil_div(p.classes, f.width);
  size_t at = 0;
  f.parts_at = at, at = up(at + strips * p.rows_p * sizeof(float2));
  f.best_at = at, at = up(at + (with_pred ? strips * p.rows_p * sizeof(int) : 0));
  f.target_at = at, at = up(at + (size_t)p.rows_p * 4);
  f.sums_at = at, at = up(at + (size_t)(p.rows_p / 16) * sizeof(Sum));
  f.max_at = at, at = up(at + (size_t)2 * kMaxParts * 4);
  f.weights_at = at, at = up(at + (weights_in_pieces(p) ? (size_t)f.width * p.ld * 2 : 0));
  f.bytes = at;
  return f;
}

template <class K>
void allow_lds(K kernel, unsigned bytes) {
  if (bytes > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

struct Call {
  const void *x, *weight, *bias, *labels;
  long long x_stride, w_stride, ignore;
  int labels_64, reduction;
  char *saved, *room;
  hipStream_t stream;
};

// The weights of the classes from class0 on as an operand of the products reads them: kept, a piece of them laid out here
// (at `room`), or where the caller has them.
template <int T>
Operand weights_of(const Plan& p, const Call& c, int class0, int classes, char* room) {
  if (p.keep_w) return {reinterpret_cast<uint16_t*>(c.saved + p.w_at) + (long long)class0 * p.ld, p.ld, classes, p.dim_p};
  constexpr int bytes = T == MI_TYPE_F32 ? 4 : 2;
  const char* w = static_cast<const char*>(c.weight) + (long long)class0 * c.w_stride * bytes;
  if (!p.copy_w) return {reinterpret_cast<const uint16_t*>(w), c.w_stride, classes, p.dim_p};
  const int most = 8 * compute_units(), grid = ceil_div(classes, 4) < most ? ceil_div(classes, 4) : most;
  uint16_t* to = reinterpret_cast<uint16_t*>(room);
  lay_out_weights<T><<<grid, 256, 0, c.stream>>>(w, c.w_stride, classes, p.dim, p.dim_p, to,
                                                reinterpret_cast<const Scalars*>(c.saved + p.scalars_at));
  return {to, p.ld, classes, p.dim_p};
}

template <int T, class LABEL>
void lay_out_all(const Plan& p, const Call& c, float* maxima) {
  const LABEL* labels = static_cast<const LABEL*>(c.labels);
  int xb = 0, wb = 0;
  if constexpr (T == MI_TYPE_F32) {
    xb = ceil_div(p.rows, 4), wb = ceil_div(p.classes, 4);
    xb = xb > kMaxParts ? kMaxParts : xb, wb = wb > kMaxParts ? kMaxParts : wb;
    largest<LABEL><<<xb + wb, 256, 0, c.stream>>>(static_cast<const float*>(c.x), c.x_stride,
                                                  static_cast<const float*>(c.weight), c.w_stride, labels, c.ignore, p.rows,
                                                  p.classes, p.dim, xb, maxima);
  }
  const int rows = p.rows_p + (p.keep_w ? p.classes : 0), most = 8 * compute_units();
  const int grid = ceil_div(rows, 4) < most ? ceil_div(rows, 4) : most;
  lay_out<T, LABEL><<<grid, 256, 0, c.stream>>>(
      c.x, c.x_stride, c.weight, c.w_stride, labels, c.ignore, p.rows, p.rows_p, p.classes, p.dim, p.dim_p,
      reinterpret_cast<uint16_t*>(c.saved + p.x_at), p.keep_w ? reinterpret_cast<uint16_t*>(c.saved + p.w_at) : nullptr,
      reinterpret_cast<int*>(c.saved + p.lab_at), maxima, xb, wb, reinterpret_cast<Scalars*>(c.saved + p.scalars_at));
}

template <class P, int T>
int launch_logits(const Plan& p, const Call& c, const ForwardRoom& f, bool with_pred, int class0, const Operand& w, int strip0) {
  const Operand x = {reinterpret_cast<uint16_t*>(c.saved + p.x_at), p.ld, p.rows_p, p.dim_p};
  const int tm = ceil_div(p.rows, P::BM), tn = ceil_div(w.rows, P::BN);
  const long long part0 = (long long)strip0 * p.rows_p;
  const auto kernel = with_pred ? logits_forward<P, T, true> : logits_forward<P, T, false>;
  allow_lds(kernel, P::kLds);
  kernel<<<tm * tn, P::kThreads, P::kLds, c.stream>>>(
      x, w, c.bias, reinterpret_cast<const int*>(c.saved + p.lab_at), reinterpret_cast<const Scalars*>(c.saved + p.scalars_at),
      p.rows, p.rows_p, class0, w.rows, tm, tn, p.dim_p / P::kStep, reinterpret_cast<float2*>(c.room + f.parts_at) + part0,
      with_pred ? reinterpret_cast<int*>(c.room + f.best_at) + part0 : nullptr, reinterpret_cast<float*>(c.room + f.target_at));
  return tn * P::WC;
}

template <int T>
int forward(const Plan& p, const Call& c, float* loss, float* losses, int64_t* pred) {
  constexpr bool split = T == MI_TYPE_F32, bf16 = T == MI_TYPE_BF16;
  const ForwardRoom f = make_room(p, pred != nullptr);
  float* maxima = reinterpret_cast<float*>(c.room + f.max_at);
  if (c.labels_64)
    lay_out_all<T, int64_t>(p, c, maxima);
  else
    lay_out_all<T, int32_t>(p, c, maxima);
  int strips = 0;
  for (int class0 = 0; class0 < p.classes; class0 += f.width) {
    const int classes = p.classes - class0 < f.width ? p.classes - class0 : f.width;
    const Operand w = weights_of<T>(p, c, class0, classes, c.room + f.weights_at);
    const bool with = pred != nullptr;
    strips += f.tile == 256   ? launch_logits<Tile256<split, bf16, false, false>, T>(p, c, f, with, class0, w, strips)
              : f.tile == 128 ? launch_logits<Tile128<split, bf16, false, false>, T>(p, c, f, with, class0, w, strips)
                              : launch_logits<Tile64<split, bf16, false, false>, T>(p, c, f, with, class0, w, strips);
  }
  join_strips<<<p.rows_p / 16, 256, 0, c.stream>>>(
      reinterpret_cast<const float2*>(c.room + f.parts_at), pred ? reinterpret_cast<const int*>(c.room + f.best_at) : nullptr,
      strips, reinterpret_cast<const int*>(c.saved + p.lab_at), p.rows, p.rows_p,
      reinterpret_cast<const float*>(c.room + f.target_at), reinterpret_cast<float*>(c.saved + p.lse_at), losses, pred,
      c.reduction == MI_REDUCTION_MEAN, loss, reinterpret_cast<Sum*>(c.room + f.sums_at),
      reinterpret_cast<Scalars*>(c.saved + p.scalars_at));
  return check_launch("mi_linear_cross_entropy_forward");
}

template <class P, int T>
int launch_q(const Plan& p, const Call& c, const Pieces& s, int class0, const Operand& w, int classes_p, bool want_bias, bool whole) {
  const Operand x = {reinterpret_cast<uint16_t*>(c.saved + p.x_at), p.ld, p.rows_p, p.dim_p};
  const int tm = ceil_div(p.rows_p, P::BM), tn = ceil_div(classes_p, P::BN);
  allow_lds(logits_backward<P, T>, P::kLds);
  logits_backward<P, T><<<tm * tn, P::kThreads, P::kLds, c.stream>>>(
      x, w, c.bias, reinterpret_cast<const int*>(c.saved + p.lab_at), reinterpret_cast<const float*>(c.saved + p.lse_at),
      c.reduction == MI_REDUCTION_NONE ? reinterpret_cast<const RowFactor*>(c.room + s.factors_at) : nullptr, whole,
      reinterpret_cast<const Scalars*>(c.saved + p.scalars_at), p.rows_p, class0, w.rows, classes_p, tm, tn,
      p.dim_p / P::kStep, reinterpret_cast<uint16_t*>(c.room + s.q_at),
      want_bias ? reinterpret_cast<float*>(c.room + s.sums_at) : nullptr);
  return tm * P::WR;
}

template <class PX, class PW, int T>
void launch_gradients(Gradient x, Gradient w, const BiasGradient& b, const Cut& cut, const Factor& factor, hipStream_t stream) {
  const auto blocks = [](Gradient& g, int slices) {
    if (g.out == nullptr) return 0;
    g.tiles_m = ceil_div(g.rows, PX::BM), g.tiles_n = ceil_div(g.cols, PX::BN), g.per_slice = ceil_div(g.steps, slices);
    return g.tiles_m * g.tiles_n * slices;
  };
  const int nx = blocks(x, cut.x), nw = blocks(w, cut.w), nb = b.out != nullptr ? ceil_div(b.classes, 64) : 0;
  if (nx + nw + nb == 0) return;
  allow_lds(gradients<PX, PW, T>, PX::kLds);
  gradients<PX, PW, T><<<nx + nw + nb, PX::kThreads, PX::kLds, stream>>>(x, w, b, nx, nw, factor);
}

template <int T>
int backward(const Plan& p, const Call& c, const float* grad, void* grad_x, void* grad_w, void* grad_b) {
  constexpr bool split = T == MI_TYPE_F32, bf16 = T == MI_TYPE_BF16;
  constexpr int words = split ? 2 : 1, step = split ? 32 : 64, out_bytes = T == MI_TYPE_F32 ? 4 : 2;
  const Pieces s = make_pieces(p);
  const Scalars* sc = reinterpret_cast<const Scalars*>(c.saved + p.scalars_at);
  RowFactor* factors = reinterpret_cast<RowFactor*>(c.room + s.factors_at);
  int* exponent = reinterpret_cast<int*>(factors + p.rows_p);
  const bool by_row = c.reduction == MI_REDUCTION_NONE, apart = by_row && grad_x != nullptr && grad_w != nullptr;
  if (by_row)
    row_factors<<<1, 1024, 0, c.stream>>>(grad, reinterpret_cast<const int*>(c.saved + p.lab_at), p.rows, p.rows_p, factors,
                                          exponent);
  const Factor factor = {by_row ? nullptr : grad, sc, by_row ? factors : nullptr, exponent, c.reduction == MI_REDUCTION_MEAN,
                         reinterpret_cast<const int*>(c.saved + p.lab_at)};
  uint16_t* q = reinterpret_cast<uint16_t*>(c.room + s.q_at);
  float* x_room = s.x_joined ? reinterpret_cast<float*>(c.room + s.x_at) : nullptr;
  float* w_room = s.cut.w > 1 ? reinterpret_cast<float*>(c.room + s.w_at) : nullptr;
  for (int k = 0; k < s.n; ++k) {
    const int class0 = k * s.width, classes = p.classes - class0 < s.width ? p.classes - class0 : s.width;
    const int classes_p = ceil_div(classes, kPad) * kPad;
    const int tile = tile_for(p.rows_p, classes_p, p.dim_p, split);
    const Operand weights = weights_of<T>(p, c, class0, classes, c.room + s.weights_at);
    const bool want_b = grad_b != nullptr, ends = k + 1 == s.n, whole = by_row && grad_x == nullptr;
    const int strips =
        tile == 256   ? launch_q<Tile256<split, bf16, false, false>, T>(p, c, s, class0, weights, classes_p, want_b, whole)
        : tile == 128 ? launch_q<Tile128<split, bf16, false, false>, T>(p, c, s, class0, weights, classes_p, want_b, whole)
                      : launch_q<Tile64<split, bf16, false, false>, T>(p, c, s, class0, weights, classes_p, want_b, whole);
    // every piece has the same slices of q W: a last, shorter piece leaves some of them empty
    const Gradient x = {{q, (long long)classes_p * words, p.rows_p, classes_p},
                        {weights.base, weights.ld, p.dim, classes},
                        p.rows, p.dim, 0, 0, classes_p / step, 0, grad_x, x_room, k > 0};
    void* w_out = grad_w == nullptr ? nullptr : static_cast<char*>(grad_w) + (size_t)class0 * p.dim * out_bytes;
    const Gradient w = {{q, (long long)classes_p * words, classes_p, p.rows_p},
                        {reinterpret_cast<uint16_t*>(c.saved + p.x_at), p.ld, p.dim, p.rows_p},
                        classes, p.dim, 0, 0, p.rows_p / step, 0, w_out, w_room, 0};
    const BiasGradient b = {reinterpret_cast<const float*>(c.room + s.sums_at), strips, classes, classes_p,
                            want_b ? static_cast<char*>(grad_b) + (size_t)class0 * out_bytes : nullptr};
    const auto multiply = [&](const Gradient& x, const Gradient& w, const BiasGradient& b) {
      if (s.cut.tile == 256)
        launch_gradients<Tile256<split, bf16, false, true>, Tile256<split, bf16, true, true>, T>(x, w, b, s.cut, factor, c.stream);
      else if (s.cut.tile == 128)
        launch_gradients<Tile128<split, bf16, false, true>, Tile128<split, bf16, true, true>, T>(x, w, b, s.cut, factor, c.stream);
      else
        launch_gradients<Tile64<split, bf16, false, true>, Tile64<split, bf16, true, true>, T>(x, w, b, s.cut, factor, c.stream);
    };
    if (apart) {
      multiply(x, Gradient{}, b);
      const int most = 8 * compute_units(), grid = ceil_div(p.rows_p, 4);
      weigh_rows<T><<<grid < most ? grid : most, 256, 0, c.stream>>>(factors, p.rows_p, classes_p, q);
      multiply(Gradient{}, w, BiasGradient{});
    } else {
      multiply(x, w, b);
    }
    const Joined jx = {x_room, s.cut.x, (long long)p.rows * p.dim, grad_x};
    const Joined jw = {w_room, s.cut.w, (long long)classes * p.dim, w_out};
    const int bx = ends && grad_x != nullptr && x_room != nullptr ? grid_for(jx.count / 4, 256) : 0;
    const int bw = grad_w != nullptr && w_room != nullptr ? grid_for(jw.count / 4, 256) : 0;
    if (bx + bw > 0) join_slices<T><<<bx + bw, 256, 0, c.stream>>>(jx, jw, bx, factor);
  }
  return check_launch("mi_linear_cross_entropy_backward");
}

// 16-bit weights are multiplied where they lie if k needs no padding and their rows start on 16 bytes.
bool in_place(const void* weight, long long stride, int dim, int dtype) {
  return dtype != MI_TYPE_F32 && dim % kPad == 0 && stride % 8 == 0 && reinterpret_cast<uintptr_t>(weight) % 16 == 0;
}

int check_sizes(int rows, int dim, int classes, int dtype) {
  MI_REQUIRE(rows >= 1 && rows <= (1 << 24), "linear_cross_entropy: %d rows, 1 to 2^24 are taken", rows);
  MI_REQUIRE(dim >= 1 && dim <= (1 << 20), "linear_cross_entropy: %d features, 1 to 2^20 are taken", dim);
  MI_REQUIRE(classes >= 1 && classes <= (1 << 24), "linear_cross_entropy: %d classes, 1 to 2^24 are taken", classes);
  MI_REQUIRE(dtype == MI_TYPE_F32 || dtype == MI_TYPE_F16 || dtype == MI_TYPE_BF16, "linear_cross_entropy: dtype %d", dtype);
  const long long r = ceil_div(rows, 64), d = ceil_div(dim, 64), c = ceil_div(classes, 64);
  // tiles of 64 x 64; where there are many, those of 128 or 256 are taken, and a launch has at most 2^32 threads, 256 a tile
  MI_REQUIRE(r * c < (1LL << 25) && r * d < (1LL << 25) && c * d < (1LL << 25),
             "linear_cross_entropy: %d rows x %d features x %d classes are more tiles than a launch takes", rows, dim, classes);
  return MI_OK;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_linear_cross_entropy_saved_bytes(int rows, int dim, int classes, int dtype, const void* weight,
                                           long long weight_stride) {
  if (check_sizes(rows, dim, classes, dtype) != MI_OK) return 0;
  return make_plan(rows, dim, classes, dtype, in_place(weight, weight_stride, dim, dtype)).saved_bytes;
}

size_t mi_linear_cross_entropy_workspace_bytes(int rows, int dim, int classes, int dtype, int pass) {
  if (check_sizes(rows, dim, classes, dtype) != MI_OK) return 0;
  const Plan p = make_plan(rows, dim, classes, dtype, true);
  return pass == MI_PASS_BACKWARD ? make_pieces(p).bytes : make_room(p, pass == MI_PASS_FORWARD_PRED).bytes;
}

static int check_call(const void* x, long long x_stride, const void* weight, long long weight_stride, const void* labels, int rows,
                      int dim, int classes, int dtype, int reduction, const void* saved, size_t saved_bytes,
                      const void* workspace, size_t workspace_bytes, size_t needed, Plan* plan) {
  if (const int rc = check_sizes(rows, dim, classes, dtype)) return rc;
  MI_REQUIRE(x != nullptr && weight != nullptr && labels != nullptr && saved != nullptr && workspace != nullptr,
             "linear_cross_entropy: null pointer");
  MI_REQUIRE(x_stride >= dim && weight_stride >= dim && weight_stride <= (1 << 22),
             "linear_cross_entropy: row strides %lld and %lld for %d features", x_stride, weight_stride, dim);
  MI_REQUIRE(reduction >= MI_REDUCTION_NONE && reduction <= MI_REDUCTION_SUM, "linear_cross_entropy: reduction %d", reduction);
  MI_REQUIRE(reinterpret_cast<uintptr_t>(saved) % 256 == 0 && reinterpret_cast<uintptr_t>(workspace) % 256 == 0,
             "linear_cross_entropy: buffers start on 256 bytes");
  *plan = make_plan(rows, dim, classes, dtype, in_place(weight, weight_stride, dim, dtype));
  if (saved_bytes < plan->saved_bytes || workspace_bytes < needed) {
    set_error("linear_cross_entropy: %zu bytes to keep and %zu of workspace are needed, %zu and %zu given", plan->saved_bytes,
              needed, saved_bytes, workspace_bytes);
    return MI_ERR_WORKSPACE;
  }
  return MI_OK;
}

int mi_linear_cross_entropy_forward(const void* x, long long x_stride, const void* weight, long long weight_stride,
                                    const void* bias, const void* labels, int labels_64, int rows, int dim, int classes, int dtype,
                                    long long ignore_index, int reduction, float* loss, int64_t* pred, void* saved,
                                    size_t saved_bytes, void* workspace, size_t workspace_bytes, mi_stream_t stream) {
  Plan p;
  if (const int rc = check_call(x, x_stride, weight, weight_stride, labels, rows, dim, classes, dtype, reduction, saved,
                                saved_bytes, workspace, workspace_bytes,
                                mi_linear_cross_entropy_workspace_bytes(rows, dim, classes, dtype,
                                                                        pred != nullptr ? MI_PASS_FORWARD_PRED : MI_PASS_FORWARD),
                                &p))
    return rc;
  MI_REQUIRE(loss != nullptr, "linear_cross_entropy: null pointer");
  begin_call();
  const Call c = {x, weight, bias, labels, x_stride, weight_stride, ignore_index, labels_64, reduction,
                  static_cast<char*>(saved), static_cast<char*>(workspace), as_stream(stream)};
  float* total = reduction == MI_REDUCTION_NONE ? nullptr : loss;
  float* each = reduction == MI_REDUCTION_NONE ? loss : nullptr;
  if (dtype == MI_TYPE_F32) return forward<MI_TYPE_F32>(p, c, total, each, pred);
  if (dtype == MI_TYPE_F16) return forward<MI_TYPE_F16>(p, c, total, each, pred);
  return forward<MI_TYPE_BF16>(p, c, total, each, pred);
}

int mi_linear_cross_entropy_backward(const float* grad_loss, const void* weight, long long weight_stride, const void* bias,
                                     int rows, int dim, int classes, int dtype, int reduction, void* grad_x, void* grad_weight,
                                     void* grad_bias, void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes,
                                     mi_stream_t stream) {
  Plan p;
  if (const int rc = check_call(saved, dim, weight, weight_stride, saved, rows, dim, classes, dtype, reduction, saved, saved_bytes,
                                workspace, workspace_bytes,
                                mi_linear_cross_entropy_workspace_bytes(rows, dim, classes, dtype, MI_PASS_BACKWARD), &p))
    return rc;
  MI_REQUIRE(grad_loss != nullptr, "linear_cross_entropy: null pointer");
  MI_REQUIRE((reinterpret_cast<uintptr_t>(grad_x) | reinterpret_cast<uintptr_t>(grad_weight)) % 16 == 0,
             "linear_cross_entropy: gradients start on 16 bytes");
  begin_call();
  const Call c = {nullptr, weight, bias, nullptr, dim, weight_stride, 0, 0, reduction,
                  static_cast<char*>(saved), static_cast<char*>(workspace), as_stream(stream)};
  if (dtype == MI_TYPE_F32) return backward<MI_TYPE_F32>(p, c, grad_loss, grad_x, grad_weight, grad_bias);
  if (dtype == MI_TYPE_F16) return backward<MI_TYPE_F16>(p, c, grad_loss, grad_x, grad_weight, grad_bias);
  return backward<MI_TYPE_BF16>(p, c, grad_loss, grad_x, grad_weight, grad_bias);
}

}  // extern "C"
