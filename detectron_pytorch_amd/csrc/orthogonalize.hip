// orthogonalize.hip -- orthogonalised updates of weight matrices by Newton-Schulz products, and the optimiser step around them.
//
// Mathematics, for a matrix G [m, n] with m <= n (a taller one is turned first and turned back at the end):
//   X_0 = G / max(|G|_F, eps);   A = X X',  C = a I + b A + c A A,  X <- C X     `steps` times
// X keeps the singular vectors of G and sends each singular value s to p(p(...p(s))) with p(s) = a s + b s^3 + c s^5, near 1 for
// all but the smallest.  The step of the optimiser around it:
//   M <- mu M + G,  U = G + mu M (nesterov) or M,  W <- (1 - lr wd) W - lr sqrt(max(1, rows / cols)) X(U)
//
// Two ways, by size:
//
// Short side up to 64 (and long side up to 16384): everything happens in the m x m space, in fp64.  A_0 = G G' / |G|^2 (the
// norm is its trace), Q = product of the C_k with A_k+1 = C_k A_k C_k, result Q G / |G|: three launches, of which the second
// is one workgroup per matrix with all its matrices in LDS.  A_0 has squared singular values, so float32 would not do.
// 64 x 256: 8 + 36 + 10 us; the middle one is bound by the fp64 matrix instructions of one compute unit (17 products, 10 tiles each
// on 4 SIMDs).
//
// Larger: the products run on the matrix cores (tile_product.h) with X, A and C as hi + lo fp16 times a power of two (22
// bits).  Their magnitudes are known -- |X| is bounded by the polynomial's largest value, which the host checks -- so no pass
// looks for a scale.  Products of plain fp16 would lose the small singular directions, whose noise the iteration
// amplifies by up to a^steps (485 for the usual a = 3.4445 and 5 steps).  Work per iteration: m^2 n for A (upper triangle), m^3
// for A A (upper triangle), 2 m^2 n for C X.  Where n is a multiple of m, two or three iterations share one pass over the
// long side: A_k+1 = C_k A_k C_k and Q = C_k+1 C_k are m x m products.  A pass in between renews A from X, which keeps the
// error at that of separate iterations (2.1e-6 to 5.2e-6 of the norm against 2.1e-6 to 4.9e-6 on Gaussian and strongly
// low-rank 256 x 1024; with all five in one pass 1e-4).
//
// Bound by the matrix cores on long matrices (1024 x 12544: Gram 45 + 9 us, C X 92 us, 285 TFLOP/s in float32 terms) and by the m x m
// products, which are too small for the chip: their 136 tiles leave nearly half of the compute units without one (1024: 16 us, 2048: 49
// to 52 us).
//
// Accumulators are float32; the norm is summed in fp64, so no gradient is too small or too large for it.
// All matrices of a call go through each stage in one launch: a workgroup finds its matrix in the call's table.
#include "common.h"
#include "tile_product.h"

#include <cmath>
#include <type_traits>

namespace mi {
namespace {

constexpr int kMany = 32;            // matrices of one table (it goes to the first kernel by value: 4 KB of kernel arguments)
constexpr float kScaleX = 4096.f;    // X is stored times this,
constexpr float kScaleA = 8192.f;    // A and C A times this,
constexpr float kScaleC = 1024.f;    // C and products of several C times this
constexpr double kMostX = 2.8;       // bounds of |X| and of |C_k ... C_1| that keep the stored forms below 65504
constexpr double kMostC = 60.0;
constexpr int kNormBlocks = 1024;    // workgroups that sum one matrix' squares, at most
constexpr int kNormElements = 8192;  // elements for which one more workgroup is worth its launch
constexpr int kNarrow = 64, kNarrowLong = 16384;
constexpr int kParts = 32;           // partial sums of A_0 in the fp64 way, at most

constexpr int kBand = 4;             // tile rows of a band of the tiles' order

enum { kA = 0, kC = 1, kQ = 2, kT = 3, kSquares = 4 };

struct Mat {
  const void* grad;
  void* out;         // the orthogonalised matrix, or the weights that are updated
  float* momentum;   // NULL: no momentum
  int m, n;          // m <= n, after turning
  int tall;          // the matrix itself is [n, m]
  int slices;        // of the sum over n in A (fp64 way: partial sums)
  float shape;       // sqrt(max(1, rows / cols))
  int pad;
  long long norm_at, x_at, y_at, square_at, square_bytes, parts_at;  // bytes into the workspace
};
struct Table {
  int count;
  int pad;
  Mat m[kMany];
};
struct Tiles {       // first workgroup of each matrix in a launch
  int first[kMany + 1];
};

struct Step {
  float a, b, c, eps;
  float mu, lr, decay;  // decay = 1 - lr * weight decay
  int nesterov, update, steps;
};

using f64x4 = __attribute__((ext_vector_type(4))) double;

__host__ __device__ inline int div_up(int a, int b) { return (a + b - 1) / b; }
__host__ __device__ inline int up32(int v) { return (v + 31) & ~31; }

__device__ __forceinline__ int find(const Tiles& t, int count, int block) {
  int i = 0;  // matrices without a workgroup in this launch are passed over
  while (i + 1 < count && block >= t.first[i + 1]) ++i;
  return i;
}

template <int T>
__device__ __forceinline__ float load_float(const void* p, long long i) {
  if constexpr (T == MI_TYPE_F32) return static_cast<const float*>(p)[i];
  if constexpr (T == MI_TYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  return __uint_as_float((unsigned)static_cast<const uint16_t*>(p)[i] << 16);
}
template <int T>
__device__ __forceinline__ void store_float(void* p, long long i, float v) {
  if constexpr (T == MI_TYPE_F32)
    static_cast<float*>(p)[i] = v;
  else if constexpr (T == MI_TYPE_F16)
    static_cast<_Float16*>(p)[i] = (_Float16)v;
  else
    static_cast<__bf16*>(p)[i] = (__bf16)v;
}
// four elements from i on; `whole`: all four exist and lie on their own alignment
template <int T>
__device__ __forceinline__ f32x4 load_four(const void* p, long long i, int left, bool whole) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (whole && left >= 4) {
    if constexpr (T == MI_TYPE_F32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
    const s16x4 h = *reinterpret_cast<const s16x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const short one = h[r];
      v[r] = load_float<T>(&one, 0);
    }
    return v;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < left) v[r] = load_float<T>(p, i + r);
  return v;
}
__device__ __forceinline__ bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// element (row, col) of a split matrix with `ld` elements a row: its hi word, the lo one is 32 words on
__device__ __forceinline__ long long split_at(int row, int col, int ld) {
  return (long long)row * ld * 2 + (col >> 5) * 64 + (col & 31);
}
__device__ __forceinline__ f32x4 get_split4(const uint16_t* p) {
  using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
  const f16x4 h = *reinterpret_cast<const f16x4*>(p), l = *reinterpret_cast<const f16x4*>(p + 32);
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = (float)h[r] + (float)l[r];
  return v;
}
__device__ __forceinline__ void put_split4(uint16_t* p, f32x4 v) {
  s16x4 h, l;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const _Float16 f = (_Float16)v[r];
    h[r] = __builtin_bit_cast(short, f);
    l[r] = __builtin_bit_cast(short, (_Float16)(v[r] - (float)f));
  }
  *reinterpret_cast<s16x4*>(p) = h;
  *reinterpret_cast<s16x4*>(p + 32) = l;
}

// The first kernel of a call has the table in its arguments and leaves it in the workspace for the others.
__device__ __forceinline__ void leave_table(const Table& t, char* ws) {
  if (blockIdx.x != 0) return;
  const int* from = reinterpret_cast<const int*>(&t);
  int* to = reinterpret_cast<int*>(ws);
  for (int i = threadIdx.x; i < (int)(sizeof(Table) / 4); i += blockDim.x) to[i] = from[i];
}
__device__ __forceinline__ const Table& table_of(const char* ws) { return *reinterpret_cast<const Table*>(ws); }
constexpr size_t kTableBytes = (sizeof(Table) + 255) / 256 * 256;

// The results of a lane, sixteen of them at at(e) where inside(e): the old weights are all asked for before the first result is written.
template <int T, class A, class I>
__device__ __forceinline__ void put_results(const Mat& q, const Step& s, A at, I inside, const float (&o)[16]) {
  float w[16] = {};
  if (s.update) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (inside(e)) w[e] = load_float<T>(q.out, at(e));
  }
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (inside(e)) store_float<T>(q.out, at(e), s.update ? fmaf(w[e], s.decay, -(s.lr * q.shape) * o[e]) : o[e]);
}
// Four of them on their alignment, with the old weights.
template <int T>
__device__ __forceinline__ void put_result4(const Mat& q, const Step& s, long long i, f32x4 o, f32x4 w) {
  if (s.update) {
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = fmaf(w[r], s.decay, -(s.lr * q.shape) * o[r]);  // one rounding of a weight's size, not three
  }
  if constexpr (T == MI_TYPE_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(q.out) + i) = o;
  } else {
    s16x4 h;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      short one;
      store_float<T>(&one, 0, o[r]);
      h[r] = one;
    }
    *reinterpret_cast<s16x4*>(static_cast<uint16_t*>(q.out) + i) = h;
  }
}

// ---- the fp64 way for a short side up to 64 ------------------------------------------------------------------------------

constexpr int kLdU = 66;  // LDS row of 64 columns of U, doubles
constexpr int kLdM = 66;  // LDS row of an m x m matrix

// 64 columns of U from column `col0` of the long side on, as doubles; rows and columns behind the matrix are zeros.  A thread's
// loads are all on their way before the first of them is used.
template <int T, bool ADVANCE>
__device__ __forceinline__ void load_columns(const Mat& q, const Step& s, int col0, double (*u)[kLdU]) {
  const int rows = (q.m + 15) & ~15, each = rows / 4;  // elements a thread
  const auto place = [&](int e, int& i, int& j) {
    const int id = e * 256 + threadIdx.x;
    j = q.tall ? id / rows : id & 63;
    i = q.tall ? id - j * rows : id >> 6;
    return i < q.m && col0 + j < q.n;
  };
  const auto at = [&](int i, int j) { return q.tall ? (long long)(col0 + j) * q.m + i : (long long)i * q.n + col0 + j; };
  float g[16], m[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    int i, j;
    g[e] = m[e] = 0.f;
    if (e < each && place(e, i, j)) {
      g[e] = load_float<T>(q.grad, at(i, j));
      if (q.momentum != nullptr) m[e] = q.momentum[at(i, j)];
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    if (e >= each) continue;
    int i, j;
    const bool inside = place(e, i, j);
    float v = g[e];
    if (q.momentum != nullptr) {
      if (ADVANCE) {
        m[e] = s.mu * m[e] + g[e];
        if (inside) q.momentum[at(i, j)] = m[e];
      }
      v = s.nesterov ? g[e] + s.mu * m[e] : m[e];
    }
    u[i][j] = (double)v;
  }
}

// tile `id` of the upper triangle of n x n tiles, row by row
__device__ __forceinline__ void triangle(int id, int n, int& i, int& j) {
  i = 0;
  while (id >= n - i) id -= n - i, ++i;
  j = i + id;
}
__host__ __device__ constexpr int triangle_tiles(int n) { return n * (n + 1) / 2; }

// Partial sums of U U': a workgroup adds up its share of 64-column chunks, each wave its tiles of the upper triangle (16 x 16;
// a lane holds column l & 15, rows (l >> 4) + 4 r) and writes them as they lie in its registers.
template <int T>
__global__ __launch_bounds__(256) void narrow_gram(Table t, Tiles tiles, Step s, char* ws) {
  leave_table(t, ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  __shared__ double u[kNarrow][kLdU];
  const int part = blockIdx.x - tiles.first[k], chunks = div_up(q.n, 64), each = div_up(chunks, q.slices);
  const int nt = div_up(q.m, 16), total = triangle_tiles(nt), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f64x4 acc[3] = {};
  for (int c = part * each; c < min(chunks, (part + 1) * each); ++c) {
    __syncthreads();
    load_columns<T, true>(q, s, c * 64, u);
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      const int id = wave + x * 4;
      if (id >= total) continue;
      int i, j;
      triangle(id, nt, i, j);
      const double *a = &u[i * 16 + (lane & 15)][lane >> 4], *b = &u[j * 16 + (lane & 15)][lane >> 4];
#pragma unroll
      for (int p = 0; p < 64; p += 4) acc[x] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[p], b[p], acc[x], 0, 0, 0);
    }
  }
  f64x4* out = reinterpret_cast<f64x4*>(ws + q.parts_at) + (long long)part * total * 64;
#pragma unroll
  for (int x = 0; x < 3; ++x)
    if (wave + x * 4 < total) out[(wave + x * 4) * 64 + lane] = acc[x];
}

// Symmetric product of commuting symmetric matrices in LDS, one tile of the upper triangle per wave; `put(i, j, v)` gets each
// element of them.  Two accumulators: a product of this type waits for the one it adds to.
template <int NT, class F>
__device__ __forceinline__ void narrow_product(const double (*x)[kLdM], const double (*y)[kLdM], F put) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave >= triangle_tiles(NT)) return;
  int i, j;
  triangle(wave, NT, i, j);
  const double *a = &x[i * 16 + (lane & 15)][lane >> 4], *b = &y[j * 16 + (lane & 15)][lane >> 4];
  double u[NT * 4], v[NT * 4];
#pragma unroll
  for (int k = 0; k < NT * 4; ++k) u[k] = a[4 * k], v[k] = b[4 * k];
  f64x4 even = {}, odd = {};
#pragma unroll
  for (int k = 0; k < NT * 4; k += 2) {
    even = __builtin_amdgcn_mfma_f64_16x16x4f64(u[k], v[k], even, 0, 0, 0);
    odd = __builtin_amdgcn_mfma_f64_16x16x4f64(u[k + 1], v[k + 1], odd, 0, 0, 0);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) put(i * 16 + (lane >> 4) + 4 * r, j * 16 + (lane & 15), even[r] + odd[r]);
}

// Q / max(|G|, eps) of one matrix per workgroup.
constexpr int kPolyThreads = 640;  // ten tiles of 16 x 16 make the upper triangle of 64 x 64
template <int NT>
__device__ __forceinline__ void polynomial_of(const Mat& q, const Step& s, char* ws, char* smem) {
  using Square = double (*)[kLdM];
  constexpr int nt = NT, total = triangle_tiles(NT);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t bytes = sizeof(double) * kNarrow * kLdM;
  Square a = reinterpret_cast<Square>(smem), c = reinterpret_cast<Square>(smem + bytes),
         p = reinterpret_cast<Square>(smem + 2 * bytes), t = reinterpret_cast<Square>(smem + 3 * bytes);
  const f64x4* parts = reinterpret_cast<const f64x4*>(ws + q.parts_at);
  if (wave < total) {
    f64x4 v = {};
#pragma unroll 8
    for (int k = 0; k < q.slices; ++k) v += parts[((long long)k * total + wave) * 64 + lane];
    int i, j;
    triangle(wave, nt, i, j);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = i * 16 + (lane >> 4) + 4 * r, col = j * 16 + (lane & 15);
      a[row][col] = v[r];
      if (i != j) a[col][row] = v[r];
    }
  }
  __syncthreads();
  double trace = 0;
  for (int i = 0; i < q.m; ++i) trace += a[i][i];
  const double length = sqrt(trace);
  const double inv = 1.0 / (length < (double)s.eps ? (double)s.eps : length);  // not fmax: a NaN stays one
  __syncthreads();
  for (int e = threadIdx.x; e < nt * 16 * nt * 16; e += kPolyThreads) a[e / (nt * 16)][e % (nt * 16)] *= inv * inv;
  __syncthreads();
  const auto both = [](Square to) {
    return [to](int i, int j, double v) {
      to[i][j] = v;
      if ((i >> 4) != (j >> 4)) to[j][i] = v;
    };
  };
  for (int k = 0; k < s.steps; ++k) {
    const Square poly = k == 0 ? p : c;
    const auto put = both(poly);
    narrow_product<NT>(a, a, [&](int i, int j, double v) {
      put(i, j, (i == j ? (double)s.a : 0.0) + (double)s.b * a[i][j] + (double)s.c * v);
    });
    __syncthreads();
    if (k > 0) {
      narrow_product<NT>(c, p, both(t));
      __syncthreads();
      const Square old = p;
      p = t, t = old;
    }
    if (k + 1 == s.steps) break;
    const Square now = k == 0 ? p : c;
    narrow_product<NT>(now, a, both(t));
    __syncthreads();
    narrow_product<NT>(t, now, both(a));
    __syncthreads();
  }
  double* out = reinterpret_cast<double*>(ws + q.square_at);
  for (int e = threadIdx.x; e < nt * 16 * nt * 16; e += kPolyThreads) out[e] = p[e / (nt * 16)][e % (nt * 16)] * inv;
}

__global__ __launch_bounds__(kPolyThreads) void narrow_polynomial(Step s, char* ws) {
  const Mat& q = table_of(ws).m[blockIdx.x];
  extern __shared__ char smem[];
  if (q.m <= 16)
    polynomial_of<1>(q, s, ws, smem);
  else if (q.m <= 32)
    polynomial_of<2>(q, s, ws, smem);
  else if (q.m <= 48)
    polynomial_of<3>(q, s, ws, smem);
  else
    polynomial_of<4>(q, s, ws, smem);
}

// Q U, 64 columns per workgroup, 16 of them a wave.
template <int T, int NT>
__device__ __forceinline__ void apply_of(const Mat& q, const Step& s, char* ws, int col0, double (*u)[kLdU], double (*w)[kLdM]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j0 = wave * 16;
  const double* in = reinterpret_cast<const double*>(ws + q.square_at);
  double v[NT * NT];  // asked for before the columns, whose loads wait for nothing of it
#pragma unroll
  for (int k = 0; k < NT * NT; ++k) v[k] = in[k * 256 + threadIdx.x];
  load_columns<T, false>(q, s, col0, u);
#pragma unroll
  for (int k = 0; k < NT * NT; ++k) {
    const int e = k * 256 + threadIdx.x;
    w[e / (NT * 16)][e % (NT * 16)] = v[k];
  }
  __syncthreads();
  double y[NT * 4];
#pragma unroll
  for (int k = 0; k < NT * 4; ++k) y[k] = u[4 * k + (lane >> 4)][j0 + (lane & 15)];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    double x[NT * 4];
#pragma unroll
    for (int k = 0; k < NT * 4; ++k) x[k] = w[4 * k + (lane >> 4)][i * 16 + (lane & 15)];
    // the matrix' own order of elements decides which side lies along the lanes; Q is symmetric
    f64x4 even = {}, odd = {};
    if (q.tall) {
#pragma unroll
      for (int k = 0; k < NT * 4; k += 2) {
        even = __builtin_amdgcn_mfma_f64_16x16x4f64(y[k], x[k], even, 0, 0, 0);
        odd = __builtin_amdgcn_mfma_f64_16x16x4f64(y[k + 1], x[k + 1], odd, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NT * 4; k += 2) {
        even = __builtin_amdgcn_mfma_f64_16x16x4f64(x[k], y[k], even, 0, 0, 0);
        odd = __builtin_amdgcn_mfma_f64_16x16x4f64(x[k + 1], y[k + 1], odd, 0, 0, 0);
      }
    }
    const auto row = [&](int r) { return i * 16 + (q.tall ? lane & 15 : (lane >> 4) + 4 * r); };
    const auto col = [&](int r) { return col0 + j0 + (q.tall ? (lane >> 4) + 4 * r : lane & 15); };
    float o[16];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (float)(even[r] + odd[r]);
    put_results<T>(q, s, [&](int r) { return q.tall ? (long long)col(r) * q.m + row(r) : (long long)row(r) * q.n + col(r); },
                   [&](int r) { return r < 4 && row(r) < q.m && col(r) < q.n; }, o);
  }
}

template <int T>
__global__ __launch_bounds__(256) void narrow_apply(Tiles tiles, Step s, char* ws) {
  const Table& t = table_of(ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  __shared__ double u[kNarrow][kLdU], w[kNarrow][kLdM];
  const int col0 = (blockIdx.x - tiles.first[k]) * 64;
  if (q.m <= 16)
    apply_of<T, 1>(q, s, ws, col0, u, w);
  else if (q.m <= 32)
    apply_of<T, 2>(q, s, ws, col0, u, w);
  else if (q.m <= 48)
    apply_of<T, 3>(q, s, ws, col0, u, w);
  else
    apply_of<T, 4>(q, s, ws, col0, u, w);
}

// ---- larger matrices: momentum, norm, X_0 --------------------------------------------------------------------------------

// M <- mu M + G, and the squares of U: one fp64 sum per workgroup.  Bound by memory: 20.9 M float32 elements in 44 us (5.7 TB/s).
template <int T>
__global__ __launch_bounds__(256) void momentum_and_norm(Table t, Tiles tiles, Step s, char* ws) {
  leave_table(t, ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int block = blockIdx.x - tiles.first[k], blocks = tiles.first[k + 1] - tiles.first[k];
  const long long n = (long long)q.m * q.n;
  const bool whole = aligned16(q.grad) && aligned16(q.momentum);
  double sum = 0;
#pragma unroll 2
  for (long long i = (block * 256LL + threadIdx.x) * 4; i < n; i += blocks * 1024LL) {
    const int left = n - i < 4 ? (int)(n - i) : 4;
    f32x4 u = load_four<T>(q.grad, i, left, whole);
    if (q.momentum != nullptr) {
      const f32x4 m = s.mu * load_four<MI_TYPE_F32>(q.momentum, i, left, whole) + u;
      if (whole && left == 4) {
        *reinterpret_cast<f32x4*>(q.momentum + i) = m;
      } else {
        for (int r = 0; r < left; ++r) q.momentum[i + r] = m[r];
      }
      u = s.nesterov ? u + s.mu * m : m;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) sum += r < left ? (double)u[r] * (double)u[r] : 0.0;
  }
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  __shared__ double part[4];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) reinterpret_cast<double*>(ws + q.norm_at)[block] = part[0] + part[1] + part[2] + part[3];
}

// X_0, 64 x 64 of the given matrix per workgroup, turned on the way if it is tall.  Bound by memory: 20.9 M elements in 48 us (5.2 TB/s).
template <int T>
__global__ __launch_bounds__(256) void normalize(Tiles tiles, Tiles norm, Step s, char* ws) {
  const Table& t = table_of(ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int rows = q.tall ? q.n : q.m, cols = q.tall ? q.m : q.n;
  const int tiles_c = div_up(cols, 64), tile = blockIdx.x - tiles.first[k];
  const int row0 = tile / tiles_c * 64, col0 = tile % tiles_c * 64;
  __shared__ double part[4];
  __shared__ float buf[64][68];
  const bool whole = aligned16(q.grad) && aligned16(q.momentum) && cols % 4 == 0;
  f32x4 u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = row0 + e * 16 + (threadIdx.x >> 4), c = col0 + (threadIdx.x & 15) * 4;
    u[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r < rows && c < cols) {
      const long long i = (long long)r * cols + c;
      const int left = cols - c < 4 ? cols - c : 4;
      u[e] = load_four<T>(q.grad, i, left, whole);
      if (q.momentum != nullptr) {
        const f32x4 m = load_four<MI_TYPE_F32>(q.momentum, i, left, whole);
        u[e] = s.nesterov ? u[e] + s.mu * m : m;
      }
    }
  }
  const double* sums = reinterpret_cast<const double*>(ws + q.norm_at);
  double sum = 0;
  for (int i = threadIdx.x; i < norm.first[k + 1] - norm.first[k]; i += 256) sum += sums[i];
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double length = sqrt(part[0] + part[1] + part[2] + part[3]);
  const double inv = (double)kScaleX / (length < (double)s.eps ? (double)s.eps : length);  // not fmax: a NaN stays one
  uint16_t* x = reinterpret_cast<uint16_t*>(ws + q.x_at);
  const int ld = up32(q.n);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = e * 16 + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 4;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      u[e][v] = (float)((double)u[e][v] * inv);
      if (q.tall) buf[c + v][r] = u[e][v];
    }
    if (!q.tall && row0 + r < q.m && col0 + c < ld) put_split4(x + split_at(row0 + r, col0 + c, ld), u[e]);
  }
  if (!q.tall) return;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = e * 16 + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 4;
    if (col0 + r < q.m && row0 + c < ld)
      put_split4(x + split_at(col0 + r, row0 + c, ld), *reinterpret_cast<const f32x4*>(&buf[r][c]));
  }
}

// ---- larger matrices: the products ---------------------------------------------------------------------------------------

// A symmetric result's tile of the upper triangle, on both sides (the padding of a row lies in its upper half; both sides are
// the same to the last bit off the diagonal's tiles).  `finish(row, col,
// v, old)` is what is still done to four columns of a row, `before(row, col)` what it wants to know of the place.
template <class P, class B, class F>
__device__ __forceinline__ void put_symmetric(f32x16 (&acc)[P::FM][P::FN], lds_bytes lds, uint16_t* out, int m, int ti, int tj,
                                              B before, F finish) {
  const int ld = up32(m);
  const auto asked = [&](int r, int c) {
    const int row = ti * P::BM + r, col = tj * P::BN + c;
    return row < m && col < ld ? before(row, col) : f32x4{0.f, 0.f, 0.f, 0.f};
  };
  const auto by_row = [&](int r, int c, f32x4 v, f32x4 old) {
    const int row = ti * P::BM + r, col = tj * P::BN + c;
    if (row >= m || col >= ld) return v;
    v = finish(row, col, v, old);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k >= m) v[k] = 0.f;
    put_split4(out + split_at(row, col, ld), v);
    return v;
  };
  if (ti == tj) {
    P::template hand_out<false>(acc, lds, asked, by_row, typename P::Nothing{});
    return;
  }
  // rows of the transposed tile: ti is not the last tile, so its 4 rows are all inside
  P::template hand_out<true>(acc, lds, asked, by_row, [&](int r, int c, f32x4 v) {
    const int row = ti * P::BM + r, col = tj * P::BN + c;
    if (col < m) put_split4(out + split_at(col, row, ld), v);
  });
}

// A = X X': one tile of the upper triangle and one slice of the sum over n.  With one slice the tile is written as it is; slices leave
// their float32 sums in the workspace, as they lie in the registers, for join_gram.  (Having the slice that comes last join
// them saves that launch, but each workgroup then writes its L2 back first: 241 us instead of 70 + 8 at 1024 x 12544, both before
// the tiles' order of today.)
template <class P>
__device__ __forceinline__ f32x4* slice_sums(const Mat& q, char* ws, int per, int tile, int slice, int i, int j, int g) {
  return reinterpret_cast<f32x4*>(ws + q.parts_at) +
         (((long long)slice * per + tile) * (P::FM * P::FN * 4) + (i * P::FN + j) * 4 + g) * P::kThreads + threadIdx.x;
}
constexpr float kGramFactor = kScaleA / (kScaleX * kScaleX);
template <class P>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void gram(Tiles tiles, char* ws, int flip) {
  extern __shared__ char smem[];
  const Table& t = table_of(ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int nt = div_up(q.m, P::BM), per = triangle_tiles(nt);
  const int id = run_of_xcd(blockIdx.x - tiles.first[k], per * q.slices), slice = id / per, tile = id - slice * per;
  int ti, tj;
  tile_in_triangle(tile, nt, kBand, ti, tj);
  const int ld = up32(q.n), steps = ld / 32, each = div_up(steps, q.slices), step0 = slice * each;
  const Operand x = {reinterpret_cast<const uint16_t*>(ws + (flip ? q.y_at : q.x_at)), (long long)ld * 2, q.m, ld};
  f32x16 acc[P::FM][P::FN];
  P::run(acc, x, x, ti * P::BM, tj * P::BN, step0, min(each, steps - step0), (lds_bytes)smem);
  if (q.slices == 1) {
    put_symmetric<P>(acc, (lds_bytes)smem, reinterpret_cast<uint16_t*>(ws + q.square_at), q.m, ti, tj,
                     [](int, int) { return f32x4{0.f, 0.f, 0.f, 0.f}; },
                     [](int, int, f32x4 v, f32x4) { return v * kGramFactor; });
    return;
  }
#pragma unroll
  for (int i = 0; i < P::FM; ++i)
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) *slice_sums<P>(q, ws, per, tile, slice, i, j, g) = P::quad(acc[i][j], g);
}

// Adds the slices up in their order, one 32 x 32 fragment of each wave of a tile per workgroup, and hands it out as a 64 tile's wave
// hands out its one (stored as it lies in the registers: 10.9 us at 1024 x 12544, so 9.3, 3.5 TB/s of slices).
template <class P>
__global__ __launch_bounds__(P::kThreads) void join_gram(Tiles tiles, char* ws) {
  using One = Tile64<true, false, false, false>;
  __shared__ char smem[P::kWaves * 32 * One::kPitch * 4];
  const Table& t = table_of(ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int nt = div_up(q.m, P::BM), per = triangle_tiles(nt), ld = up32(q.m);
  const int id = blockIdx.x - tiles.first[k], tile = id / (P::FM * P::FN), f = id % (P::FM * P::FN), i = f / P::FN, j = f % P::FN;
  int ti, tj;
  tile_in_triangle(tile, nt, kBand, ti, tj);
  f32x16 acc[1][1] = {};
#pragma unroll 2
  for (int s = 0; s < q.slices; ++s)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = *slice_sums<P>(q, ws, per, tile, s, i, j, g);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[0][0][4 * g + r] += v[r];
    }
  uint16_t* a = reinterpret_cast<uint16_t*>(ws + q.square_at);
  const int wave = uniform((int)(threadIdx.x >> 6));
  const int row0 = ti * P::BM + wave / P::WC * (P::BM / P::WR) + i * 32, col0 = tj * P::BN + wave % P::WC * (P::BN / P::WC) + j * 32;
  One::hand_out<true>(
      acc, (lds_bytes)smem, One::Nothing{},
      [&](int r, int c, f32x4 v, f32x4) {
        const int row = row0 + (r & 31), col = col0 + (c & 31);
        v *= kGramFactor;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e >= q.m) v[e] = 0.f;
        if (row < q.m && col < ld) put_split4(a + split_at(row, col, ld), v);
        return v;
      },
      [&](int r, int c, f32x4 v) {
        const int row = row0 + (r & 31), col = col0 + (c & 31);
        if (ti != tj && col < q.m) put_split4(a + split_at(col, row, ld), v);
      });
}

// out = f0 L R + f1 L + fi I of the m x m matrices, all symmetric and polynomials of one another: one tile of the upper triangle, which
// halves the work.  Its epilogue (L read, both sides written) is 6 of the 50 us at 2048.
struct Square {
  int left, right, out;
  float f0, f1, fi;
};
template <class P>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void square(Tiles tiles, Square s, char* ws) {
  extern __shared__ char smem[];
  const Table& t = table_of(ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int nt = div_up(q.m, P::BM);
  int ti, tj;
  tile_in_triangle(run_of_xcd(blockIdx.x - tiles.first[k], triangle_tiles(nt)), nt, kBand, ti, tj);
  const int ld = up32(q.m);
  const auto at = [&](int i) { return reinterpret_cast<uint16_t*>(ws + q.square_at + i * q.square_bytes); };
  const uint16_t* l = at(s.left);
  f32x16 acc[P::FM][P::FN];
  P::run(acc, {l, (long long)ld * 2, q.m, ld}, {at(s.right), (long long)ld * 2, q.m, ld}, ti * P::BM, tj * P::BN, 0, ld / 32,
         (lds_bytes)smem);
  put_symmetric<P>(acc, (lds_bytes)smem, at(s.out), q.m, ti, tj,
                   [&](int row, int col) {
                     return s.f1 != 0.f ? get_split4(l + split_at(row, col, ld)) : f32x4{0.f, 0.f, 0.f, 0.f};
                   },
                   [&](int row, int col, f32x4 v, f32x4 old) {
                     v = v * s.f0 + old * s.f1;
#pragma unroll
                     for (int r = 0; r < 4; ++r) v[r] += row == col + r ? s.fi : 0.f;
                     return v;
                   });
}

// X <- C X (or Q X, several iterations at once), or in the last pass the result itself, with the optimiser's step: the update never
// lies in memory (21 matrices, 20.9 M weights: 174 us, a pass that only writes X 103).
template <class P, int T, bool LAST>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void apply(Tiles tiles, Step s, char* ws, int factor, int flip) {
  extern __shared__ char smem[];
  const Table& t = table_of(ws);
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  int tm, tn;
  tile_of(blockIdx.x - tiles.first[k], div_up(q.m, P::BM), div_up(q.n, P::BN), kBand, tm, tn);
  const int ldm = up32(q.m), ld = up32(q.n);
  const uint16_t* x = reinterpret_cast<const uint16_t*>(ws + (flip ? q.y_at : q.x_at));
  uint16_t* y = reinterpret_cast<uint16_t*>(ws + (flip ? q.x_at : q.y_at));
  const uint16_t* c = reinterpret_cast<const uint16_t*>(ws + q.square_at + factor * q.square_bytes);
  f32x16 acc[P::FM][P::FN];
  P::run(acc, {c, (long long)ldm * 2, q.m, ldm}, {x, (long long)ld * 2, q.n, q.m}, tm * P::BM, tn * P::BN, 0, ldm / 32,
         (lds_bytes)smem);
  if constexpr (!LAST) {
    P::hand_out(acc, (lds_bytes)smem, [&](int r, int c, f32x4 v) {
      const int row = tm * P::BM + r, col = tn * P::BN + c;
      if (row < q.m && col < ld) put_split4(y + split_at(row, col, ld), v * (1.f / kScaleC));
    });
    return;
  }
  constexpr float f = 1.f / (kScaleC * kScaleX);
  if (!q.tall && aligned16(q.out) && q.n % 4 == 0) {
    P::template hand_out<false>(
        acc, (lds_bytes)smem,
        [&](int r, int c) {
          const int row = tm * P::BM + r, col = tn * P::BN + c;
          if (!s.update || row >= q.m || col >= q.n) return f32x4{0.f, 0.f, 0.f, 0.f};
          return load_four<T>(q.out, (long long)row * q.n + col, 4, true);
        },
        [&](int r, int c, f32x4 v, f32x4 old) {
          const int row = tm * P::BM + r, col = tn * P::BN + c;
          if (row < q.m && col < q.n) put_result4<T>(q, s, (long long)row * q.n + col, v * f, old);
        },
        typename P::Nothing{});
    return;
  }
  const int row0 = tm * P::BM + P::lane_row(), col0 = tn * P::BN + P::lane_col();
#pragma unroll
  for (int i = 0; i < P::FM; ++i) {
    const int row = row0 + i * 32;
    if (row >= q.m) continue;
#pragma unroll
    for (int j = 0; j < P::FN; ++j) {
      float o[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = acc[i][j][e] * f;
      const auto column = [&](int e) { return col0 + j * 32 + (e >> 2) * 8 + (e & 3); };
      put_results<T>(q, s, [&](int e) { return q.tall ? (long long)column(e) * q.m + row : (long long)row * q.n + column(e); },
                     [&](int e) { return column(e) < q.n; }, o);
    }
  }
}

// ---- launching -----------------------------------------------------------------------------------------------------------

// `go` with the tile of that side; `lone`: a launch of 128 tiles that each have a compute unit of their own.
template <bool BKM, class F>
void with_tile(int side, bool lone, F go) {
  if (side == 256)
    go(Tile256<true, false, false, BKM>{});
  else if (side == 64)
    go(Tile64<true, false, false, BKM>{});
  else if (lone)
    go(Lone128<true, false, false, BKM>{});
  else
    go(Tile128<true, false, false, BKM>{});
}

size_t up(size_t v) { return (v + 255) & ~size_t(255); }

bool is_narrow(int rows, int cols) {
  const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return m <= kNarrow && n <= kNarrowLong;
}

// Tiles and slices of X X': per side one slice, or those that deal the launch's stages evenly to all places, each at least 8 stages
// long; the side and cut with the least estimated time.  Joining costs a launch and the slices' way to memory and back.
struct GramPlan {
  int side;
  bool lone;
  float us;
};
GramPlan plan_gram(Table& t) {
  GramPlan best = {64, false, INFINITY};
  int slices[kMany];
  for (int side : {256, 128, 64})
    for (bool cut : {false, true}) {
      double stages = 0;
      for (int i = 0; i < t.count; ++i) stages += (double)triangle_tiles(div_up(t.m[i].m, side)) * (up32(t.m[i].n) / 32);
      double each = stages / tile_places(side);
      if (each < 8) each = 8;
      long long tiles = 0;
      double bytes = 0, longest = 0;
      int mine[kMany];
      for (int i = 0; i < t.count; ++i) {
        const int steps = up32(t.m[i].n) / 32, per = triangle_tiles(div_up(t.m[i].m, side));
        const double want = steps / each;
        mine[i] = !cut || want < 1.5 ? 1 : want > 32 ? 32 : (int)(want + 0.5);
        tiles += (long long)per * mine[i];
        if (mine[i] > 1) bytes += 8.0 * mine[i] * per * side * side;
        const double len = (double)div_up(steps, mine[i]);
        longest = len > longest ? len : longest;
      }
      const TileTime time = tile_time(side, true);
      float us = launch_us(side, true, tiles, (float)(stages / tiles));
      const float least = time.around + (float)longest * time.alone;
      us = (us > least ? us : least) + (bytes > 0 ? 4.f + (float)(bytes / 8e6) : 0.f);  // joined while the last tiles still run
      if (us < best.us) {
        best = {side, tiles <= compute_units(), us};
        for (int i = 0; i < t.count; ++i) slices[i] = mine[i];
      }
    }
  for (int i = 0; i < t.count; ++i) t.m[i].slices = slices[i];
  return best;
}

size_t lay_out_workspace(Table& t, bool narrow, GramPlan* plan) {
  size_t at = kTableBytes;
  if (narrow) {
    for (int i = 0; i < t.count; ++i) {
      Mat& q = t.m[i];
      const int chunks = div_up(q.n, 64), mt = div_up(q.m, 16);
      q.slices = chunks < 16 ? chunks : div_up(chunks, 8) > 16 ? div_up(chunks, 8) : 16;
      if (q.slices > kParts) q.slices = kParts;
      q.parts_at = at, at += up((size_t)q.slices * triangle_tiles(mt) * 64 * 32);
      q.square_at = at, at += up((size_t)mt * 16 * mt * 16 * 8);
    }
    return at;
  }
  *plan = plan_gram(t);
  for (int i = 0; i < t.count; ++i) {
    Mat& q = t.m[i];
    const size_t x = up((size_t)q.m * up32(q.n) * 4), a = up((size_t)q.m * up32(q.m) * 4);
    q.norm_at = at, at += up(kNormBlocks * 8);
    q.x_at = at, at += x;
    q.y_at = at, at += x;
    q.square_at = at, q.square_bytes = (long long)a, at += kSquares * a;
    q.parts_at = at;
    if (q.slices > 1) at += (size_t)q.slices * triangle_tiles(div_up(q.m, plan->side)) * plan->side * plan->side * 4;
  }
  return at;
}

template <class F>
Tiles deal(const Table& t, F per) {
  Tiles d;
  d.first[0] = 0;
  for (int i = 0; i < t.count; ++i) d.first[i + 1] = d.first[i] + per(t.m[i]);
  return d;
}

template <int THREADS, class K, class... A>
void launch(K kernel, unsigned lds, int blocks, hipStream_t stream, A... args) {
  if (lds >= 65536)  // with a kernel's own variables more than what is given unasked
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  kernel<<<blocks, THREADS, lds, stream>>>(args...);
}

// One stage of the iteration over all matrices: the workgroups of each, the tile side with the least estimated time, that time.
struct Dealt {
  Tiles tiles;
  int side;
  bool lone;
  float us;
};
template <class F>
Dealt choose(const Table& t, F tiles_of) {
  const Tiles a = deal(t, [&](const Mat& q) { return tiles_of(q, 256); }), b = deal(t, [&](const Mat& q) { return tiles_of(q, 128); }),
              c = deal(t, [&](const Mat& q) { return tiles_of(q, 64); });
  double stages = 0;
  for (int i = 0; i < t.count; ++i) stages += (double)(c.first[i + 1] - c.first[i]) * (up32(t.m[i].m) / 32);
  const float steps = (float)(stages / c.first[t.count]);
  const int side = choose_tile(a.first[t.count], b.first[t.count], c.first[t.count], steps, true);
  const Tiles& d = side == 256 ? a : side == 128 ? b : c;
  return {d, side, d.first[t.count] <= compute_units(), launch_us(side, true, d.first[t.count], steps)};
}

// How many iterations share a pass over the long side (1, 2 or 3): the least estimated time among those whose product of factors C
// stays within the stored form's range.
constexpr float kLaunch = 3.f;  // us around the tiles of a launch: start, table and a result that others read
int iterations_a_pass(int steps, float gram_us, float square_us, float apply_us, const double* growth) {
  int best = 1;
  float least = INFINITY;
  for (int g = 1; g <= 3 && g <= steps; ++g) {
    if (g > 1 && !(growth[g] <= kMostC)) break;
    float us = 0.f;
    for (int done = 0; done < steps; done += g) {
      const int now = steps - done < g ? steps - done : g;
      us += gram_us + apply_us + (4 * now - 3) * square_us + (4 * now - 1) * kLaunch;
    }
    if (us < least) least = us, best = g;
  }
  return best;
}

template <int T>
void iterate(const Table& t, const Step& s, const GramPlan& plan, const double* growth, char* ws, hipStream_t stream) {
  const Tiles norm = deal(t, [](const Mat& q) {
    const int b = ceil_div((long long)q.m * q.n, kNormElements);
    return b > kNormBlocks ? kNormBlocks : b;
  });
  momentum_and_norm<T><<<norm.first[t.count], 256, 0, stream>>>(t, norm, s, ws);
  const Tiles squares = deal(t, [](const Mat& q) { return div_up(q.m, 64) * div_up(q.n, 64); });
  normalize<T><<<squares.first[t.count], 256, 0, stream>>>(squares, norm, s, ws);
  const Tiles g = deal(t, [&](const Mat& q) { return triangle_tiles(div_up(q.m, plan.side)) * q.slices; });
  const Dealt p = choose(t, [](const Mat& q, int side) { return triangle_tiles(div_up(q.m, side)); });
  const Dealt f = choose(t, [](const Mat& q, int side) { return div_up(q.m, side) * div_up(q.n, side); });
  const auto do_square = [&](int left, int right, int out, float f0, float f1, float fi) {
    const Square q = {left, right, out, f0, f1, fi};
    with_tile<false>(p.side, p.lone, [&](auto tile) {
      using P = decltype(tile);
      launch<P::kThreads>(square<P>, P::kLds, p.tiles.first[t.count], stream, p.tiles, q, ws);
    });
  };
  const int a_pass = iterations_a_pass(s.steps, plan.us, p.us, f.us, growth);
  int flip = 0;
  for (int done = 0; done < s.steps; flip ^= 1) {
    const int now = s.steps - done < a_pass ? s.steps - done : a_pass;
    done += now;
    with_tile<false>(plan.side, plan.lone, [&](auto tile) {
      using P = decltype(tile);
      launch<P::kThreads>(gram<P>, P::kLds, g.first[t.count], stream, g, ws, flip);
      const Tiles joins = deal(t, [](const Mat& q) { return q.slices > 1 ? triangle_tiles(div_up(q.m, P::BM)) * P::FM * P::FN : 0; });
      if (joins.first[t.count] > 0) launch<P::kThreads>(join_gram<P>, 0, joins.first[t.count], stream, joins, ws);
    });
    int product = kQ, spare = kT;
    for (int i = 0; i < now; ++i) {
      const int c = i == 0 ? kQ : kC;
      do_square(kA, kA, c, s.c * kScaleC / (kScaleA * kScaleA), s.b * kScaleC / kScaleA, s.a * kScaleC);
      if (i > 0) {
        do_square(kC, product, spare, 1.f / kScaleC, 0.f, 0.f);
        const int old = product;
        product = spare, spare = old;
      }
      if (i + 1 < now) {
        const int factor = i == 0 ? product : kC;
        do_square(factor, kA, spare, 1.f / kScaleC, 0.f, 0.f);
        do_square(spare, factor, kA, 1.f / kScaleC, 0.f, 0.f);
      }
    }
    const bool last = done == s.steps;
    with_tile<true>(f.side, f.lone, [&](auto tile) {
      using P = decltype(tile);
      launch<P::kThreads>(last ? apply<P, T, true> : apply<P, T, false>, P::kLds, f.tiles.first[t.count], stream, f.tiles, s, ws,
                          product, flip);
    });
  }
}

template <int T>
void iterate_narrow(const Table& t, const Step& s, char* ws, hipStream_t stream) {
  const Tiles parts = deal(t, [](const Mat& q) { return q.slices; });
  narrow_gram<T><<<parts.first[t.count], 256, 0, stream>>>(t, parts, s, ws);
  launch<kPolyThreads>(narrow_polynomial, 4 * sizeof(double) * kNarrow * kLdM, t.count, stream, s, ws);
  const Tiles columns = deal(t, [](const Mat& q) { return div_up(q.n, 64); });
  narrow_apply<T><<<columns.first[t.count], 256, 0, stream>>>(columns, s, ws);
}

int check_matrices(int count, const int* rows, const int* cols) {
  MI_REQUIRE(count >= 1 && rows != nullptr && cols != nullptr, "orthogonalize: %d matrices", count);
  for (int i = 0; i < count; ++i)
    MI_REQUIRE(rows[i] >= 1 && cols[i] >= 1 && rows[i] <= (1 << 22) && cols[i] <= (1 << 22) &&
                   (rows[i] <= 65536 || cols[i] <= 65536),
               "orthogonalize: matrix %d is [%d, %d]; sides of 1 to 2^22 are taken, one of them up to 65536", i, rows[i], cols[i]);
  return MI_OK;
}

// growth[g]: a bound of the product of g successive factors C.  False for coefficients with which X or a single C leaves the range of
// the stored forms.  Of singular values up to `top`, C = a + b t + c t^2 (t = s^2) is largest in magnitude at an end or its
// vertex, s C at `top` or where a + 3 b t + 5 c t^2 = 0.
bool range_of(const float* coefficients, int steps, double* growth) {
  const double a = coefficients[0], b = coefficients[1], c = coefficients[2];
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  const auto factor = [&](double t) { return std::fabs(a + t * (b + t * c)); };
  const double vertex = c != 0 ? -b / (2 * c) : 0;
  double turns[2] = {0, 0};  // t where s C turns
  const double inside = 9 * b * b - 20 * a * c;
  if (c == 0) {
    if (b != 0) turns[0] = -a / (3 * b);
  } else if (inside >= 0) {
    turns[0] = (-3 * b + std::sqrt(inside)) / (10 * c), turns[1] = (-3 * b - std::sqrt(inside)) / (10 * c);
  }
  double top = 1, before = 0, second = 0;  // the two factors before
  growth[1] = growth[2] = growth[3] = 0;
  for (int i = 0; i < steps; ++i) {
    const double t = top * top;
    double most = std::fmax(factor(0), factor(t)), next = top * factor(t);
    if (vertex > 0 && vertex < t) most = std::fmax(most, factor(vertex));
    for (double u : turns)
      if (u > 0 && u < t) next = std::fmax(next, std::sqrt(u) * factor(u));
    if (!(next <= kMostX && most <= kMostC)) return false;
    growth[1] = std::fmax(growth[1], most);
    growth[2] = std::fmax(growth[2], most * before);
    growth[3] = std::fmax(growth[3], most * before * second);
    second = before, before = most, top = next;
  }
  return true;
}

int check_coefficients(const float* c, int steps, float eps, double* growth) {
  MI_REQUIRE(c != nullptr && steps >= 1 && steps <= 64, "orthogonalize: %d steps, 1 to 64 are taken", steps);
  MI_REQUIRE(eps > 0.f, "orthogonalize: eps must be positive");
  if (!range_of(c, steps, growth)) {
    set_error("orthogonalize: coefficients (%g, %g, %g) let the iteration grow beyond %g", c[0], c[1], c[2], kMostX);
    return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

// Calls `visit(table, indices, narrow)` for tables of up to kMany matrices of one way, narrow ones first, those with the longest sums of
// a table at its front: their tiles start first and the short ones fill up (21 matrices of sides 3 to 12544: 802 us, as they
// come 833).
template <class F>
void each_table(int count, const int* rows, const int* cols, F visit) {
  for (int narrow = 1; narrow >= 0; --narrow) {
    Table t = {};
    int index[kMany];
    for (int i = 0; i <= count; ++i) {
      if (i < count && is_narrow(rows[i], cols[i]) == (narrow != 0)) {
        Mat q = {};
        q.tall = rows[i] > cols[i];
        q.m = q.tall ? cols[i] : rows[i], q.n = q.tall ? rows[i] : cols[i];
        q.shape = q.tall ? std::sqrt((float)rows[i] / (float)cols[i]) : 1.f;
        int at = t.count++;
        for (; at > 0 && t.m[at - 1].m < q.m; --at) t.m[at] = t.m[at - 1], index[at] = index[at - 1];
        t.m[at] = q, index[at] = i;
      }
      if (t.count == kMany || (i == count && t.count > 0)) {
        visit(t, index, narrow != 0);
        t.count = 0;
      }
    }
  }
}

size_t workspace_bytes_of(int count, const int* rows, const int* cols) {
  size_t most = 0;
  each_table(count, rows, cols, [&](Table& t, const int*, bool narrow) {
    GramPlan plan;
    const size_t b = lay_out_workspace(t, narrow, &plan);
    most = b > most ? b : most;
  });
  return most;
}

int run_all(int count, const void* const* grads, void* const* outs, float* const* momenta, const int* rows, const int* cols,
            int dtype, const Step& s, const double* growth, void* workspace, size_t workspace_bytes, hipStream_t stream,
            const char* what) {
  MI_REQUIRE(grads != nullptr && outs != nullptr && workspace != nullptr, "%s: null pointer", what);
  MI_REQUIRE(dtype == MI_TYPE_F32 || dtype == MI_TYPE_F16 || dtype == MI_TYPE_BF16, "%s: dtype %d", what, dtype);
  MI_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "%s: the workspace starts on 256 bytes", what);
  for (int i = 0; i < count; ++i)
    MI_REQUIRE(grads[i] != nullptr && outs[i] != nullptr && (momenta == nullptr || momenta[i] != nullptr),
               "%s: null pointer for matrix %d", what, i);
  const size_t needed = workspace_bytes_of(count, rows, cols);
  if (workspace_bytes < needed) {
    set_error("%s: a workspace of %zu bytes is needed, %zu given", what, needed, workspace_bytes);
    return MI_ERR_WORKSPACE;
  }
  begin_call();
  char* ws = static_cast<char*>(workspace);
  each_table(count, rows, cols, [&](Table& t, const int* index, bool narrow) {
    GramPlan plan;
    lay_out_workspace(t, narrow, &plan);
    for (int i = 0; i < t.count; ++i) {
      t.m[i].grad = grads[index[i]];
      t.m[i].out = outs[index[i]];
      t.m[i].momentum = momenta != nullptr ? momenta[index[i]] : nullptr;
    }
    const auto go = [&](auto type) {
      constexpr int T = decltype(type)::value;
      if (narrow)
        iterate_narrow<T>(t, s, ws, stream);
      else
        iterate<T>(t, s, plan, growth, ws, stream);
    };
    if (dtype == MI_TYPE_F32)
      go(std::integral_constant<int, MI_TYPE_F32>{});
    else if (dtype == MI_TYPE_F16)
      go(std::integral_constant<int, MI_TYPE_F16>{});
    else
      go(std::integral_constant<int, MI_TYPE_BF16>{});
  });
  return check_launch(what);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_orthogonalize_workspace_bytes(int count, const int* rows, const int* cols) {
  if (check_matrices(count, rows, cols) != MI_OK) return 0;
  return workspace_bytes_of(count, rows, cols);
}

int mi_orthogonalize(int count, const void* const* in, void* const* out, const int* rows, const int* cols, int dtype, int steps,
                     const float* coefficients, float eps, void* workspace, size_t workspace_bytes, mi_stream_t stream) {
  double growth[4];
  if (const int rc = check_matrices(count, rows, cols)) return rc;
  if (const int rc = check_coefficients(coefficients, steps, eps, growth)) return rc;
  const Step s = {coefficients[0], coefficients[1], coefficients[2], eps, 0.f, 0.f, 1.f, 0, 0, steps};
  return run_all(count, in, out, nullptr, rows, cols, dtype, s, growth, workspace, workspace_bytes, as_stream(stream),
                 "mi_orthogonalize");
}

int mi_muon_step(int count, void* const* params, const void* const* grads, float* const* momenta, const int* rows, const int* cols,
                 int dtype, float lr, float momentum, int nesterov, float weight_decay, int steps, const float* coefficients,
                 float eps, void* workspace, size_t workspace_bytes, mi_stream_t stream) {
  double growth[4];
  if (const int rc = check_matrices(count, rows, cols)) return rc;
  if (const int rc = check_coefficients(coefficients, steps, eps, growth)) return rc;
  MI_REQUIRE(momenta != nullptr, "mi_muon_step: null pointer");
  const Step s = {coefficients[0], coefficients[1], coefficients[2], eps, momentum, lr, (float)(1.0 - (double)lr * weight_decay), nesterov, 1, steps};
  return run_all(count, grads, params, momenta, rows, cols, dtype, s, growth, workspace, workspace_bytes, as_stream(stream),
                 "mi_muon_step");
}

}  // extern "C"
