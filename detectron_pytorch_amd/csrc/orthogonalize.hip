// orthogonalize.hip -- orthogonalised updates of weight matrices by Newton-Schulz products, and the optimiser step around them.
//
// Mathematics, for a matrix G [m, n] with m <= n (a taller one is turned first and turned back at the end):
//   X_0 = G / max(|G|_F, eps);   A = X X',  B = b A + c A A,  X <- a X + B X     `steps` times
// X keeps the singular vectors of G and sends each singular value s to p(p(...p(s))) with p(s) = a s + b s^3 + c s^5, near 1 for
// all but the smallest.  The step of the optimiser around it:
//   M <- mu M + G,  U = G + mu M (nesterov) or M,  W <- (1 - lr wd) W - lr sqrt(max(1, rows / cols)) X(U)
//
// Work per iteration: m^2 n for A (upper triangle), m^3 for A A (upper triangle), 2 m^2 n for B X; all on the matrix cores
// (tile_product.h).  X, A and B are kept as hi + lo fp16 times 2^12 (22 bits): their magnitudes are known -- |X| is bounded
// by the polynomial's largest value, which the host checks -- so no pass looks for a scale.  Products of plain fp16 would lose the
// small singular directions, whose noise the iteration amplifies by up to a^steps (485 for the usual a = 3.4445 and 5 steps).
// Accumulators are float32; the norm is summed in fp64, so no gradient is too small or too large for it.
//
// All matrices of a call go through each stage in one launch: a workgroup finds its matrix in the launch's table.
#include "common.h"
#include "tile_product.h"

#include <cmath>

namespace mi {
namespace {

constexpr int kMany = 32;            // matrices of one table (it is passed by value: 4 KB of kernel arguments)
constexpr float kScale = 4096.f;     // X, A and B are stored times this
constexpr double kMostMagnitude = 15.0;
constexpr int kNormBlocks = 256;     // workgroups that sum one matrix' squares, at most
constexpr int kNormElements = 8192;  // elements for which one more workgroup is worth its launch

struct Mat {
  const void* grad;
  void* out;         // the orthogonalised matrix, or the weights that are updated
  float* momentum;   // NULL: no momentum
  int m, n;          // m <= n, after turning
  int tall;          // the matrix itself is [n, m]
  int slices;        // of the sum over n in A
  float shape;       // sqrt(max(1, rows / cols))
  long long norm_at, x_at, y_at, a_at, b_at, c_at;  // bytes into the workspace
};
struct Table {
  int count;
  Mat m[kMany];
};
struct Tiles {       // first workgroup of each matrix in a launch
  int first[kMany + 1];
};

struct Step {
  float a, b, c, eps;
  float mu, lr, decay;  // decay = 1 - lr * weight decay
  int nesterov, update;
};

__host__ __device__ inline int div_up(int a, int b) { return (a + b - 1) / b; }
__host__ __device__ inline int up32(int v) { return (v + 31) & ~31; }

__device__ __forceinline__ int find(const Tiles& t, int count, int block) {
  int i = 0;
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

// element (row, col) of a split matrix with `ld` elements a row: its hi word, the lo one is 32 words on
__device__ __forceinline__ long long split_at(int row, int col, int ld) {
  return (long long)row * ld * 2 + (col >> 5) * 64 + (col & 31);
}
__device__ __forceinline__ void put_split(uint16_t* p, float v) {
  const _Float16 h = (_Float16)v;
  p[0] = __builtin_bit_cast(uint16_t, h);
  p[32] = __builtin_bit_cast(uint16_t, (_Float16)(v - (float)h));
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

// ---- momentum, norm, X_0 -------------------------------------------------------------------------------------------------

template <int T>
__device__ __forceinline__ float update_of(const Mat& q, const Step& s, long long i, float momentum) {
  if (q.momentum == nullptr) return load_float<T>(q.grad, i);
  return s.nesterov ? load_float<T>(q.grad, i) + s.mu * momentum : momentum;
}

// M <- mu M + G, and the squares of U: one fp64 sum per workgroup.
template <int T>
__global__ __launch_bounds__(256) void momentum_and_norm(Table t, Tiles tiles, Step s, char* ws) {
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int block = blockIdx.x - tiles.first[k], blocks = tiles.first[k + 1] - tiles.first[k];
  const long long n = (long long)q.m * q.n;
  double sum = 0;
  for (long long i = block * 256LL + threadIdx.x; i < n; i += blocks * 256LL) {
    float m = 0.f;
    if (q.momentum != nullptr) {
      m = s.mu * q.momentum[i] + load_float<T>(q.grad, i);
      q.momentum[i] = m;
    }
    const double u = (double)update_of<T>(q, s, i, m);
    sum += u * u;
  }
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  __shared__ double part[4];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) reinterpret_cast<double*>(ws + q.norm_at)[block] = part[0] + part[1] + part[2] + part[3];
}

// X_0, 64 x 64 of the given matrix per workgroup, turned on the way if it is tall.
template <int T>
__global__ __launch_bounds__(256) void normalize(Table t, Tiles tiles, Tiles norm, Step s, char* ws) {
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int rows = q.tall ? q.n : q.m, cols = q.tall ? q.m : q.n;
  const int tiles_c = div_up(cols, 64), tile = blockIdx.x - tiles.first[k];
  const int row0 = tile / tiles_c * 64, col0 = tile % tiles_c * 64;
  __shared__ double part[4];
  const double* sums = reinterpret_cast<const double*>(ws + q.norm_at);
  double sum = 0;
  for (int i = threadIdx.x; i < norm.first[k + 1] - norm.first[k]; i += 256) sum += sums[i];
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double length = sqrt(part[0] + part[1] + part[2] + part[3]);
  // not fmax: a NaN stays one
  const double inv = (double)kScale / (length < (double)s.eps ? (double)s.eps : length);
  uint16_t* x = reinterpret_cast<uint16_t*>(ws + q.x_at);
  const int ld = up32(q.n);
  __shared__ float buf[64][65];
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int r = row0 + (e >> 6), c = col0 + (e & 63);
    float v = 0.f;
    if (r < rows && c < cols) {
      const long long i = (long long)r * cols + c;
      v = (float)((double)update_of<T>(q, s, i, q.momentum != nullptr ? q.momentum[i] : 0.f) * inv);
    }
    buf[e >> 6][e & 63] = v;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int i = e >> 6, j = e & 63;
    const int r = q.tall ? col0 + i : row0 + i, c = q.tall ? row0 + j : col0 + j;
    if (r < q.m && c < ld) put_split(x + split_at(r, c, ld), q.tall ? buf[j][i] : buf[i][j]);
  }
}

// ---- the iteration -------------------------------------------------------------------------------------------------------

// tile `id` of the upper triangle of n x n tiles, row by row
__device__ __forceinline__ void triangle(int id, int n, int& i, int& j) {
  i = 0;
  while (id >= n - i) id -= n - i, ++i;
  j = i + id;
}
__host__ __device__ inline int triangle_tiles(int n) { return n * (n + 1) / 2; }

// X X': one tile of the upper triangle and one slice of the sum over n, in float32.
template <class P>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void gram(Table t, Tiles tiles, char* ws, int flip) {
  extern __shared__ char smem[];
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int nt = div_up(q.m, P::BM), per = triangle_tiles(nt);
  const int id = blockIdx.x - tiles.first[k], slice = id / per;
  int ti, tj;
  triangle(id - slice * per, nt, ti, tj);
  const int ld = up32(q.n), steps = ld / 32, each = div_up(steps, q.slices), step0 = slice * each;
  const Operand x = {reinterpret_cast<const uint16_t*>(ws + (flip ? q.y_at : q.x_at)), (long long)ld * 2, q.m, ld};
  f32x16 acc[P::FM][P::FN];
  P::run(acc, x, x, ti * P::BM, tj * P::BN, step0, min(each, steps - step0), (lds_bytes)smem);
  float* c = reinterpret_cast<float*>(ws + q.c_at) + (long long)slice * q.m * up32(q.m);
  const int row0 = ti * P::BM + P::lane_row(), col0 = tj * P::BN + P::lane_col();
#pragma unroll
  for (int i = 0; i < P::FM; ++i)
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
      const int row = row0 + i * 32, col = col0 + j * 32 + g * 8;
      if (row < q.m && col < up32(q.m)) *reinterpret_cast<f32x4*>(c + (long long)row * up32(q.m) + col) = P::quad(acc[i][j], g);
    }
}

// A from the slices of its upper triangle: a workgroup joins 64 x 64 of them and writes both halves.
__global__ __launch_bounds__(256) void join_gram(Table t, Tiles tiles, char* ws) {
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  const int nt = div_up(q.m, 64), ld = up32(q.m);
  int ti, tj;
  triangle(blockIdx.x - tiles.first[k], nt, ti, tj);
  const float* c = reinterpret_cast<const float*>(ws + q.c_at);
  uint16_t* a = reinterpret_cast<uint16_t*>(ws + q.a_at);
  __shared__ float buf[64][65];
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int r = ti * 64 + (e >> 6), col = tj * 64 + (e & 63);
    float v = 0.f;
    if (r < q.m && col < q.m) {
      for (int s = 0; s < q.slices; ++s) v += c[((long long)s * q.m + r) * ld + col];
      v *= 1.f / kScale;
    }
    buf[e >> 6][e & 63] = v;
    if (r < q.m && col < ld) put_split(a + split_at(r, col, ld), v);
  }
  if (ti == tj) return;
  __syncthreads();
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int r = tj * 64 + (e >> 6), col = ti * 64 + (e & 63);
    if (r < q.m && col < ld) put_split(a + split_at(r, col, ld), buf[e & 63][e >> 6]);
  }
}

// B = b A + c A A: one tile of the upper triangle, written on both sides (the padding of a row lies in its upper half).
template <class P>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void polynomial(Table t, Tiles tiles, Step s, char* ws) {
  extern __shared__ char smem[];
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  int ti, tj;
  triangle(blockIdx.x - tiles.first[k], div_up(q.m, P::BM), ti, tj);
  const int ld = up32(q.m);
  const uint16_t* a = reinterpret_cast<const uint16_t*>(ws + q.a_at);
  uint16_t* b = reinterpret_cast<uint16_t*>(ws + q.b_at);
  const Operand o = {a, (long long)ld * 2, q.m, ld};
  f32x16 acc[P::FM][P::FN];
  P::run(acc, o, o, ti * P::BM, tj * P::BN, 0, ld / 32, (lds_bytes)smem);
  const int row0 = ti * P::BM + P::lane_row(), col0 = tj * P::BN + P::lane_col();
#pragma unroll
  for (int i = 0; i < P::FM; ++i)
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
      const int row = row0 + i * 32, col = col0 + j * 32 + g * 8;
      if (row >= q.m || col >= ld) continue;
      const f32x4 here = get_split4(a + split_at(row, col, ld));
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = col + r < q.m ? s.b * here[r] + s.c * (acc[i][j][g * 4 + r] * (1.f / kScale)) : 0.f;
      put_split4(b + split_at(row, col, ld), v);
      if (ti != tj)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col + r < q.m) put_split(b + split_at(col + r, row, ld), v[r]);
    }
}

// X <- a X + B X, or in the last iteration the result itself.
template <class P, int T, bool LAST>
__global__ __launch_bounds__(P::kThreads, kWavesPerSimd<P>) void apply(Table t, Tiles tiles, Step s, char* ws, int flip) {
  extern __shared__ char smem[];
  const int k = find(tiles, t.count, blockIdx.x);
  const Mat& q = t.m[k];
  int tm, tn;
  tile_of(blockIdx.x - tiles.first[k], div_up(q.m, P::BM), div_up(q.n, P::BN), 4, tm, tn);
  const int ldm = up32(q.m), ld = up32(q.n);
  const uint16_t* x = reinterpret_cast<const uint16_t*>(ws + (flip ? q.y_at : q.x_at));
  uint16_t* y = reinterpret_cast<uint16_t*>(ws + (flip ? q.x_at : q.y_at));
  const Operand b = {reinterpret_cast<const uint16_t*>(ws + q.b_at), (long long)ldm * 2, q.m, ldm};
  const Operand xo = {x, (long long)ld * 2, q.n, q.m};
  f32x16 acc[P::FM][P::FN];
  P::run(acc, b, xo, tm * P::BM, tn * P::BN, 0, ldm / 32, (lds_bytes)smem);
  const int row0 = tm * P::BM + P::lane_row(), col0 = tn * P::BN + P::lane_col();
#pragma unroll
  for (int i = 0; i < P::FM; ++i)
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
      const int row = row0 + i * 32, col = col0 + j * 32 + g * 8;
      if (row >= q.m || col >= ld) continue;
      const f32x4 here = get_split4(x + split_at(row, col, ld));
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = s.a * here[r] + acc[i][j][g * 4 + r] * (1.f / kScale);
      if constexpr (!LAST) {
        put_split4(y + split_at(row, col, ld), v);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (col + r >= q.n) continue;
          const long long at = q.tall ? (long long)(col + r) * q.m + row : (long long)row * q.n + col + r;
          const float o = v[r] * (1.f / kScale);
          store_float<T>(q.out, at, s.update ? load_float<T>(q.out, at) * s.decay - s.lr * q.shape * o : o);
        }
      }
    }
}

// ---- launching -----------------------------------------------------------------------------------------------------------

template <int SIDE, bool BKM>
struct TileOf {
  using type = TileProduct<SIDE, SIDE, 2, 2, SIDE == 64 ? 4 : 2, true, false, false, BKM>;
};
template <int SIDE>
using Gram = typename TileOf<SIDE, false>::type;
template <int SIDE>
using Apply = typename TileOf<SIDE, true>::type;

size_t up(size_t v) { return (v + 255) & ~size_t(255); }

// Slices of the sum over n: the launch's stages are dealt to two workgroups per compute unit, each at least 8 stages long.
void choose_slices(Table& t) {
  long long stages = 0;
  for (int i = 0; i < t.count; ++i) stages += (long long)triangle_tiles(div_up(t.m[i].m, 64)) * (up32(t.m[i].n) / 32);
  long long each = stages / (2 * compute_units());
  if (each < 8) each = 8;
  for (int i = 0; i < t.count; ++i) {
    const long long s = up32(t.m[i].n) / 32 / each;
    t.m[i].slices = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
  }
}

size_t lay_out_workspace(Table& t) {
  choose_slices(t);
  size_t at = 0;
  for (int i = 0; i < t.count; ++i) {
    Mat& q = t.m[i];
    const size_t x = up((size_t)q.m * up32(q.n) * 4), a = up((size_t)q.m * up32(q.m) * 4);
    q.norm_at = at, at += up(kNormBlocks * 8);
    q.x_at = at, at += x;
    q.y_at = at, at += x;
    q.a_at = at, at += a;
    q.b_at = at, at += a;
    q.c_at = at, at += a * q.slices;
  }
  return at;
}

void fill(Table& t, int first, int count, const int* rows, const int* cols) {
  t.count = count;
  for (int i = 0; i < count; ++i) {
    Mat& q = t.m[i];
    const int r = rows[first + i], c = cols[first + i];
    q = Mat{};
    q.tall = r > c;
    q.m = r < c ? r : c, q.n = r < c ? c : r;
    q.shape = r > c ? std::sqrt((float)r / (float)c) : 1.f;
  }
}

template <class F>
Tiles deal(const Table& t, F per) {
  Tiles d;
  d.first[0] = 0;
  for (int i = 0; i < t.count; ++i) d.first[i + 1] = d.first[i] + per(t.m[i]);
  return d;
}

template <class P, class K, class... A>
void launch(K kernel, int blocks, hipStream_t stream, A... args) {
  if (P::kLds > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)P::kLds);
  kernel<<<blocks, P::kThreads, P::kLds, stream>>>(args...);
}

// One stage of the iteration over all matrices: the workgroups of each for tiles of 256, 128 and 64, and the side that is taken.
struct Dealt {
  Tiles tiles;
  int side;
};
template <class F, class G>
Dealt choose(const Table& t, F tiles_of, G steps_of) {
  const Tiles a = deal(t, [&](const Mat& q) { return tiles_of(q, 256); }), b = deal(t, [&](const Mat& q) { return tiles_of(q, 128); }),
              c = deal(t, [&](const Mat& q) { return tiles_of(q, 64); });
  double stages = 0;
  for (int i = 0; i < t.count; ++i) stages += (double)(c.first[i + 1] - c.first[i]) * steps_of(t.m[i]);
  const int side = choose_tile(a.first[t.count], b.first[t.count], c.first[t.count], (float)(stages / c.first[t.count]), true);
  return {side == 256 ? a : side == 128 ? b : c, side};
}

template <int T>
void iterate(const Table& t, const Step& s, int steps, char* ws, hipStream_t stream) {
  const Tiles norm = deal(t, [](const Mat& q) {
    const int b = ceil_div((long long)q.m * q.n, kNormElements);
    return b > kNormBlocks ? kNormBlocks : b;
  });
  momentum_and_norm<T><<<norm.first[t.count], 256, 0, stream>>>(t, norm, s, ws);
  const Tiles squares = deal(t, [](const Mat& q) { return div_up(q.m, 64) * div_up(q.n, 64); });
  normalize<T><<<squares.first[t.count], 256, 0, stream>>>(t, squares, norm, s, ws);
  const Dealt g = choose(t, [](const Mat& q, int side) { return triangle_tiles(div_up(q.m, side)) * q.slices; },
                         [](const Mat& q) { return up32(q.n) / 32 / q.slices; });
  const auto short_steps = [](const Mat& q) { return up32(q.m) / 32; };
  const Dealt p = choose(t, [](const Mat& q, int side) { return triangle_tiles(div_up(q.m, side)); }, short_steps);
  const Dealt f = choose(t, [](const Mat& q, int side) { return div_up(q.m, side) * div_up(q.n, side); }, short_steps);
  const Tiles joined = deal(t, [](const Mat& q) { return triangle_tiles(div_up(q.m, 64)); });
  for (int i = 0; i < steps; ++i) {
    const int flip = i & 1;
    if (g.side == 256)
      launch<Gram<256>>(gram<Gram<256>>, g.tiles.first[t.count], stream, t, g.tiles, ws, flip);
    else if (g.side == 128)
      launch<Gram<128>>(gram<Gram<128>>, g.tiles.first[t.count], stream, t, g.tiles, ws, flip);
    else
      launch<Gram<64>>(gram<Gram<64>>, g.tiles.first[t.count], stream, t, g.tiles, ws, flip);
    join_gram<<<joined.first[t.count], 256, 0, stream>>>(t, joined, ws);
    if (p.side == 256)
      launch<Gram<256>>(polynomial<Gram<256>>, p.tiles.first[t.count], stream, t, p.tiles, s, ws);
    else if (p.side == 128)
      launch<Gram<128>>(polynomial<Gram<128>>, p.tiles.first[t.count], stream, t, p.tiles, s, ws);
    else
      launch<Gram<64>>(polynomial<Gram<64>>, p.tiles.first[t.count], stream, t, p.tiles, s, ws);
    const bool last = i + 1 == steps;
    if (f.side == 256)
      launch<Apply<256>>(last ? apply<Apply<256>, T, true> : apply<Apply<256>, T, false>, f.tiles.first[t.count], stream, t, f.tiles,
                         s, ws, flip);
    else if (f.side == 128)
      launch<Apply<128>>(last ? apply<Apply<128>, T, true> : apply<Apply<128>, T, false>, f.tiles.first[t.count], stream, t, f.tiles,
                         s, ws, flip);
    else
      launch<Apply<64>>(last ? apply<Apply<64>, T, true> : apply<Apply<64>, T, false>, f.tiles.first[t.count], stream, t, f.tiles, s,
                        ws, flip);
  }
}

int check_matrices(int count, const int* rows, const int* cols) {
  MI_REQUIRE(count >= 1 && rows != nullptr && cols != nullptr, "orthogonalize: %d matrices", count);
  for (int i = 0; i < count; ++i)
    MI_REQUIRE(rows[i] >= 1 && cols[i] >= 1 && rows[i] <= (1 << 22) && cols[i] <= (1 << 22) &&
                   (rows[i] <= 65536 || cols[i] <= 65536),
               "orthogonalize: matrix %d is [%d, %d]; sides of 1 to 2^22 are taken, one of them up to 65536", i, rows[i], cols[i]);
  return MI_OK;
}

// The largest magnitude that X, A or B can reach from |X| <= 1.  It is also the test that the scale of the stored forms holds.
int check_coefficients(const float* c, int steps, float eps) {
  MI_REQUIRE(c != nullptr && steps >= 1 && steps <= 64, "orthogonalize: %d steps, 1 to 64 are taken", steps);
  MI_REQUIRE(eps > 0.f, "orthogonalize: eps must be positive");
  const bool finite = std::isfinite(c[0]) && std::isfinite(c[1]) && std::isfinite(c[2]);
  double top = 1.0;
  for (int i = 0; i < steps; ++i) {
    double next = 0, inner = 0;
    for (int k = 0; k <= 4096; ++k) {
      const double x = top * k / 4096, x2 = x * x;
      next = std::fmax(next, std::fabs(x * (c[0] + x2 * (c[1] + x2 * c[2]))));
      inner = std::fmax(inner, std::fabs(x2 * (c[1] + x2 * c[2])));
    }
    next *= 1.001, inner *= 1.001;
    if (!(next <= kMostMagnitude && inner <= kMostMagnitude && top * top <= kMostMagnitude && finite)) {
      set_error("orthogonalize: coefficients (%g, %g, %g) let the iteration grow beyond %g", c[0], c[1], c[2], kMostMagnitude);
      return MI_ERR_UNSUPPORTED;
    }
    top = next;
  }
  return MI_OK;
}

size_t workspace_bytes_of(int count, const int* rows, const int* cols) {
  size_t most = 0;
  for (int first = 0; first < count; first += kMany) {
    Table t;
    fill(t, first, count - first < kMany ? count - first : kMany, rows, cols);
    const size_t b = lay_out_workspace(t);
    most = b > most ? b : most;
  }
  return most;
}

int run_all(int count, const void* const* grads, void* const* outs, float* const* momenta, const int* rows, const int* cols,
            int dtype, const Step& s, int steps, void* workspace, size_t workspace_bytes, hipStream_t stream, const char* what) {
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
  for (int first = 0; first < count; first += kMany) {
    Table t;
    fill(t, first, count - first < kMany ? count - first : kMany, rows, cols);
    lay_out_workspace(t);
    for (int i = 0; i < t.count; ++i) {
      t.m[i].grad = grads[first + i];
      t.m[i].out = outs[first + i];
      t.m[i].momentum = momenta != nullptr ? momenta[first + i] : nullptr;
    }
    char* ws = static_cast<char*>(workspace);
    if (dtype == MI_TYPE_F32)
      iterate<MI_TYPE_F32>(t, s, steps, ws, stream);
    else if (dtype == MI_TYPE_F16)
      iterate<MI_TYPE_F16>(t, s, steps, ws, stream);
    else
      iterate<MI_TYPE_BF16>(t, s, steps, ws, stream);
  }
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
  if (const int rc = check_matrices(count, rows, cols)) return rc;
  if (const int rc = check_coefficients(coefficients, steps, eps)) return rc;
  const Step s = {coefficients[0], coefficients[1], coefficients[2], eps, 0.f, 0.f, 1.f, 0, 0};
  return run_all(count, in, out, nullptr, rows, cols, dtype, s, steps, workspace, workspace_bytes, as_stream(stream),
                 "mi_orthogonalize");
}

int mi_muon_step(int count, void* const* params, const void* const* grads, float* const* momenta, const int* rows, const int* cols,
                 int dtype, float lr, float momentum, int nesterov, float weight_decay, int steps, const float* coefficients,
                 float eps, void* workspace, size_t workspace_bytes, mi_stream_t stream) {
  if (const int rc = check_matrices(count, rows, cols)) return rc;
  if (const int rc = check_coefficients(coefficients, steps, eps)) return rc;
  MI_REQUIRE(momenta != nullptr, "mi_muon_step: null pointer");
  const Step s = {coefficients[0], coefficients[1], coefficients[2], eps, momentum, lr, 1.f - lr * weight_decay, nesterov, 1};
  return run_all(count, grads, params, momenta, rows, cols, dtype, s, steps, workspace, workspace_bytes, as_stream(stream),
                 "mi_muon_step");
}

}  // extern "C"
