// Newton-Schulz orthogonalisation of an update on the matrix cores, to float32 accuracy.
//
//   X = G / (|G| + eps),   `steps` times:   A = X X^T,   Q = a I + b A + c A^2,   X <- Q X         (m x n with m <= n; taller matrices are turned)
//
// The first steps multiply small singular values by a (3.4 each time), and with them whatever a rounding left in their directions, so operands of 11 or 8
// bits would show in the result.  The fast matrix instructions take 16-bit operands; the float32 ones run at a sixteenth of their rate.  So every
// operand is kept as TWO float16 numbers, v = hi + lo with hi = float16(v) and lo = float16(v - hi): 22 bits, and a product of two such operands
// is hi hi + hi lo + lo hi - three float16 products, summed in float32, with nothing lost beyond 2^-21.  Values are scaled by powers of two that put
// the largest possible one just inside float16's range (|X| < 1.9, A < 3.61, |Q| < 8: the host checks the coefficients), which leaves lo's
// subnormal steps far below what matters.
//
// A, A^2 and Q are symmetric.  Every product is of the form C = L R^T with both operands stored along k: A = X X^T, A^2 = A A^T, and
// Q X = Q (X^T)^T, for which X is kept in both orders.  The polynomial is the epilogue of the product in front of it, the split into hi and lo the
// epilogue of all three; a X needs no pass of its own, it is the a on Q's diagonal.
//
//   up to 64 x 64      one workgroup per matrix, everything in LDS, one launch for a whole list: latency bound (15 dependent products of 64^3)
//   larger             tiled products over all matrices of the list at once: one launch for the norms, one for the split, three per step
#pragma once
#include "learning_common.hpp"

namespace mbt_learning {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float kScaleX = 32768.0f, kScaleA = 16384.0f, kScaleQ = 8192.0f;
constexpr int kMostGroups = 16;  // matrix shapes of one launch, by value in its arguments

struct MatrixGroup {  // `batch` matrices of one shape
  const void* in;
  void* out;
  int64_t in_batch, in_row, in_column, out_batch, out_row, out_column;  // strides of the matrix as the kernels see it: m <= n, turned if it was taller
  int32_t m, n, mp, np;        // sizes, padded to the tile
  int64_t first;               // (large) first tile of this launch, (small) first workgroup
  int64_t planes;              // (large) where its planes start in the workspace, in halfs; each matrix of the batch has `stride` of them
  int64_t stride;
  int64_t batch;
};
struct OrthogonaliseParams {
  MatrixGroup group[kMostGroups];
  int32_t groups;
  int32_t steps;
  float a, b, c;
  double eps;
  _Float16* planes;
  double* partials;       // [matrix][kNormBlocks]
  int32_t odd;            // which of the two X^T buffers holds X^T
  int32_t last;           // the product writes the output
  int64_t blocks;
};

struct Halves {
  _Float16 hi, lo;
};
__device__ __forceinline__ Halves split(float v) {
  const _Float16 hi = static_cast<_Float16>(v);
  return {hi, static_cast<_Float16>(v - static_cast<float>(hi))};
}

__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) v += lds[w];
  __syncthreads();
  return v;
}

__device__ __forceinline__ int find_group(const OrthogonaliseParams& P, int64_t block, int64_t& at) {
  int g = 0;
  while (g + 1 < P.groups && block >= P.group[g + 1].first) ++g;
  at = block - P.group[g].first;
  return g;
}

// ---- up to 64 x 64: one workgroup, four waves, a 32 x 32 quarter of every product each ----------------------------------------------
constexpr int kSmall = 64, kPitch = kSmall + 8;  // halfs; rows 144 bytes apart put the 16 rows of an operand read into 64 different banks
constexpr int kSmallPlane = kSmall * kPitch;
constexpr size_t kSmallLds = 8 * kSmallPlane * sizeof(_Float16);

// 32 x 32 of L R^T at (row, column), k up to kp
__device__ __forceinline__ void small_product(const _Float16* l, const _Float16* r, int row, int column, int kp, float4v (&acc)[2][2]) {
  const int lane = threadIdx.x & 63, at = (lane & 15) * kPitch + 8 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < kp; k += 32) {
    half8 lh[2], ll[2], rh[2], rl[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int lo = (row + 16 * i) * kPitch + k + at, ro = (column + 16 * i) * kPitch + k + at;
      lh[i] = *reinterpret_cast<const half8*>(l + lo);
      ll[i] = *reinterpret_cast<const half8*>(l + kSmallPlane + lo);
      rh[i] = *reinterpret_cast<const half8*>(r + ro);
      rl[i] = *reinterpret_cast<const half8*>(r + kSmallPlane + ro);
    }
    // (a tile's three products depend on each other: the four tiles take turns)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t >> 1][t & 1] = mfma(lh[t >> 1], rl[t & 1], acc[t >> 1][t & 1]);
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t >> 1][t & 1] = mfma(ll[t >> 1], rh[t & 1], acc[t >> 1][t & 1]);
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t >> 1][t & 1] = mfma(lh[t >> 1], rh[t & 1], acc[t >> 1][t & 1]);
  }
}

template <typename E>
__global__ __launch_bounds__(256) void orthogonalise_small(const OrthogonaliseParams P) {
  extern __shared__ _Float16 lds_small[];
  __shared__ double sums[4];
  int64_t which;
  const MatrixGroup M = P.group[find_group(P, blockIdx.x, which)];
  const E* in = static_cast<const E*>(M.in) + which * M.in_batch;
  E* out = static_cast<E*>(M.out) + which * M.out_batch;
  // planes: X (hi, lo), X^T, A, Q
  _Float16 *x = lds_small, *xt = x + 2 * kSmallPlane, *am = xt + 2 * kSmallPlane, *q = am + 2 * kSmallPlane;
  float v[16];
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {  // (threads along the longer stride-1 axis would only matter for a matrix that is read once)
    const int at = threadIdx.x + 256 * k, i = at >> 6, j = at & 63;
    v[k] = i < M.m && j < M.n ? static_cast<float>(in[i * M.in_row + j * M.in_column]) : 0.0f;
    sum += static_cast<double>(v[k]) * static_cast<double>(v[k]);
  }
  sum = block_sum(sum, sums);
  const float inverse = static_cast<float>(1.0 / (sqrt(sum) + P.eps));
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int at = threadIdx.x + 256 * k, i = at >> 6, j = at & 63;
    const Halves h = split(v[k] * inverse * kScaleX);
    x[i * kPitch + j] = h.hi;
    x[kSmallPlane + i * kPitch + j] = h.lo;
    xt[j * kPitch + i] = h.hi;
    xt[kSmallPlane + j * kPitch + i] = h.lo;
  }
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int row = 32 * (wave >> 1), column = 32 * (wave & 1);
  const int r0 = 4 * (lane >> 4), c0 = lane & 15;  // an accumulator's element r of this lane is at (r0 + r, c0) of its 16 x 16 tile
  const bool square = row < M.mp && column < M.mp, flat = row < M.mp && column < M.np;
  float4v acc[2][2];
  for (int step = 0; step < P.steps; ++step) {
    if (square) {  // A; symmetric, so a lane's four rows of one column are stored as four neighbours of a row
      small_product(x, x, row, column, M.np, acc);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          half4 hi, lo;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const Halves h = split(acc[i][j][r] * (kScaleA / kScaleX / kScaleX));
            hi[r] = h.hi;
            lo[r] = h.lo;
          }
          const int at = (column + 16 * j + c0) * kPitch + row + 16 * i + r0;
          *reinterpret_cast<half4*>(am + at) = hi;
          *reinterpret_cast<half4*>(am + kSmallPlane + at) = lo;
        }
    }
    __syncthreads();
    if (square) {
      small_product(am, am, row, column, M.mp, acc);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = (column + 16 * j + c0) * kPitch + row + 16 * i + r0;
          const half4 ah = *reinterpret_cast<const half4*>(am + at), al = *reinterpret_cast<const half4*>(am + kSmallPlane + at);
          half4 hi, lo;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float av = (static_cast<float>(ah[r]) + static_cast<float>(al[r])) * (kScaleQ / kScaleA);
            float value = __builtin_fmaf(P.b, av, P.c * (acc[i][j][r] * (kScaleQ / kScaleA / kScaleA)));
            if (row + 16 * i + r0 + r == column + 16 * j + c0) value += P.a * kScaleQ;
            const Halves h = split(value);
            hi[r] = h.hi;
            lo[r] = h.lo;
          }
          *reinterpret_cast<half4*>(q + at) = hi;
          *reinterpret_cast<half4*>(q + kSmallPlane + at) = lo;
        }
    }
    __syncthreads();
    if (flat) small_product(q, xt, row, column, M.mp, acc);
    if (step + 1 == P.steps) break;
    __syncthreads();  // X^T has been read
    if (flat) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          half4 hi, lo;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const Halves h = split(acc[i][j][r] * (1.0f / kScaleQ));
            hi[r] = h.hi;
            lo[r] = h.lo;
            const int at = (row + 16 * i + r0 + r) * kPitch + column + 16 * j + c0;
            x[at] = h.hi;
            x[kSmallPlane + at] = h.lo;
          }
          const int at = (column + 16 * j + c0) * kPitch + row + 16 * i + r0;
          *reinterpret_cast<half4*>(xt + at) = hi;
          *reinterpret_cast<half4*>(xt + kSmallPlane + at) = lo;
        }
    }
    __syncthreads();
  }
  if (flat) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = row + 16 * i + r0 + r, to = column + 16 * j + c0;
          if (at < M.m && to < M.n) out[at * M.out_row + to * M.out_column] = static_cast<E>(acc[i][j][r] * (1.0f / kScaleQ / kScaleX));
        }
  }
}

// ---- larger ------------------------------------------------------------------------------------------------------------------------
constexpr int kNormBlocks = 64;

// planes of one matrix, in halfs from its start: X hi, lo (mp x np); X^T hi, lo twice (np x mp); A hi, lo; Q hi, lo (mp x mp)
struct Planes {
  _Float16 *x, *xt, *xt_next, *a, *q;  // (X^T of this step and of the next)
  int64_t xs, as;  // from a hi plane to its lo plane
};
__device__ __forceinline__ Planes planes_of(const OrthogonaliseParams& P, const MatrixGroup& M, int64_t which) {
  Planes p;
  p.xs = static_cast<int64_t>(M.mp) * M.np;
  p.as = static_cast<int64_t>(M.mp) * M.mp;
  p.x = P.planes + M.planes + which * M.stride;
  p.xt = p.x + (P.odd ? 4 : 2) * p.xs;
  p.xt_next = p.x + (P.odd ? 2 : 4) * p.xs;
  p.a = p.x + 6 * p.xs;
  p.q = p.a + 2 * p.as;
  return p;
}

// sum of squares of one matrix, kNormBlocks workgroups each (M.first: in matrices; partials by matrix of the launch)
template <typename E>
__global__ __launch_bounds__(256) void orthogonalise_norms(const OrthogonaliseParams P) {
  __shared__ double lds[4];
  int64_t which;
  const int64_t matrix = blockIdx.x / kNormBlocks, part = blockIdx.x % kNormBlocks;
  const MatrixGroup M = P.group[find_group(P, matrix, which)];
  const E* in = static_cast<const E*>(M.in) + which * M.in_batch;
  const bool along_n = M.in_column <= M.in_row;  // neighbours in memory to neighbouring threads
  const int64_t fast = along_n ? M.n : M.m, slow = along_n ? M.m : M.n;
  const int64_t fast_stride = along_n ? M.in_column : M.in_row, slow_stride = along_n ? M.in_row : M.in_column;
  double sum = 0.0;
  for (int64_t s = part; s < slow; s += kNormBlocks)
    for (int64_t f = threadIdx.x; f < fast; f += 256) {
      const float v = static_cast<float>(in[s * slow_stride + f * fast_stride]);
      sum += static_cast<double>(v) * static_cast<double>(v);
    }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) P.partials[blockIdx.x] = sum;
}

// X = G / (|G| + eps) in both orders, 64 x 64 at a time; M.first counts such tiles
template <typename E>
__global__ __launch_bounds__(256) void orthogonalise_split(const OrthogonaliseParams P) {
  __shared__ double lds[4];
  __shared__ float tile[64][65];
  int64_t at;
  const int group = find_group(P, blockIdx.x, at);
  const MatrixGroup M = P.group[group];
  const int tiles_n = M.np / 64, tiles = M.mp / 64 * tiles_n;
  const int64_t which = at / tiles;
  const int t = static_cast<int>(at % tiles), i0 = t / tiles_n * 64, j0 = t % tiles_n * 64;
  int64_t matrix = which;
  for (int g = 0; g < group; ++g) matrix += P.group[g].batch;
  const double norm = block_sum(threadIdx.x < kNormBlocks ? P.partials[matrix * kNormBlocks + threadIdx.x] : 0.0, lds);
  const float inverse = static_cast<float>(1.0 / (sqrt(norm) + P.eps));
  const E* in = static_cast<const E*>(M.in) + which * M.in_batch;
  const bool along_n = M.in_column <= M.in_row;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int e = threadIdx.x + 256 * k, i = along_n ? e >> 6 : e & 63, j = along_n ? e & 63 : e >> 6;
    tile[i][j] = i0 + i < M.m && j0 + j < M.n ? static_cast<float>(in[(i0 + i) * M.in_row + (j0 + j) * M.in_column]) * inverse * kScaleX : 0.0f;
  }
  __syncthreads();
  const Planes p = planes_of(P, M, which);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int e = threadIdx.x + 256 * k, s = e >> 6, f = e & 63;
    const Halves h = split(tile[s][f]), g = split(tile[f][s]);
    const int64_t ax = static_cast<int64_t>(i0 + s) * M.np + j0 + f, at_t = static_cast<int64_t>(j0 + s) * M.mp + i0 + f;
    p.x[ax] = h.hi;
    p.x[p.xs + ax] = h.lo;
    p.xt[at_t] = g.hi;
    p.xt[p.xs + at_t] = g.lo;
  }
}

enum : int { kGram = 0, kPolynomial = 1, kApply = 2 };

// One T x T tile of a product, four waves of T/2 x T/2, k in steps of 32 through two LDS buffers: the next step's operands are on their way from
// memory while this one's are multiplied.
template <typename E, int T, int PRODUCT>
__global__ __launch_bounds__(256) void orthogonalise_product(const OrthogonaliseParams P) {
  constexpr int kRow = 32 + 8;                   // halfs of a row in LDS: 80 bytes apart, 16 rows in 64 different banks
  constexpr int kBuffer = 4 * T * kRow;          // L hi, L lo, R hi, R lo
  constexpr int F = T / 32;                      // 16 x 16 fragments of a wave along each side
  constexpr int kLoads = T * 32 / 8 / 256 > 0 ? T * 32 / 8 / 256 : 1;  // 16-byte loads per thread and plane
  extern __shared__ _Float16 lds_product[];
  // neighbouring tiles to the same XCD (workgroups go round the eight of them), so that its L2 sees an operand's rows again
  const int64_t blocks = P.blocks, per = (blocks + 7) / 8;
  const int64_t id = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (id >= blocks) return;
  int64_t at;
  const MatrixGroup M = P.group[find_group(P, id, at)];
  const int rows = M.mp / T, columns = PRODUCT == kApply ? M.np / T : rows;
  const int tiles = PRODUCT == kApply ? rows * columns : rows * (rows + 1) / 2;
  const int64_t which = at / tiles;
  int t = static_cast<int>(at % tiles), ti, tj;
  if (PRODUCT == kApply) {
    ti = t % rows;
    tj = t / rows;
  } else {  // the upper triangle, row by row
    ti = 0;
    while (t >= rows - ti) t -= rows - ti, ++ti;
    tj = ti + t;
  }
  const Planes p = planes_of(P, M, which);
  const int kp = PRODUCT == kGram ? M.np : M.mp;  // both operands' row length
  const _Float16* l = (PRODUCT == kGram ? p.x : PRODUCT == kPolynomial ? p.a : p.q) + static_cast<int64_t>(ti) * T * kp;
  const _Float16* r = (PRODUCT == kGram ? p.x : PRODUCT == kPolynomial ? p.a : p.xt) + static_cast<int64_t>(tj) * T * kp;
  const int64_t ls = PRODUCT == kGram ? p.xs : p.as, rs = PRODUCT == kPolynomial ? p.as : p.xs;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = T / 2 * (wave >> 1), column = T / 2 * (wave & 1);
  float4v acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};
  half8 stage[4][kLoads];
  const int load_row = threadIdx.x / 4, load_k = threadIdx.x % 4 * 8;  // 64 rows of 32 halfs per sweep
  auto fetch = [&](int k) {
#pragma unroll
    for (int s = 0; s < kLoads; ++s) {
      const int64_t off = static_cast<int64_t>(load_row + 64 * s) * kp + k + load_k;
      stage[0][s] = *reinterpret_cast<const half8*>(l + off);
      stage[1][s] = *reinterpret_cast<const half8*>(l + ls + off);
      stage[2][s] = *reinterpret_cast<const half8*>(r + off);
      stage[3][s] = *reinterpret_cast<const half8*>(r + rs + off);
    }
  };
  auto put = [&](int buffer) {
#pragma unroll
    for (int plane = 0; plane < 4; ++plane)
#pragma unroll
      for (int s = 0; s < kLoads; ++s)
        *reinterpret_cast<half8*>(lds_product + buffer * kBuffer + plane * T * kRow + (load_row + 64 * s) * kRow + load_k) = stage[plane][s];
  };
  fetch(0);
  put(0);
  __syncthreads();
  int buffer = 0;
  for (int k = 0; k < kp; k += 32, buffer ^= 1) {
    const bool more = k + 32 < kp;
    if (more) fetch(k + 32);
    const _Float16* base = lds_product + buffer * kBuffer + (lane & 15) * kRow + 8 * (lane >> 4);
    half8 lh[F], ll[F];
#pragma unroll
    for (int i = 0; i < F; ++i) {
      lh[i] = *reinterpret_cast<const half8*>(base + (row + 16 * i) * kRow);
      ll[i] = *reinterpret_cast<const half8*>(base + T * kRow + (row + 16 * i) * kRow);
    }
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const half8 rh = *reinterpret_cast<const half8*>(base + 2 * T * kRow + (column + 16 * j) * kRow);
      const half8 rl = *reinterpret_cast<const half8*>(base + 3 * T * kRow + (column + 16 * j) * kRow);
#pragma unroll
      for (int i = 0; i < F; ++i) acc[i][j] = mfma(lh[i], rl, acc[i][j]);
#pragma unroll
      for (int i = 0; i < F; ++i) acc[i][j] = mfma(ll[i], rh, acc[i][j]);
#pragma unroll
      for (int i = 0; i < F; ++i) acc[i][j] = mfma(lh[i], rh, acc[i][j]);
    }
    if (more) put(buffer ^ 1);
    __syncthreads();
  }

  const int r0 = 4 * (lane >> 4), c0 = lane & 15;
  if (PRODUCT == kApply && P.last) {
    E* out = static_cast<E*>(M.out) + which * M.out_batch;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t y = ti * T + row + 16 * i + r0 + e, z = tj * T + column + 16 * j + c0;
          if (y < M.m && z < M.n) out[y * M.out_row + z * M.out_column] = static_cast<E>(acc[i][j][e] * (1.0f / kScaleQ / kScaleX));
        }
    return;
  }
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const int y = ti * T + row + 16 * i + r0, z = tj * T + column + 16 * j + c0;  // four rows y.., one column z
      half4 hi, lo;
      half4 ah, al;
      if (PRODUCT == kPolynomial) {  // A at (y + e, z) is A at (z, y + e)
        ah = *reinterpret_cast<const half4*>(p.a + static_cast<int64_t>(z) * M.mp + y);
        al = *reinterpret_cast<const half4*>(p.a + p.as + static_cast<int64_t>(z) * M.mp + y);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float value;
        if (PRODUCT == kGram) value = acc[i][j][e] * (kScaleA / kScaleX / kScaleX);
        if (PRODUCT == kApply) value = acc[i][j][e] * (1.0f / kScaleQ);
        if (PRODUCT == kPolynomial) {
          const float av = (static_cast<float>(ah[e]) + static_cast<float>(al[e])) * (kScaleQ / kScaleA);
          value = __builtin_fmaf(P.b, av, P.c * (acc[i][j][e] * (kScaleQ / kScaleA / kScaleA)));
          if (y + e == z) value += P.a * kScaleQ;
        }
        const Halves h = split(value);
        hi[e] = h.hi;
        lo[e] = h.lo;
      }
      // turned, four neighbours at once; and as it stands, one by one (not for a tile on the diagonal, which is its own mirror image)
      _Float16* turned = PRODUCT == kGram ? p.a : PRODUCT == kPolynomial ? p.q : p.xt_next;
      _Float16* plain = PRODUCT == kGram ? p.a : PRODUCT == kPolynomial ? p.q : p.x;
      const int64_t lo_plane = PRODUCT == kApply ? p.xs : p.as;
      const int64_t to = static_cast<int64_t>(z) * M.mp + y;
      *reinterpret_cast<half4*>(turned + to) = hi;
      *reinterpret_cast<half4*>(turned + lo_plane + to) = lo;
      if (PRODUCT == kApply || ti != tj) {
        const int pitch = PRODUCT == kApply ? M.np : M.mp;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          plain[static_cast<int64_t>(y + e) * pitch + z] = hi[e];
          plain[lo_plane + static_cast<int64_t>(y + e) * pitch + z] = lo[e];
        }
      }
    }
}

}  // namespace mbt_learning
