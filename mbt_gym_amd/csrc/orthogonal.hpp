// Newton-Schulz orthogonalisation of an update on the matrix cores, to float32 accuracy.
//
//   X = G / (|G| + eps),   `steps` times:   A = X X^T,   Q = a I + b A + c A^2,   X <- Q X         (m x n with m <= n; taller matrices are turned)
//
// The first steps multiply small singular values by a (3.4 each time), and with them whatever a rounding left in their directions, so operands of 11 or 8
// bits would show in the result.  The matrix instructions that take 16-bit operands are sixteen times as fast as the float32 ones, so
//
//   min(m, n) > 64   every operand is TWO float16 numbers, v = hi + lo with hi = float16(v) and lo = float16(v - hi): 22 bits, and a product of two such
//                    operands is hi hi + hi lo + lo hi - three float16 products, summed in float32, with nothing lost beyond 2^-21.  Values are scaled by
//                    powers of two that put the largest possible one just inside float16's range (|X| < 1.9, A < 3.61, |Q| < 8: the host checks the
//                    coefficients), which leaves lo's subnormal steps far below what matters.  The errors of many entries average out: the
//                    result is as far from the exact one as that of float32 products (256 x 256: 1.5e-6 both; 1024 x 1024: 2.8e-6 and 2.6e-6).
//   min(m, n) <= 64  float32 operands and instructions: the few entries of A and Q are shared by a whole row, a rounding of theirs does not average
//                    out (4 x 64 with split operands: twice the error), and the work is too small for its rate to matter.
//
// A, A^2 and Q are symmetric.  Every product is of the form C = L R^T with both operands stored along k: A = X X^T, A^2 = A A^T, and
// Q X = Q (X^T)^T, for which X is kept in both orders.  The polynomial is the epilogue of the product in front of it, the split into hi and lo the
// epilogue of all three; a X needs no pass of its own, it is the a on Q's diagonal.
//
//   up to 64 x 64      one workgroup per matrix, everything in LDS, one launch for a whole list: bound by the latency of 15 dependent products
//   m <= 64 < n        workgroups take columns of X; each adds up everyone's share of A, works out Q for itself, and turns its columns, whose
//                      share of the next A it leaves for the next launch: one launch per step
//   larger             tiled products over all matrices of the list at once: one launch for the norms, one for the split, three per step
#pragma once
#include "learning_common.hpp"

namespace mbt_learning {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float kScaleX = 32768.0f, kScaleA = 16384.0f, kScaleQ = 8192.0f;
constexpr int kNormBlocks = 64;  // workgroups that add up one matrix's squares
constexpr int kMostGroups = 16;  // matrix shapes of one launch, by value in its arguments

struct MatrixGroup {  // `batch` matrices of one shape
  const void* in;
  void* out;
  int64_t in_batch, in_row, in_column, out_batch, out_row, out_column;  // strides of the matrix as the kernels see it: m <= n, turned if it was taller
  int32_t m, n, mp, np;        // sizes, padded to the tile
  int64_t first;               // first tile or workgroup of this launch
  int64_t planes;              // where its planes start in the workspace, in halfs (flat: floats); each matrix of the batch has `stride` of them
  int64_t stride;
  int64_t batch;
  int32_t shares;              // (flat) workgroups per matrix
  int32_t reserved;
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

// ---- min(m, n) <= 64: float32, sixteen waves, a 16 x 16 tile of every product each ----------------------------------------------------
constexpr int kSmall = 64, kPitch = kSmall + 4;  // floats; rows 272 bytes apart put the 16 rows of an operand read into 64 different banks
constexpr int kSmallPlane = kSmall * kPitch;
constexpr size_t kSmallLds = 4 * kSmallPlane * sizeof(float);  // X, X^T, A, Q
constexpr int kMostShares = 32;                                // workgroups that share one flat matrix

// the 16 x 16 tile of L R^T at (row, column).  A lane holds four neighbours along k of its row; which k an instruction's four slots stand for does not
// matter as long as both operands agree.
__device__ __forceinline__ float4v tile_product(const float* l, const float* r, int row, int column, int kp) {
  const int lane = threadIdx.x & 63, at = (lane & 15) * kPitch + 4 * (lane >> 4);
  const float *lp = l + row * kPitch + at, *rp = r + column * kPitch + at;
  float4v acc = {0.f, 0.f, 0.f, 0.f}, odd = {0.f, 0.f, 0.f, 0.f};  // (two chains: an instruction need not wait for the one before it)
#pragma unroll
  for (int k = 0; k < kSmall; k += 16) {
    if (k >= kp) break;
    const float4v a = *reinterpret_cast<const float4v*>(lp + k), b = *reinterpret_cast<const float4v*>(rp + k);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, acc, 0, 0, 0);
    odd = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, odd, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, acc, 0, 0, 0);
    odd = __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, odd, 0, 0, 0);
  }
  return acc + odd;
}

struct SmallTile {
  int row, column;  // of this wave's tile
  int r0, c0;       // an accumulator's element r of this lane is at (row + r0 + r, column + c0)
  __device__ __forceinline__ SmallTile() {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    row = 16 * (wave >> 2);
    column = 16 * (wave & 3);
    r0 = 4 * (lane >> 4);
    c0 = lane & 15;
  }
  // four rows of one column, stored as four neighbours of a row of the transpose
  __device__ __forceinline__ void put_turned(float* plane, float4v v) const { *reinterpret_cast<float4v*>(plane + (column + c0) * kPitch + row + r0) = v; }
  __device__ __forceinline__ void put(float* plane, float4v v) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) plane[(row + r0 + r) * kPitch + column + c0] = v[r];
  }
};

// Q from A, both in LDS; every wave calls it, mp a multiple of 16
__device__ __forceinline__ void small_polynomial(const OrthogonaliseParams& P, const SmallTile& T, const float* am, float* q, int mp) {
  if (T.row < mp && T.column < mp) {
    const float4v square = tile_product(am, am, T.row, T.column, mp);
    const float4v av = *reinterpret_cast<const float4v*>(am + (T.column + T.c0) * kPitch + T.row + T.r0);
    float4v v;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] = __builtin_fmaf(P.b, av[r], P.c * square[r]);
      if (T.row + T.r0 + r == T.column + T.c0) v[r] += P.a;
    }
    T.put_turned(q, v);
  }
}

template <typename E>
__global__ __launch_bounds__(1024) void orthogonalise_small(const OrthogonaliseParams P) {
  extern __shared__ float lds_small[];
  __shared__ double sums[16];
  int64_t which;
  const MatrixGroup M = P.group[find_group(P, blockIdx.x, which)];
  const E* in = static_cast<const E*>(M.in) + which * M.in_batch;
  E* out = static_cast<E*>(M.out) + which * M.out_batch;
  float *x = lds_small, *xt = x + kSmallPlane, *am = xt + kSmallPlane, *q = am + kSmallPlane;
  float v[4];
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = threadIdx.x + 1024 * k, i = at >> 6, j = at & 63;
    v[k] = i < M.m && j < M.n ? static_cast<float>(in[i * M.in_row + j * M.in_column]) : 0.0f;
    sum += static_cast<double>(v[k]) * static_cast<double>(v[k]);
  }
  sum = block_sum(sum, sums);
  const double inverse = 1.0 / (sqrt(sum) + P.eps);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = threadIdx.x + 1024 * k, i = at >> 6, j = at & 63;
    const float scaled = static_cast<float>(v[k] * inverse);
    x[i * kPitch + j] = scaled;
    xt[j * kPitch + i] = scaled;
  }
  __syncthreads();
  const SmallTile T;
  const bool square = T.row < M.mp && T.column < M.mp, flat = T.row < M.mp && T.column < M.np;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  for (int step = 0; step < P.steps; ++step) {
    if (square) T.put_turned(am, tile_product(x, x, T.row, T.column, M.np));  // (symmetric)
    __syncthreads();
    small_polynomial(P, T, am, q, M.mp);
    __syncthreads();
    if (flat) acc = tile_product(q, xt, T.row, T.column, M.mp);
    if (step + 1 == P.steps) break;
    __syncthreads();  // X^T has been read
    if (flat) {
      T.put(x, acc);
      T.put_turned(xt, acc);
    }
    __syncthreads();
  }
  if (flat) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = T.row + T.r0 + r, j = T.column + T.c0;
      if (i < M.m && j < M.n) out[i * M.out_row + j * M.out_column] = static_cast<E>(acc[r]);
    }
  }
}

// One step of a flat matrix (m <= 64 < n), `shares` workgroups each, which take its blocks of 64 columns in turn.  Workspace per matrix, in floats:
// X (64 x np, by blocks of 64 x 64), then the shares of A (64 x 64 each) of this step and the next.  Launch 0 brings X in and leaves the first shares;
// launch s = 1 .. steps turns X, the last one into the output.
template <typename E>
__global__ __launch_bounds__(1024) void orthogonalise_flat(const OrthogonaliseParams P, int launch) {
  extern __shared__ float lds_small[];
  __shared__ double sums[16];
  int64_t at;
  const int group = find_group(P, blockIdx.x, at);
  const MatrixGroup M = P.group[group];
  const int shares = M.shares, share = static_cast<int>(at % shares), column_blocks = M.np / 64;
  const int64_t which = at / shares;
  float* xs = reinterpret_cast<float*>(P.planes) + M.planes + which * M.stride;
  float* const all_shares = xs + 64 * static_cast<int64_t>(M.np);
  const float* before = all_shares + (launch & 1 ? 0 : 1) * static_cast<int64_t>(kMostShares) * 4096;
  float* after = all_shares + (launch & 1 ? 1 : 0) * static_cast<int64_t>(kMostShares) * 4096;
  float *x = lds_small, *xt = x + kSmallPlane, *am = xt + kSmallPlane, *q = am + kSmallPlane;
  const SmallTile T;
  const int mp = M.mp;
  const bool square = T.row < mp && T.column < mp, flat = T.row < mp;
  double inverse = 0.0;
  if (launch == 0) {
    int64_t matrix = which;
    for (int g = 0; g < group; ++g) matrix += P.group[g].batch;
    const double norm = block_sum(threadIdx.x < kNormBlocks ? P.partials[matrix * kNormBlocks + threadIdx.x] : 0.0, sums);
    inverse = 1.0 / (sqrt(norm) + P.eps);
  } else {  // A: everyone's shares, in their order
    float4v a = {0.f, 0.f, 0.f, 0.f};
    const int i = threadIdx.x >> 4, j = 4 * (threadIdx.x & 15);
#pragma unroll 8
    for (int w = 0; w < shares; ++w) a += *reinterpret_cast<const float4v*>(before + w * 4096 + i * 64 + j);
    *reinterpret_cast<float4v*>(am + i * kPitch + j) = a;
    __syncthreads();
    small_polynomial(P, T, am, q, mp);
  }
  const E* in = static_cast<const E*>(M.in) + which * M.in_batch;
  E* out = static_cast<E*>(M.out) + which * M.out_batch;
  const bool along_n = M.in_column <= M.in_row;
  float4v gram = {0.f, 0.f, 0.f, 0.f};
  for (int block = share; block < column_blocks; block += shares) {
    const int j0 = 64 * block;
    float* mine = xs + static_cast<int64_t>(block) * 4096;
    __syncthreads();  // (the block before has been read, Q is written)
    if (launch == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = threadIdx.x + 1024 * k, i = along_n ? e >> 6 : e & 63, j = along_n ? e & 63 : e >> 6;
        const float v = i < M.m && j0 + j < M.n ? static_cast<float>(static_cast<float>(in[i * M.in_row + (j0 + j) * M.in_column]) * inverse) : 0.0f;
        x[i * kPitch + j] = v;
        mine[i * 64 + j] = v;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = threadIdx.x + 1024 * k, i = e >> 6, j = e & 63;
        xt[j * kPitch + i] = mine[e];
      }
      __syncthreads();
      if (flat) {
        const float4v acc = tile_product(q, xt, T.row, T.column, mp);
        if (P.last) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = T.row + T.r0 + r, j = j0 + T.column + T.c0;
            if (i < M.m && j < M.n) out[i * M.out_row + j * M.out_column] = static_cast<E>(acc[r]);
          }
        } else {
          T.put(x, acc);
#pragma unroll
          for (int r = 0; r < 4; ++r) mine[(T.row + T.r0 + r) * 64 + T.column + T.c0] = acc[r];
        }
      }
    }
    if (P.last) continue;
    __syncthreads();
    if (square) gram += tile_product(x, x, T.row, T.column, 64);
  }
  if (P.last) return;
  *reinterpret_cast<float4v*>(after + share * 4096 + (T.column + T.c0) * 64 + T.row + T.r0) = gram;  // (zeros where there is no tile)
}

// ---- larger ------------------------------------------------------------------------------------------------------------------------
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
