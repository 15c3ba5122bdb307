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
constexpr int kNormBlocks = 256;  // workgroups at most that add up one matrix's squares
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
  int32_t norm_blocks;         // workgroups that add up its squares
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

// A barrier over what the workgroup has in LDS: __syncthreads() also waits for every load from memory that is on its way, which is what a pipeline
// that runs steps ahead must not do.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
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

// 1 / (|G| + eps) from the sum of squares; a matrix of zeros stays zero without an eps too
__device__ __forceinline__ double inverse_norm(double sum, double eps) {
  const double norm = sqrt(sum) + eps;
  return norm == 0.0 ? 0.0 : 1.0 / norm;
}

__device__ __forceinline__ int find_group(const OrthogonaliseParams& P, int64_t block, int64_t& at) {
  int g = 0;
  while (g + 1 < P.groups && block >= P.group[g + 1].first) ++g;
  at = block - P.group[g].first;
  return g;
}

__device__ __forceinline__ int64_t matrices_before(const OrthogonaliseParams& P, int group) {
  int64_t n = 0;
  for (int g = 0; g < group; ++g) n += P.group[g].batch;
  return n;
}

// ---- min(m, n) <= 64: float32, sixteen waves, a 16 x 16 tile of every product each ----------------------------------------------------
constexpr int kSmall = 64, kSmallPlane = kSmall * kSmall;
constexpr size_t kSmallLds = 4 * kSmallPlane * sizeof(float);  // X, X^T, A, Q
constexpr int kMostShares = 32;                                // workgroups that share one flat matrix

// where element (row, column) of a plane lies: the 16-byte pieces of a row are exchanged by its number, so that the lanes of a 16-byte read - the same piece
// of sixteen rows, or neighbouring pieces of half of them - meet different banks
__device__ __forceinline__ int small_at(int row, int column) { return row * kSmall + (((column >> 2) ^ row) & 15) * 4 + (column & 3); }

// the 16 x 16 tile of L R^T at (row, column).  A lane holds four neighbours along k of its row; which k an instruction's four slots stand for does not
// matter as long as both operands agree.
__device__ __forceinline__ float4v tile_product(const float* l, const float* r, int row, int column, int kp) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const float *lp = l + (row + i) * kSmall, *rp = r + (column + i) * kSmall;
  float4v acc = {0.f, 0.f, 0.f, 0.f}, odd = {0.f, 0.f, 0.f, 0.f};  // (two chains: an instruction need not wait for the one before it)
#pragma unroll
  for (int k = 0; k < kSmall; k += 16) {
    if (k >= kp) break;
    const int piece = ((k >> 2) + g ^ i) * 4;  // (row and column are multiples of 16: i is the row's number as far as the exchange goes)
    const float4v a = *reinterpret_cast<const float4v*>(lp + piece), b = *reinterpret_cast<const float4v*>(rp + piece);
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
  // SYMMETRIC: the ten tiles of the upper triangle to the first ten waves - at most three on a SIMD, which would have to work on four of a full product
  __device__ __forceinline__ SmallTile(bool symmetric) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int i = wave >> 2, j = wave & 3;
    if (symmetric) {
      i = 0;
      j = wave;
      while (i < 4 && j >= 4 - i) j -= 4 - i, ++i;
      j += i;
    }
    row = 16 * i;
    column = 16 * j;
    r0 = 4 * (lane >> 4);
    c0 = lane & 15;
  }
  // four rows of one column, stored as four neighbours of a row of the transpose
  __device__ __forceinline__ void put_turned(float* plane, float4v v) const { *reinterpret_cast<float4v*>(plane + small_at(column + c0, row + r0)) = v; }
  __device__ __forceinline__ void put(float* plane, float4v v) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) plane[small_at(row + r0 + r, column + c0)] = v[r];
  }
  __device__ __forceinline__ void put_symmetric(float* plane, float4v v) const {
    put_turned(plane, v);
    if (row != column) put(plane, v);
  }
};

// Q from A, both in LDS; every wave calls it with its tile of a symmetric product, mp a multiple of 16
__device__ __forceinline__ void small_polynomial(const OrthogonaliseParams& P, const SmallTile& T, const float* am, float* q, int mp) {
  if (T.row < mp && T.column < mp) {
    const float4v square = tile_product(am, am, T.row, T.column, mp);
    const float4v av = *reinterpret_cast<const float4v*>(am + small_at(T.column + T.c0, T.row + T.r0));
    float4v v;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] = __builtin_fmaf(P.b, av[r], P.c * square[r]);
      if (T.row + T.r0 + r == T.column + T.c0) v[r] += P.a;
    }
    T.put_symmetric(q, v);
  }
}

// One matrix per workgroup: 20 us for a launch with a 64 x 64 one, 15 products that wait for one another.  Their matrix instructions alone take 25600
// cycles of the fullest SIMD, 12 us (4 tiles of 16 instructions of 32 cycles; 3 tiles where the product is symmetric: 22.3 us a launch without that); the
// rest is reads of LDS and the barriers between them.
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
  const double inverse = inverse_norm(sum, P.eps);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = threadIdx.x + 1024 * k, i = at >> 6, j = at & 63;
    const float scaled = static_cast<float>(v[k] * inverse);
    x[small_at(i, j)] = scaled;
    xt[small_at(j, i)] = scaled;
  }
  __syncthreads();
  const SmallTile T(false), S(true);
  const bool square = S.row < M.mp && S.column < M.mp, flat = T.row < M.mp && T.column < M.np;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  for (int step = 0; step < P.steps; ++step) {
    if (square) S.put_symmetric(am, tile_product(x, x, S.row, S.column, M.np));
    __syncthreads();
    small_polynomial(P, S, am, q, M.mp);
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
// launch s = 1 .. steps turns X, the last one into the output.  64 x 1000: 61 us for the seven launches, each the latency of its chain of four products
// and of summing the shares; 16 x 1000: 49 us; 64 x 20000: 192 us.
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
  const SmallTile T(false), S(true);
  const int mp = M.mp;
  const bool square = S.row < mp && S.column < mp, flat = T.row < mp;
  double inverse = 0.0;
  if (launch == 0) {
    const double* partials = P.partials + (which + matrices_before(P, group)) * kNormBlocks;
    inverse = inverse_norm(block_sum(threadIdx.x < M.norm_blocks ? partials[threadIdx.x] : 0.0, sums), P.eps);
  } else {  // A: everyone's shares, in their order
    float4v a = {0.f, 0.f, 0.f, 0.f};
    const int i = threadIdx.x >> 4, j = 4 * (threadIdx.x & 15);
#pragma unroll 8
    for (int w = 0; w < shares; ++w) a += *reinterpret_cast<const float4v*>(before + w * 4096 + i * 64 + j);
    *reinterpret_cast<float4v*>(am + small_at(i, j)) = a;
    __syncthreads();
    small_polynomial(P, S, am, q, mp);
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
        x[small_at(i, j)] = v;
        mine[i * 64 + j] = v;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = threadIdx.x + 1024 * k, i = e >> 6, j = e & 63;
        xt[small_at(j, i)] = mine[e];
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
    if (square) gram += tile_product(x, x, S.row, S.column, 64);
  }
  if (P.last) return;
  // the whole 64 x 64: what this share has of A, its mirror image, and zeros where A has no tile
  if (S.row < 64) {
    float* share_of = after + share * 4096;
    *reinterpret_cast<float4v*>(share_of + (S.column + S.c0) * 64 + S.row + S.r0) = gram;
    if (S.row != S.column) {
#pragma unroll
      for (int r = 0; r < 4; ++r) share_of[(S.row + S.r0 + r) * 64 + S.column + S.c0] = gram[r];
    }
  }
}

// ---- larger ------------------------------------------------------------------------------------------------------------------------
// A matrix as a product reads it: cut into tiles of 16 rows x 32 along k, each tile 1 KB of hi followed by 1 KB of lo, the tiles of one k step
// behind one another - what a workgroup needs for a step is contiguous, and one load of a wave is one tile, whole lines of it.
struct Tiled {
  _Float16* p;
  int row_tiles;  // of the matrix
  __device__ __forceinline__ int64_t at(int row, int k) const {
    return (static_cast<int64_t>(k >> 5) * row_tiles + (row >> 4)) * 1024 + (row & 15) * 32 + (k & 31);
  }
};
constexpr int kLo = 512;  // halfs from hi to lo

// of one matrix: X (m x n), X^T twice, A, Q
struct Planes {
  Tiled x, xt, xt_next, a, q;  // (X^T of this step and of the next)
};
__device__ __forceinline__ Planes planes_of(const OrthogonaliseParams& P, const MatrixGroup& M, int64_t which) {
  const int64_t xs = 2 * static_cast<int64_t>(M.mp) * M.np, as = 2 * static_cast<int64_t>(M.mp) * M.mp;
  _Float16* p = P.planes + M.planes + which * M.stride;
  const int m = M.mp / 16, n = M.np / 16;
  return {{p, m}, {p + (P.odd ? 2 : 1) * xs, n}, {p + (P.odd ? 1 : 2) * xs, n}, {p + 3 * xs, m}, {p + 3 * xs + as, m}};
}

// sum of squares of one matrix, norm_blocks workgroups each, 4096 elements of them at a time; four loads of a thread at a time.
// 2048 x 2048 float32: 9.9 us (16 MB), small ones 6: latency, and a launch of as many workgroups as there are elements for
template <typename E>
__global__ __launch_bounds__(1024) void orthogonalise_norms(const OrthogonaliseParams P) {
  __shared__ double lds[16];
  int64_t at;
  const int group = find_group(P, blockIdx.x, at);
  const MatrixGroup M = P.group[group];
  const int64_t which = at / M.norm_blocks;
  const uint32_t part = static_cast<uint32_t>(at % M.norm_blocks);
  const E* in = static_cast<const E*>(M.in) + which * M.in_batch;
  const bool along_n = M.in_column <= M.in_row;  // neighbours in memory to neighbouring threads
  const uint32_t fast = along_n ? M.n : M.m, count = static_cast<uint32_t>(M.m) * static_cast<uint32_t>(M.n);  // (at most 2^30)
  const int64_t fast_stride = along_n ? M.in_column : M.in_row, slow_stride = along_n ? M.in_row : M.in_column;
  double sum = 0.0;
  for (uint32_t first = part * 4096; first < count; first += M.norm_blocks * 4096) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t e = first + 1024 * k + threadIdx.x;
      v[k] = e < count ? static_cast<float>(in[(e / fast) * slow_stride + (e % fast) * fast_stride]) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sum += static_cast<double>(v[k]) * static_cast<double>(v[k]);
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) P.partials[(which + matrices_before(P, group)) * kNormBlocks + part] = sum;
}

// X = G / (|G| + eps) in both orders, 64 x 64 at a time; M.first counts such tiles.  2048 x 2048: 11.6 us for 48 MB (17 with stores of single halfs)
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
  const E* in = static_cast<const E*>(M.in) + which * M.in_batch;
  const bool along_n = M.in_column <= M.in_row;
  float v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int e = threadIdx.x + 256 * k, i = along_n ? e >> 6 : e & 63, j = along_n ? e & 63 : e >> 6;
    v[k] = i0 + i < M.m && j0 + j < M.n ? static_cast<float>(in[(i0 + i) * M.in_row + (j0 + j) * M.in_column]) : 0.0f;
  }
  const double* partials = P.partials + (which + matrices_before(P, group)) * kNormBlocks;
  // (the inverse of a norm beyond 2^126 is no normal float32 number, that of one below 2^-128 no finite one: a power of two, which brings an element to at
  // most two, and what is left of it.  A product in 64 bits per element: 15.7 us instead of 11.6 at 2048 x 2048)
  int exponent;
  const float inverse = static_cast<float>(frexp(inverse_norm(block_sum(threadIdx.x < M.norm_blocks ? partials[threadIdx.x] : 0.0, lds), P.eps), &exponent));
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int e = threadIdx.x + 256 * k, i = along_n ? e >> 6 : e & 63, j = along_n ? e & 63 : e >> 6;
    tile[i][j] = ldexpf(v[k], exponent) * inverse * kScaleX;
  }
  __syncthreads();
  const Planes p = planes_of(P, M, which);
  // eight neighbours along k at once; four lanes after one another write a row of a tile
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int e = threadIdx.x + 256 * k, s = e >> 2 & 63, f = 8 * (e & 3) + 32 * (e >> 8);
    half8 xh, xl, th, tl;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const Halves h = split(tile[s][f + i]), g = split(tile[f + i][s]);
      xh[i] = h.hi;
      xl[i] = h.lo;
      th[i] = g.hi;
      tl[i] = g.lo;
    }
    half8 *x = reinterpret_cast<half8*>(p.x.p + p.x.at(i0 + s, j0 + f)), *xt = reinterpret_cast<half8*>(p.xt.p + p.xt.at(j0 + s, i0 + f));
    x[0] = xh;
    x[kLo / 8] = xl;
    xt[0] = th;
    xt[kLo / 8] = tl;
  }
}

// The order of a step's instructions: products with the reads, writes and loads strewn in between.  Left alone the requests come first, every wave's at
// once, and no product starts before LDS has taken them all.
template <int PRODUCTS, int READS, int TRANSFERS>
__device__ __forceinline__ void interleave() {
  constexpr int kRequests = READS + 2 * TRANSFERS, kEach = PRODUCTS / kRequests > 0 ? PRODUCTS / kRequests : 1;
#pragma unroll
  for (int i = 0; i < READS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      // LDS read
    __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);  // products
  }
#pragma unroll
  for (int i = 0; i < TRANSFERS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);      // LDS write
    __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);      // load from memory
    __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
  }
}

// Where the 16-byte piece `piece` of a 64-byte row lies in LDS: the pieces of four rows are exchanged differently in each of the four quarters of a tile, so
// that the sixteen lanes that a 16-byte read serves at a time - a run of rows, or half of them with the neighbouring piece of the other half - meet
// sixteen different groups of banks.  (Rows 80 bytes apart are free of conflicts only for the first of these; counters showed half of LDS's time lost.)
__device__ __forceinline__ int swizzle(int row, int piece) { return piece ^ (-(row >> 2) & 3); }

enum : int { kGram = 0, kPolynomial = 1, kApply = 2 };

// The t-th tile: by bands of eight columns of tiles, row by row within a band, so that the run of tiles that one XCD works on is compact and its L2 is
// asked for few rows of either operand.  Of a symmetric product, the upper triangle.
template <bool SYMMETRIC>
__device__ __forceinline__ void find_tile(int t, int rows, int columns, int& ti, int& tj) {
  constexpr int kBand = 8;
  for (int c0 = 0;; c0 += kBand) {
    const int width = columns - c0 < kBand ? columns - c0 : kBand;
    if (!SYMMETRIC) {
      if (t < rows * width) {
        ti = t / width;
        tj = c0 + t % width;
        return;
      }
      t -= rows * width;
    } else {
      if (t < c0 * width) {  // the rows above the band's own square have all of the band
        ti = t / width;
        tj = c0 + t % width;
        return;
      }
      t -= c0 * width;
      for (ti = c0; ti < c0 + width; ++ti) {
        const int n = c0 + width - ti;
        if (t < n) {
          tj = ti + t;
          return;
        }
        t -= n;
      }
    }
  }
}

// One T x T tile of a product, WAVES waves of T/2 x 2 T/WAVES, k in steps of 32.  Three products of matrix instructions per step of one split
// operand pair: 128 x 128 with eight waves has 768 cycles of them per SIMD and step, against 650 cycles of LDS (96 KB read, 32 KB written).
// Measured at 2048 x 2048: 41 us for a symmetric product (136 workgroups on 256 compute units), 53 for the full one (47 at best), where the matrix instructions
// alone - the loop without its reads, writes and loads - take 32 and 36; 64 x 64 tiles take 46 and 70 there, but 11 and 13 us instead of 21 and 23
// at 1024 x 1024, where 128 x 128 ones are too few.  What brought it there from 70 us: a barrier that does not wait for loads from memory (60), the
// requests strewn between the products (53), LDS without bank conflicts (44).  What bounds it now: LDS writes and the barrier per step.
template <typename E, int T, int WAVES, int PRODUCT>
__global__ __launch_bounds__(64 * WAVES, 2) void orthogonalise_product(const OrthogonaliseParams P) {
  constexpr int kRow = 32;                       // halfs of a row in LDS
  constexpr int kPlane = T * kRow, kBuffer = 4 * kPlane;  // L hi, L lo, R hi, R lo
  constexpr int FI = T / 32, FJ = 2 * T / WAVES / 16;  // 16 x 16 fragments of a wave along rows and columns
  constexpr int kSweep = 16 * WAVES;             // rows that the workgroup loads at once: a tile per wave
  constexpr int kTiles = T / kSweep, kTransfers = 4 * kTiles;  // of an operand that a wave loads; of both, in halves
  // steps whose operands wait in registers or are on their way: even, since fragments alternate with it, and a divisor of every number of steps
  constexpr int kAhead = T / 32;
  static_assert(kTiles >= 1 && FJ >= 1 && kAhead % 2 == 0, "a tile has work for every wave");
  extern __shared__ _Float16 lds_product[];
  // neighbouring tiles to the same XCD (workgroups go round the eight of them), so that its L2 sees an operand's rows again
  const int64_t blocks = P.blocks, per = (blocks + 7) / 8;
  const int64_t id = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (id >= blocks) return;
  int64_t at;
  const MatrixGroup M = P.group[find_group(P, id, at)];
  const int rows = M.mp / T, columns = (PRODUCT == kApply ? M.np : M.mp) / T;
  const int tiles = PRODUCT == kApply ? rows * columns : rows * (rows + 1) / 2;
  const int64_t which = at / tiles;
  int ti, tj;
  find_tile<PRODUCT != kApply>(static_cast<int>(at % tiles), rows, columns, ti, tj);
  const Planes p = planes_of(P, M, which);
  const int kp = PRODUCT == kGram ? M.np : M.mp;  // both operands' row length
  const Tiled left = PRODUCT == kGram ? p.x : PRODUCT == kPolynomial ? p.a : p.q;
  const Tiled right = PRODUCT == kGram ? p.x : PRODUCT == kPolynomial ? p.a : p.xt;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = T / 2 * (wave & 1), column = 16 * FJ * (wave >> 1);
  float4v acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};
  // kAhead steps' operands wait in registers or are on their way: a step takes a third of a memory latency
  half8 stage[kAhead][kTransfers];
  const int load_row = threadIdx.x / 4, load_k = 8 * swizzle(load_row, threadIdx.x % 4);  // a wave's lanes walk through one tile
  const _Float16* l = left.p + static_cast<int64_t>(ti) * (T / 16) * 1024 + wave * 1024 + lane * 8;
  const _Float16* r = right.p + static_cast<int64_t>(tj) * (T / 16) * 1024 + wave * 1024 + lane * 8;
  const int64_t l_step = left.row_tiles * 1024, r_step = right.row_tiles * 1024;
  const int steps = kp / 32;
  // (steps behind the last fetch the last one again and nobody looks: without branches around loads the compiler knows which ones a wait is for)
  auto fetch = [&](int ahead, half8 (&to)[kTransfers]) {
    const int step = ahead < steps ? ahead : steps - 1;
    const _Float16 *lp = l + step * l_step, *rp = r + step * r_step;
#pragma unroll
    for (int s = 0; s < kTiles; ++s) {
      to[4 * s] = *reinterpret_cast<const half8*>(lp + s * WAVES * 1024);
      to[4 * s + 1] = *reinterpret_cast<const half8*>(lp + s * WAVES * 1024 + kLo);
      to[4 * s + 2] = *reinterpret_cast<const half8*>(rp + s * WAVES * 1024);
      to[4 * s + 3] = *reinterpret_cast<const half8*>(rp + s * WAVES * 1024 + kLo);
    }
  };
  auto put = [&](int buffer, const half8 (&from)[kTransfers]) {
    _Float16* base = lds_product + buffer * kBuffer + load_row * kRow + load_k;
#pragma unroll
    for (int s = 0; s < kTiles; ++s)
#pragma unroll
      for (int plane = 0; plane < 4; ++plane) *reinterpret_cast<half8*>(base + plane * kPlane + s * kSweep * kRow) = from[4 * s + plane];
  };
  struct Fragments {
    half8 lh[FI], ll[FI], rh[FJ], rl[FJ];
  };
  auto read = [&](int buffer, Fragments& f) {
    const _Float16* base = lds_product + buffer * kBuffer + (lane & 15) * kRow + 8 * swizzle(lane & 15, lane >> 4);
#pragma unroll
    for (int j = 0; j < FJ; ++j) f.rl[j] = *reinterpret_cast<const half8*>(base + 3 * kPlane + (column + 16 * j) * kRow);
#pragma unroll
    for (int i = 0; i < FI; ++i) f.lh[i] = *reinterpret_cast<const half8*>(base + (row + 16 * i) * kRow);
#pragma unroll
    for (int j = 0; j < FJ; ++j) f.rh[j] = *reinterpret_cast<const half8*>(base + 2 * kPlane + (column + 16 * j) * kRow);
#pragma unroll
    for (int i = 0; i < FI; ++i) f.ll[i] = *reinterpret_cast<const half8*>(base + kPlane + (row + 16 * i) * kRow);
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) {
    fetch(d, stage[d]);
    asm volatile("" ::: "memory");  // (in their order: a wait in the loop counts the loads behind the one it is for)
    __builtin_amdgcn_sched_barrier(0);
  }
  put(0, stage[0]);
  fetch(kAhead, stage[0]);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  put(1, stage[1]);
  fetch(kAhead + 1, stage[1]);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  lds_barrier();
  // Step s multiplies the fragments it finds in registers, while those of step s + 1 come from one LDS buffer, step s + 2 is put into another - the
  // third is the one that step s itself came from - and step s + 2 + kAhead is requested from memory.
  Fragments fragments[2];
  read(0, fragments[0]);
  int next = 1, fill = 2;
  for (int first = 0; first < steps; first += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      read(next, fragments[(d + 1) & 1]);
      put(fill, stage[(d + 2) % kAhead]);
      fetch(first + d + 2 + kAhead, stage[(d + 2) % kAhead]);
      const Fragments& f = fragments[d & 1];
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int i = 0; i < FI; ++i) acc[i][j] = mfma(f.lh[i], f.rl[j], acc[i][j]);
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int i = 0; i < FI; ++i) acc[i][j] = mfma(f.lh[i], f.rh[j], acc[i][j]);
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int i = 0; i < FI; ++i) acc[i][j] = mfma(f.ll[i], f.rh[j], acc[i][j]);
      interleave<3 * FI * FJ, 2 * (FI + FJ), kTransfers>();
      __builtin_amdgcn_sched_barrier(0);  // (no product sinks below the barrier, in front of the next step's requests)
      next = fill;
      fill = fill == 2 ? 0 : fill + 1;
      lds_barrier();
    }
  }

  const int r0 = 4 * (lane >> 4), c0 = lane & 15;
  if (PRODUCT == kApply && P.last) {
    E* out = static_cast<E*>(M.out) + which * M.out_batch;
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t y = ti * T + row + 16 * i + r0 + e, z = tj * T + column + 16 * j + c0;
          if (y < M.m && z < M.n) out[y * M.out_row + z * M.out_column] = static_cast<E>(acc[i][j][e] * (1.0f / kScaleQ / kScaleX));
        }
    return;
  }
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int y = ti * T + row + 16 * i + r0, z = tj * T + column + 16 * j + c0;  // four rows y.., one column z
      half4 hi, lo;
      half4 ah, al;
      if (PRODUCT == kPolynomial) {  // A at (y + e, z) is A at (z, y + e)
        const _Float16* a = p.a.p + p.a.at(z, y);
        ah = *reinterpret_cast<const half4*>(a);
        al = *reinterpret_cast<const half4*>(a + kLo);
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
      const Tiled turned = PRODUCT == kGram ? p.a : PRODUCT == kPolynomial ? p.q : p.xt_next;
      _Float16* to = turned.p + turned.at(z, y);
      *reinterpret_cast<half4*>(to) = hi;
      *reinterpret_cast<half4*>(to + kLo) = lo;
      if (PRODUCT == kApply || ti != tj) {
        const Tiled plain = PRODUCT == kApply ? p.x : turned;
        _Float16* as_is = plain.p + plain.at(y, z);  // (y is a multiple of four: y + e stays within its tile)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          as_is[32 * e] = hi[e];
          as_is[32 * e + kLo] = lo[e];
        }
      }
    }
}

}  // namespace mbt_learning
