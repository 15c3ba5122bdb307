// The C entry point of the Newton-Schulz orthogonalisation: argument checks, how a list of matrices is cut into launches (kernels: orthogonal.hpp).
#include <atomic>
#include <cmath>

#include "orthogonal.hpp"

namespace mbt_learning {
namespace {

constexpr uint32_t kMostSize = 32768;

int64_t padded(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
enum Kind { kSmallMatrix, kFlatMatrix, kLargeMatrix };
Kind kind_of(const mbt_matrix& m) {
  const uint32_t small = m.rows < m.columns ? m.rows : m.columns, large = m.rows < m.columns ? m.columns : m.rows;
  return large <= kSmall ? kSmallMatrix : small <= kSmall ? kFlatMatrix : kLargeMatrix;
}

// 128 x 128 tiles read every operand half as often as 64 x 64 ones, but there are a quarter as many: they win where they occupy three quarters of the
// compute units (2048 x 2048: 41 and 50 us a product against 46 and 70), and lose below (1024 x 1024: 21 and 23 against 11 and 13)
int tile_of(const mbt_matrix& m) {
  const int64_t small = m.rows < m.columns ? m.rows : m.columns, large = m.rows < m.columns ? m.columns : m.rows;
  return (padded(small, 128) / 128) * (padded(large, 128) / 128) * static_cast<int64_t>(m.batch) >= 192 ? 128 : 64;
}

MatrixGroup group_of(const mbt_matrix& m, int tile) {
  MatrixGroup g{};
  const bool turn = m.rows > m.columns;
  g.in = m.in;
  g.out = m.out;
  g.in_batch = m.in_stride[0];
  g.in_row = m.in_stride[turn ? 2 : 1];
  g.in_column = m.in_stride[turn ? 1 : 2];
  g.out_batch = m.out_stride[0];
  g.out_row = m.out_stride[turn ? 2 : 1];
  g.out_column = m.out_stride[turn ? 1 : 2];
  g.m = static_cast<int32_t>(turn ? m.columns : m.rows);
  g.n = static_cast<int32_t>(turn ? m.rows : m.columns);
  g.batch = static_cast<int64_t>(m.batch);
  const Kind kind = kind_of(m);
  const int64_t norm_blocks = (static_cast<int64_t>(g.m) * g.n + 4095) / 4096;
  g.norm_blocks = static_cast<int32_t>(norm_blocks < kNormBlocks ? norm_blocks : kNormBlocks);
  if (kind == kLargeMatrix) {
    g.mp = static_cast<int32_t>(padded(g.m, tile));
    g.np = static_cast<int32_t>(padded(g.n, tile));
    g.stride = 6 * static_cast<int64_t>(g.mp) * g.np + 4 * static_cast<int64_t>(g.mp) * g.mp;  // halfs (orthogonal.hpp: Planes)
  } else {
    g.mp = static_cast<int32_t>(padded(g.m, 16));
    g.np = static_cast<int32_t>(padded(g.n, kind == kSmallMatrix ? 16 : 64));
    g.shares = g.np / 64 < kMostShares ? g.np / 64 : kMostShares;
    g.stride = 64 * static_cast<int64_t>(g.np) + 2 * kMostShares * 4096;  // floats (orthogonal.hpp: orthogonalise_flat)
  }
  return g;
}

int check_matrices(uint32_t count, const mbt_matrix* matrices) {
  if (count < 1 || matrices == nullptr) return mbt_set_error(MBT_ERR_INVALID, "no matrices");
  uint64_t total = 0, blocks = 0;
  for (uint32_t k = 0; k < count; ++k) {
    const mbt_matrix& m = matrices[k];
    if (m.in == nullptr || m.out == nullptr) return mbt_set_error(MBT_ERR_INVALID, "matrix %u: null argument", k);
    if (m.rows < 1 || m.columns < 1 || m.rows > kMostSize || m.columns > kMostSize)
      return mbt_set_error(MBT_ERR_INVALID, "matrix %u is %u x %u: rows and columns lie within 1 .. %u", k, m.rows, m.columns, kMostSize);
    if (m.batch < 1 || m.batch > (uint64_t{1} << 24)) return mbt_set_error(MBT_ERR_INVALID, "matrix %u: a batch of %llu lies outside 1 .. 2^24", k, (unsigned long long)m.batch);
    const MatrixGroup g = group_of(m, 128);
    total += m.batch * (static_cast<uint64_t>(g.mp) * g.np / 4096 + 1);
    if (total > (uint64_t{1} << 28)) return mbt_set_error(MBT_ERR_INVALID, "more elements than one call takes (2^40)");
    // a launch counts its threads in 32 bits: in workgroups of 1024, the norms' for a matrix beyond 64 x 64, or the products' 64 x 64 tiles at 256 each
    const uint64_t tiles = static_cast<uint64_t>(g.mp) * g.np / 4096 / 4;
    blocks += m.batch * (kind_of(m) == kSmallMatrix ? 1 : tiles > kNormBlocks ? tiles : kNormBlocks);
    if (blocks >= (uint64_t{1} << 22)) return mbt_set_error(MBT_ERR_INVALID, "more matrices than one launch takes");
  }
  return MBT_OK;
}

// the tile that the large matrices of the call share (one launch works on all of them), and the halfs and partial sums they need
int common_tile(uint32_t count, const mbt_matrix* matrices) {
  int tile = 64;
  for (uint32_t k = 0; k < count; ++k)
    if (kind_of(matrices[k]) == kLargeMatrix && tile_of(matrices[k]) > tile) tile = 128;
  return tile;
}
uint64_t workspace_of(uint32_t count, const mbt_matrix* matrices) {
  uint64_t bytes = 0;
  const int tile = common_tile(count, matrices);
  for (uint32_t k = 0; k < count; ++k) {
    const Kind kind = kind_of(matrices[k]);
    if (kind == kSmallMatrix) continue;
    const MatrixGroup g = group_of(matrices[k], tile);
    bytes += matrices[k].batch * (static_cast<uint64_t>(g.stride) * (kind == kFlatMatrix ? sizeof(float) : sizeof(_Float16)) + kNormBlocks * sizeof(double));
  }
  return bytes;
}

// Singular values start within [0, 1]: what the largest can become, step by step (a grid fine enough for a polynomial of degree five, and 1 % on top).
bool bounded(int steps, const double c[3]) {
  double top = 1.0;
  for (int s = 0; s < steps; ++s) {
    double next = 0.0;
    for (int k = 0; k <= 2048; ++k) {
      const double x = top * k / 2048, y = x * x, q = c[0] + c[1] * y + c[2] * y * y;
      if (!(std::fabs(q) < 7.9)) return false;
      if (std::fabs(x * q) > next) next = std::fabs(x * q);
    }
    top = next * 1.01;
    if (!(top < 1.9)) return false;
  }
  return true;
}

// three buffers of two operands in two halves, 64 bytes a row
template <int T>
constexpr size_t kProductLds = 3 * 2 * 2 * T * 64;

template <int T>
constexpr int kWaves = T == 128 ? 8 : 4;

template <typename E, int T>
int run_products(OrthogonaliseParams& P, int64_t gram_tiles, int64_t apply_tiles, const int64_t (&gram_first)[kMostGroups], const int64_t (&apply_first)[kMostGroups],
                 hipStream_t stream) {
  constexpr size_t lds = kProductLds<T>;
  auto launch = [&](auto kernel, int64_t tiles, const int64_t (&first)[kMostGroups]) {
    for (int g = 0; g < P.groups; ++g) P.group[g].first = first[g];
    P.blocks = tiles;
    kernel<<<static_cast<unsigned>((tiles + 7) / 8 * 8), 64 * kWaves<T>, lds, stream>>>(P);
  };
  P.odd = 0;
  for (int step = 0; step < P.steps; ++step) {
    P.last = step + 1 == P.steps;
    launch(orthogonalise_product<E, T, kWaves<T>, kGram>, gram_tiles, gram_first);
    launch(orthogonalise_product<E, T, kWaves<T>, kPolynomial>, gram_tiles, gram_first);
    launch(orthogonalise_product<E, T, kWaves<T>, kApply>, apply_tiles, apply_first);
    P.odd ^= 1;
  }
  return launch_status("orthogonalise");
}

template <typename E>
int run_small(uint32_t count, const mbt_matrix* matrices, OrthogonaliseParams& P, hipStream_t stream) {
  P.groups = 0;
  int64_t blocks = 0;
  for (uint32_t k = 0; k <= count; ++k) {
    if (k < count) {
      if (kind_of(matrices[k]) != kSmallMatrix) continue;
      MatrixGroup& g = P.group[P.groups++];
      g = group_of(matrices[k], 0);
      g.first = blocks;
      blocks += g.batch;
    }
    if (P.groups == kMostGroups || (k == count && P.groups > 0)) {
      orthogonalise_small<E><<<static_cast<unsigned>(blocks), 1024, kSmallLds, stream>>>(P);
      const int rc = launch_status("orthogonalise");
      if (rc != MBT_OK) return rc;
      P.groups = 0;
      blocks = 0;
    }
  }
  return MBT_OK;
}

// Flat and large matrices, kMostGroups shapes at a time; `next` walks through the workspace.
template <typename E>
int run_kind(Kind kind, uint32_t count, const mbt_matrix* matrices, int tile, OrthogonaliseParams& P, char*& next, hipStream_t stream) {
  uint32_t k = 0;
  while (k < count) {
    int64_t matrices_in = 0, norm_blocks = 0, split_tiles = 0, gram_tiles = 0, apply_tiles = 0, elements = 0, shares = 0;
    int64_t norm_first[kMostGroups] = {}, split_first[kMostGroups] = {}, gram_first[kMostGroups] = {}, apply_first[kMostGroups] = {}, share_first[kMostGroups] = {};
    P.groups = 0;
    P.odd = 0;
    P.last = 0;
    for (; k < count && P.groups < kMostGroups; ++k) {
      if (kind_of(matrices[k]) != kind) continue;
      const int at = P.groups++;
      MatrixGroup& g = P.group[at];
      g = group_of(matrices[k], tile);
      g.planes = elements;
      elements += g.batch * g.stride;
      const int64_t rows = g.mp / tile, columns = g.np / tile;
      norm_first[at] = norm_blocks;
      split_first[at] = split_tiles;
      gram_first[at] = gram_tiles;
      apply_first[at] = apply_tiles;
      share_first[at] = shares;
      matrices_in += g.batch;
      norm_blocks += g.batch * g.norm_blocks;
      split_tiles += g.batch * (g.mp / 64) * (g.np / 64);
      gram_tiles += g.batch * (rows * (rows + 1) / 2);
      apply_tiles += g.batch * rows * columns;
      shares += g.batch * g.shares;
    }
    if (P.groups == 0) break;
    P.partials = reinterpret_cast<double*>(next);
    next += matrices_in * kNormBlocks * sizeof(double);
    P.planes = reinterpret_cast<_Float16*>(next);
    next += elements * (kind == kFlatMatrix ? sizeof(float) : sizeof(_Float16));
    auto place = [&](const int64_t (&first)[kMostGroups]) {
      for (int g = 0; g < P.groups; ++g) P.group[g].first = first[g];
    };
    place(norm_first);
    orthogonalise_norms<E><<<static_cast<unsigned>(norm_blocks), 1024, 0, stream>>>(P);
    int rc;
    if (kind == kFlatMatrix) {
      place(share_first);
      for (int launch = 0; launch <= P.steps; ++launch) {
        P.last = launch == P.steps;
        orthogonalise_flat<E><<<static_cast<unsigned>(shares), 1024, kSmallLds, stream>>>(P, launch);
      }
      rc = launch_status("orthogonalise");
    } else {
      place(split_first);
      orthogonalise_split<E><<<static_cast<unsigned>(split_tiles), 256, 0, stream>>>(P);
      rc = tile == 128 ? run_products<E, 128>(P, gram_tiles, apply_tiles, gram_first, apply_first, stream)
                       : run_products<E, 64>(P, gram_tiles, apply_tiles, gram_first, apply_first, stream);
    }
    if (rc != MBT_OK) return rc;
  }
  return MBT_OK;
}

template <typename E>
int run(uint32_t count, const mbt_matrix* matrices, OrthogonaliseParams& P, void* workspace, hipStream_t stream) {
  const int tile = common_tile(count, matrices);
  char* next = static_cast<char*>(workspace);
  int rc = run_small<E>(count, matrices, P, stream);
  if (rc == MBT_OK) rc = run_kind<E>(kFlatMatrix, count, matrices, tile, P, next, stream);
  if (rc == MBT_OK) rc = run_kind<E>(kLargeMatrix, count, matrices, tile, P, next, stream);
  return rc;
}

// the kernels' shared memory is beyond the 64 KB that a launch gets unasked; set once per device
template <typename E>
int allow_lds(int device) {
  static std::atomic<uint64_t> done{0};
  if (device < 64 && (done.load(std::memory_order_relaxed) >> device & 1)) return MBT_OK;
  LEARNING_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(orthogonalise_small<E>), hipFuncAttributeMaxDynamicSharedMemorySize, kSmallLds));
  LEARNING_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(orthogonalise_flat<E>), hipFuncAttributeMaxDynamicSharedMemorySize, kSmallLds));
  const int lds = static_cast<int>(kProductLds<128>);
  LEARNING_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(orthogonalise_product<E, 128, kWaves<128>, kGram>), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  LEARNING_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(orthogonalise_product<E, 128, kWaves<128>, kPolynomial>), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  LEARNING_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(orthogonalise_product<E, 128, kWaves<128>, kApply>), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  if (device < 64) done.fetch_or(1ull << device, std::memory_order_relaxed);
  return MBT_OK;
}

}  // namespace
}  // namespace mbt_learning

extern "C" {

uint64_t mbt_orthogonalise_workspace(uint32_t count, const mbt_matrix* matrices) {
  using namespace mbt_learning;
  return check_matrices(count, matrices) == MBT_OK ? workspace_of(count, matrices) : 0;
}

int mbt_orthogonalise(int device, int dtype, uint32_t count, const mbt_matrix* matrices, int steps, const double coefficients[3], double eps, void* workspace,
                      uint64_t workspace_bytes, void* stream) {
  using namespace mbt_learning;
  if (!dtype_known(dtype)) return mbt_set_error(MBT_ERR_INVALID, "dtype %d: float32, bfloat16 and float16 are known", dtype);
  int rc = check_matrices(count, matrices);
  if (rc != MBT_OK) return rc;
  if (steps < 1 || steps > 64) return mbt_set_error(MBT_ERR_INVALID, "%d steps: 1 .. 64 are taken", steps);
  if (coefficients == nullptr || !bounded(steps, coefficients))
    return mbt_set_error(MBT_ERR_INVALID, "the coefficients let singular values grow beyond 1.9 (or are not numbers)");
  if (!(eps >= 0.0 && std::isfinite(eps))) return mbt_set_error(MBT_ERR_INVALID, "eps = %g: it has to be a finite number, not negative", eps);
  const uint64_t needed = workspace_of(count, matrices);
  if (needed > 0 && (workspace == nullptr || workspace_bytes < needed))
    return mbt_set_error(MBT_ERR_INVALID, "the workspace has %llu bytes; %llu are needed (mbt_orthogonalise_workspace)",
                         (unsigned long long)(workspace == nullptr ? 0 : workspace_bytes), (unsigned long long)needed);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return mbt_set_error(MBT_ERR_INVALID, "the workspace is not aligned to 16 bytes");
  DeviceScope scope;
  rc = scope.enter(device);
  if (rc != MBT_OK) return rc;
  rc = dtype == MBT_FLOAT32 ? allow_lds<float>(device) : dtype == MBT_BFLOAT16 ? allow_lds<bfloat16>(device) : allow_lds<float16>(device);
  if (rc != MBT_OK) return rc;
  OrthogonaliseParams P{};
  P.steps = steps;
  P.a = static_cast<float>(coefficients[0]);
  P.b = static_cast<float>(coefficients[1]);
  P.c = static_cast<float>(coefficients[2]);
  P.eps = eps;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MBT_FLOAT32) return run<float>(count, matrices, P, workspace, s);
  if (dtype == MBT_BFLOAT16) return run<bfloat16>(count, matrices, P, workspace, s);
  return run<float16>(count, matrices, P, workspace, s);
}

}  // extern "C"
