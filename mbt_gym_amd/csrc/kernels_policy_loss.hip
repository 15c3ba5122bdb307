// The C entry points of the policy-gradient loss: argument checks, the count of a mask's rows, the sum over the workgroups (kernels: policy_loss.hpp).
#include <cmath>

#include "policy_loss.hpp"

namespace mbt_learning {
extern template int launch_policy_loss<float>(const PolicyLossParams&, int, int, unsigned, hipStream_t);
extern template int launch_policy_loss<bfloat16>(const PolicyLossParams&, int, int, unsigned, hipStream_t);
extern template int launch_policy_loss<float16>(const PolicyLossParams&, int, int, unsigned, hipStream_t);

namespace {

// Rows that a mask keeps, per workgroup: the gradients of the rows are divided by their number, so it has to be known first (one byte per row).
// FLAT: the bytes lie behind one another; sixteen at a time, the bytes that are not zero counted by their carry into the top bit.
template <bool FLAT>
__global__ __launch_bounds__(256) void count_rows(Rows mask, int64_t outer, int64_t inner, uint32_t* counts) {
  __shared__ uint32_t lds[4];
  uint32_t n = 0;
  const uint8_t* p = static_cast<const uint8_t*>(mask.p);
  const int64_t total = outer * inner, each = FLAT ? 16 : 1;
  for (int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * each; at < total; at += static_cast<int64_t>(gridDim.x) * 256 * each) {
    if (FLAT && at + 16 <= total) {
      const Pack<uint8_t, 16> bytes = load_pack<uint8_t, 16>(p + at);
      uint32_t words[4];
      __builtin_memcpy(words, &bytes, 16);
#pragma unroll
      for (int w = 0; w < 4; ++w) n += __popc(((((words[w] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | words[w]) & 0x80808080u));
    } else {
      for (int64_t b = at; b < at + each && b < total; ++b) n += p[FLAT ? b : b / inner * mask.so + b % inner * mask.si] != 0;
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = lds[0] + lds[1] + lds[2] + lds[3];
}

// The workgroups' partials, added in an order that does not depend on when they came: loss, rows, and the std gradient's sums.
constexpr int kFinishThreads = 1024, kFinishWaves = kFinishThreads / 64;
__global__ __launch_bounds__(kFinishThreads) void finish_loss(const double* partials, int blocks, int actions, int columns, const uint32_t* counts, double rows,
                                                              double* sums, float* loss, float* grad_std) {
  __shared__ double lds[kFinishWaves][2 + kMostActions];
  static_assert(kCountBlocks <= kFinishThreads, "one partial count per thread");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double sum[2 + kMostActions];  // loss, components, rows
#pragma unroll
  for (int c = 0; c < 2 + kMostActions; ++c) sum[c] = 0.0;
  for (int b = threadIdx.x; b < blocks; b += kFinishThreads) {
#pragma unroll
    for (int c = 0; c < 1 + kMostActions; ++c)
      if (c < columns) sum[c] += partials[static_cast<int64_t>(b) * (1 + actions) + c];
  }
  if (counts != nullptr && threadIdx.x < kCountBlocks) sum[1 + kMostActions] = static_cast<double>(counts[threadIdx.x]);
#pragma unroll
  for (int c = 0; c < 2 + kMostActions; ++c) {
    if (c < columns || c == 1 + kMostActions) {
      sum[c] = wave_sum(sum[c]);
      if (lane == 0) lds[wave][c] = sum[c];
    }
  }
  __syncthreads();
  if (threadIdx.x >= static_cast<unsigned>(columns)) return;
  double kept = rows, s = 0.0;
  if (counts != nullptr) {
    kept = 0.0;
    for (int w = 0; w < kFinishWaves; ++w) kept += lds[w][1 + kMostActions];
  }
  const int column = threadIdx.x;
  for (int w = 0; w < kFinishWaves; ++w) s += lds[w][column];
  const float mean = kept > 0.0 ? static_cast<float>(-s / (kept * actions)) : 0.0f;
  if (column == 0) {
    sums[0] = s;
    sums[1] = kept;
    *loss = mean;
  } else {
    sums[1 + column] = s;
    if (grad_std != nullptr) grad_std[column - 1] = mean;
  }
}

struct LossPlan {
  PolicyLossParams params;
  unsigned blocks;
  uint64_t workspace;
};

int make_plan(const mbt_policy_loss* p, LossPlan& plan) {
  if (p == nullptr) return mbt_set_error(MBT_ERR_INVALID, "null argument");
  if (!dtype_known(p->dtype)) return mbt_set_error(MBT_ERR_INVALID, "dtype %d: float32, bfloat16 and float16 are known", p->dtype);
  if (p->std_kind < MBT_STD_NUMBER || p->std_kind > MBT_STD_FULL) return mbt_set_error(MBT_ERR_INVALID, "std_kind %d is none of MBT_STD_*", p->std_kind);
  if (p->actions < 1 || p->actions > kMostActions) return mbt_set_error(MBT_ERR_INVALID, "%d action components: 1 .. %d are known", p->actions, kMostActions);
  const uint64_t limit = uint64_t{1} << 40;
  if (p->outer < 1 || p->inner < 1 || p->outer > limit || p->inner > limit / p->outer) return mbt_set_error(MBT_ERR_INVALID, "outer x inner has to be within 1 .. 2^40");
  if (p->mean.data == nullptr || p->action.data == nullptr || p->weight.data == nullptr) return mbt_set_error(MBT_ERR_INVALID, "mean, action and weight are needed");
  if (p->sums == nullptr) return mbt_set_error(MBT_ERR_INVALID, "sums is needed");
  if (p->std_kind != MBT_STD_NUMBER && p->std_array.data == nullptr) return mbt_set_error(MBT_ERR_INVALID, "this std_kind needs std_array");
  if (p->std_kind == MBT_STD_NUMBER && !(p->std > 0.0 && std::isfinite(p->std))) return mbt_set_error(MBT_ERR_INVALID, "std = %g: it has to be positive", p->std);
  if (p->std_kind == MBT_STD_NUMBER && p->grad_std.data != nullptr) return mbt_set_error(MBT_ERR_INVALID, "a std given as a number has no gradient array");
  if (p->std_kind == MBT_STD_NUMBER && !std::isfinite(1.0f / static_cast<float>(p->std)))
    return mbt_set_error(MBT_ERR_INVALID, "std = %g: its inverse is not finite in float32", p->std);
  if (!std::isfinite(static_cast<float>(p->entropy_weight))) return mbt_set_error(MBT_ERR_INVALID, "entropy_weight is not finite");
  PolicyLossParams& P = plan.params;
  P = PolicyLossParams{};
  auto rows = [](const mbt_array2& a) { return Rows{a.data, a.stride[0], a.stride[1]}; };
  P.mean = rows(p->mean);
  P.action = rows(p->action);
  P.weight = rows(p->weight);
  P.mask = rows(p->mask);
  P.grad_mean = rows(p->grad_mean);
  P.grad_std = rows(p->grad_std);
  if (p->std_kind == MBT_STD_FULL) P.std_rows = rows(p->std_array);
  if (p->std_kind == MBT_STD_COMPONENT) P.std_components = static_cast<const float*>(p->std_array.data);
  P.outer = static_cast<int64_t>(p->outer);
  P.inner = static_cast<int64_t>(p->inner);
  P.num_actions = p->actions;
  P.std = static_cast<float>(p->std);
  P.log_std = p->std_kind == MBT_STD_NUMBER ? static_cast<float>(std::log(p->std)) : 0.0f;
  P.entropy_weight = static_cast<float>(p->entropy_weight);
  int log2 = 0;  // a tile lies along inner as far as inner goes
  while ((1 << log2) < kLossTile && (int64_t{1} << log2) < P.inner) ++log2;
  P.inner_log2 = log2;
  P.tiles_per_outer = (P.inner + (int64_t{1} << log2) - 1) >> log2;
  const int64_t tile_outer = kLossTile >> log2;
  P.tiles = (P.outer + tile_outer - 1) / tile_outer * P.tiles_per_outer;
  plan.blocks = static_cast<unsigned>(P.tiles < kMostLossBlocks ? P.tiles : kMostLossBlocks);
  plan.workspace = static_cast<uint64_t>(plan.blocks) * (1 + p->actions) * sizeof(double) + (p->mask.data != nullptr ? kCountBlocks * sizeof(uint32_t) : 0);
  return MBT_OK;
}

int launch(const mbt_policy_loss* p, const LossPlan& plan, hipStream_t stream) {
  if (p->dtype == MBT_FLOAT32) return launch_policy_loss<float>(plan.params, p->actions, p->std_kind, plan.blocks, stream);
  if (p->dtype == MBT_BFLOAT16) return launch_policy_loss<bfloat16>(plan.params, p->actions, p->std_kind, plan.blocks, stream);
  return launch_policy_loss<float16>(plan.params, p->actions, p->std_kind, plan.blocks, stream);
}

}  // namespace
}  // namespace mbt_learning

extern "C" {

uint64_t mbt_policy_loss_workspace(const mbt_policy_loss* p) {
  mbt_learning::LossPlan plan;
  return mbt_learning::make_plan(p, plan) == MBT_OK ? plan.workspace : 0;
}

int mbt_policy_loss_forward(int device, const mbt_policy_loss* p, void* stream) {
  using namespace mbt_learning;
  LossPlan plan;
  int rc = make_plan(p, plan);
  if (rc != MBT_OK) return rc;
  if (p->loss == nullptr) return mbt_set_error(MBT_ERR_INVALID, "the forward call needs loss");
  if (p->workspace == nullptr || p->workspace_bytes < plan.workspace)
    return mbt_set_error(MBT_ERR_INVALID, "the workspace has %llu bytes; %llu are needed (mbt_policy_loss_workspace)",
                         (unsigned long long)(p->workspace == nullptr ? 0 : p->workspace_bytes), (unsigned long long)plan.workspace);
  if (reinterpret_cast<uintptr_t>(p->workspace) % sizeof(double) != 0) return mbt_set_error(MBT_ERR_INVALID, "the workspace is not aligned to 8 bytes");
  DeviceScope scope;
  rc = scope.enter(device);
  if (rc != MBT_OK) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  PolicyLossParams& P = plan.params;
  P.partials = static_cast<double*>(p->workspace);
  if (P.mask.p != nullptr) {
    uint32_t* counts = reinterpret_cast<uint32_t*>(P.partials + static_cast<int64_t>(plan.blocks) * (1 + p->actions));
    P.counts = counts;
    const bool flat = (P.inner == 1 || P.mask.si == 1) && (P.outer == 1 || P.mask.so == P.inner);
    if (flat) count_rows<true><<<kCountBlocks, 256, 0, s>>>(P.mask, P.outer, P.inner, counts);
    else count_rows<false><<<kCountBlocks, 256, 0, s>>>(P.mask, P.outer, P.inner, counts);
    rc = launch_status("policy loss (rows)");
    if (rc != MBT_OK) return rc;
  }
  rc = launch(p, plan, s);
  if (rc != MBT_OK) return rc;
  const bool components = p->std_kind == MBT_STD_COMPONENT;
  finish_loss<<<1, kFinishThreads, 0, s>>>(P.partials, static_cast<int>(plan.blocks), p->actions, components ? 1 + p->actions : 1, P.counts,
                                static_cast<double>(P.outer) * static_cast<double>(P.inner), p->sums, p->loss,
                                components ? static_cast<float*>(P.grad_std.p) : nullptr);
  return launch_status("policy loss (sum)");
}

uint64_t mbt_stream_capture_id(void* stream) {
  if (stream == nullptr) return 0;  // (the default stream cannot be captured)
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id : 0;
}

int mbt_policy_loss_backward(int device, const mbt_policy_loss* p, void* stream) {
  using namespace mbt_learning;
  LossPlan plan;
  int rc = make_plan(p, plan);
  if (rc != MBT_OK) return rc;
  if (p->grad_loss == nullptr) return mbt_set_error(MBT_ERR_INVALID, "the backward call needs grad_loss");
  DeviceScope scope;
  rc = scope.enter(device);
  if (rc != MBT_OK) return rc;
  plan.params.grad_loss = p->grad_loss;
  plan.params.sums = p->sums;
  plan.params.ready = p->gradients_ready != 0;
  return launch(p, plan, static_cast<hipStream_t>(stream));
}

}  // extern "C"
