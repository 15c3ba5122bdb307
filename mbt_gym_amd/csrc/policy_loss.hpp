// The policy-gradient loss of recorded actions and its gradient in ONE pass over the recording.
//
//   z = (a - mean) / std,   log N = - z^2 / 2 - log std - log(2 pi) / 2,   H = log std + log(2 pi e) / 2
//   loss = - 1 / (R A) sum over kept rows and components of  w log N + c H                               (R rows kept, A components)
//   d loss / d mean = - w z / (std R A),     d loss / d std = - (w (z^2 - 1) + c) / (std R A)
//
// What bounds it: memory.  A row of two float32 components is read once (mean, action, weight: 20 B) and its gradient written once (8 B).  The
// gradients for a loss gradient of one are written while the row is in registers; the backward call looks at the loss gradient on the device
// and has nothing to do when it is one, which is what loss.backward() hands it, and recomputes (one more pass, one rounding) when it is not.
//
// 2^18 lanes x 200 float32 rows of two components: 268 us, 5.5 TB/s of the 1.47 GB it cannot do without - past the caches, for which it is too large
// (305 us through them); 1000 x 200 in 9.5 us, two launches; 16411 x 50 bfloat16 rows of four
// components with their own std under a mask in 23 us, three launches, 43 MB: there the launches count.
//
// Sums: a row's value in float32, everything above it in float64 - per thread, per wave, per workgroup, then one workgroup over the workgroups'
// partials in a fixed order, so repeated calls give the same bits.
#pragma once
#include "learning_common.hpp"

namespace mbt_learning {

constexpr int kMostActions = 8;
constexpr int kLossThreads = 256, kRowsPerThread = 4, kLossTile = kLossThreads * kRowsPerThread;
constexpr int kMostLossBlocks = 2048, kCountBlocks = 256;
static_assert(MBT_POLICY_LOSS_SUMS >= 2 + kMostActions, "the loss, the number of rows, one sum per component");

struct Rows {  // strides in elements along (outer, inner)
  void* p;
  int64_t so, si;
};

struct PolicyLossParams {
  Rows mean, action, weight, mask, std_rows, grad_mean, grad_std;
  const float* std_components;
  const float* grad_loss;  // null: one
  double* partials;        // [block][1 + A], null in the backward call
  const uint32_t* counts;  // [kCountBlocks] rows kept, null without a mask (and in the backward call, which has them in `sums`)
  const double* sums;      // backward: the forward call's
  int64_t outer, inner;
  int64_t tiles, tiles_per_outer;  // a tile is 2^inner_log2 rows along inner x kLossTile >> inner_log2 along outer
  int32_t inner_log2;
  int32_t ready;           // the gradient arrays hold the gradients for a loss gradient of one
  int32_t num_actions;
  float std, log_std;
  float entropy_weight;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

template <typename E, int A, bool STREAM>
__device__ __forceinline__ Pack<E, A> read_row(const E* p) {
  if constexpr (STREAM) return stream_load_pack<E, A>(p);
  else return load_pack<E, A>(p);
}
template <typename E, int A, bool STREAM>
__device__ __forceinline__ void write_row(E* p, const Pack<E, A>& v) {
  if constexpr (STREAM) stream_store_pack<E, A>(p, v);
  else store_pack<E, A>(p, v);
}

template <typename E, int A, int KIND, bool STREAM>
__global__ __launch_bounds__(kLossThreads) void policy_loss_kernel(const PolicyLossParams P) {
  __shared__ double lds[kLossThreads / 64][1 + kMostActions];
  __shared__ double kept;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float g = P.grad_loss == nullptr ? 1.0f : *P.grad_loss;
  if (P.ready && g == 1.0f) return;
  double rows = static_cast<double>(P.outer) * static_cast<double>(P.inner);
  if (P.sums != nullptr) {
    rows = P.sums[1];
  } else if (P.counts != nullptr) {  // every workgroup adds the few partial counts up for itself
    double c = threadIdx.x < kCountBlocks ? static_cast<double>(P.counts[threadIdx.x]) : 0.0;
    static_assert(kCountBlocks <= kLossThreads, "one partial count per thread");
    c = wave_sum(c);
    if (lane == 0) lds[wave][0] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int w = 0; w < kLossThreads / 64; ++w) all += lds[w][0];
      kept = all;
    }
    __syncthreads();
    rows = kept;
  }
  const float scale = rows > 0.0 ? static_cast<float>(static_cast<double>(g) / (rows * A)) : 0.0f;
  float std_c[A], inv_c[A], log_c[A];
#pragma unroll
  for (int j = 0; j < A; ++j) {
    std_c[j] = KIND == MBT_STD_COMPONENT ? P.std_components[j] : P.std;
    inv_c[j] = 1.0f / std_c[j];
    log_c[j] = KIND == MBT_STD_COMPONENT ? logf(std_c[j]) : P.log_std;
  }
  constexpr float kHalfLog2Pi = 0.918938533f, kHalfLog2PiE = 1.418938533f;
  double total = 0.0, by_component[A];
#pragma unroll
  for (int j = 0; j < A; ++j) by_component[j] = 0.0;
  const int wi = 1 << P.inner_log2, tile_outer = kLossTile >> P.inner_log2;

  for (int64_t tile = blockIdx.x; tile < P.tiles; tile += gridDim.x) {
    const int64_t o0 = tile / P.tiles_per_outer * tile_outer, i0 = tile % P.tiles_per_outer * wi;
    Pack<E, A> mean[kRowsPerThread], std_row[kRowsPerThread];
    Pack<float, A> action[kRowsPerThread];
    float w[kRowsPerThread];
    bool in[kRowsPerThread], keep[kRowsPerThread];
#pragma unroll
    for (int r = 0; r < kRowsPerThread; ++r) {  // every load of the thread's rows first
      const int at = threadIdx.x + r * kLossThreads;
      const int64_t o = o0 + (at >> P.inner_log2), i = i0 + (at & (wi - 1));
      in[r] = o < P.outer && i < P.inner;
      keep[r] = in[r];
      w[r] = 0.0f;
      if (in[r]) {
        mean[r] = read_row<E, A, STREAM>(static_cast<const E*>(P.mean.p) + o * P.mean.so + i * P.mean.si);
        action[r] = read_row<float, A, STREAM>(static_cast<const float*>(P.action.p) + o * P.action.so + i * P.action.si);
        w[r] = static_cast<const float*>(P.weight.p)[o * P.weight.so + i * P.weight.si];
        if (KIND == MBT_STD_FULL) std_row[r] = read_row<E, A, STREAM>(static_cast<const E*>(P.std_rows.p) + o * P.std_rows.so + i * P.std_rows.si);
        if (P.mask.p != nullptr) keep[r] = static_cast<const uint8_t*>(P.mask.p)[o * P.mask.so + i * P.mask.si] != 0;
      }
    }
#pragma unroll
    for (int r = 0; r < kRowsPerThread; ++r) {
      if (!in[r]) continue;
      const int at = threadIdx.x + r * kLossThreads;
      const int64_t o = o0 + (at >> P.inner_log2), i = i0 + (at & (wi - 1));
      float value = 0.0f;
      Pack<E, A> gm, gs;
#pragma unroll
      for (int j = 0; j < A; ++j) {
        const float std = KIND == MBT_STD_FULL ? static_cast<float>(std_row[r].e[j]) : std_c[j];
        const float inv = KIND == MBT_STD_FULL ? 1.0f / std : inv_c[j];
        const float log_std = KIND == MBT_STD_FULL ? logf(std) : log_c[j];
        const float z = (action[r].e[j] - static_cast<float>(mean[r].e[j])) * inv;
        const float log_prob = __builtin_fmaf(-0.5f * z, z, -log_std - kHalfLog2Pi);
        value += __builtin_fmaf(w[r], log_prob, P.entropy_weight * (log_std + kHalfLog2PiE));
        const float ds = __builtin_fmaf(w[r], __builtin_fmaf(z, z, -1.0f), P.entropy_weight) * inv;
        if (KIND == MBT_STD_COMPONENT && keep[r]) by_component[j] += static_cast<double>(ds);
        gm.e[j] = static_cast<E>(keep[r] ? -scale * (w[r] * z * inv) : 0.0f);
        gs.e[j] = static_cast<E>(keep[r] ? -scale * ds : 0.0f);
      }
      if (keep[r]) total += static_cast<double>(value);
      if (P.grad_mean.p != nullptr) write_row<E, A, STREAM>(static_cast<E*>(P.grad_mean.p) + o * P.grad_mean.so + i * P.grad_mean.si, gm);
      if (KIND == MBT_STD_FULL && P.grad_std.p != nullptr) write_row<E, A, STREAM>(static_cast<E*>(P.grad_std.p) + o * P.grad_std.so + i * P.grad_std.si, gs);
    }
  }
  if (P.partials == nullptr) {
    if (KIND == MBT_STD_COMPONENT && P.grad_std.p != nullptr && blockIdx.x == 0 && threadIdx.x < A)
      static_cast<float*>(P.grad_std.p)[threadIdx.x] = rows > 0.0 ? static_cast<float>(-P.sums[2 + threadIdx.x] * static_cast<double>(g) / (rows * A)) : 0.0f;
    return;
  }
  __syncthreads();
  total = wave_sum(total);
  if (lane == 0) lds[wave][0] = total;
  if (KIND == MBT_STD_COMPONENT) {
#pragma unroll
    for (int j = 0; j < A; ++j) {
      const double s = wave_sum(by_component[j]);
      if (lane == 0) lds[wave][1 + j] = s;
    }
  }
  __syncthreads();
  if (threadIdx.x < (KIND == MBT_STD_COMPONENT ? 1 + A : 1)) {
    double s = 0.0;
    for (int w = 0; w < kLossThreads / 64; ++w) s += lds[w][threadIdx.x];
    P.partials[static_cast<int64_t>(blockIdx.x) * (1 + A) + threadIdx.x] = s;
  }
}

template <typename E, int A, bool STREAM>
void (*pick_policy_loss(int kind))(PolicyLossParams) {
  if (kind == MBT_STD_NUMBER) return policy_loss_kernel<E, A, MBT_STD_NUMBER, STREAM>;
  if (kind == MBT_STD_COMPONENT) return policy_loss_kernel<E, A, MBT_STD_COMPONENT, STREAM>;
  return policy_loss_kernel<E, A, MBT_STD_FULL, STREAM>;
}

// one translation unit per element type (kernels_policy_loss_*.hip)
template <typename E>
int launch_policy_loss(const PolicyLossParams& P, int actions, int kind, unsigned blocks, hipStream_t stream) {
  // past the caches where the recording is larger than the last of them (2^18 x 200 rows of two float32 components: 268 us, through them 305)
  const int64_t bytes = P.outer * P.inner * actions * static_cast<int64_t>(2 * sizeof(E) + 4);
  const bool stream_it = bytes > (int64_t{256} << 20);
  void (*kernel)(PolicyLossParams) = nullptr;
#define LEARNING_PICK(A) if (actions == A) kernel = stream_it ? pick_policy_loss<E, A, true>(kind) : pick_policy_loss<E, A, false>(kind);
  LEARNING_PICK(1) LEARNING_PICK(2) LEARNING_PICK(3) LEARNING_PICK(4) LEARNING_PICK(5) LEARNING_PICK(6) LEARNING_PICK(7) LEARNING_PICK(8)
#undef LEARNING_PICK
  kernel<<<blocks, kLossThreads, 0, stream>>>(P);
  return launch_status("policy loss");
}

}  // namespace mbt_learning
