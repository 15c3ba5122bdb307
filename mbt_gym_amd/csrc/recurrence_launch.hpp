// Which instantiation of recurrence.hpp a launch runs; included by one translation unit per element type.
#pragma once
#include "recurrence.hpp"

namespace mbt_learning {

template <typename E>
constexpr int kVector = 16 / static_cast<int>(sizeof(E));  // columns of one 16-byte access

template <typename E, int FORM, int V, bool BACKWARD>
void (*columns_kernel(int mode))(RecurrenceParams) {
  constexpr int kJoinedSteps = chunk_steps(FORM, BACKWARD, V, false), kAloneSteps = chunk_steps(FORM, BACKWARD, V, true);
  if (mode == kAlone) return recurrence_columns<E, FORM, V, kAloneSteps, BACKWARD, kAlone>;
  if (mode == kJoined) return recurrence_columns<E, FORM, V, kJoinedSteps, BACKWARD, kJoined>;
  return recurrence_columns<E, FORM, V, kJoinedSteps, BACKWARD, kComposites>;
}

template <typename E, int FORM, bool BACKWARD>
void (*pick_recurrence(int which))(RecurrenceParams) {
  if (which >= kRows) {
    if (which - kRows == kComposites) return recurrence_rows<E, FORM, kRowSteps, BACKWARD, true>;
    return recurrence_rows<E, FORM, kRowSteps, BACKWARD, false>;
  }
  if constexpr (!BACKWARD) {
    constexpr int V = kVector<E>, K = chunk_steps(FORM, false, V, true);
    if (which == kColumnsWide) return recurrence_columns<E, FORM, V, K, false, kAlone>;
    if (which == kColumnsWide + kStreamed) return recurrence_columns<E, FORM, V, K, false, kAlone, true>;
  }
  if constexpr (sizeof(E) == 2) {
    if (which >= kColumnsPair) return columns_kernel<E, FORM, 2, BACKWARD>(which - kColumnsPair);
  }
  return columns_kernel<E, FORM, 1, BACKWARD>(which - kColumnsScalar);
}

template <typename E>
int launch_recurrence(const RecurrenceParams& P, int form, bool backward, int which, unsigned blocks, unsigned threads, size_t lds, hipStream_t stream) {
  void (*kernel)(RecurrenceParams) = nullptr;
  if (form == kGateConstant) kernel = backward ? pick_recurrence<E, kGateConstant, true>(which) : pick_recurrence<E, kGateConstant, false>(which);
  if (form == kGateValue) kernel = backward ? pick_recurrence<E, kGateValue, true>(which) : pick_recurrence<E, kGateValue, false>(which);
  if (form == kGateLogit) kernel = backward ? pick_recurrence<E, kGateLogit, true>(which) : pick_recurrence<E, kGateLogit, false>(which);
  kernel<<<blocks, threads, lds, stream>>>(P);
  return launch_status("recurrence");
}

template <typename E>
int launch_recurrence_step(const float* state, const void* x, const void* g, const uint8_t* reset, int64_t reset_columns, int64_t rs, int64_t rc, void* out,
                           float* new_state, int64_t n, int form, hipStream_t stream) {
  // 16 bytes per thread only where the chip is full anyway (2^22 bfloat16: 9.3 us, 11.6 with one element each); below that more and smaller waves
  // finish sooner (2^16: 2.3 us, 2.8 wide; 2^21: 5.4 and 5.8)
  const bool wide = n >= (1 << 22);
  const int v = wide ? kVector<E> : 1;
  const unsigned blocks = static_cast<unsigned>((n + 256 * static_cast<int64_t>(v) - 1) / (256 * static_cast<int64_t>(v)));
  const E *xe = static_cast<const E*>(x), *ge = static_cast<const E*>(g);
  E* oe = static_cast<E*>(out);
  if (form == kGateValue) {
    if (wide) recurrence_step<E, kGateValue, kVector<E>><<<blocks, 256, 0, stream>>>(state, xe, ge, reset, reset_columns, rs, rc, oe, new_state, n);
    else recurrence_step<E, kGateValue, 1><<<blocks, 256, 0, stream>>>(state, xe, ge, reset, reset_columns, rs, rc, oe, new_state, n);
  } else {
    if (wide) recurrence_step<E, kGateLogit, kVector<E>><<<blocks, 256, 0, stream>>>(state, xe, ge, reset, reset_columns, rs, rc, oe, new_state, n);
    else recurrence_step<E, kGateLogit, 1><<<blocks, 256, 0, stream>>>(state, xe, ge, reset, reset_columns, rs, rc, oe, new_state, n);
  }
  return launch_status("recurrence step");
}

}  // namespace mbt_learning
