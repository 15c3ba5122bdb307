// The gated linear recurrence for float16 elements (recurrence.hpp).
#include "recurrence_launch.hpp"

namespace mbt_learning {
template int launch_recurrence<float16>(const RecurrenceParams&, int, bool, int, unsigned, unsigned, size_t, hipStream_t);
template int launch_recurrence_step<float16>(const float*, const void*, const void*, const uint8_t*, int64_t, int64_t, int64_t, void*, float*, int64_t, int, hipStream_t);
}  // namespace mbt_learning
