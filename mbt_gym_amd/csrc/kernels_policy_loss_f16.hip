// The policy-gradient loss for a network of float16 (policy_loss.hpp).
#include "policy_loss.hpp"

namespace mbt_learning {
template int launch_policy_loss<float16>(const PolicyLossParams&, int, int, unsigned, hipStream_t);
}  // namespace mbt_learning
