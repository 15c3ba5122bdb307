// The policy-gradient loss for a network of float (policy_loss.hpp).
#include "policy_loss.hpp"

namespace mbt_learning {
template int launch_policy_loss<float>(const PolicyLossParams&, int, int, unsigned, hipStream_t);
}  // namespace mbt_learning
