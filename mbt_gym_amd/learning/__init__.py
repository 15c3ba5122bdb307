"""What a learner runs between two rollouts, as HIP kernels on torch tensors that live on the device (csrc/kernels_recurrence.hip and its
neighbours, behind the C ABI of include/mbt_env.h):

  linear_recurrence, linear_recurrence_step, rewards_to_go     the gated linear recurrence along the time axis of a recording
  policy_gradient_loss                                         the loss of recorded actions, with its gradient
  RecurrentPolicy                                              an actor on the recurrence: steps while it quotes, sequences while it learns
  orthogonalise, Muon                                          Newton-Schulz products of an update, and the optimiser that steps along it

Every function takes CUDA tensors only (there is no CPU path), works on the current stream of the tensors' device, allocates its outputs and
workspaces from torch and never synchronises, so it may be captured into a `torch.cuda.graph`."""
from mbt_gym_amd.learning.muon import Muon, orthogonalise
from mbt_gym_amd.learning.policy_loss import policy_gradient_loss
from mbt_gym_amd.learning.recurrence import linear_recurrence, linear_recurrence_step, rewards_to_go
from mbt_gym_amd.learning.recurrent_policy import RecurrentPolicy

__all__ = ["Muon", "RecurrentPolicy", "linear_recurrence", "linear_recurrence_step", "orthogonalise", "policy_gradient_loss", "rewards_to_go"]
