"""A recurrent actor: what it answers with depends on the episode so far - order flow that comes in bursts, a trend - through a state that a gated linear
recurrence carries.  One step at a time while it quotes, the whole recording at once while it learns."""
import torch

from mbt_gym_amd.learning.recurrence import linear_recurrence, linear_recurrence_step


class RecurrentPolicy(torch.nn.Module):
    """mean_t = V tanh(h_t) + c,   h_t = f_t h_{t-1} + (1 - f_t) x_t,   (x_t, gate_t) = W obs_t + b,   f_t = sigmoid(gate_t)

    forward(observations)  (T, N, D) -> (T, N, A), differentiable: the recurrence runs along T (mbt_gym_amd.learning.linear_recurrence)
    step(observation)      (N, D) -> (N, A) for the next step of the episode; begin_episode() puts the state back to zero, and lanes whose episode
                           starts anew in between are named by `reset`
    `PolicyGradientAgent` trains it as it is.  Parameters and tensors live on the device."""

    def __init__(self, observation_size: int, action_size: int, hidden_size: int = 64, memory: float = 2.0):
        super().__init__()
        self.inputs = torch.nn.Linear(observation_size, 2 * hidden_size)
        self.output = torch.nn.Linear(hidden_size, action_size)
        self.hidden_size = hidden_size
        with torch.no_grad():
            self.inputs.bias[hidden_size:] += memory  # (the forget gates start open: sigmoid(2) = 0.88)
        self.state = None

    def forward(self, observations: torch.Tensor, reset: torch.Tensor = None) -> torch.Tensor:
        x, gate = self.inputs(observations).split(self.hidden_size, dim=-1)
        if reset is not None:
            reset = reset.unsqueeze(-1).expand(x.shape)
        return self.output(torch.tanh(linear_recurrence(x, gate, dim=0, reset=reset, gate_is_logit=True)))

    def begin_episode(self):
        self.state = None

    @torch.no_grad()
    def step(self, observation: torch.Tensor, reset: torch.Tensor = None) -> torch.Tensor:
        x, gate = self.inputs(observation).split(self.hidden_size, dim=-1)
        if self.state is None or self.state.shape != x.shape or self.state.device != x.device:
            self.state = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
        if reset is not None:
            reset = reset.unsqueeze(-1).expand(x.shape)
        hidden, _ = linear_recurrence_step(self.state, x, gate, reset=reset, gate_is_logit=True, new_state=self.state)
        return self.output(torch.tanh(hidden))
