"""The reference's REINFORCE learner (mbt_gym/agents/PolicyGradientAgent.py:14-73) as a consumer of the device path.

Same interface - `PolicyGradientAgent(policy, action_std, optimizer, env, lr_scheduler)`, `get_action(state, deterministic,
include_log_probs)`, `train(num_epochs, reporting_freq) -> (losses, mean rewards)` - and the same objective (log-probabilities
of the sampled actions weighted by the rewards-to-go, PG:49-73).  What differs is where an epoch's data comes from: when the
actor is a network the kernels can evaluate ([Linear, act, Linear, act, Linear], hidden width <= 64, tanh or relu) the whole
episode is sampled by ONE fused rollout launch - the network on the matrix cores, a ~ N(mean, std) drawn from Philox in the
kernel, observations / actions / rewards recorded straight into torch tensors - and what is learnt from them is computed there
too: the rewards-to-go, the loss log N(a | policy(obs), std) x reward-to-go and its gradient with respect to the network's
answers are kernels (mbt_gym_amd/learning), PyTorch carries that gradient on through the network.  Any other torch module takes
the reference's loop (generate_trajectory with include_log_probs=True: one host forward pass and one env.step per time step); a
`learning.RecurrentPolicy` quotes step by step in that loop and is scored on the whole recording at once.  PyTorch is the consumer
here, not the product."""
from typing import Callable, Tuple, Union

import numpy as np

from mbt_gym_amd.agents.Agent import Agent
from mbt_gym_amd.gym.helpers.generate_trajectory import generate_trajectory


def _actor_layers(policy):
    """([(W, b)] * 3, activation) when the kernels can evaluate the module, else None."""
    import torch

    modules = list(policy) if isinstance(policy, torch.nn.Sequential) else None
    if modules is None or len(modules) != 5:
        return None
    first, act1, second, act2, last = modules
    if not all(isinstance(m, torch.nn.Linear) for m in (first, second, last)) or type(act1) is not type(act2):
        return None
    activation = {torch.nn.Tanh: "tanh", torch.nn.ReLU: "relu"}.get(type(act1))
    hidden = first.out_features
    if activation is None or hidden > 64 or second.in_features != hidden or second.out_features != hidden or last.in_features != hidden:
        return None
    if any(m.bias is None for m in (first, second, last)):
        return None
    return [(m.weight.detach().cpu().numpy(), m.bias.detach().cpu().numpy()) for m in (first, second, last)], activation


class PolicyGradientAgent(Agent):
    def __init__(self, policy, action_std: Union[float, Callable] = 0.01, optimizer=None, env=None, lr_scheduler=None, discount: float = 1.0):
        """Beyond the reference's arguments: `discount` of the rewards-to-go (the reference's learner has none: 1), and `optimizer` may be the name
        "muon" (mbt_gym_amd.learning.Muon over the policy's parameters)."""
        import torch
        from torch.optim.lr_scheduler import StepLR

        if not 0.0 <= discount <= 1.0:
            raise ValueError(f"discount = {discount}: it has to lie in [0, 1]")
        if isinstance(optimizer, str):
            if optimizer != "muon":
                raise ValueError(f"optimizer = {optimizer!r}: an optimizer, or the name 'muon'")
            from mbt_gym_amd.learning import Muon

            optimizer = Muon(policy.parameters())

        if env is None:
            from mbt_gym_amd.gym.TradingEnvironment import TradingEnvironment

            env = TradingEnvironment()
        self.env = env
        self.input_size = env.observation_space.shape[0]
        self.action_size = env.action_space.shape[0]
        first = policy[0] if hasattr(policy, "__getitem__") else None
        assert first is None or self.input_size == first.in_features
        self.policy_net = policy
        self.action_std = action_std
        self.discount = float(discount)
        self.optimizer = optimizer or torch.optim.SGD(self.policy_net.parameters(), lr=1e-1)
        self.lr_scheduler = lr_scheduler or StepLR(self.optimizer, step_size=1, gamma=0.995)
        self.noise_dist = torch.distributions.Normal
        self.proportion_completed: float = 0.0

    # ---- the policy -------------------------------------------------------------------------------------------------------
    def _std(self) -> float:
        return float(self.action_std(self.proportion_completed)) if isinstance(self.action_std, Callable) else float(self.action_std)

    def _module_device(self):
        import torch

        return next((p.device for p in self.policy_net.parameters()), torch.device("cpu"))

    def get_action(self, state: np.ndarray, deterministic: bool = False, include_log_probs: bool = False):
        import torch

        assert not (deterministic and include_log_probs), "include_log_probs is only an option for deterministic output"
        observation = torch.as_tensor(np.asarray(state), dtype=torch.float, device=self._module_device())
        mean_value = self.policy_net.step(observation) if self._is_recurrent else self.policy_net(observation)
        if deterministic:
            return mean_value.detach().cpu().numpy()
        action_dist = self.noise_dist(loc=mean_value, scale=self._std() * torch.ones_like(mean_value))
        action = action_dist.sample()
        if include_log_probs:
            return action.detach().cpu().numpy(), action_dist.log_prob(action)
        return action.detach().cpu().numpy()

    @property
    def _is_recurrent(self) -> bool:
        from mbt_gym_amd.learning import RecurrentPolicy

        return isinstance(self.policy_net, RecurrentPolicy)

    def begin_episode(self):
        """What an actor carries from step to step starts anew (generate_trajectory calls this after env.reset())."""
        if self._is_recurrent:
            self.policy_net.begin_episode()

    @property
    def has_device_policy(self) -> bool:
        """The fused rollout can sample this actor on this environment: a [Linear, act, Linear, act, Linear] network, Philox
        noise, and observations the matrix cores can read as fp16 (normalised, or bounded by 4: SbAgent.observations_fit_fp16) -
        otherwise `train` takes the reference's host loop."""
        from mbt_gym_amd.agents.SbAgent import observations_fit_fp16

        return (_actor_layers(self.policy_net) is not None and hasattr(self.env, "rollout_device") and getattr(self.env, "noise", "philox") == "philox"
                and observations_fit_fp16(self.env))

    def kernel_mean(self, obs):
        """The actor's mean AS THE KERNEL EVALUATES IT (csrc/policy_mlp.hpp), in torch and differentiable: the observation row,
        [W1 | b1], the hidden activations, W2 and W3 rounded to fp16 - fp32 accumulation, b2 / b3 in fp32 - with a
        straight-through estimator for the rounding of the weights.  The kernel samples a ~ N(kernel mean, std); scoring those
        actions against the float32 `policy_net(obs)` instead would add (kernel mean - float32 mean) / std^2 x grad(mean) x
        reward-to-go to the REINFORCE gradient - a bias the reference's loop, which samples and scores with ONE mean, does not
        have, and which grows as the exploration std is annealed."""
        import torch

        first, act1, second, act2, last = list(self.policy_net)

        def half(t):  # value rounded to fp16, gradient passed straight through
            return t + (t.detach().half().float() - t.detach())

        x = obs.half().float()
        h = act1(torch.nn.functional.linear(x, half(first.weight), half(first.bias)))
        h = act2(torch.nn.functional.linear(half(h), half(second.weight), second.bias))
        return torch.nn.functional.linear(half(h), half(last.weight), last.bias)

    def device_policy(self, deterministic: bool = False):
        """The actor as the kernels evaluate it: sampling with the current std unless `deterministic`; never clipped (PG:34-47)."""
        from mbt_gym_amd import _native

        layers, activation = _actor_layers(self.policy_net)
        std = None if deterministic else [self._std()] * self.action_size
        return _native.mlp_policy(layers, activation, action_std=std, clip=False)

    @property
    def _epoch_is_its_own(self) -> bool:
        """The sampling, the rewards-to-go and the distribution are the ones of this class.  Where a subclass, or a program, has put its own in
        their place, `train` asks those for them and takes the loss of what they answer."""
        import torch

        return (getattr(self._sample_on_device, "__func__", None) is _OWN_SAMPLE and self._calculate_future_rewards is _OWN_FUTURE_REWARDS
                and self.noise_dist is torch.distributions.Normal)

    # ---- one epoch of data ----------------------------------------------------------------------------------------------------
    def _record_on_device(self):
        """One fused rollout launch: (observations (T, N, D), actions (T, N, A), rewards (T, N)), views of the padded recording on the device."""
        import torch

        env = self.env
        n, n_pad, horizon = env.num_trajectories, env.padded_lanes, env.n_steps
        cuda = torch.device("cuda", env.device)
        obs = torch.empty((horizon + 1, n_pad, env.observation_dim), dtype=torch.float32, device=cuda)
        act = torch.empty((horizon, n_pad, env.action_dim), dtype=torch.float32, device=cuda)
        rew = torch.empty((horizon, n_pad), dtype=torch.float32, device=cuda)
        env.set_stream(torch.cuda.current_stream(cuda).cuda_stream)  # torch's allocator and the kernel share a stream
        env.reset_device()
        steps, _ = env.rollout_device(self.device_policy(), max_steps=horizon, obs_ptr=obs.data_ptr(), act_ptr=act.data_ptr(), rew_ptr=rew.data_ptr())
        return obs[:steps, :n], act[:steps, :n], rew[:steps, :n]

    def _sample_on_device(self):
        """(rewards (N, 1, T) tensor, log-probabilities (N, A, T) tensor with gradients), from one fused rollout launch."""
        where = self._module_device()
        o, a, r = (t.to(where) for t in self._record_on_device())
        return self._scored(self.kernel_mean(o), a, r)  # the actions the KERNEL sampled, around ITS mean

    def _sample_sequence(self):
        """The same of a recurrent actor, which quoted step by step and is scored on the whole recording."""
        o, a, r = self._record_sequence()
        return self._scored(self.policy_net(o), a, r)

    def _scored(self, mean, actions, rewards):
        log_prob = self.noise_dist(mean, self._std()).log_prob(actions)  # (T, N, A)
        return rewards.t().unsqueeze(1), log_prob.permute(1, 2, 0)

    def _record_sequence(self):
        """One episode of the reference's loop: (observations (T, N, D), actions (T, N, A), rewards (T, N)) on the policy's device."""
        observations, actions, rewards, where = *generate_trajectory(self.env, self), self._module_device()
        return tuple(self._time_first(t, where) for t in (observations[:, :, :-1], actions, rewards[:, 0]))

    def _device_epoch(self):
        """(rewards, loss) of one epoch whose data never leaves the device: - mean of log N(a | mean, std) x reward-to-go (PG:58-59) as kernels"""
        import torch

        from mbt_gym_amd.learning import policy_gradient_loss, rewards_to_go

        if self._is_recurrent:
            o, a, r = self._record_sequence()
            mean = self.policy_net(o)
        else:
            o, a, r = self._record_on_device()
            mean = self.kernel_mean(o)
        loss = policy_gradient_loss(mean, a, rewards_to_go(r, self.discount, dim=0), self._std())
        if bool(torch.isnan(loss)):  # (as any NaN in the means and actions makes it: the distribution refuses those, and says what it was given)
            self.noise_dist(mean, self._std()).log_prob(a)
        return r, loss

    @staticmethod
    def _time_first(array, where):
        """(N, ..., T) on the host -> (T, N, ...) on the device"""
        import torch

        return torch.as_tensor(np.ascontiguousarray(np.moveaxis(array, -1, 0)), device=where)

    def train(self, num_epochs: int = 1, reporting_freq: int = 100):
        import torch

        learning_losses, learning_rewards = [], []
        self.proportion_completed = 0.0
        for epoch in range(num_epochs):
            on_device = self._is_recurrent or (self.has_device_policy and self._module_device() == torch.device("cuda", self.env.device))
            if on_device and self._epoch_is_its_own:
                rewards, loss = self._device_epoch()
                learning_rewards.append(float(rewards.mean()))
            else:
                if self._is_recurrent:
                    rewards, log_probs = self._sample_sequence()
                elif self.has_device_policy:
                    rewards, log_probs = self._sample_on_device()
                else:
                    _, _, rewards, log_probs = generate_trajectory(self.env, self, include_log_probs=True)
                    rewards = torch.as_tensor(rewards, device=log_probs.device)
                learning_rewards.append(float(rewards.mean()))
                future_rewards = self._calculate_future_rewards(rewards, *([] if self.discount == 1.0 else [self.discount]))  # (PG:69 takes the rewards alone)
                loss = -torch.mean(log_probs * future_rewards)  # PG:58-59
            self.optimizer.zero_grad()
            loss.backward()
            self.optimizer.step()
            if epoch % reporting_freq == 0:
                print(loss.item())
            learning_losses.append(loss.item())
            self.proportion_completed += 1 / max(1, num_epochs - 1)
            self.lr_scheduler.step()
        return learning_losses, learning_rewards

    @staticmethod
    def _calculate_future_rewards(rewards, discount: float = 1.0):
        """Rewards-to-go along the last axis (PG:69-73): a kernel where the rewards live on the device, torch where they live on the host or are
        something to differentiate (any number of times, either way) or to transform."""
        import torch

        from mbt_gym_amd.learning._tensors import DTYPES, transformed

        if rewards.is_cuda and rewards.dtype in DTYPES and not (torch.is_grad_enabled() and rewards.requires_grad) and not transformed():
            from mbt_gym_amd.learning import rewards_to_go

            return rewards_to_go(rewards, discount)
        if discount == 1.0:
            return torch.flip(torch.cumsum(torch.flip(rewards, dims=(-1,)), dim=-1), dims=(-1,))
        out, following = torch.empty_like(rewards), torch.zeros_like(rewards[..., 0])
        for k in range(rewards.shape[-1] - 1, -1, -1):
            following = rewards[..., k] + discount * following
            out[..., k] = following
        return out


_OWN_SAMPLE, _OWN_FUTURE_REWARDS = PolicyGradientAgent._sample_on_device, PolicyGradientAgent._calculate_future_rewards
