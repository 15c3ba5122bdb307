"""The policy-gradient loss of recorded actions (the reference's objective, mbt_gym/agents/PolicyGradientAgent.py:49-62) with its gradient in the same
pass over the recording.  Kernels and what bounds them: csrc/policy_loss.hpp."""
import math
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from mbt_gym_amd import _native
from mbt_gym_amd.learning._tensors import DTYPES, batch_groups, current_stream, refuse_recording, require


class _Plan:
    """How operands of these shapes, strides and settings look to the library, with every field of struct mbt_policy_loss filled in but the addresses and
    the entropy's weight, and the workspace it asks for.  It depends on nothing else, so it is kept."""

    def __init__(self, shape, dtype, kind, number, mean, actions, weights, mask, std):
        axis, components = len(shape) - 1, shape[-1]
        given = [mean, actions, weights + (1,)] + ([] if mask is None else [mask + (1,)]) + ([std] if kind == _native.STD_FULL else [])
        dense, run = [0] * len(shape), 1  # of the gradients
        for d in range(axis, -1, -1):
            dense[d] = run
            run *= max(1, shape[d])
        groups = batch_groups(shape, axis, given + [dense])
        # components of a row lie side by side; batch axes fold to two
        self.folds = groups is not None and (components == 1 or all(s[-1] == 1 for s in given))
        if not self.folds:
            return
        outer_dim = groups[0][1] if len(groups) == 2 else None
        inner_dim = groups[-1][1] if groups else None

        def array(s):
            return (None, (0 if outer_dim is None else s[outer_dim], 0 if inner_dim is None else s[inner_dim]))

        p = _native.MbtPolicyLoss(groups[0][0] if len(groups) == 2 else 1, groups[-1][0] if groups else 1, components, DTYPES[dtype], kind, 0, number)
        p.mean, p.action, p.weight = array(mean), array(actions), array(weights)
        if mask is not None:
            p.mask = array(mask)
        if kind == _native.STD_FULL:
            p.std_array = array(std)
        p.grad_mean = p.grad_std = array(dense)
        self.template = bytes(p)
        p.mean.data = p.action.data = p.weight.data = p.sums = 16  # (the size goes by shapes alone; any address stands for "this operand is there")
        if mask is not None:
            p.mask.data = 16
        if kind != _native.STD_NUMBER:
            p.std_array.data = 16
        self.workspace = _native.load_library().mbt_policy_loss_workspace(p)


_LARGEST = torch.finfo(torch.float32).max
_plans = {}


def _plan_of(mean, std, actions, weights, mask, number):
    kind = _native.STD_NUMBER if std is None else _native.STD_COMPONENT if std.dim() == 1 else _native.STD_FULL
    key = (mean.shape, mean.dtype, kind, number, mean.stride(), actions.stride(), weights.stride(), None if mask is None else mask.stride(),
           None if std is None else std.stride())
    plan = _plans.get(key)
    if plan is None:
        if len(_plans) >= 512:
            _plans.clear()
        plan = _plans[key] = _Plan(*key)
    return plan


def _operands(mean, std, actions, weights, mask, number):
    """(plan, the operands it belongs to): as given, or as copies where their axes do not fold"""
    plan = _plan_of(mean, std, actions, weights, mask, number)
    if not plan.folds:
        mean, std, actions, weights, mask = (None if t is None else t.contiguous() for t in (mean, std, actions, weights, mask))
        plan = _plan_of(mean, std, actions, weights, mask, number)
    p = _native.MbtPolicyLoss.from_buffer_copy(plan.template)
    p.mean.data, p.action.data, p.weight.data = mean.data_ptr(), actions.data_ptr(), weights.data_ptr()
    if mask is not None:
        p.mask.data = mask.data_ptr()
    if std is not None:
        p.std_array.data = std.data_ptr()
    return plan, p, (mean, std, actions, weights, mask)


def _gradients(ctx, p, mean, std):
    """(gradient of mean, gradient of std) as empty tensors that the struct points to, None where none is wanted"""
    grad_mean = grad_std = None
    if ctx.needs_input_grad[0]:
        grad_mean = torch.empty_like(mean, memory_format=torch.contiguous_format)
        p.grad_mean.data = grad_mean.data_ptr()
    if ctx.needs_input_grad[1]:
        grad_std = torch.empty_like(std, memory_format=torch.contiguous_format)
        p.grad_std.data = grad_std.data_ptr()
    return grad_mean, grad_std


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, mean, std, actions, weights, mask, number, entropy_weight):
        device = mean.device
        plan, p, operands = _operands(mean, std, actions, weights, mask, number)
        loss = torch.empty((), dtype=torch.float32, device=device)
        sums = torch.empty(_native.POLICY_LOSS_SUMS, dtype=torch.float64, device=device)
        workspace = torch.empty(plan.workspace, dtype=torch.uint8, device=device)
        p.entropy_weight, p.loss, p.sums = entropy_weight, loss.data_ptr(), sums.data_ptr()
        p.workspace, p.workspace_bytes = workspace.data_ptr(), plan.workspace
        ctx.gradients = _gradients(ctx, p, *operands[:2])
        lib, index = _native.load_library(), device.index
        stream = current_stream(index)
        code = lib.mbt_policy_loss_forward(index, p, stream)
        if code < 0:
            _native.check(code)
        ctx.capture = lib.mbt_stream_capture_id(stream)
        ctx.save_for_backward(*operands, sums)
        ctx.settings = number, entropy_weight
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        *operands, sums = ctx.saved_tensors
        number, entropy_weight = ctx.settings
        _, p, operands = _operands(*operands, number)
        lib, index = _native.load_library(), sums.device.index
        stream = current_stream(index)
        capture = lib.mbt_stream_capture_id(stream)
        # The arrays that the forward call filled are handed out once; a graph that is walked again gets new ones.  So does a pass that is captured without the
        # forward call - its replays come again and again, with other loss gradients and after what the program did to the arrays - and one that is not captured
        # behind a forward call that was, whose replays would write over what it handed out.
        gradients, ctx.gradients = ctx.gradients, None
        if gradients is not None and capture == ctx.capture:
            grad_mean, grad_std = gradients
            p.gradients_ready = 1
            if grad_mean is not None:
                p.grad_mean.data = grad_mean.data_ptr()
            if grad_std is not None:
                p.grad_std.data = grad_std.data_ptr()
        else:
            gradients = _gradients(ctx, p, *operands[:2])
        grad_loss = grad_loss.contiguous()
        p.entropy_weight, p.sums, p.grad_loss = entropy_weight, sums.data_ptr(), grad_loss.data_ptr()
        code = lib.mbt_policy_loss_backward(index, p, stream)
        if code < 0:
            _native.check(code)
        return gradients + (None,) * 5


def policy_gradient_loss(mean: torch.Tensor, actions: torch.Tensor, weights: torch.Tensor, std: Union[float, torch.Tensor], *,
                         mask: Optional[torch.Tensor] = None, entropy_weight: float = 0.0) -> torch.Tensor:
    """- mean of [weight * log N(action | mean, std) + entropy_weight * H(std)] over rows and components: a float32 scalar, differentiable in mean
    and std.

    mean            (..., A) float32, bfloat16 or float16 - what the network answers with for the recorded observations; A from 1 to 8
    actions         (..., A) float32, as recorded; weights (...) float32, e.g. rewards_to_go.  Both are data: no gradient reaches them
    std             a positive number (from 3e-39 on); a float32 tensor (A,), one per component; or a tensor like mean, one per row and component
    mask            bool (or uint8) (...): rows that count.  The others count for nothing, NaN and infinities in them too, and get gradients of zero;
                    with no row left the loss is zero
    entropy_weight  of the entropy bonus H(std) = log std + log(2 pi e) / 2, per component

    The gradients are computed with the loss, in one pass over the recording; backward() only has more to do when the loss was scaled on the way."""
    refuse_recording("policy_gradient_loss", by_autograd=True)
    require(mean, "mean", dtypes=DTYPES)
    if mean.dim() == 0 or not 1 <= mean.shape[-1] <= 8:
        raise ValueError(f"mean has the shape {tuple(mean.shape)}: the last axis holds 1 to 8 action components")
    device = mean.device
    require(actions, "actions", device, (torch.float32,), mean.shape)
    require(weights, "weights", device, (torch.float32,), mean.shape[:-1])
    if torch.is_grad_enabled() and (actions.requires_grad or weights.requires_grad):
        raise ValueError("actions and weights are data of the loss: detach them")
    if mask is not None:
        require(mask, "mask", device, (torch.bool, torch.uint8), mean.shape[:-1])
    entropy_weight = float(entropy_weight)
    if not abs(entropy_weight) <= _LARGEST:
        raise ValueError(f"entropy_weight = {entropy_weight}: it has to be finite, in float32")
    number = 0.0
    if isinstance(std, torch.Tensor):
        require(std, "std", device)
        if std.dim() == 1 and std.shape[0] == mean.shape[-1]:
            require(std, "std (one per component)", device, (torch.float32,))
            std = std.contiguous()
            if mean.dim() == 1:  # (a single row: per component is per element)
                mean, actions, weights = mean.unsqueeze(0), actions.unsqueeze(0), weights.unsqueeze(0)
                mask = None if mask is None else mask.unsqueeze(0)
        else:
            require(std, "std (one per row and component)", device, (mean.dtype,), mean.shape)
    else:
        number, std = float(std), None
        if not (number > 0.0 and math.isfinite(number)):
            raise ValueError(f"std = {number}: it has to be positive")
        if not 1.0 / number <= _LARGEST:
            raise ValueError(f"std = {number}: its inverse has to be finite, in float32")
    if mean.numel() == 0:
        zero = mean.sum(dtype=torch.float32) if std is None else mean.sum(dtype=torch.float32) + 0.0 * std.sum(dtype=torch.float32)
        return zero  # (no rows: a loss of zero that is still connected to its leaves)
    if not torch.is_grad_enabled():  # (nothing will ask for the gradients)
        mean, std = mean.detach(), None if std is None else std.detach()
    return _PolicyLoss.apply(mean, std, actions, weights, mask, number, entropy_weight)
