"""The policy-gradient loss of recorded actions (the reference's objective, mbt_gym/agents/PolicyGradientAgent.py:49-62) with its gradient in the same
pass over the recording.  Kernels and what bounds them: csrc/policy_loss.hpp."""
import math
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from mbt_gym_amd import _native
from mbt_gym_amd.learning._tensors import DTYPES, batch_groups, current_stream, require


def _rows(tensor, groups):
    """struct mbt_array2 of a tensor: its address and its strides along (outer, inner)"""
    s = tensor.stride()
    return _native.MbtArray2(tensor.data_ptr(), (s[groups[0][1]] if len(groups) == 2 else 0, s[groups[-1][1]] if groups else 0))


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, mean, std, actions, weights, mask, number, entropy_weight):
        components = mean.shape[-1]
        axis = mean.dim() - 1
        full = std is not None and std.dim() > 1
        # components of a row lie side by side; batch axes fold to two
        mean, actions = (t if components == 1 or t.stride(-1) == 1 else t.contiguous() for t in (mean, actions))
        if full and components > 1 and std.stride(-1) != 1:
            std = std.contiguous()

        def fold():
            strides = [t.stride() for t in ((mean, actions, std) if full else (mean, actions))]
            return batch_groups(mean.shape, axis, strides + [t.stride() + (1,) for t in (weights, mask) if t is not None])

        groups = fold()
        if groups is None:
            mean, actions, weights = mean.contiguous(), actions.contiguous(), weights.contiguous()
            mask, std = None if mask is None else mask.contiguous(), std.contiguous() if full else std
            groups = fold()
        device = mean.device
        loss = torch.empty((), dtype=torch.float32, device=device)
        sums = torch.empty(_native.POLICY_LOSS_SUMS, dtype=torch.float64, device=device)
        p = _native.MbtPolicyLoss(groups[0][0] if len(groups) == 2 else 1, groups[-1][0] if groups else 1, components, DTYPES[mean.dtype],
                                  _native.STD_NUMBER if std is None else _native.STD_FULL if full else _native.STD_COMPONENT, 0, number, entropy_weight)
        p.mean, p.action, p.weight = _rows(mean, groups), _rows(actions, groups), _rows(weights, groups)
        if mask is not None:
            p.mask = _rows(mask, groups)
        if full:
            p.std_array = _rows(std, groups)
        elif std is not None:
            p.std_array.data = std.data_ptr()
        p.loss, p.sums = loss.data_ptr(), sums.data_ptr()
        ctx.gradients = _gradients(ctx, p, mean, std, groups)
        lib = _native.load_library()
        size = lib.mbt_policy_loss_workspace(p)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = workspace.data_ptr(), size
        _native.check(lib.mbt_policy_loss_forward(device.index, p, current_stream(device.index)))
        ctx.save_for_backward(mean, std, actions, weights, mask, sums)
        ctx.struct, ctx.groups = p, groups
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        mean, std, actions, weights, mask, sums = ctx.saved_tensors
        # the arrays that the forward call filled are handed out once; a graph that is walked again gets new ones
        ready, ctx.gradients = ctx.gradients, None
        p, groups = _native.MbtPolicyLoss.from_buffer_copy(ctx.struct), ctx.groups
        p.mean, p.action, p.weight = _rows(mean, groups), _rows(actions, groups), _rows(weights, groups)
        if mask is not None:
            p.mask = _rows(mask, groups)
        if std is not None:
            p.std_array.data = std.data_ptr()
        p.sums, p.loss, p.workspace, p.workspace_bytes = sums.data_ptr(), None, None, 0
        gradients = ready or _gradients(ctx, p, mean, std, groups)
        p.gradients_ready = int(ready is not None)
        grad_loss = grad_loss.contiguous()
        p.grad_loss = grad_loss.data_ptr()
        index = mean.device.index
        _native.check(_native.load_library().mbt_policy_loss_backward(index, p, current_stream(index)))
        return gradients + (None,) * 5


def _gradients(ctx, p, mean, std, groups):
    """(gradient of mean, gradient of std) as empty tensors that the struct points to, None where none is wanted"""
    out = [None, None]
    if ctx.needs_input_grad[0]:
        out[0] = torch.empty_like(mean, memory_format=torch.contiguous_format)
        p.grad_mean = _rows(out[0], groups)
    if ctx.needs_input_grad[1]:
        out[1] = torch.empty_like(std, memory_format=torch.contiguous_format)
        if std.dim() > 1:
            p.grad_std = _rows(out[1], groups)
        else:
            p.grad_std.data = out[1].data_ptr()
    return tuple(out)


def policy_gradient_loss(mean: torch.Tensor, actions: torch.Tensor, weights: torch.Tensor, std: Union[float, torch.Tensor], *,
                         mask: Optional[torch.Tensor] = None, entropy_weight: float = 0.0) -> torch.Tensor:
    """- mean of [weight * log N(action | mean, std) + entropy_weight * H(std)] over rows and components: a float32 scalar, differentiable in mean
    and std.

    mean            (..., A) float32, bfloat16 or float16 - what the network answers with for the recorded observations; A from 1 to 8
    actions         (..., A) float32, as recorded; weights (...) float32, e.g. rewards_to_go.  Both are data: no gradient reaches them
    std             a positive number; a float32 tensor (A,), one per component; or a tensor like mean, one per row and component
    mask            bool (or uint8) (...): rows that count.  The others count for nothing, NaN and infinities in them too, and get gradients of zero;
                    with no row left the loss is zero
    entropy_weight  of the entropy bonus H(std) = log std + log(2 pi e) / 2, per component

    The gradients are computed with the loss, in one pass over the recording; backward() only has more to do when the loss was scaled on the way."""
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
    if not math.isfinite(entropy_weight):
        raise ValueError(f"entropy_weight = {entropy_weight}: it has to be finite")
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
    if mean.numel() == 0:
        zero = mean.sum(dtype=torch.float32) if std is None else mean.sum(dtype=torch.float32) + 0.0 * std.sum(dtype=torch.float32)
        return zero  # (no rows: a loss of zero that is still connected to its leaves)
    return _PolicyLoss.apply(mean, std, actions, weights, mask, number, entropy_weight)
