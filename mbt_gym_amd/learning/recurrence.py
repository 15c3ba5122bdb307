"""The gated linear recurrence h_t = g_t h_{t-1} + x_t along the time axis of a recording, its backward pass, and its single step.

The rewards-to-go of the reference's learner (mbt_gym/agents/PolicyGradientAgent.py:69-73) are the recurrence walked backwards with a constant
gate; the state of a recurrent actor is the one with learnt gates.  Kernels, splits and what bounds them: csrc/recurrence.hpp."""
import ctypes
import math
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from mbt_gym_amd import _native
from mbt_gym_amd.learning._tensors import DTYPES, dense_like, require, where


def _batch_axes(tensors, axis):
    """The batch dimensions (all but `axis`) as at most two groups of neighbours that are one stride apart in EVERY tensor: [(size, last dim)]
    ordered outer, inner; or None when they do not fold into two."""
    shape = tensors[0].shape
    groups = []
    for d in range(len(shape)):
        if d == axis or shape[d] == 1:
            continue
        if groups and all(t.stride(groups[-1][1]) == t.stride(d) * shape[d] for t in tensors):
            groups[-1] = (groups[-1][0] * shape[d], d)
        else:
            groups.append((shape[d], d))
    return groups if len(groups) <= 2 else None


class _Call:
    """One call's tensors as struct mbt_recurrence sees them: arrays of (outer, time, inner)."""

    def __init__(self, tensors, axis):
        self.axis = axis
        self.groups = _batch_axes(list(tensors.values()), axis)
        if self.groups is None:  # (batch axes that do not fold: copies that do)
            tensors = {name: t.contiguous() for name, t in tensors.items()}
            self.groups = _batch_axes(list(tensors.values()), axis)
        self.tensors = tensors  # (kept: the copies live until the launch)
        first = next(iter(tensors.values()))
        sizes = [1] * (2 - len(self.groups)) + [size for size, _ in self.groups]
        self.struct = _native.MbtRecurrence(outer=sizes[0], steps=first.shape[axis], inner=sizes[1], dtype=DTYPES[first.dtype])
        for name, t in tensors.items():
            array = getattr(self.struct, name)
            array.data = t.data_ptr()
            strides = [0] * (2 - len(self.groups)) + [t.stride(d) for _, d in self.groups]
            array.stride[0], array.stride[1], array.stride[2] = strides[0], t.stride(axis), strides[1]

    def run(self, entry, backward, device):
        lib = _native.load_library()
        size = lib.mbt_recurrence_workspace(ctypes.byref(self.struct), int(backward))
        workspace = None
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
            self.struct.workspace, self.struct.workspace_bytes = workspace.data_ptr(), size
        index, stream = where(device)
        _native.check(getattr(lib, entry)(index, ctypes.byref(self.struct), stream))


def _forward(inputs, gate, initial, reset, axis, form, constant, reverse):
    states = dense_like(inputs)
    final = torch.empty([n for d, n in enumerate(inputs.shape) if d != axis], dtype=torch.float32, device=inputs.device)
    tensors = {"inputs": inputs, "states": states}
    if gate is not None:
        tensors["gate"] = gate
    if reset is not None:
        tensors["reset"] = reset
    call = _Call(tensors, axis)
    call.struct.form, call.struct.constant, call.struct.reverse = form, constant, int(reverse)
    call.struct.initial = None if initial is None else initial.data_ptr()
    call.struct.final_state = final.data_ptr()
    call.run("mbt_recurrence_forward", False, inputs.device)
    return call.tensors["states"], final


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs, gate, initial, reset, axis, form, constant, reverse):
        states, final = _forward(inputs, gate, initial, reset, axis, form, constant, reverse)
        ctx.save_for_backward(*((None, None, initial, reset, None) if gate is None else (inputs, gate, initial, reset, states)))
        ctx.settings = (axis, form, constant, reverse)
        ctx.shape, ctx.dtype = inputs.shape, inputs.dtype
        ctx.set_materialize_grads(False)
        return states, final

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_states, grad_final):
        inputs, gate, initial, reset, states = ctx.saved_tensors
        axis, form, constant, reverse = ctx.settings
        if grad_states is None and grad_final is None:
            return (None,) * 8
        if grad_states is None:
            grad_states = torch.zeros(ctx.shape, dtype=ctx.dtype, device=grad_final.device) if states is None else torch.zeros_like(states)
        layout = inputs if inputs is not None else grad_states
        if states is not None and grad_states.stride() != states.stride():  # (an expanded or transposed gradient: one copy, then the fast layout)
            grad_states = torch.empty_like(states).copy_(grad_states)
        elif states is None and not (grad_states.is_contiguous() or grad_states.stride(axis) == 1):
            grad_states = grad_states.contiguous()
        tensors = {"grad_states": grad_states}
        if gate is not None:
            tensors.update(inputs=inputs, gate=gate, states=states)
        if reset is not None:
            tensors["reset"] = reset
        grads = [None, None, None]
        if ctx.needs_input_grad[0]:
            grads[0] = tensors["grad_inputs"] = dense_like(layout)
        if gate is not None and ctx.needs_input_grad[1]:
            grads[1] = tensors["grad_gate"] = dense_like(layout)
        if initial is not None and ctx.needs_input_grad[2]:
            grads[2] = torch.empty_like(initial)
        call = _Call(tensors, axis)
        call.struct.form, call.struct.constant, call.struct.reverse = form, constant, int(reverse)
        call.struct.initial = None if initial is None else initial.data_ptr()
        if grad_final is not None:
            grad_final = grad_final.contiguous()
            call.struct.grad_final = grad_final.data_ptr()
        if grads[2] is not None:
            call.struct.grad_initial = grads[2].data_ptr()
        call.run("mbt_recurrence_backward", True, grad_states.device)
        for position, name in ((0, "grad_inputs"), (1, "grad_gate")):
            if grads[position] is not None:
                grads[position] = call.tensors[name]
        return (grads[0], grads[1], grads[2], None, None, None, None, None)


def linear_recurrence(inputs: torch.Tensor, gate: Union[float, torch.Tensor], initial: Optional[torch.Tensor] = None, *, dim: int = 0,
                      reverse: bool = False, reset: Optional[torch.Tensor] = None, gate_is_logit: bool = False, return_final: bool = False):
    """States of h_t = g_t h_{t-1} + x_t along axis `dim`, in the shape and dtype of `inputs`; differentiable in inputs, gate and initial.

    inputs        float32, bfloat16 or float16, any strides; the walk along `dim` is carried in float32 and rounded once, when a state is stored
    gate          a number, or a tensor of the inputs' shape and dtype (expand a shared one).  With `gate_is_logit` the gate is f = sigmoid(gate)
                  and the input is weighted with what the gate leaves: h_t = f h_{t-1} + (1 - f) x_t.  Gates are meant to lie in [-1, 1]: products
                  of gates along the axis have to stay inside float32's range
    initial       the state before the first step (the inputs' shape without `dim`; zeros when None)
    reverse       walk from the last step to the first; `initial` then stands behind the last
    reset         bool (or uint8) of the inputs' shape: where it is set, the step starts from a state of zero
    return_final  also return the last state of the walk in float32, for a recording that comes in pieces

    A gate of exactly zero, like a reset, drops the state it meets whatever that holds: infinities and NaN do not pass it.  A sequence without
    steps has no states, and its final state is the initial one.  Gradients are exact for the stored inputs and gates: the states that they
    need are recomputed from them.  Second derivatives are refused."""
    require(inputs, "inputs", dtypes=DTYPES)
    if inputs.dim() == 0:
        raise ValueError("inputs is a scalar: it has no time axis")
    if not -inputs.dim() <= dim < inputs.dim():
        raise IndexError(f"dim {dim} of a tensor with {inputs.dim()} dimensions")
    axis = dim % inputs.dim()
    batch = [n for d, n in enumerate(inputs.shape) if d != axis]
    constant = 0.0
    if isinstance(gate, torch.Tensor):
        require(gate, "gate", inputs.device, (inputs.dtype,), inputs.shape)
        form = _native.GATE_LOGIT if gate_is_logit else _native.GATE_VALUE
    else:
        if gate_is_logit:
            raise TypeError("gate_is_logit needs a gate tensor")
        form, constant, gate = _native.GATE_CONSTANT, float(gate), None
        if not math.isfinite(constant):
            raise ValueError(f"gate = {constant}: a constant gate has to be finite")
    if initial is not None:
        require(initial, "initial", inputs.device, (torch.float32, inputs.dtype), batch)
        initial = initial.to(torch.float32).contiguous()
    if reset is not None:
        require(reset, "reset", inputs.device, (torch.bool, torch.uint8), inputs.shape)
    if inputs.numel() == 0:
        states = inputs.clone()
        final = torch.zeros(batch, dtype=torch.float32, device=inputs.device) if initial is None else initial.clone()
        return (states, final) if return_final else states
    tracked = torch.is_grad_enabled() and (inputs.requires_grad or (gate is not None and gate.requires_grad) or (initial is not None and initial.requires_grad))
    run = _LinearRecurrence.apply if tracked else _forward
    states, final = run(inputs, gate, initial, reset, axis, form, constant, bool(reverse))
    return (states, final) if return_final else states


def linear_recurrence_step(state: torch.Tensor, inputs: torch.Tensor, gate: torch.Tensor, *, reset: Optional[torch.Tensor] = None,
                           gate_is_logit: bool = False, new_state: Optional[torch.Tensor] = None):
    """One step of `linear_recurrence`, for an actor that quotes: (the state in the inputs' dtype, the same state in float32 to carry on with).

    state      float32, the inputs' shape; contiguous
    new_state  where the float32 state goes: None = a new tensor; `state` itself updates it in place
    Not differentiable: an actor is trained on whole sequences."""
    require(inputs, "inputs", dtypes=DTYPES)
    require(state, "state", inputs.device, (torch.float32,), inputs.shape)
    require(gate, "gate", inputs.device, (inputs.dtype,), inputs.shape)
    if torch.is_grad_enabled() and (state.requires_grad or inputs.requires_grad or gate.requires_grad):
        raise ValueError("linear_recurrence_step is not differentiable: use torch.no_grad(), or linear_recurrence on the sequence")
    if new_state is None:
        new_state = torch.empty(inputs.shape, dtype=torch.float32, device=inputs.device)
    elif new_state is not state:
        require(new_state, "new_state", inputs.device, (torch.float32,), inputs.shape)
    if not (state.is_contiguous() and new_state.is_contiguous()):
        raise ValueError("state and new_state have to be contiguous")
    out = torch.empty(inputs.shape, dtype=inputs.dtype, device=inputs.device)
    if inputs.numel() == 0:
        return out, new_state
    columns = inputs.shape[-1] if inputs.dim() else 1
    rows = inputs.numel() // columns
    flags = row_stride = column_stride = 0
    if reset is not None:
        require(reset, "reset", inputs.device, (torch.bool, torch.uint8), inputs.shape)
        folded = reset.reshape(rows, columns)
        flags, row_stride, column_stride = folded.data_ptr(), folded.stride(0), folded.stride(1)
    inputs, gate = inputs.contiguous(), gate.contiguous()
    index, stream = where(inputs.device)
    _native.check(_native.load_library().mbt_recurrence_step(
        index, DTYPES[inputs.dtype], _native.GATE_LOGIT if gate_is_logit else _native.GATE_VALUE, rows, columns, state.data_ptr(), inputs.data_ptr(),
        gate.data_ptr(), flags or None, row_stride, column_stride, out.data_ptr(), new_state.data_ptr(), stream))
    return out, new_state


def rewards_to_go(rewards: torch.Tensor, discount: float = 1.0, *, dim: int = -1, done: Optional[torch.Tensor] = None) -> torch.Tensor:
    """G_t = r_t + discount G_{t+1} along `dim` (PolicyGradientAgent.py:69-73, where the discount is 1); `done` marks the last step of an
    episode, behind which nothing counts."""
    discount = float(discount)
    if not 0.0 <= discount <= 1.0:
        raise ValueError(f"discount = {discount}: it has to lie in [0, 1]")
    return linear_recurrence(rewards, discount, dim=dim, reverse=True, reset=done)
