"""The gated linear recurrence h_t = g_t h_{t-1} + x_t along the time axis of a recording, its backward pass, and its single step.

The rewards-to-go of the reference's learner (mbt_gym/agents/PolicyGradientAgent.py:69-73) are the recurrence walked backwards with a constant
gate; the state of a recurrent actor is the one with learnt gates.  Kernels, splits and what bounds them: csrc/recurrence.hpp."""
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from mbt_gym_amd import _native
from mbt_gym_amd.learning._tensors import DTYPES, batch_groups, current_stream, dense_strides, refuse_recording, require


class _Plan:
    """How operands of these shapes, strides and settings look to the library - (outer, time, inner) - with every field of struct mbt_recurrence filled
    in but the addresses, and the workspaces it asks for.  It depends on nothing else, so it is kept: filling it in costs more than a short call."""

    def __init__(self, shape, strides, dtype, axis, form, constant, reverse, inputs, gate, reset):
        # `strides` are the states' - and the gradients' - own: the inputs' order of axes without gaps
        given = [t for t in (inputs, gate, reset) if t is not None]
        groups = batch_groups(shape, axis, given + [strides])
        self.folds = groups is not None
        if not self.folds:
            return
        self.strides, self.batch = strides, [n for d, n in enumerate(shape) if d != axis]
        outer_dim = groups[0][1] if len(groups) == 2 else None
        inner_dim = groups[-1][1] if groups else None

        def array(s):
            return (None, (0 if outer_dim is None else s[outer_dim], s[axis], 0 if inner_dim is None else s[inner_dim]))

        r = _native.MbtRecurrence(groups[0][0] if len(groups) == 2 else 1, shape[axis], groups[-1][0] if groups else 1, DTYPES[dtype], form, reverse, 0,
                                  constant)
        for name, s in (("inputs", inputs), ("gate", gate), ("reset", reset), ("states", strides), ("grad_states", strides), ("grad_inputs", strides),
                        ("grad_gate", strides)):
            if s is not None:
                setattr(r, name, array(s))
        self.template = bytes(r)
        lib = _native.load_library()
        # (the sizes go by strides alone; any address stands for "this operand is there")
        for name in ("inputs", "states", "grad_states", "grad_inputs") + (() if gate is None else ("gate", "grad_gate")):
            getattr(r, name).data = 16
        self.workspace = lib.mbt_recurrence_workspace(r, 0), lib.mbt_recurrence_workspace(r, 1)
        self.edge_steps = lib.mbt_recurrence_edge_steps(r)
        self.edges = -(-shape[axis] // self.edge_steps) - 1 if self.edge_steps else 0

    def struct(self):
        return _native.MbtRecurrence.from_buffer_copy(self.template)

    def launch(self, entry, struct, backward, device):
        size = self.workspace[backward]
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
            struct.workspace, struct.workspace_bytes = workspace.data_ptr(), size
        index = device.index
        code = entry(index, struct, current_stream(index))
        if code < 0:
            _native.check(code)


_LARGEST = torch.finfo(torch.float32).max
_plans = {}


def _plan_of(inputs, gate, reset, settings):
    key = (inputs.shape, inputs.stride(), inputs.dtype, None if gate is None else gate.stride(), None if reset is None else reset.stride(), settings)
    plan = _plans.get(key)
    if plan is None:
        if len(_plans) >= 512:
            _plans.clear()
        plan = _plans[key] = _Plan(inputs.shape, dense_strides(inputs), inputs.dtype, *settings, inputs.stride(), key[3], key[4])
    return plan


def _forward(inputs, gate, initial, reset, settings, for_gate=False):
    """(states, final state, edges - for the gate's gradient, if it is wanted and they are needed, else None - plan, and the operands it belongs to)"""
    plan = _plan_of(inputs, gate, reset, settings)
    if not plan.folds:  # (batch axes that do not fold into two: copies that do)
        inputs, gate, reset = (None if t is None else t.contiguous() for t in (inputs, gate, reset))
        plan = _plan_of(inputs, gate, reset, settings)
    device = inputs.device
    states = torch.empty_strided(inputs.shape, plan.strides, dtype=inputs.dtype, device=device)
    final = torch.empty(plan.batch, dtype=torch.float32, device=device)
    r = plan.struct()
    r.inputs.data, r.states.data, r.final_state = inputs.data_ptr(), states.data_ptr(), final.data_ptr()
    if gate is not None:
        r.gate.data = gate.data_ptr()
    if reset is not None:
        r.reset.data = reset.data_ptr()
    if initial is not None:
        r.initial = initial.data_ptr()
    edges = None
    if for_gate and plan.edges:
        edges = torch.empty([plan.edges] + plan.batch, dtype=torch.float32, device=device)
        r.edge_steps, r.edges, r.edges_bytes = plan.edge_steps, edges.data_ptr(), 4 * edges.numel()
    plan.launch(_native.load_library().mbt_recurrence_forward, r, 0, device)
    return states, final, edges, plan, inputs, gate, reset


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs, gate, initial, reset, settings):
        states, final, edges, plan, inputs, gate, reset = _forward(inputs, gate, initial, reset, settings, ctx.needs_input_grad[1])
        if gate is None:
            ctx.save_for_backward(None, None, initial, reset, None, None)
        else:  # (the backward pass looks at states only for the gate's gradient: float32 ones as they were stored, or the edges)
            ctx.save_for_backward(inputs, gate, initial, reset, states if ctx.needs_input_grad[1] and states.dtype is torch.float32 else None, edges)
        ctx.edge_steps = plan.edge_steps
        ctx.plan, ctx.settings, ctx.shape, ctx.dtype, ctx.device = plan, settings, states.shape, states.dtype, states.device
        ctx.reset_strides = None if reset is None else reset.stride()
        ctx.set_materialize_grads(False)
        return states, final

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_states, grad_final):
        inputs, gate, initial, reset, states, edges = ctx.saved_tensors
        if grad_states is None and grad_final is None:
            return (None,) * 5
        plan, device = ctx.plan, ctx.device
        if initial is not None:
            initial = initial.contiguous()  # (as it was saved, unless a hook brought it back otherwise)
        if gate is not None:
            plan = _plan_of(inputs, gate, reset, ctx.settings)  # (the same one, unless a hook on saved tensors brought them back in another layout)
            if not plan.folds:
                inputs, gate, reset = (None if t is None else t.contiguous() for t in (inputs, gate, reset))
                plan = _plan_of(inputs, gate, reset, ctx.settings)
            if states is not None and states.stride() != plan.strides:
                states = _laid_out(states, plan.strides)
            if ctx.needs_input_grad[1] and plan.edges and plan.edge_steps != ctx.edge_steps:  # (that layout is walked in other pieces)
                edges = _forward(inputs, gate, initial, reset, ctx.settings, True)[2]
        elif reset is not None and reset.stride() != ctx.reset_strides:
            reset = _laid_out(reset, ctx.reset_strides)
        if grad_states is None:
            grad_states = torch.empty_strided(ctx.shape, plan.strides, dtype=ctx.dtype, device=device).zero_()
        elif grad_states.stride() != plan.strides:  # (an expanded or transposed gradient: one copy, then the states' layout)
            grad_states = _laid_out(grad_states, plan.strides)
        r = plan.struct()
        r.grad_states.data = grad_states.data_ptr()
        if gate is not None:
            r.inputs.data, r.gate.data = inputs.data_ptr(), gate.data_ptr()
            if states is not None:
                r.states.data = states.data_ptr()
            if ctx.needs_input_grad[1] and plan.edges:
                edges = edges.contiguous()
                r.edge_steps, r.edges, r.edges_bytes = plan.edge_steps, edges.data_ptr(), 4 * edges.numel()
        if reset is not None:
            r.reset.data = reset.data_ptr()
        if initial is not None:
            r.initial = initial.data_ptr()
        wanted = ctx.needs_input_grad
        grad_inputs = grad_gate = grad_initial = None
        if wanted[0]:
            grad_inputs = torch.empty_like(grad_states)
            r.grad_inputs.data = grad_inputs.data_ptr()
        if wanted[1]:
            grad_gate = torch.empty_like(grad_states)
            r.grad_gate.data = grad_gate.data_ptr()
        if wanted[2]:
            grad_initial = torch.empty_like(initial)
            r.grad_initial = grad_initial.data_ptr()
        if grad_final is not None:
            grad_final = grad_final.contiguous()
            r.grad_final = grad_final.data_ptr()
        plan.launch(_native.load_library().mbt_recurrence_backward, r, 1, device)
        return grad_inputs, grad_gate, grad_initial, None, None


def _laid_out(tensor, strides):
    return torch.empty_strided(tensor.shape, strides, dtype=tensor.dtype, device=tensor.device).copy_(tensor)


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
    steps has no states, and its final state is the initial one.  Gradients are those of the stored inputs and gates: the
    states that they need are recomputed from them, in float32 whatever the states are stored in.  Second and
    forward-mode derivatives are refused."""
    tracing = refuse_recording("linear_recurrence", by_autograd=True)
    require(inputs, "inputs", dtypes=DTYPES)
    if inputs.dim() == 0:
        raise ValueError("inputs is a scalar: it has no time axis")
    if not -inputs.dim() <= dim < inputs.dim():
        raise IndexError(f"dim {dim} of a tensor with {inputs.dim()} dimensions")
    axis = dim % inputs.dim()
    batch = tuple(n for d, n in enumerate(inputs.shape) if d != axis)
    constant = 0.0
    if isinstance(gate, torch.Tensor):
        require(gate, "gate", inputs.device, (inputs.dtype,), inputs.shape)
        form = _native.GATE_LOGIT if gate_is_logit else _native.GATE_VALUE
    else:
        if gate_is_logit:
            raise TypeError("gate_is_logit needs a gate tensor")
        form, constant, gate = _native.GATE_CONSTANT, float(gate), None
        if not abs(constant) <= _LARGEST:
            raise ValueError(f"gate = {constant}: a constant gate has to be finite, in float32")
    if initial is not None:
        require(initial, "initial", inputs.device, (torch.float32, inputs.dtype), batch)
        initial = initial.to(torch.float32).contiguous()
    if reset is not None:
        require(reset, "reset", inputs.device, (torch.bool, torch.uint8), inputs.shape)
    if inputs.numel() == 0:
        # (nothing is added to the initial state, but the results depend on every operand, whose gradients are zeros)
        joined = inputs if gate is None else inputs + gate
        first = torch.zeros(batch, dtype=torch.float32, device=inputs.device) if initial is None else initial
        states, final = joined + first.unsqueeze(axis).to(inputs.dtype), first + joined.sum(dim=axis, dtype=torch.float32)
        return (states, final) if return_final else states
    tracked = torch.is_grad_enabled() and (inputs.requires_grad or (gate is not None and gate.requires_grad) or (initial is not None and initial.requires_grad))
    settings = (axis, form, constant, 1 if reverse else 0)
    if tracked or tracing:
        states, final = _LinearRecurrence.apply(inputs, gate, initial, reset, settings)
    else:
        states, final = _forward(inputs, gate, initial, reset, settings)[:2]
    return (states, final) if return_final else states


def linear_recurrence_step(state: torch.Tensor, inputs: torch.Tensor, gate: torch.Tensor, *, reset: Optional[torch.Tensor] = None,
                           gate_is_logit: bool = False, new_state: Optional[torch.Tensor] = None):
    """One step of `linear_recurrence`, for an actor that quotes: (the state in the inputs' dtype, the same state in float32 to carry on with).

    state      float32, the inputs' shape; contiguous
    new_state  where the float32 state goes: None = a new tensor; `state` itself updates it in place
    Not differentiable: an actor is trained on whole sequences."""
    refuse_recording("linear_recurrence_step")
    require(inputs, "inputs", dtypes=DTYPES)
    shape, dtype, device = inputs.shape, inputs.dtype, inputs.device
    require(state, "state", device, (torch.float32,), shape)
    require(gate, "gate", device, (dtype,), shape)
    if torch.is_grad_enabled() and (state.requires_grad or inputs.requires_grad or gate.requires_grad):
        raise ValueError("linear_recurrence_step is not differentiable: use torch.no_grad(), or linear_recurrence on the sequence")
    given = new_state is not None
    if not given:
        new_state = torch.empty(shape, dtype=torch.float32, device=device)
    elif new_state is not state:
        require(new_state, "new_state", device, (torch.float32,), shape)
    if not (state.is_contiguous() and new_state.is_contiguous()):
        raise ValueError("state and new_state have to be contiguous")
    out, count = torch.empty(shape, dtype=dtype, device=device), inputs.numel()
    if not count:
        return out, new_state
    columns = shape[-1] if shape else 1
    rows = count // columns
    flags, row_stride, column_stride = None, 0, 0
    if reset is not None:
        require(reset, "reset", device, (torch.bool, torch.uint8), shape)
        folded = reset.reshape(rows, columns)
        flags, (row_stride, column_stride) = folded.data_ptr(), folded.stride()
    inputs, gate = inputs.contiguous(), gate.contiguous()
    state_at, inputs_at, gate_at, new_at = state.data_ptr(), inputs.data_ptr(), gate.data_ptr(), new_state.data_ptr()
    if given:
        size = 4 * count
        width = size if dtype is torch.float32 else size // 2
        if (new_at != state_at and -size < new_at - state_at < size) or -width < new_at - inputs_at < width or -width < new_at - gate_at < width:
            _refuse_overlap(new_at, size, (("state", state_at, size), ("inputs", inputs_at, width), ("gate", gate_at, width)))
        if not new_state.is_inference():
            torch.autograd.graph.increment_version(new_state)  # (so that a backward pass that saved it notices)
    index = device.index
    code = _native.load_library().mbt_recurrence_step(
        index, DTYPES[dtype], _native.GATE_LOGIT if gate_is_logit else _native.GATE_VALUE, rows, columns, state_at, inputs_at, gate_at, flags, row_stride,
        column_stride, out.data_ptr(), new_at, current_stream(index))
    if code < 0:
        _native.check(code)
    return out, new_state


def _refuse_overlap(new_at, size, operands):
    """Each element is read before its own place is written, by the thread that writes it: the very same place is all right, another is not."""
    for name, at, width in operands:
        if at < new_at + size and new_at < at + width and not (at == new_at and width == size):
            raise ValueError(f"new_state lies over {name}, but not in its place")


def rewards_to_go(rewards: torch.Tensor, discount: float = 1.0, *, dim: int = -1, done: Optional[torch.Tensor] = None) -> torch.Tensor:
    """G_t = r_t + discount G_{t+1} along `dim` (PolicyGradientAgent.py:69-73, where the discount is 1); `done` marks the last step of an
    episode, behind which nothing counts."""
    discount = float(discount)
    if not 0.0 <= discount <= 1.0:
        raise ValueError(f"discount = {discount}: it has to lie in [0, 1]")
    return linear_recurrence(rewards, discount, dim=dim, reverse=True, reset=done)
