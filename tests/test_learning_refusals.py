"""What the learner's operators refuse, without a device: the Python side's checks of its tensors and the C side's checks of its arguments (which
come before any device is touched)."""
import ctypes as C
import os
import subprocess

import pytest

from mbt_gym_amd import _native

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mbt_env.h")


@pytest.fixture(scope="module")
def lib():
    return _native.load_library()


def refused(lib, rc, text):
    assert rc == -1 and text.encode() in lib.mbt_last_error(), (rc, lib.mbt_last_error())


def offsets_match(struct, name, tmp_path):
    """sizeof / offsetof from a C compiler on the header == the ctypes binding"""
    fields = [f for f, _ in struct._fields_]
    body = "".join(f'  printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f in fields)
    source = tmp_path / f"{name}.c"
    source.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n  printf("sizeof %zu\\n", sizeof({name}));\n{body}  return 0; }}\n')
    exe = tmp_path / name
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(source), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(out.pop("sizeof")) == C.sizeof(struct)
    for field, offset in out.items():
        assert getattr(struct, field).offset == int(offset), field


# ---- the recurrence --------------------------------------------------------------------------------------------------------------------
def test_recurrence_struct_layout(tmp_path):
    offsets_match(_native.MbtArray3, "mbt_array3", tmp_path)
    offsets_match(_native.MbtRecurrence, "mbt_recurrence", tmp_path)


def recurrence_struct(**changes):
    """valid arguments over addresses that nothing reads: a refusal comes first, and without a device so does the lack of one"""
    r = _native.MbtRecurrence(outer=2, steps=3, inner=4, dtype=_native.FLOAT32, form=_native.GATE_VALUE, workspace_bytes=0)
    for name in ("inputs", "gate", "states", "grad_states", "grad_inputs", "grad_gate"):
        array = getattr(r, name)
        array.data = 4096
        array.stride[0], array.stride[1], array.stride[2] = 12, 4, 1
    for name, value in changes.items():
        setattr(r, name, value)
    return r


def test_the_library_refuses_a_malformed_recurrence(lib):
    def forward(r):
        return lib.mbt_recurrence_forward(0, C.byref(r), None)

    refused(lib, lib.mbt_recurrence_forward(0, None, None), "null argument")
    refused(lib, forward(recurrence_struct(dtype=7)), "dtype 7")
    refused(lib, forward(recurrence_struct(form=3)), "form 3")
    for name in ("outer", "steps", "inner"):
        refused(lib, forward(recurrence_struct(**{name: 0})), "at least 1")
        refused(lib, forward(recurrence_struct(**{name: 1 << 41})), "beyond 2^40")
    refused(lib, forward(recurrence_struct(outer=1 << 30, inner=1 << 30)), "beyond 2^40")
    missing = recurrence_struct()
    missing.gate.data = None
    refused(lib, forward(missing), "needs a gate")
    missing = recurrence_struct()
    missing.states.data = None
    refused(lib, forward(missing), "inputs and states")
    missing = recurrence_struct()
    missing.grad_states.data = None
    refused(lib, lib.mbt_recurrence_backward(0, C.byref(missing), None), "needs grad_states")
    constant = recurrence_struct(form=_native.GATE_CONSTANT, constant=float("nan"))
    constant.grad_gate.data = None
    refused(lib, forward(constant), "not finite")
    constant = recurrence_struct(form=_native.GATE_CONSTANT, constant=0.5)
    refused(lib, lib.mbt_recurrence_backward(0, C.byref(constant), None), "no gradient array")


def test_a_long_walk_needs_its_workspace(lib):
    r = recurrence_struct(outer=1, steps=1 << 16, inner=4)
    size = lib.mbt_recurrence_workspace(C.byref(r), 0)
    assert size > 0
    refused(lib, lib.mbt_recurrence_forward(0, C.byref(r), None), f"{size} are needed")
    r.workspace, r.workspace_bytes = 4096, size - 1
    refused(lib, lib.mbt_recurrence_forward(0, C.byref(r), None), f"{size} are needed")
    r.workspace, r.workspace_bytes = 4100, size
    refused(lib, lib.mbt_recurrence_forward(0, C.byref(r), None), "aligned")
    assert lib.mbt_recurrence_workspace(C.byref(recurrence_struct()), 0) == 0


def test_more_sequences_than_a_launch_has_threads_are_refused(lib):
    for sizes in (dict(outer=1 << 40, inner=1), dict(outer=1, inner=1 << 34), dict(outer=1 << 20, inner=(1 << 12) + 1)):
        r = recurrence_struct(steps=1, **sizes)
        refused(lib, lib.mbt_recurrence_forward(0, C.byref(r), None), "more than one launch can walk")
        refused(lib, lib.mbt_recurrence_backward(0, C.byref(r), None), "more than one launch can walk")


def test_the_library_refuses_a_malformed_step(lib):
    args = dict(device=0, dtype=0, form=_native.GATE_VALUE, rows=3, columns=4, state=4096, inputs=4096, gate=4096, reset=None, rs=0, cs=0, out=4096, new=4096)

    def step(**changes):
        return lib.mbt_recurrence_step(*{**args, **changes}.values(), None)

    refused(lib, step(dtype=3), "dtype 3")
    refused(lib, step(form=_native.GATE_CONSTANT), "MBT_GATE_VALUE or MBT_GATE_LOGIT")
    for name in ("state", "inputs", "gate", "out", "new"):
        refused(lib, step(**{name: None}), "null argument")
    for sizes in ((0, 1), (1, 0), (1 << 20, 1 << 20), ((1 << 33) + 1, 1), (1, (1 << 33) + 1)):
        refused(lib, step(rows=sizes[0], columns=sizes[1]), "2^33")


def test_tensors_that_are_not_on_the_device_are_refused():
    from mbt_gym_amd import learning

    x = torch.randn(5, 3)
    with pytest.raises(ValueError, match="no CPU path"):
        learning.linear_recurrence(x, 0.5)
    with pytest.raises(ValueError, match="no CPU path"):
        learning.linear_recurrence_step(x, x, x)
    with pytest.raises(ValueError, match="no CPU path"):
        learning.rewards_to_go(x)
    with pytest.raises(TypeError, match="torch tensor"):
        learning.linear_recurrence([1.0, 2.0], 0.5)
    with pytest.raises(ValueError, match="discount"):
        learning.rewards_to_go(x, 1.5)


# ---- the policy-gradient loss ------------------------------------------------------------------------------------------------------------
def loss_struct(**changes):
    p = _native.MbtPolicyLoss(outer=3, inner=5, actions=2, dtype=_native.FLOAT32, std_kind=_native.STD_NUMBER, std=0.1, loss=4096, sums=4096, grad_loss=4096)
    for name in ("mean", "action", "weight"):
        array = getattr(p, name)
        array.data, array.stride[0], array.stride[1] = 4096, 10, 2
    for name, value in changes.items():
        setattr(p, name, value)
    return p


def test_policy_loss_struct_layout(tmp_path):
    offsets_match(_native.MbtArray2, "mbt_array2", tmp_path)
    offsets_match(_native.MbtPolicyLoss, "mbt_policy_loss", tmp_path)


def test_the_library_refuses_a_malformed_policy_loss(lib):
    def forward(**changes):
        return lib.mbt_policy_loss_forward(0, C.byref(loss_struct(**changes)), None)

    refused(lib, lib.mbt_policy_loss_forward(0, None, None), "null argument")
    refused(lib, forward(dtype=5), "dtype 5")
    refused(lib, forward(std_kind=3), "std_kind 3")
    for n in (0, 9):
        refused(lib, forward(actions=n), f"{n} action components")
    for sizes in ((0, 1), (1, 0), (1 << 41, 1), (1 << 30, 1 << 30)):
        refused(lib, forward(outer=sizes[0], inner=sizes[1]), "2^40")
    for name in ("mean", "action", "weight"):
        p = loss_struct()
        getattr(p, name).data = None
        refused(lib, lib.mbt_policy_loss_forward(0, C.byref(p), None), "are needed")
    refused(lib, forward(sums=None), "sums")
    refused(lib, forward(loss=None), "needs loss")
    refused(lib, forward(std_kind=_native.STD_FULL), "std_array")
    for std in (0.0, -1.0, float("nan"), float("inf")):
        refused(lib, forward(std=std), "positive")
    refused(lib, forward(entropy_weight=float("nan")), "entropy_weight")
    p = loss_struct()
    p.grad_std.data = 4096
    refused(lib, lib.mbt_policy_loss_forward(0, C.byref(p), None), "no gradient array")
    size = lib.mbt_policy_loss_workspace(C.byref(loss_struct()))
    assert size > 0
    refused(lib, forward(), f"{size} are needed")
    refused(lib, forward(workspace=4096, workspace_bytes=size - 1), f"{size} are needed")
    refused(lib, forward(workspace=4100, workspace_bytes=size), "aligned")
    refused(lib, lib.mbt_policy_loss_backward(0, C.byref(loss_struct(grad_loss=None)), None), "needs grad_loss")


def test_a_policy_loss_off_the_device_is_refused():
    from mbt_gym_amd import learning

    with pytest.raises(ValueError, match="no CPU path"):
        learning.policy_gradient_loss(torch.randn(3, 2), torch.randn(3, 2), torch.randn(3), 0.1)


# ---- the orthogonalisation --------------------------------------------------------------------------------------------------------------
def test_matrix_struct_layout(tmp_path):
    source = {"in_": "in"}
    fields = [f for f, _ in _native.MbtMatrix._fields_]
    body = "".join(f'  printf("{f} %zu\\n", offsetof(mbt_matrix, {source.get(f, f)}));\n' for f in fields)
    path = tmp_path / "matrix.c"
    path.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n  printf("sizeof %zu\\n", sizeof(mbt_matrix));\n{body}  return 0; }}\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(path), "-o", str(tmp_path / "matrix")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "matrix")], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(out.pop("sizeof")) == C.sizeof(_native.MbtMatrix)
    assert all(getattr(_native.MbtMatrix, f).offset == int(o) for f, o in out.items())


def matrix(rows=100, columns=90, batch=1, given=4096, out=4096):
    m = _native.MbtMatrix(in_=given, out=out, rows=rows, columns=columns, batch=batch)
    m.in_stride[:] = m.out_stride[:] = (rows * columns, columns, 1)
    return m


def test_the_library_refuses_malformed_matrices(lib):
    good = (C.c_double * 3)(3.4445, -4.7750, 2.0315)

    def call(*matrices, dtype=0, steps=5, coefficients=good, eps=1e-7, workspace=None, size=0, count=None):
        array = (_native.MbtMatrix * max(1, len(matrices)))(*matrices)
        return lib.mbt_orthogonalise(0, dtype, len(matrices) if count is None else count, array, steps, coefficients, eps, workspace, size, None)

    refused(lib, call(matrix(), dtype=9), "dtype 9")
    refused(lib, call(), "no matrices")
    refused(lib, lib.mbt_orthogonalise(0, 0, 1, None, 5, good, 1e-7, None, 0, None), "no matrices")
    refused(lib, call(matrix(), matrix(given=None)), "matrix 1: null argument")
    refused(lib, call(matrix(out=None)), "null argument")
    for bad in (matrix(rows=0), matrix(columns=0), matrix(rows=32769)):
        refused(lib, call(bad), "1 .. 32768")
    refused(lib, call(matrix(batch=0)), "batch of 0")
    refused(lib, call(matrix(rows=32768, columns=32768, batch=1 << 20)), "more elements")
    for many in (matrix(rows=3, columns=2, batch=1 << 22), matrix(rows=80, columns=66, batch=1 << 14), matrix(rows=66, columns=5, batch=1 << 14)):
        refused(lib, call(many), "more matrices than one launch takes")
    for steps in (0, -1, 65):
        refused(lib, call(matrix(), steps=steps), f"{steps} steps")
    for c in ((4.5, 0.0, 0.0), (1.0, 2.0, 0.0), (float("inf"), 0.0, 0.0), (0.0, float("nan"), 0.0)):
        refused(lib, call(matrix(), coefficients=(C.c_double * 3)(*c)), "1.9")
    refused(lib, call(matrix(), coefficients=None), "1.9")
    for eps in (-1.0, float("nan"), float("inf")):
        refused(lib, call(matrix(), eps=eps), "eps")
    size = lib.mbt_orthogonalise_workspace(1, matrix())
    assert size > 0 and lib.mbt_orthogonalise_workspace(1, matrix(64, 64)) == 0
    refused(lib, call(matrix()), f"{size} are needed")
    refused(lib, call(matrix(), workspace=4096, size=size - 1), f"{size} are needed")
    refused(lib, call(matrix(), workspace=4104, size=size), "aligned")


def test_updates_off_the_device_are_refused():
    from mbt_gym_amd import learning

    with pytest.raises(ValueError, match="no CPU path"):
        learning.orthogonalise(torch.randn(3, 2))
    parameter = torch.nn.Parameter(torch.randn(3, 2))
    parameter.grad = torch.ones(3, 2)
    with pytest.raises(ValueError, match="no CPU path"):
        learning.Muon([parameter]).step()
