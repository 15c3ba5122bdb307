"""What the recurrence's C side says about the float32 states that a 16-bit gate's gradient starts from, without a device."""
import ctypes as C

import pytest

from mbt_gym_amd import _native
from tests.test_learning_refusals import recurrence_struct, refused


@pytest.fixture(scope="module")
def lib():
    return _native.load_library()


def test_how_far_apart_the_backward_pass_needs_them(lib):
    def apart(**changes):
        return lib.mbt_recurrence_edge_steps(C.byref(recurrence_struct(**changes)))

    assert apart(steps=1000) == 0 and lib.mbt_recurrence_edge_steps(None) == 0  # (float32 states are stored unrounded)
    for dtype in (_native.BFLOAT16, _native.FLOAT16):
        distance = apart(steps=1000, dtype=dtype)
        assert distance > 0 and distance & (distance - 1) == 0
        assert apart(steps=1, dtype=dtype) == apart(steps=2, dtype=dtype) == 0  # (one piece, from the initial state)
        assert apart(steps=17, dtype=dtype) > 0
        assert apart(steps=1000, dtype=dtype, form=_native.GATE_CONSTANT, constant=0.5) == 0


def test_malformed_edges_are_refused(lib):
    def call(backward, **changes):
        r = recurrence_struct(**{**dict(steps=1000, dtype=_native.BFLOAT16), **changes})
        return (lib.mbt_recurrence_backward if backward else lib.mbt_recurrence_forward)(0, C.byref(r), None)

    distance = lib.mbt_recurrence_edge_steps(C.byref(recurrence_struct(steps=1000, dtype=_native.BFLOAT16)))
    needed = (-(-1000 // distance) - 1) * 2 * 4 * 4
    for backward in (False, True):
        for steps in (3, -4):
            refused(lib, call(backward, edge_steps=steps, edges=4096, edges_bytes=1 << 20), "no power of two")
        refused(lib, call(backward, edge_steps=distance), f"{needed} are needed")
        refused(lib, call(backward, edge_steps=distance, edges=4096, edges_bytes=needed - 1), f"{needed} are needed")
        refused(lib, call(backward, edge_steps=distance, edges=4098, edges_bytes=needed), "aligned")
        refused(lib, call(backward, edge_steps=distance, edges=4096, edges_bytes=needed, dtype=_native.FLOAT32), "16-bit")
    refused(lib, call(True, edge_steps=2 * distance, edges=4096, edges_bytes=needed), f"every {distance} steps")
    bare = recurrence_struct(steps=1000, dtype=_native.BFLOAT16)
    bare.states.data = None
    refused(lib, lib.mbt_recurrence_backward(0, C.byref(bare), None), "states or edges")


def test_constants_that_float32_does_not_hold_are_refused(lib):
    """3.5e38 is a finite double and an infinite float32; the largest float32 is taken as far as the check of the device"""
    for constant in (3.5e38, -1e39, 1e300):
        r = recurrence_struct(form=_native.GATE_CONSTANT, constant=constant)
        r.grad_gate.data = None
        for call in (lib.mbt_recurrence_forward, lib.mbt_recurrence_backward):
            refused(lib, call(0, C.byref(r), None), "not finite in float32")
    r.constant = -3.4028234663852886e38
    assert lib.mbt_recurrence_workspace(C.byref(r), 0) == 0 and lib.mbt_recurrence_forward(-1, C.byref(r), None) < 0
    assert b"float32" not in lib.mbt_last_error()


def test_numbers_that_the_loss_cannot_use_in_float32_are_refused(lib):
    """1 / 1e-39 is an infinity in float32, whose product with a difference of zero is NaN; the next ones up are taken as far as the workspace"""
    from tests.test_learning_refusals import loss_struct

    def forward(**changes):
        return lib.mbt_policy_loss_forward(0, C.byref(loss_struct(**changes)), None)

    for std in (1e-39, 2.9e-39, 1e-50, 5e-324):
        refused(lib, forward(std=std), "not finite in float32")
    for weight in (3.5e38, -1e300):
        refused(lib, forward(entropy_weight=weight), "entropy_weight is not finite")
    for std in (3e-39, 1e-20, 1e39):
        refused(lib, forward(std=std, entropy_weight=-3.4e38), "are needed")
