"""Forward-mode derivatives: refused, since a tangent would be passed by in silence."""
import pytest

torch = pytest.importorskip("torch")


def calls(x):
    from mbt_gym_amd import learning

    plain = torch.rand(x.shape, device=x.device)
    row = torch.rand(x.shape[0], device=x.device)
    return {"inputs": lambda: learning.linear_recurrence(x, plain), "gate": lambda: learning.linear_recurrence(plain, x),
            "initial": lambda: learning.linear_recurrence(plain, 0.5, x[0]), "to go": lambda: learning.rewards_to_go(x),
            "step": lambda: learning.linear_recurrence_step(plain, x, plain), "state": lambda: learning.linear_recurrence_step(x, plain, plain),
            "orthogonalise": lambda: learning.orthogonalise([plain, x]), "mean": lambda: learning.policy_gradient_loss(x, plain, row, 0.5),
            "actions": lambda: learning.policy_gradient_loss(plain, x, row, 0.5), "std": lambda: learning.policy_gradient_loss(plain, plain, row, x)}


def tangents_are_refused(device):
    import torch.autograd.forward_ad as forward_ad

    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.rand(5, 3, device=device), torch.ones(5, 3, device=device))
        for name, call in calls(x).items():
            with pytest.raises(ValueError, match="tangent" if device == "cuda" or name in ("inputs", "to go", "step", "mean") else "tangent|no CPU path"):
                call()


def test_tangents_are_refused():
    tangents_are_refused("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_device():
    tangents_are_refused("cuda")
