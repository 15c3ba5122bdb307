"""Parameters that Muon refuses, without a device."""
import pytest

torch = pytest.importorskip("torch")


def test_complex_parameters_are_refused():
    """their momentum would be that of the real parts"""
    from mbt_gym_amd.learning import Muon

    p = torch.nn.Parameter(torch.zeros(4, 3, dtype=torch.complex64))
    p.grad = torch.ones_like(p)
    optimizer = Muon([p])
    with pytest.raises(ValueError, match="complex64"):
        optimizer.step()
    assert not optimizer.state[p] and torch.equal(p.detach(), torch.zeros(4, 3, dtype=torch.complex64))
