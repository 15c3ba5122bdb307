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


def test_operands_on_the_host_are_refused_without_a_device_too():
    """the question whether a stream is being captured is not asked for them: without a device it is an error"""
    from mbt_gym_amd.learning import Muon, RecurrentPolicy

    p = torch.nn.Parameter(torch.zeros(4, 3))
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="no CPU path"):
        Muon([p]).step()
    policy = RecurrentPolicy(3, 2, hidden_size=4)
    policy.begin_episode()
    with pytest.raises(ValueError, match="no CPU path"):
        policy.step(torch.zeros(5, 3))
    policy.begin_episode()
    with pytest.raises(ValueError, match="no CPU path"):
        policy(torch.zeros(2, 5, 3))
