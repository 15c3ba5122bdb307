"""mbt_gym_amd.learning in HIP graphs: calls that are captured apart from the ones they belong to."""
import pytest

from tests.learning_oracle import U

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kind", ["number", "component", "full"])
def test_a_backward_pass_captured_without_its_forward_pass(kind):
    """every replay writes the gradients for the loss gradient of that replay, whatever became of the arrays in between"""
    gen = torch.Generator(device="cuda").manual_seed(3)
    mean, actions = (torch.randn(500, 3, generator=gen, device="cuda") for _ in range(2))
    weights = torch.randn(500, generator=gen, device="cuda")
    std = {"number": 0.5, "component": torch.full((3,), 0.5, device="cuda"), "full": torch.full((500, 3), 0.5, device="cuda")}[kind]
    leaves = [t.requires_grad_(True) for t in (mean, std) if isinstance(t, torch.Tensor)]
    loss_gradient, stream = torch.tensor(1.0, device="cuda"), torch.cuda.Stream()

    def forward():
        from mbt_gym_amd import learning

        return learning.policy_gradient_loss(mean, actions, weights, std, entropy_weight=0.1)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(forward(), leaves, loss_gradient)
        loss = forward()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = torch.autograd.grad(loss, leaves, loss_gradient)
    torch.cuda.synchronize()
    expected = [g.double() for g in torch.autograd.grad(forward(), leaves)]
    for factor in (1.0, 3.0, 1.0, -0.5, 1.0):
        loss_gradient.fill_(factor)
        graph.replay()
        torch.cuda.synchronize()
        for out, one in zip(outs, expected):  # (a scaled gradient is off by the rounding of its scale and of its product)
            assert float((out.double() - factor * one).abs().max()) <= 4 * U * abs(factor) * float(one.abs().max())
            out.mul_(0.0)


def test_a_whole_pass_captured_twice_has_its_gradients_on_every_replay():
    """forward and backward in one graph, the loss gradient one, while the program clips the gradients in place; and both calls in graphs of their own"""
    from mbt_gym_amd import learning

    mean, actions, weights = torch.randn(300, 2, device="cuda", requires_grad=True), torch.randn(300, 2, device="cuda"), torch.randn(300, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(learning.policy_gradient_loss(mean, actions, weights, 0.5), mean)
        torch.cuda.synchronize()
        whole, front, back = (torch.cuda.CUDAGraph() for _ in range(3))
        with torch.cuda.graph(whole, stream=stream):
            together, = torch.autograd.grad(learning.policy_gradient_loss(mean, actions, weights, 0.5), mean)
        with torch.cuda.graph(front, stream=stream):
            loss = learning.policy_gradient_loss(mean, actions, weights, 0.5)
        with torch.cuda.graph(back, stream=stream):
            apart, = torch.autograd.grad(loss, mean)
    for _ in range(4):
        with torch.no_grad():
            mean.copy_(torch.randn(300, 2, device="cuda"))
            weights.copy_(torch.randn(300, device="cuda"))
        torch.cuda.synchronize()
        for graph in (whole, front, back, back):
            apart.zero_() if graph is back else None
            graph.replay()
        torch.cuda.synchronize()
        expected, = torch.autograd.grad(learning.policy_gradient_loss(mean, actions, weights, 0.5), mean)
        assert torch.equal(together, expected) and torch.equal(apart, expected)
        together.mul_(0.25)
