"""mbt_gym_amd.learning.policy_gradient_loss and its gradients against their definition in float64."""
import numpy as np
import pytest

from tests.learning_oracle import PolicyLoss, assert_within

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def loss_of(*arguments, **options):
    from mbt_gym_amd.learning import policy_gradient_loss

    return policy_gradient_loss(*arguments, **options)


def to64(t):
    return t.detach().double().cpu().numpy()


def make(rows, components, dtype, std, seed=0, padded=False, mask=False):
    """(mean, actions, weights, std, mask); padded: actions and weights are views of a wider recording"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    mean = normal(*rows, components) * 0.5
    spread = {"number": 0.07, "component": torch.exp(normal(components) * 0.3 - 1.5), "full": torch.exp(normal(*rows, components) * 0.3 - 1.5)}[std]
    wide = rows[:-1] + (rows[-1] + (13 if padded else 0),)
    actions, weights = torch.full(wide + (components,), float("nan"), device="cuda"), torch.full(wide, float("nan"), device="cuda")
    actions[..., :rows[-1], :] = mean + spread * normal(*rows, components)
    weights[..., :rows[-1]] = normal(*rows)
    keep = torch.rand(rows, generator=gen, device="cuda") < 0.7 if mask else None
    mean = mean.to(DTYPES[dtype]).requires_grad_(True)
    if std != "number":
        spread = (spread.to(DTYPES[dtype]) if std == "full" else spread).requires_grad_(True)
    return mean, actions[..., :rows[-1], :], weights[..., :rows[-1]], spread, keep


def check(mean, actions, weights, std, mask, entropy, dtype, factor=1.0):
    loss = loss_of(mean, actions, weights, std, mask=mask, entropy_weight=entropy)
    assert loss.shape == () and loss.dtype == torch.float32
    leaves = [mean] + ([std] if isinstance(std, torch.Tensor) else [])
    grads = torch.autograd.grad(loss * factor if factor != 1.0 else loss, leaves)
    ref = PolicyLoss(to64(mean), to64(actions), to64(weights), to64(std) if isinstance(std, torch.Tensor) else float(np.float32(std)),
                     None if mask is None else mask.cpu().numpy(), entropy, dtype, float(np.float32(factor)))
    what = (tuple(mean.shape), dtype, entropy, factor, mask is not None)
    assert_within(to64(loss), ref.loss, ref.loss_bound, ("loss",) + what)
    assert grads[0].dtype == mean.dtype and grads[0].shape == mean.shape
    assert_within(to64(grads[0]), ref.grad_mean, ref.grad_mean_bound, ("grad mean",) + what)
    if len(leaves) == 2:
        assert grads[1].dtype == std.dtype and grads[1].shape == std.shape
        assert_within(to64(grads[1]), ref.grad_std, ref.grad_std_bound, ("grad std",) + what)


ROWS = [(1,), (7,), (1023,), (1025,), (20, 1000), (50, 77), (3, 5, 11), (200, 3), (2, 70000)]


@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("std", ["number", "component", "full"])
@pytest.mark.parametrize("components", [1, 2, 4])
def test_loss_and_gradients_float32(rows, std, components):
    print(rows, std, components, flush=True)
    check(*make(rows, components, "float32", std), 0.0, "float32")
    check(*make(rows, components, "float32", std, seed=1, padded=True, mask=len(rows) > 1 or rows[0] > 50), 0.01, "float32")


@pytest.mark.parametrize("components", [3, 5, 6, 7, 8])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("std", ["number", "component", "full"])
def test_every_number_of_components_and_type(components, dtype, std):
    check(*make((13, 301), components, dtype, std, seed=2, padded=True, mask=True), 0.02, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("std", ["number", "component", "full"])
@pytest.mark.parametrize("factor", [1.0, 0.5, -3.0, 1.0e-3])
def test_a_scaled_loss(dtype, std, factor):
    """backward() looks at the gradient of the loss on the device: one is what the forward pass wrote, anything else is computed once more"""
    check(*make((31, 129), 2, dtype, std, seed=3, mask=True), 0.01, dtype, factor)
    check(*make((31, 129), 2, "float32", std, seed=4), 0.0, "float32", factor)


def test_a_large_recording():
    check(*make((100, 1 << 17), 2, "float32", "component", seed=5, padded=True), 0.01, "float32")


def test_without_gradients_none_are_computed():
    mean, actions, weights, std, _ = make((20, 30), 2, "float32", "component", seed=14)
    expected = loss_of(mean, actions, weights, std)
    with torch.no_grad():
        before = torch.cuda.memory_allocated()
        loss = loss_of(mean, actions, weights, std)
        assert torch.cuda.memory_allocated() - before < mean.numel() * 4  # (no room for a gradient of mean was taken and kept)
    assert not loss.requires_grad and torch.equal(loss, expected.detach())


def test_rows_beyond_32_bits_of_offset():
    """2^30 + 777 rows of two bfloat16 components and float32 actions (8.6 GB): the last rows count, and their gradients are where they belong"""
    rows = (1 << 30) + 777
    mean = torch.zeros(rows, 2, dtype=torch.bfloat16, device="cuda")
    actions = torch.zeros(rows, 2, device="cuda")
    weights = torch.zeros(rows, device="cuda")
    mean[-3:], actions[-3:], weights[-3:] = 0.25, torch.tensor([0.5, 0.125], device="cuda"), torch.tensor([1e9, -2e9, 3e9], device="cuda")
    mean.requires_grad_(True)
    loss = loss_of(mean, actions, weights, 0.5)
    grad, = torch.autograd.grad(loss, mean)
    ref = PolicyLoss(to64(mean[-3:]), to64(actions[-3:]), to64(weights[-3:]) * 3 / rows, 0.5, dtype="bfloat16")
    assert_within(to64(loss), ref.loss, ref.loss_bound, "loss")
    assert_within(to64(grad[-3:]), ref.grad_mean, ref.grad_mean_bound, "grad")
    assert int((grad != 0).sum()) == 6


def test_masked_rows_count_for_nothing_whatever_they_hold():
    mean, actions, weights, std, _ = make((40, 100), 2, "float32", "full", seed=6)
    keep = torch.rand(40, 100, device="cuda") < 0.5
    with torch.no_grad():
        for t, bad in ((mean, float("nan")), (actions, float("inf")), (weights, float("-inf")), (std, -1.0)):
            t[~keep] = bad
    check(mean, actions, weights, std, keep, 0.01, "float32")
    loss = loss_of(mean, actions, weights, std, mask=torch.zeros_like(keep))
    grads = torch.autograd.grad(loss, [mean, std])
    assert loss.item() == 0.0 and all(torch.equal(g, torch.zeros_like(g)) for g in grads)
    one = torch.zeros_like(keep)
    one[17, 3] = True
    with torch.no_grad():
        mean[17, 3], actions[17, 3], weights[17, 3], std[17, 3] = 0.1, 0.2, 1.5, 0.3
    check(mean, actions, weights, std, one, 0.0, "float32")
    component = torch.tensor([0.1, 0.2], device="cuda", requires_grad=True)
    empty = loss_of(mean, actions, weights, component, mask=torch.zeros_like(keep))
    assert torch.autograd.grad(empty * 2.0, component)[0].tolist() == [0.0, 0.0]


def test_an_unmasked_nan_is_not_hidden():
    mean, actions, weights, std, _ = make((4, 9), 2, "float32", "number", seed=7)
    with torch.no_grad():
        mean[2, 3, 1] = float("nan")
    loss = loss_of(mean, actions, weights, std)
    grad, = torch.autograd.grad(loss, mean)
    assert torch.isnan(loss) and torch.isnan(grad[2, 3, 1]) and torch.isfinite(grad).sum() == grad.numel() - 1


def test_layouts():
    mean, actions, weights, std, keep = make((6, 50, 30), 2, "float32", "full", seed=8, mask=True)
    turned = lambda t: t.detach().transpose(0, 2)  # noqa: E731 - batch axes that do not fold: the copies that do
    check(turned(mean).requires_grad_(True), turned(actions), turned(weights), turned(std).requires_grad_(True), turned(keep), 0.0, "float32")
    component_first = torch.randn(2, 80, 3, device="cuda").permute(1, 2, 0).requires_grad_(True)
    check(component_first, torch.randn(80, 3, 2, device="cuda"), torch.randn(3, 80, device="cuda").t(), 0.3, None, 0.0, "float32")
    row, single = torch.randn(3, device="cuda", requires_grad=True), torch.tensor([0.2, 0.3, 0.4], device="cuda", requires_grad=True)
    check(row, torch.randn(3, device="cuda"), torch.tensor(1.3, device="cuda"), 0.2, None, 0.0, "float32")
    loss = loss_of(row, torch.zeros(3, device="cuda"), torch.tensor(1.0, device="cuda"), single)
    assert torch.autograd.grad(loss, single)[0].shape == (3,)
    shared = torch.randn(2, device="cuda").expand(70, 2)  # one action for every row
    check(torch.randn(70, 2, device="cuda").requires_grad_(True), shared, torch.ones(1, device="cuda").expand(70), 0.5, None, 0.0, "float32")


def test_no_rows():
    mean = torch.empty(0, 2, device="cuda", requires_grad=True)
    loss = loss_of(mean, torch.empty(0, 2, device="cuda"), torch.empty(0, device="cuda"), 0.1)
    loss.backward()
    assert loss.item() == 0.0 and mean.grad.shape == (0, 2)


def test_a_graph_that_is_walked_twice():
    mean, actions, weights, std, _ = make((17, 23), 2, "float32", "component", seed=9)
    loss = loss_of(mean, actions, weights, std)
    first = torch.autograd.grad(loss, [mean, std], retain_graph=True)
    kept = [g.clone() for g in first]
    third = torch.autograd.grad(loss, [mean, std], torch.tensor(3.0, device="cuda"), retain_graph=True)
    again = torch.autograd.grad(loss, [mean, std])
    for a, b, c, d in zip(first, kept, third, again):
        assert torch.equal(a, b)  # nothing wrote to what had been handed out
        assert torch.equal(a, d)
        assert torch.allclose(c, 3.0 * a, rtol=4 * 2.0 ** -24, atol=0.0)
    mean.grad = None
    for _ in range(2):  # gradients accumulate
        loss_of(mean, actions, weights, std).backward()
    assert torch.allclose(mean.grad, 2 * first[0], rtol=2 * 2.0 ** -24, atol=0.0)


def test_gradients_agree_with_differences():
    mean, actions, weights, std, keep = make((5, 4), 2, "float32", "component", seed=10, mask=True)
    grads = torch.autograd.grad(loss_of(mean, actions, weights, std, mask=keep, entropy_weight=0.1), [mean, std])
    point = [to64(mean), to64(std)]
    step = 2.0 ** -12

    def value(m, s):
        return PolicyLoss(m, to64(actions), to64(weights), s, keep.cpu().numpy(), 0.1).loss

    for which, grad in enumerate(grads):
        for at in np.ndindex(point[which].shape):
            moved = []
            for sign in (1, -1):
                q = [p.copy() for p in point]
                q[which][at] += sign * step
                moved.append(value(*q))
            # the loss is quadratic in mean; its third derivative in std is a mean of |w| (12 z^2 + 2 + c) / std^3, |w| < 4, |z| < 5, std > 0.08
            third = 0.0 if which == 0 else 4 * (12 * 25 + 3) / 0.08 ** 3
            assert abs(float(grad[at]) - (moved[0] - moved[1]) / (2 * step)) <= step ** 2 / 6 * third + 1e-5


def test_captured_graphs_and_repeated_calls():
    mean, actions, weights, std, keep = make((60, 3000), 2, "float32", "component", seed=11, mask=True)
    other = make((60, 3000), 2, "float32", "component", seed=12, mask=True)

    def step():
        loss = loss_of(mean, actions, weights, std, mask=keep, entropy_weight=0.01)
        return [loss.detach()] + list(torch.autograd.grad(loss, [mean, std]))

    expected = step()
    assert all(torch.equal(a, b) for a, b in zip(expected, step()))  # the same bits
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = step()
    for turn in range(4):
        with torch.no_grad():
            for t, s in zip((mean, actions, weights, std, keep), other if turn % 2 == 0 else make((60, 3000), 2, "float32", "component", seed=20 + turn, mask=True)):
                t.copy_(s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step())), turn


def test_refusals_on_the_device():
    mean, actions, weights, std, keep = make((4, 5), 2, "float32", "number", seed=13, mask=True)
    for arguments, error, text in [
        ((mean.double(), actions, weights, 0.1), TypeError, "float64"), ((mean, actions[:3], weights, 0.1), ValueError, "shape"),
        ((mean, actions, weights[..., None], 0.1), ValueError, "shape"), ((mean, actions.half(), weights, 0.1), TypeError, "actions"),
        ((mean, actions, weights, 0.0), ValueError, "positive"), ((mean, actions, weights, float("nan")), ValueError, "positive"),
        ((mean, actions, weights, torch.ones(3, device="cuda")), ValueError, "std"), ((mean, actions, weights, torch.ones(2, device="cuda").half()), TypeError, "std"),
        ((mean, actions.clone().requires_grad_(True), weights, 0.1), ValueError, "detach"), ((mean, actions, weights.cpu(), 0.1), ValueError, "no CPU path"),
        ((torch.randn(4, 9, device="cuda"), torch.randn(4, 9, device="cuda"), torch.randn(4, device="cuda"), 0.1), ValueError, "1 to 8"),
    ]:
        with pytest.raises(error, match=text):
            loss_of(*arguments)
    with pytest.raises(TypeError, match="mask"):
        loss_of(mean, actions, weights, 0.1, mask=weights)
    with pytest.raises(ValueError, match="entropy_weight"):
        loss_of(mean, actions, weights, 0.1, entropy_weight=float("inf"))
    grad, = torch.autograd.grad(loss_of(mean, actions, weights, 0.1), mean, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), mean)


def test_numbers_that_float32_does_not_hold_are_refused():
    from mbt_gym_amd.learning import policy_gradient_loss

    mean = torch.zeros(4, 2, device="cuda")
    for std in (1e-39, 1e-50):
        with pytest.raises(ValueError, match="inverse"):
            policy_gradient_loss(mean, mean, mean[:, 0], std)
    with pytest.raises(ValueError, match="entropy_weight"):
        policy_gradient_loss(mean, mean, mean[:, 0], 0.5, entropy_weight=3.5e38)
    assert float(policy_gradient_loss(mean, mean, mean[:, 0] + 1.0, 4e-39)) == pytest.approx(np.log(4e-39) + 0.5 * np.log(2 * np.pi), rel=1e-6)
