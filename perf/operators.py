"""The operators a learner of this package runs between two rollouts, as measured work: cases, inputs, one pass, and what is exact.

Three families, in the order a training epoch uses them (mbt_gym_amd/learning):

  recurrence    h_t = g_t h_{t-1} + x_t along the time axis of a recording: the rewards-to-go of an episode (g a number, time reversed), the
                state of a recurrent actor (g a tensor, or f = sigmoid(gate) with h_t = f h_{t-1} + (1 - f) x_t) with its backward pass, and
                the single step that actor takes when it quotes
  policy_loss   minus the mean of log N(action | mean, std) x weight minus an entropy bonus, over the rows of a recording, with gradients
  orthogonalise five Newton-Schulz products X <- a X + (b X X^T + c (X X^T)^2) X of an update of a weight matrix

With `own` false `run` evaluates the plain forms: elementary torch operations in float32 (float64 for the long sums), rounded once at the end."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NORM_EPS = 1e-7


def listed():
    return [
        # 1000 trajectories x 200 steps (the default environment of the reference's examples): one learner's rewards-to-go, latency counts
        {"name": "to_go_1000_lanes", "op": "rewards_to_go", "lanes": 1000, "steps": 200, "discount": 1.0, "dtype": "float32"},
        # the benchmark's own recording, 2^20 lanes x 200 steps, discounted: read once, written once
        {"name": "to_go_2e20_lanes", "op": "rewards_to_go", "lanes": 1 << 20, "steps": 200, "discount": 0.99, "dtype": "float32"},
        # a recurrent actor of width 64 takes one step on 1000 lanes between two env.step calls
        {"name": "actor_step_1000_lanes", "op": "recurrence_step", "lanes": 1000, "width": 64, "dtype": "float32", "logit": True, "reset": True},
        # the same actor trained on a recording of 200 steps: forward and backward, (T, N, C) as recorded
        {"name": "actor_train_200_steps", "op": "recurrence", "form": "logit", "layout": "time_first", "steps": 200, "lanes": 1024, "width": 64,
         "dtype": "bfloat16", "reset": False, "reverse": False, "train": True},
        # episodes of odd length packed behind one another, gates as values, time contiguous as generate_trajectory returns it (N, C, T)
        {"name": "packed_1001_time_last", "op": "recurrence", "form": "value", "layout": "time_last", "steps": 1001, "lanes": 333, "width": 5,
         "dtype": "float32", "reset": True, "reverse": False, "train": True},
        # one market's tick history: few channels, a very long time axis, forward and backward
        {"name": "tick_history_65536", "op": "recurrence", "form": "logit", "layout": "time_first", "steps": 65536, "lanes": 1, "width": 64,
         "dtype": "float32", "reset": False, "reverse": False, "train": True},
        # the loss of one epoch of the agent's defaults (limit orders: two components), a fixed std
        {"name": "loss_1000_lanes", "op": "policy_loss", "steps": 200, "lanes": 1000, "actions": 2, "dtype": "float32", "std": "number",
         "mask": False, "entropy": 0.0},
        # a learnt std per component over the recording of 2^18 lanes; the actions are a view of the padded recording
        {"name": "loss_2e18_lanes", "op": "policy_loss", "steps": 200, "lanes": 1 << 18, "actions": 2, "dtype": "float32", "std": "component",
         "mask": False, "entropy": 0.01},
        # limit and market orders (four components), the std an output of the network, rows behind an episode's end masked, bfloat16 network
        {"name": "loss_masked_bf16", "op": "policy_loss", "steps": 50, "lanes": 16411, "actions": 4, "dtype": "bfloat16", "std": "full",
         "mask": True, "entropy": 0.01},
        # the weights of the actor that the fused rollout evaluates: 4 -> 64 -> 64 -> 2
        {"name": "actor_4_64_64_2", "op": "orthogonalise", "shapes": "64x4,64x64,2x64", "dtype": "float32"},
        # a mid-sized network with a flat and a tall matrix of odd size, gradients in bfloat16
        {"name": "layers_300x1000_bf16", "op": "orthogonalise", "shapes": "300x1000,1000x300,257x255", "dtype": "bfloat16"},
        # the largest square layer
        {"name": "layer_2048", "op": "orthogonalise", "shapes": "2048x2048", "dtype": "float32"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rewards_to_go", "recurrence_step", "recurrence", "recurrence", "policy_loss", "orthogonalise", "orthogonalise"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "rewards_to_go":
        lanes = _log_uniform(rng, 1, 1 << 20)
        steps = _log_uniform(rng, 1, min(1 << 16, max(1, (1 << 27) // lanes)))
        return {"op": op, "lanes": lanes, "steps": steps, "discount": rng.choice([1.0, 0.999, 0.9]), "dtype": "float32"}
    if op == "recurrence_step":
        width = _log_uniform(rng, 1, 256)
        return {"op": op, "lanes": _log_uniform(rng, 1, max(1, (1 << 24) // width)), "width": width, "dtype": dtype,
                "logit": rng.random() < 0.5, "reset": rng.random() < 0.5}
    if op == "recurrence":
        steps = _log_uniform(rng, 1, 1 << 16)
        width = _log_uniform(rng, 1, 256)
        lanes = _log_uniform(rng, 1, max(1, (1 << 24) // (steps * width)))
        return {"op": op, "form": rng.choice(["value", "logit"]), "layout": rng.choice(["time_first", "time_last"]), "steps": steps, "lanes": lanes,
                "width": width, "dtype": dtype, "reset": rng.random() < 0.4, "reverse": rng.random() < 0.3, "train": rng.random() < 0.75}
    if op == "policy_loss":
        lanes = _log_uniform(rng, 1, 1 << 18)
        return {"op": op, "steps": _log_uniform(rng, 1, max(1, min(1000, (1 << 24) // lanes))), "lanes": lanes, "actions": rng.randint(1, 8),
                "dtype": dtype, "std": rng.choice(["number", "component", "full"]), "mask": rng.random() < 0.4, "entropy": rng.choice([0.0, 0.01])}
    count, shapes = rng.randint(1, 4), []
    for _ in range(count):
        shapes.append("%dx%d" % (_log_uniform(rng, 2, 1024), _log_uniform(rng, 2, 1024)))
    return {"op": op, "shapes": ",".join(shapes), "dtype": dtype}


def _shapes(case):
    return [tuple(int(v) for v in text.split("x")) for text in case["shapes"].split(",")]


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    device = torch.device("cuda", 0)
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=device)

    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "rewards_to_go":
        # as the fused rollout records them: time first, lanes padded to a tile; the learner sees (N, 1, T)
        lanes, steps = case["lanes"], case["steps"]
        padded = -(-lanes // 512) * 512
        recorded = normal(steps, padded).mul_(0.3).add_(0.02)
        state["rewards"] = recorded[:, :lanes].t().unsqueeze(1)
    elif case["op"] == "recurrence_step":
        shape = (case["lanes"], case["width"])
        state["state"] = normal(*shape)
        state["inputs"] = normal(*shape).to(dtype)
        gate = normal(*shape) + 2.0
        state["gate"] = (gate if case["logit"] else torch.sigmoid(gate)).to(dtype)
        state["reset"] = (uniform(case["lanes"], 1) < 0.01).expand(shape) if case["reset"] else None
        state["new_state"] = torch.empty(shape, device=device)
    elif case["op"] == "recurrence":
        steps, lanes, width = case["steps"], case["lanes"], case["width"]
        last = case["layout"] == "time_last"
        shape = (lanes, width, steps) if last else (steps, lanes, width)
        state["inputs"] = normal(*shape).to(dtype)
        gate = normal(*shape) + 2.0
        state["gate"] = (gate if case["form"] == "logit" else torch.sigmoid(gate)).to(dtype)
        state["initial"] = normal(lanes, width)
        one = (lanes, 1, steps) if last else (steps, lanes, 1)
        state["reset"] = (uniform(*one) < 3.0 / steps).expand(shape) if case["reset"] else None
        if case["train"]:
            state["inputs"].requires_grad_(True)
            state["gate"].requires_grad_(True)
            state["initial"].requires_grad_(True)
            state["grad_states"] = normal(*shape).to(dtype)
            state["grad_final"] = normal(lanes, width)
    elif case["op"] == "policy_loss":
        steps, lanes, a = case["steps"], case["lanes"], case["actions"]
        padded = -(-lanes // 512) * 512
        mean = normal(steps, lanes, a).mul_(0.5)
        std = 0.05 if case["std"] == "number" else torch.exp(normal(a).mul_(0.2) - 2.0) if case["std"] == "component" else torch.exp(
            normal(steps, lanes, a).mul_(0.2) - 2.0)
        actions = torch.zeros(steps, padded, a, device=device)
        actions[:, :lanes] = mean + std * normal(steps, lanes, a)
        weights = torch.zeros(steps, padded, device=device)
        weights[:, :lanes] = normal(steps, lanes)
        state["mean"] = mean.to(dtype).requires_grad_(True)
        state["actions"], state["weights"] = actions[:, :lanes], weights[:, :lanes]
        state["std"] = std if case["std"] == "number" else (std.to(dtype) if case["std"] == "full" else std).requires_grad_(True)
        state["mask"] = None
        if case["mask"]:  # lanes end at their own step
            ends = torch.randint(1, steps + 1, (lanes,), generator=gen, device=device)
            state["mask"] = torch.arange(steps, device=device)[:, None] < ends[None, :]
    else:
        # a few strong directions over noise, as gradients of a network have them
        updates = []
        for m, n in _shapes(case):
            r = max(1, min(m, n) // 8)
            updates.append((normal(m, r) @ normal(r, n) / math.sqrt(r) * 1e-2 + normal(m, n) * 3e-3).to(dtype))
        state["updates"] = updates
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from mbt_gym_amd import learning

    case = state["case"]
    if case["op"] == "rewards_to_go":
        return learning.rewards_to_go(state["rewards"], case["discount"])
    if case["op"] == "recurrence_step":
        return learning.linear_recurrence_step(state["state"], state["inputs"], state["gate"], reset=state["reset"], gate_is_logit=case["logit"],
                                               new_state=state["new_state"])
    if case["op"] == "recurrence":
        axis = -1 if case["layout"] == "time_last" else 0
        states, final = learning.linear_recurrence(state["inputs"], state["gate"], state["initial"], dim=axis, reverse=case["reverse"],
                                                   reset=state["reset"], gate_is_logit=case["form"] == "logit", return_final=True)
        if not case["train"]:
            return states, final
        grads = torch.autograd.grad([states, final], [state["inputs"], state["gate"], state["initial"]], [state["grad_states"], state["grad_final"]])
        return (states.detach(), final.detach()) + tuple(grads)
    if case["op"] == "policy_loss":
        loss = learning.policy_gradient_loss(state["mean"], state["actions"], state["weights"], state["std"], mask=state["mask"],
                                             entropy_weight=case["entropy"])
        wanted = [state["mean"]] + ([] if case["std"] == "number" else [state["std"]])
        return (loss.detach(),) + tuple(torch.autograd.grad(loss, wanted))
    return learning.orthogonalise(state["updates"])


def _doubling(a, b):
    """Prefix of (a, b) -> h_t = a_t h_{t-1} + b_t along axis 0, h_{-1} = 0, in log2(T) elementwise passes."""
    steps, span = b.shape[0], 1
    while span < steps:
        b = torch.cat([b[:span], torch.addcmul(b[span:], a[span:], b[:-span])])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return b


def _run_plain(state):
    with torch.no_grad():
        case = state["case"]
        if case["op"] == "rewards_to_go":
            out, span = torch.flip(state["rewards"].float(), dims=(-1,)), 1
            while span < out.shape[-1]:
                out = torch.cat([out[..., :span], out[..., span:] + case["discount"] ** span * out[..., :-span]], dim=-1)
                span *= 2
            return torch.flip(out, dims=(-1,))
        if case["op"] == "recurrence_step":
            x, g, h = state["inputs"].float(), state["gate"].float(), state["state"]
            if state["reset"] is not None:
                h = torch.where(state["reset"], torch.zeros_like(h), h)
            if case["logit"]:
                f = torch.sigmoid(g)
                new = f * h + (1.0 - f) * x
            else:
                new = g * h + x
            return new.to(state["inputs"].dtype), new
        if case["op"] == "recurrence":
            return _plain_recurrence(state)
        if case["op"] == "policy_loss":
            return _plain_loss(state)
        return [_plain_orthogonalise(u) for u in state["updates"]]


def _plain_recurrence(state):
    case = state["case"]
    last = case["layout"] == "time_last"

    def arrange(t):  # time to the front, in the order in which it is walked
        t = t.movedim(-1, 0) if last else t
        return torch.flip(t, dims=(0,)) if case["reverse"] else t

    def back(t):
        t = torch.flip(t, dims=(0,)) if case["reverse"] else t
        return (t.movedim(0, -1) if last else t).to(state["inputs"].dtype)

    x, g, h0 = arrange(state["inputs"]).float(), arrange(state["gate"]).float(), state["initial"]
    logit = case["form"] == "logit"
    f = torch.sigmoid(g) if logit else g
    keep = f if state["reset"] is None else torch.where(arrange(state["reset"]), torch.zeros_like(f), f)  # what the carried state is multiplied by
    b = (1.0 - torch.sigmoid(g)) * x if logit else x.clone()
    b[0] += keep[0] * h0
    h = _doubling(keep, b)
    if not case["train"]:
        return back(h), h[-1].clone()
    d = arrange(state["grad_states"]).float().clone()
    d[-1] += state["grad_final"]
    shifted = torch.cat([keep[1:], torch.zeros_like(keep[:1])])
    d = torch.flip(_doubling(torch.flip(shifted, dims=(0,)), torch.flip(d, dims=(0,))), dims=(0,))  # d_t = dh_t + keep_{t+1} d_{t+1}
    before = torch.cat([h0[None], h[:-1]])
    if state["reset"] is not None:
        before = torch.where(arrange(state["reset"]), torch.zeros_like(before), before)
    grad_x = (1.0 - f) * d if logit else d
    grad_g = d * f * (1.0 - f) * (before - x) if logit else d * before
    return back(h), h[-1].clone(), back(grad_x), back(grad_g), keep[0] * d[0]


def _plain_loss(state):
    case = state["case"]
    mean, actions, w = state["mean"].float(), state["actions"].float(), state["weights"].float()[..., None]
    std = state["std"] if case["std"] != "number" else torch.tensor(state["std"], device=mean.device)
    std = std.float().expand_as(mean)
    rows = torch.ones_like(w, dtype=torch.bool) if state["mask"] is None else state["mask"][..., None]
    count = rows.sum(dtype=torch.float64) * mean.shape[-1]
    z = (actions - mean) / std
    log_prob = -0.5 * z * z - torch.log(std) - 0.5 * math.log(2.0 * math.pi)
    entropy = torch.log(std) + 0.5 * math.log(2.0 * math.pi * math.e)
    value = torch.where(rows, log_prob * w + case["entropy"] * entropy, torch.zeros_like(mean))
    loss = (-value.sum(dtype=torch.float64) / count).float()
    scale = (1.0 / count).float()
    grad_mean = torch.where(rows, -scale * w * z / std, torch.zeros_like(mean)).to(state["mean"].dtype)
    if case["std"] == "number":
        return loss, grad_mean
    grad_std = torch.where(rows, -scale * (w * (z * z - 1.0) / std + case["entropy"] / std), torch.zeros_like(mean))
    if case["std"] == "component":
        grad_std = grad_std.reshape(-1, mean.shape[-1]).sum(dim=0, dtype=torch.float64)
    return loss, grad_mean, grad_std.to(state["std"].dtype)


def _plain_orthogonalise(update):
    a, b, c = COEFFICIENTS
    x = update.float()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (torch.sqrt((x * x).sum()) + NORM_EPS)
    for _ in range(5):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.t() if tall else x).contiguous().to(update.dtype)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rewards_to_go":
            r = state["rewards"].double()
            out, carry = torch.empty_like(r), torch.zeros_like(r[..., 0])
            for t in range(case["steps"] - 1, -1, -1):
                carry = r[..., t] + case["discount"] * carry
                out[..., t] = carry
            return out
        if case["op"] == "recurrence_step":
            return _exact_step(state)
        if case["op"] == "recurrence":
            return _exact_recurrence(state)
        if case["op"] == "policy_loss":
            return _exact_loss(state)
        return [_exact_orthogonalise(u) for u in state["updates"]]


def _gates(gate, logit):
    """(what multiplies the state, what multiplies the input)"""
    gate = gate.double()
    if not logit:
        return gate, torch.ones_like(gate)
    return 1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))


def _exact_step(state):
    f, i = _gates(state["gate"], state["case"]["logit"])
    h = state["state"].double()
    if state["reset"] is not None:
        h = h.masked_fill(state["reset"], 0.0)
    new = f * h + i * state["inputs"].double()
    return new, new


def _exact_recurrence(state):
    case = state["case"]
    axis = 2 if case["layout"] == "time_last" else 0
    logit, steps = case["form"] == "logit", case["steps"]
    order = list(range(steps))[::-1] if case["reverse"] else list(range(steps))
    x = state["inputs"].double().movedim(axis, 0).contiguous()
    f, i = _gates(state["gate"].movedim(axis, 0).contiguous(), logit)
    cut = None if state["reset"] is None else state["reset"].movedim(axis, 0)
    h, carry, before = torch.empty_like(x), state["initial"].double(), torch.empty_like(x)
    for t in order:
        before[t] = carry if cut is None else carry.masked_fill(cut[t], 0.0)
        carry = torch.addcmul(i[t] * x[t], f[t], before[t])
        h[t] = carry
    if not case["train"]:
        return h.movedim(0, axis), carry
    up = state["grad_states"].double().movedim(axis, 0)
    d, flow = torch.empty_like(x), state["grad_final"].double()
    for t in reversed(order):
        d[t] = up[t] + flow
        flow = f[t] * d[t]
        if cut is not None:
            flow = flow.masked_fill(cut[t], 0.0)
    grad_gate = f * i * (before - x) * d if logit else before * d
    return h.movedim(0, axis), carry, (i * d).movedim(0, axis), grad_gate.movedim(0, axis), flow


def _exact_loss(state):
    case = state["case"]
    mean = state["mean"].detach().double().requires_grad_(True)
    given = state["std"]
    std = torch.tensor(given, dtype=torch.float64, device=mean.device) if case["std"] == "number" else given.detach().double().requires_grad_(True)
    with torch.enable_grad():
        spread = std.expand_as(mean)
        score = -((state["actions"].double() - mean) ** 2) / (2.0 * spread ** 2) - torch.log(spread * math.sqrt(2.0 * math.pi))
        total = score * state["weights"].double().unsqueeze(-1) + case["entropy"] * (0.5 + torch.log(spread * math.sqrt(2.0 * math.pi)))
        if state["mask"] is not None:
            total = total[state["mask"]]
        loss = -total.mean()
        grads = torch.autograd.grad(loss, [mean] if case["std"] == "number" else [mean, std])
    return (loss.detach(),) + tuple(grads)


def _exact_orthogonalise(update):
    g = update.double()
    if g.shape[0] < g.shape[1]:
        return _exact_orthogonalise(update.t()).t().contiguous()
    a, b, c = COEFFICIENTS  # tall: the products on the right, X (a + b X^T X + c (X^T X)^2)
    x = g / (torch.linalg.vector_norm(g) + NORM_EPS)
    eye = torch.eye(x.shape[1], dtype=torch.float64, device=x.device)
    for _ in range(5):
        inner = x.t().contiguous() @ x
        x = x @ (a * eye + inner @ (b * eye + c * inner))
    return x


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------
def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "rewards_to_go":
        n = case["lanes"] * case["steps"]
        return {"bytes": 2 * n * size, "flops": 2 * n}
    if case["op"] == "recurrence_step":
        n = case["lanes"] * case["width"]
        return {"bytes": n * (8 + 3 * size) + (case["lanes"] if case["reset"] else 0), "flops": (8 if case["logit"] else 2) * n}
    if case["op"] == "recurrence":
        lanes, n = case["lanes"] * case["width"], case["lanes"] * case["width"] * case["steps"]
        flags = case["lanes"] * case["steps"] if case["reset"] else 0
        arrays = 6 if case["train"] else 3
        return {"bytes": arrays * n * size + flags + (16 if case["train"] else 8) * lanes, "flops": (16 if case["train"] else 4) * n}
    if case["op"] == "policy_loss":
        rows, a = case["lanes"] * case["steps"], case["actions"]
        per_row = a * (2 * size + 4) + 4 + (2 * a * size if case["std"] == "full" else 0) + (1 if case["mask"] else 0)
        return {"bytes": rows * per_row + 4, "flops": 16 * rows * a}
    total = {"bytes": 0, "flops": 0}
    for m, n in _shapes(case):
        m, n = min(m, n), max(m, n)
        total["bytes"] += 2 * m * n * size
        total["flops"] += 5 * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)  # the two symmetric products, and Q X
    return total
