"""The learner's operators from their definitions in float64 on the CPU, with bounds on what a float32 evaluation may differ by.

The bounds are derived, not fitted.  u is half a float32 step (2^-24) and v half a step of the element type.  A recurrence h = keep h + b that is
evaluated in any association - one step after another, or chunks whose composites are joined - sends every input through at most the products and
sums that stand between it and the output.  Per step of the walk these are two roundings (product, sum), four more for gates that are computed
(sigmoid and its complement, each good to two ulps); joining chunks adds at most 64 (six levels within a wave, sixteen waves, the composites of
segments in front: two roundings each).  With M the same recurrence over absolute values, the error E obeys E_t <= |keep| E_{t-1} + 6 u M_t, plus 64 u M_t
once."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
# below the smallest normal number the steps of a type stop shrinking: a rounding is then off by up to half of the smallest subnormal number
# (float16: 2^-24 / 2; of the others, nothing that counts)
HALF_SUBNORMAL = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}


def sigmoid_pair(k):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-k)), 1.0 / (1.0 + np.exp(k))


def _drop(keep, state):
    """keep * state, where a keep of zero drops the state whatever it holds"""
    with np.errstate(invalid="ignore", over="ignore"):
        return np.where(keep == 0.0, 0.0, keep * np.where(keep == 0.0, 0.0, state))


class Recurrence:
    """time first: x (T, B...), gate (T, B...) or a number, reset bool or None, initial (B...) or None"""

    def __init__(self, x, gate, form, initial=None, reset=None, reverse=False, dtype="float32"):
        self.reverse, self.form, self.v, self.w = reverse, form, HALF_STEP[dtype], HALF_SUBNORMAL[dtype]
        turn = self.turn
        self.x = turn(np.asarray(x, np.float64))
        if form == "constant":
            f, i = np.full_like(self.x, float(np.float32(gate))), np.ones_like(self.x)
        else:
            g = turn(np.asarray(gate, np.float64))
            f, i = (g, np.ones_like(g)) if form == "value" else sigmoid_pair(g)
        self.f, self.i = f, i
        self.cut = np.zeros(self.x.shape, bool) if reset is None else turn(np.asarray(reset, bool))
        self.keep = np.where(self.cut, 0.0, f)
        self.h0 = np.zeros(self.x.shape[1:]) if initial is None else np.asarray(initial, np.float64)
        h, m, e, r = self.h0, np.abs(self.h0), np.zeros_like(self.h0), np.zeros_like(self.h0)
        self.h, self.before, self.bound, self.before_bound = (np.empty_like(self.x) for _ in range(4))
        for t in range(len(self.x)):
            self.before[t] = np.where(self.cut[t], 0.0, h)
            self.before_bound[t] = np.where(self.cut[t], 0.0, e + 64 * U * m + r)
            b = i[t] * self.x[t]
            h = _drop(self.keep[t], h) + b
            m = _drop(np.abs(self.keep[t]), m) + np.abs(b)
            e = _drop(np.abs(self.keep[t]), e) + 6 * U * m
            r = np.maximum(self.v * np.abs(h) + self.w, np.abs(self.keep[t]) * r)  # (a stored state that the backward pass starts a chunk from)
            self.h[t], self.bound[t] = h, e + 64 * U * m
        self.final, self.final_bound = h, e + 64 * U * m

    def turn(self, a):
        return a[::-1] if self.reverse else a

    def states(self):
        return self.turn(self.h), self.turn(self.bound + self.v * np.abs(self.h) + self.w)

    def gradients(self, up, up_final=None):
        """{name: (value, bound)} of inputs, gate, initial"""
        up = self.turn(np.asarray(up, np.float64))
        steps = len(up)
        d = np.zeros_like(self.h0) if up_final is None else np.asarray(up_final, np.float64)
        m, e, keep = np.abs(d), np.zeros_like(self.h0), np.ones_like(self.h0)
        ds, db = np.empty_like(up), np.empty_like(up)
        for t in range(steps - 1, -1, -1):
            d = _drop(keep, d) + up[t]
            m = _drop(np.abs(keep), m) + np.abs(up[t])
            e = _drop(np.abs(keep), e) + 6 * U * m
            ds[t], db[t] = d, e + 64 * U * m
            keep = self.keep[t]
        out = {"initial": (_drop(keep, d), np.abs(keep) * (e + 64 * U * m) + 6 * U * np.abs(keep * d))}
        gx = self.i * ds
        out["inputs"] = (self.turn(gx), self.turn(np.abs(self.i) * db + (6 * U + self.v) * np.abs(gx) + self.w))
        if self.form == "value":
            gg = ds * self.before
            bound = db * np.abs(self.before) + np.abs(ds) * self.before_bound + (2 * U + self.v) * np.abs(gg) + self.w
        else:
            p, diff = self.f * self.i, self.before - self.x
            gg = p * diff * ds
            bound = p * (db * np.abs(diff) + np.abs(ds) * (self.before_bound + 2 * U * (np.abs(self.before) + np.abs(self.x)))) + (16 * U + self.v) * np.abs(gg) + self.w
        if self.form != "constant":
            out["gate"] = (self.turn(gg), self.turn(bound))
        return out


def assert_within(got, expected, bound, what):
    got, expected, bound = (np.asarray(a, np.float64) for a in (got, expected, bound))
    assert got.shape == expected.shape, (what, got.shape, expected.shape)
    off = np.abs(got - expected) - bound - 1e-37  # (subnormal results: the hardware's exponential flushes them)
    if off.size:
        worst = np.unravel_index(np.argmax(np.where(np.isnan(off), np.inf, off)), off.shape)
        assert off[worst] <= 0.0, (what, worst, got[worst], expected[worst], bound[worst])


class PolicyLoss:
    """rows x components in float64; std a number, (A,) or rows x components; mask bool over rows or None.  Bounds: z = (a - mean) / std carries four
    roundings, its square nine, the logarithm two ulps; a row is summed in float32, the rows in float64; one rounding at the end."""

    def __init__(self, mean, actions, weights, std, mask=None, entropy_weight=0.0, dtype="float32", grad_loss=1.0):
        mean, actions = np.asarray(mean, np.float64), np.asarray(actions, np.float64)
        keep = np.ones(mean.shape[:-1], bool) if mask is None else np.asarray(mask, bool)
        clean = lambda a, fill: np.where(keep[..., None], a, fill)  # noqa: E731
        w = clean(np.asarray(weights, np.float64)[..., None], 0.0)
        mean, actions = clean(mean, 0.0), clean(actions, 0.0)
        full = np.ndim(std) > 1
        sigma = np.broadcast_to(np.asarray(std, np.float64), mean.shape)
        sigma = clean(sigma, 1.0) if full else sigma
        n = keep.sum() * mean.shape[-1]
        c = float(np.float32(entropy_weight))
        v, tiny = HALF_STEP[dtype], HALF_SUBNORMAL[dtype]
        z = (actions - mean) / sigma
        log_prob, entropy = -0.5 * z * z - np.log(sigma) - 0.5 * np.log(2 * np.pi), np.log(sigma) + 0.5 * np.log(2 * np.pi * np.e)
        value = clean(w * log_prob + c * entropy, 0.0)
        size = clean(np.abs(w) * (0.5 * z * z + np.abs(np.log(sigma)) + 1.0) + abs(c) * (np.abs(np.log(sigma)) + 1.5), 0.0)
        scale = grad_loss / n if n else 0.0
        self.loss = -value.sum() / n if n else 0.0
        self.loss_bound = (16 + mean.shape[-1]) * U * size.sum() / max(n, 1) + U * abs(self.loss)
        self.grad_mean = -scale * w * z / sigma
        self.grad_mean_bound = (12 * U + v) * np.abs(self.grad_mean) + tiny
        each = clean((w * (z * z - 1.0) + c) / sigma, 0.0)
        each_bound = clean(16 * U * (np.abs(w) * (z * z + 1.0) + abs(c)) / sigma, 0.0)
        if full:
            self.grad_std = -scale * each
            self.grad_std_bound = abs(scale) * each_bound + (4 * U + v) * np.abs(self.grad_std) + tiny
        else:
            axes = tuple(range(mean.ndim - 1))
            self.grad_std = -scale * each.sum(axis=axes)
            self.grad_std_bound = abs(scale) * each_bound.sum(axis=axes) + 4 * U * np.abs(self.grad_std)


def orthogonalise(g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """(the formula in float64, a bound on the Frobenius norm of a float32-accurate evaluation's error).

    The bound follows the errors through the products.  Operands are good to 2^-21 (two float16 numbers and the product of their low parts that is left
    out), sums of k terms are float32: a product L R^T is off by at most e_k |L|_F |R|_F with e_k = 2^-20 + k U in Frobenius norm (the classical bound, k
    the terms of a sum).  One step maps singular values by f(s) = a s + b s^3 + c s^5; in the singular vectors' basis its derivative multiplies the entries of
    an error by the divided differences (f(s) - f(t)) / (s - t) and (f(s) + f(t)) / (s + t), all at most max |f'| over [0, |X|_2], so an error is passed on
    at most that many times in Frobenius norm, and the step adds those of its three products and of the split results.  The classical bound takes
    every rounding at its worst and all of one sign; a sum of k terms is off by a random walk, sqrt(k) instead of k, with overwhelming probability,
    and that is used here: e_k = 2^-20 + 4 sqrt(k) U."""
    a, b, c = coefficients
    x = np.asarray(g, np.float64)
    turned = x.shape[0] > x.shape[1]
    x = x.T if turned else x
    m, n = x.shape
    x = x / (np.sqrt((x * x).sum()) + eps)
    frob = np.linalg.norm
    en, em = 2.0 ** -20 + 4 * np.sqrt(n) * U, 2.0 ** -20 + 4 * np.sqrt(m) * U
    error = 4 * U * frob(x)
    for _ in range(steps):
        gram = x @ x.T
        q = a * np.eye(m) + b * gram + c * (gram @ gram)
        s = np.linalg.norm(x, 2)
        gram_error = en * frob(x) * s + 2 * U * frob(gram)
        square_error = em * frob(gram) * s * s
        q_error = (abs(b) + 2 * abs(c) * s * s) * gram_error + abs(c) * square_error + 4 * U * (frob(b * gram) + frob(c * gram @ gram) + abs(a) * np.sqrt(m))
        apply_error = em * frob(q @ x) + em * frob(x) * np.linalg.norm(q, 2)
        grid = np.linspace(0.0, s, 2001) ** 2
        error = error * np.abs(a + 3 * b * grid + 5 * c * grid * grid).max() + q_error * s + apply_error
        x = q @ x
    return (x.T if turned else x), error
