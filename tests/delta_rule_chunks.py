"""The gated delta rule and its gradients by chunks, in float64 on the CPU: the formulas of the device's
kernels with a rounding of one's own where they round, and with any of their terms left out.

Operands are arrays [batch, time, heads, ...] with as many key heads as heads."""

import numpy as np

CHUNK = 64


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


def same(x):
    return x


def chunked(q, k, v, gate, write, gradient=None, scale=None, state=None, final=None, low=same,
            high=None, drop=()):
    """{name: array}: the output, the last state and, with a `gradient`, the operands' gradients and
    the first state's, from the first `state` and the `final` one's gradient (None: 0).  `low` rounds what the kernels keep in the operands' bits, `high` what a state that is handed on is
    made of (None: as `low`); `drop` names terms that are left out."""
    high = low if high is None else high
    keep = lambda name, x: 0.0 * x if name in drop else x  # noqa: E731
    q, k, v, gate, write = (np.moveaxis(x, 1, 2) for x in (q, k, v, gate, write))
    batch, heads, time, keys = k.shape
    scale = keys ** -0.5 if scale is None else scale
    log_a, b = -np.log1p(np.exp(-gate)), sigmoid(write)
    t_ = lambda x: np.swapaxes(x, -1, -2)  # noqa: E731
    s = np.zeros((batch, heads, keys, v.shape[3])) if state is None else state
    out, kept = np.zeros_like(v), []
    for first in range(0, time, CHUNK):
        at = slice(first, min(time, first + CHUNK))
        kc, qc, vc, bc = k[:, :, at], q[:, :, at], v[:, :, at], b[:, :, at]
        g = np.cumsum(log_a[:, :, at], -1)
        n = kc.shape[2]
        lower = np.tril(np.ones((n, n), bool))
        between = np.where(lower, np.exp(np.where(lower, g[..., :, None] - g[..., None, :], 0.0)), 0.0)
        a = kc @ t_(kc) * between * np.tril(np.ones((n, n)), -1)
        system = np.linalg.solve(np.eye(n) + a * bc[..., None, :], a)
        within = qc @ t_(kc) * between * scale
        since, until = np.exp(g)[..., None], np.exp(g[..., -1:] - g)[..., None]
        y = vc - keep("keys of the state", since * (kc @ high(s)))
        e = y - keep("system", high(system) @ high(bc[..., None] * y))
        u = bc[..., None] * e
        out[:, :, at] = keep("queries of the state", scale * since * (qc @ low(s))) + \
            keep("scores", low(within) @ low(u))
        kept.append((at, kc, qc, bc, g, between, system, within, since, until, low(s), low(e)))
        s = keep("decay", since[..., -1:, :] * s) + t_(kc) @ high(until * u)
    result = {"output": np.moveaxis(out, 2, 1), "state": s}
    if gradient is None:
        return result
    do = np.moveaxis(gradient, 1, 2)
    grads = [np.zeros_like(x) for x in (q, k, v, gate, write)]
    ds = np.zeros_like(s) if final is None else final
    for at, kc, qc, bc, g, between, system, within, since, until, s0, e in reversed(kept):
        doc, bb = do[:, :, at], bc[..., None]
        strict = between * np.tril(np.ones(between.shape[-2:]), -1)
        d_low = low(ds)
        du = keep("scores'", t_(low(within)) @ doc) + keep("keys of the state's gradient",
                                                           until * (kc @ d_low))
        x = du - keep("system'", t_(low(system)) @ low(bb * du))
        x_low = low(x)
        one = scale * between * (doc @ t_(e)) * bc[..., None, :]
        two = -strict * (x_low @ t_(e)) * bb * bc[..., None, :]
        q1 = keep("queries' state", scale * since * (doc @ t_(s0)))
        k1 = keep("keys' state", -since * bb * (x_low @ t_(s0)))
        k2 = keep("keys' state gradient", until * bb * (e @ t_(d_low)))
        qk, kk = qc @ t_(kc), kc @ t_(kc)
        worth = keep("pairs of queries", one * qk * (strict != 0)) + keep("pairs of keys", two * kk)
        after = worth.sum(-1) + keep("queries in the decay", (qc * q1).sum(-1)) + \
            keep("keys in the decay", (kc * k1).sum(-1)) - worth.sum(-2)
        before = keep("keys of the gradient in the decay", (kc * k2).sum(-1))
        suffix = np.flip(np.cumsum(np.flip(after, -1), -1), -1)
        whole = keep("state in the decay", since[..., -1, 0] * (d_low * s0).sum((-1, -2)))
        decay = suffix + np.cumsum(before, -1) - before + whole[..., None]
        grads[0][:, :, at] = q1 + keep("queries' pairs", low(one) @ kc)
        grads[1][:, :, at] = k1 + k2 + keep("keys' pairs of queries", t_(low(one)) @ qc) + \
            keep("keys' earlier pairs", low(two) @ kc) + keep("keys' later pairs", t_(low(two)) @ kc)
        grads[2][:, :, at] = low(bb * x)
        grads[3][:, :, at] = decay * sigmoid(-gate[:, :, at])
        grads[4][:, :, at] = (e * x_low).sum(-1) * bc * (1 - bc)
        ds = keep("decay of the gradient", since[..., -1:, :] * ds) + \
            keep("queries into the gradient", t_(qc) @ low(scale * since * doc)) - \
            keep("keys out of the gradient", t_(kc) @ low(since * bb * x))
    for name, x in zip(("query", "key", "value", "gate", "write"), grads):
        result[name] = np.moveaxis(x, 2, 1)
    result["first state"] = ds
    return result


def off(got, ref):
    """The Frobenius norm of the difference over the reference's."""
    return np.linalg.norm(got - ref) / np.linalg.norm(ref)
