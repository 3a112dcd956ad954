"""The workloads on which the sequence operators' speed is measured: the calls that a program
training or running a recurrent sequence model makes, from a single token to the largest.

A case is a dict of plain values; ``kind`` says which operator it calls:

* ``norm_forward`` / ``norm_backward``: root-mean-square norm of a residual sum over the features
  of each row, and its gradients (the residual stream's own gradient added in);
* ``scan_forward`` / ``scan_backward``: the gated linear recurrence
  ``h_t = a_t h_{t-1} + (1 - a_t) u_t``, ``a_t = sigmoid(g_t)``, along the time axis, from an
  initial state to a final one (``ragged``: each row has a length of its own), and its gradients;
* ``orthogonalize``: five quintic Newton-Schulz rounds over a stack of matrices;
* ``muon``: one optimizer step (momentum, orthogonalisation, decayed update) over the matrices of
  ``count`` layers, in place.

``own`` false computes the plain forms (elementary torch operations in float32), ``own`` true
calls the framework.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PACKAGE = Path(__file__).resolve().parents[1] / "oxide-beta_amd"

EPSILON = 1e-6  # of the norm
QUINTIC = (3.4445, -4.7750, 2.0315)
ROUNDS, NS_EPSILON = 5, 1e-7
LR, DECAY, MOMENTUM = 0.02, 0.01, 0.95
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # one token between two layers of a model that answers: latency
        {"name": "norm fwd bf16 1x1024", "kind": "norm_forward", "dtype": "bf16", "rows": 1,
         "cols": 1024},
        # a large training batch at a wide layer
        {"name": "norm fwd bf16 16384x4096", "kind": "norm_forward", "dtype": "bf16",
         "rows": 16384, "cols": 4096},
        # 128 images of 28 rows (MNIST read row by row) at the repository's widest layer
        {"name": "norm bwd f32 3584x1280", "kind": "norm_backward", "dtype": "f32",
         "rows": 3584, "cols": 1280},
        # an odd number of odd rows: no row but the first is aligned
        {"name": "norm bwd bf16 1021x1537", "kind": "norm_backward", "dtype": "bf16",
         "rows": 1021, "cols": 1537},
        # one token for each of 64 streams, the state updated in place: latency
        {"name": "scan fwd f32 64x1x2048", "kind": "scan_forward", "dtype": "f32", "batch": 64,
         "time": 1, "channels": 2048, "ragged": False},
        # one long document: few independent rows, the time axis has to be split
        {"name": "scan fwd bf16 1x131072x512", "kind": "scan_forward", "dtype": "bf16",
         "batch": 1, "time": 131072, "channels": 512, "ragged": False},
        # an ordinary training batch
        {"name": "scan bwd f32 8x2048x2048", "kind": "scan_backward", "dtype": "f32",
         "batch": 8, "time": 2048, "channels": 2048, "ragged": False},
        # a ragged batch at odd sizes, one row of it empty
        {"name": "scan bwd bf16 5x1537x333", "kind": "scan_backward", "dtype": "bf16",
         "batch": 5, "time": 1537, "channels": 333, "ragged": True},
        # one 1 x 1 convolution's update (the repository's most frequent inverted bottleneck)
        {"name": "muon 1x192x96", "kind": "muon", "count": 1, "rows": 192, "cols": 96},
        # a model's layers of one shape in one step
        {"name": "muon 12x512x2048", "kind": "muon", "count": 12, "rows": 512, "cols": 2048},
        # the repository's 1000-class head: not a multiple of any tile
        {"name": "orthogonalize 1x1000x1280", "kind": "orthogonalize", "count": 1, "rows": 1000,
         "cols": 1280},
        # one large square matrix
        {"name": "orthogonalize 1x4096x4096", "kind": "orthogonalize", "count": 1, "rows": 4096,
         "cols": 4096},
    ]


def _log_uniform(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["norm_forward", "norm_backward", "scan_forward", "scan_backward",
                       "orthogonalize", "muon"])
    if kind.startswith("norm"):
        dtype = rng.choice(["f32", "bf16"])
        cols = _log_uniform(rng, 24, 8192)
        rows = _log_uniform(rng, 1, min(65536, (1 << 25) // cols))
        return {"kind": kind, "dtype": dtype, "rows": rows, "cols": cols}
    if kind.startswith("scan"):
        dtype = rng.choice(["f32", "bf16"])
        channels = _log_uniform(rng, 24, 4096)
        time = _log_uniform(rng, 1, min(131072, (1 << 24) // channels))
        batch = _log_uniform(rng, 1, max(1, min(64, (1 << 24) // (channels * time))))
        return {"kind": kind, "dtype": dtype, "batch": batch, "time": time,
                "channels": channels, "ragged": rng.random() < 0.5}
    rows, cols = _log_uniform(rng, 24, 2048), _log_uniform(rng, 24, 2048)
    count = _log_uniform(rng, 1, 12) if rows * cols <= 1 << 18 else 1
    return {"kind": kind, "count": count, "rows": rows, "cols": cols}


# ----------------------------------------------------------------------------- inputs

def _matrices(generator, count, rows, cols, scale):
    """Gradients as a mini-batch leaves them: some directions that matter, their strengths
    falling off, and the noise of the sample over all of them."""
    rank = min(64, rows, cols)
    strength = torch.arange(1, rank + 1, device="cuda", dtype=torch.float32) ** -0.75
    left = torch.randn(count, rows, rank, device="cuda", generator=generator) * strength
    right = torch.randn(count, rank, cols, device="cuda", generator=generator)
    noise = torch.randn(count, rows, cols, device="cuda", generator=generator)
    return (left @ right + noise) * scale


def _inputs(case: dict, seed: int) -> dict:
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    kind = case["kind"]

    def normal(*shape, dtype=torch.float32, scale=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=generator) * scale + mean).to(dtype)

    if kind.startswith("norm"):
        dtype, shape = DTYPES[case["dtype"]], (case["rows"], case["cols"])
        s = {"weight": normal(case["cols"], scale=0.2, mean=1.0)}
        if kind == "norm_forward":
            # a residual stream that has grown over the layers before, and one layer's output
            return s | {"x": normal(*shape, dtype=dtype),
                        "residual": normal(*shape, dtype=dtype, scale=3.0)}
        s["sum"] = normal(*shape, dtype=dtype, scale=3.0)
        s["inverse_rms"] = torch.rsqrt(s["sum"].float().square().mean(1) + EPSILON)
        return s | {"gradient": normal(*shape, dtype=dtype, scale=0.1),
                    "sum_gradient": normal(*shape, dtype=dtype, scale=0.1)}
    if kind.startswith("scan"):
        dtype = DTYPES[case["dtype"]]
        batch, time, channels = case["batch"], case["time"], case["channels"]
        shape = (batch, time, channels)
        s = {"x": normal(*shape, dtype=dtype),
             # most gates keep between half and 99 per cent of the state
             "gate": normal(*shape, dtype=dtype, scale=1.5, mean=2.0),
             "state": normal(batch, channels), "lengths": None}
        if case["ragged"]:
            lengths = torch.randint(0, time + 1, (batch,), device="cuda", dtype=torch.int32,
                                    generator=generator)
            lengths[0] = time
            if batch > 1:
                lengths[batch - 1] = 0
            s["lengths"] = lengths
        if kind == "scan_backward":
            s["h"] = _plain_scan_forward(s)[0]
            s["gradient"] = normal(*shape, dtype=dtype, scale=0.1)
            s["final_gradient"] = normal(batch, channels, scale=0.1)
        return s
    shape = (case["count"], case["rows"], case["cols"])
    s = {"update": _matrices(generator, *shape, 1e-3)}
    if kind == "muon":
        s["momentum"] = _matrices(generator, *shape, 1e-2)
        s["parameter"] = normal(*shape, scale=math.sqrt(2.0 / case["cols"]))
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    kind = case["kind"]
    # the buffers that a program keeps for the results
    if kind == "norm_forward":
        s["outputs"] = (torch.empty_like(s["x"]), torch.empty_like(s["x"]),
                        torch.empty(case["rows"], device="cuda"))
    elif kind == "norm_backward":
        s["outputs"] = (torch.empty_like(s["sum"]), torch.empty_like(s["weight"]))
    elif kind == "scan_forward":
        s["outputs"] = (torch.empty_like(s["x"]), torch.empty_like(s["state"]))
    elif kind == "scan_backward":
        s["outputs"] = (torch.empty_like(s["x"]), torch.empty_like(s["x"]),
                        torch.empty_like(s["state"]))
    elif kind == "orthogonalize":
        s["outputs"] = (torch.empty_like(s["update"]),)
    s["kind"] = kind
    return s


# ----------------------------------------------------------------------------- plain forms

def _plain_norm_forward(s):
    total = s["x"].float() + s["residual"].float()
    q = torch.rsqrt(total.square().mean(1) + EPSILON)
    y = total * q[:, None] * s["weight"]
    return y.to(s["x"].dtype), total.to(s["x"].dtype), q


def _plain_norm_backward(s):
    total, q, dy = s["sum"].float(), s["inverse_rms"][:, None], s["gradient"].float()
    unit = total * q
    d = dy * s["weight"]
    dx = s["sum_gradient"].float() + q * (d - unit * (unit * d).mean(1, keepdim=True))
    return dx.to(s["sum"].dtype), (dy * unit).sum(0)


def _live(s):
    """[batch, time, 1] truth values of the steps below each row's length."""
    steps = torch.arange(s["x"].shape[1], device=s["x"].device, dtype=torch.int32)
    return (steps < s["lengths"][:, None])[:, :, None]


def _compose(a, b):
    """h_t = a_t h_{t-1} + b_t from h_0 = 0 for every t, by doubling: after the round of span k
    (a, b)_t is the composition of the last 2 k steps up to t."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return a, b


def _plain_scan_forward(s):
    x, gate = s["x"].float(), s["gate"].float()
    a, b = torch.sigmoid(gate), torch.sigmoid(-gate) * x
    if s["lengths"] is not None:
        live = _live(s)
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    through, h = _compose(a, b)
    h = h + through * s["state"][:, None, :]
    final = h[:, -1].clone()
    if s["lengths"] is not None:
        h = torch.where(live, h, 0.0)
    return h.to(s["x"].dtype), final


def _plain_scan_backward(s):
    x, gate, dh = s["x"].float(), s["gate"].float(), s["gradient"].float()
    a, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    before = torch.cat([s["state"][:, None, :], s["h"][:, :-1].float()], 1)
    if s["lengths"] is not None:
        live = _live(s)
        a, keep, dh = torch.where(live, a, 1.0), torch.where(live, keep, 0.0), \
            torch.where(live, dh, 0.0)
    # l_t = dh_t + a_{t+1} l_{t+1}, the final state's gradient coming in behind the last step
    after = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    through, grad = _compose(after, dh.flip(1))
    grad = (grad + through * s["final_gradient"][:, None, :]).flip(1)
    dx, dg = keep * grad, a * keep * (before - x) * grad
    return dx.to(s["x"].dtype), dg.to(s["x"].dtype), a[:, 0] * grad[:, 0]


def _plain_orthogonalize(v):
    a, b, c = QUINTIC
    tall = v.shape[1] > v.shape[2]
    x = v.mT if tall else v
    x = x / (v.square().sum((1, 2), keepdim=True).sqrt() + NS_EPSILON)
    for _ in range(ROUNDS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT.contiguous() if tall else x


def _plain_muon(s):
    parameter, momentum, gradient = s["parameter"], s["momentum"], s["update"]
    momentum.mul_(MOMENTUM).add_(gradient)
    direction = _plain_orthogonalize(gradient + MOMENTUM * momentum)
    scale = math.sqrt(max(1.0, parameter.shape[1] / parameter.shape[2]))
    parameter.sub_(LR * (DECAY * parameter + scale * direction))
    return parameter, momentum


def _plain(s):
    kind = s["kind"]
    if kind == "norm_forward":
        return _plain_norm_forward(s)
    if kind == "norm_backward":
        return _plain_norm_backward(s)
    if kind == "scan_forward":
        return _plain_scan_forward(s)
    if kind == "scan_backward":
        return _plain_scan_backward(s)
    if kind == "orthogonalize":
        return _plain_orthogonalize(s["update"])
    return _plain_muon(s)


# ----------------------------------------------------------------------------- the framework

_loaded = None


def _module():
    """The framework's launchers on the current GPU, loaded once as a program does."""
    global _loaded
    if _loaded is None:
        if str(_PACKAGE) not in sys.path:
            sys.path.insert(0, str(_PACKAGE))
        import oxide_hip

        _loaded = oxide_hip.load_kernels(0)
    return _loaded


def _framework(s):
    m, kind = _module(), s["kind"]
    if kind == "norm_forward":
        y, total, q = s["outputs"]
        m.rms_norm_forward(s["x"], s["weight"], y, q, residual=s["residual"], sum=total,
                           epsilon=EPSILON)
    elif kind == "norm_backward":
        dx, dw = s["outputs"]
        m.rms_norm_backward(s["gradient"], s["sum"], s["weight"], s["inverse_rms"], dx, dw,
                            sum_gradient=s["sum_gradient"])
    elif kind == "scan_forward":
        h, final = s["outputs"]
        m.gated_recurrence_forward(s["x"], s["gate"], h, initial_state=s["state"],
                                   final_state=final, lengths=s["lengths"])
    elif kind == "scan_backward":
        dx, dg, ds = s["outputs"]
        m.gated_recurrence_backward(s["gradient"], s["x"], s["gate"], s["h"], dx, dg,
                                    initial_state=s["state"],
                                    final_state_gradient=s["final_gradient"],
                                    initial_state_gradient=ds, lengths=s["lengths"])
    elif kind == "orthogonalize":
        m.orthogonalize(s["update"], s["outputs"][0], rounds=ROUNDS, epsilon=NS_EPSILON)
        return s["outputs"][0]
    else:
        layers = list(zip(s["parameter"], s["update"], s["momentum"]))
        m.muon(LR, DECAY, MOMENTUM, layers, nesterov=True, rounds=ROUNDS, epsilon=NS_EPSILON)
        return s["parameter"], s["momentum"]
    return s["outputs"]


def run(state: dict):
    return _framework(state) if own else _plain(state)


# ----------------------------------------------------------------------------- work and oracle

def work(case: dict) -> dict:
    kind = case["kind"]
    if kind.startswith("norm"):
        rows, cols = case["rows"], case["cols"]
        n, size = rows * cols, DTYPES[case["dtype"]].itemsize
        if kind == "norm_forward":  # x, r in; sum, y, 1 / rms out
            return {"bytes": 4 * n * size + 4 * (rows + cols), "flops": 5 * n}
        # dy, ds, sum, 1 / rms in; dx, dw out
        return {"bytes": 4 * n * size + 4 * (rows + 2 * cols), "flops": 9 * n}
    if kind.startswith("scan"):
        states = case["batch"] * case["channels"]
        n, size = states * case["time"], DTYPES[case["dtype"]].itemsize
        if kind == "scan_forward":  # u, g, state in; h, state out
            return {"bytes": 3 * n * size + 8 * states, "flops": 8 * n}
        # dh, u, g, h, state, its gradient in; du, dg, the state's gradient out
        return {"bytes": 6 * n * size + 12 * states, "flops": 12 * n}
    count, rows, cols = case["count"], case["rows"], case["cols"]
    short, long = min(rows, cols), max(rows, cols)
    # X X' and A A are symmetric: half of each is enough; B X is whole
    flops = ROUNDS * count * (short * short * long + short ** 3 + 2 * short * short * long)
    # the matrix in and out; the optimizer: gradient in, momentum and parameter in and out
    moved = (5 if kind == "muon" else 2) * 4 * count * rows * cols
    return {"bytes": moved, "flops": flops}


def _f64(t):
    return t.detach().cpu().double().numpy()


def _exact_orthogonal(v):
    """By the definition in float64 (the products on the GPU where there is one)."""
    k1, k3, k5 = QUINTIC
    wide = v if v.shape[-2] <= v.shape[-1] else v.transpose(-1, -2).contiguous()
    norms = torch.linalg.vector_norm(wide, dim=(-2, -1), keepdim=True)
    y = wide / (norms + NS_EPSILON)
    for _ in range(ROUNDS):
        yyt = torch.matmul(y, y.transpose(-1, -2))
        y3 = torch.matmul(yyt, y)
        y = k1 * y + k3 * y3 + k5 * torch.matmul(yyt, y3)
    return y if v.shape[-2] <= v.shape[-1] else y.transpose(-1, -2).contiguous()


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm_forward":
        t = _f64(s["x"]) + _f64(s["residual"])
        q = 1.0 / np.sqrt(np.einsum("ij,ij->i", t, t) / t.shape[1] + EPSILON)
        return t * q[:, None] * _f64(s["weight"]), t, q
    if kind == "norm_backward":
        t, q, g, w = (_f64(s[k]) for k in ("sum", "inverse_rms", "gradient", "weight"))
        inner = np.einsum("ij,ij,j->i", g, t, w)
        dx = _f64(s["sum_gradient"]) + g * w * q[:, None] \
            - t * (inner * q ** 3 / t.shape[1])[:, None]
        return dx, np.einsum("ij,ij,i->j", g, t, q)
    if kind.startswith("scan"):
        batch, time, _ = s["x"].shape
        lengths = [time] * batch if s["lengths"] is None else s["lengths"].tolist()
        u, g, state = _f64(s["x"]), _f64(s["gate"]), _f64(s["state"])
        keep = 1.0 / (1.0 + np.exp(-g))
        new = 1.0 / (1.0 + np.exp(g))
        if kind == "scan_forward":
            h = np.zeros_like(u)
            for i in range(batch):
                for t in range(lengths[i]):
                    state[i] = keep[i, t] * state[i] + new[i, t] * u[i, t]
                    h[i, t] = state[i]
            return h, state
        h, dh, back = _f64(s["h"]), _f64(s["gradient"]), _f64(s["final_gradient"])
        du, dg = np.zeros_like(u), np.zeros_like(u)
        for i in range(batch):
            for t in range(lengths[i] - 1, -1, -1):
                back[i] += dh[i, t]
                du[i, t] = new[i, t] * back[i]
                before = h[i, t - 1] if t else state[i]
                dg[i, t] = keep[i, t] * new[i, t] * (before - u[i, t]) * back[i]
                back[i] *= keep[i, t]
        return du, dg, back
    update = s["update"].double()
    if kind == "orthogonalize":
        return _exact_orthogonal(update)
    momentum = MOMENTUM * s["momentum"].double() + update
    parameter = s["parameter"].double()
    direction = _exact_orthogonal(update + MOMENTUM * momentum)
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return parameter - LR * (DECAY * parameter + scale * direction), momentum
