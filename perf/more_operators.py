"""The workloads on which the speed of the layers and the loss of a sequence model that learns from
rewards is measured: the calls that a program makes that trains it, reads a prompt with it or lets
it answer token by token.

A case is a dict of plain values; ``kind`` says which operator it calls:

* ``layer_forward`` / ``layer_backward``: layer norm of a residual sum over the features of each
  row, and its gradients (the residual stream's own gradient added in);
* ``delta_step``: one token of the gated delta rule for each stream, the state updated in place;
* ``delta_forward``: the gated delta rule along the time axis, from an initial state to a final one
  (``ragged``: each row has a length of its own);
* ``delta_train``: its forward and every gradient, from zero states;
* ``policy``: the clipped policy loss with a KL term of rows of logits, its gradient and the log
  probabilities (``masked``: a third of the rows has weight 0).

The gated delta rule keeps a state S [key_dim, value_dim] for each head,
``S_t = P + b_t k_t (v_t - P' k_t)'``, ``P = a_t S_{t-1}``, ``o_t = scale S_t' q_t`` with
``a_t = sigmoid(gate_t)`` and ``b_t = sigmoid(write_t)``.

``own`` false computes the plain forms (elementary torch operations in float32), ``own`` true
calls the framework.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parents[1] / "oxide-beta_amd"

EPSILON = 1e-5  # of the norm
CHUNK = 64  # steps that the plain form of the delta rule takes at a time
CLIP, KL = (0.2, 0.28), 0.05
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # one token between two layers of a model that answers: latency
        {"name": "layer fwd bf16 1x2048", "kind": "layer_forward", "dtype": "bf16", "rows": 1,
         "cols": 2048},
        # a large training batch at a wide layer
        {"name": "layer bwd bf16 16384x4096", "kind": "layer_backward", "dtype": "bf16",
         "rows": 16384, "cols": 4096},
        # an odd number of odd rows: no row but the first is aligned
        {"name": "layer bwd f32 1021x1537", "kind": "layer_backward", "dtype": "f32",
         "rows": 1021, "cols": 1537},
        # one token of one stream: latency
        {"name": "delta step bf16 1x16", "kind": "delta_step", "dtype": "bf16", "batch": 1,
         "key_heads": 16, "heads": 16, "key_dim": 128, "value_dim": 128},
        # one token for each of 64 streams, two value heads to a key head
        {"name": "delta step bf16 64x32", "kind": "delta_step", "dtype": "bf16", "batch": 64,
         "key_heads": 16, "heads": 32, "key_dim": 128, "value_dim": 128},
        # one long prompt: few independent heads, the time axis is long
        {"name": "delta fwd bf16 1x32768x16", "kind": "delta_forward", "dtype": "bf16",
         "batch": 1, "time": 32768, "key_heads": 16, "heads": 16, "key_dim": 128,
         "value_dim": 128, "ragged": False},
        # a ragged batch at odd sizes, one row of it empty
        {"name": "delta fwd f32 5x333x6", "kind": "delta_forward", "dtype": "f32", "batch": 5,
         "time": 333, "key_heads": 3, "heads": 6, "key_dim": 48, "value_dim": 75,
         "ragged": True},
        # an ordinary training batch
        {"name": "delta train bf16 8x2048x16", "kind": "delta_train", "dtype": "bf16",
         "batch": 8, "time": 2048, "key_heads": 16, "heads": 16, "key_dim": 128,
         "value_dim": 128},
        # 128 images of 28 rows (MNIST read row by row) at 128 features in four heads
        {"name": "delta train f32 128x28x4", "kind": "delta_train", "dtype": "f32",
         "batch": 128, "time": 28, "key_heads": 4, "heads": 4, "key_dim": 32, "value_dim": 32},
        # the repository's batch and classes
        {"name": "policy f32 128x10", "kind": "policy", "dtype": "f32", "rows": 128,
         "cols": 10, "masked": False},
        # the tokens of a batch of answers over a vocabulary
        {"name": "policy bf16 8192x32768", "kind": "policy", "dtype": "bf16", "rows": 8192,
         "cols": 32768, "masked": False},
        # odd rows, a third of them padding
        {"name": "policy f32 509x1003 masked", "kind": "policy", "dtype": "f32", "rows": 509,
         "cols": 1003, "masked": True},
    ]


def _log_uniform(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["layer_forward", "layer_backward", "delta_step", "delta_forward",
                       "delta_train", "policy"])
    dtype = rng.choice(["f32", "bf16"])
    if kind.startswith("layer"):
        cols = _log_uniform(rng, 24, 8192)
        rows = _log_uniform(rng, 1, min(65536, (1 << 25) // cols))
        return {"kind": kind, "dtype": dtype, "rows": rows, "cols": cols}
    if kind == "policy":
        cols = _log_uniform(rng, 2, 65536)
        rows = _log_uniform(rng, 1, min(16384, (1 << 26) // cols))
        return {"kind": kind, "dtype": dtype, "rows": rows, "cols": cols,
                "masked": rng.random() < 0.5}
    key_heads, group = _log_uniform(rng, 1, 16), rng.choice([1, 1, 2, 3])
    heads = key_heads * group
    case = {"kind": kind, "dtype": dtype, "batch": 1, "key_heads": key_heads, "heads": heads,
            "key_dim": rng.choice([16, 32, 64, 96, 128, rng.randint(16, 128)]),
            "value_dim": rng.choice([32, 64, 128, 192, rng.randint(16, 200)])}
    if kind == "delta_step":
        case["batch"] = _log_uniform(rng, 1, max(1, 2048 // heads))
        return case
    most = 1 << (17 if dtype == "bf16" else 15)  # steps of all heads
    case["time"] = _log_uniform(rng, 1, min(8192, most // heads))
    case["batch"] = _log_uniform(rng, 1, max(1, min(64, most // (heads * case["time"]))))
    if kind == "delta_forward":
        case["ragged"] = rng.random() < 0.5
    return case


# ----------------------------------------------------------------------------- inputs

def _inputs(case: dict, seed: int) -> dict:
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32, scale=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=generator) * scale + mean).to(dtype)

    if kind.startswith("layer"):
        rows, cols = case["rows"], case["cols"]
        s = {"weight": normal(cols, scale=0.2, mean=1.0)}
        if kind == "layer_forward":
            # a residual stream that has grown over the layers before, and one layer's output
            return s | {"bias": normal(cols, scale=0.1), "x": normal(rows, cols, dtype=dtype),
                        "residual": normal(rows, cols, dtype=dtype, scale=3.0, mean=0.3)}
        s["sum"] = normal(rows, cols, dtype=dtype, scale=3.0, mean=0.3)
        wide = s["sum"].double()
        s["mean"] = wide.mean(1).float()
        s["inverse_deviation"] = torch.rsqrt(wide.var(1, unbiased=False) + EPSILON).float()
        return s | {"gradient": normal(rows, cols, dtype=dtype, scale=0.1),
                    "sum_gradient": normal(rows, cols, dtype=dtype, scale=0.1)}
    if kind == "policy":
        rows, cols = case["rows"], case["cols"]
        logits = normal(rows, cols, dtype=dtype, scale=2.0)
        actions = torch.randint(0, cols, (rows,), device="cuda", generator=generator)
        chosen = torch.log_softmax(logits.float(), 1).gather(1, actions[:, None])[:, 0]
        s = {"logits": logits, "actions": actions.float(),
             # the policy has moved on since the answers were drawn, some of them past the clip
             "old_log_probs": chosen + normal(rows, scale=0.15),
             "reference_log_probs": chosen + normal(rows, scale=0.3),
             "advantages": normal(rows, mean=0.2), "weights": None}
        if case["masked"]:
            live = torch.rand(rows, device="cuda", generator=generator) < 0.67
            live[0] = True
            s["weights"] = live.float() / live.sum()
        return s
    batch, key_heads, heads = case["batch"], case["key_heads"], case["heads"]
    time = case.get("time", 1)

    def unit(*shape):  # what the layer before leaves: directions
        v = normal(*shape)
        return (v / v.square().sum(-1, keepdim=True).sqrt()).to(dtype)

    s = {"query": unit(batch, time, key_heads, case["key_dim"]),
         "key": unit(batch, time, key_heads, case["key_dim"]),
         "value": normal(batch, time, heads, case["value_dim"], dtype=dtype),
         # most gates keep between 80 and 99.5 per cent of the state
         "gate": normal(batch, time, heads, dtype=dtype, scale=1.5, mean=3.0),
         "write": normal(batch, time, heads, dtype=dtype), "lengths": None}
    if kind == "delta_train":
        s["gradient"] = normal(batch, time, heads, case["value_dim"], dtype=dtype, scale=0.1)
        return s
    s["state"] = normal(batch, heads, case["key_dim"], case["value_dim"], scale=0.3)
    if case.get("ragged"):
        lengths = torch.randint(0, time + 1, (batch,), device="cuda", dtype=torch.int32,
                                generator=generator)
        lengths[0] = time
        if batch > 1:
            lengths[batch - 1] = 0
        s["lengths"] = lengths
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    kind = s["kind"] = case["kind"]
    # the buffers that a program keeps for the results
    if kind == "layer_forward":
        statistics = [torch.empty(case["rows"], device="cuda") for _ in range(2)]
        s["outputs"] = (torch.empty_like(s["x"]), torch.empty_like(s["x"]), *statistics)
    elif kind == "layer_backward":
        s["outputs"] = (torch.empty_like(s["sum"]), torch.empty_like(s["weight"]),
                        torch.empty_like(s["weight"]))
    elif kind == "policy":
        s["outer"] = torch.ones(1, device="cuda")
        s["outputs"] = (torch.empty(1, device="cuda"), torch.empty_like(s["advantages"]),
                        torch.empty_like(s["logits"]))
    elif kind == "delta_step":
        s["outputs"] = (torch.empty_like(s["value"]), s["state"])
    elif kind == "delta_forward":
        s["outputs"] = (torch.empty_like(s["value"]), torch.empty_like(s["state"]))
    else:
        s["outputs"] = (torch.empty_like(s["value"]),
                        *(torch.empty_like(s[k])
                          for k in ("query", "key", "value", "gate", "write")))
    return s


# ----------------------------------------------------------------------------- plain forms

def _plain_layer_forward(s):
    total = s["x"].float() + s["residual"].float()
    mean = total.mean(1)
    off = total - mean[:, None]
    q = torch.rsqrt(off.square().mean(1) + EPSILON)
    y = off * q[:, None] * s["weight"] + s["bias"]
    return y.to(s["x"].dtype), total.to(s["x"].dtype), mean, q


def _plain_layer_backward(s):
    dy, q = s["gradient"].float(), s["inverse_deviation"][:, None]
    unit = (s["sum"].float() - s["mean"][:, None]) * q
    d = dy * s["weight"]
    dx = s["sum_gradient"].float() + q * (d - d.mean(1, keepdim=True) -
                                          unit * (unit * d).mean(1, keepdim=True))
    return dx.to(s["sum"].dtype), (dy * unit).sum(0), dy.sum(0)


def _plain_policy(s):
    logits = s["logits"].float()
    rows = logits.shape[0]
    # what a row comes to is in 64 bits: a ratio beside the clip's border, a loss that cancels
    index = s["actions"].long()[:, None]
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, dtype=torch.float64)
    log_prob = (logits.gather(1, index) - top)[:, 0].double() - torch.log(total)
    weight = torch.full_like(log_prob, 1.0 / rows) if s["weights"] is None else \
        s["weights"].double()
    advantage = s["advantages"].double()
    ratio = torch.exp(log_prob - s["old_log_probs"].double())
    free, held = ratio * advantage, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * advantage
    away = s["reference_log_probs"].double() - log_prob
    loss = KL * (torch.exp(away) - away - 1) - torch.minimum(free, held)
    slope = KL * (1 - torch.exp(away)) - torch.where(free <= held, free, 0.0)
    live = weight != 0
    slope, loss = torch.where(live, slope * weight, 0.0), torch.where(live, loss * weight, 0.0)
    gradient = e * (-slope / total).float()[:, None]
    gradient.scatter_add_(1, index, slope.float()[:, None])
    return (loss.sum().float()[None], torch.where(live, log_prob, 0.0).float(),
            gradient.to(s["logits"].dtype))


def _log_sigmoid(x):
    return x.clamp(max=0) - torch.log1p(torch.exp(-x.abs()))


def _plain_delta(query, key, value, gate, write, state, lengths):
    """(out, final state) in float32, CHUNK steps at a time: within a chunk the errors
    e_t = v_t - (what the state holds for k_t) solve a triangular system."""
    batch, time, key_heads, key_dim = query.shape
    heads, scale = value.shape[2], key_dim ** -0.5
    short = -time % CHUNK

    def chunks(x):  # [batch, time, heads, ...] -> [batch, heads, chunks, CHUNK, ...]
        x = x.float()
        if x.shape[2] != heads:
            x = x.repeat_interleave(heads // key_heads, 2)
        x = torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, short))
        return x.unflatten(1, (-1, CHUNK)).movedim(3, 1)

    q, k, v = chunks(query), chunks(key), chunks(value)
    decay, beta = _log_sigmoid(chunks(gate).double()), torch.sigmoid(chunks(write).double())
    steps = torch.arange(time + short, device=q.device).view(1, 1, -1, CHUNK)
    ends = torch.full((batch,), time, device=q.device) if lengths is None else lengths
    live = steps < ends.view(-1, 1, 1, 1)
    k, v = torch.where(live[..., None], k, 0.0), torch.where(live[..., None], v, 0.0)
    decay, beta = torch.where(live, decay, 0.0), torch.where(live, beta, 0.0)
    # angles of decay grow with the chunk: their differences in 64 bits
    sums = decay.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    between = torch.exp((sums[..., :, None] - sums[..., None, :]).masked_fill(~lower, -math.inf))
    since, until = torch.exp(sums).float(), torch.exp(sums[..., -1:] - sums).float()
    # (1 + B)^-1 = (1 - B)(1 + B^2)(1 + B^4)...: alternating sums, in 64 bits
    power = (k @ k.mT).double() * between * beta[..., None, :]
    power = power.masked_fill(~lower.tril(-1), 0.0)
    one = torch.eye(CHUNK, device=q.device, dtype=torch.float64)
    inverse = one - power
    for _ in range(int(math.log2(CHUNK)) - 1):
        power = power @ power
        inverse = inverse + inverse @ power
    inverse, beta = inverse.float(), beta.float()
    fresh, stale = inverse @ v, inverse @ (since[..., None] * k)
    within = (q @ k.mT) * between.float() * beta[..., None, :]
    carry, old = (until * beta)[..., None] * k, since[..., None] * q
    s = torch.zeros(batch, heads, key_dim, value.shape[3], device=q.device) if state is None \
        else state
    out = []
    for c in range(q.shape[2]):  # the state goes from chunk to chunk
        error = fresh[:, :, c] - stale[:, :, c] @ s
        out.append(old[:, :, c] @ s + within[:, :, c] @ error)
        s = since[:, :, c, -1, None, None] * s + carry[:, :, c].mT @ error
    out = torch.where(live[..., None], torch.stack(out, 2), 0.0) * scale
    return out.movedim(1, 3).flatten(1, 2)[:, :time], s


def _plain_delta_step(s):
    query, key = (s[k][:, 0].float() for k in ("query", "key"))
    value, state = s["value"][:, 0].float(), s["state"]
    group = state.shape[1] // key.shape[1]
    query, key = query.repeat_interleave(group, 1), key.repeat_interleave(group, 1)
    state.mul_(torch.sigmoid(s["gate"][:, 0].float())[..., None, None])
    error = value - (state * key[..., None]).sum(2)
    error = error * torch.sigmoid(s["write"][:, 0].float())[..., None]
    state.add_(key[..., None] * error[:, :, None])
    out = (state * query[..., None]).sum(2) * key.shape[2] ** -0.5
    return out[:, None].to(s["value"].dtype), state


def _plain(s):
    kind = s["kind"]
    if kind == "layer_forward":
        return _plain_layer_forward(s)
    if kind == "layer_backward":
        return _plain_layer_backward(s)
    if kind == "policy":
        return _plain_policy(s)
    if kind == "delta_step":
        return _plain_delta_step(s)
    operands = [s[k] for k in ("query", "key", "value", "gate", "write")]
    if kind == "delta_forward":
        out, state = _plain_delta(*operands, s["state"], s["lengths"])
        return out.to(s["value"].dtype), state
    # reverse mode over the plain forward, in 32 bits
    leaves = [x.float().requires_grad_() for x in operands]
    out, _ = _plain_delta(*leaves, None, None)
    gradients = torch.autograd.grad(out, leaves, s["gradient"].float())
    dtype = s["value"].dtype
    return (out.detach().to(dtype), *(g.to(dtype) for g in gradients))


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
    m, kind, out = _module(), s["kind"], s["outputs"]
    if kind == "layer_forward":
        y, total, mean, q = out
        m.layer_norm_forward(s["x"], s["weight"], s["bias"], y, mean, q, residual=s["residual"],
                             sum=total, epsilon=EPSILON)
    elif kind == "layer_backward":
        m.layer_norm_backward(s["gradient"], s["sum"], s["weight"], s["mean"],
                              s["inverse_deviation"], *out, sum_gradient=s["sum_gradient"])
    elif kind == "policy":
        loss, log_probs, gradient = out
        m.policy_loss(s["logits"], s["actions"], s["old_log_probs"], s["advantages"], loss,
                      gradient, s["outer"], log_probs=log_probs,
                      reference_log_probs=s["reference_log_probs"], weights=s["weights"],
                      clip=CLIP, kl=KL)
    elif kind == "delta_step":
        m.gated_delta_rule_forward(s["query"], s["key"], s["value"], s["gate"], s["write"],
                                   out[0], initial_state=s["state"], final_state=s["state"])
    elif kind == "delta_forward":
        m.gated_delta_rule_forward(s["query"], s["key"], s["value"], s["gate"], s["write"],
                                   out[0], initial_state=s["state"], final_state=out[1],
                                   lengths=s["lengths"])
    else:
        saved = s.get("saved")
        if saved is None:  # once in a program's life
            saved = s["saved"] = m.gated_delta_rule_saved(s["key"], s["value"])
        m.gated_delta_rule_forward(s["query"], s["key"], s["value"], s["gate"], s["write"],
                                   out[0], saved=saved)
        m.gated_delta_rule_backward(s["gradient"], s["query"], s["key"], s["value"], s["gate"],
                                    s["write"], saved, *out[1:])
    return out


def run(state: dict):
    return _framework(state) if own else _plain(state)


# ----------------------------------------------------------------------------- work and oracle

def work(case: dict) -> dict:
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind.startswith("layer"):
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        if kind == "layer_forward":  # x, r in; sum, y, the statistics out
            return {"bytes": 4 * n * size + 8 * (rows + cols), "flops": 8 * n}
        # dy, ds, sum, the statistics in; dx, dw, db out
        return {"bytes": 4 * n * size + 8 * rows + 12 * cols, "flops": 13 * n}
    if kind == "policy":  # logits in, gradient out (a masked row: out)
        n = case["rows"] * case["cols"]
        read = 0.67 if case["masked"] else 1.0
        return {"bytes": int((1 + read) * n * size) + 28 * case["rows"], "flops": 6 * n}
    batch, time, heads = case["batch"], case.get("time", 1), case["heads"]
    keys, values = case["key_dim"], case["value_dim"]
    steps, state = batch * time * heads, batch * heads * keys * values
    q = batch * time * case["key_heads"] * keys * size
    v, g = steps * values * size, steps * size
    if kind == "delta_step":  # the state through k, the update, and q
        return {"bytes": 2 * q + 2 * v + 2 * g + 8 * state, "flops": 7 * state}
    # by chunks of c: two products with the state and its update, q k and k k, two triangles
    # with the values, and the triangular system (halves where a triangle is all that counts)
    c = min(CHUNK, time)
    forward = steps * (6 * keys * values + 2 * c * keys + 2 * c * values + c * c // 3)
    if kind == "delta_forward":
        return {"bytes": 2 * q + 2 * v + 2 * g + 8 * state, "flops": forward}
    # do with the state and its gradient, three times; the state's own way back; triangles
    backward = steps * (14 * keys * values + 4 * c * keys + 6 * c * values)
    # forward: q, k, v, gates in, o out; backward: the same and do in, five gradients out
    return {"bytes": (2 + 2 + 2) * q + (2 + 2 + 1) * v + 6 * g, "flops": forward + backward}


def _exact_delta(s, backward):
    """The recurrence step by step in float64; backward: its gradients from s["gradient"], with
    the states of one stretch of steps at a time formed again from those kept."""
    q, k, v = (s[x].double() for x in ("query", "key", "value"))
    a, b = torch.sigmoid(s["gate"].double()), torch.sigmoid(s["write"].double())
    batch, time, key_heads, keys = q.shape
    heads, values = v.shape[2:]
    group, scale = heads // key_heads, 1.0 / math.sqrt(keys)
    ends = [time] * batch if s["lengths"] is None else s["lengths"].tolist()
    live = torch.tensor([[t < n for n in ends] for t in range(time)], device=q.device)
    state = s["state"].double().clone() if "state" in s else torch.zeros(
        batch, heads, keys, values, dtype=torch.float64, device=q.device)

    def at(x, t):  # one step's values, key heads shared among their value heads
        x = x[:, t]
        return torch.repeat_interleave(x, group, 1) if x.shape[1] != heads else x

    def step(state, t):
        shrunk = a[:, t, :, None, None] * state
        wrong = at(v, t) - torch.matmul(at(k, t)[:, :, None], shrunk)[:, :, 0]
        new = torch.addcmul(shrunk, at(k, t)[..., None],
                            (b[:, t, :, None] * wrong)[:, :, None])
        return new, shrunk, wrong

    out, kept, stretch = torch.zeros_like(v), [], 64
    whole = all(n == time for n in ends)
    for t in range(time):
        if backward and t % stretch == 0:
            kept.append(state)
        new = step(state, t)[0]
        y = torch.matmul(at(q, t)[:, :, None], new)[:, :, 0] * scale
        if whole:
            state, out[:, t] = new, y
        else:
            on = live[t].view(-1, 1, 1, 1)
            state = torch.where(on, new, state)
            out[:, t] = torch.where(on[..., 0], y, 0.0)
    if not backward:
        return out, state
    g = s["gradient"].double()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    ds = torch.zeros_like(state)

    def shared(x):
        return x.view(batch, key_heads, group, keys).sum(2)

    for start in reversed(range(0, time, stretch)):
        states, last = [kept.pop()], min(time, start + stretch)
        for t in range(start, last):
            states.append(step(states[-1], t)[0])
        for t in reversed(range(start, last)):
            old, new = states[t - start], states[t - start + 1]
            _, shrunk, wrong = step(old, t)
            kt, bt, gt = at(k, t), b[:, t, :, None], g[:, t] * scale
            dq[:, t] = shared(torch.matmul(new, gt[..., None])[..., 0])
            ds = torch.addcmul(ds, at(q, t)[..., None], gt[:, :, None])
            # through S = P + b k (v - P'k)'
            into = torch.matmul(kt[:, :, None], ds)[:, :, 0]  # of b * wrong
            db[:, t] = (into * wrong).sum(-1)
            dv[:, t] = bt * into
            dk[:, t] = shared(torch.matmul(ds, (bt * wrong)[..., None])[..., 0]
                              - torch.matmul(shrunk, (bt * into)[..., None])[..., 0])
            ds = torch.addcmul(ds, kt[..., None], (-bt * into)[:, :, None])
            da[:, t] = (ds * old).sum((2, 3))
            ds = a[:, t, :, None, None] * ds
    return out, dq, dk, dv, da * a * (1 - a), db * b * (1 - b)


def _exact_policy(s):
    x, rows = s["logits"].double(), s["logits"].shape[0]
    picked = torch.nn.functional.one_hot(s["actions"].long(), x.shape[1]).bool()
    lse = torch.logsumexp(x, 1)
    log_prob = x[picked] - lse
    w = torch.full((rows,), 1.0 / rows, dtype=torch.float64, device=x.device) \
        if s["weights"] is None else s["weights"].double()
    adv = s["advantages"].double()
    r = torch.exp(log_prob - s["old_log_probs"].double())
    up, down = r > 1 + CLIP[1], r < 1 - CLIP[0]
    cut = (up & (adv >= 0)) | (down & (adv < 0))  # the clip holds the ratio
    bound = torch.where(adv >= 0, 1 + CLIP[1], 1 - CLIP[0])
    d = s["reference_log_probs"].double() - log_prob
    loss = (w * (-torch.where(cut, bound, r) * adv + KL * (torch.expm1(d) - d))).sum()
    c = w * (torch.where(cut, 0.0, -r * adv) - KL * torch.expm1(d))
    gradient = torch.exp(x - lse[:, None]).mul_(-c[:, None])
    gradient[picked] += c
    return loss[None], torch.where(w != 0, log_prob, 0.0), gradient


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "layer_forward":
        t = s["x"].double() + s["residual"].double()
        var, mean = torch.var_mean(t, 1, unbiased=False)
        q = (var + EPSILON) ** -0.5
        return (t - mean[:, None]) * (q[:, None] * s["weight"].double()) + s["bias"].double(), \
            t, mean, q
    if kind == "layer_backward":
        g, q = s["gradient"].double(), s["inverse_deviation"].double()
        n = g.shape[1]
        hat = (s["sum"].double() - s["mean"].double()[:, None]) * q[:, None]
        gw = g * s["weight"].double()
        along = torch.linalg.vecdot(gw, hat) / n
        dx = q[:, None] * (gw - (gw.sum(1) / n)[:, None] - hat * along[:, None])
        return s["sum_gradient"].double() + dx, torch.linalg.vecdot(g, hat, dim=0), g.sum(0)
    if kind == "policy":
        return _exact_policy(s)
    if kind == "delta_train":
        return _exact_delta(s, True)
    out, state = _exact_delta(s, False)
    return out, state
