"""The clipped policy loss with a KL term and its gradient against the formulas in float64.

Tolerances, with u = 2^-24.  An exponential of d = x - max is off by 2 u, of bfloat16 logits by
(|d| + 2) u (the product with log2 e is rounded); a sum of positive ones over a thread's at most 128
values by 128 u in the worst order and in practice by a few, its logarithm as much absolutely, and
what follows is float64.  So l is within 64 u (the terms that count have |d| < 32) and its rounding;
a row's loss is within that times its slope's terms T = r |A| + kl (1 + exp(ref - l)); a gradient
w c p within 192 u of w T p (the action's of w T), for the logits whose |d| is below 64.  A bfloat16
result has half a unit of 2^-8 more."""

import numpy as np
import pytest
import torch

import oxide_hip as ox
from test_gpu_rms_norm import TYPES, f64, make, within

pytestmark = pytest.mark.gpu
F32, U = torch.float32, 2.0 ** -24
# small and one block, one value, waves per row, odd, blocks, the registers' last, two passes
SHAPES = [(1, 1), (5, 2), (128, 10), (1024, 32), (1025, 10), (3, 33), (130, 100), (7, 509),
          (5, 1003), (9, 2047), (3, 4097), (2, 8192), (2, 16387), (2, 32768), (1, 65536),
          (2, 65541), (1, 131072), (2, 131077)]


def operands(shape, t, dev, seed=1, masked=False):
    rows, classes = shape
    g = torch.Generator().manual_seed(seed)
    x = make(shape, t, dev, seed) * 2
    a = torch.randint(0, classes, (rows,), generator=g)
    lp = torch.log_softmax(f64_t(x), 1).gather(1, a[:, None])[:, 0]
    old = (lp + 0.2 * torch.randn(rows, generator=g)).float()
    ref = (lp + 0.4 * torch.randn(rows, generator=g)).float()
    adv = torch.randn(rows, generator=g)
    w = None
    if masked:
        w = torch.rand(rows, generator=g) * (torch.rand(rows, generator=g) < 0.7)
        w[0] = 0.5
        w = w.to(dev)
    return [x, a.float().to(dev), old.to(dev), adv.to(dev), ref.to(dev), w]


def f64_t(x):
    return x.detach().cpu().double()


def reference(x, a, old, adv, ref, w, clip, kl, outer):
    x6, rows = f64(x), x.shape[0]
    a6 = f64(a).astype(int)
    w6 = np.full(rows, 1.0 / rows) if w is None else f64(w)
    top = x6.max(1, keepdims=True)
    e = np.exp(x6 - top)
    p = e / e.sum(1, keepdims=True)
    at = np.arange(rows), a6
    lp = x6[at] - top[:, 0] - np.log(e.sum(1))
    r = np.exp(lp - f64(old))
    adv = f64(adv)
    loss, slope, size = -np.minimum(r * adv, np.clip(r, 1 - clip[0], 1 + clip[1]) * adv), \
        np.where(r * adv <= np.clip(r, 1 - clip[0], 1 + clip[1]) * adv, -r * adv, 0.0), \
        r * np.abs(adv)
    if kl:
        d = f64(ref) - lp
        loss = loss + kl * (np.expm1(d) - d)
        slope = slope - kl * np.expm1(d)
        size = size + kl * (1 + np.exp(d))
    live = w6 != 0
    lp = np.where(live, lp, 0.0)
    loss, slope, size = (np.where(live, v * w6, 0.0) for v in (loss, slope, size))
    grad, mag = -p * slope[:, None], p * size[:, None]
    grad[at] += slope
    mag[at] = size
    near = 64 * U * size.sum() + U * np.abs(loss).sum()
    return loss.sum(), near, lp, grad * outer, mag * abs(outer)


def clear_of_borders(ops, clip):
    """Rows whose ratio lies within rounding of a border take either side: none of these do."""
    x, a, old = ops[0], ops[1], ops[2]
    lp = torch.log_softmax(f64_t(x), 1).gather(1, a.cpu().long()[:, None])[:, 0]
    r = torch.exp(lp - old.cpu().double())
    assert ((r - 1 + clip[0]).abs() > 1e-5).all() and ((r - 1 - clip[1]).abs() > 1e-5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("masked", [False, True])
def test_loss_and_gradient(module, dev, shape, dtype, masked):
    t, clip, kl, outer = TYPES[dtype], (0.2, 0.3), 0.1 if masked else 0.0, -1.5
    ops = operands(shape, t, dev, 3, masked)
    clear_of_borders(ops, clip)
    x, a, old, adv, ref, w = ops
    loss, lp, g = torch.empty(1, device=dev), torch.empty(shape[0], device=dev), torch.empty_like(x)
    flag = torch.zeros(1, dtype=torch.int32, device=dev)
    module.policy_loss(x, a, old, adv, loss, g, torch.full((1,), outer, device=dev), log_probs=lp,
                       reference_log_probs=ref if kl else None, weights=w, clip=clip, kl=kl,
                       error_flag=flag)
    want, near, want_lp, grad, mag = reference(x, a, old, adv, ref, w, clip, kl, outer)
    assert abs(float(loss) - want) <= near + U * abs(want), (float(loss), want, near)
    within(lp, want_lp, 64 + np.abs(want_lp), 1, F32, "log probabilities")
    within(g, grad, mag, 192, t, "gradient")
    assert int(flag) == 0


def test_each_output_alone(module, dev):
    x, a, old, adv, ref, w = operands((300, 700), F32, dev, 5, True)
    one = torch.ones(1, device=dev)
    loss, lp, g = torch.empty(1, device=dev), torch.empty(300, device=dev), torch.empty_like(x)
    rest = dict(reference_log_probs=ref, weights=w, kl=0.1)
    module.policy_loss(x, a, old, adv, loss, g, one, log_probs=lp, **rest)
    alone = torch.empty(1, device=dev), torch.empty(300, device=dev), torch.empty_like(x)
    module.policy_loss(x, a, old, adv, alone[0], **rest)
    module.policy_loss(x, a, old, adv, log_probs=alone[1], **rest)
    module.policy_loss(x, a, old, adv, None, alone[2], one, **rest)
    assert all(torch.equal(p, q) for p, q in zip((loss, lp, g), alone))


@pytest.mark.parametrize("classes", [10, 300, 5000, 70000, 140001])
def test_masked_places(module, dev, classes):
    """What a row of weight 0 holds never counts; a logit of minus infinity has no probability."""
    t = torch.bfloat16 if classes > 100000 else F32
    x, a, old, adv, ref, _ = operands((6, classes), t, dev, 7)
    w = torch.tensor([1.0, 0, 0.5, 0, 0, 2.0], device=dev)
    dead = w == 0
    x[:, 1::3] = -float("inf")
    a[~dead] = 3.0 * torch.tensor([0.0, 1, 2], device=dev)
    one, rest = torch.ones(1, device=dev), dict(weights=w, kl=0.1)

    def run():
        out = torch.empty(1, device=dev), torch.empty(6, device=dev), torch.empty_like(x)
        module.policy_loss(x, a, old, adv, out[0], out[2], one, log_probs=out[1],
                           reference_log_probs=ref, **rest)
        return out

    clean = run()
    assert clean[0].isfinite().all() and clean[2].isfinite().all()
    assert (clean[2][:, 1::3] == 0).all() and (clean[2][dead] == 0).all()
    assert (clean[1][dead] == 0).all()
    x[dead], old[dead], adv[dead], ref[dead] = float("nan"), float("inf"), float("nan"), float("nan")
    a[dead] = -7.0
    assert all(torch.equal(p, q) for p, q in zip(clean, run()))


def test_the_clip(module, dev):
    """Two classes of equal logits: l = -ln 2 for both, so r is exp of what `old` is put below it.
    On either side of a border, and on it (a ratio of 1 with no room): the border is inside."""
    old = torch.log(torch.tensor([0.5])).double()
    ratios = torch.tensor([1.5, 1.5, 0.5, 0.5, 1.0, 1.0], dtype=torch.float64)
    adv = torch.tensor([1.0, -1, 1, -1, 1, -1], device=dev)
    x = torch.zeros(6, 2, device=dev)
    a = torch.zeros(6, device=dev)
    olds = (old - torch.log(ratios)).float().to(dev)
    loss, g = torch.empty(1, device=dev), torch.empty_like(x)
    module.policy_loss(x, a, olds, adv, loss, g, torch.ones(1, device=dev), clip=(0.25, 0.25),
                       weights=torch.ones(6, device=dev))
    free = torch.tensor([0.0, 1.5, -0.5, 0, -1, 1], device=dev)  # slopes: 0 where the clip holds
    assert torch.allclose(g[:, 0], 0.5 * free, atol=1e-6)
    assert torch.allclose(g[:, 1], -0.5 * free, atol=1e-6)
    want = -(1.25 - 1.5 + 0.5 - 0.75 + 1 - 1)
    assert abs(float(loss) - want) < 1e-6
    # no room at all: a ratio of exactly 1 is its own border
    lp = torch.empty(6, device=dev)
    module.policy_loss(x, a, olds, adv, log_probs=lp)
    module.policy_loss(x, a, lp, adv, None, g, torch.ones(1, device=dev), clip=(1.0, 0.0),
                       weights=torch.ones(6, device=dev))
    assert (g[:, 0][adv < 0] != 0).all()


@pytest.mark.parametrize("shape", [(4, 10), (4, 3000), (2, 131077)])
def test_actions_that_are_no_class(module, dev, shape):
    for bad in (-1.0, 0.5, float(shape[1]), float("nan"), float("inf"), 1e20):
        x, a, old, adv, _, _ = operands(shape, F32, dev, 9)
        a[1] = bad
        loss, g = torch.empty(1, device=dev), torch.empty_like(x)
        flag = torch.zeros(1, dtype=torch.int32, device=dev)
        module.policy_loss(x, a, old, adv, loss, g, torch.ones(1, device=dev), error_flag=flag)
        assert int(flag) == 1 and loss.isnan().all() and g[1].isnan().all()
        assert g[0].isfinite().all()


def test_gradient_against_differences(module, dev):
    """Central differences of the loss along a random direction; h = 2^-8 of logits of size 2 on
    rows of 20 classes: truncation and rounding stay below 2e-3 of the slope's terms."""
    x, a, old, adv, ref, w = operands((40, 20), F32, dev, 11, True)
    v, h = make((40, 20), F32, dev, 12), 2.0 ** -8
    rest = dict(reference_log_probs=ref, weights=w, kl=0.2, clip=(0.9, 5.0))  # away from borders

    def value(step):
        loss = torch.empty(1, device=dev)
        module.policy_loss(x + step * v, a, old, adv, loss, **rest)
        return float(loss)

    g = torch.empty_like(x)
    module.policy_loss(x, a, old, adv, None, g, torch.ones(1, device=dev), **rest)
    slope = float((g.double() * v.double()).sum())
    size = float((g.double() * v.double()).abs().sum())
    assert abs((value(h) - value(-h)) / (2 * h) - slope) <= 2e-3 * size


def test_another_stream_graphs_and_repeats(module, dev):
    x, a, old, adv, ref, w = operands((700, 1003), torch.bfloat16, dev, 13, True)
    one = torch.ones(1, device=dev)

    def outputs():
        return torch.empty(1, device=dev), torch.empty(700, device=dev), torch.empty_like(x)

    def run(out, stream=None):
        module.policy_loss(x, a, old, adv, out[0], out[2], one, log_probs=out[1],
                           reference_log_probs=ref, weights=w, kl=0.1, stream=stream)

    want, outs = outputs(), (outputs(), outputs())
    run(want)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = [ox.HipGraphExec.capture(st, lambda o=o, st=st: run(o, st))
              for o, st in zip(outs, streams)]
    for _ in range(3):
        for o in outs:
            for v in o:
                v.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            graph.launch(st)
        eager = outputs()
        run(eager)
        torch.cuda.synchronize()
        for o in (*outs, eager):
            assert all(torch.equal(p, q) for p, q in zip(o, want))


def test_offsets_past_32_bits(module, dev):
    """More than 2^32 bytes of logits: rows at both ends against the formulas."""
    rows, classes = 40000, 60001
    x = torch.zeros(rows, classes, dtype=torch.bfloat16, device=dev)
    some = [0, 1, rows - 2, rows - 1]
    x[some] = make((4, classes), torch.bfloat16, dev, 1)
    a = torch.arange(rows, device=dev).float()
    old, adv = torch.full((rows,), -11.0, device=dev), torch.ones(rows, device=dev)
    w = torch.zeros(rows, device=dev)
    w[some] = 1.0
    g, one = torch.empty_like(x), torch.ones(1, device=dev)
    module.policy_loss(x, a, old, adv, None, g, one, weights=w, clip=(1.0, 1e6))
    pick = lambda v: v[some].contiguous()  # noqa: E731
    _, _, _, grad, mag = reference(pick(x), pick(a), pick(old), pick(adv), None, pick(w), (1.0, 1e6),
                                   0.0, 1.0)
    within(pick(g), grad, mag, 192, torch.bfloat16, "gradient")
    assert (g[2:4] == 0).all()
