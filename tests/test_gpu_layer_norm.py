"""Layer norm of a residual sum and its gradients on the device against the formulas in float64.

Tolerances, with u = 2^-24.  A sum over a row is a serial chain of at most 64 terms per thread, a
tree of 6 levels and 16 wave sums: its error is below 90 u of the sum of magnitudes.  So the mean is
off by at most 90 u of the mean magnitude A; a deviation s - m by that and one rounding; the sum of
squared deviations by 90 u of itself and, through the mean, by less than (90 u A)^2 per value; q by
half of that and 4 roundings.  y therefore is within 64 u of |y| and 128 u of q |w| A.  dx sums four
terms whose factors carry the errors of two dot products of that length: 192 u of the sum of the
terms' magnitudes.  dw and db add at most rows / groups + 128 + 16 terms in a chain: 256 u of the
sum of magnitudes, dw with the error of its deviations besides.  A bfloat16 result has half a unit
of 2^-8 relative rounding more."""

import numpy as np
import pytest
import torch

import oxide_hip as ox
from test_gpu_rms_norm import TYPES, f64, make, within

pytestmark = pytest.mark.gpu
F32 = torch.float32
SHAPES = [(1, 1), (3, 63), (5, 64), (7, 65), (1, 1024), (33, 333), (130, 96), (9, 2049), (4, 4096),
          (3, 8192), (2, 8193), (2, 16385), (2, 40000), (1, 70001), (2500, 40)]


def forward_ref(x, r, w, b, eps):
    s = f64(x) + (0.0 if r is None else f64(r))
    m = s.mean(-1)
    off = s - m[..., None]
    q = 1.0 / np.sqrt((off * off).mean(-1) + eps)
    y = off * q[..., None] * f64(w) + (0.0 if b is None else f64(b))
    size = np.abs(s).mean(-1)
    err = 64 * np.abs(y) + 128 * (q * size)[..., None] * np.abs(f64(w)) + \
        (0.0 if b is None else 2 * np.abs(f64(b)))
    return s, m, size, q, y, err


def check_forward(x, r, w, b, y, s, m, q, t, eps=1e-5):
    s_ref, m_ref, size, q_ref, y_ref, err = forward_ref(x, r, w, b, eps)
    if s is not None:
        within(s, s_ref, np.abs(s_ref), 1, t, "sum")
    if m is not None:
        within(m, m_ref, size, 90, F32, "mean")
        within(q, q_ref, q_ref * (1 + 90 * 2.0 ** -24 * (q_ref * size) ** 2), 64, F32, "deviation")
    within(y, y_ref, err, 1, t, "output")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("whole", [True, False])
def test_forward(module, dev, shape, dtype, whole):
    """With a residual, a bias and every output, and without them."""
    t = TYPES[dtype]
    x, w = make(shape, t, dev, 1), make(shape[-1:], F32, dev, 2) + 1.0
    if not whole:
        y = torch.empty_like(x)
        module.layer_norm_forward(x, w, None, y)
        return check_forward(x, None, w, None, y, None, None, None, t)
    r, b = make(shape, t, dev, 3) * 3 + 1, make(shape[-1:], F32, dev, 4)
    y, s = torch.empty_like(x), torch.empty_like(x)
    m, q = torch.empty(shape[0], device=dev), torch.empty(shape[0], device=dev)
    module.layer_norm_forward(x, w, b, y, m, q, residual=r, sum=s)
    check_forward(x, r, w, b, y, s, m, q, t)


def statistics(s, dev, eps=1e-5):
    _, m, _, q, _, _ = forward_ref(s, None, torch.ones(s.shape[-1]), None, eps)
    return torch.from_numpy(m).float().to(dev), torch.from_numpy(q).float().to(dev)


def check_backward(s, g, w, sg, m, q, dx, dw, db, t):
    s6, g6, w6, m6, q6 = f64(s), f64(g), f64(w), f64(m)[:, None], f64(q)[:, None]
    unit, d = (s6 - m6) * q6, g6 * w6
    size = np.abs(unit) + q6 * np.abs(m6) * 2.0 ** -6  # a deviation's own rounding is of s and m
    mean = lambda v: v.mean(-1, keepdims=True)  # noqa: E731
    ref = q6 * (d - mean(d) - unit * mean(unit * d))
    mag = q6 * (np.abs(d) + mean(np.abs(d)) + size * mean(size * np.abs(d)))
    if sg is not None:
        ref, mag = ref + f64(sg), mag + np.abs(f64(sg))
    within(dx, ref, mag, 192, t, "input gradient")
    if dw is not None:
        within(dw, (g6 * unit).sum(0), (np.abs(g6) * size).sum(0), 256, F32, "weight gradient")
    if db is not None:
        within(db, g6.sum(0), np.abs(g6).sum(0), 256, F32, "bias gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("outputs", ["all", "weight", "bias", "none"])
def test_backward(module, dev, shape, dtype, outputs):
    t = TYPES[dtype]
    s, g = make(shape, t, dev, 1) * 2 + 0.5, make(shape, t, dev, 2)
    w = make(shape[-1:], F32, dev, 3) + 1.0
    sg = make(shape, t, dev, 4) if outputs in ("all", "none") else None
    m, q = statistics(s, dev)
    dx = torch.empty_like(s)
    dw = torch.empty_like(w) if outputs in ("all", "weight") else None
    db = torch.empty_like(w) if outputs in ("all", "bias") else None
    module.layer_norm_backward(g, s, w, m, q, dx, dw, db, sum_gradient=sg)
    check_backward(s, g, w, sg, m, q, dx, dw, db, t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_other_alignments(module, dev, dtype, offset):
    t, shape = TYPES[dtype], (6, 512)
    x, r = make(shape, t, dev, 1, offset), make(shape, t, dev, 2)
    w, b = make((512,), F32, dev, 3, offset), make((512,), F32, dev, 8, 1)
    y, s = make(shape, t, dev, 4, offset), make(shape, t, dev, 5)
    m, q = torch.empty(6, device=dev), torch.empty(6, device=dev)
    module.layer_norm_forward(x, w, b, y, m, q, residual=r, sum=s)
    check_forward(x, r, w, b, y, s, m, q, t)
    g, dx, dw = make(shape, t, dev, 6), make(shape, t, dev, 7, offset), torch.empty(512, device=dev)
    db = make((512,), F32, dev, 9, offset)
    module.layer_norm_backward(g, s, w, m, q, dx, dw, db)
    check_backward(s, g, w, None, m, q, dx, dw, db, t)


@pytest.mark.parametrize("columns", [96, 1001, 40000])
def test_sum_in_place_and_gradient_in_place(module, dev, columns):
    shape = (5, columns)
    x, r = make(shape, F32, dev, 1), make(shape, F32, dev, 2)
    w, b = make((columns,), F32, dev, 3), make((columns,), F32, dev, 6)
    for into in ("x", "r"):
        a, c, y = x.clone(), r.clone(), torch.empty_like(x)
        module.layer_norm_forward(a, w, b, y, residual=c, sum=a if into == "x" else c)
        check_forward(x, r, w, b, y, a if into == "x" else c, None, None, F32)
    m, q = statistics(r, dev)
    g, sg = make(shape, F32, dev, 4), make(shape, F32, dev, 5)
    dx = sg.clone()
    module.layer_norm_backward(g, r, w, m, q, dx, None, sum_gradient=dx)
    check_backward(r, g, w, sg, m, q, dx, None, None, F32)


def test_rows_far_from_zero(module, dev):
    """A mean a thousand deviations away costs its own rounding, not the square's."""
    x = make((40, 1000), F32, dev, 1) + 1000.0
    w, b, y = torch.ones(1000, device=dev), torch.zeros(1000, device=dev), torch.empty_like(x)
    m, q = torch.empty(40, device=dev), torch.empty(40, device=dev)
    module.layer_norm_forward(x, w, b, y, m, q)
    check_forward(x, None, w, b, y, None, m, q, F32)


def test_gradients_against_differences(module, dev):
    """Central differences of sum(c . y) along random directions of x, w and b.  Their truncation is
    below h^2 / 6 of the third derivative (h = 2^-6: 1e-4 of the slope's scale), the rounding below
    4 u |c . y| sqrt(n) / h, n = 2880: 2e-3 of the largest slope covers both."""
    shape, h = (30, 96), 2.0 ** -6
    x, w, b, c = make(shape, F32, dev, 1), make((96,), F32, dev, 2) + 1, make((96,), F32, dev, 3), \
        make(shape, F32, dev, 4)
    vx, vw, vb = make(shape, F32, dev, 5), make((96,), F32, dev, 6), make((96,), F32, dev, 7)

    def value(step, dx, dw, db):
        y = torch.empty_like(x)
        module.layer_norm_forward(x + step * dx * vx, w + step * dw * vw, b + step * db * vb, y)
        return float((y.double() * c.double()).sum())

    y, m, q = torch.empty_like(x), torch.empty(30, device=dev), torch.empty(30, device=dev)
    module.layer_norm_forward(x, w, b, y, m, q)
    gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    module.layer_norm_backward(c, x, w, m, q, gx, gw, gb)
    slopes = [float((g.double() * v.double()).sum()) for g, v in ((gx, vx), (gw, vw), (gb, vb))]
    scale = max(abs(s) for s in slopes)
    for which, slope in zip(((1, 0, 0), (0, 1, 0), (0, 0, 1)), slopes):
        diff = (value(h, *which) - value(-h, *which)) / (2 * h)
        assert abs(diff - slope) <= 2e-3 * scale, (which, diff, slope)


def test_degenerate_rows(module, dev):
    """Rows of one repeated value have no deviation (epsilon keeps them finite); rows that are not
    finite stay rows; no rows leave parameter gradients of 0."""
    x, w, b = make((4, 300), F32, dev, 1), torch.ones(300, device=dev), torch.zeros(300, device=dev)
    clean = torch.empty_like(x)
    module.layer_norm_forward(x, w, b, clean)
    x[1], x[2, 7] = 3.0, float("nan")
    y = torch.empty_like(x)
    module.layer_norm_forward(x, w, b, y)
    assert torch.equal(y[[0, 3]], clean[[0, 3]]) and (y[1] == 0).all() and y[2].isnan().all()
    none = x[:0]
    module.layer_norm_forward(none, w, b, torch.empty_like(none))
    dw, db = torch.ones(300, device=dev), torch.ones(300, device=dev)
    empty = torch.empty(0, device=dev)
    module.layer_norm_backward(none, none, w, empty, empty, torch.empty_like(none), dw, db)
    assert (dw == 0).all() and (db == 0).all()


def test_another_stream_graphs_and_repeats(module, dev):
    """The same bits on a stream of the caller's, from two graphs replayed in turn and every run."""
    shape = (300, 1000)
    s, g = make(shape, torch.bfloat16, dev, 1), make(shape, torch.bfloat16, dev, 2)
    w, b = make((1000,), F32, dev, 3), make((1000,), F32, dev, 4)

    def outputs():
        return (torch.empty_like(s), torch.empty(300, device=dev), torch.empty(300, device=dev),
                torch.empty_like(s), torch.empty_like(w), torch.empty_like(b))

    def run(out, stream=None):
        y, m, q, dx, dw, db = out
        module.layer_norm_forward(s, w, b, y, m, q, stream=stream)
        module.layer_norm_backward(g, s, w, m, q, dx, dw, db, stream=stream)

    want = outputs()
    run(want)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    outs = outputs(), outputs()
    graphs = [ox.HipGraphExec.capture(st, lambda o=o, st=st: run(o, st))
              for o, st in zip(outs, (one, two))]
    for _ in range(3):
        for o in outs:
            for x in o:
                x.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, (one, two)):
            graph.launch(st)
        eager = outputs()
        run(eager)
        torch.cuda.synchronize()
        for o in (*outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(o, want))
