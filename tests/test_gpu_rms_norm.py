"""RMS norm of a residual sum and its gradients on the device against the formulas in float64.

Tolerances, with u = 2^-24.  A row's sum of squares (all terms positive) is a serial chain of at
most 64 terms per thread, a tree of 6 levels and 16 wave sums, so its relative error is below 90 u
and that of q = (mean + eps)^-1/2 below half of it plus 4 roundings; y has three more.  64 u covers
it.  dx sums three terms whose factors carry the errors of q and of one dot product of the same
length: 128 u of the sum of the terms' magnitudes (the dot product's own magnitudes inside).  dw
adds at most rows / groups + 128 + 16 terms in a chain: 256 u of the sum of magnitudes.  A bfloat16
result has half a unit of 2^-8 relative rounding more."""

import numpy as np
import pytest
import torch

import oxide_hip as ox

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# rows, columns: one value, a wave's share and one more, odd, whole packs, a block, several
# accesses per thread, longer than a block's registers
SHAPES = [(1, 1), (3, 63), (5, 64), (7, 65), (1, 1024), (33, 333), (130, 96), (9, 2049), (4, 4096),
          (3, 8192), (2, 8193), (2, 40000), (1, 70001), (2500, 40)]


def make(shape, dtype, dev, seed=1, offset=0):
    """Random values; ``offset`` elements into a larger buffer (another alignment)."""
    g = torch.Generator().manual_seed(seed)
    n = int(np.prod(shape))
    flat = torch.zeros(n + offset, dtype=dtype, device=dev)
    flat[offset:] = torch.randn(n, generator=g).to(dev).to(dtype)
    return flat[offset:].view(shape)


def f64(t):
    return t.detach().cpu().double().numpy()


def within(got, ref, magnitude, units, dtype, what):
    tol = units * U * magnitude + (2.0 ** -8 * np.abs(ref) if dtype == torch.bfloat16 else 0.0)
    bad = ~(np.abs(f64(got) - ref) <= tol + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3],
                           np.abs(f64(got) - ref).max())


def forward_ref(x, r, w, eps):
    s = f64(x) + (0.0 if r is None else f64(r))
    q = 1.0 / np.sqrt((s * s).mean(-1) + eps)
    return s, q, s * q[..., None] * f64(w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_forward(module, dev, shape, dtype, residual):
    t = TYPES[dtype]
    x, w = make(shape, t, dev, 1), make(shape[-1:], torch.float32, dev, 2) + 1.0
    r = make(shape, t, dev, 3) * 3 if residual else None
    y, s, q = torch.empty_like(x), torch.empty_like(x), torch.empty(shape[0], device=dev)
    module.rms_norm_forward(x, w, y, q, residual=r, sum=s, epsilon=1e-6)
    s_ref, q_ref, y_ref = forward_ref(x, r, w, 1e-6)
    within(s, s_ref, np.abs(s_ref), 1, t, "sum")
    within(q, q_ref, q_ref, 64, torch.float32, "inverse rms")
    within(y, y_ref, np.abs(y_ref), 64, t, "output")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("stream_gradient", [True, False])
def test_backward(module, dev, shape, dtype, stream_gradient):
    t = TYPES[dtype]
    s, g = make(shape, t, dev, 1) * 2, make(shape, t, dev, 2)
    w = make(shape[-1:], torch.float32, dev, 3) + 1.0
    sg = make(shape, t, dev, 4) if stream_gradient else None
    q = torch.from_numpy(1.0 / np.sqrt((f64(s) ** 2).mean(-1) + 1e-6)).float().to(dev)
    dx, dw = torch.empty_like(s), torch.empty_like(w)
    module.rms_norm_backward(g, s, w, q, dx, dw, sum_gradient=sg)
    check_backward(s, g, w, sg, q, dx, dw, t)


def check_backward(s, g, w, sg, q, dx, dw, t):
    s6, g6, w6, q6 = f64(s), f64(g), f64(w), f64(q)[:, None]
    unit, d = s6 * q6, g6 * w6
    inner = (unit * d).mean(-1, keepdims=True)
    ref = q6 * (d - unit * inner)
    mag = q6 * (np.abs(d) + np.abs(unit) * np.abs(unit * d).mean(-1, keepdims=True))
    if sg is not None:
        ref, mag = ref + f64(sg), mag + np.abs(f64(sg))
    within(dx, ref, mag, 128, t, "input gradient")
    if dw is not None:
        within(dw, (g6 * unit).sum(0), np.abs(g6 * unit).sum(0), 256, torch.float32,
               "weight gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_other_alignments(module, dev, dtype, offset):
    t, shape = TYPES[dtype], (6, 512)
    x, r = make(shape, t, dev, 1, offset), make(shape, t, dev, 2)
    w = make((512,), torch.float32, dev, 3, offset)
    y, s = make(shape, t, dev, 4, offset), make(shape, t, dev, 5)
    q = torch.empty(6, device=dev)
    module.rms_norm_forward(x, w, y, q, residual=r, sum=s)
    s_ref, _, y_ref = forward_ref(x, r, w, 1e-6)
    within(y, y_ref, np.abs(y_ref), 64, t, "output")
    within(s, s_ref, np.abs(s_ref), 1, t, "sum")
    g, dx, dw = make(shape, t, dev, 6), make(shape, t, dev, 7, offset), torch.empty(512, device=dev)
    module.rms_norm_backward(g, s, w, q, dx, dw)
    check_backward(s, g, w, None, q, dx, dw, t)


@pytest.mark.parametrize("columns", [96, 1001, 40000])
def test_sum_in_place_and_gradient_in_place(module, dev, columns):
    """The residual stream is updated where it lies; its gradient too."""
    shape = (5, columns)
    x, r = make(shape, torch.float32, dev, 1), make(shape, torch.float32, dev, 2)
    w = make((columns,), torch.float32, dev, 3)
    s_ref, _, y_ref = forward_ref(x, r, w, 1e-6)
    for into in ("x", "r"):
        a, b, y = x.clone(), r.clone(), torch.empty_like(x)
        module.rms_norm_forward(a, w, y, residual=b, sum=a if into == "x" else b)
        within(a if into == "x" else b, s_ref, np.abs(s_ref), 1, torch.float32, into)
        within(y, y_ref, np.abs(y_ref), 64, torch.float32, "output")
    q = torch.from_numpy(1.0 / np.sqrt((f64(r) ** 2).mean(-1))).float().to(dev)
    g, sg = make(shape, torch.float32, dev, 4), make(shape, torch.float32, dev, 5)
    dx = sg.clone()
    module.rms_norm_backward(g, r, w, q, dx, None, sum_gradient=dx)
    check_backward(r, g, w, sg, q, dx, None, torch.float32)


def test_gradient_against_differences(module, dev):
    """d loss / d(x, w) along random directions against central differences of the kernel's own
    forward.  With step h = 2^-6 the truncation is below h^2 of the terms' magnitudes (the third
    derivative of s / rms(s) along a unit-variance direction is of order 1) and the rounding of
    two float32 sums below 64 u / h of them: 1e-3 of the magnitudes covers both."""
    shape, h = (17, 200), 2.0 ** -6
    x, r = make(shape, torch.float32, dev, 1), make(shape, torch.float32, dev, 2)
    w, c = make((200,), torch.float32, dev, 3) + 1, make(shape, torch.float32, dev, 4)
    vx, vw = make(shape, torch.float32, dev, 5), make((200,), torch.float32, dev, 6)

    def loss(step):
        y, s, q = torch.empty_like(x), torch.empty_like(x), torch.empty(17, device=dev)
        module.rms_norm_forward(x + step * vx, w + step * vw, y, q, residual=r, sum=s)
        return float((f64(y) * f64(c)).sum()), s, q

    _, s, q = loss(0.0)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    module.rms_norm_backward(c, s, w, q, dx, dw)
    want = (f64(dx) * f64(vx)).sum() + (f64(dw) * f64(vw)).sum()
    size = np.abs(f64(dx) * f64(vx)).sum() + np.abs(f64(dw) * f64(vw)).sum()
    got = (loss(h)[0] - loss(-h)[0]) / (2 * h)
    assert abs(got - want) <= 1e-3 * size


def test_values_that_are_not_finite_stay_in_their_row(module, dev):
    x, w = make((4, 300), torch.float32, dev, 1), make((300,), torch.float32, dev, 2)
    clean = torch.empty_like(x)
    module.rms_norm_forward(x, w, clean)
    x[1, 7], x[2, 299] = float("nan"), float("inf")
    y = torch.empty_like(x)
    module.rms_norm_forward(x, w, y)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
    assert y[1].isnan().all()
    assert y[2, 299].isnan() and (y[2, :299] == 0).all()  # 1 / rms of an infinite row is 0
    zero = torch.zeros_like(x)
    module.rms_norm_forward(zero, w, y)
    assert (y == 0).all()


def test_no_rows(module, dev):
    x, w = torch.empty(0, 64, device=dev), torch.ones(64, device=dev)
    module.rms_norm_forward(x, w, torch.empty_like(x))
    dw = torch.ones(64, device=dev)
    module.rms_norm_backward(x, x, w, torch.empty(0, device=dev), torch.empty_like(x), dw)
    assert (dw == 0).all()


def test_another_stream_a_graph_and_repeats(module, dev):
    """The same bits on a stream of the caller's, from a replayed graph and on every run."""
    shape = (300, 1000)
    s, g = make(shape, torch.bfloat16, dev, 1), make(shape, torch.bfloat16, dev, 2)
    w = make((1000,), torch.float32, dev, 3)
    y, q = torch.empty_like(s), torch.empty(300, device=dev)
    dx, dw = torch.empty_like(s), torch.empty_like(w)

    def both(stream=None):
        module.rms_norm_forward(s, w, y, q, stream=stream)
        module.rms_norm_backward(g, s, w, q, dx, dw, stream=stream)

    both()
    torch.cuda.synchronize()
    want = [t.clone() for t in (y, q, dx, dw)]
    stream = torch.cuda.Stream()
    graph = ox.HipGraphExec.capture(stream, lambda: both(stream))
    for run in (lambda: both(stream), lambda: graph.launch(stream), lambda: graph.launch(stream)):
        for t in (y, q, dx, dw):
            t.zero_()
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        for a, b in zip((y, q, dx, dw), want):
            assert torch.equal(a, b)


# columns that are no multiple of an access: less than one, one and a value, one short of what a
# wave, four, and sixteen hold, past the registers; rows that make several turns of every group
RAGGED = [(3, 2), (5, 5), (9, 9), (4100, 33), (6, 255), (3, 513), (2100, 1283), (700, 2047),
          (4, 4095), (3, 8191), (2, 12001), (2, 16383), (2, 16385), (2, 32767), (2, 65535)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", RAGGED)
def test_ragged_rows(module, dev, shape, dtype):
    """Both directions, the sum over its operand and the gradient over the stream's, and nothing
    written behind or before an output."""
    t, rows = TYPES[dtype], shape[0]
    size = int(np.prod(shape))
    r, w = make(shape, t, dev, 2), make(shape[-1:], torch.float32, dev, 3) + 1.0
    x = make(shape, t, dev, 1)
    s_ref, q_ref, y_ref = forward_ref(x, r, w, 1e-6)
    around = torch.full((size + 64,), 7.0, dtype=t, device=dev)
    y = around[32:32 + size].view(shape)
    q = torch.empty(rows, device=dev)
    module.rms_norm_forward(x, w, y, q, residual=r, sum=x)
    within(x, s_ref, np.abs(s_ref), 1, t, "sum")
    within(q, q_ref, q_ref, 64, torch.float32, "inverse rms")
    within(y, y_ref, np.abs(y_ref), 64, t, "output")
    assert (around[:32] == 7).all() and (around[32 + size:] == 7).all()
    g, sg = make(shape, t, dev, 4), make(shape, t, dev, 5)
    dx = around[33:33 + size].view(shape)
    dx.copy_(sg)
    around[32], dw = 7.0, torch.empty_like(w)
    module.rms_norm_backward(g, x, w, q, dx, dw, sum_gradient=dx)
    check_backward(x, g, w, sg, q, dx, dw, t)
    assert (around[:33] == 7).all() and (around[33 + size:] == 7).all()


def test_offsets_past_32_bits(module, dev):
    """More than 2^31 elements: the last rows against the formulas."""
    t, shape = torch.bfloat16, (70001, 32765)
    x = torch.randn(shape, dtype=t, device=dev)
    w = torch.randn(shape[1], device=dev)
    y, q = torch.empty_like(x), torch.empty(shape[0], device=dev)
    module.rms_norm_forward(x, w, y, q)
    s_ref, q_ref, y_ref = forward_ref(x[-3:], None, w, 1e-6)
    within(q[-3:], q_ref, q_ref, 64, torch.float32, "inverse rms")
    within(y[-3:], y_ref, np.abs(y_ref), 64, t, "output")
    dx = torch.empty_like(x)
    module.rms_norm_backward(y, x, w, q, dx, None)
    check_backward(x[-3:], y[-3:], w, None, q[-3:], dx[-3:], None, t)


@pytest.mark.parametrize("shape", [(1, 1024), (16, 1024), (17, 1024), (16, 33), (5, 7), (2, 4096),
                                   (3, 4096), (1, 40000)])
def test_few_rows(module, dev, shape):
    """The weight gradient that one block writes by itself, and the row counts beside it."""
    t = torch.float32
    s, g = make(shape, t, dev, 1), make(shape, t, dev, 2)
    w = make(shape[-1:], t, dev, 3) + 1.0
    q = torch.from_numpy(1.0 / np.sqrt((f64(s) ** 2).mean(-1) + 1e-6)).float().to(dev)
    dx, around = torch.empty_like(s), torch.full((shape[1] + 20,), 7.0, device=dev)
    dw = around[9:9 + shape[1]]
    module.rms_norm_backward(g, s, w, q, dx, dw)
    check_backward(s, g, w, None, q, dx, dw, t)
    assert (around[:9] == 7).all() and (around[9 + shape[1]:] == 7).all()


def test_more_rows_than_a_launch_takes(module, dev):
    """2^26 rows and a few, 64 threads each: more than 2^32, which one launch cannot number.  The
    rows beside every 2^25th and the last ones, the sum where its operand lay."""
    t, shape = torch.bfloat16, ((1 << 26) + 5, 8)
    x, w = torch.randn(shape, dtype=t, device=dev), make((8,), torch.float32, dev, 2) + 1.0
    r = torch.randn(shape, dtype=t, device=dev)
    some = [0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, (1 << 26) - 1, 1 << 26, (1 << 26) + 4]
    ref = forward_ref(x[some], r[some], w, 1e-6)
    y, q = torch.zeros_like(x), torch.zeros(shape[0], device=dev)
    module.rms_norm_forward(x, w, y, q, residual=r, sum=x)
    within(x[some], ref[0], np.abs(ref[0]), 1, t, "sum")
    within(q[some], ref[1], ref[1], 64, torch.float32, "inverse rms")
    within(y[some], ref[2], np.abs(ref[2]), 64, t, "output")
    assert bool((q > 0).all())
    dx = torch.empty_like(x)
    module.rms_norm_backward(y, x, w, q, dx, None, sum_gradient=r)
    check_backward(x[some], y[some], w, r[some], q[some], dx[some], None, t)


def test_more_columns_than_a_launch_takes(module, dev):
    """The weight gradient of 2^26 columns and a few, 64 threads each.  A row's dot product is a
    chain of 2^26 / 1024 terms per thread, and its error's part in dx is q unit times it over the
    columns: 2^16 u of the mean magnitude, which 128 u of dx's other terms leave out."""
    t, shape = torch.float32, (3, (1 << 26) + 3)
    s, g = torch.randn(shape, device=dev), torch.randn(shape, device=dev)
    w, q = torch.ones(shape[1], device=dev), torch.rsqrt(s.square().mean(1))
    dx, dw = torch.empty_like(s), torch.zeros(shape[1], device=dev)
    module.rms_norm_backward(g, s, w, q, dx, dw)
    some = [0, 15, 16, (1 << 25) - 1, 1 << 25, (1 << 25) + 16, (1 << 26) - 1, 1 << 26, (1 << 26) + 2]
    unit = f64(s[:, some]) * f64(q)[:, None]
    terms = f64(g[:, some]) * unit
    within(dw[some], terms.sum(0), np.abs(terms).sum(0), 256, t, "weight gradient")
    inner = (s.double() * g.double()).mean(1).cpu().numpy() * f64(q)
    size = (s.double() * g.double()).abs().mean(1).cpu().numpy() * f64(q)
    ref = f64(q)[:, None] * (f64(g[:, some]) - unit * inner[:, None])
    bound = f64(q)[:, None] * (128 * U * (np.abs(f64(g[:, some])) + np.abs(unit) * size[:, None]) +
                               2.0 ** 16 * U * np.abs(unit) * size[:, None])
    assert (np.abs(f64(dx[:, some]) - ref) <= bound).all()
