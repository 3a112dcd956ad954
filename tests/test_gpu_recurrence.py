"""The gated linear recurrence and its gradients on the device against the formulas in float64.

Tolerances, with u = 2^-24.  A gate's two values carry the rounding of exp's scaled argument (|g|
log2(e) u relative to exp(-|g|), which is at most 0.54 u log2(e) of the value itself for the larger
one and |g| 1.45 u for the smaller), of exp, of the reciprocal and two products: below 24 u for the
|g| <= 10 here.  Every step of a serial or composed sum adds two roundings.  So a term that passes
through n steps has a relative error below 32 n u, and the error of h_t is below 32 u e_t with
e_t = a_t e_{t-1} + (a_t |h_{t-1}| + (1 - a_t) |u_t|) in magnitudes; likewise for l_t backwards.  A
bfloat16 result has half a unit of 2^-8 more."""

import numpy as np
import pytest
import torch

import oxide_hip as ox

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# batch, time, channels
SHAPES = [(1, 1, 1), (3, 1, 65), (64, 1, 256), (2, 2, 64), (2, 7, 130), (1, 63, 33), (3, 64, 128),
          (2, 65, 72), (1, 129, 1000), (5, 200, 31), (1, 2500, 24), (1, 4099, 96), (40, 17, 512),
          (2, 1000, 2056), (1, 20000, 8)]


def make(shape, dtype, dev, seed, scale=1.0, mean=0.0, offset=0):
    g = torch.Generator().manual_seed(seed)
    n = int(np.prod(shape))
    flat = torch.zeros(n + offset, dtype=dtype, device=dev)
    flat[offset:] = (torch.randn(n, generator=g) * scale + mean).to(dev).to(dtype)
    return flat[offset:].view(shape)


def f64(t):
    return t.detach().cpu().double().numpy()


def gates(shape, dtype, dev, seed, offset=0):
    return make(shape, dtype, dev, seed, 1.5, 2.0, offset).clamp_(-10, 10)


def lengths_of(batch, time, dev, seed=9):
    n = np.random.default_rng(seed).integers(0, time + 1, batch)
    n[0] = time
    if batch > 1:
        n[-1] = 0
    return torch.from_numpy(n.astype(np.int32)).to(dev)


def within(got, ref, magnitude, dtype, what):
    tol = 32 * U * magnitude + (2.0 ** -8 * np.abs(ref) if dtype == torch.bfloat16 else 0.0)
    bad = ~(np.abs(f64(got) - ref) <= tol + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3],
                           np.nanmax(np.abs(f64(got) - ref)))


def forward_ref(u, g, state, lengths):
    batch, time, channels = u.shape
    u6, keep, take = f64(u), 1 / (1 + np.exp(-f64(g))), 1 / (1 + np.exp(f64(g)))
    h = np.zeros((batch, channels)) if state is None else f64(state)
    e, n = np.zeros_like(h), [time] * batch if lengths is None else lengths.tolist()
    out, err = np.zeros_like(u6), np.zeros_like(u6)
    for t in range(time):
        for i in range(batch):
            if t >= n[i]:
                continue
            e[i] = keep[i, t] * (e[i] + np.abs(h[i])) + take[i, t] * np.abs(u6[i, t])
            h[i] = keep[i, t] * h[i] + take[i, t] * u6[i, t]
            out[i, t], err[i, t] = h[i], e[i]
    return out, err, h, e


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_forward(module, dev, shape, dtype, ragged):
    t = TYPES[dtype]
    u, g = make(shape, t, dev, 1), gates(shape, t, dev, 2)
    state = make((shape[0], shape[2]), torch.float32, dev, 3)
    lengths = lengths_of(shape[0], shape[1], dev) if ragged else None
    h, final = torch.empty_like(u), torch.empty_like(state)
    module.gated_recurrence_forward(u, g, h, initial_state=state, final_state=final,
                                    lengths=lengths)
    ref, err, ref_final, err_final = forward_ref(u, g, state, lengths)
    within(h, ref, err, t, "output")
    within(final, ref_final, err_final, torch.float32, "final state")


def backward_ref(dh, u, g, h, state, dfinal, lengths):
    batch, time, channels = u.shape
    keep, take = 1 / (1 + np.exp(-f64(g))), 1 / (1 + np.exp(f64(g)))
    dh6, u6, h6 = f64(dh), f64(u), f64(h)
    s6 = np.zeros((batch, channels)) if state is None else f64(state)
    back = np.zeros((batch, channels)) if dfinal is None else f64(dfinal)
    size, err = np.abs(back), np.zeros_like(back)
    n = [time] * batch if lengths is None else lengths.tolist()
    out = [np.zeros_like(u6) for _ in range(4)]
    for i in range(batch):
        for t in range(n[i] - 1, -1, -1):
            back[i] += dh6[i, t]
            size[i] += np.abs(dh6[i, t])
            err[i] += size[i]
            before = h6[i, t - 1] if t else s6[i]
            out[0][i, t] = take[i, t] * back[i]
            out[1][i, t] = take[i, t] * err[i]
            out[2][i, t] = keep[i, t] * take[i, t] * (before - u6[i, t]) * back[i]
            out[3][i, t] = keep[i, t] * take[i, t] * (np.abs(before) + np.abs(u6[i, t])) * err[i]
            back[i] *= keep[i, t]
            size[i] *= keep[i, t]
            err[i] = keep[i, t] * err[i]
    return out, back, err + size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_backward(module, dev, shape, dtype, ragged):
    t = TYPES[dtype]
    dh, u, g, h = (make(shape, t, dev, 1), make(shape, t, dev, 2), gates(shape, t, dev, 3),
                   make(shape, t, dev, 4))
    state, dfinal = (make((shape[0], shape[2]), torch.float32, dev, k) for k in (5, 6))
    lengths = lengths_of(shape[0], shape[1], dev) if ragged else None
    du, dg, ds = torch.empty_like(u), torch.empty_like(u), torch.empty_like(state)
    module.gated_recurrence_backward(dh, u, g, h, du, dg, initial_state=state,
                                     final_state_gradient=dfinal, initial_state_gradient=ds,
                                     lengths=lengths)
    (rdu, edu, rdg, edg), rds, eds = backward_ref(dh, u, g, h, state, dfinal, lengths)
    within(du, rdu, edu, t, "input gradient")
    within(dg, rdg, edg, t, "gate gradient")
    within(ds, rds, eds, torch.float32, "state gradient")


def test_without_states(module, dev):
    shape = (3, 150, 70)
    u, g = make(shape, torch.float32, dev, 1), gates(shape, torch.float32, dev, 2)
    h = torch.empty_like(u)
    module.gated_recurrence_forward(u, g, h)
    ref, err, _, _ = forward_ref(u, g, None, None)
    within(h, ref, err, torch.float32, "output")
    dh, du, dg = make(shape, torch.float32, dev, 3), torch.empty_like(u), torch.empty_like(u)
    module.gated_recurrence_backward(dh, u, g, h, du, dg)
    (rdu, edu, rdg, edg), _, _ = backward_ref(dh, u, g, h, None, None, None)
    within(du, rdu, edu, torch.float32, "input gradient")
    within(dg, rdg, edg, torch.float32, "gate gradient")


@pytest.mark.parametrize("shape", [(4, 1, 100), (2, 300, 64), (1, 5000, 40)])
def test_state_in_place(module, dev, shape):
    """The final state over the initial one, the state's gradient over the final's."""
    u, g = make(shape, torch.float32, dev, 1), gates(shape, torch.float32, dev, 2)
    state = make((shape[0], shape[2]), torch.float32, dev, 3)
    want, h2 = torch.empty_like(state), torch.empty_like(u)
    h, kept = torch.empty_like(u), state.clone()
    module.gated_recurrence_forward(u, g, h2, initial_state=state, final_state=want)
    module.gated_recurrence_forward(u, g, h, initial_state=kept, final_state=kept)
    assert torch.equal(kept, want) and torch.equal(h, h2)
    back, ds = state.clone(), torch.empty_like(state)
    a, b = torch.empty_like(u), torch.empty_like(u)
    module.gated_recurrence_backward(u, u, g, h, a, b, final_state_gradient=state,
                                     initial_state_gradient=ds)
    module.gated_recurrence_backward(u, u, g, h, a, b, final_state_gradient=back,
                                     initial_state_gradient=back)
    assert torch.equal(back, ds)


def test_token_by_token_equals_the_whole(module, dev):
    """A sequence in one call and one token at a time with the state in place."""
    shape = (3, 40, 48)
    u, g = make(shape, torch.float32, dev, 1), gates(shape, torch.float32, dev, 2)
    h, final = torch.empty_like(u), torch.empty(3, 48, device=dev)
    module.gated_recurrence_forward(u, g, h, final_state=final)
    state, one = torch.zeros(3, 48, device=dev), torch.empty(3, 1, 48, device=dev)
    _, err, _, _ = forward_ref(u, g, None, None)
    for t in range(40):
        module.gated_recurrence_forward(u[:, t:t + 1].contiguous(), g[:, t:t + 1].contiguous(),
                                        one, initial_state=state, final_state=state)
        within(one[:, 0], f64(h[:, t]), 2 * err[:, t], torch.float32, t)
    within(state, f64(final), 2 * err[:, -1], torch.float32, "final state")


@pytest.mark.parametrize("shape", [(4, 9, 50), (3, 700, 64), (2, 6000, 24)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -3.4e38])
def test_masked_places_may_hold_anything(module, dev, shape, poison):
    u, g = make(shape, torch.float32, dev, 1), gates(shape, torch.float32, dev, 2)
    state = make((shape[0], shape[2]), torch.float32, dev, 3)
    n = lengths_of(shape[0], shape[1], dev)
    dh, h = make(shape, torch.float32, dev, 4), torch.empty_like(u)
    final, outs = torch.empty_like(state), [torch.empty_like(u) for _ in range(2)]
    ds = torch.empty_like(state)
    masked = (torch.arange(shape[1], device=dev)[None] >= n[:, None])[:, :, None]

    def run(u, g, dh):
        module.gated_recurrence_forward(u, g, h, initial_state=state, final_state=final,
                                        lengths=n)
        hp = torch.where(masked, poison, h)
        module.gated_recurrence_backward(dh, u, g, hp, *outs, initial_state=state,
                                         final_state_gradient=state, initial_state_gradient=ds,
                                         lengths=n)
        return [t.clone() for t in (h, final, *outs, ds)]

    want = run(u, g, dh)
    got = run(*(torch.where(masked, poison, t) for t in (u, g, dh)))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert (want[0][-1] == 0).all() and torch.equal(want[1][-1], state[-1])
    assert torch.equal(want[4][-1], state[-1])


def test_gates_at_their_limits(module, dev):
    """A closed gate keeps the state, an open one takes the input; what is not finite stays in
    its channel and does not reach earlier steps."""
    u = make((1, 90, 64), torch.float32, dev, 1)
    state = make((1, 64), torch.float32, dev, 2)
    h = torch.empty_like(u)
    for g, want in ((float("inf"), state[:, None].expand(1, 90, 64)), (float("-inf"), u),
                    (200.0, state[:, None].expand(1, 90, 64)), (-200.0, u)):
        module.gated_recurrence_forward(u, torch.full_like(u, g), h, initial_state=state)
        assert torch.equal(h, want)
    gate = gates((1, 90, 64), torch.float32, dev, 3)
    clean = torch.empty_like(u)
    module.gated_recurrence_forward(u, gate, clean, initial_state=state)
    v = u.clone()
    v[0, 40, 5] = float("nan")
    module.gated_recurrence_forward(v, gate, h, initial_state=state)
    hit = h.isnan()
    assert hit[0, 40:, 5].all() and int(hit.sum()) == 50
    assert torch.equal(h[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_other_alignments(module, dev, dtype, offset):
    t, shape = TYPES[dtype], (2, 300, 64)
    u, g = make(shape, t, dev, 1, offset=offset), gates(shape, t, dev, 2)
    h = make(shape, t, dev, 3, offset=offset)
    state = make((2, 64), torch.float32, dev, 4, offset=offset)
    final = torch.empty(2, 64, device=dev)
    module.gated_recurrence_forward(u, g, h, initial_state=state, final_state=final)
    ref, err, ref_final, err_final = forward_ref(u, g, state, None)
    within(h, ref, err, t, "output")
    within(final, ref_final, err_final, torch.float32, "final state")
    du, dg = make(shape, t, dev, 5, offset=offset), torch.empty_like(g)
    dh = make(shape, t, dev, 6)
    module.gated_recurrence_backward(dh, u, g, h, du, dg, initial_state=state)
    (rdu, edu, rdg, edg), _, _ = backward_ref(dh, u, g, h, state, None, None)
    within(du, rdu, edu, t, "input gradient")
    within(dg, rdg, edg, t, "gate gradient")


def test_gradient_against_differences(module, dev):
    """The gradients of sum(c h) + sum(k final) along random directions against central
    differences of the kernel's own forward: step 2^-7, truncation of the order of its square and
    rounding of 64 u / step of the magnitudes; 1e-3 covers both."""
    shape, step = (2, 60, 33), 2.0 ** -7
    u, g = make(shape, torch.float32, dev, 1), gates(shape, torch.float32, dev, 2)
    state = make((2, 33), torch.float32, dev, 3)
    c, k = make(shape, torch.float32, dev, 4), make((2, 33), torch.float32, dev, 5)
    vu, vg = make(shape, torch.float32, dev, 6), make(shape, torch.float32, dev, 7)
    vs = make((2, 33), torch.float32, dev, 8)
    h, final = torch.empty_like(u), torch.empty_like(state)

    def loss(s):
        module.gated_recurrence_forward(u + s * vu, g + s * vg, h, initial_state=state + s * vs,
                                        final_state=final)
        return float((f64(h) * f64(c)).sum() + (f64(final) * f64(k)).sum())

    numeric = (loss(step) - loss(-step)) / (2 * step)
    loss(0.0)
    du, dg, ds = torch.empty_like(u), torch.empty_like(u), torch.empty_like(state)
    module.gated_recurrence_backward(c, u, g, h, du, dg, initial_state=state,
                                     final_state_gradient=k, initial_state_gradient=ds)
    parts = [f64(a) * f64(b) for a, b in ((du, vu), (dg, vg), (ds, vs))]
    assert abs(numeric - sum(p.sum() for p in parts)) <= \
        1e-3 * sum(np.abs(p).sum() for p in parts)


def test_empty(module, dev):
    """No steps leave the state; no rows or channels do nothing; lengths are clamped."""
    state, final = torch.randn(2, 8, device=dev), torch.empty(2, 8, device=dev)
    nothing = torch.empty(2, 0, 8, device=dev)
    module.gated_recurrence_forward(nothing, nothing, torch.empty_like(nothing),
                                    initial_state=state, final_state=final)
    assert torch.equal(state, final)
    module.gated_recurrence_backward(nothing, nothing, nothing, nothing,
                                     torch.empty_like(nothing), torch.empty_like(nothing),
                                     final_state_gradient=state, initial_state_gradient=final)
    assert torch.equal(state, final)
    for shape in ((0, 5, 8), (2, 5, 0)):
        z = torch.empty(shape, device=dev)
        module.gated_recurrence_forward(z, z.clone(), z.clone())
    u = torch.randn(2, 5, 8, device=dev)
    h, want = torch.empty_like(u), torch.empty_like(u)
    n = torch.tensor([-3, 1000], dtype=torch.int32, device=dev)
    module.gated_recurrence_forward(u, u.clone(), want)
    module.gated_recurrence_forward(u, u.clone(), h, lengths=n)
    assert (h[0] == 0).all() and torch.equal(h[1], want[1])


@pytest.mark.parametrize("shape", [(2, 500, 200), (1, 9000, 64)])
def test_another_stream_a_graph_and_repeats(module, dev, shape):
    u, g = make(shape, torch.bfloat16, dev, 1), gates(shape, torch.bfloat16, dev, 2)
    state = make((shape[0], shape[2]), torch.float32, dev, 3)
    h, final = torch.empty_like(u), torch.empty_like(state)
    du, dg, ds = torch.empty_like(u), torch.empty_like(u), torch.empty_like(state)
    outs = (h, final, du, dg, ds)

    def both(stream=None):
        module.gated_recurrence_forward(u, g, h, initial_state=state, final_state=final,
                                        stream=stream)
        module.gated_recurrence_backward(u, u, g, h, du, dg, initial_state=state,
                                         final_state_gradient=state, initial_state_gradient=ds,
                                         stream=stream)

    both()
    torch.cuda.synchronize()
    want = [t.clone() for t in outs]
    stream = torch.cuda.Stream()
    graph = ox.HipGraphExec.capture(stream, lambda: both(stream))
    for run in (lambda: both(stream), lambda: graph.launch(stream), lambda: graph.launch(stream)):
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_more_than_the_caches_hold(module, dev):
    """Inputs and outputs of over 256 MB, whose accesses bypass the caches: a few channels against
    the formulas."""
    t = torch.float32
    u, g = make((1, 46001, 512), t, dev, 1), gates((1, 46001, 512), t, dev, 2)
    h = torch.empty_like(u)
    module.gated_recurrence_forward(u, g, h)
    some = [0, 3, 130, 509, 511]
    pick = lambda x: x[:, :, some].contiguous()  # noqa: E731
    ref, err, _, _ = forward_ref(pick(u), pick(g), None, None)
    within(pick(h), ref, err, t, "output")
    n = 23003
    u, g, h = u[:, :n].contiguous(), g[:, :n].contiguous(), h[:, :n].contiguous()
    dh = make(u.shape, t, dev, 4)
    du, dg = torch.empty_like(u), torch.empty_like(g)
    module.gated_recurrence_backward(dh, u, g, h, du, dg)
    out, _, _ = backward_ref(pick(dh), pick(u), pick(g), pick(h), None, None, None)
    within(pick(du), out[0], out[1], t, "input gradient")
    within(pick(dg), out[2], out[3], t, "gate gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 5, 65), (3, 40, 5), (2, 300, 65), (1, 3000, 67),
                                   (2, 9, 2051), (300, 20, 7), (2, 300, 3)])
def test_ragged_channels(module, dev, shape, dtype):
    """Channels that are no multiple of an access, of one in another block among them: the state
    where it lay, and nothing written before or behind an output."""
    t, size = TYPES[dtype], int(np.prod(shape))
    u, g = make(shape, t, dev, 1), gates(shape, t, dev, 2)
    first = make((shape[0], shape[2]), torch.float32, dev, 3)
    lengths = lengths_of(shape[0], shape[1], dev)
    ref, err, ref_final, err_final = forward_ref(u, g, first, lengths)
    around = torch.full((size + 40,), 7.0, dtype=t, device=dev)
    more = torch.full((size + 40,), 7.0, dtype=t, device=dev)
    h, state = around[21:21 + size].view(shape), first.clone()
    module.gated_recurrence_forward(u, g, h, initial_state=state, final_state=state,
                                    lengths=lengths)
    within(h, ref, err, t, "output")
    within(state, ref_final, err_final, torch.float32, "state")
    dh, dfinal = make(shape, t, dev, 4), make((shape[0], shape[2]), torch.float32, dev, 5)
    h = h.clone()
    du, dg, ds = around[21:21 + size].view(shape), more[21:21 + size].view(shape), dfinal.clone()
    module.gated_recurrence_backward(dh, u, g, h, du, dg, initial_state=first,
                                     final_state_gradient=ds, initial_state_gradient=ds,
                                     lengths=lengths)
    (rdu, edu, rdg, edg), rds, eds = backward_ref(dh, u, g, h, first, dfinal, lengths)
    within(du, rdu, edu, t, "input gradient")
    within(dg, rdg, edg, t, "gate gradient")
    within(ds, rds, eds, torch.float32, "state gradient")
    for b in (around, more):
        assert (b[:21] == 7).all() and (b[21 + size:] == 7).all()


def test_offsets_past_32_bits(module, dev):
    """More than 2^31 elements: the last steps against the formulas from 40 steps before them, which
    reach no further (keep is below 0.02 there: 0.02^30 of anything is below the tolerance)."""
    t, shape, n = torch.bfloat16, (1, 4200001, 512), 40
    u = torch.randn(shape, dtype=t, device=dev)
    g = torch.randn(shape, dtype=t, device=dev).sub_(8).clamp_(-10, -4)
    h = torch.empty_like(u)
    module.gated_recurrence_forward(u, g, h)
    tail = lambda x: x[:, -n:].contiguous()  # noqa: E731
    ref, err, _, _ = forward_ref(tail(u), tail(g), None, None)
    within(tail(h)[:, 30:], ref[:, 30:], err[:, 30:], t, "output")
    du, dg = torch.empty_like(u), torch.empty_like(u)
    module.gated_recurrence_backward(u, u, g, h, du, dg)
    out, _, _ = backward_ref(tail(u), tail(u), tail(g), tail(h), None, None, None)
    within(tail(du)[:, 1:], out[0][:, 1:], out[1][:, 1:], t, "input gradient")
    within(tail(dg)[:, 1:], out[2][:, 1:], out[3][:, 1:], t, "gate gradient")


def test_workspaces_of_streams_and_graphs(module, dev):
    """Streams share no scratch memory, and a captured call keeps its own when the stream's next
    ones need more."""
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    ws = ox.StreamWorkspaces()
    a, b = (ws.ptr_bytes(1000, s.cuda_stream)[0] for s in (one, two))
    c, size = ws.ptr_bytes(1001, one.cuda_stream)
    assert len({a, b, c}) == 3 and size >= 2000
    assert ws.ptr_bytes(10, one.cuda_stream) == (c, size)
    assert ws.ptr_bytes(0, one.cuda_stream) == (None, 0)

    t, shape = torch.float32, (1, 3000, 24)
    u, g = make(shape, t, dev, 1), gates(shape, t, dev, 2)
    want, h = torch.empty_like(u), torch.empty_like(u)
    own = ox.load_kernels(0)
    own.gated_recurrence_forward(u, g, want)
    run = lambda: own.gated_recurrence_forward(u, g, h, stream=one)  # noqa: E731
    torch.cuda.synchronize()
    run()
    graph = ox.HipGraphExec.capture(one, run)
    large = make((1, 60000, 96), t, dev, 3)
    out = torch.empty_like(large)
    torch.cuda.synchronize()
    for _ in range(3):
        own.gated_recurrence_forward(large, large, out, stream=one)
        fill = torch.full((1 << 20,), 3.0, device=dev)  # takes memory that was given back
        torch.cuda.synchronize()
        h.zero_()
        torch.cuda.synchronize()
        graph.launch(one)
        torch.cuda.synchronize()
        assert torch.equal(h, want) and (fill == 3).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(4, 9, 50), (3, 700, 64), (2, 6000, 24), (300, 3, 5)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_steps_beside_a_final_gradient_that_is_not_finite(module, dev, shape, dtype, bad):
    """Steps at or past a row's length take gradients of 0 whatever reaches the row's last step."""
    t = TYPES[dtype]
    u, g = make(shape, t, dev, 1), gates(shape, t, dev, 2)
    n = lengths_of(shape[0], shape[1], dev)
    du, dg = torch.ones_like(u), torch.ones_like(u)
    ds, final = torch.empty(shape[0], shape[2], device=dev), torch.zeros(shape[0], shape[2],
                                                                         device=dev)
    final[:, 1::2] = bad
    module.gated_recurrence_backward(u, u, g, u, du, dg, final_state_gradient=final,
                                     initial_state_gradient=ds, lengths=n)
    masked = (torch.arange(shape[1], device=dev)[None] >= n[:, None])[:, :, None].expand(shape)
    assert (du[masked] == 0).all() and (dg[masked] == 0).all()
    assert torch.equal(ds[-1].nan_to_num(7.0), final[-1].nan_to_num(7.0))  # a row of no steps
    assert du[:, :, ::2].isfinite().all() and dg[:, :, ::2].isfinite().all()
    assert not du[0, -1, 1::2].isfinite().any()  # the first row is whole


@pytest.mark.parametrize("time", [1, 100])
@pytest.mark.parametrize("closed", [True, False])
def test_small_gate_values(module, dev, time, closed):
    """What a nearly closed gate takes and a nearly open one keeps, in a single step between steps
    that add nothing and keep all, up to the smallest normal numbers.  exp2's argument g log2(e)
    carries the constant's rounding (0.22 u) and its own (u), |g| times as much in the result; exp2
    and the reciprocal are within a unit in the last place (2 u each), 1 + e and the product within
    u: (8 + 1.25 |g|) u with what is of second order."""
    g = torch.linspace(0, 86.5, 20001, device=dev) * (1.0 if closed else -1.0)
    gate = torch.full((1, time, g.numel()), 200.0, device=dev)
    u, at = torch.zeros_like(gate), time // 2
    gate[0, at] = g
    u[0, at] = 1.0 if closed else 0.0
    state = torch.full((1, g.numel()), 0.0 if closed else 1.0, device=dev)
    h, final = torch.empty_like(u), torch.empty_like(state)
    module.gated_recurrence_forward(u, gate, h, initial_state=state, final_state=final)
    small, bound = 1 / (1 + np.exp(np.abs(f64(g)))), (8 + 1.25 * np.abs(f64(g))) * U
    for got in (h[0, at], final[0]):
        assert (np.abs(f64(got) / small - 1) <= bound).all()
    # gate gradient: keep take (h_{t-1} - u_t) l, of l = 1 here: the larger value's 4 u and three
    # products more
    dh, du, dg = torch.zeros_like(u), torch.empty_like(u), torch.empty_like(u)
    dh[0, at] = 1.0
    module.gated_recurrence_backward(dh, u, gate, h, du, dg, initial_state=state)
    large = 1 / (1 + np.exp(-np.abs(f64(g))))
    want = small * large * (-1.0 if closed else 1.0)
    assert (np.abs(f64(dg[0, at]) / want - 1) <= bound + 8 * U).all()
    take = small if closed else large
    assert (np.abs(f64(du[0, at]) / take - 1) <= (bound if closed else 4 * U) + U).all()


@pytest.mark.parametrize("time", [1, 100])
def test_gates_that_are_not_finite(module, dev, time):
    """A NaN gate gives NaN; infinite ones keep or take exactly, also of large values."""
    u = make((1, time, 8), torch.float32, dev, 1)
    u[0, -1, 5] = 3e38
    gate, state = gates((1, time, 8), torch.float32, dev, 2), make((1, 8), torch.float32, dev, 3)
    state[0, 6] = 3e38
    gate[0, -1, 0], gate[0, -1, 1] = float("nan"), -float("nan")
    gate[0, -1, 2:5:2] = float("inf")
    gate[0, -1, 3] = gate[0, -1, 6] = float("-inf")
    gate[0, -1, 5] = float("inf")
    h = torch.empty_like(u)
    module.gated_recurrence_forward(u, gate, h, initial_state=state)
    assert h[0, -1, :2].isnan().all()
    before = state if time == 1 else h[:, -2]
    assert torch.equal(h[0, -1, [2, 4, 5]], before[0, [2, 4, 5]])
    assert torch.equal(h[0, -1, [3, 6]], u[0, -1, [3, 6]])
