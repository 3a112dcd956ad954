"""The gated delta rule and its gradients on the device against its steps in float64.

Tolerances.  Columns of values never meet, and for keys of length at most 1 a step's map of a
column of the state, a (1 - b k k'), shortens every vector: an error made at a step never grows.  So
with M_t the running sum of the lengths of what the steps add to a column (decayed as the state is),
the state is within c of M, an output within c scale |q| M, where c counts the roundings between the
operands and it.  The state's gradient shrinks the same way backwards, D_t its running sum; dv is
within c b |k| D, dq, dk and both gates' gradients within c of the sums over the columns of the
products of D, M and the errors' sizes that they are made of.

float32: sums of at most 128 + 64 + 64 products, whose order's worst case is their count; exponentials
of at most 2 roundings: c = 512 u, u = 2^-24, for the gradients, which chain two of them, twice that.
bfloat16 operands: an output passes the state, the chunk's matrix and its own rounding, 2^-8 each,
and the system's 2^-17: c = 4 of 2^-8; a gradient the states, both matrices, the errors and its own:
c = 8.  The state's own path has 2^-17 roundings of four operands, a rounding of q k' none: c = 16
of 2^-17.  Steps one by one are float32."""

import numpy as np
import pytest
import torch

import oxide_hip as ox
from test_gpu_rms_norm import TYPES, f64, make

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
# batch, time, key heads, heads, key_dim, value_dim: single values, single tokens, the last steps
# taken one by one and the first by chunks, whole chunks and one step more or less, odd widths,
# shared heads, every count of 32 keys
SHAPES = [(1, 1, 1, 1, 1, 1), (3, 1, 2, 4, 32, 32), (1, 5, 1, 3, 17, 33), (2, 16, 2, 2, 64, 64),
          (2, 17, 1, 2, 33, 15), (2, 63, 2, 2, 32, 16), (1, 64, 1, 1, 64, 48),
          (2, 65, 1, 3, 96, 40), (1, 128, 2, 2, 100, 130), (3, 130, 2, 4, 128, 128),
          (2, 200, 1, 1, 128, 7), (5, 28, 4, 4, 32, 32)]


def unit(shape, t, dev, seed):
    v = make(shape, F32, dev, seed)
    return (v / v.norm(dim=-1, keepdim=True) * 0.99).to(t)  # rounded: not above 1


def operands(shape, t, dev, seed=1):
    batch, time, key_heads, heads, keys, values = shape
    return [unit((batch, time, key_heads, keys), t, dev, seed),
            unit((batch, time, key_heads, keys), t, dev, seed + 1),
            make((batch, time, heads, values), t, dev, seed + 2),
            make((batch, time, heads), t, dev, seed + 3) * 1.5 + 2,
            make((batch, time, heads), t, dev, seed + 4)]


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


class Reference:
    """The steps in float64, and the running sums that errors are held to."""

    def __init__(self, q, k, v, gate, write, state=None, lengths=None, scale=None):
        self.group = v.shape[2] // k.shape[2]
        wide = lambda x: np.repeat(f64(x), self.group, 2)  # noqa: E731
        self.q, self.k, self.v = wide(q), wide(k), f64(v)
        self.gate, self.write = f64(gate), f64(write)
        self.a, self.b = sigmoid(self.gate), sigmoid(self.write)
        # 1 - a and 1 - b from their own exponentials: a gate of 80 leaves 1.8e-35, not 0
        self.less_a, self.less_b = sigmoid(-self.gate), sigmoid(-self.write)
        batch, time, heads, keys = self.k.shape
        self.scale = keys ** -0.5 if scale is None else scale
        self.n = [time] * batch if lengths is None else [min(max(int(i), 0), time) for i in lengths]
        s = np.zeros((batch, heads, keys, self.v.shape[3])) if state is None else f64(state)
        m = np.linalg.norm(s, axis=2)
        self.states, self.sizes, self.out = [s], [m], np.zeros_like(self.v)
        self.near = np.zeros_like(self.v)
        for t in range(time):
            on = self.on(t)
            shrunk, wrong, size = self.step(t, s)
            extra = self.b[:, t, :, None] * self.length(self.k, t) * size
            new = shrunk + (self.b[:, t, :, None] * self.k[:, t])[..., None] * wrong[:, :, None]
            s = np.where(on[..., None], new, s)
            m = np.where(on, self.a[:, t, :, None] * m + extra, m)
            self.out[:, t] = np.where(on, self.scale * self.dot(self.q[:, t], s), 0.0)
            self.near[:, t] = np.where(on, abs(self.scale) * self.length(self.q, t) * m, 0.0)
            self.states.append(s)
            self.sizes.append(m)

    def on(self, t):
        return np.array([t < n for n in self.n])[:, None, None]

    @staticmethod
    def dot(x, s):
        return np.einsum("bhk,bhkv->bhv", x, s)

    @staticmethod
    def length(x, t):
        return np.linalg.norm(x[:, t], axis=-1)[..., None]

    def step(self, t, s):
        shrunk = self.a[:, t, :, None, None] * s
        seen = self.dot(self.k[:, t], shrunk)
        # a sum through a key is rounded by the lengths of the key and of the state's column
        size = np.abs(self.v[:, t]) + self.length(self.k, t) * np.linalg.norm(shrunk, axis=2)
        return shrunk, self.v[:, t] - seen, size

    def gradients(self, g, final=None):
        """(name: (gradient, what its error is held to))."""
        g = f64(g)
        batch, time, heads, keys = self.k.shape
        ds = np.zeros_like(self.states[0]) if final is None else f64(final)
        big = np.linalg.norm(ds, axis=2)
        got = {x: [np.zeros(y.shape), np.zeros(y.shape)] for x, y in (
            ("query", self.q), ("key", self.k), ("value", self.v), ("gate", self.a),
            ("write", self.b))}
        for t in reversed(range(time)):
            on = self.on(t)
            old, new, m = self.states[t], self.states[t + 1], self.sizes[t + 1]
            shrunk, wrong, size = self.step(t, old)
            gt, kt, b = g[:, t] * self.scale, self.k[:, t], self.b[:, t, :, None]
            klen, qlen = self.length(self.k, t), self.length(self.q, t)

            def put(name, value, near, live=on[..., 0]):
                live = live if value.ndim == 2 else live[..., None]
                got[name][0][:, t] = np.where(live, value, 0.0)
                got[name][1][:, t] = np.where(live, near, 0.0)

            put("query", np.einsum("bhkv,bhv->bhk", new, gt), (np.abs(gt) * m).sum(-1)[..., None])
            full = ds + self.q[:, t][..., None] * gt[:, :, None]
            wide = big + qlen * np.abs(gt)
            into = self.dot(kt, full)
            slope = self.b[:, t] * self.less_b[:, t]
            put("write", (into * wrong).sum(-1) * slope, (klen * wide * size).sum(-1) * slope)
            put("value", b * into, b * klen * wide)
            put("key", np.einsum("bhkv,bhv->bhk", full, b * wrong)
                - np.einsum("bhkv,bhv->bhk", shrunk, b * into),
                (b * wide * size + b * klen * wide * m).sum(-1)[..., None])
            back = full - kt[..., None] * (b * into)[:, :, None]
            a, less = self.a[:, t], self.less_a[:, t]
            put("gate", (back * old).sum((2, 3)) * a * less,
                (wide * (self.sizes[t] + m)).sum(-1) * less)
            ds = np.where(on[..., None], a[..., None, None] * back, ds)
            big = np.where(on, a[..., None] * wide, big)
        for name in ("query", "key"):
            got[name] = [x.reshape(batch, time, -1, self.group, keys).sum(3) for x in got[name]]
        return got, ds, big


def held(got, ref, near, units, t, what):
    tol = units * near + (2.0 ** -8 if t == BF16 else U) * np.abs(ref) + 1e-37
    bad = ~(np.abs(f64(got) - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3], np.abs(f64(got) - ref).max(),
                           (np.abs(f64(got) - ref) / tol).max())


def units_of(t, chunks):
    """(of an output, of the state)."""
    if t == F32 or not chunks:
        return 512 * U, 512 * U
    return 4 * 2.0 ** -8, 16 * 2.0 ** -17


def check_forward(ops, out, state, t, chunks, first=None, lengths=None, scale=None):
    ref = Reference(*ops, first, lengths, scale)
    of_out, of_state = units_of(t, chunks)
    held(out, ref.out, ref.near, of_out, t, "output")
    if state is not None:
        held(state, ref.states[-1], ref.sizes[-1][:, :, None], of_state, F32, "state")
    return ref


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("states", [True, False])
@pytest.mark.parametrize("saves", [True, False])
def test_forward(module, dev, shape, dtype, states, saves):
    t = TYPES[dtype]
    batch, time, _, heads, keys, values = shape
    ops = operands(shape, t, dev)
    first = make((batch, heads, keys, values), F32, dev, 9) * 0.3 if states else None
    final = torch.empty(batch, heads, keys, values, device=dev) if states else None
    out = torch.full_like(ops[2], 7.0)
    saved = module.gated_delta_rule_saved(ops[1], ops[2]) if saves else None
    module.gated_delta_rule_forward(*ops, out, initial_state=first, final_state=final, saved=saved)
    check_forward(ops, out, final, t, saves or time > 16, first)


def backward(module, ops, g, saved, **k):
    outs = [torch.full_like(x, 7.0) for x in ops]
    module.gated_delta_rule_backward(g, *ops, saved, *outs, **k)
    return outs


def check_gradients(ref, g, outs, t, final=None, back=None):
    got, ds, big = ref.gradients(g, final)
    units = 1024 * U if t == F32 else 8 * 2.0 ** -8
    for name, x in zip(("query", "key", "value", "gate", "write"), outs):
        held(x, *got[name], units, t, name + " gradient")
    if back is not None:
        held(back, ds, big[:, :, None], units, F32, "state gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("states", [True, False])
def test_backward(module, dev, shape, dtype, states):
    t = TYPES[dtype]
    batch, time, _, heads, keys, values = shape
    ops, g = operands(shape, t, dev), make((batch, time, heads, values), t, dev, 21)
    state = (batch, heads, keys, values)
    first = make(state, F32, dev, 9) * 0.3 if states else None
    dfinal = make(state, F32, dev, 22) if states else None
    back = torch.empty(state, device=dev) if states else None
    out, saved = torch.empty_like(ops[2]), module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, initial_state=first, saved=saved)
    outs = backward(module, ops, g, saved, final_state_gradient=dfinal, initial_state_gradient=back)
    check_gradients(Reference(*ops, first), g, outs, t, dfinal, back)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(6, 10, 1, 2, 20, 18), (6, 150, 2, 2, 64, 33)])
def test_lengths(module, dev, shape, dtype):
    """Rows of every kind of length, empty ones among them; what lies behind a row's end is never
    read, its outputs and gradients are 0, nothing around an output is written, and the state of the
    row is that at its end, in place."""
    t = TYPES[dtype]
    batch, time, _, heads, keys, values = shape
    lengths = [time, 0, 1, time // 2, -3, time + 9]
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    ops, g = operands(shape, t, dev), make((batch, time, heads, values), t, dev, 21)
    state = (batch, heads, keys, values)
    first, dfinal = make(state, F32, dev, 9) * 0.3, make(state, F32, dev, 22)
    ref = Reference(*ops, first, lengths)
    poisoned = [x.clone() for x in (*ops, g)]
    for x in poisoned:
        for b, end in enumerate(ref.n):
            x[b, end:] = float("nan")
    *ops, g = poisoned
    around = torch.full((ops[2].numel() + 48,), 7.0, dtype=t, device=dev)
    out = around[24:-24].view(ops[2].shape)
    for saves in (False, True):
        final = first.clone()
        saved = module.gated_delta_rule_saved(ops[1], ops[2]) if saves else None
        out.fill_(5.0)
        module.gated_delta_rule_forward(*ops, out, initial_state=final, final_state=final,
                                        saved=saved, lengths=n)
        of_out, of_state = units_of(t, saves or time > 16)
        held(out, ref.out, ref.near, of_out, t, "output")
        held(final, ref.states[-1], ref.sizes[-1][:, :, None], of_state, F32, "state")
    assert (around[:24] == 7).all() and (around[-24:] == 7).all()
    rooms = [torch.full((x.numel() + 48,), 7.0, dtype=t, device=dev) for x in ops]
    outs = [r[24:-24].view(x.shape) for r, x in zip(rooms, ops)]
    back = dfinal.clone()
    module.gated_delta_rule_backward(g, *ops, saved, *outs, final_state_gradient=back,
                                     initial_state_gradient=back, lengths=n)
    got, ds, big = ref.gradients(torch.nan_to_num(g), dfinal)
    units = 1024 * U if t == F32 else 8 * 2.0 ** -8
    for name, x in zip(("query", "key", "value", "gate", "write"), outs):
        held(x, *got[name], units, t, name + " gradient")
    held(back, ds, big[:, :, None], units, F32, "state gradient")
    for r in rooms:
        assert (r[:24] == 7).all() and (r[-24:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_token_by_token(module, dev, dtype):
    """A prompt by chunks, its end by single tokens and by a few at once: the one sequence."""
    t, shape = TYPES[dtype], (2, 90, 2, 4, 64, 40)
    ops = operands(shape, t, dev)
    out, state = torch.empty_like(ops[2]), torch.empty(2, 4, 64, 40, device=dev)
    ref = Reference(*ops)
    done = 0
    for count in (70, 1, 1, 7, 11):
        part = [x[:, done:done + count].contiguous() for x in ops]
        o = torch.empty_like(part[2])
        module.gated_delta_rule_forward(*part, o, initial_state=state if done else None,
                                        final_state=state)
        out[:, done:done + count] = o
        done += count
    of_out, of_state = units_of(t, True)
    held(out, ref.out, ref.near, of_out, t, "output")
    held(state, ref.states[-1], ref.sizes[-1][:, :, None], of_state, F32, "state")


@pytest.mark.parametrize("time", [9, 70])
def test_gates_at_their_ends(module, dev, time):
    """Gates that keep all or nothing and writes of all or nothing, for a step or for all of them;
    keys of 0."""
    shape = (2, time, 1, 2, 32, 24)
    inf = float("inf")
    for gate, write in ((inf, None), (-inf, None), (-300.0, None), (80.0, None), (None, -inf),
                        (None, inf), (None, -200.0), ("some", "some")):
        ops = operands(shape, F32, dev, 31)
        if gate == "some":
            ops[3][:, ::5], ops[3][:, 2::7] = -inf, inf
            ops[4][:, 1::3], ops[4][:, 4::6] = -inf, inf
            ops[1][:, 3::4] = 0.0
        else:
            if gate is not None:
                ops[3].fill_(gate)
            if write is not None:
                ops[4].fill_(write)
        first = make((2, 2, 32, 24), F32, dev, 9)
        out, final = torch.empty_like(ops[2]), torch.empty_like(first)
        saved = module.gated_delta_rule_saved(ops[1], ops[2])
        for s in (None, saved):
            module.gated_delta_rule_forward(*ops, out, initial_state=first, final_state=final,
                                            saved=s)
            ref = check_forward(ops, out, final, F32, True, first)
        g = make(ops[2].shape, F32, dev, 21)
        check_gradients(ref, g, backward(module, ops, g, saved), F32)


def test_many_resets_in_a_chunk(module, dev):
    """Decays of e^-60 over and over: sums of hundreds whose differences still count."""
    ops = operands((1, 128, 1, 1, 32, 32), F32, dev, 41)
    ops[3][:, ::3] = -60.0
    out, saved = torch.empty_like(ops[2]), module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, saved=saved)
    ref = check_forward(ops, out, None, F32, True)
    g = make(ops[2].shape, F32, dev, 21)
    check_gradients(ref, g, backward(module, ops, g, saved), F32)


def test_scale_and_repeated_keys(module, dev):
    """One key over and over, written whole each time: the state holds the last value for it."""
    shape = (1, 100, 1, 1, 64, 32)
    ops = operands(shape, F32, dev, 51)
    ops[1][:] = ops[1][:, :1].clone() / ops[1][:, :1].norm()
    ops[0][:] = ops[1]
    ops[3].fill_(40.0)
    ops[4].fill_(40.0)
    out = torch.empty_like(ops[2])
    module.gated_delta_rule_forward(*ops, out, scale=-2.0)
    check_forward(ops, out, None, F32, True, scale=-2.0)
    assert torch.allclose(out, -2.0 * ops[2], atol=1e-3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 3, 8])
def test_other_alignments(module, dev, dtype, offset):
    t, shape = TYPES[dtype], (2, 70, 2, 2, 64, 32)
    ops = [make(x.shape, t, dev, 60, offset).copy_(x) for x in operands(shape, t, dev, 61)]
    first = make((2, 2, 64, 32), F32, dev, 9, offset)
    out, final = make(ops[2].shape, t, dev, 1, offset), make(first.shape, F32, dev, 2, offset)
    saved = module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, initial_state=first, final_state=final, saved=saved)
    ref = check_forward(ops, out, final, t, True, first)
    g = make(ops[2].shape, t, dev, 21, offset)
    outs = [make(x.shape, t, dev, 3, offset) for x in ops]
    module.gated_delta_rule_backward(g, *ops, saved, *outs)
    check_gradients(ref, g, outs, t)
    few = [x[:, :4].contiguous() for x in ops]
    few = [make(x.shape, t, dev, 60, offset).copy_(x) for x in few]
    out = make(few[2].shape, t, dev, 1, offset)
    module.gated_delta_rule_forward(*few, out, initial_state=first, final_state=final)
    check_forward(few, out, final, t, False, first)


def test_gradients_against_differences(module, dev):
    """Central differences of sum(c . o) + sum(d . S) along random directions of each operand and of
    the state; h = 2^-7: truncation below h^2 of the slopes' scale, rounding below 1e-4 of it."""
    shape, h = (2, 70, 1, 2, 24, 20), 2.0 ** -7
    ops = operands(shape, F32, dev, 71)
    first = make((2, 2, 24, 20), F32, dev, 9) * 0.3
    c, d = make(ops[2].shape, F32, dev, 72), make(first.shape, F32, dev, 73)
    ways = [make(x.shape, F32, dev, 80 + i) * (0.1 if i < 2 else 1.0)
            for i, x in enumerate((*ops, first))]

    def value(which, step):
        at = [x + step * v if i == which else x for i, (x, v) in enumerate(zip((*ops, first), ways))]
        out, final = torch.empty_like(ops[2]), torch.empty_like(first)
        module.gated_delta_rule_forward(*at[:5], out, initial_state=at[5], final_state=final)
        return float((out.double() * c.double()).sum() + (final.double() * d.double()).sum())

    out, saved = torch.empty_like(ops[2]), module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, initial_state=first, saved=saved)
    back = torch.empty_like(first)
    outs = backward(module, ops, c, saved, final_state_gradient=d, initial_state_gradient=back)
    slopes = [float((g.double() * v.double()).sum()) for g, v in zip((*outs, back), ways)]
    for i, slope in enumerate(slopes):
        diff = (value(i, h) - value(i, -h)) / (2 * h)
        assert abs(diff - slope) <= 2e-3 * max(abs(s) for s in slopes), (i, diff, slope)


def test_empty(module, dev):
    for batch, time in ((0, 5), (2, 0)):
        ops = operands((batch, time, 1, 2, 8, 8), F32, dev)
        first, final = torch.ones(batch, 2, 8, 8, device=dev), torch.zeros(batch, 2, 8, 8, device=dev)
        saved = module.gated_delta_rule_saved(ops[1], ops[2])
        for s in (None, saved):
            module.gated_delta_rule_forward(*ops, torch.empty_like(ops[2]), initial_state=first,
                                            final_state=final, saved=s)
        assert torch.equal(final, first)
        back = torch.zeros_like(first)
        backward(module, ops, ops[2], saved, final_state_gradient=first,
                 initial_state_gradient=back)
        assert torch.equal(back, first)
        backward(module, ops, ops[2], saved, initial_state_gradient=back)
        assert (back == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_more_chunks_than_are_prepared_at_once(module, dev, dtype):
    """A sequence whose operands exceed the workspace: in parts, the state handed on."""
    t, shape = TYPES[dtype], (1, 10000, 16, 16, 128, 8)
    ops, g = operands(shape, t, dev, 91), make((1, 10000, 16, 8), t, dev, 92)
    first = make((1, 16, 128, 8), F32, dev, 9)
    out, final = torch.empty_like(ops[2]), torch.empty_like(first)
    saved = module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, initial_state=first, final_state=final, saved=saved)
    ref = check_forward(ops, out, final, t, True, first)
    dfinal, back = make(first.shape, F32, dev, 10), torch.empty_like(first)
    outs = backward(module, ops, g, saved, final_state_gradient=dfinal, initial_state_gradient=back)
    check_gradients(ref, g, outs, t, dfinal, back)


def test_offsets_past_32_bits(module, dev):
    """More than 2^31 values: the last steps against the formulas from 40 steps before them (a gate
    below -4 keeps less than 0.02 of the state each step)."""
    shape, n = (1, 4200001, 1, 1, 16, 512), 40
    make_one = lambda *s: torch.randn(*s, dtype=BF16, device=dev)  # noqa: E731
    k, q = (torch.nn.functional.normalize(make_one(1, shape[1], 1, 16), dim=-1) for _ in range(2))
    v = make_one(1, shape[1], 1, 512)
    gate, write = make_one(1, shape[1], 1).sub_(8).clamp_(-10, -4), make_one(1, shape[1], 1)
    out = torch.empty_like(v)
    module.gated_delta_rule_forward(q, k, v, gate, write, out)
    tail = [x[:, -n:].contiguous() for x in (q, k, v, gate, write, out)]
    ref = Reference(*tail[:5])
    late = slice(30, None)
    held(tail[5][:, late], ref.out[:, late], ref.near[:, late], 4 * 2.0 ** -8, BF16, "output")


def test_streams_graphs_and_repeats(module, dev):
    """The same bits every time: on a stream of the caller's, from two graphs that share nothing,
    replayed beside an eager call."""
    shape = (3, 200, 2, 4, 64, 48)
    ops, g = operands(shape, BF16, dev, 95), make((3, 200, 4, 48), BF16, dev, 96)

    def buffers():
        return (torch.empty_like(ops[2]), torch.empty(3, 4, 64, 48, device=dev),
                module.gated_delta_rule_saved(ops[1], ops[2]), *[torch.empty_like(x) for x in ops])

    def run(b, stream=None):
        out, final, saved, *grads = b
        module.gated_delta_rule_forward(*ops, out, final_state=final, saved=saved, stream=stream)
        module.gated_delta_rule_backward(g, *ops, saved, *grads, stream=stream)

    want, rooms = buffers(), (buffers(), buffers())
    run(want)
    torch.cuda.synchronize()
    results = lambda b: (b[0], b[1], *b[3:])  # noqa: E731
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = [ox.HipGraphExec.capture(st, lambda b=b, st=st: run(b, st))
              for b, st in zip(rooms, streams)]
    for _ in range(3):
        for b in rooms:
            for x in results(b):
                x.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            graph.launch(st)
        eager = buffers()
        run(eager)
        torch.cuda.synchronize()
        for b in (*rooms, eager):
            assert all(torch.equal(x, y) for x, y in zip(results(b), results(want)))


def test_wrong_tensors(module, dev):
    q, k, v, gate, write = operands((2, 5, 2, 4, 8, 6), F32, dev)
    out = torch.empty_like(v)
    call = module.gated_delta_rule_forward
    for bad in ((q[:, :4], k, v, gate, write, out), (q, k, v, gate, write[..., :2], out),
                (q, k, v.bfloat16(), gate, write, out), (q, k, v, gate, write, out[:, :, :2]),
                (q.transpose(2, 3), k.transpose(2, 3), v, gate, write, out),
                (q[0], k[0], v, gate, write, out)):
        with pytest.raises(ox.OxideError):
            call(*bad)
    for rest in (dict(initial_state=out), dict(lengths=torch.zeros(2, device=dev)),
                 dict(saved=torch.empty(8, dtype=torch.uint8, device=dev)),
                 dict(scale=float("nan"))):
        with pytest.raises(ox.OxideError):
            call(q, k, v, gate, write, out, **rest)


def shifted(x):
    """The same values one element behind an aligned place."""
    room = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    room[1:] = x.flatten()
    return room[1:].view(x.shape)


# enough heads for blocks of 32 columns, whose rows are staged: rows of whole 16 bytes, odd ones,
# every count of 32 keys, odd counts of 16 columns, shared heads, one chunk and several
MANY = [(32, 66, 2, 4, 128, 40), (43, 130, 1, 6, 17, 7), (86, 65, 1, 3, 96, 24),
        (32, 129, 4, 4, 64, 33), (256, 20, 1, 1, 32, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", MANY)
@pytest.mark.parametrize("aligned", [True, False])
def test_many_heads(module, dev, shape, dtype, aligned):
    t = TYPES[dtype]
    batch, time, _, heads, keys, values = shape
    place = (lambda x: x) if aligned else shifted
    ops = [place(x) for x in operands(shape, t, dev)]
    g = place(make((batch, time, heads, values), t, dev, 21))
    lengths = [time - 7 * (b % 3) if b % 5 else (b * 37) % (time + 1) for b in range(batch)]
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    for x in (*ops, g):
        for b, end in enumerate(lengths):
            x[b, end:] = float("nan")
    state = (batch, heads, keys, values)
    first, dfinal = make(state, F32, dev, 9) * 0.3, make(state, F32, dev, 22)
    out, final, back = place(torch.empty_like(ops[2])), torch.empty_like(first), torch.empty_like(first)
    saved = module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, initial_state=first, final_state=final, saved=saved,
                                    lengths=n)
    clean = [torch.nan_to_num(x) for x in ops]
    ref = check_forward(clean, out, final, t, True, first, lengths)
    # without the state's exact way, and without what the backward reads
    out.fill_(3.0)
    module.gated_delta_rule_forward(*ops, out, initial_state=first, lengths=n)
    held(out, ref.out, ref.near, units_of(t, True)[0], t, "output alone")
    module.gated_delta_rule_forward(*ops, out, initial_state=first, saved=saved, lengths=n)
    outs = [place(torch.full_like(x, 7.0)) for x in ops]
    module.gated_delta_rule_backward(g, *ops, saved, *outs, final_state_gradient=dfinal,
                                     initial_state_gradient=back, lengths=n)
    check_gradients(ref, torch.nan_to_num(g), outs, t, dfinal, back)


@pytest.mark.parametrize("time", [17, 48, 49])
def test_steps_of_many_heads(module, dev, time):
    """float32 heads enough to be taken one by one further, and the first count of steps that is not."""
    shape = (128, time, 8, 16, 32, 24)
    ops = operands(shape, F32, dev, 61)
    first = make((128, 16, 32, 24), F32, dev, 9) * 0.3
    out, final = torch.empty_like(ops[2]), torch.empty_like(first)
    module.gated_delta_rule_forward(*ops, out, initial_state=first, final_state=final)
    check_forward(ops, out, final, F32, True, first)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_heads_in_parts(module, dev, dtype):
    """More chunks of many heads than are prepared at once: to the bit what two calls give that hand
    each other the state and its gradient."""
    t, shape = TYPES[dtype], (64, 1024, 8, 16, 8, 8)
    ops, g = operands(shape, t, dev, 71), make((64, 1024, 16, 8), t, dev, 72)
    state = torch.empty(64, 16, 8, 8, device=dev)
    whole, parts, back = (torch.empty_like(state) for _ in range(3))
    dfinal = make(state.shape, F32, dev, 73)
    out, saved = torch.empty_like(ops[2]), module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, final_state=whole, saved=saved)
    outs = backward(module, ops, g, saved, final_state_gradient=dfinal, initial_state_gradient=back)
    halves = [[x[:, i:i + 512].contiguous() for x in (*ops, g)] for i in (0, 512)]
    kept = []
    for i, (*half, _) in enumerate(halves):
        o = torch.empty_like(half[2])
        kept.append(module.gated_delta_rule_saved(half[1], half[2]))
        module.gated_delta_rule_forward(*half, o, initial_state=parts if i else None,
                                        final_state=parts, saved=kept[i])
        assert torch.equal(o, out[:, 512 * i:512 * i + 512])
    assert torch.equal(parts, whole)
    into = dfinal.clone()
    for i in (1, 0):
        *half, gradient = halves[i]
        got = backward(module, half, gradient, kept[i], final_state_gradient=into,
                       initial_state_gradient=into)
        for name, a, b in zip(("query", "key", "value", "gate", "write"), got, outs):
            assert torch.equal(a, b[:, 512 * i:512 * i + 512]), name
    assert torch.equal(into, back)
