"""Sequence layers in traced graphs: every gradient of small graphs against torch float64 autograd
of the same graph, the optimizer's step against the definition, replays against the eager run, and
the row classifier trained.

Tolerance of a gradient: at most 16 operations lie between it and the loss, each within 256 * 2^-24
of its terms' magnitudes (the operators' own tests), so 2.5e-4 of the gradient's Frobenius norm; the
terms here do not cancel by more than the factor 2 left to reach 5e-4."""

import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import jit
import nn
import oxide_hip as ox
import sequence
import tensor as tn
import training
from test_data_checkpoint import _idx_images, _idx_labels
from test_gpu_muon import orthogonal

pytestmark = pytest.mark.gpu


def close(got, ref, what=""):
    ref = ref.detach().numpy() if hasattr(ref, "detach") else ref
    off = np.linalg.norm(got.astype(np.float64) - ref)
    assert off <= 5e-4 * np.linalg.norm(ref) + 1e-9, (what, off, np.linalg.norm(ref))


def leaf(a):
    return torch.tensor(np.asarray(a, np.float64), requires_grad=True)


def norm64(x, w, eps=1e-6):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def recurrence64(x, gate):
    a, h, out = torch.sigmoid(gate), torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        out.append(h)
    return torch.stack(out, 1)


def randn(*shape, seed):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def kinds(program):
    return [op.kind for op in program.ops]


def run_checked(program):
    """Group by group, as an inspecting caller runs it."""
    for op in program.ops:
        op.launch()
    program.check()


def test_residual_norms_and_recurrence():
    """s1 = a + b, y1 = norm(s1) (one launch), r = recurrence(y1, g), s2 = s1 + r, y2 = norm(s2)
    (one launch), both norms of one weight, s1 used twice."""
    B, T, D = 3, 9, 20
    av, bv, gv, tv = (randn(B, T, D, seed=i) for i in range(4))
    wv = 1 + 0.1 * randn(D, seed=5)
    targets = np.arange(B, dtype=np.float32) * 7
    a, b, g = (tn.input((B, T, D), requires_grad=True) for _ in range(3))
    w, t = nn.Parameter(wv), tn.input((B,))
    s1 = a.add(b)
    y1 = s1.rms_norm(w.tensor())
    s2 = s1.add(y1.gated_recurrence(g))
    y2 = s2.rms_norm(w.tensor())
    loss = y2.mul(tn.constant(tv)).reshape((B, T * D)).cross_entropy(t)
    program = tn.training_program(loss)
    assert kinds(program).count("add_rms_norm_forward") == 2
    assert "add_forward" not in kinds(program) and "rms_norm_forward" not in kinds(program)
    for node, v in ((a, av), (b, bv), (g, gv), (t, targets)):
        program.feed(node, v)
    bytes_of = {op.kind: training.op_bytes(op) for op in program.ops}
    assert bytes_of["add_rms_norm_forward"] == ("rms_norm", 4 * 4 * B * T * D)
    assert bytes_of["gated_recurrence_backward"] == ("gated_recurrence", 6 * 4 * B * T * D)
    run_checked(program)
    A, Bt, G, W = leaf(av), leaf(bv), leaf(gv), leaf(wv)
    S1 = A + Bt
    S2 = S1 + recurrence64(norm64(S1, W), G)
    Y2 = norm64(S2, W)
    L = F.cross_entropy((Y2 * torch.tensor(tv, dtype=torch.float64)).reshape(B, -1),
                        torch.tensor(targets, dtype=torch.long))
    L.backward()
    close(program.value(s1).host(), S1, "sum")
    close(program.value(y2).host(), Y2, "second norm")
    close(program.value(loss).host()[0], L, "loss")
    for node, ref in ((a, A), (b, Bt), (g, G)):
        close(program.gradient(node).host(), ref.grad, node)
    close(program.gradient(w.tensor()).host(), W.grad, "weight")


def test_one_value_as_input_and_gate_and_what_needs_no_gradient():
    """A recurrence of one value twice; a norm of a fed input (only its weight takes a gradient)
    and one with a constant weight (only its input does); a gate without a gradient."""
    B, T, D = 2, 5, 12
    fv, xv, gv, cv = (randn(B, T, D, seed=i) for i in range(4))
    wv, kv = 1 + 0.1 * randn(D, seed=7), 1 + 0.1 * randn(D, seed=8)
    targets = np.array([3, 17], np.float32)
    f, t = tn.input((B, T, D)), tn.input((B,))
    x, w = tn.input((B, T, D), requires_grad=True), nn.Parameter(wv)
    n = f.rms_norm(w.tensor(), 1e-3)
    m = x.rms_norm(tn.constant(kv)).add(n)
    loss = (m.gated_recurrence(m).gated_recurrence(tn.constant(gv)).mul(tn.constant(cv))
            .reshape((B, T * D)).cross_entropy(t))
    program = tn.training_program(loss)
    for node, v in ((f, fv), (x, xv), (t, targets)):
        program.feed(node, v)
    run_checked(program)
    X, W = leaf(xv), leaf(wv)
    c = lambda v: torch.tensor(v, dtype=torch.float64)  # noqa: E731
    M = norm64(X, c(kv)) + norm64(c(fv), W, 1e-3)
    L = F.cross_entropy((recurrence64(recurrence64(M, M), c(gv)) * c(cv)).reshape(B, -1),
                        torch.tensor(targets, dtype=torch.long))
    L.backward()
    close(program.gradient(x).host(), X.grad, "input")
    close(program.gradient(w.tensor()).host(), W.grad, "weight")
    assert program.gradient(f) is None


def test_forward_program_forms_a_norm_with_its_add():
    x, y = (tn.input((4, 30)) for _ in range(2))
    w = nn.Parameter(1 + 0.1 * randn(30, seed=1))
    s = x.add(y)
    out = s.rms_norm(w.tensor()).add(s)
    program = tn.forward_program(out, [x, y])
    assert kinds(program) == ["add_rms_norm_forward", "add_forward"]
    a, b = randn(4, 30, seed=2), randn(4, 30, seed=3)
    program.feed(x, a)
    program.feed(y, b)
    program.run()
    S = torch.tensor(a, dtype=torch.float64) + torch.tensor(b, dtype=torch.float64)
    close(program.value(out).host(),
          norm64(S, torch.tensor(w.host(), dtype=torch.float64)) + S, "output")


def images_of(count, seed=0):
    """Byte images whose class is where a bright band lies, with noise."""
    r = np.random.default_rng(seed)
    labels = r.integers(0, 10, count).astype(np.uint8)
    images = r.integers(0, 60, (count, 28, 28)).astype(np.uint8)
    for i, c in enumerate(labels):
        images[i, 2 * c + 4:2 * c + 7, 3 + c:20 + c % 5] += 150
    return images.reshape(count, 784), labels


def step_of(batch=16, update=None):
    model = sequence.RowClassifier(features=32, depth=2)
    return model, sequence.Training(model, batch, update)


def test_step_of_the_optimizer_in_a_program():
    """Matrices move by the orthogonalised momentum of the program's own gradients, the others as
    AdamW alone moves them."""
    images, labels = images_of(16)
    model, step = step_of()
    assert training.op_bytes(step.program.ops[-1]) == ("muon", 6 * 5 * 4 * 32 * 32)
    before = [p.host().copy() for p in model.parameters()]
    step.images.copy_from(images.astype(np.float32).reshape(16, 1, 28, 28) / 255)
    step.labels.copy_from(labels.astype(np.float32))
    step.step()
    assert np.isfinite(step.loss())
    matrices = {id(p) for p in sequence.optimizer(model).matrices}
    assert len(matrices) == 6
    c1, c2 = ox.adamw_corrections(0.9, 0.999, 1)
    for p, old in zip(model.parameters(), before):
        g = step.program.gradient(p.tensor()).host().astype(np.float64)
        if id(p) in matrices:
            flat = g.reshape(g.shape[0], -1)
            x = orthogonal(flat + 0.95 * flat).reshape(g.shape)
            ref = old - 0.02 * math.sqrt(max(1.0, flat.shape[0] / flat.shape[1])) * x
        else:
            ref = old - 3e-3 * ((0.1 * g / c1) / (np.sqrt(0.001 * g * g / c2) + 1e-8) + 1e-4 * old)
        moved = np.linalg.norm(ref - old)
        assert np.linalg.norm(p.host() - ref) <= 1e-3 * moved + 1e-7 * np.linalg.norm(old), p.shape


def test_replays_equal_eager_steps():
    images, labels = images_of(16)
    x, y = images.astype(np.float32).reshape(16, 1, 28, 28) / 255, labels.astype(np.float32)
    results = []
    for replay in (True, False):
        model, step = step_of()
        step.images.copy_from(x)
        step.labels.copy_from(y)
        for _ in range(4):
            step.step() if replay else step.program.run()
            torch.cuda.synchronize()
        results.append([p.host() for p in model.parameters()])
    for a, b in zip(*results):
        assert np.array_equal(a, b)


def test_all_parameters_matrices_without_adamw():
    """A program whose every trained parameter is a matrix, and no AdamW."""
    w = nn.Parameter(randn(12, 9, 1, 1, seed=1))
    x, t = tn.input((6, 9, 1, 1)), tn.input((6,))
    loss = x.conv2d(w.tensor(), tn.constant(np.zeros(12)), 1, 0, 1).reshape((6, 12)) \
        .cross_entropy(t)
    update = nn.Muon([w], None, learning_rate=0.1, nesterov=False)
    program = tn.training_program(loss, update)
    program.feed(x, randn(6, 9, 1, 1, seed=2))
    program.feed(t, np.arange(6, dtype=np.float32))
    old = w.host().copy()
    program.capture()
    program.replay()
    program.check()
    g = program.gradient(w.tensor()).host().astype(np.float64).reshape(12, 9)
    ref = old.reshape(12, 9) - 0.1 * math.sqrt(12 / 9) * orthogonal(g)
    assert np.linalg.norm(w.host().reshape(12, 9) - ref) <= 1e-3 * np.linalg.norm(
        ref - old.reshape(12, 9))
    assert program.steps() == 0


def test_row_classifier_learns():
    images, labels = images_of(640)
    model = sequence.RowClassifier(features=64, depth=2)
    losses = []
    sequence.train(model, images, labels, batch=64, epochs=8,
                   report=lambda line: losses.append(float(line.split()[-1])))
    assert losses[-1] < 0.2 and losses[-1] < losses[0]
    test_images, test_labels = images_of(200, seed=1)
    assert sequence.accuracy(model, test_images, test_labels) > 0.9


def test_builders_refuse():
    with pytest.raises(ox.OxideError) as err:
        tn.input((2, 3)).rms_norm(tn.constant(np.ones(2)))
    assert err.value.kind == "InvalidShape"
    with pytest.raises(ox.OxideError) as err:
        tn.input((2, 3)).rms_norm(tn.constant(np.ones(3)), float("nan"))
    assert err.value.kind == "Execution"
    for other in ((2, 3, 5), (2, 3)):
        with pytest.raises(ox.OxideError):
            tn.input((2, 3, 4)).gated_recurrence(tn.input(other))
    for bad in (dict(learning_rate=0.0), dict(weight_decay=-1.0), dict(momentum=1.0)):
        with pytest.raises(ox.OxideError):
            nn.Muon([], nn.AdamW(1e-3, 0.0), **bad)


def test_compiled_block():
    """jit.compile of a block: no fused plan takes it, so it runs as a program."""
    block, x = nn.GatedRecurrentBlock(24), randn(2, 11, 24, seed=1)
    module = jit.compile(block, x)
    with torch.no_grad():
        X = torch.tensor(x, dtype=torch.float64)
        weight = lambda m: torch.tensor(m.conv.weight.host()[:, :, 0, 0].astype(np.float64))  # noqa: E731
        linear = lambda m, v: v @ weight(m).T + torch.tensor(m.conv.bias.host().astype(np.float64))  # noqa: E731
        y = norm64(X, torch.tensor(block.norm.weight.host().astype(np.float64)))
        ref = X + linear(block.project, recurrence64(linear(block.value, y), linear(block.gate, y)))
    for _ in range(2):
        close(np.asarray(module.run([x])).reshape(x.shape), ref, "block")


def test_adamw_alone_over_sequence_layers():
    images, labels = images_of(16)
    model, step = step_of(update=nn.AdamW(1e-2, 0.1))
    before = [p.host().copy() for p in model.parameters()]
    step.images.copy_from(images.astype(np.float32).reshape(16, 1, 28, 28) / 255)
    step.labels.copy_from(labels.astype(np.float32))
    step.step()
    assert np.isfinite(step.loss()) and step.program.steps() == 1
    c1, c2 = ox.adamw_corrections(0.9, 0.999, 1)
    for p, old in zip(model.parameters(), before):
        g = step.program.gradient(p.tensor()).host().astype(np.float64)
        moved = 1e-2 * ((0.1 * g / c1) / (np.sqrt(0.001 * g * g / c2) + 1e-8) + 0.1 * old)
        off = np.linalg.norm(p.host() - (old - moved))
        assert off <= 1e-3 * np.linalg.norm(moved) + 1e-7 * np.linalg.norm(old), p.shape


def test_example_on_idx_files(tmp_path, capsys):
    """The example's command: IDX files in, a line per epoch and the test accuracy out."""
    for name, count, seed in (("train", 384, 0), ("t10k", 200, 1)):
        images, labels = images_of(count, seed)
        (tmp_path / f"{name}-images-idx3-ubyte").write_bytes(_idx_images(images))
        (tmp_path / f"{name}-labels-idx1-ubyte").write_bytes(_idx_labels(labels))
    sequence.main(str(tmp_path), 2)
    lines = capsys.readouterr().out.splitlines()
    assert [line.split()[0] for line in lines] == ["epoch", "epoch", "test"]
    assert math.isfinite(float(lines[1].split()[-1])) and 0 <= float(lines[2].split()[-1]) <= 1


@pytest.mark.parametrize("uses", ["alone", "added", "multiplied"])
def test_norm_of_a_value_by_itself(uses):
    """A value that is input and weight of a norm takes both gradients, beside those of other uses
    (an add's waits for the norm's, a product's is there before it)."""
    D = 24
    wv, cv = 1 + 0.3 * randn(D, seed=5), randn(D, seed=6)
    w, t = nn.Parameter(wv), tn.input((1,))
    v = w.tensor()
    y = v.rms_norm(v)
    if uses == "added":
        y = y.add(v)
    if uses == "multiplied":
        y = y.mul(v)
    loss = y.mul(tn.constant(cv)).reshape((1, D)).cross_entropy(t)
    program = tn.training_program(loss)
    program.feed(t, np.array([3], np.float32))
    run_checked(program)
    W = leaf(wv)
    Y = norm64(W, W)
    Y = {"alone": Y, "added": Y + W, "multiplied": Y * W}[uses]
    F.cross_entropy((Y * torch.tensor(cv, dtype=torch.float64)).reshape(1, D),
                    torch.tensor([3])).backward()
    close(program.gradient(v).host(), W.grad, "gradient")
    for _ in range(2):
        program.run()
    close(program.gradient(v).host(), W.grad, "gradient of the whole program")


def test_bytes_of_norm_backwards():
    """A norm's backward counts the other gradient of its input that it reads: a waiting add's, or
    the one it adds to in place; none where the norm is the only use."""
    B, T, D = 2, 3, 16
    a, b, c = (tn.input((B, T, D), requires_grad=True) for _ in range(3))
    w, t = nn.Parameter(1 + 0.1 * randn(D, seed=1)), tn.input((B,))
    s = a.add(b)
    added = s.add(s.rms_norm(w.tensor()))            # s takes the add's gradient
    p = added.mul(c)
    in_place = p.mul(p.rms_norm(w.tensor()))         # p takes the product's first
    alone = in_place.rms_norm(w.tensor())
    loss = alone.reshape((B, T * D)).cross_entropy(t)
    program = tn.training_program(loss)
    ops = [op for op in program.ops if op.kind == "rms_norm_backward"]
    assert [("addend" in op.reads, "input_gradient" in op.by_role) for op in ops] == \
        [(False, False), (False, True), (True, False)]
    assert [training.op_bytes(op) for op in ops] == \
        [("rms_norm", n * 4 * B * T * D) for n in (3, 4, 4)]
