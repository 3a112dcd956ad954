"""Newton-Schulz orthogonalisation and the optimizer step over it against the definition in float64.

Tolerance.  An operand of a product keeps 22 bits, so each round perturbs X by about 2^-22 of its
norm, and five rounds stretch what lies in the directions of the smallest singular values by at
most 3.4445^5 = 485; the perturbation of a whole round in those directions is the float32 rounding
of X alone, so 485 * 2^-22 = 1.2e-4 of the result's Frobenius norm is a bound that random matrices
stay far below.  One round: 3.4445 * 2^-22 * 4."""

import math

import numpy as np
import pytest
import torch

import oxide_hip as ox

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315
BOUND = A ** 5 * 2.0 ** -22
SHAPES = [(1, 1), (1, 200), (200, 1), (2, 3), (31, 33), (32, 32), (33, 64), (64, 65), (96, 192),
          (192, 96), (130, 127), (128, 512), (512, 96), (257, 300), (100, 1280), (10, 1280),
          (700, 710), (300, 2000), (2000, 300)]


def orthogonal(v, rounds=5, eps=1e-7):
    x = v.T if v.shape[0] > v.shape[1] else v
    x = x / (np.linalg.norm(x) + eps)
    for _ in range(rounds):
        gram = x @ x.T
        x = A * x + (B * gram + C * (gram @ gram)) @ x
    return x.T if v.shape[0] > v.shape[1] else x


def matrix(shape, seed, scale=1e-3):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(np.float32)


def close(got, ref, bound, what=""):
    off = np.linalg.norm(got.detach().cpu().double().numpy() - ref)
    assert off <= bound * max(np.linalg.norm(ref), 1e-30), (what, off, np.linalg.norm(ref))


@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(module, dev, shape):
    v = matrix(shape, 1)
    x, out = torch.from_numpy(v).to(dev), torch.empty(shape, device=dev)
    module.orthogonalize(x, out)
    close(out, orthogonal(v.astype(np.float64)), BOUND)
    singular = np.linalg.svd(orthogonal(v.astype(np.float64)), compute_uv=False)
    assert singular.max() < 1.25


@pytest.mark.parametrize("shape", [(40, 70), (70, 40), (200, 200)])
@pytest.mark.parametrize("rounds", [1, 2, 3, 8])
def test_rounds(module, dev, shape, rounds):
    v = matrix(shape, 2)
    out = torch.empty(shape, device=dev)
    module.orthogonalize(torch.from_numpy(v).to(dev), out, rounds=rounds)
    close(out, orthogonal(v.astype(np.float64), rounds), A ** min(rounds, 5) * 2.0 ** -20)


@pytest.mark.parametrize("scale", [1e-15, 1e-6, 1.0, 1e15])
def test_any_scale(module, dev, scale):
    """The norm is taken first, so only its own range limits the values (the sum of squares is a
    float32)."""
    v = matrix((60, 90), 3, scale)
    out = torch.empty(60, 90, device=dev)
    module.orthogonalize(torch.from_numpy(v).to(dev), out, epsilon=1e-20)
    close(out, orthogonal(v.astype(np.float64), eps=1e-20), BOUND)


def test_low_rank_and_decaying_spectrum(module, dev):
    """Directions far below the largest one: the ones that five rounds stretch most."""
    r = np.random.default_rng(4)
    v = ((r.standard_normal((150, 20)) * np.exp(-np.arange(20) / 4)) @
         r.standard_normal((20, 260))).astype(np.float32)
    out = torch.empty(150, 260, device=dev)
    module.orthogonalize(torch.from_numpy(v).to(dev), out)
    close(out, orthogonal(v.astype(np.float64)), BOUND)


def test_stack_equals_its_matrices(module, dev):
    """More matrices than one launch group takes, each with the bits it has alone."""
    v = torch.from_numpy(matrix((70, 24, 40), 5)).to(dev)
    out, one = torch.empty_like(v), torch.empty(24, 40, device=dev)
    module.orthogonalize(v, out)
    for i in (0, 31, 32, 69):
        module.orthogonalize(v[i], one)
        assert torch.equal(out[i], one)


def test_zero_and_not_finite(module, dev):
    v = torch.from_numpy(matrix((4, 50, 60), 6)).to(dev)
    v[1] = 0.0
    v[2, 3, 4] = float("nan")
    out, clean = torch.empty_like(v), torch.empty(50, 60, device=dev)
    module.orthogonalize(v, out)
    assert (out[1] == 0).all() and out[2].isnan().all()
    for i in (0, 3):
        module.orthogonalize(v[i], clean)
        assert torch.equal(out[i], clean)


SETS = [[(96, 192)], [(192, 96, 1, 1)], [(32, 16, 3, 3), (10, 1280, 1, 1), (7, 5)],
        [(300, 200), (200, 300), (64, 64), (1, 9)], [(24, 24 + i) for i in range(40)]]


@pytest.mark.parametrize("shapes", SETS)
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(module, dev, shapes, nesterov):
    """Two steps over a list of matrices (convolution weights among them)."""
    r = np.random.default_rng(7)
    p, g, m = ([r.standard_normal(s).astype(np.float32) * k for s in shapes]
               for k in (0.05, 1e-3, 1e-2))
    dev_p, dev_g, dev_m = ([torch.from_numpy(a).to(dev) for a in t] for t in (p, g, m))
    p, g, m = ([a.astype(np.float64).reshape(a.shape[0], -1) for a in t] for t in (p, g, m))
    for _ in range(2):
        module.muon(0.02, 0.1, 0.95, list(zip(dev_p, dev_g, dev_m)), nesterov=nesterov)
        for i in range(len(p)):
            m[i] = 0.95 * m[i] + g[i]
            x = orthogonal(g[i] + 0.95 * m[i] if nesterov else m[i])
            scale = math.sqrt(max(1.0, p[i].shape[0] / p[i].shape[1]))
            moved = 0.02 * (0.1 * p[i] + scale * x)
            p[i] = p[i] - moved
            flat = lambda t: t.reshape(t.shape[0], -1)  # noqa: E731
            close(flat(dev_m[i]), m[i], 4 * 2.0 ** -24, "momentum")
            off = flat(dev_p[i]).cpu().double().numpy() - p[i]
            tol = 2 * BOUND * np.linalg.norm(moved) + 4 * 2.0 ** -24 * np.linalg.norm(p[i])
            assert np.linalg.norm(off) <= tol


def test_another_stream_a_graph_and_repeats(module, dev):
    shapes = [(96, 192), (130, 70), (512, 520)]
    start = [[torch.from_numpy(matrix(s, 10 * i + j, k)).to(dev) for j, s in enumerate(shapes)]
             for i, k in enumerate((0.05, 1e-3, 1e-2))]
    p, g, m = ([t.clone() for t in ts] for ts in start)

    def reset():
        for now, then in zip((p, g, m), start):
            for a, b in zip(now, then):
                a.copy_(b)
        torch.cuda.synchronize()

    def step(stream=None):
        module.muon(0.02, 0.01, 0.9, list(zip(p, g, m)), stream=stream)

    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in p + m]
    stream = torch.cuda.Stream()
    reset()
    graph = ox.HipGraphExec.capture(stream, lambda: step(stream))
    for run in (lambda: step(stream), lambda: graph.launch(stream), lambda: graph.launch(stream)):
        reset()
        run()
        torch.cuda.synchronize()
        for a, b in zip(p + m, want):
            assert torch.equal(a, b)


# sides at which tiles of 64 fill the compute units once or more often, of 128, and of 192
LARGE = [(1000, 1280), (520, 2050), (1537, 1660), (4000, 1030), (2050, 2300), (3900, 3870)]


def orthogonal_on(v, rounds=5, eps=1e-7):
    """``orthogonal`` of a float64 tensor where it lies."""
    x = v.T.contiguous() if v.shape[0] > v.shape[1] else v
    x = x / (x.norm() + eps)
    for _ in range(rounds):
        gram = x @ x.T.contiguous()
        x = A * x + (B * gram + C * (gram @ gram)) @ x
    return x.T.contiguous() if v.shape[0] > v.shape[1] else x


@pytest.mark.parametrize("shape", LARGE)
def test_large(module, dev, shape):
    """Both entry points, with a spectrum that falls by 10^4 over an eighth of the directions."""
    g = torch.Generator().manual_seed(11)
    rank = min(shape) // 8
    left = torch.randn(shape[0], rank, generator=g) * torch.logspace(0, -4, rank)
    v = (left @ torch.randn(rank, shape[1], generator=g) +
         1e-4 * torch.randn(*shape, generator=g)).to(dev)
    out = torch.empty_like(v)
    module.orthogonalize(v, out)
    ref = orthogonal_on(v.double())
    assert (out.double() - ref).norm() <= BOUND * ref.norm()
    p = torch.randn(*shape, generator=g).to(dev)
    m = torch.zeros_like(p)
    moved = 0.1 * math.sqrt(max(1.0, shape[0] / shape[1])) * ref
    want = p.double() - moved
    module.muon(0.1, 0.0, 0.9, [(p, v, m)], nesterov=False)
    assert torch.equal(m, v)
    tol = BOUND * moved.norm() + 4 * 2.0 ** -24 * want.norm()
    assert (p.double() - want).norm() <= tol


# short sides of up to 128 with more columns than one block takes
SLABS = [(87, 1091), (1091, 87), (1, 4000), (20, 1500), (32, 1025), (64, 700), (700, 61), (96, 193),
         (193, 96), (90, 384), (385, 70), (128, 2049), (2500, 100), (96, 19200), (33, 19201)]


@pytest.mark.parametrize("shape", SLABS)
@pytest.mark.parametrize("rounds", [1, 2, 5])
def test_slabs(module, dev, shape, rounds):
    v = matrix(shape, 13)
    x, out = torch.from_numpy(v).to(dev), torch.empty(shape, device=dev)
    module.orthogonalize(x, out, rounds=rounds)
    ref = orthogonal_on(x.double(), rounds).cpu().numpy()
    close(out, ref, A ** rounds * 2.0 ** -22 if rounds == 5 else A ** rounds * 2.0 ** -20)


def test_step_of_every_kind(module, dev):
    """One list with matrices that a block takes, that go in slabs (more than a launch group of one
    side, and of several) and in tiles; each moves as it does alone, and a replay repeats it."""
    shapes = [(30, 40), (128, 150), (300, 310), (128, 600), (90, 700), (2100, 120)] + \
        [(64, 600 + 7 * i) for i in range(34)] + [(1300, 33)]
    r = np.random.default_rng(14)
    start = [[torch.from_numpy(r.standard_normal(s).astype(np.float32) * k).to(dev)
              for s in shapes] for k in (0.05, 1e-3, 1e-2)]
    alone = [[t.clone() for t in ts] for ts in start]
    for one in zip(*alone):
        module.muon(0.02, 0.01, 0.9, [one])
    for i, (p, g, m) in enumerate(zip(*start)):
        want = orthogonal_on((g + 0.9 * (0.9 * m + g)).double())
        scale = math.sqrt(max(1.0, shapes[i][0] / shapes[i][1]))
        moved = 0.02 * (0.01 * p.double() + scale * want)
        off = (alone[0][i].double() - (p.double() - moved)).norm()
        assert off <= BOUND * moved.norm() + 4 * 2.0 ** -24 * p.double().norm(), shapes[i]
    p, g, m = ([t.clone() for t in ts] for ts in start)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def step():
        module.muon(0.02, 0.01, 0.9, list(zip(p, g, m)), stream=stream)

    step()
    torch.cuda.synchronize()
    graph = ox.HipGraphExec.capture(stream, step)
    for _ in range(2):
        for now, then in zip((p, g, m), start):
            for a, b in zip(now, then):
                a.copy_(b)
        torch.cuda.synchronize()
        graph.launch(stream)
        torch.cuda.synchronize()
        for a, b in zip(p + m, alone[0] + alone[2]):
            # tiles are chosen for a list, so (128, 600) and (300, 310) may differ in rounding
            assert (a - b).norm() <= 1e-5 * b.norm()
            if a.shape[0] not in (128, 300):
                assert torch.equal(a, b)


# sides that a block takes, that go in slabs and in tiles of each size
SMALL_NORMS = [(60, 90), (96, 700), (257, 300), (300, 200), (700, 710), (520, 2050), (2050, 2300)]


@pytest.mark.parametrize("shape", SMALL_NORMS)
@pytest.mark.parametrize("norm", [2e-8, 1e-8, 1e-9, 1e-11, 1e-13, 1e-15])
def test_norms_below_epsilon(module, dev, shape, norm):
    """|V|_F / (|V|_F + epsilon) far below 1: X starts small and keeps its bits.  From 1e-11 on X stays
    below 485e-4, where a round multiplies it by 3.4445 but for a part of 3.3e-3 at most: its
    rounding to 22 bits, of which half a unit is 2^-23, the product's in float32 and the entries'
    floor (2^-39 of an X of at least 1/4) add up, below 2^-22 a round."""
    g = torch.Generator().manual_seed(21)
    v = torch.randn(*shape, generator=g).double()
    v = (v / v.norm() * norm).float().to(dev)
    out = torch.empty_like(v)
    module.orthogonalize(v, out)
    ref = orthogonal_on(v.double())
    bound = BOUND if norm > 1e-11 else 5 * 2.0 ** -22
    assert (out.double() - ref).norm() <= bound * ref.norm()


@pytest.mark.parametrize("norm", [1.0, 9e-8, 6e-8, 4e-8, 3.4e-8, 2e-8, 1e-8, 1e-9, 1e-12])
@pytest.mark.parametrize("rounds", [1, 5])
def test_one_direction_at_any_norm(module, dev, norm, rounds):
    """A matrix of rank 1, whose whole norm is one singular value: the largest entries that A and B
    can have."""
    left, right = torch.randn(300, 1, generator=torch.Generator().manual_seed(22)), \
        torch.ones(1, 310)
    left[7], right[0, 9] = 300.0, 300.0  # one entry holds most of it
    v = (left @ right).double()
    v = (v / v.norm() * norm).float().to(dev)
    out = torch.empty_like(v)
    module.orthogonalize(v, out, rounds=rounds)
    ref = orthogonal_on(v.double(), rounds)
    assert (out.double() - ref).norm() <= BOUND * ref.norm()


@pytest.mark.parametrize("shape", [(100, 130), (64, 700), (300, 310), (700, 710), (1000, 1280)])
def test_small_rows(module, dev, shape):
    """Eight rows of 1e-6 of the others: what they lose to the halves' floor.  A round leaves them
    2^-39 an entry of X off, and as much of A and of B (b and 1 times), each of which a round's X of
    norm 1 turns into rows: sqrt(8 columns) (a + b + 2) 2^-39 at most, and every later round takes
    3.4445 times it on: 684 (1 + a + .. + a^5) times that in all, beside the bound on the whole."""
    v = torch.randn(*shape, generator=torch.Generator().manual_seed(24)).to(dev)
    v[:8] *= 1e-6
    out = torch.empty_like(v)
    module.orthogonalize(v, out)
    ref = orthogonal_on(v.double())
    floor = 684 * (A - B + 2) * 2.0 ** -39 * math.sqrt(8 * shape[1])
    assert (out[:8].double() - ref[:8]).norm() <= floor + BOUND * ref[:8].norm()
    assert (out.double() - ref).norm() <= BOUND * ref.norm()


@pytest.mark.parametrize("shape", [(60, 90), (96, 700), (300, 310), (700, 710), (1000, 1280),
                                   (2050, 2300), (3900, 3870)])
def test_bits_of_one_round(module, dev, shape):
    """A round's bound from its operands' bits, 2^-23 each (half a unit of 22): a X has a (1 more for
    its rounding); A of |A|_F <= 1 two of them, its rounding, and b A and B's rounding after it, c A A
    two A's and their rounding, and B X those of B and of X, for |B|_F <= b + c: in all a + 1 + 4 b +
    8 c + 2 (b + c) = 54 units of 2^-23 in the worst case, were all errors of one sign.  They are
    independent, and a sum of thousands of them is below an eighth of that."""
    v = torch.randn(*shape, generator=torch.Generator().manual_seed(23)).to(dev)
    out = torch.empty_like(v)
    module.orthogonalize(v, out, rounds=1)
    assert (out.double() - orthogonal_on(v.double(), 1)).norm() <= 54 / 8 * 2.0 ** -23
