"""What the accuracy of the gated delta rule's bfloat16 results is held to, and that a lost term
exceeds it: on the CPU, by the chunks' formulas with the device's roundings in float64.

BOUND.  A rounding to bfloat16 is at most half a step off, 2^-8 of the smallest value with its exponent;
evenly spread errors and mantissas as products have them make that 2^-8 / sqrt(3) * sqrt(3 / (8 ln 2))
= 1.66e-3 in the mean square.  A path from the operands to a result meets at most six: the state, b y
(b du, x), the system or a matrix of pairs, b e (e, u), what is made of the state's gradient, and the
result's own.  They are independent: sqrt(6) * 1.66e-3 = 4.1e-3 of the result's Frobenius norm.  2^-7 =
7.8e-3 leaves a factor of nearly 2 for terms that cancel.

STATE_BOUND, of a state that is handed on: two parts leave 2^-18, so 2^-18 / sqrt(3) * 0.74 = 1.6e-6 in
the mean square, five of them 3.6e-6, and float32 sums of at most 256 terms sqrt(256) * 2^-24 = 1e-6:
2^-16 = 1.5e-5 leaves a factor of 3."""

import functools

import numpy as np
import pytest
import torch

from delta_rule_chunks import chunked, off
from test_gpu_delta_rule import Reference

BOUND, STATE_BOUND = 2.0 ** -7, 2.0 ** -16
SHAPES = [(2, 200, 2, 64, 48), (4, 130, 2, 128, 128), (3, 70, 2, 17, 40), (2, 300, 2, 32, 16),
          (4, 28, 4, 32, 32), (1, 520, 2, 96, 24)]


def low(x):
    return torch.from_numpy(np.ascontiguousarray(x)).float().bfloat16().double().numpy()


def high(x):
    return low(x) + low(x - low(x))


def operands(shape, seed=1, mean=4.0):
    """Of bfloat16 values: unit keys and queries, gates that keep most of the state over a chunk."""
    r = np.random.default_rng(seed)
    batch, time, heads, keys, values = shape

    def unit():
        v = r.standard_normal((batch, time, heads, keys))
        return low(0.99 * v / np.linalg.norm(v, axis=-1, keepdims=True))

    row = (batch, time, heads)
    return [unit(), unit(), low(r.standard_normal((*row, values))),
            low(1.5 * r.standard_normal(row) + mean), low(r.standard_normal(row))], \
        low(r.standard_normal((*row, values)))


@pytest.mark.parametrize("shape", SHAPES)
def test_the_formulas_are_the_steps(shape):
    ops, g = operands(shape)
    r = np.random.default_rng(9)
    first, final = (r.standard_normal((shape[0], *shape[2:])) for _ in range(2))
    got = chunked(*ops, g, state=first, final=final)
    wide = torch.from_numpy
    steps = Reference(*[wide(x) for x in ops], wide(first))
    gradients, back, _ = steps.gradients(wide(g), wide(final))
    assert off(got["output"], steps.out) < 1e-11 and off(got["state"], steps.states[-1]) < 1e-11
    assert off(got["first state"], back) < 1e-11
    for name, (ref, _) in gradients.items():
        assert off(got[name], ref) < 1e-10, name


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("mean", [2.0, 4.0, 7.0])
def test_the_roundings_keep_within_the_bounds(shape, mean):
    ops, g = operands(shape, 2, mean)
    ref, got = chunked(*ops, g), chunked(*ops, g, low=low)
    for name in got:
        if name not in ("state", "first state"):
            assert off(low(got[name]), ref[name]) < BOUND, name
    assert off(got["first state"], ref["first state"]) < BOUND
    handed = chunked(*ops, low=low, high=high)
    assert off(low(handed["output"]), ref["output"]) < BOUND
    assert off(handed["state"], ref["state"]) < STATE_BOUND


# each term of the formulas, and a result that its loss must show in
TERMS = {"keys of the state": "output", "system": "output", "queries of the state": "output",
         "scores": "output", "decay": "state", "scores'": "value",
         "keys of the state's gradient": "value", "system'": "value", "queries' state": "query",
         "keys' state": "key", "keys' state gradient": "key", "pairs of queries": "gate",
         "pairs of keys": "gate", "queries in the decay": "gate", "keys in the decay": "gate",
         "keys of the gradient in the decay": "gate", "state in the decay": "gate",
         "queries' pairs": "query", "keys' pairs of queries": "key", "keys' earlier pairs": "key",
         "keys' later pairs": "key", "decay of the gradient": "value",
         "queries into the gradient": "value", "keys out of the gradient": "value"}


@functools.cache
def complete(shape):
    ops, g = operands(shape, 3, 7.0)
    return ops, g, chunked(*ops, g)


@pytest.mark.parametrize("term", TERMS)
@pytest.mark.parametrize("shape", [SHAPES[1], SHAPES[3]])
def test_a_lost_term_exceeds_them(shape, term):
    ops, g, ref = complete(shape)
    name = TERMS[term]
    assert off(chunked(*ops, g, drop=(term,))[name], ref[name]) > 2 * BOUND
