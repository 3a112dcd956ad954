"""The gated delta rule's bfloat16 results in the mean square: outputs, gradients and states within the
bounds of test_delta_rule_chunks, which any lost term of the formulas exceeds, of the norms of the
float64 ones."""

import numpy as np
import pytest
import torch

from delta_rule_chunks import chunked, off
from test_delta_rule_chunks import BOUND, STATE_BOUND, operands
from test_gpu_delta_rule import shifted
from test_gpu_rms_norm import f64

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
# batch, time, key heads, heads, keys, values: few blocks (of 16 columns) and many (of 32), every
# count of 32 keys, rows of whole 16 bytes and odd ones, shared heads
SHAPES = [(2, 200, 1, 2, 64, 48), (4, 130, 2, 4, 128, 128), (3, 70, 2, 2, 17, 40),
          (2, 300, 2, 2, 32, 16), (1, 520, 1, 2, 96, 24), (32, 200, 2, 4, 64, 40),
          (32, 130, 4, 8, 128, 32), (64, 70, 2, 4, 17, 40), (128, 129, 1, 2, 96, 24),
          (64, 28, 4, 4, 32, 32), (43, 130, 6, 6, 33, 7)]


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("mean", [4.0, 7.0])
@pytest.mark.parametrize("shape", SHAPES)
def test_results_in_the_mean_square(module, dev, shape, mean, aligned):
    batch, time, key_heads, heads, keys, values = shape
    group = heads // key_heads
    (q, k, v, gate, write), g = operands((batch, time, heads, keys, values), 5, mean)
    q, k = (np.ascontiguousarray(x[:, :, ::group]) for x in (q, k))
    place = (lambda x: x) if aligned else shifted
    ops = [place(torch.from_numpy(x).to(dev, BF16)) for x in (q, k, v, gate, write)]
    go = place(torch.from_numpy(g).to(dev, BF16))
    r = np.random.default_rng(6)
    states = [torch.from_numpy(0.3 * r.standard_normal((batch, heads, keys, values))).to(dev, F32)
              for _ in range(2)]
    first, dfinal = states
    ref = chunked(np.repeat(q, group, 2), np.repeat(k, group, 2), v, gate, write, g,
                  state=f64(first), final=f64(dfinal))
    for name in ("query", "key"):
        ref[name] = ref[name].reshape(batch, time, key_heads, group, keys).sum(3)
    out, final, back = torch.empty_like(ops[2]), torch.empty_like(first), torch.empty_like(first)
    got = {}

    def note(name, x, to, bound=BOUND):
        got[name] = off(f64(x), to) / bound

    saved = module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, initial_state=first, final_state=final, saved=saved)
    note("output with a state", out, ref["output"])
    note("state", final, ref["state"], STATE_BOUND)
    for name, keep in (("output alone", None), ("output", saved)):
        module.gated_delta_rule_forward(*ops, out.fill_(7.0), initial_state=first, saved=keep)
        note(name, out, ref["output"])
    grads = [torch.full_like(x, 7.0) for x in ops]
    module.gated_delta_rule_backward(go, *ops, saved, *grads, final_state_gradient=dfinal,
                                     initial_state_gradient=back)
    for name, x in zip(("query", "key", "value", "gate", "write"), grads):
        note(name, x, ref[name])
    note("first state", back, ref["first state"])
    assert max(got.values()) <= 1.0, got
