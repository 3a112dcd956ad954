"""The gated delta rule writes its outputs and its workspace and nothing around them: a workspace of
exactly the bytes that the library names, and outputs of every width, between guard bytes.  Values
against the steps in float64, with the tolerances of test_gpu_delta_rule."""

import ctypes

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import nn
import oxide_hip as ox
import sequence
from test_gpu_delta_rule import TYPES, backward, check_forward, check_gradients, operands
from test_gpu_reward_net import c64, model64
from test_gpu_rms_norm import make
from test_gpu_sequence_net import close, images_of, leaf

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def at(x):
    return None if x is None else x.data_ptr()


@pytest.mark.parametrize("saves", [False, True])
@pytest.mark.parametrize("shape", [
    (1, 12160, 16, 16, 128, 8),   # few blocks: one part, two where a state is handed on
    (64, 832, 8, 16, 8, 8),       # many blocks: the same
    (1, 13120, 64, 64, 8, 4)])    # two parts, and three
def test_workspace_without_a_final_state(module, dev, shape, saves):
    """bfloat16, where calls with and without a final state prepare different operands."""
    batch, time, _, heads, keys, values = shape
    ops = operands(shape, BF16, dev, 5)
    out = torch.full_like(ops[2], 7.0)
    _, alone, size, kept, _ = ox._delta_plan(ox.BF16, *shape)
    if not saves:
        size = alone
    guard = 128 << 20  # more than the plans of one call differ by
    room = torch.full((size + guard,), 0x5A, dtype=torch.uint8, device=dev)
    saved = module.gated_delta_rule_saved(ops[1], ops[2]) if saves else None
    ox.check(ox.lib().oxh_gated_delta_rule_forward(
        ox.current_stream(), ox.BF16, ctypes.byref(ox.DeltaShape(*shape)), keys ** -0.5,
        *[at(x) for x in ops], None, None, at(out), None, at(saved), kept if saves else 0,
        at(room), size))
    assert (room[size:] == 0x5A).all()
    check_forward(ops, out, None, BF16, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 130, 1, 2, 64, 40), (64, 130, 4, 8, 40, 12),
                                   (1, 9000, 16, 16, 128, 8), (64, 640, 8, 16, 8, 8)])
def test_saved_and_both_workspaces(module, dev, shape, dtype):
    """Training by a caller with buffers of exactly the sizes named: one part, and several."""
    t, code = TYPES[dtype], {"f32": ox.F32, "bf16": ox.BF16}[dtype]
    ops = operands(shape, t, dev, 6)
    g = make(ops[2].shape, t, dev, 21)
    out, grads = torch.empty_like(ops[2]), [torch.empty_like(x) for x in ops]
    _, _, forward, kept, back = ox._delta_plan(code, *shape)
    dims, scale, edge = ctypes.byref(ox.DeltaShape(*shape)), shape[4] ** -0.5, 1 << 20
    saved, ws, ws_back = (torch.full((n + edge,), 0x5A, dtype=torch.uint8, device=dev)
                          for n in (kept, forward, back))
    stream = ox.current_stream()
    ox.check(ox.lib().oxh_gated_delta_rule_forward(
        stream, code, dims, scale, *[at(x) for x in ops], None, None, at(out), None, at(saved), kept,
        at(ws), forward))
    ox.check(ox.lib().oxh_gated_delta_rule_backward(
        stream, code, dims, scale, at(g), *[at(x) for x in ops], at(saved), kept, None, None,
        *[at(x) for x in grads], None, at(ws_back), back))
    for x, n in ((saved, kept), (ws, forward), (ws_back, back)):
        assert (x[n:] == 0x5A).all()
    ref = check_forward(ops, out, None, t, True)
    check_gradients(ref, g, grads, t)


# widths of every remainder by the columns that one access stores, of many heads (blocks of 32
# columns) and of few (16)
WIDTHS = [(64, 66, 2, 4, 32, 36), (256, 70, 1, 1, 32, 12), (32, 65, 4, 8, 20, 20),
          (64, 70, 1, 1, 64, 100), (1, 130, 1, 256, 8, 28), (128, 28, 4, 4, 20, 20),
          (86, 65, 1, 3, 12, 4), (32, 66, 2, 8, 16, 56), (2, 70, 1, 2, 8, 12), (1, 66, 2, 4, 4, 36)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", WIDTHS)
def test_outputs_of_every_width(module, dev, shape, dtype):
    """16-byte aligned rows, which are stored 16 bytes at a time, and nothing around them: outputs
    and gradients, the same bits when asked again."""
    t = TYPES[dtype]
    ops = operands(shape, t, dev, 3)
    g = make(ops[2].shape, t, dev, 21)
    edge = 64  # elements
    rooms = [torch.full((x.numel() + 2 * edge,), 7.0, dtype=t, device=dev)
             for x in (ops[2], *ops)]
    out, *grads = [r[edge:-edge].view(x.shape) for r, x in zip(rooms, (ops[2], *ops))]
    assert out.data_ptr() % 16 == 0
    saved = module.gated_delta_rule_saved(ops[1], ops[2])
    module.gated_delta_rule_forward(*ops, out, saved=saved)
    ref = check_forward(ops, out, None, t, True)
    module.gated_delta_rule_backward(g, *ops, saved, *grads)
    check_gradients(ref, g, grads, t)
    for r in rooms:
        assert (r[:edge] == 7).all() and (r[-edge:] == 7).all()
    again = torch.full_like(out, 3.0)
    module.gated_delta_rule_forward(*ops, again, saved=saved)
    assert torch.equal(again, out)
    for x, y in zip(backward(module, ops, g, saved), grads):
        assert torch.equal(x, y)


def test_classifier_of_20_columns_a_head():
    """Its training forward and gradients, at the example's batch."""
    images, labels = images_of(128)
    pixels = images.astype(np.float32).reshape(128, 1, 28, 28) / 255
    model = sequence.RowClassifier(features=80, depth=1, block=nn.DeltaRuleBlock, norm=nn.LayerNorm)
    step = sequence.Training(model, 128)
    step.images.copy_from(pixels)
    step.labels.copy_from(labels.astype(np.float32))
    params = [leaf(p.host()) for p in model.parameters()]
    step.step()
    logits = model64(model, params, c64(pixels[:, 0]))
    F.cross_entropy(logits, torch.tensor(labels.astype(np.int64))).backward()
    close(step.logits.host(), logits, "logits")
    for p, ref in zip(model.parameters(), params):
        close(step.program.gradient(p.tensor()).host(), ref.grad, p.shape)
