"""The gated delta rule writes its outputs and its workspace and nothing around them: a workspace of
exactly the bytes that the library names, and outputs of every width, between guard bytes.  Values
against the steps in float64, with the tolerances of test_gpu_delta_rule."""

import ctypes

import pytest
import torch

import oxide_hip as ox
from test_gpu_delta_rule import TYPES, check_forward, operands

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
