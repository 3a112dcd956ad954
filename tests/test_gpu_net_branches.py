"""A BatchNorm (+ ReLU) that runs inside the launches of the depthwise layer behind it while other
layers read its output, too: their contributions reach its gradient.  Against torch float64 autograd,
with the tolerance of test_gpu_sequence_net."""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import nn
import tensor as tn
from test_gpu_reward_net import c64
from test_gpu_sequence_net import close, kinds, leaf, randn, run_checked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("relu", [True, False])
@pytest.mark.parametrize("others", [1, 2, 3])
def test_other_readers_of_a_norm_before_a_depthwise_layer(relu, others):
    """Later readers of the norm's output: a loss of its values, a product, a convolution."""
    x, first = tn.input((4, 8, 8, 8), requires_grad=True), nn.Conv2d(8, 8, 1)
    norm, layer = nn.BatchNorm2d(8), nn.ConvNormAct(8, 8, 3, 2, 8, True)
    behind = nn.Conv2d(8, 4, 3, 2)
    y = norm(first(x))
    y = y.relu() if relu else y
    mask, targets = randn(4, 8, 8, 8, seed=2), np.arange(512, dtype=np.float32) % 4
    t, few = tn.constant(targets), tn.constant(targets[:128])
    loss = layer(y).reshape((128, 4)).cross_entropy(few)
    loss = loss.add(y.reshape((512, 4)).cross_entropy(t))
    if others > 1:
        loss = loss.add(y.mul(tn.constant(mask)).reshape((512, 4)).cross_entropy(t))
    if others > 2:
        loss = loss.add(behind(y).reshape((64, 4)).cross_entropy(tn.constant(targets[:64])))
    program = tn.training_program(loss)
    joined = "batch_norm2d_relu_" if relu else "batch_norm2d_"
    assert joined + "depthwise_conv2d_batch_norm_relu_backward" in kinds(program)
    xv = randn(4, 8, 8, 8, seed=6)
    program.feed(x, xv)
    run_checked(program)
    params = [*first.parameters(), *norm.parameters(), *layer.parameters(), *behind.parameters()]
    P = [leaf(p.host()) for p in params]
    X = leaf(xv)
    bn = lambda v, w, b: F.batch_norm(v, None, None, w, b, training=True)  # noqa: E731
    Y = bn(F.conv2d(X, P[0], P[1]), P[2], P[3])
    Y = Y.relu() if relu else Y
    T = torch.tensor(targets.astype(np.int64))
    L = F.cross_entropy(bn(F.conv2d(Y, P[4], P[5], 2, 1, groups=8), P[6], P[7]).relu()
                        .reshape(128, 4), T[:128]) + F.cross_entropy(Y.reshape(512, 4), T)
    if others > 1:
        L = L + F.cross_entropy((Y * c64(mask)).reshape(512, 4), T)
    if others > 2:
        L = L + F.cross_entropy(F.conv2d(Y, P[8], P[9], 2, 1).reshape(64, 4), T[:64])
    L.backward()
    close(program.value(loss).host()[0], L, "loss")
    close(program.gradient(x).host(), X.grad, "input")
    for i, (p, ref) in enumerate(zip(params, P)):
        if ref.grad is None:
            continue
        got = program.gradient(p.tensor()).host()
        # a bias before a norm, or one that all classes of a row share: a sum that is 0, of at most
        # 512 terms below 1/64, each within 8 * 2^-24 of itself: 4e-6
        if i in (1, 5, 9):
            assert np.abs(got).max() < 4e-6
        else:
            close(got, ref.grad, i)
