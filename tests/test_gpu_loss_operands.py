"""What a loss's rows are beside their logits takes no gradient: targets, actions, old log
probabilities, advantages, reference log probabilities and weights may be computed from parameters
and from inputs that require gradients, which take their gradients from the logits' side alone.
Against torch float64 autograd with those operands detached; the tolerance is that of
test_gpu_sequence_net."""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import nn
import oxide_hip as ox
import tensor as tn
from test_gpu_reward_net import c64, drawn, policy64
from test_gpu_sequence_net import close, kinds, leaf, randn, run_checked

pytestmark = pytest.mark.gpu


def test_policy_operands_of_parameters():
    """Weights from a parameter that nothing else uses (it is not trained), log probabilities from a
    part of the logits' own parameter, advantages from an input that asks for a gradient."""
    rows, classes = 6, 4
    action, old, advantage, _, weight = drawn(rows, classes, 3)
    pv, wv = randn(rows, classes, seed=1), np.abs(weight) + 0.1
    P, W = nn.Parameter(pv), nn.Parameter(wv)
    x = tn.input((rows,), requires_grad=True)
    a, o = tn.input((rows,)), tn.input((rows,))
    logits = P.tensor().mul(tn.constant(np.full((rows, classes), 2.0)))
    flat = W.tensor().mul(tn.constant(np.full(rows, 0.5)))
    advantages = x.add(tn.constant(np.full(rows, 0.25)))
    loss = logits.policy_loss(a, o, advantages, reference_log_probs=o.add(x), weights=flat, kl=0.1)
    program = tn.training_program(loss, nn.AdamW(0.1, 0.01))
    for node, value in ((x, advantage), (a, action), (o, old)):
        program.feed(node, value)
    run_checked(program)
    ref = leaf(pv)
    L = policy64(2 * ref, action, old, advantage + 0.25, np.float32(old + advantage), 0.5 * wv,
                 kl=0.1)
    L.backward()
    close(program.value(loss).host()[0], L, "loss")
    close(program.gradient(P.tensor()).host(), ref.grad, "logits' parameter")
    assert program.gradient(W.tensor()) is None and program.gradient(x) is None
    assert np.array_equal(W.host(), wv.astype(np.float32))  # decay would have changed it
    assert not np.array_equal(P.host(), pv)


@pytest.mark.parametrize("root", [True, False])
def test_targets_that_are_computed(root):
    """Cross entropy's targets from an input that asks for a gradient, which it has from the logits."""
    xv, tv = randn(5, 7, seed=2), np.arange(5, dtype=np.float32)
    x, t = tn.input((5, 7), requires_grad=True), tn.input((5,), requires_grad=True)
    loss = x.cross_entropy(t.mul(tn.constant(np.ones(5))))
    if not root:
        loss = loss.mul(tn.constant(np.full(1, 3.0)))
    program = tn.training_program(loss)
    program.feed(x, xv)
    program.feed(t, tv)
    run_checked(program)
    ref = leaf(xv)
    (F.cross_entropy(ref, torch.arange(5)) * (1 if root else 3)).backward()
    close(program.gradient(x).host(), ref.grad, "logits")
    assert program.gradient(t) is None


def branches(trained):
    """A norm whose first use is a depthwise layer; `trained`: that layer's values are logits, else
    the weights of the rows of a loss."""
    x = tn.input((4, 8, 8, 8), requires_grad=True)
    norm, layer = nn.BatchNorm2d(8), nn.ConvNormAct(8, 8, 3, 2, 8, True)
    y = norm(x).relu()
    z = layer(y)
    fed = [tn.input((512,)) for _ in range(4)]  # actions, old, advantages, targets
    own = nn.Parameter(randn(512, 3, seed=5))
    if trained:
        side = z.reshape((128, 4)).cross_entropy(tn.constant(np.zeros(128)))
    else:
        side = own.tensor().policy_loss(*fed[:3], weights=z.reshape((512,)))
    loss = side.add(y.reshape((512, 4)).cross_entropy(fed[3]))
    return x, layer, own, fed, loss


def test_layers_of_a_branch_without_gradient():
    """The norm's launch joins the depthwise layer's where both have a gradient; where the layer's
    values only weigh rows the norm's gradient still comes from its other use."""
    joined = "batch_norm2d_relu_depthwise_conv2d_batch_norm_relu_"
    assert joined + "backward" in kinds(tn.training_program(branches(True)[-1]))
    x, layer, own, fed, loss = branches(False)
    program = tn.training_program(loss, nn.AdamW(0.1, 0.01))
    assert not any(k.startswith(joined) for k in kinds(program))
    xv = randn(4, 8, 8, 8, seed=6)
    action, old, advantage, _, _ = drawn(512, 3, 7)
    target = np.arange(512, dtype=np.float32) % 4
    for node, value in zip((x, *fed), (xv, action, old, advantage, target)):
        program.feed(node, value)
    before = [p.host() for p in layer.parameters()]
    P = leaf(own.host())
    run_checked(program)
    X = leaf(xv)
    bn = lambda v: F.batch_norm(v, None, None, training=True)  # noqa: E731
    Y = bn(X).relu()
    z = bn(F.conv2d(Y.detach(), c64(before[0]), c64(before[1]), 2, 1, groups=8)).relu()
    L = policy64(P, action, old, advantage, weights=z.reshape(-1)) + \
        F.cross_entropy(Y.reshape(512, 4), torch.tensor(target.astype(np.int64)))
    L.backward()
    close(program.value(loss).host()[0], L, "loss")
    close(program.gradient(x).host(), X.grad, "input")
    close(program.gradient(own.tensor()).host(), P.grad, "other logits")
    for p, was in zip(layer.parameters(), before):
        assert program.gradient(p.tensor()) is None and np.array_equal(p.host(), was)


def test_what_the_check_says_of_an_action():
    x, rows = tn.input((2, 3), requires_grad=True), [tn.input((2,)) for _ in range(3)]
    program = tn.training_program(x.policy_loss(*rows))
    for node in (x, *rows):
        program.feed(node, np.zeros(node.shape))
    program.feed(rows[0], np.array([1.0, 3.0]))
    program.run()
    with pytest.raises(ox.OxideError, match="action is not a class index") as err:
        program.check()
    assert err.value.kind == "InvalidShape"
    program.feed(rows[0], np.array([1.0, 2.0]))
    program.run()
    program.check()
