"""What layer norm, the gated delta rule and the policy loss refuse on the host, before any launch
(the pointers are never followed)."""

import ctypes

import pytest

import oxide_hip as ox
from test_sequence_refusals import places, refused

NAN, INF = float("nan"), float("inf")


def norm_forward(**k):
    x, r, w, b, s, y, m, q = places(8)
    a = dict(dtype=0, rows=4, columns=8, epsilon=1e-5, x=x, r=r, w=w, b=b, s=s, y=y, m=m, q=q) | k
    return ox.lib().oxh_layer_norm_forward(
        None, a["dtype"], a["rows"], a["columns"], a["epsilon"], *[a[n] for n in "xrwbsymq"])


def test_layer_norm_forward():
    x, r, w, b, s, y, m, q = places(8)
    refused(norm_forward(dtype=2), b"dtype")
    refused(norm_forward(columns=0), b"columns")
    refused(norm_forward(rows=1 << 31), b"rows")
    for eps in (-1e-6, NAN, INF):
        refused(norm_forward(epsilon=eps), b"epsilon", ox.EXECUTION)
    for name in "xwy":
        refused(norm_forward(**{name: None}), b"null")
    for name, at in (("x", x + 2), ("b", b + 1), ("m", m + 2)):
        refused(norm_forward(**{name: at}), b"aligned")
    refused(norm_forward(dtype=1, y=y + 1), b"aligned")
    for name, at in (("y", x), ("y", b), ("s", x + 4), ("s", r - 4), ("s", w), ("m", w), ("q", x)):
        refused(norm_forward(**{name: at}), b"overlaps an operand")
    for name, at in (("y", s + 4), ("m", y), ("q", m), ("m", s)):
        refused(norm_forward(**{name: at}), b"two outputs")
    assert norm_forward(rows=0, x=None, y=None) == ox.OK


def norm_backward(**k):
    g, sg, s, w, m, q, dx, dw, db, ws = places(10)
    a = dict(dtype=0, rows=4, columns=8, g=g, sg=sg, s=s, w=w, m=m, q=q, dx=dx, dw=dw, db=db,
             ws=ws, n=ox.layer_norm_backward_workspace_size(4, 8)) | k
    return ox.lib().oxh_layer_norm_backward(
        None, a["dtype"], a["rows"], a["columns"],
        *[a[n] for n in ("g", "sg", "s", "w", "m", "q", "dx", "dw", "db", "ws", "n")])


def test_layer_norm_backward():
    g, sg, s, w, m, q, dx, dw, db, ws = places(10)
    for name in ("g", "s", "w", "m", "q", "dx"):
        refused(norm_backward(**{name: None}), b"null")
    refused(norm_backward(columns=1 << 30), b"columns")
    for bad in (dict(n=0), dict(ws=None), dict(ws=ws + 4), dict(ws=None, dw=None)):
        refused(norm_backward(**bad), b"workspace")
    for name, at in (("dx", g), ("dx", s), ("dx", sg + 4), ("dw", w), ("db", m), ("ws", s)):
        refused(norm_backward(**{name: at}), b"overlaps an operand")
    for name, at in (("dw", dx), ("db", dw), ("ws", db)):
        refused(norm_backward(**{name: at}), b"two outputs")
    refused(norm_backward(db=db + 2), b"aligned")
    with pytest.raises(ox.OxideError):
        ox.layer_norm_backward_workspace_size(4, 0)


DIMS = dict(batch=2, time=100, key_heads=2, heads=4, key_dim=8, value_dim=6)


def sizes(code, dims):
    return ox._delta_plan(code, *[dims[f] for f, _ in ox.DeltaShape._fields_])


def delta_forward(**k):
    names = ("q", "k", "v", "gate", "write", "first", "n", "o", "final", "saved", "ws")
    a = dict(zip(names, places(11))) | dict(dtype=0, scale=1.0) | DIMS | k
    shape = ox.DeltaShape(*[a[f] for f, _ in ox.DeltaShape._fields_])
    _, _, ws, kept, _ = sizes(0, DIMS)
    return ox.lib().oxh_gated_delta_rule_forward(
        None, a["dtype"], ctypes.byref(shape), a["scale"], *[a[n] for n in names[:9]], a["saved"],
        a.get("kept", kept), a["ws"], a.get("bytes", ws))


BAD_DIMS = [(dict(key_dim=0), b"key_dim"), (dict(key_dim=129), b"key_dim"),
            (dict(value_dim=0), b"value_dim"), (dict(value_dim=4097), b"value_dim"),
            (dict(heads=3), b"heads"), (dict(key_heads=0), b"heads"),
            (dict(heads=65536), b"heads"), (dict(batch=65536), b"batch"),
            (dict(time=(1 << 31) - 5), b"steps"),
            (dict(batch=60000, heads=60000, time=64), b"one call"),
            (dict(batch=1, heads=64000, key_heads=64000, value_dim=4096, time=64, dtype=1,
                  kept=1 << 62),
             b"2^24"),
            (dict(batch=1, heads=64000, key_heads=64000, value_dim=256, time=64, dtype=1,
                  kept=1 << 62),
             b"workspace"), (dict(dtype=2), b"dtype")]


def test_gated_delta_rule_forward():
    q, k, v, gate, write, first, n, o, final, saved, ws = places(11)
    for bad, text in BAD_DIMS:
        refused(delta_forward(**bad), text)
    assert ox.lib().oxh_gated_delta_rule_forward(None, 0, None, 1.0, *[None] * 10, 0, None,
                                                 0) == ox.INVALID_SHAPE
    for scale in (NAN, INF):
        refused(delta_forward(scale=scale), b"scale", ox.EXECUTION)
    for name in ("q", "k", "v", "gate", "write", "o"):
        refused(delta_forward(**{name: None}), b"null")
    for bad in (dict(ws=None), dict(bytes=0), dict(ws=ws + 8)):
        refused(delta_forward(**bad), b"workspace")
    for bad in (dict(kept=0), dict(saved=saved + 8)):
        refused(delta_forward(**bad), b"saved")
    for name, at in (("q", q + 2), ("n", n + 1), ("first", first + 2), ("final", final + 2)):
        refused(delta_forward(**{name: at}), b"aligned")
    for name, at in (("o", v), ("final", k), ("saved", gate), ("ws", q), ("final", first + 4),
                     ("o", first)):
        refused(delta_forward(**{name: at}), b"overlap")
    for name, at in (("final", o), ("saved", ws), ("ws", final)):
        refused(delta_forward(**{name: at}), b"two outputs")
    assert delta_forward(batch=0, q=None) == ox.OK


def delta_backward(**k):
    names = ("g", "q", "k", "v", "gate", "write", "saved", "dfinal", "n", "dq", "dk", "dv", "dgate",
             "dwrite", "dfirst", "ws")
    a = dict(zip(names, places(16))) | dict(dtype=0, scale=1.0) | DIMS | k
    shape = ox.DeltaShape(*[a[f] for f, _ in ox.DeltaShape._fields_])
    _, _, _, kept, ws = sizes(0, DIMS)
    return ox.lib().oxh_gated_delta_rule_backward(
        None, a["dtype"], ctypes.byref(shape), a["scale"], *[a[n] for n in names[:7]],
        a.get("kept", kept), *[a[n] for n in names[7:]], a.get("bytes", ws))


def test_gated_delta_rule_backward():
    g, q, k, v, gate, write, saved, dfinal, n, dq, dk, dv, dgate, dwrite, dfirst, ws = places(16)
    for bad, text in BAD_DIMS:
        refused(delta_backward(**bad), text)
    refused(delta_backward(scale=NAN), b"scale", ox.EXECUTION)
    for name in ("g", "q", "k", "v", "gate", "write", "saved", "dq", "dk", "dv", "dgate", "dwrite",
                 "ws"):
        refused(delta_backward(**{name: None}), b"null")
    refused(delta_backward(kept=0), b"saved")
    refused(delta_backward(bytes=0), b"workspace")
    for name, at in (("g", g + 2), ("ws", ws + 8), ("saved", saved + 4), ("dfirst", dfirst + 1)):
        refused(delta_backward(**{name: at}), b"aligned")
    for name, at in (("dq", q), ("dv", g), ("dk", saved), ("dfirst", dfinal + 4), ("ws", v)):
        refused(delta_backward(**{name: at}), b"overlaps an operand")
    for name, at in (("dk", dq), ("dwrite", dgate), ("ws", dv), ("dfirst", dq)):
        refused(delta_backward(**{name: at}), b"two outputs")
    assert delta_backward(batch=0, q=None) == ox.OK


def policy(**k):
    names = ("x", "a", "old", "adv", "ref", "w", "outer", "loss", "lp", "g", "flag", "ws")
    p = dict(zip(names, places(12))) | dict(dtype=0, rows=4, classes=8, low=0.2, high=0.2, kl=0.1,
                                            n=ox.policy_loss_workspace_size(4, 8)) | k
    return ox.lib().oxh_policy_loss(None, p["dtype"], p["rows"], p["classes"], p["low"], p["high"],
                                    p["kl"], *[p[n] for n in names], p["n"])


def test_policy_loss():
    x, a, old, adv, ref, w, outer, loss, lp, g, flag, ws = places(12)
    refused(policy(dtype=3), b"dtype")
    for bad in (dict(rows=0), dict(classes=0)):
        refused(policy(**bad), b"empty")
    for bad in (dict(rows=(1 << 21) + 1), dict(classes=1 << 31)):
        refused(policy(**bad), b"too large")
    for bad in (dict(low=-0.1), dict(low=1.5), dict(low=NAN), dict(high=-1.0), dict(high=INF)):
        refused(policy(**bad), b"clip", ox.EXECUTION)
    for kl in (-1.0, NAN, INF):
        refused(policy(kl=kl), b"KL", ox.EXECUTION)
    refused(policy(ref=None), b"KL")
    for name in ("x", "a", "old", "adv"):
        refused(policy(**{name: None}), b"null")
    refused(policy(outer=None), b"upstream")
    for bad in (dict(n=0), dict(ws=None), dict(ws=ws + 8)):
        refused(policy(**bad), b"workspace")
    for name, at in (("x", x + 2), ("w", w + 1), ("loss", loss + 2), ("flag", flag + 1)):
        refused(policy(**{name: at}), b"aligned")
    for name, at in (("g", x), ("lp", old), ("loss", adv), ("ws", x), ("g", outer)):
        refused(policy(**{name: at}), b"overlaps an operand")
    for name, at in (("lp", loss), ("g", lp), ("ws", g)):
        refused(policy(**{name: at}), b"two outputs")


def test_net_builders():
    """oxh_net_* of the three, before anything is allocated."""
    import tensor

    L, h, u32 = tensor._lib(), ctypes.c_void_p(), ctypes.c_uint32
    none = tensor.NO_NODE
    assert L.oxh_net_create(ctypes.byref(h)) == ox.OK

    def leaf(*d):
        n = u32()
        shape = (ctypes.c_uint64 * len(d))(*d)
        assert L.oxh_net_input(h, len(d), shape, 0, ctypes.byref(n)) == ox.OK
        return n.value

    n = u32()
    out = ctypes.byref(n)
    x, w, short = leaf(2, 3, 8), leaf(8), leaf(7)
    for a, b, c in ((x, short, short), (x, w, short), (x, w, x), (x, 99, w), (99, w, w),
                    (x, w, 99)):
        assert L.oxh_net_layer_norm(h, a, b, c, 1e-5, out) == ox.INVALID_SHAPE
    for eps in (-1.0, NAN, INF):
        refused(L.oxh_net_layer_norm(h, x, w, w, eps, out), b"epsilon", ox.EXECUTION)
    assert L.oxh_net_layer_norm(h, x, w, w, 0.0, out) == ox.OK

    k, v, g = leaf(2, 5, 2, 8), leaf(2, 5, 4, 6), leaf(2, 5, 4)

    def rule(query=k, key=k, value=v, gate=g, write=g, scale=1.0):
        return L.oxh_net_gated_delta_rule(h, query, key, value, gate, write, scale, out)

    for bad in (dict(query=leaf(2, 5, 2, 7)), dict(value=leaf(2, 4, 4, 6)), dict(value=x),
                dict(value=leaf(3, 5, 4, 6)), dict(gate=leaf(2, 5, 2)), dict(write=x),
                dict(key=99), dict(write=99)):
        assert rule(**bad) == ox.INVALID_SHAPE, bad
    odd = dict(value=leaf(2, 5, 3, 6), gate=leaf(2, 5, 3))
    assert rule(**odd, write=odd["gate"]) == ox.INVALID_SHAPE  # 3 heads of 2 key heads
    wide = leaf(2, 5, 2, 129)
    refused(rule(query=wide, key=wide), b"key_dim")
    refused(rule(scale=NAN), b"scale", ox.EXECUTION)
    assert rule() == ox.OK
    rank, dims = u32(), (ctypes.c_uint64 * 4)()
    assert L.oxh_net_node_shape(h, n.value, ctypes.byref(rank), dims) == ox.OK
    assert rank.value == 4 and list(dims) == [2, 5, 4, 6]

    logits, row = leaf(6, 8), leaf(6)

    def policy(a=logits, b=row, c=row, d=row, reference=none, weights=none, low=0.2, high=0.2,
               kl=0.0):
        return L.oxh_net_policy_loss(h, a, b, c, d, reference, weights, low, high, kl, out)

    for bad in (dict(a=x), dict(b=short), dict(c=x), dict(d=99), dict(weights=short),
                dict(weights=99), dict(reference=none - 1), dict(kl=0.1)):
        assert policy(**bad) == ox.INVALID_SHAPE, bad
    for bad in (dict(low=-0.1), dict(low=1.1), dict(high=INF), dict(kl=-1.0), dict(kl=NAN)):
        assert policy(**bad) == ox.EXECUTION, bad
    assert policy(reference=row, weights=row, kl=0.1) == ox.OK
    assert policy(reference=row) == ox.OK
    assert L.oxh_net_layer_norm(None, x, w, w, 0.0, out) == ox.INVALID_SHAPE
    assert L.oxh_net_policy_loss(h, logits, row, row, row, none, none, 0.2, 0.2, 0.0,
                                 None) == ox.INVALID_SHAPE
    assert L.oxh_net_destroy(h) == ox.OK


def test_tensor_methods():
    """The Python graph's own checks."""
    import nn
    import tensor as tn

    i = tn.input
    for call in (lambda: i((2, 3)).layer_norm(i((2,)), i((2,))),
                 lambda: i((2, 3)).layer_norm(i((3,)), i((2,))),
                 lambda: i((2, 5, 2, 8)).gated_delta_rule(i((2, 5, 2, 7)), i((2, 5, 2, 3)),
                                                          i((2, 5, 2)), i((2, 5, 2))),
                 lambda: i((2, 5, 2, 8)).gated_delta_rule(i((2, 5, 2, 8)), i((2, 5, 3, 3)),
                                                          i((2, 5, 3)), i((2, 5, 3))),
                 lambda: i((2, 5, 2, 8)).gated_delta_rule(i((2, 5, 2, 8)), i((2, 5, 2, 3)),
                                                          i((2, 5, 2)), i((2, 5, 1))),
                 lambda: i((2, 5, 2, 129)).gated_delta_rule(i((2, 5, 2, 129)), i((2, 5, 2, 3)),
                                                            i((2, 5, 2)), i((2, 5, 2))),
                 lambda: i((4, 3)).policy_loss(i((4,)), i((4,)), i((3,))),
                 lambda: i((4, 3)).policy_loss(i((4,)), i((4,)), i((4,)), kl=0.1),
                 lambda: i((4, 3)).policy_loss(i((4,)), i((4,)), i((4,)), clip=0.2),
                 lambda: nn.LayerNorm(0), lambda: nn.DeltaRuleBlock(10, heads=4),
                 lambda: nn.DeltaRuleBlock(12, heads=4, key_heads=3)):
        with pytest.raises(ox.OxideError) as err:
            call()
        assert err.value.kind == "InvalidShape"
    for call in (lambda: i((2, 3)).layer_norm(i((3,)), i((3,)), NAN),
                 lambda: i((2, 5, 2, 8)).gated_delta_rule(i((2, 5, 2, 8)), i((2, 5, 2, 3)),
                                                          i((2, 5, 2)), i((2, 5, 2)), INF),
                 lambda: i((4, 3)).policy_loss(i((4,)), i((4,)), i((4,)), clip=(1.5, 0.2)),
                 lambda: i((4, 3)).policy_loss(i((4,)), i((4,)), i((4,)), kl=-0.1)):
        with pytest.raises(ox.OxideError) as err:
            call()
        assert err.value.kind == "Execution"
