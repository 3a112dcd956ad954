"""What the sequence operators refuse on the host, before any launch (the pointers are never
followed)."""

import ctypes

import numpy as np
import pytest

import oxide_hip as ox

BASE = 1 << 30
STEP = 1 << 24


def places(n):
    return [BASE + i * STEP for i in range(n)]


def refused(status, text, kind=ox.INVALID_SHAPE):
    assert status == kind, (status, ox.lib().oxh_last_error())
    assert text in ox.lib().oxh_last_error(), ox.lib().oxh_last_error()


def norm_forward(**k):
    x, r, w, s, y, q = places(6)
    a = dict(dtype=0, rows=4, columns=8, epsilon=1e-6, x=x, r=r, w=w, s=s, y=y, q=q) | k
    return ox.lib().oxh_rms_norm_forward(None, a["dtype"], a["rows"], a["columns"], a["epsilon"],
                                         a["x"], a["r"], a["w"], a["s"], a["y"], a["q"])


def test_rms_norm_forward():
    x, r, w, s, y, q = places(6)
    refused(norm_forward(dtype=2), b"dtype")
    refused(norm_forward(columns=0), b"columns")
    refused(norm_forward(rows=1 << 31), b"rows")
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(norm_forward(epsilon=eps), b"epsilon", ox.EXECUTION)
    for name in ("x", "w", "y"):
        refused(norm_forward(**{name: None}), b"null")
    refused(norm_forward(x=x + 2), b"aligned")
    refused(norm_forward(dtype=1, y=y + 1), b"aligned")
    refused(norm_forward(y=x), b"overlaps")
    refused(norm_forward(y=s + 4), b"overlaps")
    refused(norm_forward(s=x + 4), b"partially overlaps")
    refused(norm_forward(s=r - 4), b"partially overlaps")
    refused(norm_forward(q=y), b"overlaps")
    assert norm_forward(rows=0, x=None, y=None) == ox.OK


def norm_backward(**k):
    g, sg, s, w, q, dx, dw, ws = places(8)
    a = dict(dtype=0, rows=4, columns=8, g=g, sg=sg, s=s, w=w, q=q, dx=dx, dw=dw, ws=ws,
             n=ox.rms_norm_backward_workspace_size(4, 8)) | k
    return ox.lib().oxh_rms_norm_backward(None, a["dtype"], a["rows"], a["columns"], a["g"],
                                          a["sg"], a["s"], a["w"], a["q"], a["dx"], a["dw"],
                                          a["ws"], a["n"])


def test_rms_norm_backward():
    g, sg, s, w, q, dx, dw, ws = places(8)
    for name in ("g", "s", "w", "q", "dx"):
        refused(norm_backward(**{name: None}), b"null")
    refused(norm_backward(n=0), b"workspace")
    refused(norm_backward(ws=None), b"workspace")
    refused(norm_backward(ws=ws + 4), b"workspace")
    refused(norm_backward(dx=g), b"overlaps")
    refused(norm_backward(dx=s), b"overlaps")
    refused(norm_backward(dx=sg + 4), b"overlaps")
    refused(norm_backward(dw=w), b"overlaps")
    refused(norm_backward(dw=dx), b"overlap")
    refused(norm_backward(ws=s), b"overlaps")
    with pytest.raises(ox.OxideError):
        ox.rms_norm_backward_workspace_size(4, 0)


def scan_forward(**k):
    u, g, st, n, h, f, ws = places(7)
    a = dict(dtype=0, batch=2, time=2000, channels=8, u=u, g=g, st=st, n=n, h=h, f=f, ws=ws,
             bytes=ox.gated_recurrence_workspace_size(2, 2000, 8)) | k
    return ox.lib().oxh_gated_recurrence_forward(
        None, a["dtype"], a["batch"], a["time"], a["channels"], a["u"], a["g"], a["st"], a["n"],
        a["h"], a["f"], a["ws"], a["bytes"])


def test_gated_recurrence_forward():
    u, g, st, n, h, f, ws = places(7)
    refused(scan_forward(dtype=7), b"dtype")
    refused(scan_forward(batch=65536), b"batch")
    refused(scan_forward(time=1 << 31), b"time")
    refused(scan_forward(batch=65535, time=(1 << 31) - 1, channels=(1 << 31) - 1), b"overflow")
    for name in ("u", "g", "h"):
        refused(scan_forward(**{name: None}), b"null")
    refused(scan_forward(u=u + 2), b"aligned")
    refused(scan_forward(n=n + 2), b"aligned")
    refused(scan_forward(bytes=0), b"workspace")
    refused(scan_forward(h=u), b"overlaps")
    refused(scan_forward(f=st + 4), b"overlaps")
    refused(scan_forward(f=h), b"overlap")
    refused(scan_forward(ws=g), b"overlap")
    assert scan_forward(batch=0, u=None) == ox.OK
    assert scan_forward(channels=0, u=None) == ox.OK


def scan_backward(**k):
    dh, u, g, h, st, df, n, du, dg, ds, ws = places(11)
    a = dict(dtype=0, dh=dh, u=u, g=g, h=h, st=st, df=df, n=n, du=du, dg=dg, ds=ds, ws=ws,
             bytes=ox.gated_recurrence_workspace_size(2, 2000, 8)) | k
    return ox.lib().oxh_gated_recurrence_backward(
        None, a["dtype"], 2, 2000, 8, a["dh"], a["u"], a["g"], a["h"], a["st"], a["df"], a["n"],
        a["du"], a["dg"], a["ds"], a["ws"], a["bytes"])


def test_gated_recurrence_backward():
    dh, u, g, h, st, df, n, du, dg, ds, ws = places(11)
    for name in ("dh", "u", "g", "h", "du", "dg"):
        refused(scan_backward(**{name: None}), b"null")
    refused(scan_backward(dtype=1, dg=dg + 1), b"aligned")
    refused(scan_backward(ws=None), b"workspace")
    for bad in (dh, u, g, h):
        refused(scan_backward(du=bad), b"overlaps")
        refused(scan_backward(dg=bad + 4), b"overlaps")
    refused(scan_backward(du=dg), b"overlap")
    refused(scan_backward(ds=df + 4), b"overlaps")
    refused(scan_backward(ds=st), b"overlaps")


def test_orthogonalize():
    x, y, ws = places(3)
    lib, need = ox.lib(), ox.orthogonalize_workspace_size(2, 300, 400)

    def call(count=2, rows=300, columns=400, rounds=5, eps=1e-7, x=x, y=y, ws=ws, n=need):
        return lib.oxh_orthogonalize(None, count, rows, columns, rounds, eps, x, y, ws, n)

    refused(call(rows=0), b"empty")
    refused(call(rows=65537, columns=65537), b"too large")
    refused(call(rows=(1 << 20) + 1), b"too large")
    refused(call(rows=8192, columns=(1 << 20)), b"too large")
    refused(call(rounds=0), b"rounds")
    refused(call(rounds=65), b"rounds")
    for eps in (0.0, -1.0, float("nan")):
        refused(call(eps=eps), b"epsilon", ox.EXECUTION)
    refused(call(x=None), b"null")
    refused(call(y=y + 2), b"misaligned")
    refused(call(n=need - 1), b"workspace")
    refused(call(ws=ws + 8), b"workspace")
    refused(call(y=x), b"overlap")
    refused(call(ws=x), b"overlap")
    assert call(count=0, x=None, ws=None) == ox.OK


def test_muon():
    p, g, m, ws = places(4)
    lib = ox.lib()

    def call(entries=((p, g, m, 300, 400),), lr=0.1, wd=0.0, mu=0.9, eps=1e-7, rounds=5, ws=ws,
             n=None):
        table = (ox.MuonTensor * len(entries))(*[ox.MuonTensor(*e) for e in entries])
        if n is None:
            out = ctypes.c_uint64()
            if lib.oxh_muon_workspace_size(table, len(entries), ctypes.byref(out)) != ox.OK:
                return ox.INVALID_SHAPE
            n = out.value
        return lib.oxh_muon_multi_tensor(None, lr, wd, mu, 1, eps, rounds, table, len(entries), ws,
                                         n)

    for k in ({"lr": float("nan")}, {"wd": float("inf")}, {"mu": float("nan")}):
        refused(call(**k), b"finite")
    refused(call(eps=0.0), b"epsilon", ox.EXECUTION)
    refused(call(rounds=0), b"rounds")
    refused(call(((p, g, m, 0, 400),)), b"empty")
    refused(call(((p, g, None, 300, 400),)), b"null")
    refused(call(((p + 1, g, m, 300, 400),)), b"misaligned")
    refused(call(n=16), b"workspace")
    refused(call(((p, p, m, 300, 400),)), b"overlaps")
    refused(call(((p, g, p + 400, 300, 400),)), b"overlaps")
    refused(call(((p, g, m, 300, 400), (p + 4000, g + 500000, m + 500000, 300, 400))), b"overlaps")
    refused(call(ws=m), b"overlaps")
    assert call((), ws=None) == ox.OK


def test_front_end_checks_shapes():
    """The Python front end refuses before it reaches the library."""
    torch = pytest.importorskip("torch")
    z = torch.zeros
    with pytest.raises(ox.OxideError):
        ox.muon_table([(z(3), z(3), z(3))])
    with pytest.raises(ox.OxideError):
        ox.muon_table([(z(3, 4), z(3, 5), z(3, 4))])
    with pytest.raises(ox.OxideError):  # host tensors
        ox._activations((z(2, 3),), (2, 3), "rms_norm")
    assert np.isfinite(ox.gated_recurrence_workspace_size(1, 1, 1))


def test_net_builders():
    """oxh_net_* of the sequence layers and of the optimizer, before anything is allocated."""
    import tensor

    L, h, u32 = tensor._lib(), ctypes.c_void_p(), ctypes.c_uint32
    shape = lambda *d: (ctypes.c_uint64 * len(d))(*d)  # noqa: E731
    assert L.oxh_net_create(ctypes.byref(h)) == ox.OK

    def leaf(*d, parameter=False):
        n = u32()
        if parameter:
            st = L.oxh_net_parameter(h, len(d), shape(*d), BASE, ctypes.byref(n))
        else:
            st = L.oxh_net_input(h, len(d), shape(*d), 0, ctypes.byref(n))
        assert st == ox.OK
        return n.value

    x, other, flat = leaf(2, 3, 8), leaf(2, 4, 8), leaf(6, 8)
    w, short, square = leaf(8, parameter=True), leaf(7, parameter=True), leaf(8, 8, parameter=True)
    n = u32()
    out = ctypes.byref(n)
    for a, b in ((x, short), (x, square), (x, 99), (99, w)):
        assert L.oxh_net_rms_norm(h, a, b, 1e-6, out) == ox.INVALID_SHAPE
    for eps in (-1.0, float("nan"), float("inf")):
        refused(L.oxh_net_rms_norm(h, x, w, eps, out), b"epsilon", ox.EXECUTION)
    for a, b in ((x, other), (flat, flat), (x, 99), (99, x)):
        assert L.oxh_net_gated_recurrence(h, a, b, out) == ox.INVALID_SHAPE
    assert L.oxh_net_rms_norm(h, x, w, 0.0, out) == ox.OK
    assert L.oxh_net_gated_recurrence(h, n.value, x, out) == ox.OK
    rank, dims = u32(), (ctypes.c_uint64 * 4)()
    assert L.oxh_net_node_shape(h, n.value, ctypes.byref(rank), dims) == ox.OK
    assert rank.value == 3 and list(dims)[:3] == [2, 3, 8]
    assert L.oxh_net_rms_norm(None, x, w, 0.0, out) == ox.INVALID_SHAPE
    assert L.oxh_net_gated_recurrence(h, x, x, None) == ox.INVALID_SHAPE

    targets = leaf(6)
    assert L.oxh_net_cross_entropy(h, flat, targets, out) == ox.OK
    loss, program = n.value, ctypes.c_void_p()

    def muon(nodes=(square,), root=loss, config=True, **k):
        a = dict(learning_rate=0.1, weight_decay=0.0, momentum=0.9, epsilon=1e-7, nesterov=1,
                 rounds=5) | k
        c = tensor.MuonConfig(**a)
        return L.oxh_net_training_program_muon(
            h, root, ctypes.byref(c) if config else None, (u32 * len(nodes))(*nodes), len(nodes),
            None, ctypes.byref(program))

    refused(muon(root=x), b"scalar", ox.EXECUTION)
    refused(muon(config=False), b"null")
    for k in (dict(learning_rate=0.0), dict(learning_rate=float("nan")), dict(weight_decay=-0.1),
              dict(momentum=1.0), dict(momentum=float("nan")), dict(epsilon=0.0),
              dict(epsilon=float("inf"))):
        assert muon(**k) == ox.EXECUTION, k
    refused(muon(rounds=0), b"rounds")
    refused(muon(rounds=65), b"rounds")
    for node in (w, x, 99):
        assert muon((node,)) == ox.INVALID_SHAPE
    assert program.value is None
    assert L.oxh_net_destroy(h) == ox.OK


@pytest.mark.parametrize("dtype", [0, 1])
def test_gated_recurrence_of_more_than_a_launch_takes(dtype):
    """2^32 threads and more, which a launch cannot number: 256 channels a wave for a few steps, 64
    a block of 8 waves for more.  Refused before any launch, where blocks alone still fit 31 bits."""
    at = [i << 46 for i in range(1, 8)]

    def forward(batch, time, channels):
        need = ox.gated_recurrence_workspace_size(batch, time, channels)
        return ox.lib().oxh_gated_recurrence_forward(None, dtype, batch, time, channels, at[0],
                                                     at[1], None, None, at[2], None, at[3], need)

    def backward(batch, time, channels):
        need = ox.gated_recurrence_workspace_size(batch, time, channels)
        return ox.lib().oxh_gated_recurrence_backward(None, dtype, batch, time, channels, *at[:4],
                                                      None, None, None, at[4], at[5], None, at[6],
                                                      need)

    for call in (forward, backward):
        for batch, time, channels in ((65535, 1, 1 << 19), (1 << 12, 8, 1 << 22),
                                      (1, 100, 1 << 29), (60000, 65, 9000)):
            refused(call(batch, time, channels), b"too many rows and channels")


def test_stream_is_capturing():
    out = ctypes.c_int(7)
    assert ox.lib().oxh_stream_is_capturing(None, ctypes.byref(out)) == ox.OK and out.value == 0
    refused(ox.lib().oxh_stream_is_capturing(None, None), b"null")
