"""Host threads that share a stream take turns at its scratch: between a call's choice of scratch and
its last launch no other thread's call comes, as its launches would write what this one's later ones
read.  The library's entries are stood in for, so no GPU is needed."""

import threading
import time

import pytest
import torch

import oxide_hip as ox


class Device:
    """What the launchers ask of a device tensor."""

    is_cuda, device = True, "cuda:0"

    def __init__(self, *shape, dtype=torch.float32):
        self.shape, self.dtype = torch.Size(shape), dtype

    def numel(self):
        return self.shape.numel()

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 30


class Library:
    """The library with its launching entries replaced by one that takes its time and notes whether
    another began meanwhile."""

    ENTRIES = {"oxh_rms_norm_backward", "oxh_gated_recurrence_forward",
               "oxh_gated_recurrence_backward", "oxh_orthogonalize", "oxh_muon_multi_tensor"}

    def __init__(self, real):
        self.real, self.inside, self.calls, self.met = real, 0, 0, False

    def __getattr__(self, name):
        return self.launch if name in self.ENTRIES else getattr(self.real, name)

    def launch(self, *arguments):
        self.inside += 1
        self.calls += 1
        self.met |= self.inside > 1
        time.sleep(0.01)
        self.met |= self.inside > 1
        self.inside -= 1
        return ox.OK


def recurrence(m):
    x = Device(1, 3000, 24)
    m.gated_recurrence_forward(x, x, x, stream=0)


def recurrence_backward(m):
    x = Device(1, 3000, 24)
    m.gated_recurrence_backward(x, x, x, x, x, x, stream=0)


def norm_backward(m):
    x = Device(600, 700)
    m.rms_norm_backward(x, x, Device(700), Device(600), x, Device(700), stream=0)


def orthogonalize(m):
    m.orthogonalize(Device(300, 310), Device(300, 310), stream=0)


def muon(m):
    m.muon(0.1, 0.0, 0.9, [(Device(300, 310),) * 3], stream=0)


@pytest.mark.parametrize("call", [recurrence, recurrence_backward, norm_backward, orthogonalize,
                                  muon])
def test_threads_on_one_stream_take_turns(monkeypatch, call):
    library = Library(ox.lib())
    monkeypatch.setattr(ox, "lib", lambda: library)
    monkeypatch.setattr(ox.StreamWorkspaces, "_allocate",
                        staticmethod(lambda nbytes, stream: torch.empty(nbytes, dtype=torch.uint8)))
    module = object.__new__(ox.LoadedModule)
    module._sequence_ws = ox.StreamWorkspaces()
    errors = []

    def run():
        try:
            for _ in range(3):
                call(module)
        except Exception as error:  # noqa: BLE001 - reported below
            errors.append(error)

    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and library.calls == 12 and not library.met


def test_types_are_known_before_they_are_said_to_be(monkeypatch):
    """A thread whose first call comes while another's fills the table of types: what it reads as
    ready is whole."""
    class Table(dict):
        def update(self, *arguments):
            began.set()
            late.wait(0.5)
            super().update(*arguments)

    began, late, seen = threading.Event(), threading.Event(), []
    monkeypatch.setattr(ox, "_codes", Table())
    monkeypatch.setattr(ox, "_float32", None)
    monkeypatch.setattr(ox, "_int32", None)

    def second():
        began.wait(5)
        x = Device(2, 3)
        try:
            seen.append(ox._activations((x,), x.shape, "rms_norm")[0])
        except ox.OxideError as error:
            seen.append(error)
        late.set()

    thread = threading.Thread(target=second)
    thread.start()
    assert ox._activations((Device(2, 3),), torch.Size((2, 3)), "rms_norm")[0] == ox.F32
    thread.join()
    assert seen == [ox.F32]
