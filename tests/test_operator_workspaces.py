"""Whose device memory a call works in: one workspace per device, stream and host thread (CPU only, a library that is not there)."""
import importlib
import threading

import pytest


class Library:
    """The few entry points that a workspace takes, of a process with several devices."""

    def __init__(self):
        self.current = threading.local()
        self.lies_on = {}
        self.synced = []
        self.freed = []
        self.lock = threading.Lock()

    def device(self):
        return getattr(self.current, "index", 0)

    def call(self, name, *args):
        if name == "sb_set_device":
            self.current.index = args[0]
        elif name == "sb_get_device":
            args[0]._obj.value = self.device()
        elif name == "sb_malloc":
            with self.lock:
                at = 0x100000 * (len(self.lies_on) + 1)
                self.lies_on[at] = self.device()
            args[0]._obj.value = at
        elif name == "sb_stream_sync":
            self.synced.append(args[0])
        else:
            assert name == "sb_free", name
            self.freed.append(args[0])


@pytest.fixture
def library(sb, monkeypatch):
    lib = Library()
    from spiral_b200 import _lib, device
    monkeypatch.setattr(_lib, "call", lib.call)
    monkeypatch.setattr(device, "_WORKSPACES", type(device._WORKSPACES)())    # none of other tests, and none left to them
    return lib


def test_of_a_device(sb, library):
    """The default stream has one handle on all devices; its workspaces lie where the kernels run."""
    from spiral_b200.device import stream_workspace
    held = []
    for device in (0, 1, 0, 1):
        sb.set_device(device)
        held.append(stream_workspace(100000, None))
        assert library.lies_on[held[-1].ptr] == device
    assert held[0] is held[2] and held[1] is held[3]


def test_of_a_stream(sb, library):
    from spiral_b200.device import stream_workspace
    sb.set_device(2)
    a, b = stream_workspace(100000, 0x71), stream_workspace(100000, 0x72)
    assert a.ptr != b.ptr and stream_workspace(5, 0x71) is a and not library.synced
    grown = stream_workspace(200000, 0x71)                             # the old one may be in use: a wait for its stream
    assert grown.nbytes >= 200000 and library.synced == [0x71] and stream_workspace(5, 0x72) is b


def test_of_a_host_thread(sb, library):
    """The launches of one call may have those of another thread between them."""
    from spiral_b200.device import stream_workspace
    mine, others = stream_workspace(100000, None), []
    meet = threading.Barrier(3)                                        # alive together: numbers of threads come again

    def work():
        others.append(stream_workspace(100000, None))
        meet.wait()
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len({w.ptr for w in others}) == 3
    assert mine.ptr not in {w.ptr for w in others} and stream_workspace(100000, None) is mine


def test_outlives_its_thread(sb, library):
    """What a thread launched, or captured in a graph, may run after it has ended."""
    from spiral_b200.device import stream_workspace
    at = []
    thread = threading.Thread(target=lambda: at.append(stream_workspace(100000, 0x71).ptr))
    thread.start()
    thread.join()
    assert not library.freed and at[0] in library.lies_on


def test_split_operands_of_the_fp32_class(sb, library, monkeypatch):
    """matmul in the fp32 class keeps its split operands under the same rule."""
    matmul = importlib.import_module("spiral_b200.matmul")             # the module, not the function of its name

    def call(name, *args):
        if name == "sb_matmul_f32_workspace_bytes":
            args[3]._obj.value = 8 * (args[0] + args[1]) * args[2] + 1024
        else:
            library.call(name, *args)
    monkeypatch.setattr(matmul._lib, "call", call)
    monkeypatch.setattr(matmul, "_F32X3_WORKSPACES", type(matmul._F32X3_WORKSPACES)())
    held, others = [], []
    for device in (0, 1, 0):
        sb.set_device(device)
        held.append(matmul._f32x3_workspace(64, 64, 64, None))
        assert library.lies_on[held[-1].ptr] == device
    assert held[0] is held[2] and matmul._f32x3_workspace(8, 8, 8, None) is held[0]
    grown = matmul._f32x3_workspace(64, 64, 128, None)
    assert grown.nbytes >= 8 * 128 * 128 and library.synced == [None]
    thread = threading.Thread(target=lambda: others.append(matmul._f32x3_workspace(64, 64, 64, None)))
    thread.start()
    thread.join()
    assert others[0].ptr not in {w.ptr for w in held} | {grown.ptr}
