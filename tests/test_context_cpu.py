"""ops.context() binds the shared context to torch's current stream by every call, also when a
caller has set another stream on the handle in between, and leaves the current device as it was. A
stand-in for the library records the calls, so this needs no GPU."""
import contextlib
import types

import pytest


class _Library:
    def __init__(self):
        self.stream = None
        self.device = 0                  # the thread's current device
        self.created = 0

    def tb_ctx_create(self, device, stream, out):
        self.created += 1
        self.device = device             # as the library does, for good
        self.stream = stream.value
        out._obj.value = 0x1000 + device
        return 0

    def tb_ctx_set_stream(self, handle, stream):
        assert handle.value & ~15 == 0x1000
        self.stream = getattr(stream, "value", stream)
        return 0

    def tb_ctx_last_error(self, handle):
        return b""


@pytest.fixture()
def bound(tb, monkeypatch):
    """(ops, the library, a way to change torch's current stream), no context yet."""
    import torch
    from trellis_cpp_b200 import _lib, ops
    lib, now = _Library(), types.SimpleNamespace(cuda_stream=100)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_ctxs", {})
    monkeypatch.setattr(ops, "_raw_stream", lambda index: now.cuda_stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: now)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: lib.device)

    @contextlib.contextmanager
    def device(index):
        before, lib.device = lib.device, index
        yield
        lib.device = before

    monkeypatch.setattr(torch.cuda, "device", device)
    return ops, lib, now


def test_follows_torch(bound):
    ops, lib, now = bound
    ops.context()
    assert lib.stream == 100 and lib.created == 1
    now.cuda_stream = 200
    for device in (None, 0, "cuda", "cuda:0"):
        ops.context(device)
    assert lib.stream == 200 and lib.created == 1


def test_a_stream_set_on_the_handle_does_not_stay(bound):
    import ctypes
    ops, lib, now = bound
    h = ops.context(0)
    lib.tb_ctx_set_stream(h, ctypes.c_void_p(300))
    assert lib.stream == 300
    ops.context(0)
    assert lib.stream == 100


def test_a_first_call_on_another_device_leaves_the_current_one(bound):
    ops, lib, now = bound
    ops.context(3)
    assert lib.created == 1 and lib.device == 0
    ops.context(3)
    ops.context()
    assert lib.created == 2 and lib.device == 0
