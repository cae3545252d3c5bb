"""ops.context() binds the shared context to torch's current stream by every call, also when a
caller has set another stream on the handle in between. A stand-in for the library records the
calls, so this needs no GPU."""
import types

import pytest


class _Library:
    def __init__(self):
        self.stream = None
        self.created = 0

    def tb_ctx_create(self, device, stream, out):
        self.created += 1
        self.stream = stream.value
        out._obj.value = 0x1000 + device
        return 0

    def tb_ctx_set_stream(self, handle, stream):
        assert handle.value == 0x1000
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
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
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
