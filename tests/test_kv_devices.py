"""The attention-side ops on several GPUs, on the host: stand-ins for tensors of two devices and for the library record on
which device each call is made.  Tensors of one call must share a device; the call is made on it, whatever is current."""

import contextlib

import pytest
import torch

from gguf_onnx_ops_b200 import ops


EMPTY = torch.empty  # (the tests replace it)


class Fake:
    """A tensor's host side: shape, type and device number."""

    is_cuda = True

    def __init__(self, *shape, dtype=torch.bfloat16, dev=0):
        self.t, self.dev = EMPTY(*shape, dtype=dtype, device="meta"), dev
        self.dtype, self.shape, self.device = dtype, self.t.shape, torch.device("cuda", dev)

    def __getattr__(self, name):  # dim, stride, numel, is_contiguous
        return getattr(self.t, name)

    def get_device(self):
        return self.dev

    def data_ptr(self):
        return 0x10000

    def new_empty(self, shape):
        return Fake(*shape, dtype=self.dtype, dev=self.dev)


class Library:
    """Every entry point notes the device that is current and succeeds."""

    def __init__(self, current):
        self.current, self.calls = current, []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, self.current[0]))
            return 0

        return call


@pytest.fixture
def fakes(monkeypatch):
    current = [0]

    @contextlib.contextmanager
    def device(dev):
        was, current[0] = current[0], dev if isinstance(dev, int) else dev.index
        yield
        current[0] = was

    lib = Library(current)
    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch, "empty", lambda *shape, dtype=None, device=None: Fake(*shape, dtype=dtype, dev=current[0]))
    monkeypatch.setattr(torch, "zeros", lambda *shape, dtype=None, device=None: Fake(*shape, dtype=dtype, dev=current[0]))
    monkeypatch.setattr(torch, "empty_like", lambda t, memory_format=None: Fake(*t.shape, dtype=t.dtype, dev=t.dev))
    monkeypatch.setattr(ops, "load", lambda: lib)
    monkeypatch.setattr(ops, "_raw_stream", lambda t: 0)
    monkeypatch.setattr(ops, "_kv_workspaces", {})
    return lib



def arguments(devs):
    """(op, calls of it) with the i-th tensor of every op on devs[i % len(devs)]."""
    d = lambda i: devs[i % len(devs)]  # noqa: E731
    i32, f32 = torch.int32, torch.float32
    cache = ops.KvCache(Fake(4, 2, 16, 64, dtype=torch.int8, dev=d(0)), Fake(4, 2, 16, 64, dtype=torch.int8, dev=d(0)),
                        Fake(4, 2, dtype=f32, dev=d(0)), Fake(4, 2, dtype=f32, dev=d(0)))
    rows = lambda i, heads=2: Fake(1, 1, heads, 64, dev=d(i))  # noqa: E731
    table, lens = Fake(1, 2, dtype=i32, dev=d(0)), Fake(1, dtype=i32, dev=d(0))
    return [
        ("gguf_qk_norm_rope", lambda: ops.QkNormRope(Fake(2, 6 * 64, dev=d(0)), Fake(64, dtype=f32, dev=d(1)), None,
                                                     Fake(8, 32, dtype=f32, dev=d(0)), Fake(8, 32, dtype=f32, dev=d(0)),
                                                     Fake(2, dtype=i32, dev=d(0)), heads=4, kv_heads=1)),
        ("gguf_kv_cache_write", lambda: ops.KvCacheWrite(rows(0), rows(1), cache, table, lens)),
        ("gguf_kv_cache_read", lambda: ops.KvCacheRead(cache, table, Fake(1, dtype=i32, dev=d(1)), rows=3)),
        ("gguf_kv_cache_attention", lambda: ops.KvCacheAttention(rows(1, 4), cache, table, lens)),
        ("gguf_draft_verify", lambda: ops.DraftVerify(Fake(1, 2, 8, dtype=f32, dev=d(0)), None, Fake(1, 1, dtype=i32, dev=d(0)),
                                                      Fake(1, 1, dtype=f32, dev=d(1)), Fake(1, dtype=f32, dev=d(0)))),
    ]


@pytest.mark.parametrize("dev", [0, 1])
def test_calls_are_made_on_the_tensors_device(fakes, dev):
    for name, call in arguments([dev]):
        fakes.calls.clear()
        call()
        assert fakes.calls[-1] == (name, dev) and {c[1] for c in fakes.calls} == {dev}
    assert ops._current_device() == 0


@pytest.mark.parametrize("devs", [[0, 1], [1, 0]])
def test_tensors_of_two_devices_are_refused(fakes, devs):
    for _, call in arguments(devs):
        with pytest.raises(ValueError, match="one device"):
            call()
    assert not fakes.calls
