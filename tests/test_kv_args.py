"""The attention-side entry points of the C ABI refuse bad arguments before any CUDA call (fake pointers, no GPU)."""

import ctypes

import pytest

from gguf_onnx_ops_b200 import _lib

FAKE = 0x10000


def cache(pages=8, kv_heads=2, page=64, head_dim=128, k=FAKE, scale=FAKE):
    return _lib.GgufKvCache(k, FAKE, scale, FAKE, pages, kv_heads, page, head_dim)


def refused(lib, fn, args, msg):
    assert getattr(lib, fn)(*args) == _lib.GGUF_ERR_INVALID_ARGUMENT
    assert msg in lib.gguf_last_error().decode()


ROPE = dict(x=FAKE, gq=FAKE, gk=FAKE, cos=FAKE, sin=FAKE, pos=FAKE, q=FAKE, k=FAKE, T=4, stride=1024, heads=4, kv=2, D=128,
            rot=128, max_pos=64, eps=1e-6, inter=0, stream=None)


@pytest.mark.parametrize("change,msg", [
    (dict(D=129), "head_dim"), (dict(D=264), "head_dim"), (dict(rot=136), "rotated width"), (dict(rot=12), "rotated width"),
    (dict(T=-1), "number of tokens"), (dict(T=1 << 31), "number of tokens"), (dict(heads=0), "number of heads"),
    (dict(stride=1023), "multiples of 4"), (dict(x=None), "null"), (dict(cos=None), "null"), (dict(x=FAKE + 4), "aligned"),
    (dict(q=FAKE + 8), "aligned"), (dict(gq=FAKE + 4), "aligned"), (dict(max_pos=0), "table rows")])
def test_rope(lib, change, msg):
    refused(lib, "gguf_qk_norm_rope", tuple({**ROPE, **change}.values()), "QkNormRope")
    assert msg in lib.gguf_last_error().decode()


def test_rope_empty(lib):
    assert lib.gguf_qk_norm_rope(*{**ROPE, "T": 0}.values()) == _lib.GGUF_OK


@pytest.mark.parametrize("c,cols,B,msg", [
    (dict(head_dim=80), 4, 2, "head_dim"), (dict(page=48), 4, 2, "page"), (dict(page=8), 4, 2, "page"),
    (dict(page=512), 4, 2, "page"), (dict(kv_heads=0), 4, 2, "kv heads"), (dict(pages=0), 4, 2, "pages"),
    (dict(pages=1 << 31), 4, 2, "pages"), (dict(k=None), 4, 2, "null"), (dict(scale=None), 4, 2, "null"),
    (dict(k=FAKE + 8), 4, 2, "aligned"), ({}, 0, 2, "page table"), ({}, 1 << 26, 2, "page table"), ({}, 4, -1, "batch"),
    ({}, 4, 65536, "batch")])
def test_cache(lib, c, cols, B, msg):
    kc = cache(**c)
    ref = ctypes.addressof(kc)
    refused(lib, "gguf_kv_cache_write", (ref, FAKE, FAKE, FAKE, FAKE, None, B, 1, cols, 256, 256, 256, 256, None), msg)
    refused(lib, "gguf_kv_cache_read", (ref, FAKE, FAKE, FAKE, FAKE, B, 1, cols, None), msg)
    refused(lib, "gguf_kv_cache_attention", (ref, FAKE, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, B, 1, 4, cols, 512, 512, 0.1, 0,
                                             None), msg)


def test_write_read(lib):
    kc = cache()
    ref = ctypes.addressof(kc)
    write = [ref, FAKE, FAKE, FAKE, FAKE, None, 2, 1, 4, 256, 256, 256, 256, None]
    for i, v, msg in ((1, FAKE + 2, "aligned"), (1, None, "null"), (9, 255, "strides"), (7, -1, "rows"), (0, None, "null"),
                      (3, None, "null")):
        refused(lib, "gguf_kv_cache_write", tuple(write[:i] + [v] + write[i + 1:]), msg)
    read = [ref, FAKE, FAKE, FAKE, FAKE, 2, 1, 4, None]
    for i, v, msg in ((3, FAKE + 16, "32-byte"), (3, None, "null"), (6, -1, "rows"), (6, (1 << 31) - 1, "rows")):
        refused(lib, "gguf_kv_cache_read", tuple(read[:i] + [v] + read[i + 1:]), msg)
    assert lib.gguf_kv_cache_write(*(write[:7] + [0] + write[8:])) == _lib.GGUF_OK  # nothing to do
    assert lib.gguf_kv_cache_read(*(read[:6] + [0] + read[7:])) == _lib.GGUF_OK


def test_attention(lib):
    kc = cache()
    args = [ctypes.addressof(kc), FAKE, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, 2, 1, 4, 4, 512, 512, 0.1, 0, None]
    for i, v, msg in ((1, None, "null"), (1, FAKE + 8, "aligned"), (5, FAKE + 8, "aligned"), (7, None, "null"), (8, None, "null"),
                      (9, 4097, "batch"), (11, 5, "multiple of kv heads"), (11, 0, "multiple of kv heads"), (13, 4, "strides"),
                      (15, float("inf"), "finite"), (15, float("nan"), "finite"), (16, -1, "window")):
        refused(lib, "gguf_kv_cache_attention", tuple(args[:i] + [v] + args[i + 1:]), msg)
    n = ctypes.c_int64(0)
    refused(lib, "gguf_kv_cache_attention_workspace", (1, 1, 4, 2, 80, ctypes.byref(n), ctypes.byref(n)), "head_dim")
    refused(lib, "gguf_kv_cache_attention_workspace", (1, 1, 4, 2, 128, None, ctypes.byref(n)), "null")


@pytest.mark.parametrize("page,cols,B,R,heads", [(256, 1 << 22, 4096, 1, 4), (64, 1 << 14, 8, 1 << 20, 32), (64, 4, 1, 1 << 24, 512)])
def test_attention_of_more_than_32_bits_count(lib, page, cols, B, R, heads):
    """Page tables and rows whose tiles, summed over the call, would pass 32 bits."""
    kc = cache(page=page)
    refused(lib, "gguf_kv_cache_attention", (ctypes.addressof(kc), FAKE, FAKE, FAKE, None, FAKE, None, FAKE, FAKE, B, R, heads, cols,
                                             512, 512, 0.1, 0, None), "too many")


def test_draft(lib):
    args = [FAKE] * 5 + [None, FAKE, FAKE, 2, 3, 1000, None]
    for i, v, msg in ((9, 0, "[1, 32]"), (9, 33, "[1, 32]"), (10, 0, "vocabulary"), (10, (1 << 24) + 1, "vocabulary"), (8, -1, "batch"),
                      (0, None, "null"), (2, None, "null"), (6, None, "null")):
        refused(lib, "gguf_draft_verify", tuple(args[:i] + [v] + args[i + 1:]), msg)
    assert lib.gguf_draft_verify(*(args[:8] + [0] + args[9:])) == _lib.GGUF_OK


def test_host_tensors_are_refused():
    import torch

    from gguf_onnx_ops_b200 import ops

    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.KvCache.empty(2, 1, 16, 64, "cpu")
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.QkNormRope(torch.zeros(1, 192, dtype=torch.bfloat16), None, None, torch.zeros(4, 32), torch.zeros(4, 32),
                       torch.zeros(1, dtype=torch.int32), heads=1, kv_heads=1)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.DraftVerify(torch.zeros(1, 2, 8), None, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1), torch.zeros(1))
