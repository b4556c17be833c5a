"""KvCacheWrite / KvCacheRead: every step of their definition is one fp32 operation, so codes, scales and the values
read back are compared bit for bit; against 64 bits, a value just written is within half a code (and fp32's last bits) of x."""

import numpy as np
import pytest
import torch

from gguf_onnx_ops_b200 import ops
from tests import kv_ref as K

pytestmark = pytest.mark.gpu


def run_case(cuda, B, R, H, page, D, lens, news=None, seed=0, scale=1.0, strided=False):
    cols = max(1, -(-max(max(lens), 1) // page)) + 1
    pages = B * cols + 2
    cache_t = K.make_cache(pages, H, page, D, seed, cuda)
    table = K.make_table(B, cols, pages, seed + 1, cuda)
    g = K.gen(seed + 2)
    if strided:
        kv = (torch.randn(B, R, 2, H, D, generator=g) * scale).to(torch.bfloat16).to(cuda)
        k, v = kv[:, :, 0], kv[:, :, 1]
    else:
        k, v = ((torch.randn(B, R, H, D, generator=g) * scale).to(torch.bfloat16).to(cuda) for _ in range(2))
    want = [t.cpu().numpy().copy() for t in cache_t]
    tn, ln = table.cpu().numpy(), np.array(lens)
    K.write(want[0], want[2], k.float().cpu().numpy(), tn, ln, news)
    K.write(want[1], want[3], v.float().cpu().numpy(), tn, ln, news)
    cache = ops.KvCache(*cache_t)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    nt = None if news is None else torch.tensor(news, dtype=torch.int32, device=cuda)
    ops.KvCacheWrite(k, v, cache, table, lt, nt)
    for got, ref, name in zip(cache_t, want, ("k", "v", "k_scale", "v_scale")):
        assert np.array_equal(got.cpu().numpy(), ref), name
    ops.KvCacheWrite(k, v, cache, table, lt, nt)  # the same tokens again change nothing
    for got, ref in zip(cache_t, want):
        assert np.array_equal(got.cpu().numpy(), ref)
    # read back, all rows and some before the start
    rows = max(lens) + 3
    rk, rv = ops.KvCacheRead(cache, table, lt, rows=rows)
    for got, codes, scales in ((rk, want[0], want[2]), (rv, want[1], want[3])):
        for b in range(B):
            n = lens[b]
            x = K.dense(torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda), table[b], n) if n else None
            assert (got[b, :rows - n] == 0).all()
            if n:
                assert torch.equal(got[b, rows - n:], x.float().to(torch.bfloat16))
    return cache, table, lt, k, v


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_ragged_writes(cuda, page, D):
    run_case(cuda, 6, 19, 2, page, D, [19, 20, 100, 1, 0, 300], seed=page + D)


@pytest.mark.parametrize("R,lens,news", [(1, [1, 2, 16, 17, 64, 65], None), (1, [0, 5, 0], None),
                                         (5, [5, 64, 69, 3], [1, 5, 0, 3]), (130, [130, 193, 500], None),
                                         (300, [300, 301], [300, 7])])
def test_tokens_and_prompts(cuda, R, lens, news):
    run_case(cuda, len(lens), R, 3, 64, 128, lens, news, seed=R)
    run_case(cuda, len(lens), R, 3, 16, 64, lens, news, seed=R, strided=True)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 0.0])
def test_magnitudes(cuda, scale):
    """Scales near the smallest normal float and below it, large ones, zeros."""
    run_case(cuda, 3, 4, 2, 16, 64, [4, 8, 37], seed=9, scale=scale)


def test_token_by_token_and_rollback(cuda):
    """Sixty single tokens of growing size: the scale follows the largest, older codes are rescaled; a rollback keeps it."""
    H, page, D = 2, 64, 64
    cache = ops.KvCache.empty(3, H, page, D, cuda)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=cuda)
    x = torch.randn(70, H, D, generator=K.gen(1)) * torch.linspace(0.1, 2, 70)[:, None, None]
    xb = x.to(torch.bfloat16).to(cuda)
    want = [t.cpu().numpy().copy() for t in (cache.k, cache.k_scale)]
    for i in range(70):
        lens = torch.tensor([i + 1], dtype=torch.int32, device=cuda)
        t = xb[i].reshape(1, 1, H, D)
        ops.KvCacheWrite(t, t, cache, table, lens)
        K.write(want[0], want[1], t.float().cpu().numpy(), table.cpu().numpy(), [i + 1], None)
    assert np.array_equal(cache.k.cpu().numpy(), want[0]) and np.array_equal(cache.k_scale.cpu().numpy(), want[1])
    assert torch.equal(cache.k, cache.v)
    got, _ = ops.KvCacheRead(cache, table, lens, rows=70)
    # each rescaling rounds a code once more, by half a code of the scale of that time at most
    assert (got[0].double().cpu() - xb.double().cpu()).abs().max() <= 70 * 0.51 * float(cache.k_scale.max())
    before = float(cache.k_scale[2, 0])
    small = xb[:1].reshape(1, 1, H, D) * 0
    ops.KvCacheWrite(small, small, cache, table, torch.tensor([30], dtype=torch.int32, device=cuda))
    assert float(cache.k_scale[2, 0]) == before
    ops.KvCacheWrite(small, small, cache, table, torch.tensor([1], dtype=torch.int32, device=cuda))  # begun again
    assert float(cache.k_scale[2, 0]) == 0


def test_within_half_a_code_of_the_values(cuda):
    cache, table, lens, k, _ = run_case(cuda, 2, 200, 2, 64, 128, [200, 200], seed=4)
    rk, _ = ops.KvCacheRead(cache, table, lens, rows=200)
    for b in range(2):
        codes = K.dense(cache.k, cache.k_scale, table[b], 200)
        step = cache.k_scale[table[b, :4].long()].repeat_interleave(64, 0)[:200].double()
        assert ((codes - k[b].double()).abs() <= step[..., None] * 0.5001).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_value_that_is_not_finite_marks_its_page_and_head_only(cuda, bad):
    cache = ops.KvCache.empty(4, 2, 16, 64, cuda)
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=cuda)
    x = torch.ones(1, 20, 2, 64, dtype=torch.bfloat16, device=cuda)
    y = x.clone()
    y[0, 17, 1, 5] = bad
    lens = torch.tensor([20], dtype=torch.int32, device=cuda)
    ops.KvCacheWrite(y, x, cache, table, lens)
    k, v = ops.KvCacheRead(cache, table, lens, rows=20)
    assert torch.isnan(k[0, 16:, 1]).all()
    assert (k[0, :16] == 1).all() and (k[0, 16:, 0] == 1).all() and (v == 1).all()


def test_pages_outside_the_cache_are_reported_and_skipped(cuda):
    cache = ops.KvCache.empty(2, 1, 16, 64, cuda)
    x = torch.ones(1, 20, 1, 64, dtype=torch.bfloat16, device=cuda)
    ops.device_status()
    for table, lens in (([[1, 2]], [20]), ([[1, -1]], [20]), ([[1]], [20])):
        t = torch.tensor(table, dtype=torch.int32, device=cuda)
        n = torch.tensor(lens, dtype=torch.int32, device=cuda)
        ops.KvCacheWrite(x, x, cache, t, n)
        assert ops.device_status() == (4, 7)
        k, _ = ops.KvCacheRead(cache, t, n, rows=20)
        assert ops.device_status() == (4, 7)
        assert (k[0, :16] == 1).all() and (k[0, 16:] == 0).all()
    assert (cache.k[0] == 0).all()


def test_codes_past_four_gigabytes(cuda):
    """Page numbers whose byte offsets need 33 bits."""
    H, page, D = 8, 256, 256
    pages = (1 << 32) // (H * page * D) + 8
    k = torch.empty(pages, H, page, D, dtype=torch.int8, device=cuda)
    s = torch.zeros(pages, H, device=cuda)
    cache = ops.KvCache(k, torch.empty_like(k), s, s.clone())
    table = torch.tensor([[pages - 1, 3]], dtype=torch.int32, device=cuda)
    x = torch.randn(1, 300, H, D, generator=K.gen(2)).to(torch.bfloat16).to(cuda)
    lens = torch.tensor([300], dtype=torch.int32, device=cuda)
    ops.KvCacheWrite(x, x, cache, table, lens)
    got, _ = ops.KvCacheRead(cache, table, lens, rows=300)
    assert torch.equal(got[0], K.dense(k, s, table[0], 300).float().to(torch.bfloat16))
    q = x[:, -2:, :8]
    out = ops.KvCacheAttention(q, cache, table, lens)
    ref, mag, _ = K.attention(q, (k, cache.v, s, cache.v_scale), table, lens, None, D ** -0.5, 0)
    assert ((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -11 * mag).all()


def test_refusals(cuda):
    c = ops.KvCache.empty(4, 2, 16, 64, cuda)
    table = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    lens = torch.ones(1, dtype=torch.int32, device=cuda)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="page must be"):
        ops.KvCache.empty(4, 2, 48, 64, cuda)
    with pytest.raises(ValueError, match="head_dim must be"):
        ops.KvCache.empty(4, 2, 16, 80, cuda)
    with pytest.raises(ValueError, match="must be torch.int8"):
        ops.KvCache(c.k.float(), c.v, c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="needs k, v"):
        ops.KvCache(c.k, c.v[:2].contiguous(), c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.KvCacheWrite(x.float(), x, c, table, lens)
    with pytest.raises(ValueError, match=r"\[B, rows, 2, 64\]"):
        ops.KvCacheWrite(x[:, :, :1], x, c, table, lens)
    with pytest.raises(ValueError, match="heads of a row"):
        ops.KvCacheWrite(torch.zeros(1, 1, 64, 2, dtype=torch.bfloat16, device=cuda).transpose(2, 3), x, c, table, lens)
    with pytest.raises(ValueError, match="page_table"):
        ops.KvCacheWrite(x, x, c, table.repeat(2, 1), lens)
    with pytest.raises(ValueError, match="new_lens"):
        ops.KvCacheWrite(x, x, c, table, lens, lens.repeat(2))
    with pytest.raises(ValueError, match="16-byte aligned"):
        flat = torch.zeros(129 + 8, dtype=torch.bfloat16, device=cuda)
        ops.KvCacheWrite(flat[1:129].view(1, 1, 2, 64), x, c, table, lens)
    with pytest.raises(ValueError, match="rows must be"):
        ops.KvCacheRead(c, table, lens, rows=-1)
