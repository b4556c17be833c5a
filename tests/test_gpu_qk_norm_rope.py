"""QkNormRope against its formula in 64 bits.

Tolerance, derived: fp32 arithmetic with one rounding to bf16.  The rounding is at most 2^-9 of the result; the norm
factor, two products and a sum in fp32 add a few 2^-24 of |a| + |b|, which stays when a and b cancel: 2^-8 |y| + 2^-20 (|a| + |b|)."""

import pytest
import torch

from gguf_onnx_ops_b200 import ops
from tests.kv_ref import gen

pytestmark = pytest.mark.gpu


def tables(max_pos, rot, device, base=10000.0):
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * f
    return a.cos().float().to(device).contiguous(), a.sin().float().to(device).contiguous()


def reference(qkv, gq, gk, cos, sin, pos, hq, hk, eps, inter):
    D = qkv.shape[-1] // (hq + 2 * hk)
    x = qkv.double().reshape(-1, hq + 2 * hk, D)[:, :hq + hk]
    out = torch.empty_like(x)
    bound = torch.zeros_like(x)
    rot = 2 * cos.shape[1]
    for h in range(hq + hk):
        gamma = gq if h < hq else gk
        y = x[:, h]
        if gamma is not None:
            y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * gamma.double()
        out[:, h] = y
        bound[:, h] = y.abs()
        if rot:
            c, s = cos.double()[pos.long()], sin.double()[pos.long()]
            ia = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
            ib = ia + (1 if inter else rot // 2)
            a, b = y[:, ia], y[:, ib]
            out[:, h, ia], out[:, h, ib] = a * c - b * s, b * c + a * s
            bound[:, h, ia] = bound[:, h, ib] = a.abs() + b.abs()
    return (out[:, :hq], out[:, hq:]), (bound[:, :hq], bound[:, hq:])


def check(got, want, bound):
    for g, w, m in zip(got, want, bound):
        d = (g.double().reshape(w.shape) - w).abs()
        tol = 2.0 ** -8 * w.abs() + 2.0 ** -20 * m
        assert (d <= tol).all(), (d - tol).max()


@pytest.mark.parametrize("T,hq,hk,D,rot", [(1, 32, 8, 128, 128), (1, 1, 1, 8, 8), (3, 5, 1, 64, 32), (7, 9, 3, 96, 96),
                                           (2, 4, 2, 80, 40), (5, 6, 2, 256, 64), (4, 3, 1, 192, 192), (2, 2, 2, 128, 0),
                                           (1025, 33, 7, 128, 128), (2049, 16, 4, 256, 256), (4097, 20, 4, 64, 64)])
@pytest.mark.parametrize("inter", [False, True])
def test_shapes(cuda, T, hq, hk, D, rot, inter):
    g = gen(T + D + rot)
    qkv = (torch.randn(T, (hq + 2 * hk) * D, generator=g) * 2).to(torch.bfloat16).to(cuda)
    gq, gk = (torch.rand(D, generator=g) + 0.5).to(cuda), (torch.rand(D, generator=g) - 0.5).to(cuda)
    cos, sin = tables(517, rot, cuda)
    pos = torch.randint(0, 517, (T,), generator=g, dtype=torch.int32).to(cuda)
    got = ops.QkNormRope(qkv, gq, gk, cos, sin, pos, heads=hq, kv_heads=hk, epsilon=1e-6, interleaved=inter)
    assert got[0].shape == (T, hq, D) and got[1].shape == (T, hk, D)
    check(got, *reference(qkv, gq, gk, cos, sin, pos, hq, hk, 1e-6, inter))


def test_without_norm_strided_rows_and_leading_dims(cuda):
    g = gen(3)
    hq, hk, D, T = 4, 2, 64, 9
    wide = torch.randn(T, (hq + 2 * hk) * D + 36, generator=g).to(torch.bfloat16).to(cuda)
    qkv = wide[:, 4:4 + (hq + 2 * hk) * D]  # 8-byte aligned rows, another row stride
    cos, sin = tables(64, D, cuda)
    pos = torch.arange(T, dtype=torch.int32, device=cuda)
    gk = (torch.rand(D, generator=g) + 0.5).to(cuda)
    got = ops.QkNormRope(qkv, None, gk, cos, sin, pos, heads=hq, kv_heads=hk)
    check(got, *reference(qkv, None, gk, cos, sin, pos, hq, hk, 1e-6, False))
    x3 = qkv.contiguous().reshape(3, 3, -1)
    q3, k3 = ops.QkNormRope(x3, None, gk, cos, sin, pos, heads=hq, kv_heads=hk)
    assert torch.equal(q3.reshape(T, hq, D), got[0]) and torch.equal(k3.reshape(T, hk, D), got[1])
    e = ops.QkNormRope(qkv[:0], None, gk, cos, sin, pos[:0], heads=hq, kv_heads=hk)
    assert e[0].shape == (0, hq, D)


@pytest.mark.parametrize("T", [3, 700])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_norm,k_norm", [(False, True), (True, False), (False, False)])
def test_a_norm_on_one_side_only(cuda, T, D, q_norm, k_norm):
    """A warp has query and key heads side by side, with one head a lane group (few tokens) and with four; heads without a
    norm come out as their rounded rotation, whatever the others have."""
    g = gen(T + D)
    hq, hk = 5, 3
    qkv = (torch.randn(T, (hq + 2 * hk) * D, generator=g) * 2).to(torch.bfloat16).to(cuda)
    gq = (torch.rand(D, generator=g) + 0.5).to(cuda) if q_norm else None
    gk = (torch.rand(D, generator=g) + 0.5).to(cuda) if k_norm else None
    cos, sin = tables(301, D, cuda)
    pos = torch.randint(0, 301, (T,), generator=g, dtype=torch.int32).to(cuda)
    got = ops.QkNormRope(qkv, gq, gk, cos, sin, pos, heads=hq, kv_heads=hk)
    check(got, *reference(qkv, gq, gk, cos, sin, pos, hq, hk, 1e-6, False))
    bare = ops.QkNormRope(qkv, None, None, cos, sin, pos, heads=hq, kv_heads=hk)
    for y, z, norm in zip(got, bare, (q_norm, k_norm)):
        assert norm or torch.equal(y, z)


def test_extreme_rows(cuda):
    """Zero heads, tiny and huge values; an infinite value makes its own head NaN and no other."""
    hq, hk, D = 3, 1, 64
    x = torch.ones(4, (hq + 2 * hk) * D)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e15
    x[3, 5] = float("inf")
    qkv = x.to(torch.bfloat16).to(cuda)
    one = torch.ones(D, device=cuda)
    cos, sin = tables(8, D, cuda)
    pos = torch.arange(4, dtype=torch.int32, device=cuda)
    q, k = ops.QkNormRope(qkv, one, one, cos, sin, pos, heads=hq, kv_heads=hk)
    (rq, rk), (bq, bk) = reference(qkv, one, one, cos, sin, pos, hq, hk, 1e-6, False)
    check((q[:3], k[:3]), (rq[:3], rk[:3]), (bq[:3], bk[:3]))
    assert torch.isnan(q[3, 0]).any() and torch.isfinite(q[3, 1:].float()).all() and torch.isfinite(k[3].float()).all()


def test_position_outside_the_tables_is_reported(cuda):
    x = torch.ones(2, 3 * 64, dtype=torch.bfloat16, device=cuda)
    cos, sin = tables(4, 64, cuda)
    ops.device_status()
    q, _ = ops.QkNormRope(x, None, None, cos, sin, torch.tensor([4, 0], dtype=torch.int32, device=cuda), heads=1, kv_heads=1)
    rc, site = ops.device_status()
    assert rc != 0 and site == 8
    assert torch.equal(q[0], q[1])  # row 0 was used
    assert ops.device_status()[0] == 0


def test_refusals(cuda):
    x = torch.zeros(2, 6 * 64, dtype=torch.bfloat16, device=cuda)
    cos, sin = tables(8, 64, cuda)
    pos = torch.zeros(2, dtype=torch.int32, device=cuda)
    ok = dict(heads=4, kv_heads=1)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.QkNormRope(x.float(), None, None, cos, sin, pos, **ok)
    with pytest.raises(ValueError, match="width"):
        ops.QkNormRope(x, None, None, cos, sin, pos, heads=5, kv_heads=1)
    with pytest.raises(ValueError, match="one position per row"):
        ops.QkNormRope(x, None, None, cos, sin, pos[:1], **ok)
    with pytest.raises(ValueError, match="q_gamma size"):
        ops.QkNormRope(x, torch.ones(32, device=cuda), None, cos, sin, pos, **ok)
    with pytest.raises(ValueError, match="rotated width"):
        ops.QkNormRope(x, None, None, cos[:, :31].contiguous(), sin[:, :31].contiguous(), pos, **ok)
    with pytest.raises(ValueError, match="contiguous"):
        ops.QkNormRope(x[:, ::2], None, None, cos, sin, pos, heads=1, kv_heads=1)
