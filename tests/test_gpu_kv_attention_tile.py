"""KvCacheAttention, the tile kernel's range: softmax scales of any sign, scores flat and sharp, magnitudes of q, page scales
and strides with more than 16 rows a kv head of 128 values (32 of 64), over a page table so wide that it takes the call.
Tolerances as in test_gpu_kv_attention_edges.py."""

import pytest
import torch

from gguf_onnx_ops_b200 import ops
from tests import kv_ref as K
from tests.test_gpu_kv_attention_edges import check, reference

pytestmark = pytest.mark.gpu

# R, heads, kv heads, D: one row tile and two, half-filled ones, groups that do not divide 128
FORMS = [(17, 2, 2, 128), (5, 35, 5, 128), (33, 2, 2, 64), (130, 2, 1, 128), (43, 21, 3, 64)]


def run(cuda, form, lens, news=None, page=32, window=0, scale=None, seed=0, spread=1.0, qmul=1.0, q=None, edit=None):
    R, H, Hk, D = form
    B, cols = len(lens), max(1, -(-max(lens) // page))
    cache = K.make_cache(B * cols + 3, Hk, page, D, seed, cuda, spread)
    table = K.make_table(B, cols, B * cols + 3, seed + 1, cuda)
    if edit:
        edit(cache, table)
    if q is None:
        q = (torch.randn(B, R, H, D, generator=K.gen(seed + 2)) * qmul).to(torch.bfloat16).to(cuda)
    scale = D ** -0.5 if scale is None else scale
    # The rule: units of 16 rows, each of as many 16-token tiles as the table holds and 32 more, 150 (64 values: 250) an SM.
    sms, units = torch.cuda.get_device_properties(cuda).multi_processor_count, B * Hk * -(-R * (H // Hk) // 16)
    tiles = -(-sms * (250 if D == 64 else 150) // units)
    wide = torch.nn.functional.pad(table, (0, tiles * 16 // page), value=-1)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    nt = None if news is None else torch.tensor(news, dtype=torch.int32, device=cuda)
    ref = reference(q, cache, table, lens, news, scale, window)
    c = ops.KvCache(*cache)
    out, lse = ops.KvCacheAttention(q, c, wide, lt, nt, window=window, scale=scale, return_lse=True)
    check(out, lse, ref, cache, table, lens)
    assert torch.equal(out, ops.KvCacheAttention(q, c, wide, lt, nt, window=window, scale=scale))
    return out


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("qmul,scale", [(30.0, None), (0.0, None), (1.0, -0.3), (8.0, -0.5), (1.0, 0.0), (1.0, 1e-20)])
def test_scores(cuda, form, qmul, scale):
    """One token takes nearly all (the moving maximum jumps), all are alike, the softmax scale is negative or 0."""
    run(cuda, form, [form[0] + 300, 2000], qmul=qmul, scale=scale, seed=4)


@pytest.mark.parametrize("form", FORMS)
def test_scores_that_rise_and_fall_along_the_tokens(cuda, form):
    """The page scales of K grow (the maximum moves at nearly every step) or shrink (it never does) by 2^1/2 a page."""
    def edit(c, table):
        n = table.shape[1]
        up = torch.exp2(torch.arange(n, device=cuda) / 2 - n / 2 - 2)
        c[2][table[0].long()] = up[:, None]
        c[2][table[1].long()] = up.flip(0)[:, None]

    run(cuda, form, [700, 700], seed=5, edit=edit)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("mul", [1e-36, 1e-20, 1e20])
def test_query_magnitudes(cuda, form, mul):
    R, H, _, D = form
    q = (torch.randn(2, R, H, D, generator=K.gen(8)) * mul).to(torch.bfloat16).to(cuda)
    run(cuda, form, [R + 60, R + 300], q=q, scale=0.05 / mul, seed=8)


@pytest.mark.parametrize("form", FORMS)
def test_page_scales_of_all_sizes(cuda, form):
    run(cuda, form, [form[0] + 480, form[0] + 900], seed=9, spread=6.0, page=16)


@pytest.mark.parametrize("form", FORMS)
def test_pages_of_zeros(cuda, form):
    def edit(c, table):
        p = table[0, ::3].long()
        for t in c:
            t[p] = 0
        p = table[1].long()
        c[1][p], c[3][p] = 0, 0  # a whole sequence of zero V

    out = run(cuda, form, [form[0] + 200, form[0] + 90], seed=10, edit=edit, page=16)
    assert (out[1] == 0).all()


@pytest.mark.parametrize("form", FORMS)
def test_strided_queries_and_a_second_stream(cuda, form):
    R, H, _, D = form
    lens, news = [R + 77, R + 200, R + 1030], [R, max(1, R // 3), R]
    wide = torch.randn(3, R, 3, H, D, generator=K.gen(13)).to(torch.bfloat16).to(cuda)
    a = run(cuda, form, lens, news, q=wide[:, :, 1], seed=13)
    assert torch.equal(a, run(cuda, form, lens, news, q=wide[:, :, 1].contiguous(), seed=13))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(cuda, form, lens, news, q=wide[:, :, 1], seed=13)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_lengths_around_steps_and_pages(cuda, form, page):
    R = form[0]
    lens = [R, R + 1, 63, 64, 65, 127, 128, 129, 255, 256, 257, 0, 1]
    run(cuda, form, lens, [min(R, n) for n in lens], page=page, seed=page)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_stays_in_its_row(cuda, form, bad):
    R, H, Hk, D = form
    q = torch.randn(2, R, H, D, generator=K.gen(3)).to(torch.bfloat16).to(cuda)
    good = run(cuda, form, [R + 100, R + 50], q=q, seed=3)
    q2 = q.clone()
    q2[1, R // 2, H - 1, 3] = bad
    B, page, cols = 2, 32, -(-(R + 100) // 32)
    cache = ops.KvCache(*K.make_cache(B * cols + 3, Hk, page, D, 3, cuda, 1.0))
    table = torch.nn.functional.pad(K.make_table(B, cols, B * cols + 3, 4, cuda), (0, 40000), value=-1)
    out = ops.KvCacheAttention(q2, cache, table, torch.tensor([R + 100, R + 50], dtype=torch.int32, device=cuda))
    assert torch.isnan(out[1, R // 2, H - 1]).all()
    out[1, R // 2, H - 1] = good[1, R // 2, H - 1]
    assert (out.float() - good.float()).abs().max() <= 2.0 ** -7 * good.float().abs().max()
