"""KvCacheAttention against softmax attention in 64 bits on the cache's values.

Tolerance, derived: q and the codes enter exactly, scores and sums are fp32; a token's weight is rounded to f16 once
(2^-12 of it, or 2^-40 absolute of the largest), so the output is off by at most 2^-11 sum p |v| + 2^-40 n max |v| before it is
rounded to bf16 (2^-9, bounded here by 2^-8).  The log-sum-exp is fp32 throughout: 1e-5 (4 + |lse|)."""

import pytest
import torch

from gguf_onnx_ops_b200 import ops
from tests import kv_ref as K

pytestmark = pytest.mark.gpu
WIDE = 1 << 20  # positions of a wide table, over all (sequence, kv head) pairs


def check(out, ref, mag, cache, lens):
    d = (out.double() - ref).abs()
    scales = cache[3][torch.isfinite(cache[3])]
    least = 2.0 ** -40 * max(lens) * 127 * float(scales.max())
    tol = 2.0 ** -8 * ref.abs() + 2.0 ** -11 * mag + least
    assert torch.isfinite(out.float()).all()
    assert (d <= tol).all(), float((d - tol).max())


def run_case(cuda, B, R, H, Hk, page, D, lens, news=None, window=0, scale=None, seed=0, spread=1.0, qmul=1.0, q=None,
             edit=None):
    cols = max(1, -(-max(lens) // page)) + 1
    pages = B * cols + 3
    cache_t = K.make_cache(pages, Hk, page, D, seed, cuda, spread)
    table = K.make_table(B, cols, pages, seed + 1, cuda)
    if edit:
        edit(cache_t, table)
    if q is None:
        q = (torch.randn(B, R, H, D, generator=K.gen(seed + 2)) * qmul).to(torch.bfloat16).to(cuda)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    nt = None if news is None else torch.tensor(news, dtype=torch.int32, device=cuda)
    ref, mag, ref_lse = K.attention(q, cache_t, table, lens, news, D ** -0.5 if scale is None else scale, window)
    seen = torch.isfinite(ref_lse)
    # A page table that is much wider than the lengths: for many rows another kernel takes the call.
    wide = torch.nn.functional.pad(table, (0, WIDE // (B * Hk * page)), value=-1)
    for t in (table, wide):
        out, lse = ops.KvCacheAttention(q, ops.KvCache(*cache_t), t, lt, nt, window=window, scale=scale, return_lse=True)
        check(out, ref, mag, cache_t, lens)
        assert torch.equal(seen, torch.isfinite(lse))
        assert ((lse.double() - ref_lse)[seen].abs() <= 1e-5 * (4 + ref_lse[seen].abs())).all()
        assert (out[~seen] == 0).all()
        again = ops.KvCacheAttention(q, ops.KvCache(*cache_t), t, lt, nt, window=window, scale=scale)
        assert torch.equal(out, again)  # whatever the order in which CTAs finish
    return out


@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("H,Hk,R", [(1, 1, 1), (8, 1, 1), (5, 1, 3), (4, 4, 2), (14, 2, 1), (32, 2, 5)])
def test_heads_and_rows(cuda, D, H, Hk, R):
    run_case(cuda, 3, R, H, Hk, 64, D, [R, 130, 517], seed=D + H + R)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages_and_lengths(cuda, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 300, 0]
    run_case(cuda, len(lens), 1, 8, 2, page, 128, lens, seed=page)
    run_case(cuda, len(lens), 4, 8, 2, page, 64, lens, seed=page)


def test_fewer_new_tokens_than_rows(cuda):
    run_case(cuda, 6, 6, 16, 2, 32, 128, [6, 100, 3, 0, 1000, 64], news=[6, 1, 3, 0, 4, 0], seed=5)
    run_case(cuda, 4, 4, 4, 2, 32, 128, [2, 1, 40, 7], news=[4, 4, 9, -3], seed=6)  # never more than rows or length


@pytest.mark.parametrize("window", [1, 5, 16, 100, 1000, 1 << 30])
def test_windows(cuda, window):
    run_case(cuda, 4, 5, 10, 2, 16, 64, [5, 37, 400, 999], window=window, seed=window % 97)
    run_case(cuda, 2, 40, 10, 2, 16, 64, [40, 399], window=window, seed=window % 97)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_windows_of_many_rows(cuda, window, D):
    run_case(cuda, 8, 200, 10, 2, 16, D, [200, 201, 215, 300, 399, 777, 1210, 260], window=window, seed=window,
             news=[200, 200, 200, 1, 200, 130, 200, 0])


@pytest.mark.parametrize("R", [17, 33, 64, 129, 300])
def test_many_rows(cuda, R):
    run_case(cuda, 2, R, 6, 2, 64, 128, [R, R + 211], seed=R)
    run_case(cuda, 1, R, 3, 1, 16, 64, [R + 1], seed=R)
    run_case(cuda, 3, R, 4, 2, 256, 64, [R, R + 3, 900], seed=R, news=[R, 3, R // 2])


@pytest.mark.parametrize("R,D", [(40, 128), (70, 64), (300, 128)])
def test_units_follow_one_another_in_a_block(cuda, R, D):
    """More (sequence, kv head) units than blocks, of one to a few 64-token steps each: a unit's first scores go where the
    last unit's weights were.  The lengths leave odd and even numbers of steps; one and two row tiles."""
    B = 60 if R < 100 else 24
    lens = [R + (61 * i) % 530 for i in range(B)]
    run_case(cuda, B, R, 8, 8, 64, D, lens, news=[R if i % 5 else 1 + i % R for i in range(B)], seed=R)


def test_one_long_sequence(cuda):
    run_case(cuda, 1, 1, 8, 2, 64, 128, [40007], seed=1)
    run_case(cuda, 1, 2, 4, 1, 64, 64, [70001], seed=2, window=60000)


def test_many_short_sequences(cuda):
    lens = [(37 * i) % 91 for i in range(700)]
    run_case(cuda, 700, 1, 4, 1, 16, 64, lens, seed=3)


def test_sharp_and_flat_scores(cuda):
    run_case(cuda, 2, 3, 8, 2, 64, 128, [300, 2000], qmul=30.0, seed=4)  # one token takes nearly all
    run_case(cuda, 2, 3, 8, 2, 64, 128, [300, 2000], qmul=0.0, seed=4)  # q = 0: the mean of v
    run_case(cuda, 2, 3, 8, 2, 64, 128, [300, 2000], scale=-0.3, seed=4)
    run_case(cuda, 2, 3, 8, 2, 64, 128, [300, 2000], scale=0.0, seed=4)


@pytest.mark.parametrize("mul", [1e-36, 1e-20, 1e20])
def test_query_magnitudes(cuda, mul):
    """q's power of two is taken out row by row: tiny and huge rows keep their precision."""
    g = K.gen(8)
    q = (torch.randn(2, 2, 8, 128, generator=g) * mul).to(torch.bfloat16).to(cuda)
    run_case(cuda, 2, 2, 8, 2, 64, 128, [100, 300], q=q, scale=0.05 / mul, seed=8)


def test_page_scales_of_all_sizes(cuda):
    run_case(cuda, 2, 2, 8, 2, 16, 128, [500, 900], seed=9, spread=6.0)


def test_pages_of_zeros(cuda):
    def edit(c, table):
        for i in (0, 3, 4):
            p = table[0, i].long()
            c[1][p], c[3][p] = 0, 0  # V zero
            c[0][p], c[2][p] = 0, 0  # K zero
        p = table[1].long()
        c[1][p], c[3][p] = 0, 0  # a whole sequence of zero V

    out = run_case(cuda, 2, 2, 8, 2, 16, 64, [200, 90], seed=10, edit=edit)
    assert (out[1] == 0).all()


def test_hidden_places_do_not_matter(cuda):
    """Pages past a sequence's end and pages of others may hold anything, scales that are not numbers among it."""
    def edit(c, table):
        used = table[0, :4].long()
        keep = [t[used].clone() for t in c]
        for t in c[2:]:
            t.fill_(float("nan"))
        for t, x in zip(c, keep):
            t[used] = x

    run_case(cuda, 1, 3, 8, 2, 32, 128, [101], seed=11, edit=edit)
    # the window hides whole pages at the front
    def front(c, table):
        for t in c[2:]:
            t[table[0, :2].long()] = float("inf")

    run_case(cuda, 1, 1, 8, 2, 32, 128, [161], window=97, seed=12, edit=front)
    run_case(cuda, 1, 20, 8, 2, 32, 128, [161 + 19], window=97, seed=12, edit=front)
    # the same for many rows
    run_case(cuda, 1, 20, 8, 2, 32, 128, [101], seed=11, edit=edit)

    def fronts(c, table):
        for t in c[2:]:
            t[table[:, :2].long()] = float("inf")

    run_case(cuda, 16, 100, 8, 2, 32, 128, [260 - 100 // (b + 1) % 3 for b in range(16)], window=97, seed=12,
             news=[100 - 100 // (b + 1) % 3 for b in range(16)], edit=fronts)


@pytest.mark.parametrize("R,D,cols", [(1, 64, 3), (20, 128, 8000)])
def test_marked_pages_are_seen(cuda, R, D, cols):
    """A page whose scale is NaN makes the rows that see it NaN, and no others."""
    c = K.make_cache(8, 2, 16, D, 1, cuda)
    table = torch.full((2, cols), -1, dtype=torch.int32, device=cuda)
    table[:, :3] = torch.arange(6, dtype=torch.int32, device=cuda).view(2, 3)
    c[3][4, 1] = float("nan")
    q = torch.randn(2, R, 4, D, generator=K.gen(2)).to(torch.bfloat16).to(cuda)
    lens = torch.tensor([40, 40], dtype=torch.int32, device=cuda)
    out = ops.KvCacheAttention(q, ops.KvCache(*c), table, lens)
    assert torch.isfinite(out[0].float()).all() and torch.isfinite(out[1, :, :2].float()).all()
    assert torch.isnan(out[1, :, 2:]).all()


def test_strided_queries_streams_and_workspaces(cuda):
    g = K.gen(13)
    B, R, H, Hk, D = 3, 2, 8, 2, 128
    wide = torch.randn(B, R, 3, H, D, generator=g).to(torch.bfloat16).to(cuda)
    lens = [77, 200, 1030]
    a = run_case(cuda, B, R, H, Hk, 64, D, lens, q=wide[:, :, 1], seed=13)
    b = run_case(cuda, B, R, H, Hk, 64, D, lens, q=wide[:, :, 1].contiguous(), seed=13)
    assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = run_case(cuda, B, R, H, Hk, 64, D, lens, q=wide[:, :, 1], seed=13)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, c)


@pytest.mark.parametrize("R,extra", [(2, 0), (12, 4000)])
def test_captured_graph_serves_other_lengths(cuda, R, extra):
    B, H, Hk, page, D = 4, 8, 2, 64, 128
    c = K.make_cache(200, Hk, page, D, 14, cuda)
    cache = ops.KvCache(*c)
    table = torch.nn.functional.pad(K.make_table(B, 40, 200, 15, cuda), (0, extra), value=-1)
    q = torch.randn(B, R, H, D, generator=K.gen(16)).to(torch.bfloat16).to(cuda)
    lens = torch.tensor([5, 100, 900, 2000], dtype=torch.int32, device=cuda)
    ws = ops.KvAttentionWorkspace(cuda)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(ValueError, match="fit"):
            ops.KvCacheAttention(q, cache, table, lens, workspace=ws)
    ws.fit(B, R, H, Hk, D)
    for own in (ws, None):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.KvCacheAttention(q, cache, table, lens, workspace=own)
        for case in ([5, 100, 900, 2000], [2560, 2, 0, 31], [64, 64, 64, 64]):
            lens.copy_(torch.tensor(case, dtype=torch.int32))
            graph.replay()
            graph.replay()
            ref, mag, _ = K.attention(q, c, table, case, None, D ** -0.5, 0)
            check(out, ref, mag, c, case)


def test_a_workspace_that_grows_leaves_captured_graphs_what_they_use(cuda):
    B, R, H, Hk, page, D = 2, 2, 8, 2, 64, 128
    c = K.make_cache(120, Hk, page, D, 14, cuda)
    cache, case = ops.KvCache(*c), [3000, 2900]
    table = K.make_table(B, 50, 120, 15, cuda)
    q = torch.randn(B, R, H, D, generator=K.gen(16)).to(torch.bfloat16).to(cuda)
    lens = torch.tensor(case, dtype=torch.int32, device=cuda)
    ws = ops.KvAttentionWorkspace(cuda).fit(B, R, H, Hk, D)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.KvCacheAttention(q, cache, table, lens, workspace=ws)
    small = [(t.data_ptr(), t.numel() * t.element_size()) for t in (ws.scratch, ws.counters)]
    ws.fit(64, 300, 32, 8, D)
    assert ws.scratch.numel() > small[0][1] and ws.counters.numel() * 4 > small[1][1]
    # Allocations of the same sizes get other memory, and the replays leave them alone.
    others = [torch.full((n,), 77, dtype=torch.uint8, device=cuda) for _, n in small for _ in range(8)]
    for t in others:
        for at, n in small:
            assert t.data_ptr() + t.numel() <= at or at + n <= t.data_ptr()
    ref, mag, _ = K.attention(q, c, table, case, None, D ** -0.5, 0)
    for _ in range(3):
        out.zero_()
        graph.replay()
        check(out, ref, mag, c, case)
        check(ops.KvCacheAttention(q, cache, table, lens, workspace=ws), ref, mag, c, case)
    assert all((t == 77).all() for t in others)


def test_lengths_past_the_table_are_reported(cuda):
    c = K.make_cache(4, 1, 16, 64, 1, cuda)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device=cuda)
    table = torch.tensor([[1, 2]], dtype=torch.int32, device=cuda)
    ops.device_status()
    ops.KvCacheAttention(q, ops.KvCache(*c), table, torch.tensor([33], dtype=torch.int32, device=cuda))
    assert ops.device_status() == (4, 7)
    ops.KvCacheAttention(q, ops.KvCache(*c), table + 3, torch.tensor([20], dtype=torch.int32, device=cuda))
    assert ops.device_status() == (4, 7)
    ops.KvCacheAttention(q, ops.KvCache(*c), table, torch.tensor([32], dtype=torch.int32, device=cuda))
    assert ops.device_status()[0] == 0


def test_empty_calls(cuda):
    c = ops.KvCache(*K.make_cache(4, 2, 16, 64, 1, cuda))
    table = torch.zeros(0, 2, dtype=torch.int32, device=cuda)
    lens = torch.zeros(0, dtype=torch.int32, device=cuda)
    out = ops.KvCacheAttention(torch.zeros(0, 1, 4, 64, dtype=torch.bfloat16, device=cuda), c, table, lens)
    assert out.shape == (0, 1, 4, 64)
    out = ops.KvCacheAttention(torch.zeros(2, 0, 4, 64, dtype=torch.bfloat16, device=cuda), c, table.new_zeros(2, 2),
                               lens.new_zeros(2))
    assert out.shape == (2, 0, 4, 64)


def test_refusals(cuda):
    c = ops.KvCache.empty(4, 2, 16, 64, cuda)
    table = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    lens = torch.ones(1, dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="multiple of kv heads"):
        ops.KvCacheAttention(q[:, :, :3], c, table, lens)
    with pytest.raises(ValueError, match=r"q must be \[B, rows"):
        ops.KvCacheAttention(q.view(1, 1, 2, 128), c, table, lens)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.KvCacheAttention(q.half(), c, table, lens)
    with pytest.raises(ValueError, match="window"):
        ops.KvCacheAttention(q, c, table, lens, window=-1)
    with pytest.raises(ValueError, match="finite"):
        ops.KvCacheAttention(q, c, table, lens, scale=float("nan"))
    with pytest.raises(ValueError, match="int32"):
        ops.KvCacheAttention(q, c, table.long(), lens)
    with pytest.raises(ValueError, match=r"batch must be in \[0, 4096\]"):
        ops.KvCacheAttention(q.expand(4097, 1, 4, 64), c, table.expand(4097, 2).contiguous(), lens.expand(4097).contiguous())
