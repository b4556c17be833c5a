"""KvCacheAttention where pages are marked, missing, empty or of unusual scale, through both kernels.

A call of few rows is the streaming kernel's; one of many rows over a wide page table is the tile kernel's.  Tolerances are
those of test_gpu_kv_attention.py with the tile kernel's absolute term: a weight is off by 2^-12 of it or by 2^-36 of the
largest one, so the output is off by 2^-11 sum p |v| + 2^-36 n max |v|, and 2^-8 of it for the rounding to bf16."""

import numpy as np
import pytest
import torch

from gguf_onnx_ops_b200 import ops
from tests import kv_ref as K

pytestmark = pytest.mark.gpu

# name, R, heads, kv heads, D, page-table columns beside the needed ones
FORMS = [("stream", 3, 8, 2, 128, 0), ("stream", 3, 4, 2, 64, 0), ("stream", 1, 5, 1, 256, 0), ("stream", 2, 16, 2, 96, 0), ("stream", 40, 4, 2, 128, 0),
         ("tile", 40, 4, 2, 128, 4000), ("tile", 70, 2, 2, 64, 9000), ("tile", 300, 2, 1, 128, 9000)]
IDS = [f"{f[0]}-R{f[1]}-D{f[4]}" for f in FORMS]


def reference(q, cache, table, lens, news, scale, window=0):
    """As kv_ref.attention, rows by matrix products; positions whose page is not in the cache are left out."""
    B, R, H, D = q.shape
    Hk, page, pages = cache[0].shape[1], cache[0].shape[2], cache[0].shape[0]
    out = torch.zeros(B, R, H, D, dtype=torch.float64, device=q.device)
    mag, lse = torch.zeros_like(out), torch.full((B, R, H), -np.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lens[b])
        m = min(R if news is None else int(news[b]), n, R)
        if m <= 0:
            continue
        t = table[b, :-(-n // page)].long()
        ok = ((t >= 0) & (t < pages)).repeat_interleave(page)[:n]
        k, v = (K.dense(cache[i], cache[i + 2], torch.where((t >= 0) & (t < pages), t, 0), n) for i in (0, 1))
        pos, j = torch.arange(n - m, n, device=q.device)[:, None], torch.arange(n, device=q.device)
        see = (j <= pos) & ok
        if window:
            see &= j > pos - window
        for h in range(H):
            kh, vh = k[:, h // (H // Hk)], v[:, h // (H // Hk)]
            s = (q[b, :m, h].double() @ kh.T * scale).masked_fill(~see, -np.inf)
            lse[b, :m, h] = torch.logsumexp(s, -1)
            p = torch.softmax(s, -1).masked_fill(~see.any(-1, keepdim=True), 0.0)
            if torch.isfinite(vh).all():
                out[b, :m, h], mag[b, :m, h] = p @ vh, p @ vh.abs()
            else:  # row by row, so that hidden places stay out of it
                for r in range(m):
                    at = see[r].nonzero()[:, 0]
                    out[b, r, h], mag[b, r, h] = p[r, at] @ vh[at], p[r, at] @ vh[at].abs()
    return out, mag, lse


def call(cuda, form, lens, page=16, news=None, window=0, scale=None, seed=0, edit=None, qmul=1.0):
    _, R, H, Hk, D, extra = form
    B, cols = len(lens), max(1, -(-max(lens) // page))
    pages = B * cols + 3
    cache = K.make_cache(pages, Hk, page, D, seed, cuda)
    table = K.make_table(B, cols, pages, seed + 1, cuda)
    if edit:
        edit(cache, table)
    q = (torch.randn(B, R, H, D, generator=K.gen(seed + 2)) * qmul).to(torch.bfloat16).to(cuda)
    scale = D ** -0.5 if scale is None else scale
    wide = torch.nn.functional.pad(table, (0, extra * 64 // page // B), value=-1)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    nt = None if news is None else torch.tensor(news, dtype=torch.int32, device=cuda)
    out, lse = ops.KvCacheAttention(q, ops.KvCache(*cache), wide, lt, nt, window=window, scale=scale, return_lse=True)
    return out, lse, reference(q, cache, table, lens, news, scale, window), cache, table


def check(out, lse, ref, cache, table, lens, where=None):
    want, mag, want_lse = ref
    t = table[(table >= 0) & (table < cache[0].shape[0])].long()
    scales = cache[3][t]
    most = float(scales[torch.isfinite(scales)].max()) * 127
    where = torch.isfinite(want) if where is None else where
    assert torch.isfinite(out.float())[where].all()
    d = (out.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -11 * mag + 2.0 ** -36 * max(lens) * most + 2.0 ** -133  # (bf16's smallest steps)
    assert (d <= tol)[where].all(), float((d - tol)[where].max())
    rows = where.all(-1)
    seen = torch.isfinite(want_lse) & rows
    assert (lse[~torch.isfinite(want_lse) & rows] == -np.inf).all() and (out[~torch.isfinite(want_lse) & rows] == 0).all()
    assert ((lse.double() - want_lse)[seen].abs() <= 1e-5 * (4 + want_lse[seen].abs())).all()


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_marked_page_reaches_only_rows_that_see_it(cuda, form, which, bad):
    """The last token begins a page whose scale is not finite: the rows before it are what they are without that page."""
    R, page = form[1], 16
    lens = [16 * (R // 16 + 3) + 1, 16 * (R // 16 + 1) + 1]

    def edit(c, table):
        for b, n in enumerate(lens):
            for i in {"k": (2,), "v": (3,), "both": (2, 3)}[which]:
                c[i][table[b, n // page].long()] = bad

    out, lse, ref, cache, table = call(cuda, form, lens, edit=edit)
    last = torch.zeros(out.shape, dtype=torch.bool, device=cuda)
    last[:, -1] = True
    check(out, lse, ref, cache, table, lens, ~last)
    assert not torch.isfinite(out[:, -1].float()).any()


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_a_marked_page_that_the_window_hides(cuda, form):
    """Only the first row's window reaches back into the marked page."""
    R, window = form[1], 64
    lens = [160 + R, 97 + R] * (1 if form[0] == "stream" else 50 if R < 100 else 12)  # (work decides, and the window cuts it)

    def edit(c, table):
        for b, n in enumerate(lens):
            first = n - R - window + 1  # the first position that row 0 sees
            c[3][table[b, first // 16].long()] = float("nan")

    out, lse, ref, cache, table = call(cuda, form, lens, window=window, edit=edit)
    sees = ~torch.isfinite(ref[0])
    assert sees[:, 0].all() and (R < 20 or not sees[:, 16:].any())
    check(out, lse, ref, cache, table, lens)
    assert torch.isnan(out[sees]).all()


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("page", [16, 64])
def test_pages_outside_the_cache_are_skipped(cuda, form, page):
    """Positions of such a page do not count, whatever page 0 or an earlier step holds; a sequence of nothing else gives 0."""
    R = form[1]
    lens = [R + 7 * page + 5, R + 3 * page, R + 2]

    def edit(c, table):
        n = c[0].shape[0]
        table[0, 1], table[0, 4], table[1, 0] = -1, n, 1 << 30
        table[2] = -7
        for x in c[2:]:
            x[0] = 1e4  # page 0 shows where it is taken in

    ops.device_status()
    out, lse, ref, cache, table = call(cuda, form, lens, page=page, edit=edit, seed=3)
    assert ops.device_status() == (4, 7)
    assert torch.isfinite(ref[0]).all() and (ref[0][2] == 0).all()
    check(out, lse, ref, cache, table, lens)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("log2", [-70, -40, -30, -8, 20])
def test_pages_of_zeros_beside_pages_of_any_scale(cuda, form, log2):
    """A page whose V scale is 0 takes its softmax mass and adds nothing, whatever its codes are and however small the other
    pages' values are."""
    R = form[1]
    lens = [R + 150, R + 40]

    def edit(c, table):
        c[3].mul_(64 * 2.0 ** log2)
        for b in range(2):
            c[3][table[b, ::2].long()] = 0

    out, lse, ref, cache, table = call(cuda, form, lens, edit=edit, seed=4)
    check(out, lse, ref, cache, table, lens)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("scale", [3e-38, 1e-36, 1e-33, 1e-30, 1e25, 1e33])
def test_values_of_any_size(cuda, form, scale):
    """V scales over the range of what KvCacheWrite makes: tiny values keep their softmax and its sum."""
    lens = [form[1] + 900, form[1] + 3]

    def edit(c, table):
        c[3].mul_(64 * scale / 2)

    out, lse, ref, cache, table = call(cuda, form, lens, edit=edit, seed=5)
    check(out, lse, ref, cache, table, lens)
