"""The operators of a decode / verify step's attention side, as measured cases.

QkNormRope (head norms and position rotation), KvCacheWrite / KvCacheRead (8-bit paged cache, one scale
for each page and head), KvCacheAttention (attention over that cache) and DraftVerify (which drafted
tokens stand).  ``run`` computes a case with elementary torch operations where ``own`` is false, and
through the library's public functions where it is true.
"""

import math
import random

import torch

own = False

DEV = "cuda"
BF16_B, F32_B = 2, 4
MAX_POS = 16384


def listed():
    rope = {"op": "norm_rope", "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False}
    write = {"op": "cache_write", "kv_heads": 8, "dim": 128, "page": 64}
    attn = {"op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "ragged": False}
    return [
        # one token of one sequence: the call's latency
        {**rope, "name": "norm_rope_token", "tokens": 1},
        # the tokens of a few prompts at once, larger than the L2
        {**rope, "name": "norm_rope_prompt", "tokens": 8191},
        # 64 sequences decoding: one token each into pages that are partly full, the last page's worth read back
        {**write, "name": "cache_write_token", "batch": 64, "rows": 1, "lo": 37, "hi": 4001, "back": 64},
        # three prompts written whole into empty pages and read back
        {**write, "name": "cache_write_prompt", "batch": 3, "rows": 5003, "lo": 5003, "hi": 5003, "back": 5003},
        # one sequence, short context: the call's latency
        {**attn, "name": "attn_token_short", "batch": 1, "rows": 1, "lo": 777, "hi": 777},
        # a serving batch with contexts of all lengths
        {**attn, "name": "attn_token_batch", "batch": 64, "rows": 1, "lo": 131, "hi": 8009},
        # one sequence, long context: the work is split over its length
        {**attn, "name": "attn_token_long", "batch": 1, "rows": 1, "lo": 131071, "hi": 131071},
        # drafted tokens verified, some sequences with fewer drafts than others; 8 query heads on each kv head
        {**attn, "name": "attn_verify", "batch": 16, "rows": 6, "heads": 64, "lo": 801, "hi": 9001, "ragged": True},
        # narrow heads, an odd group, small pages and a sliding window
        {**attn, "name": "attn_window", "batch": 32, "rows": 3, "heads": 20, "kv_heads": 4, "dim": 64, "page": 16,
         "lo": 1, "hi": 20011, "window": 4096},
        # a prompt continued by a long chunk over what the cache holds: matrix products
        {**attn, "name": "attn_chunk", "batch": 1, "rows": 1001, "lo": 9001, "hi": 9001},
        # one sequence, small vocabulary: the call's latency
        {"op": "draft_verify", "name": "draft_verify_one", "batch": 1, "rows": 5, "vocab": 32000},
        # a serving batch at this library's LM-head width
        {"op": "draft_verify", "name": "draft_verify_batch", "batch": 64, "rows": 7, "vocab": 131072},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["norm_rope", "cache_write", "attention", "attention", "draft_verify"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "norm_rope":
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
        tokens = max(1, min(_spread(rng, 1, 8191), 8191 * 40 * 128 // ((heads + kv_heads) * dim)))
        return {"op": op, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.3}
    if op == "cache_write":
        batch, rows = _spread(rng, 1, 64), _spread(rng, 1, 5003)
        most = 3 * 5003 * 8 * 128
        rows = max(1, min(rows, most // (batch * kv_heads * dim)))
        lo = rows + rng.choice([0, 0, 1, 17, 64])
        hi = lo + rng.randint(0, 999)
        return {"op": op, "kv_heads": kv_heads, "dim": dim, "page": page, "batch": batch, "rows": rows, "lo": lo,
                "hi": hi, "back": min(hi, rows + page - 1)}
    if op == "attention":
        group = rng.choice([1, 2, 4, 5, 7, 8])
        rows = rng.choice([1, 1, 1, 2, 3, 5, 8, 16, _spread(rng, 17, 1001)])
        batch = _spread(rng, 1, 64) if rows <= 16 else rng.choice([1, 1, 2])
        hi = max(rows, _spread(rng, 32, 131071))
        hi = max(rows, min(hi, 64 * 4070 * 8 * 128 // (batch * kv_heads * dim)))  # no more cache than the listed batch
        # nor more work than the listed chunk
        hi = max(rows, min(hi, 1001 * 8500 * 32 * 128 // (batch * rows * kv_heads * group * dim)))
        return {"op": op, "batch": batch, "rows": rows, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "page": page, "lo": rng.choice([hi, max(1, hi // 8), max(1, hi // 2)]), "hi": hi,
                "window": rng.choice([0, 0, 0, 128, 1024]), "ragged": rng.random() < 0.3}
    batch, rows, vocab = _spread(rng, 1, 64), rng.randint(1, 8), _spread(rng, 1000, 131072)
    return {"op": op, "batch": batch, "rows": min(rows, 7), "vocab": vocab}


def _lens(case):
    """Context lengths, evenly from lo to hi; the seed only changes their order."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [lo + (hi - lo) * i // max(1, b - 1) if b > 1 else hi for i in range(b)]


def _news(case):
    """New tokens of each sequence (ragged: 1 .. rows in turn; never more than its length)."""
    r = case["rows"]
    return [min(n, r - i % r if case.get("ragged") else r) for i, n in enumerate(_lens(case))]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _pages(case, lens, g):
    """A pool of pages with one spare, and a table that takes its pages in random order."""
    per = -(-max(lens) // case["page"])
    pool = case["batch"] * per + 1
    table = torch.randperm(pool - 1, generator=g, device=DEV).to(torch.int32).reshape(case["batch"], per)
    return pool, table


def _codes(shape, g):
    """Codes as a quantised normal distribution leaves them."""
    out = torch.empty(shape, dtype=torch.int8, device=DEV)
    flat, step = out.view(-1), 1 << 26
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), generator=g, device=DEV).mul_(32).round_().clamp_(-127, 127))
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "norm_rope":
        t, hq, hk, d, rot = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rot"]
        s["qkv"] = torch.randn(t, (hq + 2 * hk) * d, generator=g, device=DEV).to(torch.bfloat16)
        s["gq"] = torch.rand(d, generator=g, device=DEV) + 0.5
        s["gk"] = torch.rand(d, generator=g, device=DEV) + 0.5
        freq = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
        angle = torch.arange(MAX_POS, device=DEV, dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["pos"] = torch.randint(0, MAX_POS, (t,), generator=g, device=DEV, dtype=torch.int32)
        return s
    if op == "draft_verify":
        b, r, v = case["batch"], case["rows"], case["vocab"]
        logits = torch.randn(b, r + 1, v, generator=g, device=DEV) * 3
        noise = torch.randn(b, r, v, generator=g, device=DEV)
        s["p"] = torch.softmax(logits, -1)
        s["q"] = torch.softmax(logits[:, :r] + 0.5 * noise, -1)
        del logits, noise
        s["draft"] = torch.multinomial(s["q"].view(b * r, v), 1, generator=g).view(b, r).to(torch.int32)
        s["u"] = torch.rand(b, r, generator=g, device=DEV)
        s["us"] = torch.rand(b, generator=g, device=DEV)
        return s
    hk, d, page, b, r = case["kv_heads"], case["dim"], case["page"], case["batch"], case["rows"]
    order = torch.randperm(b, generator=g, device=DEV)
    lens = _lens(case)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)[order].contiguous()
    s["new"] = torch.tensor(_news(case), dtype=torch.int32, device=DEV)[order].contiguous()
    s["most"] = max(lens)
    pool, s["table"] = _pages(case, lens, g)
    s["k"], s["v"] = _codes((pool, hk, page, d), g), _codes((pool, hk, page, d), g)
    s["ks"] = (torch.rand(pool, hk, generator=g, device=DEV) + 0.5) / 32
    s["vs"] = (torch.rand(pool, hk, generator=g, device=DEV) + 0.5) / 32
    if op == "cache_write":
        kv = torch.randn(b, r, 2, hk, d, generator=g, device=DEV).to(torch.bfloat16)  # as one projection leaves them
        s["nk"], s["nv"] = kv[:, :, 0], kv[:, :, 1]
    else:
        s["q"] = (2 * torch.randn(b, r, case["heads"], d, generator=g, device=DEV)).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _rotate(y, cos, sin, rot, interleaved):
    """Rotates the first `rot` of each head's values; y [T, H, D], cos and sin [T, 1, rot/2]."""
    x = y[..., :rot]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((r, y[..., rot:]), -1)


def _plain_norm_rope(s):
    c = s["case"]
    t, hq, hk, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].float().view(t, hq + 2 * hk, d)[:, :hq + hk]
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    y = torch.cat((y[:, :hq] * s["gq"], y[:, hq:] * s["gk"]), 1)
    pos = s["pos"].long()
    y = _rotate(y, s["cos"][pos][:, None], s["sin"][pos][:, None], c["rot"], c["interleaved"]).to(torch.bfloat16)
    return y[:, :hq].contiguous(), y[:, hq:].contiguous()


def _write_one(x, codes, scales, pages, pos, first, lens):
    """One of K and V: x [B, R, H, D] at positions first .. lens - 1, into the touched pages [B, N], pos [B, N, page]."""
    b, r = x.shape[:2]
    new = (pos >= first[:, None, None]) & (pos < lens[:, None, None])
    old = (pos < first[:, None, None]) & (pos[:, :, :1] < first[:, None, None])
    at = (pos - first[:, None, None]).clamp(0, r - 1)
    xf = x.float()[torch.arange(b, device=x.device)[:, None, None], at].permute(0, 1, 3, 2, 4)  # [B, N, H, page, D]
    isn, iso = new[:, :, None, :, None], old[:, :, None, :, None]
    amax = torch.where(isn, xf.abs(), 0.0).amax((-1, -2))
    was = torch.where(old[:, :, :1].expand(-1, -1, amax.shape[2]), scales[pages], 0.0)
    scale = torch.maximum(was, amax / 127.0)
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, 0.0, scale)
    some = scale > 0
    inv = torch.where(some, 1.0 / scale, 0.0)[..., None, None]
    ratio = torch.where(some, was / scale, 0.0)[..., None, None]
    have = codes[pages]
    fresh = (xf * inv).round().clamp(-127, 127)
    kept = (have.float() * ratio).round()
    codes[pages] = torch.where(isn, fresh, torch.where(iso, kept, have.float())).to(torch.int8)
    scales[pages] = scale


def _read_one(codes, scales, table, at, ok):
    """bf16 values of positions at [B, rows] (ok: those that exist) as [B, rows, H, D]."""
    page = codes.shape[2]
    p = table.long().gather(1, at // page)
    x = codes[p, :, at % page].float() * scales[p][..., None]
    return torch.where(ok[..., None, None], x, 0.0).to(torch.bfloat16)


def _plain_write(s):
    c = s["case"]
    page, r, n = c["page"], c["rows"], s["table"].shape[1]
    lens, first = s["lens"].long(), (s["lens"] - s["new"]).long()
    touched = (r + page - 2) // page + 1
    index = first[:, None] // page + torch.arange(touched, device=DEV)
    spare = s["k"].shape[0] - 1  # pages past the sequence's end go to the pool's spare page
    pages = torch.where(index * page < lens[:, None], s["table"].long().gather(1, index.clamp(max=n - 1)), spare)
    pos = index[..., None] * page + torch.arange(page, device=DEV)
    _write_one(s["nk"], s["k"], s["ks"], pages, pos, first, lens)
    _write_one(s["nv"], s["v"], s["vs"], pages, pos, first, lens)
    at = lens[:, None] - c["back"] + torch.arange(c["back"], device=DEV)
    ok = at >= 0
    at = at.clamp(min=0)
    return _read_one(s["k"], s["ks"], s["table"], at, ok), _read_one(s["v"], s["vs"], s["table"], at, ok)


def _sequence(codes, scales, table):
    """The cache's values of every sequence, f32 [B, H, tokens, D]."""
    t = table.long()
    x = codes[t].float() * scales[t][..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _seen(c, lens, new, tokens):
    """[B, R, tokens]: which tokens each row sees."""
    row, j = torch.arange(c["rows"], device=DEV), torch.arange(tokens, device=DEV)
    pos = (lens - new)[:, None] + row
    see = (j <= pos[..., None]) & (row < new[:, None])[..., None]
    return see & (j > pos[..., None] - c["window"]) if c["window"] else see


def _plain_attention(s):
    c = s["case"]
    b, r, hq, hk, d = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["dim"]
    k, v = _sequence(s["k"], s["ks"], s["table"]), _sequence(s["v"], s["vs"], s["table"])
    q = s["q"].float().view(b, r, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    score = (q @ k.transpose(-1, -2)) * d ** -0.5  # [B, Hk, G * R, tokens]
    see = _seen(c, s["lens"].long(), s["new"].long(), k.shape[2])
    score = score.view(b, hk, hq // hk, r, -1).masked_fill_(~see[:, None, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(m.isinf(), 0.0, m)).exp_()
    total = score.sum(-1, keepdim=True)
    o = (score.view(b, hk, -1, k.shape[2]) @ v).view(b, hk, hq // hk, r, d) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, r, hq, d).to(torch.bfloat16)


def _plain_draft(s):
    p, q, x = s["p"], s["q"], s["draft"].long()
    b, r = x.shape
    at = torch.arange(b, device=DEV)
    px, qx = p[:, :r].gather(2, x[..., None])[..., 0], q.gather(2, x[..., None])[..., 0]
    stand = (s["u"] * qx < px).int().cumprod(1).sum(1)  # drafts before the first that does not stand
    row = torch.where((stand < r)[:, None], q[at, stand.clamp(max=r - 1)], 0.0)
    rest = (p[at, stand] - row).clamp(0, 1)
    w = (rest.double() * 2.0 ** 38).floor().long().cumsum(1)
    w = torch.where(w[:, -1:] > 0, w, (p[at, stand].clamp(0, 1).double() * 2.0 ** 38).floor().long().cumsum(1))
    total = w[:, -1]
    u = (s["us"] * 2.0 ** 24).long().clamp(0, (1 << 24) - 1)
    target = (total >> 24) * u + (((total & ((1 << 24) - 1)) * u) >> 24)
    token = (w <= target[:, None]).sum(1)
    i = torch.arange(r + 1, device=DEV)
    out = torch.cat((x, x[:, :1]), 1)
    out = torch.where(i < stand[:, None], out, torch.where(i == stand[:, None], token[:, None], -1))
    return stand.to(torch.int32), out.to(torch.int32)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _own(s):
    from gguf_onnx_ops_b200 import ops

    c = s["case"]
    if c["op"] == "norm_rope":
        return ops.QkNormRope(s["qkv"], s["gq"], s["gk"], s["cos"], s["sin"], s["pos"], heads=c["heads"],
                              kv_heads=c["kv_heads"], epsilon=1e-6, interleaved=c["interleaved"])
    if c["op"] == "draft_verify":
        return ops.DraftVerify(s["p"], s["q"], s["draft"], s["u"], s["us"])
    if "cache" not in s:
        s["cache"] = ops.KvCache(s["k"], s["v"], s["ks"], s["vs"])
    if c["op"] == "cache_write":
        ops.KvCacheWrite(s["nk"], s["nv"], s["cache"], s["table"], s["lens"], s["new"])
        return ops.KvCacheRead(s["cache"], s["table"], s["lens"], rows=c["back"])
    return ops.KvCacheAttention(s["q"], s["cache"], s["table"], s["lens"], s["new"], window=c["window"])


def run(state):
    if own:
        return _own(state)
    plain = {"norm_rope": _plain_norm_rope, "cache_write": _plain_write, "attention": _plain_attention,
             "draft_verify": _plain_draft}
    return plain[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "norm_rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        tables = min(case["tokens"], MAX_POS) * case["rot"] * F32_B
        return {"bytes": 2 * n * BF16_B + tables + case["tokens"] * 4 + 2 * case["dim"] * F32_B, "flops": 10 * n}
    if op == "draft_verify":
        # the drafted tokens' probabilities, and one row of the target's and one of the drafter's
        b, r = case["batch"], case["rows"]
        return {"bytes": b * (2 * case["vocab"] * F32_B + r * 5 * 4 + 4 + 8), "flops": b * 4 * case["vocab"]}
    lens, news, page = _lens(case), _news(case), case["page"]
    if op == "cache_write":
        row = 2 * case["kv_heads"] * case["dim"]  # K and V
        back = sum(min(n, case["back"]) for n in lens)
        scales = sum(-(-n // page) - (n - m) // page for n, m in zip(lens, news)) * 2 * case["kv_heads"] * F32_B
        return {"bytes": sum(news) * row * (BF16_B + 1) + back * row + case["batch"] * case["back"] * row * BF16_B + 2 * scales,
                "flops": (sum(news) * 3 + back) * row}
    seen = pairs = 0
    for n, m in zip(lens, news):
        w = case["window"] or n
        seen += min(n, w + m - 1)
        pairs += sum(min(n - m + i + 1, w) for i in range(m))
    kv = seen * 2 * case["kv_heads"] * (case["dim"] + F32_B / page)
    rows = case["batch"] * case["rows"] * case["heads"] * case["dim"]
    return {"bytes": kv + 2 * rows * BF16_B, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------------------------
# in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "draft_verify":
        return None  # whole numbers
    if op == "norm_rope":
        hq, hk, d, rot = case["heads"], case["kv_heads"], case["dim"], case["rot"]
        x = s["qkv"].double().reshape(-1, hq + 2 * hk, d)[:, :hq + hk]
        gamma = torch.cat((s["gq"].double().expand(hq, d), s["gk"].double().expand(hk, d)))
        y = x / (x.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * gamma
        z = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
        if case["interleaved"]:
            w = torch.view_as_complex(y[..., :rot].reshape(*y.shape[:-1], rot // 2, 2).contiguous()) * z
            y[..., :rot] = torch.view_as_real(w).flatten(-2)
        else:
            w = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * z
            y[..., :rot // 2], y[..., rot // 2:rot] = w.real, w.imag
        return y[:, :hq].contiguous(), y[:, hq:].contiguous()
    lens, news, page = s["lens"].tolist(), s["new"].tolist(), case["page"]
    if op == "cache_write":
        outs = []
        for x, codes, scales in ((s["nk"], s["k"], s["ks"]), (s["nv"], s["v"], s["vs"])):
            out = torch.zeros(case["batch"], case["back"], case["kv_heads"], case["dim"], dtype=torch.float64, device=DEV)
            for b, (n, m) in enumerate(zip(lens, news)):
                whole = torch.zeros(n, case["kv_heads"], case["dim"], dtype=torch.float64, device=DEV)
                for i in range(max(0, n - case["back"]) // page, -(-n // page)):
                    p, begin, end = int(s["table"][b, i]), i * page, min(n, (i + 1) * page)
                    was, first = scales[p].double(), max(begin, n - m)
                    if first >= end:
                        whole[begin:end] = (codes[p, :, :end - begin].double() * was[:, None, None]).transpose(0, 1)
                        continue
                    fresh = x[b, first - (n - m):end - (n - m)].double()
                    now = fresh.abs().amax((0, 2)).div(127)
                    now = (torch.maximum(now, was) if first > begin else now).float().double()  # a scale is held in f32
                    whole[first:end] = (fresh / now[:, None]).round().clamp(-127, 127) * now[:, None]
                    if first > begin:
                        held = codes[p, :, :first - begin].double() * (was / now)[:, None, None]
                        whole[begin:first] = (held.round() * now[:, None, None]).transpose(0, 1)
                tail = whole[max(0, n - case["back"]):]
                out[b, case["back"] - len(tail):] = tail
            outs.append(out)
        return tuple(outs)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(case["batch"], case["rows"], hq, d, dtype=torch.float64, device=DEV)
    for b, (n, m) in enumerate(zip(lens, news)):
        t = s["table"][b, :-(-n // page)].long()
        low = max(0, n - m - case["window"] + 1) if case["window"] else 0
        pos = torch.arange(n - m, n, device=DEV)[:, None]
        j = torch.arange(low, n, device=DEV)
        hide = (j > pos) | (j <= pos - case["window"]) if case["window"] else j > pos
        for h in range(hk):
            k = (s["k"][t, h].double() * s["ks"][t, h].double()[:, None, None]).reshape(-1, d)[low:n]
            v = (s["v"][t, h].double() * s["vs"][t, h].double()[:, None, None]).reshape(-1, d)[low:n]
            for e in range(h * hq // hk, (h + 1) * hq // hk):
                score = (s["q"][b, :m, e].double() @ k.T / math.sqrt(d)).masked_fill(hide, -math.inf)
                out[b, :m, e] = torch.softmax(score, -1) @ v
    return out
