"""Plain references of the attention-side ops for the tests: the definitions, in 64 bits where values are compared and in
single fp32 steps where bits are."""

from __future__ import annotations

import numpy as np
import torch


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_cache(pages, kv_heads, page, D, seed, device, spread=1.0):
    """Random codes and scales; page scales vary by 2^+-spread."""
    g = gen(seed)
    codes = [torch.randint(-127, 128, (pages, kv_heads, page, D), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [(torch.rand(pages, kv_heads, generator=g) * 2 - 1).mul(spread).exp2() / 64 for _ in range(2)]
    return [t.to(device).contiguous() for t in codes + scales]


def make_table(B, cols, pages, seed, device):
    return torch.randperm(pages, generator=gen(seed))[:B * cols].reshape(B, cols).to(torch.int32).to(device)


def dense(codes, scales, table_row, n):
    """float64 [n, kv_heads, D] of one sequence."""
    page = codes.shape[2]
    t = table_row[:-(-n // page)].long()
    x = codes[t].double() * scales[t].double()[..., None, None]
    return x.permute(0, 2, 1, 3).reshape(-1, codes.shape[1], codes.shape[3])[:n]


def attention(q, cache, table, lens, news, scale, window):
    """(out, sum of p |v|, lse) in float64, [B, R, heads, D] / [B, R, heads]."""
    k_c, v_c, k_s, v_s = cache
    B, R, H, D = q.shape
    Hk = k_c.shape[1]
    out = torch.zeros(B, R, H, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((B, R, H), -np.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lens[b])
        m = R if news is None else int(news[b])
        m = min(m, n, R)
        if m <= 0:
            continue
        k, v = dense(k_c, k_s, table[b], n), dense(v_c, v_s, table[b], n)
        for r in range(m):
            t = n - m + r
            lo = max(0, t - window + 1) if window else 0
            kk = k[lo:t + 1].repeat_interleave(H // Hk, 1)
            vv = v[lo:t + 1].repeat_interleave(H // Hk, 1)
            s = torch.einsum("hd,jhd->hj", q[b, r].double(), kk) * scale
            lse[b, r] = torch.logsumexp(s, -1)
            p = torch.softmax(s, -1)
            out[b, r] = torch.einsum("hj,jhd->hd", p, vv)
            mag[b, r] = torch.einsum("hj,jhd->hd", p, vv.abs())
    return out, mag, lse


def write(codes, scales, x, table, lens, news):
    """The definition of KvCacheWrite on one of K and V in fp32 steps, in place on numpy arrays; x float32 [B, R, H, D]."""
    f = np.float32
    B, R = x.shape[:2]
    page = codes.shape[2]
    for b in range(B):
        n = min(int(news[b]) if news is not None else R, R, int(lens[b]))
        if n <= 0:
            continue
        first = int(lens[b]) - n
        for i in range(first // page, -(-int(lens[b]) // page)):
            p, begin = int(table[b, i]), i * page
            t0, t1 = max(first, begin), min(int(lens[b]), begin + page)
            for h in range(codes.shape[1]):
                new = x[b, t0 - first:t1 - first, h]
                was = scales[p, h] if t0 > begin else f(0)
                a = np.abs(new).max() if np.isfinite(new).all() else f(np.nan)
                s = f(np.nan) if np.isnan(a) or np.isnan(was) else max(was, f(a / f(127)))
                if s < np.finfo(f).tiny:
                    s = f(0)
                with np.errstate(invalid="ignore"):
                    inv = f(1) / s if s > 0 else f(0)
                    ratio = f(was / s) if s > 0 else f(0)
                scales[p, h] = s
                if np.isnan(s):
                    continue  # codes of a page without a scale mean nothing
                codes[p, h, t0 - begin:t1 - begin] = np.rint((new * inv).astype(f)).astype(np.int8)
                if t0 > begin and s != was:
                    old = codes[p, h, :t0 - begin].astype(f)
                    codes[p, h, :t0 - begin] = np.rint((old * ratio).astype(f)).astype(np.int8)


def draft(p, q, x, u, us, drafts=None):
    """DraftVerify's definition with Python integers; numpy inputs."""
    B, R = x.shape
    V = p.shape[2]
    accepted, tokens = np.zeros(B, np.int32), np.full((B, R + 1), -1, np.int32)

    def mass(w):
        w = np.nan_to_num(w.astype(np.float32), nan=0.0, posinf=1.0, neginf=0.0).clip(0, 1)
        return [int(v) for v in np.floor(w.astype(np.float64) * 2.0 ** 38)]

    for b in range(B):
        most = R if drafts is None else max(0, min(R, int(drafts[b])))
        n = 0
        while n < most:
            t = int(x[b, n])
            if not 0 <= t < V:
                break
            qx = np.float32(1) if q is None else q[b, n, t]
            if not np.float32(u[b, n] * qx) < p[b, n, t]:
                break
            n += 1
        with np.errstate(invalid="ignore"):
            if n < most and q is not None:
                w = mass(p[b, n] - q[b, n])
            else:
                w = mass(p[b, n])
                if n < most and 0 <= x[b, n] < V:
                    w[int(x[b, n])] = 0
        if sum(w) == 0:
            w = mass(p[b, n])
        total, token = sum(w), -1
        if total:
            u24 = min(max(int(np.float32(us[b]) * 2.0 ** 24), 0), 2 ** 24 - 1)
            target, run = (total * u24) >> 24, 0
            for v in range(V):
                run += w[v]
                if run > target:
                    token = v
                    break
        accepted[b] = n
        tokens[b, :n] = x[b, :n]
        tokens[b, n] = token
    return accepted, tokens
