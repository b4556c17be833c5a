"""One attention layer decoding with drafted tokens: the products, norms, cache, attention and verification run together.

    python examples/verify_step.py            # needs a GPU; random weights, prints the tokens of a few steps

A step feeds every sequence its last token and R drafted ones:
    Q8Embed -> RmsNorm -> Q8Gemv (q, k, v) -> QkNormRope -> KvCacheWrite -> KvCacheAttention -> Q8Gemv -> SkipRmsNorm
    -> Q8Gemv (LM head) -> softmax -> DraftVerify
DraftVerify's counts say how many drafts stand: the cache's lengths go back by the rest (nothing is moved: their codes are
written over by the next step), and in a hybrid model they are the `state_row` of the next MambaVerify.
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from gguf_onnx_ops_b200 import ops  # noqa: E402


def q8_0(w: torch.Tensor) -> torch.Tensor:
    """Raw GGUF Q8_0 rows (fp16 d, 32 int8) of a float matrix [N, K]."""
    b = w.float().reshape(w.shape[0], -1, 32)
    d = (b.abs().amax(-1, keepdim=True) / 127).half()
    q = torch.where(d > 0, b / d.float(), 0.0).round().clamp(-127, 127).to(torch.int8)
    return torch.cat((d.contiguous().view(torch.uint8), q.view(torch.uint8)), -1).reshape(w.shape[0], -1).contiguous()


class Layer:
    """Random weights of one attention layer and a drafter's table."""

    def __init__(self, device, *, vocab=1000, hidden=512, heads=8, kv_heads=2, head_dim=64, max_pos=4096, seed=0):
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, scale=1.0):
            return torch.randn(*shape, generator=g) * scale

        self.device, self.vocab, self.hidden = device, vocab, hidden
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        width = heads * head_dim
        self.embed = q8_0(normal(vocab, hidden)).to(device)
        self.w_qkv = q8_0(normal((heads + 2 * kv_heads) * head_dim, hidden, scale=hidden ** -0.5)).to(device)
        self.w_out = q8_0(normal(hidden, width, scale=width ** -0.5)).to(device)
        self.w_head = q8_0(normal(vocab, hidden, scale=4 * hidden ** -0.5)).to(device)
        self.g_in, self.g_out = (torch.rand(hidden, generator=g).add(0.5).to(device) for _ in range(2))
        self.g_q, self.g_k = (torch.rand(head_dim, generator=g).add(0.5).to(device) for _ in range(2))
        freq = 10000.0 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
        angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * freq
        self.cos, self.sin = angle.cos().float().to(device), angle.sin().float().to(device)


class Sequences:
    """The cache of B sequences and how far each has come."""

    def __init__(self, layer: Layer, batch: int, tokens: int, page: int = 32):
        cols = -(-tokens // page)
        self.cache = ops.KvCache.empty(batch * cols, layer.kv_heads, page, layer.head_dim, layer.device)
        self.table = torch.randperm(batch * cols).reshape(batch, cols).to(torch.int32).to(layer.device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=layer.device)


def forward(layer: Layer, seqs: Sequences, tokens: torch.Tensor) -> torch.Tensor:
    """Feeds tokens int64 [B, R] (B * R <= 16) at the sequences' ends; returns the target's probabilities f32 [B, R, vocab]."""
    B, R = tokens.shape
    H, Hk, D = layer.heads, layer.kv_heads, layer.head_dim
    seqs.lens += R
    positions = (seqs.lens[:, None] - R + torch.arange(R, dtype=torch.int32, device=layer.device)).reshape(-1).contiguous()
    x = ops.Q8Embed(layer.embed, tokens).reshape(B * R, -1)
    qkv = ops.Q8Gemv(ops.RmsNorm(x, layer.g_in), layer.w_qkv)
    q, k = ops.QkNormRope(qkv, layer.g_q, layer.g_k, layer.cos, layer.sin, positions, heads=H, kv_heads=Hk)
    v = qkv.view(B, R, H + 2 * Hk, D)[:, :, H + Hk:]  # where the projection left it
    ops.KvCacheWrite(k.view(B, R, Hk, D), v, seqs.cache, seqs.table, seqs.lens)
    o = ops.KvCacheAttention(q.view(B, R, H, D), seqs.cache, seqs.table, seqs.lens)
    y, _ = ops.SkipRmsNorm(ops.Q8Gemv(o.view(B * R, H * D), layer.w_out), x, layer.g_out)
    return torch.softmax(ops.Q8Gemv(y, layer.w_head).float(), -1).view(B, R, -1)


def verify(layer: Layer, seqs: Sequences, last: torch.Tensor, drafts: torch.Tensor, draft_probs, u, u_sample):
    """One step: last int32 [B], drafts int32 [B, R], draft_probs f32 [B, R, vocab] or None.  Returns DraftVerify's
    (accepted [B], tokens [B, R + 1]); the cache keeps the last token and the drafts that stand."""
    R = drafts.shape[1]
    p = forward(layer, seqs, torch.cat((last[:, None], drafts), 1).long())
    accepted, tokens = ops.DraftVerify(p.contiguous(), draft_probs, drafts, u, u_sample)
    seqs.lens -= R - accepted
    return accepted, tokens


def draft(layer: Layer, last: torch.Tensor, count: int, g: torch.Generator):
    """`count` tokens after last int32 [B], drafted by the model without its attention layer, and their distributions."""
    tokens, probs = [], []
    for _ in range(count):
        x = ops.Q8Embed(layer.embed, last.long())
        q = torch.softmax(ops.Q8Gemv(ops.RmsNorm(x, layer.g_out), layer.w_head).float(), -1)
        last = torch.multinomial(q, 1, generator=g)[:, 0].to(torch.int32)
        tokens.append(last)
        probs.append(q)
    return torch.stack(tokens, 1).contiguous(), torch.stack(probs, 1).contiguous()


def main():
    dev = torch.device("cuda:0")
    layer = Layer(dev)
    B, R, steps = 2, 3, 6
    seqs = Sequences(layer, B, 256)
    g = torch.Generator(device=dev).manual_seed(1)
    prompt = torch.randint(0, layer.vocab, (B, 8), generator=g, device=dev)
    last = forward(layer, seqs, prompt)[:, -1].argmax(-1).to(torch.int32)
    for i in range(steps):
        drafts, q = draft(layer, last, R, g)
        accepted, tokens = verify(layer, seqs, last, drafts, q, torch.rand(B, R, generator=g, device=dev),
                                  torch.rand(B, generator=g, device=dev))
        last = tokens.gather(1, accepted.long()[:, None])[:, 0]
        print(f"step {i}: accepted {accepted.tolist()}, tokens {tokens.tolist()}, lengths {seqs.lens.tolist()}")


if __name__ == "__main__":
    main()
