"""examples/verify_step.py: the attention-side ops with the products and norms around them.

Greedy decoding token by token must come out the same when the tokens are drafted and verified several at a time: with a
certain drafter that proposes exactly those tokens all of them stand, with a wrong one none from it on, and the cache
that a rollback leaves serves the next step.  The target's distributions are made one-hot (their best token), so the random
numbers do not matter; a token whose two best candidates are within 2 % is left out of the comparison (the cache's
rounding depends on how many tokens a write brings)."""

import importlib.util
import os

import pytest
import torch

from gguf_onnx_ops_b200 import ops

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("verify_step", os.path.join(ROOT, "examples", "verify_step.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_drafted_tokens_reproduce_plain_decoding(cuda, ex):
    layer = ex.Layer(cuda, seed=3)
    g = torch.Generator(device=cuda).manual_seed(4)
    prompt = torch.randint(0, layer.vocab, (1, 12), generator=g, device=cuda)
    n = 24
    seqs = ex.Sequences(layer, 1, 128)
    p = ex.forward(layer, seqs, prompt)[:, -1]
    plain, clear = [], []
    for _ in range(n):
        top = p.topk(2, -1).values[0]
        clear.append(bool(top[0] > 1.02 * top[1]))
        plain.append(int(p.argmax(-1)))
        p = ex.forward(layer, seqs, torch.tensor([[plain[-1]]], device=cuda))[:, -1]
    assert all(clear), "choose another seed: two candidates too near"

    class Greedy:  # one-hot target rows
        def __init__(self, p):
            self.p = torch.nn.functional.one_hot(p.argmax(-1), p.shape[-1]).float()

    seqs = ex.Sequences(layer, 1, 128)
    first = int(ex.forward(layer, seqs, prompt)[:, -1].argmax(-1))
    got, wrong_at, step = [first], {2: 1, 4: 0}, 0  # in steps 2 and 4 the drafter is wrong at draft 1 and 0
    while len(got) < n:
        R = min(5, n - len(got))
        drafts = [plain[len(got) + i] for i in range(R)]
        bad = wrong_at.get(step, R)
        if bad < R:
            drafts[bad] = (drafts[bad] + 1) % layer.vocab
        d = torch.tensor([drafts], dtype=torch.int32, device=cuda)
        before = int(seqs.lens)
        probs = ex.forward(layer, seqs, torch.tensor([[got[-1]] + drafts], device=cuda))
        accepted, tokens = ops.DraftVerify(Greedy(probs).p, None, d, torch.full((1, R), 0.5, device=cuda),
                                           torch.tensor([0.7], device=cuda))
        seqs.lens -= R - accepted
        a = int(accepted)
        assert a == min(bad, R) and int(seqs.lens) == before + 1 + a
        got += tokens[0, :a + 1].tolist()
        step += 1
    assert got[:n] == plain
    assert ops.device_status()[0] == 0


def test_counts_start_the_next_mamba_state(cuda, ex):
    """accepted is what MambaVerify takes as its state row: int32 on the device, usable without a copy to the host."""
    layer = ex.Layer(cuda, seed=5)
    seqs = ex.Sequences(layer, 2, 64)
    prompt = torch.randint(0, layer.vocab, (2, 8), device=cuda)
    p = ex.forward(layer, seqs, prompt)[:, -1]
    last = p.argmax(-1).to(torch.int32)
    q = p[:, None].expand(2, 3, -1).contiguous()
    drafts = torch.multinomial(q.view(6, -1), 1).view(2, 3).to(torch.int32)
    accepted, tokens = ex.verify(layer, seqs, last, drafts, q, torch.rand(2, 3, device=cuda), torch.rand(2, device=cuda))
    heads, groups, rows = 8, 1, 4
    di, cd = heads * 64, heads * 64 + 2 * groups * 128
    proj = torch.randn(1, di + cd + heads, device=cuda).to(torch.bfloat16)
    conv = torch.randn(rows, cd, 3, device=cuda).to(torch.bfloat16)
    ssm = torch.randn(rows, heads, 128, 64, device=cuda)
    args = (torch.randn(cd, 4, device=cuda).to(torch.bfloat16), torch.randn(cd, device=cuda).to(torch.bfloat16),
            torch.randn(heads, device=cuda), -torch.rand(heads, device=cuda), torch.randn(heads, device=cuda),
            torch.rand(di, device=cuda))
    row = accepted[:1]
    y = ops.MambaVerify(proj, conv, ssm, *args, row, heads=heads, n_groups=groups)[0]
    k = int(row)
    ref = ops.MambaStep(proj, conv[k:k + 1].contiguous(), ssm[k:k + 1].contiguous(), *args, heads=heads, n_groups=groups)[0]
    assert torch.equal(y, ref)
    assert ((tokens >= 0).sum(1) == accepted + 1).all()


def test_example_runs(cuda, ex, capsys):
    ex.main()
    assert capsys.readouterr().out.count("accepted") == 6
