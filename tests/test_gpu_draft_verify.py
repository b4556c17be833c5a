"""DraftVerify against its definition with Python integers: accepted counts and tokens are equal."""

import numpy as np
import pytest
import torch

from gguf_onnx_ops_b200 import ops
from tests import kv_ref as K

pytestmark = pytest.mark.gpu


def make(B, R, V, seed, sharp=3.0, noise=0.7):
    g = K.gen(seed)
    logits = torch.randn(B, R + 1, V, generator=g) * sharp
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits[:, :R] + noise * torch.randn(B, R, V, generator=g), -1)
    x = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, R).to(torch.int32)
    return p, q, x, torch.rand(B, R, generator=g), torch.rand(B, generator=g)


def run_case(cuda, p, q, x, u, us, drafts=None):
    dev = [None if t is None else t.to(cuda).contiguous() for t in (p, q, x, u, us, drafts)]
    accepted, tokens = ops.DraftVerify(*dev)
    ra, rt = K.draft(p.numpy(), None if q is None else q.numpy(), x.numpy(), u.numpy(), us.numpy(),
                     None if drafts is None else drafts.numpy())
    assert np.array_equal(accepted.cpu().numpy(), ra)
    assert np.array_equal(tokens.cpu().numpy(), rt)
    return ra, rt


@pytest.mark.parametrize("B,R,V", [(1, 1, 1), (2, 1, 2), (3, 4, 33), (5, 3, 128), (4, 8, 1000), (2, 32, 515), (64, 5, 257),
                                   (3, 2, 32000), (2, 3, 50257), (1, 2, 131072)])
def test_shapes(cuda, B, R, V):
    p, q, x, u, us = make(B, R, V, B + R + V)
    run_case(cuda, p, q, x, u, us)
    run_case(cuda, p, None, x, u, us)
    n = torch.tensor([i % (R + 1) for i in range(B)], dtype=torch.int32)
    run_case(cuda, p, q, x, u, us, n)
    run_case(cuda, p, None, x, u * 0.1, us, n)


def test_all_and_none_stand(cuda):
    p, q, x, u, us = make(6, 4, 100, 1)
    a, t = run_case(cuda, p, p[:, :4].contiguous(), x, u, us)  # the drafter is the target: u q < q
    assert (a == 4).all()
    zero = p.clone()
    zero[:, :4].scatter_(2, x.long()[..., None], 0.0)
    a, t = run_case(cuda, zero, q, x, u * 0, us)  # a token without probability never stands, even at u = 0
    assert (a == 0).all() and (t[:, 1:] == -1).all()


def test_random_numbers_at_the_edges(cuda):
    p, q, x, u, _ = make(4, 2, 77, 2)
    for v in (0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, 0.5):
        run_case(cuda, p, q, x, u, torch.full((4,), v))


def test_one_token_holds_everything(cuda):
    """Greedy rows (all mass on one token), its last token among them, and rows with a huge tail of zeros."""
    V = 4099
    p = torch.zeros(3, 3, V)
    p[0, :, 17] = 1
    p[1, :, V - 1] = 1
    p[2, :, 0] = 1
    x = torch.tensor([[17, 17], [V - 1, 3], [5, 0]], dtype=torch.int32)
    us = torch.tensor([0.3, 0.999, 0.0])
    a, t = run_case(cuda, p, None, x, torch.full((3, 2), 0.999), us)
    assert a.tolist() == [2, 1, 0] and t[:, :].tolist() == [[17, 17, 17], [V - 1, V - 1, -1], [0, -1, -1]]


def test_empty_residuals_and_rows(cuda):
    p = torch.zeros(4, 2, 50)
    q = torch.full((4, 1, 50), 0.02)
    p[0, 0, 7] = 0.01  # below q everywhere: the residual is empty, the target's own row is drawn from
    p[2, 0] = float("nan")
    p[3, 0, 4] = float("inf")
    p[3, 1, 4] = 1e30
    x = torch.tensor([[3], [3], [3], [99]], dtype=torch.int32)  # the last is no token at all
    _, t = run_case(cuda, p, q, x, torch.full((4, 1), 0.5), torch.full((4,), 0.4))
    assert t[0, 0] == 7 and t[1, 0] == -1 and t[2, 0] == -1 and t[3, 0] == 4


def test_draws_follow_the_distribution(cuda):
    """20000 sequences of one drafted token: the tokens' frequencies are the target's (five standard deviations)."""
    B, V = 20000, 8
    g = K.gen(5)
    p = torch.softmax(torch.randn(V, generator=g), 0)
    q = torch.softmax(torch.randn(V, generator=g), 0)
    x = torch.multinomial(q, B, replacement=True, generator=g).view(B, 1).to(torch.int32)
    _, t = ops.DraftVerify(p.expand(B, 2, V).contiguous().to(cuda), q.expand(B, 1, V).contiguous().to(cuda), x.to(cuda),
                           torch.rand(B, 1, generator=g).to(cuda), torch.rand(B, generator=g).to(cuda))
    freq = torch.bincount(t[:, 0].cpu().long(), minlength=V).double() / B
    assert ((freq - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / B).sqrt()).all()


def test_empty_batch_and_refusals(cuda):
    p, q, x, u, us = (t.to(cuda) for t in make(2, 3, 64, 9))
    a, t = ops.DraftVerify(p[:0], q[:0], x[:0], u[:0], us[:0])
    assert a.shape == (0,) and t.shape == (0, 4)
    with pytest.raises(ValueError, match="R \\+ 1"):
        ops.DraftVerify(p[:, :3].contiguous(), q, x, u, us)
    with pytest.raises(ValueError, match="draft_probs must be"):
        ops.DraftVerify(p, p, x, u, us)
    with pytest.raises(ValueError, match="float32"):
        ops.DraftVerify(p.half(), q, x, u, us)
    with pytest.raises(ValueError, match="int32"):
        ops.DraftVerify(p, q, x.long(), u, us)
    with pytest.raises(ValueError, match="drafts must have"):
        ops.DraftVerify(p, q, x, u, us, x[0])
    with pytest.raises(ValueError, match=r"\[1, 32\]"):
        ops.DraftVerify(p.repeat(1, 12, 1)[:, :34].contiguous(), None, x.repeat(1, 11), u.repeat(1, 11), us)
