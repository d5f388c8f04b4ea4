"""The operators on logits at the largest sizes that they take, on inputs whose results are known in closed form."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LAST = 2 ** 31 - 2  # the last token of the widest row


@pytest.fixture(autouse=True)
def released(supa):
    yield
    torch.supa.empty_cache()


@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
def test_distillation_of_the_widest_row(rest, no_fallback):
    """A student who thinks all tokens alike: q = 1 / vocab.  The sums of ones are exact in float32 (a thread's below 2^18, the
    whole a power of two within one rounding), so a logarithm is off by a few 2^-24 of itself, under 64 of 2^-24."""
    vocab = LAST + 1
    x = torch.zeros(1, vocab, dtype=torch.bfloat16, device="supa", requires_grad=True)
    at = [0, 131072, 33554431, 33554432, 2 ** 30 + 5, LAST - 1, LAST]
    i = torch.tensor([at])
    t = torch.tensor([[0.5, 1.0, -1.0, 0.0, 2.0, 1.5, -0.5]])
    lse = torch.logsumexp(t.double(), 1) + 0.25 if rest else None
    p = (t.double() - (torch.logsumexp(t.double(), 1, keepdim=True) if lse is None else lse[:, None])).exp()[0]
    loss = torch.supa.distillation_loss(x, i.to("supa"), t.to("supa"), teacher_lse=None if lse is None else lse.to("supa"))
    (g,) = torch.autograd.grad(loss, x, torch.tensor(1024.0, device="supa"))
    want = float((p * (p.log() + math.log(vocab))).sum())
    r = float(1 - p.sum()) if rest else 0.0
    if rest:
        want += r * (math.log(r) - math.log1p(-len(at) / vocab))
    assert abs(float(loss.detach()) - want) <= 64 * U
    for n, c in enumerate(at):
        w = (1 / vocab - float(p[n])) * 1024
        assert abs(float(g[0, c]) - w) <= abs(w) * (2.0 ** -8 + 64 * U), c
    other = (1 / vocab - (r / (vocab - len(at)) if rest else 0.0)) * 1024
    for c in (1, 8, 131071, 131073, 33554433, 2 ** 30, 2 ** 30 + 6, LAST - 2, LAST - 9):
        # with the rest it is a difference of a quarter or so of its terms
        assert abs(float(g[0, c]) - other) <= abs(other) * 2.0 ** -8 + 64 * U * 1024 / vocab, c


def test_adjustments_of_the_widest_row(no_fallback):
    vocab = 2 ** 29 - 1
    x = torch.ones(1, vocab, dtype=torch.float32, device="supa")
    said = [0, 32767, 32768, 2 ** 28 + 3, vocab - 1]
    tokens = torch.tensor([said + [vocab, 2 ** 33, -1, 7]])
    bias_tokens = torch.tensor([[vocab - 2, 7, 2 ** 28]])
    y = torch.supa.adjust_logits(x, tokens=tokens.to("supa"), repetition=2.0, presence=0.25, bias_tokens=bias_tokens.to("supa"),
                                 bias=torch.tensor([[4.0, 8.0, 16.0]], device="supa"))
    want = {c: 0.25 for c in said} | {vocab - 2: 5.0, 7: 8.25, 2 ** 28: 17.0}
    for c, v in want.items():
        assert float(y[0, c]) == v, c
    # all others are 1: the sum is theirs, of whole runs
    for lo in range(0, vocab, 2 ** 26):
        part = y[0, lo: lo + 2 ** 26].cpu()
        changed = [c - lo for c in want if lo <= c < lo + 2 ** 26]
        part[changed] = 1.0
        assert (part == 1).all(), lo


def test_balance_of_the_most_tokens(no_fallback):
    """One expert takes every token: its share is 1, the loss 1 and the gradient 0; whole numbers below 2^24 until float64."""
    tokens = 2 ** 31 - 1
    x = torch.ones(tokens, 1, dtype=torch.bfloat16, device="supa", requires_grad=True)
    e = torch.zeros(tokens, 1, dtype=torch.int32, device="supa")
    loss, counts = torch.supa.router_balance_loss(x, e)
    assert counts.cpu().tolist() == [tokens] and float(loss.detach()) == 1
    (g,) = torch.autograd.grad(loss, x)
    assert g.shape == x.shape
    for lo in range(0, tokens, 2 ** 28):
        assert not g[lo: lo + 2 ** 28].any().item(), lo
