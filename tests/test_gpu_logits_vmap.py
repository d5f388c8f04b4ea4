"""The operators on logits under torch.vmap: each sample's results are those of a call of its own, bit for bit."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:There is a performance drop")]


def test_a_call_for_each_sample(no_fallback):
    g = torch.Generator().manual_seed(0)
    n, rows, vocab, k, experts = 3, 5, 300, 4, 12
    x, t, r = (torch.randn(n, rows, w, generator=g) for w in (vocab, k, experts))
    e = r.topk(2).indices.to("supa")
    x, t, r = x.to("supa"), t.to("supa"), r.to("supa")
    i = torch.randint(0, vocab, (n, rows, k), generator=g).to("supa")
    lse = (torch.logsumexp(t.cpu(), -1) + 0.2).to("supa")
    x.requires_grad_()
    r.requires_grad_()
    kd = lambda x, i, t, lse: torch.supa.distillation_loss(x, i, t, teacher_lse=lse, temperature=1.5)  # noqa: E731
    loss = torch.vmap(kd)(x, i, t, lse)
    balance, counts = torch.vmap(lambda r, e: torch.supa.router_balance_loss(r, e))(r, e)
    gx, gr = torch.autograd.grad([loss.sum(), balance.sum()], [x, r])
    y = torch.vmap(lambda x, h: torch.supa.adjust_logits(x, tokens=h, repetition=1.25))(x.detach(), i)
    for s in range(n):
        xs, rs = x[s].detach().requires_grad_(), r[s].detach().requires_grad_()
        a = kd(xs, i[s], t[s], lse[s])
        b, c = torch.supa.router_balance_loss(rs, e[s])
        ga, gb = torch.autograd.grad([a, b], [xs, rs])
        one = torch.supa.adjust_logits(x[s].detach(), tokens=i[s], repetition=1.25)
        for u, v in ((loss[s], a), (balance[s], b), (counts[s], c), (gx[s], ga), (gr[s], gb), (y[s], one)):
            assert torch.equal(u.detach().cpu(), v.detach().cpu())
