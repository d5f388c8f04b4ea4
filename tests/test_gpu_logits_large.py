"""The operators on logits past 2^31 elements: offsets of 64 bits.  Some rows
against the same rows alone, which other tests hold to their definitions."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, VOCAB = 33000, 70001  # 2.31e9 elements
AT = [0, 1, 15000, 30676, 30678, 32999]  # around the 2^31st element, which row 30677 holds


@pytest.fixture(scope="module")
def logits(supa):
    x = torch.empty(ROWS, VOCAB, dtype=torch.bfloat16, device="supa")
    g = torch.Generator().manual_seed(0)
    x.normal_()
    for r in AT:
        x[r] = torch.randn(VOCAB, generator=g).bfloat16().to("supa")
    yield x
    del x
    torch.supa.empty_cache()


def rows(t):
    return torch.stack([t[r].cpu() for r in AT])


@pytest.mark.parametrize("rest", [False, True])
def test_distillation(logits, rest, no_fallback):
    g = torch.Generator().manual_seed(1)
    i = torch.randint(0, VOCAB, (ROWS, 5), generator=g)
    t = torch.randn(ROWS, 5, generator=g)
    lse = torch.logsumexp(t, 1) + 0.2
    x = logits.detach().requires_grad_()
    loss = torch.supa.distillation_loss(x, i.to("supa"), t.to("supa"), teacher_lse=lse.to("supa") if rest else None, reduction="none")
    (gx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    few = rows(logits).to("supa").requires_grad_()
    want = torch.supa.distillation_loss(few, i[AT].to("supa"), t[AT].to("supa"), reduction="none",
                                        teacher_lse=lse[AT].to("supa") if rest else None)
    (gw,) = torch.autograd.grad(want, few, torch.ones_like(want))
    # the few rows are split over workgroups: sums in another order, (vocab / 64 + 128) of 2^-24 on either side
    s = 2 * (VOCAB / 64 + 128) * 2.0 ** -24
    assert ((loss.detach().cpu()[AT] - want.detach().cpu()).abs() <= s + 2.0 ** -23 * want.detach().cpu().abs()).all()
    a, b = rows(gx).float(), gw.cpu().float()
    assert ((a - b).abs() <= b.abs() * 2.0 ** -7 + 4 * s).all() and float(gx[32999].float().sum().cpu().abs()) < 1e-2


def test_adjust(logits, no_fallback):
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, VOCAB, (ROWS, 20), generator=g)
    kw = dict(repetition=1.5, presence=0.25)
    out = torch.supa.adjust_logits(logits, tokens=tokens.to("supa"), **kw)
    want = torch.supa.adjust_logits(rows(logits).to("supa"), tokens=tokens[AT].to("supa"), **kw)
    assert torch.equal(rows(out), want.cpu())


def test_wide_rows_apart(supa, no_fallback):
    """Few rows far apart in a large buffer, in place; what lies between stays."""
    buf = torch.zeros(3 * (1 << 30), dtype=torch.bfloat16, device="supa")
    x = buf.view(3, 1 << 30)[:, 5: 5 + 9001]
    g = torch.Generator().manual_seed(3)
    v = torch.randn(3, 9001, generator=g).bfloat16()
    x.copy_(v.to("supa"))
    i, t = torch.randint(0, 9001, (3, 4), generator=g).to("supa"), torch.randn(3, 4, generator=g).to("supa")
    d = x.detach().requires_grad_()
    loss = torch.supa.distillation_loss(d, i, t)
    (gx,) = torch.autograd.grad(loss, d)
    e = v.to("supa").requires_grad_()
    want = torch.supa.distillation_loss(e, i, t)
    (gw,) = torch.autograd.grad(want, e)
    # the views' vectors begin elsewhere: another order of the sums
    s = 2 * (9001 / 64 + 128) * 2.0 ** -24
    assert abs(float(loss) - float(want)) <= 2 * s
    assert ((gx.cpu().float() - gw.cpu().float()).abs() <= gw.cpu().float().abs() * 2.0 ** -7 + 4 * s).all()
    torch.supa.adjust_logits_(x, tokens=i, repetition=2.0)
    assert torch.equal(x.cpu(), torch.supa.adjust_logits(v.to("supa"), tokens=i, repetition=2.0).cpu())
    for r in range(3):
        row = buf.view(3, 1 << 30)[r]
        assert not row[:5].cpu().any() and not row[9006: 9100].cpu().any()


def test_balance(supa, no_fallback):
    tokens, experts = 2200000, 1000
    x = torch.empty(tokens, experts, dtype=torch.bfloat16, device="supa").normal_()
    g = torch.Generator().manual_seed(4)
    e = torch.randint(0, experts, (tokens, 2), generator=g)
    d = x.detach().requires_grad_()
    loss, counts = torch.supa.router_balance_loss(d, e.to("supa"))
    assert torch.equal(counts.cpu(), torch.bincount(e.flatten(), minlength=experts))
    (gx,) = torch.autograd.grad(loss, d, torch.full((), 1e6, device="supa"))
    load = torch.bincount(e.flatten(), minlength=experts).double() * experts / (2 * tokens) - 1
    for t in (0, 2147482, 2147484, tokens - 1):
        p = torch.softmax(x[t].double().cpu(), 0)
        want = p * (load - (p * load).sum()) * 1e6 / tokens
        # one rounding to bf16, and 368 of 2^-24 of the magnitudes as in test_gpu_router_balance.py
        tol = want.abs() * 2.0 ** -8 + 368 * 2.0 ** -24 * p * (load.abs() + (p * load.abs()).sum()) * 1e6 / tokens + 1e-38
        assert ((gx[t].double().cpu() - want).abs() <= tol).all()
    assert abs(float(loss) - 1) < 0.01
