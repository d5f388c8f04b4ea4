"""torch.supa.distillation_loss with a teacher_lse of every float type: a float64 one is
taken as it is.  What the teacher leaves to the tokens that are not listed, r = 1 - sum p, is a
difference of near values: a log-sum-exp of 2000 rounded to float32 is off by up to 2^-14 = 6e-5, which
moves a rest of 1e-4 by half of itself.

Tolerances are those of test_gpu_distillation.py, which know of no such rounding."""
import pytest
import torch

from test_gpu_distillation import T, check, make

pytestmark = pytest.mark.gpu


def near(rows, vocab, k, x, left, shift, seed, temperature=1.0):
    """Teachers whose listed tokens leave `left` of the mass, of logits about `shift`."""
    logits, i, t, _ = make(rows, vocab, k, x, "f32", False, seed)
    t = (t + shift).float()
    z = t.double() / temperature
    share = left * (0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(seed), dtype=torch.float64))
    return logits, i, t, torch.logsumexp(z, 1) - torch.log1p(-share)


@pytest.mark.parametrize("x", T)
@pytest.mark.parametrize("left", [1e-2, 1e-4, 1e-7])
@pytest.mark.parametrize("shift", [20.0, 2000.0])
def test_float64(x, left, shift, no_fallback):
    logits, i, t, lse = near(9, 700, 12, x, left, shift, 3)
    for reduction in ("none", "mean", "sum"):
        check(logits, i, t, lse, reduction=reduction)


@pytest.mark.parametrize("rows, vocab, k", [(1, 5, 2), (4, 40000, 30), (600, 300, 7), (4100, 65, 5), (530, 9000, 300)], ids=str)
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_float64_in_every_form_of_the_forward(rows, vocab, k, temperature, no_fallback):
    """Rows in parts, in workgroups, in wavefronts; many pairs."""
    check(*near(rows, vocab, k, "bf16", 1e-3, 500.0, rows, temperature), temperature)


def test_float64_rows_at_any_distance(no_fallback):
    logits, i, t, lse = near(12, 200, 5, "f32", 1e-4, 900.0, 7)
    dx = logits.view(3, 4, 200).to("supa")
    ids, tt = i.view(3, 4, 5).to("supa"), t.view(3, 4, 5).to("supa")
    want = torch.supa.distillation_loss(dx, ids, tt, teacher_lse=lse.view(3, 4).to("supa"), reduction="none").cpu()
    check(logits.view(3, 4, 200), i.view(3, 4, 5), t.view(3, 4, 5), lse.view(3, 4))
    wide = torch.zeros(4, 7, dtype=torch.float64, device="supa")
    wide[:3, 1:5] = lse.view(3, 4).to("supa")
    for view in (wide[:3, 1:5], lse.view(3, 4).t().contiguous().to("supa").t()):
        assert not view.is_contiguous()
        assert torch.equal(torch.supa.distillation_loss(dx, ids, tt, teacher_lse=view, reduction="none").cpu(), want)
    same = lse[:1].to("supa").expand(12)
    got = torch.supa.distillation_loss(logits.to("supa"), i.to("supa"), t.to("supa"), teacher_lse=same, reduction="none").cpu()
    one = torch.supa.distillation_loss(logits.to("supa"), i.to("supa"), t.to("supa"), reduction="none",
                                       teacher_lse=lse[:1].repeat(12).to("supa")).cpu()
    assert torch.equal(got, one)


@pytest.mark.parametrize("lse", [torch.float32, torch.bfloat16, torch.float16])
def test_narrower_types(lse, no_fallback):
    """Their values are float64's too: the same bits."""
    logits, i, t, exact = near(9, 700, 12, "f32", 0.3, 5.0, 4)
    rounded = (exact + 0.1).to(lse)
    check(logits, i, t, rounded)
    args = (logits.to("supa"), i.to("supa"), t.to("supa"))
    a = torch.supa.distillation_loss(*args, teacher_lse=rounded.to("supa"), reduction="none")
    b = torch.supa.distillation_loss(*args, teacher_lse=rounded.double().to("supa"), reduction="none")
    assert torch.equal(a.cpu(), b.cpu())


def test_no_rows(no_fallback):
    x = torch.empty(0, 5, device="supa", requires_grad=True)
    loss = torch.supa.distillation_loss(x, torch.empty(0, 2, dtype=torch.int64, device="supa"), torch.empty(0, 2, device="supa"),
                                        teacher_lse=torch.empty(0, dtype=torch.float64, device="supa"), reduction="sum")
    assert float(loss.detach()) == 0
    (g,) = torch.autograd.grad(loss, x)
    assert g.shape == (0, 5)
