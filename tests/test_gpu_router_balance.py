"""torch.supa.router_balance_loss against its definition in float64 (CPU), its
counts exactly, its gradient against torch's autograd of the definition.

Tolerances, derived (u = 2^-24): a share p is an exponential over a sum of at most 16
of a thread and a tree of 6 steps; its exponent has three roundings relative to itself,
|x - max| < 40 here: p is off by under K = 3 * 40 + 32 = 152 u of itself.  A column's sum adds at
most 64 values in sequence here, then trees and float64: under (K + 96) u of it, and so the loss, a sum of
positive terms.  The gradient p (a - sum p a) scale: under 2 K + 64 u of p (|a| + sum p |a|) scale.  The
definition's own gradient is formed in float64 with the loads a + 1, whose even part cancels there: each of its
at most 1024 products and sums is off by 2^-53 of p (load + sum p load) scale, which counts where a is 0 (k =
num_experts: every load is 1, the gradient is 0, and the definition's 1e-17)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24
K = 152 * U


def make(shape, k, x="f32", mask=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(shape, generator=g) + torch.randn(shape[-1], generator=g)).to(T[x])
    experts = torch.rand(shape, generator=g).argsort(-1)[..., :k].contiguous()
    m = torch.rand(shape[:-1], generator=g) < 0.7 if mask else None
    return logits, experts, m


def definition(x, experts, mask, scores, per_sequence):
    """float64: loss, counts, and the loads and number of tokens per sequence."""
    e, k = x.shape[-1], experts.shape[-1]
    n_seq = math.prod(x.shape[:-2]) if per_sequence else 1
    x3, c3 = x.reshape(n_seq, -1, e), experts.reshape(n_seq, -1, k)
    on = torch.ones(x3.shape[:2], dtype=torch.bool) if mask is None else mask.reshape(n_seq, -1)
    ok = on[..., None] & (c3 >= 0)
    counts = torch.zeros(n_seq, e, dtype=torch.int64)
    for s in range(n_seq):
        counts[s] = torch.bincount(c3[s][ok[s]], minlength=e)[:e]
    p = torch.softmax(x3, -1)
    if scores == "sigmoid":  # in logarithms: no underflow
        p = torch.softmax(torch.nn.functional.logsigmoid(x3), -1)
    p = torch.where(on[..., None], p, 0.0)
    n = on.sum(1).double()
    some = n > 0
    load = e * counts / (k * n.clamp(min=1))[:, None]
    each = (load * p.sum(1)).sum(1) / n.clamp(min=1)
    loss = each.sum() / some.sum().clamp(min=1)
    return loss, counts.reshape(x.shape[:-2] + (e,) if per_sequence else (e,)), p, load, n


def check(x, experts, mask=None, scores="softmax", per_sequence=False, upstream=1.0, view=lambda v: v):
    d = x.double().requires_grad_()
    want, counts, p, load, n = definition(d, experts, mask, scores, per_sequence)
    (want_g,) = torch.autograd.grad(want * upstream, d)
    want_g = torch.zeros_like(want_g) if mask is not None and not mask.any() else want_g
    dx = view(x.to("supa")).detach().requires_grad_()
    m = None if mask is None else mask.to("supa")
    loss, c = torch.supa.router_balance_loss(dx, experts.to("supa"), mask=m, scores=scores, per_sequence=per_sequence)
    assert torch.equal(c.cpu(), counts) and c.dtype == torch.int64
    want, got = want.detach(), float(loss.detach())
    assert abs(got - float(want)) <= (K + 96 * U) * float(want) + U * abs(got), (got, float(want))
    (g,) = torch.autograd.grad(loss, dx, torch.tensor(float(upstream), device="supa"))
    assert g.dtype == x.dtype and g.shape == x.shape
    with torch.no_grad():
        again, c2 = torch.supa.router_balance_loss(dx, experts.to("supa"), mask=m, scores=scores, per_sequence=per_sequence)
    assert float(again) == got and torch.equal(c2.cpu(), counts)
    a = (load - 1).abs()[:, None, :]
    p = p.detach()
    sequences = max(1, int((n > 0).sum()))
    size = p * (a + (p * a).sum(-1, keepdim=True)) * (abs(upstream) / sequences / n.clamp(min=1))[:, None, None]
    size64 = p * (load[:, None, :] + (p * load[:, None, :]).sum(-1, keepdim=True)) * (abs(upstream) / sequences / n.clamp(min=1))[:, None, None]
    off = ((2 * K + 64 * U) * size + 1024 * 2.0 ** -53 * size64).view(x.shape)
    fi = torch.finfo(g.dtype)
    tol = (want_g.abs() + off) * fi.eps / 2 + fi.tiny * fi.eps + off
    err = (g.double().cpu() - want_g).abs()
    assert (err <= tol).all(), float((err / tol).max())
    return loss, c, g


SIZES = [
    # shape, k
    ((1, 1), 1), ((1, 4), 2), ((5, 3), 3), ((64, 8), 2), ((37, 7), 1), ((100, 60), 4), ((33, 64), 6), ((130, 65), 8),
    ((2, 50, 128), 8), ((17, 129), 2), ((9, 161), 6), ((300, 256), 8), ((21, 257), 3), ((15, 512), 4), ((7, 513), 20),
    ((6, 1000), 100), ((5, 1024), 1024), ((5000, 16), 2), ((3000, 33), 4),
]


@pytest.mark.parametrize("shape, k", SIZES, ids=str)
@pytest.mark.parametrize("x", T)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_sizes(shape, k, x, scores, no_fallback):
    check(*make(shape, k, x, seed=shape[-1] + k), scores, upstream=3.5 if x != "f16" else 256.0)


@pytest.mark.parametrize("x", T)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("shape, k", [((4, 33, 8), 2), ((3, 7, 129), 4), ((2, 3, 20, 64), 6), ((50, 1, 16), 2), ((1, 700, 300), 3)], ids=str)
def test_sequences_and_masks(x, scores, shape, k, no_fallback):
    logits, experts, mask = make(shape, k, x, True, seed=k)
    up = 512.0 if x == "f16" else 1.0
    check(logits, experts, mask, scores, False, up)
    check(logits, experts, mask, scores, True, up)
    mask[0] = False  # a sequence without a token
    check(logits, experts, mask, scores, True, up)
    check(logits, experts, None, scores, True, up)


def test_masked_tokens_say_nothing(no_fallback):
    """Their logits may be anything, and their gradient is 0."""
    logits, experts, mask = make((40, 24), 3, mask=True)
    logits[~mask] = math.nan
    experts[~mask] = 5
    x = torch.where(mask[:, None], logits, 0.0)
    for scores in ("softmax", "sigmoid"):
        loss, c, g = check(x, experts, mask, scores)
        dx = logits.to("supa").requires_grad_()
        other, c2 = torch.supa.router_balance_loss(dx, experts.to("supa"), mask=mask.to("supa"), scores=scores)
        (g2,) = torch.autograd.grad(other, dx)
        assert float(other.detach()) == float(loss.detach()) and torch.equal(c2.cpu(), c.cpu()) and torch.equal(g2.cpu(), g.cpu())
        assert not g2.cpu()[~mask].any()


def test_nothing_counts(no_fallback):
    logits, experts, _ = make((3, 4, 6), 2)
    none = torch.zeros(3, 4, dtype=torch.bool)
    for per_sequence in (False, True):
        loss, c, g = check(logits, experts, none, per_sequence=per_sequence)
        assert float(loss.detach()) == 0 and not c.cpu().any() and not g.cpu().any()
    for shape in ((0, 6), (2, 0, 6), (0, 4, 6)):
        dx = torch.empty(shape, device="supa", requires_grad=True)
        loss, c = torch.supa.router_balance_loss(dx, torch.empty(shape[:-1] + (2,), dtype=torch.int64, device="supa"),
                                                 per_sequence=len(shape) == 3)
        (g,) = torch.autograd.grad(loss, dx)
        assert float(loss.detach()) == 0 and g.shape == shape and not c.cpu().any() and c.shape == ((shape[0], 6) if len(shape) == 3 else (6,))


def test_dropped_choices(no_fallback):
    logits, experts, mask = make((60, 10), 4, mask=True)
    experts[::3, 1] = -1
    experts[5] = -7
    for index in (torch.int64, torch.int32):
        check(logits, experts.to(index), mask)
        check(logits, experts.to(index), None, "sigmoid")
    experts[2] = 4  # the same expert for every choice of a token
    check(logits, experts)


def test_past_the_end(supa):
    logits, experts, _ = make((20, 5), 2)
    experts[3, 0], experts[9, 1] = 5, 2 ** 40
    want = experts[experts < 5].bincount(minlength=5)
    _, c = torch.supa.router_balance_loss(logits.to("supa"), experts.to("supa"))
    with pytest.raises(IndexError, match="router_balance_loss"):
        torch.supa.synchronize()
    assert torch.equal(c.cpu(), want)


def test_extreme_logits(no_fallback):
    """Logits of -inf (experts that are switched off), far apart and large, and a NaN's reach."""
    logits, experts, _ = make((30, 12), 2)
    logits[:, 3] = -math.inf
    for scores in ("softmax", "sigmoid"):
        loss, _ = torch.supa.router_balance_loss(logits.to("supa").requires_grad_(), experts.to("supa"), scores=scores)
        want = definition(logits.double(), experts, None, scores, False)[0]
        assert abs(float(loss.detach()) - float(want)) <= (K + 97 * U) * float(want)
    logits, experts, _ = make((30, 12), 2)
    for shift in (-200.0, 200.0):  # sigmoids that float32 does not hold, and ones
        check(logits + shift, experts, None, "sigmoid")
    logits[4, 4] = math.nan
    dx = logits.to("supa").requires_grad_()
    loss, _ = torch.supa.router_balance_loss(dx, experts.to("supa"))
    (g,) = torch.autograd.grad(loss, dx)
    assert loss.isnan() and g[4].isnan().all() and g[:4].cpu().isfinite().all() and g[5:].cpu().isfinite().all()


@pytest.mark.parametrize("x", T)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_lowest_values(x, scores, no_fallback):
    """Tokens that a mask of the type's lowest value leaves no expert are spread evenly."""
    logits, experts, _ = make((30, 20), 2, x)
    logits[::3] = torch.finfo(T[x]).min
    logits[1::3, 4:] = torch.finfo(T[x]).min
    logits[6, 1::2] = -math.inf
    loss, _ = torch.supa.router_balance_loss(logits.to("supa"), experts.to("supa"), scores=scores)
    want = definition(logits.double(), experts, None, scores, False)[0]
    assert abs(float(loss.detach()) - float(want)) <= (K + 97 * U) * float(want)
    logits[6] = torch.finfo(T[x]).min
    check(logits, experts, None, scores, upstream=256.0)


def test_even_loads(no_fallback):
    """Loads next to 1: the gradient is a small difference."""
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(4096, 8, generator=g) * 0.01
    experts = (torch.arange(4096)[:, None] + torch.arange(2)) % 8
    experts[0, 0] = 5
    check(logits, experts)


def test_strides(no_fallback):
    logits, experts, mask = make((6, 11, 40), 3, mask=True)
    view = lambda v: torch.stack([v, v], 2)[:, :, 1]  # noqa: E731
    check(logits, experts, mask, view=view)
    check(logits, experts, mask, per_sequence=True, view=lambda v: v.transpose(0, 2).contiguous().transpose(0, 2))
    a, _ = torch.supa.router_balance_loss(logits.to("supa"), experts.to("supa"), mask=mask.to("supa"))
    b, _ = torch.supa.router_balance_loss(logits.to("supa"), experts.transpose(0, 2).contiguous().to("supa").transpose(0, 2), mask=torch.stack([mask, mask], -1).to("supa")[..., 0])
    assert float(a) == float(b)


def test_differences(no_fallback):
    logits, experts, mask = make((10, 6), 2, mask=True, seed=5)
    mask[:3] = True
    for scores in ("softmax", "sigmoid"):
        f = lambda v: float(torch.supa.router_balance_loss(v.to("supa"), experts.to("supa"), mask=mask.to("supa"), scores=scores)[0])  # noqa: E731
        dx = logits.to("supa").requires_grad_()
        loss, _ = torch.supa.router_balance_loss(dx, experts.to("supa"), mask=mask.to("supa"), scores=scores)
        (g,) = torch.autograd.grad(loss, dx)
        h = 2.0 ** -5
        # third derivatives are under 2 max load / tokens < 2; the losses' own roundings on both sides
        tol = 2 * h * h / 6 + 2 * (K + 97 * U) * float(loss.detach()) / (2 * h)
        for r, c in ((0, 0), (1, 3), (2, 5)):
            v = [logits.clone(), logits.clone()]
            v[0][r, c] += h
            v[1][r, c] -= h
            assert abs((f(v[0]) - f(v[1])) / (2 * h) - float(g[r, c])) <= tol


def test_saved_tensors(no_fallback):
    logits, experts, mask = make((12, 9), 2, mask=True)
    dx = logits.to("supa").requires_grad_()
    loss, _ = torch.supa.router_balance_loss(dx, experts.to("supa"), mask=mask.to("supa"))
    (a,) = torch.autograd.grad(loss, dx, retain_graph=True)
    (b,) = torch.autograd.grad(loss, dx)
    assert torch.equal(a.cpu(), b.cpu())
    m = mask.to("supa")
    loss, _ = torch.supa.router_balance_loss(dx, experts.to("supa"), mask=m)
    m.fill_(True)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_many_sequences(no_fallback):
    """More sequences than one launch's grid takes."""
    logits, experts, mask = make((66000, 2, 4), 1, mask=True, seed=1)
    check(logits, experts, mask, per_sequence=True, upstream=1e4)
