"""torch.supa.distillation_loss against its definition in float64 (CPU), its
gradient against torch's autograd of that definition and against central
differences.

Tolerances, derived (u = 2^-24).  A row's sum of exponentials: an exponent
(x - m) c has three roundings, relative to itself, and |t| e^t weighed over a
row stays under ln(vocab) < 16: 3 * 16 u of the sum; the exponential itself one
u; a thread adds at most vocab / 64 + 32 values in sequence, then a tree.  So
the sum, and absolutely the log-sum-exp and the loss, is off by under
S = (vocab / 64 + 128) u.  What depends on the pairs is float64, rounded once at the
end.  A probability's exponent next to 0 is formed to 24 bits, in all under
(|log2 q| + 4) u with |log2 q| < 140: q is off by under (S + 150 u) q, and with
the rest class its mass by S of itself, which the coefficient w q_R - r takes
over: the gradient is off by under (3 S + 300 u) (w q + r q / q_R + p), times
the scale, before its one rounding to the logits' type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def S(vocab):
    return (vocab / 64 + 128) * U


def make(rows, vocab, k, x="f32", teacher="f32", rest=False, seed=0, temperature=1.0, spread=3.0):
    """logits, indices, teacher's logits and lse; k distinct tokens a row."""
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=g) * spread)
    indices = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)]) if rows else torch.zeros(0, k, dtype=torch.int64)
    t = torch.randn(rows, k, generator=g) * 3
    logits.scatter_add_(1, indices, t)
    t = t.to(T[teacher])
    lse = None
    if rest:
        z = t.double() / temperature
        lse = (torch.logsumexp(z, 1) + torch.rand(rows, generator=g) * 0.5 + 0.01).float()
    return logits.to(T[x]), indices, t, lse


def definition(x, indices, t, lse, temperature, reduction):
    """float64; (loss, the rows' losses, which rows count)."""
    vocab, k = x.shape[-1], indices.shape[-1]
    x2, i2, t2 = x.reshape(-1, vocab), indices.reshape(-1, k), t.double().reshape(-1, k)
    there = (i2 >= 0) & (i2 < vocab) & (t2 != -math.inf)
    counted = there.any(1)
    at = torch.where(there, i2, 0)
    log_q = torch.log_softmax(x2 / temperature, 1)
    z = torch.where(there, t2 / temperature, -math.inf)
    if lse is None:
        log_p = torch.log_softmax(torch.where(counted[:, None], z, 0.0), 1)
    else:
        log_p = z - lse.double().reshape(-1, 1)
    p = torch.where(there, log_p.exp(), 0.0)
    some = p > 0
    rows = torch.where(some, p * (torch.where(some, log_p, 0.0) - torch.where(some, log_q.gather(1, at), 0.0)), 0.0).sum(1)
    if lse is not None:
        listed = torch.zeros(x2.shape[0], vocab + 1, dtype=torch.bool)
        listed.scatter_(1, torch.where(there, i2, vocab), True)
        listed = listed[:, :vocab]
        r = torch.where(listed.all(1), 0.0, (1 - p.sum(1)).clamp(min=0))
        # rows without a rest go in as zeros: the gradient of a log-sum-exp of nothing is NaN
        rest = torch.logsumexp(torch.where((r > 0)[:, None], torch.where(listed, -math.inf, log_q), 0.0), 1)
        rows = rows + torch.where(r > 0, torch.xlogy(r, r) - r * rest, 0.0)
    rows = torch.where(counted, rows, 0.0)
    if reduction == "none":
        return rows.view(x.shape[:-1]), rows, counted
    total = rows.sum()
    return (total / counted.sum() if reduction == "mean" else total), rows, counted


def magnitude(x, indices, t, lse, temperature):
    """w q + r q / q_R (at tokens that are not listed) + p, of each logit."""
    vocab, k = x.shape[-1], indices.shape[-1]
    x2, i2, t2 = x.double().reshape(-1, vocab), indices.reshape(-1, k), t.double().reshape(-1, k)
    there = (i2 >= 0) & (i2 < vocab) & (t2 != -math.inf)
    q = torch.softmax(x2 / temperature, 1)
    z = torch.where(there, t2 / temperature, -math.inf)
    norm = torch.logsumexp(z, 1, keepdim=True) if lse is None else lse.double().reshape(-1, 1)
    p = torch.where(there, (z - norm).exp(), 0.0)
    out = q * p.sum(1, keepdim=True).clamp(min=1.0)
    wide = torch.zeros(x2.shape[0], vocab + 1, dtype=torch.float64)
    at = torch.where(there, i2, vocab)
    out = out + wide.scatter_add(1, at, p)[:, :vocab]
    if lse is not None:
        listed = wide.scatter(1, at, 1.0)[:, :vocab] > 0
        r = (1 - p.sum(1, keepdim=True)).clamp(min=0)
        rest = torch.where(listed, 0.0, q)
        out = out + r * rest / rest.sum(1, keepdim=True).clamp(min=1e-300)
    return out.view(x.shape)


def check(x, indices, t, lse=None, temperature=1.0, reduction="mean", upstream=None, view=lambda v: v):
    """Forward and backward; `view` makes the caller's view of the logits on the device."""
    vocab = x.shape[-1]
    d = x.double().requires_grad_()
    want, rows, counted = definition(d, indices, t, lse, temperature, reduction)
    up = torch.ones_like(want) if upstream is None else upstream.double()
    (want_g,) = torch.autograd.grad(want, d, up)
    dx = view(x.to("supa")).detach().requires_grad_()
    assert dx.shape == x.shape
    loss = torch.supa.distillation_loss(dx, indices.to("supa"), t.to("supa"), teacher_lse=None if lse is None else lse.to("supa"),
                                        temperature=temperature, reduction=reduction)
    (g,) = torch.autograd.grad(loss, dx, up.float().to("supa"))
    with torch.no_grad():  # the same without a graph, bit for bit
        again = torch.supa.distillation_loss(dx, indices.to("supa"), t.to("supa"), temperature=temperature, reduction=reduction,
                                             teacher_lse=None if lse is None else lse.to("supa"))
    assert torch.equal(again.cpu().nan_to_num(7e9), loss.detach().cpu().nan_to_num(7e9))
    got = loss.detach().double().cpu()
    each = S(vocab) * counted.double() + 2 * U * rows.detach().abs()
    n = counted.sum().double()
    tol = {"none": each.view(x.shape[:-1]), "sum": each.sum() + U * want.detach().abs(),
           "mean": each.sum() / n + 2 * U * want.detach().abs()}[reduction]
    if not (reduction == "mean" and n == 0):
        near = (got - want.detach()).abs() <= tol
        assert got.shape == want.shape and (near | (got == want.detach())).all(), (got, want, tol)  # inf is inf
    else:
        assert got.isnan()
    assert g.dtype == x.dtype and g.shape == x.shape
    scale = up.abs().view(x.shape[:-1] + (1,)) if reduction == "none" else up.abs()
    if reduction == "mean":
        scale = scale / n
    scale = torch.where(counted.view(x.shape[:-1] + (1,)), scale / temperature, 0.0)
    fi = torch.finfo(g.dtype)
    off = scale * (3 * S(vocab) + 300 * U) * magnitude(x, indices, t, lse, temperature)
    off = torch.where(counted.view(x.shape[:-1] + (1,)), off, 0.0)
    want_g = torch.where(counted.view(x.shape[:-1] + (1,)), want_g, 0.0)
    tol = (want_g.abs() + off) * fi.eps / 2 + fi.tiny * fi.eps + off
    err = (g.double().cpu() - want_g).abs()
    bad = ~(err <= tol) & rows.detach().isfinite().view(x.shape[:-1] + (1,))  # an infinite loss has no gradient
    assert not bad.any(), (int(bad.sum()), float((err / tol).max()), bad.nonzero()[:4])
    return loss, g


SIZES = [
    # rows, vocab, k
    (1, 1, 1), (1, 2, 1), (3, 7, 3), (5, 64, 8), (4, 100, 64), (9, 257, 5), (130, 512, 16), (7, 1000, 100), (3, 2048, 256),
    (5, 2047, 257), (3, 4096, 1024), (2, 4099, 1000), (17, 8191, 20), (6, 32000, 64), (3, 50257, 20), (2, 131077, 33),
    (1, 300000, 7),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
def test_sizes(size, rest, no_fallback):
    rows, vocab, k = size
    x = ["f32", "bf16", "f16"][(rows + vocab) % 3]
    check(*make(rows, vocab, k, x, ["f32", "bf16", "f16"][k % 3], rest, seed=vocab))


@pytest.mark.parametrize("x", T)
@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("temperature", [1.0, 2.5, 0.3])
def test_types(x, rest, reduction, temperature, no_fallback):
    a = make(13, 1003, 17, x, "f32", rest, 3, temperature)
    up = torch.rand(13, generator=torch.Generator().manual_seed(1)) + 0.5 if reduction == "none" else torch.tensor(3.25)
    if x == "f16":
        up = up * 64
    check(*a, temperature, reduction, up)


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_short_rows(index, no_fallback):
    """Rows that store fewer pairs, one or none; logits of -inf and indices past the end are not there."""
    for rest in (False, True):
        x, i, t, lse = make(8, 700, 9, "bf16", "bf16", rest, 5)
        i[0] = -1
        i[1, 4:] = -100
        i[2, :8] = -1
        t[3, 2] = -math.inf
        t[4] = -math.inf
        i[5, ::2] = -(2 ** 31)
        for reduction in ("mean", "sum", "none"):
            loss, g = check(x, i.to(index), t, lse, reduction=reduction)
            assert not g[0].cpu().any() and not g[4].cpu().any()


def test_no_row_counts(no_fallback):
    x, i, t, _ = make(4, 300, 3)
    i.fill_(-1)
    for reduction in ("mean", "sum", "none"):
        loss, g = check(x, i, t, reduction=reduction)
        assert not g.cpu().any() and (loss.isnan().all() if reduction == "mean" else not loss.cpu().any())
    for reduction in ("mean", "sum", "none"):  # and no row at all
        dx = torch.empty(0, 5, device="supa", requires_grad=True)
        loss = torch.supa.distillation_loss(dx, torch.empty(0, 2, dtype=torch.int64, device="supa"),
                                            torch.empty(0, 2, device="supa"), reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and (reduction != "mean" or loss.isnan())
        (g,) = torch.autograd.grad(loss, dx, torch.ones_like(loss))
        assert g.shape == (0, 5)


@pytest.mark.parametrize("k", [4, 200, 700])
@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
def test_a_token_listed_twice(k, rest, no_fallback):
    x, i, t, lse = make(6, 1500, k, "f32", "f32", rest, 9)
    i[0, -1] = i[0, 0]
    i[1] = i[1, 0]
    i[2, 1::2] = i[2, 0]
    i[3, -2:] = i[3, 0]
    i[4, 1] = i[4, 0]
    t[4, 0] = -math.inf  # the first of the two is not there
    check(x, i, t, lse)


@pytest.mark.parametrize("k", [64, 256, 1000])
@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
def test_tokens_listed_many_times(k, rest, no_fallback):
    """All, in pairs, far apart and at random: the same bits each time."""
    for vocab in (40, 1500, 70001):
        x, i, t, lse = make(6, max(vocab, k), k, "f32", "f32", rest, vocab)
        i[0] = i[0, 3]
        i[1] = (torch.arange(k) // 2) % vocab
        i[2] = torch.arange(k) % (k // 2 + 1) % vocab
        i[3] = torch.randint(0, min(vocab, 90), (k,), generator=torch.Generator().manual_seed(k))
        i[4] = (torch.arange(k) * 65536) % max(vocab, k)
        i[4, ::3] = -1
        loss, g = check(x, i, t, lse, reduction="none")
        again, g2 = check(x, i, t, lse, reduction="none")
        assert torch.equal(loss.detach().cpu(), again.detach().cpu()) and torch.equal(g.cpu(), g2.cpu())


def test_every_token_listed(no_fallback):
    """No rest: what the teacher's lse leaves over has nowhere to go."""
    for vocab in (1, 5, 300):
        x, i, t, lse = make(4, vocab, vocab, "f32", "f32", True, 2)
        check(x, i, t, lse)
        check(x, i, t, lse - 2.0)  # and a teacher of more than 1


def test_teacher_of_more_than_one(no_fallback):
    x, i, t, lse = make(5, 900, 12, "f32", "f32", True, 4)
    check(x, i, t, torch.logsumexp(t, 1) - 0.25)
    check(x, i, t, torch.logsumexp(t, 1) + 1e-6)


def test_extremes(no_fallback):
    """Confident students, logits of -inf, masked tails and far temperatures."""
    x, i, t, lse = make(6, 2500, 6, "f32", "f32", True, 8)
    x[0] = -60.0
    x[0, i[0]] = 20.0  # the rest holds e^-80 of the mass
    x[1, 3:] = -math.inf
    i[1, 0], i[1, 1], i[1, 2], t[1, 3:] = 0, 1, 2, -math.inf
    keep = torch.ones(2500, dtype=torch.bool)
    keep[i[2]] = False
    x[2, keep.nonzero()[5:, 0]] = -math.inf
    x[3] = torch.finfo(torch.float32).min
    x[3, 7] = 0.0
    x[4] = 0.0
    lse[1] = torch.logsumexp(t[1, :3], 0) - 0.1  # no mass for a rest that has none
    x[3, i[3]] = torch.linspace(-5, 5, 6)
    for v in (None, lse):
        check(x, i, t, v, reduction="none")
        check(x, i, t, v if v is None else torch.logsumexp(t / 50, 1) + 0.1, 50.0, "none")


@pytest.mark.parametrize("temperature", [math.log2(math.e), 2 * math.log2(math.e), 0.7, 1.1, 3.0, 1e-3, 1e4])
def test_excluded_tokens_at_any_temperature(temperature, no_fallback):
    """Logits of -inf, where log2(e) / temperature is a float32, or rounds either way."""
    x, i, t, lse = make(4, 130, 5, "f32", "f32", True, 21, temperature)
    keep = torch.zeros(4, 130, dtype=torch.bool).scatter(1, i, True)
    keep[:, ::3] = True
    x[~keep] = -math.inf
    for v in (None, lse):
        check(x * min(1.0, temperature), i, t * min(1.0, temperature), v if v is None else torch.logsumexp(t * min(1.0, temperature) / temperature, 1) + 0.1,
              temperature, "none")


@pytest.mark.parametrize("x", T)
@pytest.mark.parametrize("temperature", [1.0, 0.25, 1e-3])
def test_lowest_values(x, temperature, no_fallback):
    """Rows that a mask of the type's lowest value leaves nothing of are even, in part or whole; the largest value too."""
    logits, i, t, lse = make(7, 530, 6, x, "f32", True, 31, temperature)
    fi = torch.finfo(T[x])
    logits[0] = fi.min
    logits[1] = fi.min
    logits[1, i[1]] = 0.0
    logits[2] = fi.min
    logits[2, ::2] = -math.inf
    logits[2, i[2]] = fi.min
    logits[3] = fi.max
    logits[4] = torch.where(torch.arange(530) % 3 == 0, fi.max, fi.min).to(T[x])
    logits[4, i[4]] = fi.max
    logits[5] = fi.min
    logits[5, i[5, :3]] = fi.max
    t[5, 3:] = -math.inf
    # a teacher without a rest where the student's would cost (largest - lowest) / temperature: no float32
    lse[1], lse[5] = torch.logsumexp(t[1].double() / temperature, 0) - 0.1, torch.logsumexp(t[5].double() / temperature, 0) - 0.1
    for v in (None, lse):
        for reduction in ("none", "sum"):
            rows = slice(0, 5) if reduction == "sum" else slice(0, 7)
            check(logits[rows], i[rows], t[rows], v if v is None else v[rows], temperature, reduction)


def test_infinite_losses_and_nans(no_fallback):
    x, i, t, lse = make(5, 400, 4, "f32", "f32", True, 6)
    x[0, i[0, 0]] = -math.inf  # a listed token that the student excludes
    x[1, 17] = math.nan
    t[2, 1] = math.nan
    x[3, 5] = math.inf
    for v in (None, lse):
        dx = x.to("supa").requires_grad_()
        loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"), teacher_lse=None if v is None else v.to("supa"),
                                            reduction="none")
        (g,) = torch.autograd.grad(loss, dx, torch.ones_like(loss))
        got = loss.detach().cpu()
        assert got[0] == math.inf and got[1].isnan() and got[2].isnan() and got[3].isnan() and got[4].isfinite()
        assert g[1].isnan().any() and g[2].isnan().any() and g[4].cpu().isfinite().all()
    only = torch.full((1, 400), -math.inf)
    only[0, i[4]] = 1.0
    with torch.no_grad():  # a rest whose tokens the student excludes, and a teacher who does not
        assert torch.supa.distillation_loss(only.to("supa"), i[4:].to("supa"), t[4:].to("supa"), teacher_lse=lse[4:].to("supa")).item() == math.inf


def strided(kind):
    def view(v):
        b, s, n = v.shape
        if kind == "shifted":  # [:, :-1] of a longer batch
            w = torch.full((b, s + 1, n), math.nan, dtype=v.dtype, device="supa")
            w[:, :-1] = v
            return w[:, :-1]
        if kind == "columns":  # the first columns of wider rows
            w = torch.full((b, s, n + 37), math.nan, dtype=v.dtype, device="supa")
            w[..., :n] = v
            return w[..., :n]
        if kind == "both":
            w = torch.full((b + 1, s + 2, n + 5), math.nan, dtype=v.dtype, device="supa")
            w[1:, 1:-1, 3:-2] = v
            return w[1:, 1:-1, 3:-2]
        if kind == "sequence_first":
            w = torch.empty((s, b, n), dtype=v.dtype, device="supa")
            w.transpose(0, 1).copy_(v)
            return w.transpose(0, 1)
        w = torch.empty((b, n, s), dtype=v.dtype, device="supa")  # tokens before positions
        w.transpose(1, 2).copy_(v)
        return w.transpose(1, 2)
    return view


@pytest.mark.parametrize("kind", ["shifted", "columns", "both", "sequence_first", "transposed"])
@pytest.mark.parametrize("x, vocab", [("bf16", 1003), ("f32", 512), ("f16", 2600)])
def test_strides(kind, x, vocab, no_fallback):
    logits, i, t, lse = make(15, vocab, 6, x, "f32", True, 12)
    check(logits.view(3, 5, vocab), i.view(3, 5, 6), t.view(3, 5, 6), lse.view(3, 5), reduction="mean", view=strided(kind))


def test_strided_indices_and_upstream(no_fallback):
    x, i, t, lse = make(6, 300, 8, rest=True, seed=2)
    dx = x.to("supa").requires_grad_()
    wide_i, wide_t = i.repeat_interleave(2, 1).to("supa"), t.repeat_interleave(2, 1).to("supa")
    base = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"), teacher_lse=lse.to("supa"), reduction="none")
    other = torch.supa.distillation_loss(dx, wide_i[:, ::2], wide_t[:, ::2], reduction="none",
                                         teacher_lse=torch.stack([lse, lse], 1).to("supa")[:, 1])
    assert torch.equal(base.detach().cpu(), other.detach().cpu())
    (a,) = torch.autograd.grad(base.sum(), dx)  # an expanded gradient
    (b,) = torch.autograd.grad(other, dx, torch.ones(6, device="supa"))
    assert torch.equal(a.cpu(), b.cpu())


def test_differences(no_fallback):
    """Central differences of the float64 definition are its gradient's check elsewhere; here of the operator itself."""
    x, i, t, lse = make(3, 40, 4, rest=True, seed=7)
    up = torch.tensor([1.0, -0.5, 2.0])
    dx = x.to("supa").requires_grad_()
    f = lambda v: (torch.supa.distillation_loss(v, i.to("supa"), t.to("supa"), teacher_lse=lse.to("supa"),  # noqa: E731
                                                temperature=1.5, reduction="none").cpu().double() * up).sum()
    loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"), teacher_lse=lse.to("supa"), temperature=1.5, reduction="none")
    (g,) = torch.autograd.grad(loss, dx, up.to("supa"))
    h = 2.0 ** -6
    # a difference's error: three third derivatives, each under 2 in size, times h^2 / 6, and the losses' own S on both sides
    tol = 2 * h * h + 3.5 * 2 * (S(40) + 16 * U) / (2 * h)
    for r in range(3):
        for c in (0, int(i[r, 0]), int(i[r, 3]), 39):
            v = [x.clone(), x.clone()]
            v[0][r, c] += h
            v[1][r, c] -= h
            with torch.no_grad():
                d = float(f(v[0].to("supa")) - f(v[1].to("supa"))) / (2 * h)
            assert abs(d - float(g[r, c])) <= tol, (r, c, d, float(g[r, c]))


def test_past_the_end(supa):
    x, i, t, _ = make(4, 50, 3)
    i[2, 1] = 50
    dx = x.to("supa").requires_grad_()
    loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"), reduction="none")
    with pytest.raises(IndexError, match="distillation_loss"):
        torch.supa.synchronize()
    i[2, 1] = -1
    want, _, _ = definition(x.double(), i, t, None, 1.0, "none")
    assert torch.allclose(loss.detach().double().cpu(), want, atol=S(50) + 1e-5, rtol=0)


def test_past_the_end_but_not_there(no_fallback):
    """Padding by a teacher's logit of -inf may list any token."""
    x, i, t, _ = make(4, 50, 6)
    i[1, 2:], t[1, 2:] = 50, -math.inf
    i[2], t[2] = 2 ** 31 - 1, -math.inf
    check(x, i, t)
    check(x, i.int(), t)
    torch.supa.synchronize()


def test_many_rows(no_fallback):
    """More rows than one launch of the sum adds, and more than one slab of the gradient's grid."""
    rows, vocab = 70000, 16
    g = torch.Generator().manual_seed(0)
    x = torch.randn(rows, vocab, generator=g)
    i = torch.randint(0, vocab // 2, (rows, 1), generator=g).repeat(1, 2)
    i[:, 1] += vocab // 2
    i[::3] = -1
    check(x, i, torch.randn(rows, 2, generator=g), reduction="mean")


@pytest.mark.parametrize("x, vocab", [("bf16", 5003), ("f16", 20001), ("f32", 15999), ("bf16", 33001)])
@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
def test_many_long_rows(x, vocab, rest, no_fallback):
    """Enough rows for a wavefront each: copies of a few, which are checked, have their losses and gradients
    but for the order of the sums."""
    few, k = 41, 30
    logits, i, t, lse = make(few, vocab, k, x, "f32", rest, 5, 0.8)
    i[3] = -1
    i[4, 20:] = i[4, 0]
    loss, g = check(logits, i, t, lse, 0.8, "none", torch.full((few,), 64.0))
    copies = lambda v: v.repeat((101,) + (1,) * (v.dim() - 1)).to("supa")  # noqa: E731
    dx = copies(logits).requires_grad_()
    many = torch.supa.distillation_loss(dx, copies(i), copies(t), temperature=0.8, reduction="none",
                                        teacher_lse=None if lse is None else copies(lse))
    (gm,) = torch.autograd.grad(many, dx, torch.full((101 * few,), 64.0, device="supa"))
    many, gm = many.detach().cpu().view(101, few), gm.cpu().view(101, few, vocab)
    # Copies are not the same bits: vectors lie at multiples of 16 bytes, so a row's address decides which element falls to
    # which thread, and a float32 sum depends on that order.  Each order's sum is within S of the exact one, relative, so two
    # are within 2 S, and the losses, logarithms of them, absolutely; a gradient off by at most `off` each way and rounded once
    # (half an eps of a value that is |g| + off at most) is within 2 off + eps (|g| + off) of the other.
    assert ((many - loss.detach().cpu()).abs() <= 2 * S(vocab) + 4 * U * many.abs()).all()
    off = (3 * S(vocab) + 300 * U) * magnitude(logits, i, t, lse, 0.8) * 64 / 0.8
    fi, g = torch.finfo(T[x]), g.double().cpu()
    far = 2 * off + fi.eps * (g.abs() + off) + fi.tiny * fi.eps
    for each in gm:
        assert ((each.double() - g).abs() <= far).all()


def test_saved_tensors(no_fallback):
    """Twice through the graph; a write to the logits in between is noticed; a hook's copies do."""
    x, i, t, _ = make(5, 600, 4)
    dx = x.to("supa").requires_grad_()
    loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"))
    (a,) = torch.autograd.grad(loss, dx, retain_graph=True)
    (b,) = torch.autograd.grad(loss, dx)
    assert torch.equal(a.cpu(), b.cpu())
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, dx)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), lambda v: v.to("supa")):
        loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"))
    (c,) = torch.autograd.grad(loss, dx)
    assert torch.equal(a.cpu(), c.cpu())
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: v.cpu()):
        loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"))
    with pytest.raises(RuntimeError, match="saved tensor came back"):
        torch.autograd.grad(loss, dx)
    y = dx * 1
    loss = torch.supa.distillation_loss(y, i.to("supa"), t.to("supa"))
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
