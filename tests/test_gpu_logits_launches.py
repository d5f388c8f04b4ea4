"""The operators on logits where a call is cut into several: columns past one bitmap of listed tokens, rows past one
launch, and rows whose ranges lie eight workgroups apart.

Tolerances are those derived in test_gpu_distillation.py, against the definition in float64."""
import math

import pytest
import torch

from test_gpu_distillation import S, T, U, definition, magnitude, make

pytestmark = pytest.mark.gpu

SEGMENT = 1 << 17  # columns of one bitmap


def against(x, i, t, lse, up, loss, g, temperature=1.0):
    """The rows' losses and gradients (reduction none, upstream `up`) of the operator against the definition."""
    vocab = x.shape[-1]
    d = x.double().requires_grad_()
    want, rows, counted = definition(d, i, t, lse, temperature, "none")
    (want_g,) = torch.autograd.grad(want, d, up.double())
    rows, want = rows.detach(), want.detach()
    assert ((loss.double() - want).abs() <= S(vocab) * counted + 2 * U * rows.abs()).all(), (loss, want)
    scale = torch.where(counted, up.double().abs() / temperature, 0.0)[:, None]
    off = torch.where(counted[:, None], scale * (3 * S(vocab) + 300 * U) * magnitude(x, i, t, lse, temperature), 0.0)
    want_g = torch.where(counted[:, None], want_g, 0.0)
    fi = torch.finfo(g.dtype)
    err, tol = (g.double() - want_g).abs(), (want_g.abs() + off) * fi.eps / 2 + fi.tiny * fi.eps + off
    assert (err <= tol).all(), (float((err / tol).max()), (err > tol).nonzero()[:4])


def crossing(vocab, k, x, rest, edges):
    """Rows that list tokens around `edges`, with a student who thinks most of the tokens that lie one bitmap further on or
    back: one that a bitmap left over from there would take away."""
    few = 8
    logits, i, t, lse = make(few, vocab, k, x, "f32", rest, vocab, spread=1.0)
    around = torch.tensor([e + o for e in edges for o in (-1, 0, 1, -9, 8) if 0 <= e + o < vocab])
    i[0, : min(k, len(around))] = around[:k]
    i[1, 0] = edges[0]  # alone in its bitmap, if that begins there
    i[2] = torch.arange(k)
    i[3] = vocab - 1 - torch.arange(k)
    i[4, :2] = edges[0]  # twice
    i[5] = -1
    i[6] = torch.arange(k) * 3 + max(0, edges[0] - 10)
    i[6] = torch.where(i[6] < vocab, i[6], -1)
    for r in range(few):
        listed = {int(c) for c in i[r] if c >= 0}
        for c in listed:
            for o in (c - SEGMENT, c + SEGMENT):
                if 0 <= o < vocab and o not in listed:
                    logits[r, o] = 10.0
    return logits, i, t, lse


def tiled(v, rows):
    """As many rows: v's, again and again."""
    v, times = v.to("supa"), rows // len(v)
    return torch.cat([v[None].expand((times,) + v.shape).reshape((-1,) + v.shape[1:]), v[: rows - times * len(v)]])


def copies(rows, few, *tensors):
    at = torch.arange(rows) % few
    return [None if v is None else v[at].to("supa") for v in tensors]


@pytest.mark.parametrize("vocab", [SEGMENT + 1, 151937, 2 * SEGMENT, 2 * SEGMENT + 3])
@pytest.mark.parametrize("x, rest", [("bf16", True), ("f32", True), ("bf16", False), ("f16", True)])
def test_columns_past_one_bitmap(vocab, x, rest, no_fallback):
    """Enough rows for a workgroup each, at every alignment that an odd width gives."""
    few, rows, k = 8, 517, 12
    logits, i, t, lse = crossing(vocab, k, x, rest, [SEGMENT] if vocab < 2 * SEGMENT else [SEGMENT, 2 * SEGMENT])
    up = torch.arange(rows) % 7 + 1.0
    at = torch.arange(rows) % few
    dx, ids, tt, lt = copies(rows, few, logits, i, t, lse)
    dx.requires_grad_()
    loss = torch.supa.distillation_loss(dx, ids, tt, teacher_lse=lt, reduction="none")
    (g,) = torch.autograd.grad(loss, dx, up.to("supa"))
    loss = loss.detach().cpu()
    for c in [0, 1, 2, 3, 63]:
        r = slice(c * few, (c + 1) * few)
        against(logits, i, t, lse, up[r], loss[r], g[r].cpu())
    tail = torch.arange(rows - 5, rows)
    against(logits[at[tail]], i[at[tail]], t[at[tail]], None if lse is None else lse[at[tail]], up[tail], loss[tail], g[rows - 5:].cpu())
    # copies differ by the order of their sums, which their alignment gives
    whole = loss[: rows // few * few].view(-1, few)
    assert ((whole - whole[0]).abs() <= 2 * S(vocab) + 4 * U * whole.abs()).all()


@pytest.mark.parametrize("x, rest", [("bf16", True), ("f32", True), ("f16", False)])
def test_parts_of_more_columns_than_one_bitmap(x, rest, no_fallback):
    """Rows in three parts, each of a bitmap and some columns."""
    few, rows, vocab, k = 8, 500, 400001, 12
    part = (vocab // 3 + 256) // 256 * 256
    assert SEGMENT < part
    logits, i, t, lse = crossing(vocab, k, x, rest, [SEGMENT, part, part + SEGMENT, 2 * part, 2 * part + SEGMENT])
    dx, ids, tt, lt = copies(rows, few, logits, i, t, lse)
    dx.requires_grad_()
    up = torch.arange(rows) % 5 + 1.0
    loss = torch.supa.distillation_loss(dx, ids, tt, teacher_lse=lt, reduction="none")
    (g,) = torch.autograd.grad(loss, dx, up.to("supa"))
    loss = loss.detach().cpu()
    for c in (0, 1, 61):
        r = slice(c * few, (c + 1) * few)
        against(logits, i, t, lse, up[r], loss[r], g[r].cpu())
    whole = loss[: rows // few * few].view(-1, few)
    assert ((whole - whole[0]).abs() <= 2 * S(vocab) + 4 * U * whole.abs()).all()


@pytest.mark.parametrize("rows, vocab, x", [(66001, 1037, "bf16"), (66001, 1032, "bf16"), (65537, 700, "f32"), (262147, 16, "f32"),
                                            (262161, 21, "f16")], ids=str)
@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
def test_gradients_past_one_launch(rows, vocab, x, rest, no_fallback):
    """Launches of 65535 rows, of 262140 where four share a workgroup; another upstream value for each row, some of them
    without a pair.  The rows about the border and some of all, and that every row's gradient sums to nothing."""
    g = torch.Generator().manual_seed(rows)
    logits = torch.randn(rows, vocab, generator=g).to(T[x])
    i = torch.randint(0, vocab // 2, (rows, 3), generator=g) + torch.tensor([0, vocab // 2, 0])
    t = torch.randn(rows, 3, generator=g)
    lse = torch.logsumexp(t, 1) + 0.4 if rest else None
    i[::5] = -1
    up = 1 + torch.arange(rows) % 11 / 4
    dx = logits.to("supa").requires_grad_()
    loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"), teacher_lse=None if lse is None else lse.to("supa"), reduction="none")
    (gx,) = torch.autograd.grad(loss, dx, up.to("supa"))
    gx, loss = gx.cpu(), loss.detach().cpu()
    border = 65535 if vocab > 500 else 262140
    at = torch.unique(torch.cat([torch.arange(border - 6, rows)[:12], torch.arange(0, rows, 977), torch.arange(rows - 4, rows)]))
    against(logits[at], i[at], t[at], None if lse is None else lse[at], up[at], loss[at], gx[at])
    # each element is off by its rounding and 2 (3 S + 300 u) of what it adds up, which sums to 3 at most
    total = gx.double().sum(1).abs()
    fi = torch.finfo(T[x])
    assert (total <= up * (3 * fi.eps / 2 + 3 * (3 * S(vocab) + 300 * U)) + vocab * fi.tiny).all()
    assert not gx[::5].any() and not loss[::5].any()


def test_short_rows_past_one_launch(no_fallback):
    """A launch of the forward holds 4 (2^24 - 1) rows of a wavefront each."""
    rows, few, vocab = 4 * ((1 << 24) - 1) + 5, 1013, 2
    logits, _, t, _ = make(few, vocab, 1, "bf16", "f16", False, 1)
    i = (torch.arange(few) % 3 - 1)[:, None].int()
    up = 1 + torch.arange(few) % 11 / 4
    dx, ids, tt, u = (tiled(v, rows) for v in (logits, i, t, up))
    dx.requires_grad_()
    loss = torch.supa.distillation_loss(dx, ids, tt, reduction="none")
    (g,) = torch.autograd.grad(loss, dx, u)
    loss, g = loss.detach().cpu(), g.cpu()
    against(logits, i.long(), t, None, up, loss[:few], g[:few])
    n = rows // few * few
    assert torch.equal(loss[:n].view(-1, few), loss[:few].expand(n // few, few)) and torch.equal(loss[n:], loss[: rows - n])
    assert torch.equal(g[:n].view(-1, few, 2), g[:few].expand(n // few, few, 2)) and torch.equal(g[n:], g[: rows - n])
    del dx, ids, tt, u
    torch.supa.empty_cache()


@pytest.mark.parametrize("history", [False, True])
def test_adjusted_rows_past_one_launch(history, no_fallback):
    """A launch holds 2^26 - 8 rows of one wavefront: in order, and (with a history) eight apart, where the last workgroups
    of a launch have no row."""
    rows, few, vocab = (1 << 26) - 8 + 13, 1013, 3
    x = (torch.randn(few, vocab, generator=torch.Generator().manual_seed(2)) * 4).bfloat16()
    tokens = (torch.arange(few) % 5 - 1)[:, None].int()
    allowed = torch.tensor([5], dtype=torch.int32)
    buf = torch.full((rows * vocab + 64,), 7.0, dtype=torch.bfloat16, device="supa")
    dx = buf[: rows * vocab].view(rows, vocab)
    dx.copy_(tiled(x, rows))
    kw = dict(tokens=tiled(tokens, rows), repetition=2.0, presence=0.5) if history else {}
    torch.supa.adjust_logits_(dx, allowed=allowed.to("supa"), **kw)
    got = dx.cpu()
    want = x.float()
    if history:
        said = torch.arange(vocab) == tokens
        want = torch.where(said, torch.where(want > 0, want / 2, want * 2) - 0.5, want)
    want[:, 1] = -math.inf
    want = want.bfloat16()  # halves, doubles and one difference, in float32 exact or rounded once as here
    n = rows // few * few
    assert torch.equal(got[:n].view(-1, few, vocab), want.expand(n // few, few, vocab)) and torch.equal(got[n:], want[: rows - n])
    assert (buf[rows * vocab:].cpu() == 7).all()
    del buf, dx, kw
    torch.supa.empty_cache()


@pytest.mark.parametrize("rows, length", [(69, 65000), (71, 65000), (66, 70001), (513, 9001)], ids=str)
def test_rows_eight_apart(rows, length, no_fallback):
    """Long histories, whose rows' ranges are eight workgroups apart, of rows that are no multiple of eight: each row is
    what a call for it alone gives, and what lies beside and behind the rows stays."""
    vocab = 9001
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, vocab, generator=g) * 4).bfloat16()
    tokens = (vocab * torch.rand(rows, length, generator=g) ** 3).int().clamp_(max=vocab - 1)
    kw = {"tokens": tokens, "lengths": length - torch.arange(rows), "prompt_lengths": torch.arange(rows) * 37,
          "repetition": 1 + torch.rand(rows, generator=g), "presence": torch.rand(rows, generator=g),
          "frequency": torch.rand(rows, generator=g) / 8, "bias_tokens": torch.randint(0, vocab, (rows, 9), generator=g),
          "bias": torch.randn(rows, 9, generator=g)}
    kw = {n: v.to("supa") for n, v in kw.items()}
    wide = torch.full((rows + 9, vocab + 6), 7.0, dtype=torch.bfloat16, device="supa")
    view = wide[:rows, 3: 3 + vocab]
    view.copy_(x.to("supa"))
    out = torch.supa.adjust_logits(view, **kw).cpu()
    torch.supa.adjust_logits_(view, **kw)
    got = wide.cpu()
    assert torch.equal(got[:rows, 3: 3 + vocab], out)
    assert (got[rows:] == 7).all() and (got[:, :3] == 7).all() and (got[:, 3 + vocab:] == 7).all()
    dx = x.to("supa")
    for r in range(rows):
        one = torch.supa.adjust_logits(dx[r: r + 1], **{n: v[r: r + 1] for n, v in kw.items()})
        assert torch.equal(one.cpu()[0], out[r]), r
