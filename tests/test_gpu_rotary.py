"""torch.supa.rotary_embedding and rotary_embedding_ against complex rotations
in float64 (CPU); its gradient against the inverse rotation, autograd's second
derivative, and a difference.

Tolerance, derived: the fraction of a turn is formed in float64 (off by
2^-52 |turns|, below 1e-9 at the positions here), rounded to float32 (2^-24 of
half a turn: an angle off by 1.9e-7), its sine and cosine are off by at most 2
units of 2^-24, the scale's product and the rotation's three operations each by
one: under 8 of 2^-24 times |a| + |b| in all, then the output's own half step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def turned(x, angle, half, scale, inverse=False):
    """x [batch, seq, heads, dim] by angle [batch, seq, pairs], in float64; and |a| + |b| of each element."""
    r = 2 * angle.shape[-1]
    v = x[..., :r].double()
    p = v.unflatten(-1, (2, r // 2)).transpose(-1, -2) if half else v.unflatten(-1, (r // 2, 2))
    by = torch.polar(torch.full_like(angle, scale), -angle if inverse else angle).unsqueeze(2)
    got = torch.view_as_real(torch.view_as_complex(p.contiguous()) * by)
    mag = p.abs().sum(-1, keepdim=True).expand_as(p) * abs(scale)
    join = (lambda t: t.transpose(-1, -2).flatten(-2)) if half else (lambda t: t.flatten(-2))
    rest = x[..., r:].double()
    return torch.cat((join(got), rest), -1), torch.cat((join(mag), 0 * rest), -1)


def check(got, want, mag):
    fi = torch.finfo(got.dtype)
    err = (got.double().cpu() - want).abs()
    tol = want.abs() * fi.eps / 2 + fi.tiny * fi.eps + 8 * 2.0 ** -24 * mag * (1 + fi.eps)
    assert not (err > tol).any(), float((err / tol.clamp_min(1e-300)).max())


CASES = [
    # batch, seq, heads, kv_heads, dim, rotary, type, layout, memory, start, scale
    (2, 33, 8, 2, 128, 128, "bf16", "half", "bshd", 0, 1.0),
    (3, 21, 12, 12, 72, 36, "f32", "interleaved", "bhsd", 1000000, 1.0),
    (1, 1, 1, 1, 64, 64, "f32", "half", "bshd", 7, 1.0),
    (64, 1, 32, 8, 128, 128, "bf16", "half", "bshd", 250000, 1.0),
    (2, 17, 5, 1, 80, 32, "f16", "half", "bshd", 0, 1.25),
    (2, 17, 5, 1, 80, 32, "f16", "interleaved", "bhsd", 5000, 1.25),
    (1, 130, 3, 1, 10, 6, "bf16", "half", "bshd", 3, 1.0),
    (1, 130, 3, 2, 11, 6, "bf16", "interleaved", "bhsd", 3, 1.0),
    (2, 9, 7, 1, 257, 254, "f32", "half", "bhsd", 12, 1.0),
    (1, 5, 64, 8, 256, 256, "f16", "half", "bshd", 100, 1.0),
    (1, 3, 100, 30, 192, 190, "bf16", "interleaved", "bshd", 0, 1.0),
    (1, 2, 2, 1, 1200, 1024, "f32", "half", "bshd", 0, 1.0),
    (1, 1000, 1, 1, 2, 2, "f32", "interleaved", "bshd", 0, 1.0),
]


def inputs(c, seed=0):
    b, s, hq, hk, dim, rotary, t, layout, memory, start, scale = c
    g = torch.Generator().manual_seed(seed)

    def one(h):
        if memory == "bhsd":
            return torch.randn(b, h, s, dim, generator=g).to(T[t]).transpose(1, 2)
        return torch.randn(b, s, h, dim, generator=g).to(T[t])

    f = 10000.0 ** (-torch.arange(rotary // 2, dtype=torch.float64) * 2 / rotary)
    return one(hq), one(hk), f


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c))
def test_rotation_and_gradient(case, no_fallback):
    b, s, hq, hk, dim, rotary, t, layout, memory, start, scale = case
    q, k, f = inputs(case)
    gq, gk, _ = inputs(case, 1)
    g = torch.Generator().manual_seed(2)
    pos = start + (torch.arange(s).expand(b, s) if s > 1 else torch.randint(0, 4096, (b, 1), generator=g))
    angle = pos.double().unsqueeze(-1) * f
    half = layout == "half"
    dq, dk = q.to("supa").requires_grad_(), k.to("supa").requires_grad_()
    assert dq.stride() == q.stride()
    fd = f.to("supa")
    oq, ok = torch.supa.rotary_embedding(dq, dk, fd, pos.to("supa"), layout=layout, scale=scale)
    assert oq.stride() == q.stride() and ok.stride() == k.stride() and oq.dtype == T[t]
    check(oq.detach(), *turned(q, angle, half, scale))
    check(ok.detach(), *turned(k, angle, half, scale))
    got = torch.autograd.grad([oq, ok], [dq, dk], [gq.to("supa"), gk.to("supa")])
    for a, src in zip(got, (gq, gk)):
        check(a, *turned(src, angle, half, scale, inverse=True))
    # int32 positions, narrower frequencies' type and q alone: the same bits
    with torch.no_grad():
        alone, none = torch.supa.rotary_embedding(dq, None, fd, pos.to("supa", torch.int32), layout=layout, scale=scale)
        assert none is None and torch.equal(alone.cpu(), oq.detach().cpu())
        if s > 1:
            for p in (pos[0].to("supa"), pos[:1].to("supa"), start):
                again, _ = torch.supa.rotary_embedding(dq, dk, fd, p, layout=layout, scale=scale)
                assert torch.equal(again.cpu(), oq.detach().cpu())


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c))
def test_in_place_in_a_packed_projection(case, no_fallback):
    """q and k as views of one tensor: the same values, and what does not turn
    (the rest of the heads, v) as it was."""
    b, s, hq, hk, dim, rotary, t, layout, memory, start, scale = case
    g = torch.Generator().manual_seed(3)
    _, _, f = inputs(case)
    shape = (b, hq + 2 * hk, s, dim) if memory == "bhsd" else (b, s, hq + 2 * hk, dim)
    host = torch.randn(shape, generator=g).to(T[t])
    dev = host.to("supa")

    def views(p):
        p = p.transpose(1, 2) if memory == "bhsd" else p
        return p[:, :, :hq], p[:, :, hq: hq + hk], p[:, :, hq + hk:]

    q, k, v = views(dev)
    want = torch.supa.rotary_embedding(q, k, f.to("supa"), start, layout=layout, scale=scale)
    version = dev._version
    got = torch.supa.rotary_embedding_(q, k, f.to("supa"), start, layout=layout, scale=scale)
    assert got[0] is q and got[1] is k and dev._version > version
    hv = views(host)
    assert torch.equal(q.cpu(), want[0].cpu()) and torch.equal(k.cpu(), want[1].cpu())
    assert torch.equal(v.cpu(), hv[2]) and torch.equal(q.cpu()[..., rotary:], hv[0][..., rotary:])


def test_positions_far_out(no_fallback):
    """Positions past 2^31 and negative ones: the angle keeps its fraction of a turn."""
    f = torch.tensor([1.0, 0.3, 1e-3, 1e-5], dtype=torch.float64)
    pos = torch.tensor([0, -5, 10 ** 6, 2 ** 31 + 3, 2 ** 40 + 1, -(2 ** 33)])
    x = torch.randn(6, 2, 8, generator=torch.Generator().manual_seed(1))
    got, _ = torch.supa.rotary_embedding(x.to("supa"), None, f.to("supa"), pos.to("supa"))
    want, mag = turned(x.unsqueeze(0), (pos.double().unsqueeze(-1) * f).unsqueeze(0), True, 1.0)
    # 2^-52 of 2^40 / 6.28 turns is an angle off by 2.5e-4 at most there, less elsewhere
    slack = (2.0 ** -51 * pos.double().abs() * 1.0).view(1, -1, 1, 1) * mag
    err = (got.double().cpu() - want[0]).abs()
    assert not (err > (8 * 2.0 ** -24 * mag + slack)[0] + 2.0 ** -24 * want[0].abs()).any()
    one, _ = torch.supa.rotary_embedding(x[3:4].to("supa"), None, f.to("supa"), 2 ** 31 + 3)
    assert torch.equal(one.cpu(), got[3:4].cpu())


def test_offsets_past_32_bits(no_fallback):
    """Samples that lie 2^31 elements apart, and almost 2^31 tokens: the same
    bits as the same rows close together."""
    g = torch.Generator().manual_seed(8)
    f = torch.tensor([1.0, 0.01], dtype=torch.float64, device="supa")
    near = torch.randn(2, 3, 2, 5, generator=g).half().to("supa")
    room = torch.empty(2 ** 31 + 64, dtype=torch.half, device="supa")
    far = room.as_strided((2, 3, 2, 5), (2 ** 31, 10, 5, 1), 7)
    far.copy_(near)
    for layout in ("half", "interleaved"):
        want, _ = torch.supa.rotary_embedding(near, None, f, 9, layout=layout)
        assert torch.equal(torch.supa.rotary_embedding(far, None, f, 9, layout=layout)[0].cpu(), want.cpu())
    torch.supa.rotary_embedding_(far, None, f, 9, layout="interleaved")
    assert torch.equal(far.cpu(), want.cpu())
    del far, room
    n, last = 2 ** 31 - 3, 700
    row = torch.tensor([[[0.5, -1.5]]], device="supa", dtype=torch.bfloat16)
    got, _ = torch.supa.rotary_embedding(row.expand(n, 1, 2), None, f[1:])
    for at in (0, 2 ** 30 - 300, n - last):
        want, _ = torch.supa.rotary_embedding(row.expand(last, 1, 2), None, f[1:], at)
        assert torch.equal(got[at: at + last].cpu(), want.cpu())


def test_second_derivative_and_difference(no_fallback):
    q = torch.randn(4, 2, 16, generator=torch.Generator().manual_seed(5)).to("supa").requires_grad_()
    f, scale = torch.supa.rotary_frequencies(12, scaling="yarn", factor=4.0, original_length=64)
    def loss(x):
        o, _ = torch.supa.rotary_embedding(x, None, f, 100, layout="interleaved", scale=scale)
        return (o * o * o).sum()
    (g,) = torch.autograd.grad(loss(q), q, create_graph=True)
    (gg,) = torch.autograd.grad(g.sum(), q)
    pos = torch.arange(100, 104).double().view(1, 4, 1)
    ref = q.detach().double().cpu().requires_grad_()
    a = pos * f.cpu()
    def ref_loss(x):
        r = 12
        p = x[..., :r].unflatten(-1, (6, 2))
        c, s = a.cos()[0].unsqueeze(1) * scale, a.sin()[0].unsqueeze(1) * scale
        o = torch.stack((p[..., 0] * c - p[..., 1] * s, p[..., 1] * c + p[..., 0] * s), -1).flatten(-2)
        return (o ** 3).sum() + (x[..., r:] ** 3).sum()
    (rg,) = torch.autograd.grad(ref_loss(ref), ref, create_graph=True)
    (rgg,) = torch.autograd.grad(rg.sum(), ref)
    # cubes of two rotated terms: a dozen float32 operations on values up to 3 * 4^2 * 1.2^3
    assert (g.detach().double().cpu() - rg.detach()).abs().max() <= 40 * 2.0 ** -24 * rg.abs().max()
    assert (gg.double().cpu() - rgg).abs().max() <= 60 * 2.0 ** -24 * rgg.abs().max()
    way = torch.randn(4, 2, 16, generator=torch.Generator().manual_seed(6), dtype=torch.float64)
    with torch.no_grad():
        slope = (ref_loss(ref + 1e-4 * way) - ref_loss(ref - 1e-4 * way)) / 2e-4
    assert abs(float((g.detach().double().cpu() * way).sum() - slope)) <= 1e-5 * float((rg.detach().abs() * way.abs()).sum())


def test_only_k_has_a_gradient(no_fallback):
    q, k, f = inputs(CASES[0])
    dk = k.to("supa").requires_grad_()
    oq, ok = torch.supa.rotary_embedding(q.to("supa"), dk, f.to("supa"), 3)
    ones = torch.ones_like(ok)
    (g,) = torch.autograd.grad((ok * ones).sum(), dk)
    want, mag = turned(torch.ones_like(k), (3 + torch.arange(33).double()).view(1, -1, 1) * f, True, 1.0, inverse=True)
    check(g, want.expand_as(k), mag.expand_as(k))


def test_empty(no_fallback):
    f = torch.ones(4, dtype=torch.float64, device="supa")
    for shape in ((0, 3, 8), (2, 0, 3, 8), (2, 5, 0, 8)):
        q = torch.ones(shape, device="supa")
        o, _ = torch.supa.rotary_embedding(q, None, f)
        assert o.shape == q.shape
        torch.supa.rotary_embedding_(q, q.clone(), f)


def test_refusals(supa):
    f = torch.ones(4, dtype=torch.float64, device="supa")
    q = torch.ones(2, 5, 3, 8, device="supa")
    rot = torch.supa.rotary_embedding
    for args, kw, text in [
        ((q.cpu(), None, f), {}, "supa"), ((q, q.cpu(), f), {}, "k is on"), ((q, None, f.cpu()), {}, "frequencies is on"),
        ((q.double(), None, f), {}, "float32, bfloat16"), ((q, q.half(), f), {}, "k of"),
        ((q, q[:, :4], f), {}, "more than their heads"), ((q[0, 0], None, f), {}, "shape"),
        ((q, None, torch.ones(8, dtype=torch.float64, device="supa")), {}, "rotate"), ((q, None, f[:0]), {}, "rotate"), ((q, None, f.long()), {}, "floats"),
        ((q, None, f, torch.ones(4, dtype=torch.long, device="supa")), {}, "positions"),
        ((q, None, f, torch.ones(3, 5, dtype=torch.long, device="supa")), {}, "positions"),
        ((q, None, f, torch.ones(5, device="supa")), {}, "int64 or int32"),
        ((q, None, f, torch.ones(5, dtype=torch.long)), {}, "positions is on"),
        ((q, None, f, 1.5), {}, "positions"), ((q, None, f), dict(layout="third"), "layout"),
        ((q, None, f), dict(scale=math.inf), "scale"),
    ]:
        with pytest.raises((RuntimeError, ValueError, TypeError, NotImplementedError), match=text):
            rot(*args, **kw)
    with pytest.raises(RuntimeError, match="no gradient"):
        rot(q, None, f.clone().requires_grad_())
    put = torch.supa.rotary_embedding_
    with pytest.raises(RuntimeError, match="overlap"):
        put(q, q, f)
    with pytest.raises(RuntimeError, match="overlap"):
        put(q[:, :, :2], q[:, :, 1:], f)
    with pytest.raises(RuntimeError, match="overlap"):
        put(q[:, :4], q[:, 1:], f)
    with pytest.raises(RuntimeError, match="overlap"):  # windows that slide over each other
        put(torch.ones(100, device="supa").as_strided((4, 5, 1, 8), (10, 11, 8, 1)), None, f)
    with pytest.raises(RuntimeError, match="contiguous"):
        put(torch.ones(2, 5, 8, 3, device="supa").transpose(2, 3), None, f)
    with pytest.raises(RuntimeError):
        put(torch.ones(1, 5, 3, 8, device="supa").expand(2, 5, 3, 8), None, f)
    with pytest.raises(RuntimeError, match="no gradient"):
        put(q.clone().requires_grad_(), None, f)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, q.clone())
        for call in (rot, put):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual, None, f)
