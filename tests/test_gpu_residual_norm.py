"""torch.supa.residual_norm against its definition in float64 (CPU), its
gradients against torch's autograd of that definition and against central
differences.

Tolerances, derived: an output rounds once, by eps/2 of its type relative to
the value (f16 subnormals: half their spacing).  Everything before that is
float32: a sum over a row adds at most 16 values a thread, then a tree of at
most 4 + 4 steps and 16 wavefronts, so it is off by under 40 of 2^-24 times the
sum of magnitudes; with the products around it no result is off by more than
K = 128 of 2^-24 times its magnitude, the same formula evaluated on absolute
values.  Column sums add at most 16 rows' values in sequence here, then their
partials.  Where the backward starts from a rounded h (no gate, no post norm,
16-bit residual and parameters) the relative half step of h's type enters the
normalised value too, and is propagated."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
K = 128 * 2.0 ** -24
NAMES = ("x", "residual", "gate", "post_weight", "post_bias", "weight", "bias")


def make(shape, x, residual, params, gate, post, norm, seed):
    g = torch.Generator().manual_seed(seed)
    width = shape[-1]

    def rnd(s, t, scale=1.0, shift=0.0):
        return (torch.randn(s, generator=g, dtype=torch.float64) * scale + shift).to(T[t])

    loud = 1 + 15 * (torch.rand(width, generator=g) < 0.02).double()
    d = {"x": rnd(shape, x), "residual": (torch.randn(shape, generator=g, dtype=torch.float64) * loud).to(T[residual])}
    if gate is not None:
        gs = {"channel": (width,), "sample": (shape[0],) + (1,) * (len(shape) - 2) + (width,), "full": shape}[gate]
        d["gate"] = rnd(gs, params, 0.3, 0.5)
    for kind, w, b in ((post, "post_weight", "post_bias"), (norm, "weight", "bias")):
        if kind is not None:
            d[w] = rnd((width,), params, 0.1, 1.0)
        if kind == "layer":
            d[b] = rnd((width,), params, 0.1)
    return d, rnd(shape, residual), rnd(shape, x) if norm else None


def normed(v, kind, w, b, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    v = v if w is None else v * w
    return v if b is None else v + b


def definition(d, scale, post, norm, eps):
    u = d["x"] if post is None else normed(d["x"], post, d.get("post_weight"), d.get("post_bias"), eps)
    h = scale * d["residual"] + (u if d.get("gate") is None else u * d["gate"])
    return h, None if norm is None else normed(h, norm, d.get("weight"), d.get("bias"), eps)


def magnitudes(d, gh, gy, scale, post, norm, eps, rounded_h):
    """The formulas of outputs and gradients on absolute values (float64);
    rounded_h: relative error of the h that the backward starts from."""
    v = {k: t.double() for k, t in d.items()}
    one = torch.ones((), dtype=torch.float64)

    def stats(t, kind):
        c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
        r = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
        return r, (t.abs() + (t.abs().mean(-1, keepdim=True) if kind == "layer" else 0.0)) * r

    def back(a, n, r, kind):
        return r * (a + (a.mean(-1, keepdim=True) if kind == "layer" else 0.0) + n * (a * n).mean(-1, keepdim=True))

    m, u = {}, v["x"].abs()
    if post:
        pr, pn = stats(v["x"], post)
        u = pn * v.get("post_weight", one).abs() + v.get("post_bias", 0 * one).abs()
    gate = v.get("gate", one).abs()
    H = abs(scale) * v["residual"].abs() + gate * u
    m["h"] = H
    dH = gh.double().abs() if gh is not None else torch.zeros_like(H)
    extra = {}
    if norm:
        h, _ = definition(v, scale, post, None, eps)
        r, _ = stats(h, norm)
        n = (H + (H.mean(-1, keepdim=True) if norm == "layer" else 0.0)) * r
        m["y"] = n * v.get("weight", one).abs() + v.get("bias", 0 * one).abs()
        if gy is not None:
            a = gy.double().abs()
            m["weight"] = (a * n).reshape(-1, a.shape[-1]).sum(0)
            m["bias"] = a.reshape(-1, a.shape[-1]).sum(0)
            dn = rounded_h * h.abs() * r
            extra["weight"] = (a * dn).reshape(-1, a.shape[-1]).sum(0)
            a = a * v.get("weight", one).abs()
            dH = dH + back(a, n, r, norm)
            extra["x"] = r * (dn * (a * n).mean(-1, keepdim=True) + n * (a * dn).mean(-1, keepdim=True))
            extra["residual"] = abs(scale) * extra["x"]
    m["residual"] = abs(scale) * dH
    if d.get("gate") is not None:
        m["gate"] = (u * dH).sum_to_size(d["gate"].shape)
    du = gate * dH
    if post:
        m["post_weight"] = (du * pn).reshape(-1, du.shape[-1]).sum(0)
        m["post_bias"] = du.reshape(-1, du.shape[-1]).sum(0)
        du = back(du * v.get("post_weight", one).abs(), pn, pr, post)
    m["x"] = du
    return m, extra


def check(name, got, want, m, extra):
    assert got.shape == want.shape, name
    fi = torch.finfo(got.dtype)
    tol = want.abs() * fi.eps / 2 + fi.tiny * fi.eps + (1 + fi.eps) * (K * m[name] + extra.get(name, 0.0))
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((err / tol.clamp_min(1e-300)).max()))


CASES = [
    # shape, x, residual, params, gate, post, norm, scale
    ((1, 1, 4096), "bf16", "bf16", "bf16", "channel", "rms", "rms", 1.0),
    ((3, 5, 4096), "bf16", "bf16", "bf16", "channel", "rms", "rms", 1.0),
    ((3, 37, 2047), "f32", "f32", "f32", "sample", "layer", "layer", 0.5),
    ((2, 33, 8192), "bf16", "f32", "f32", None, None, "rms", 1.0),
    ((2, 9, 8192), "bf16", "bf16", "bf16", None, None, "rms", 1.0),
    ((41, 8200), "bf16", "bf16", "f32", "full", "layer", "layer", 0.7071),
    ((17, 16384), "f16", "f32", "f16", "channel", "layer", "layer", 1.0),
    ((5, 16381), "f32", "f32", "f32", "channel", "layer", "rms", 1.0),
    ((4, 61, 64), "f16", "f16", "f16", "sample", "rms", "layer", 1.0),
    ((1000, 128), "bf16", "bf16", "bf16", "channel", "rms", "rms", 1.0),
    ((300, 3, 40), "f32", "f32", "f32", "sample", "layer", "rms", 1.0),
    ((515, 129), "bf16", "f32", "bf16", "channel", "layer", None, 1.0),
    ((131, 512), "f16", "f32", "f32", None, "layer", "layer", 2.0),
    ((77, 513), "f32", "f32", "f32", None, None, "layer", 1.0),
    ((259, 1025), "bf16", "bf16", "f32", None, None, "layer", 1.0),
    ((700, 7), "f32", "f32", "f32", "full", "rms", "rms", 1.0),
    ((5, 3), "f16", "f16", "f16", None, "rms", None, 1.0),
    ((9, 1), "f32", "f32", "f32", "channel", "rms", "rms", 1.0),
    ((2, 130, 2048), "f32", "f32", "f32", "sample", None, "rms", 1.0),
    ((6, 4095), "bf16", "bf16", "bf16", "channel", None, None, 1.0),
    ((64, 96), "bf16", "bf16", "bf16", None, None, None, 0.5),
    ((4097,), "f32", "f32", "f32", "channel", "layer", "layer", 1.0),
    ((270, 2, 8200), "bf16", "bf16", "bf16", "sample", "layer", "layer", 1.0),
    ((270, 2, 8201), "bf16", "bf16", "bf16", "sample", "layer", "layer", 1.0),
    ((300, 2, 8195), "f32", "f32", "f32", "sample", "rms", "rms", 1.0),
    ((261, 3, 4099), "bf16", "f32", "f32", "sample", "layer", "rms", 1.0),
    ((3, 40, 9001), "f32", "f32", "f32", "sample", "rms", "rms", 1.0),
    ((160, 24, 520), "bf16", "bf16", "bf16", "sample", "layer", "layer", 1.0),
    ((300, 9, 260), "f32", "f32", "f32", "sample", "rms", "layer", 1.0),
    ((1100, 2, 70), "f32", "f32", "f32", "sample", "layer", "rms", 1.0),
    ((600, 1, 256), "bf16", "bf16", "bf16", "sample", "rms", "rms", 1.0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c))
def test_forward_and_gradients(case, no_fallback):
    shape, x, residual, params, gate, post, norm, scale = case
    eps = 1e-6
    d, gh, gy = make(shape, x, residual, params, gate, post, norm, 7)
    ref = {k: t.double().requires_grad_() for k, t in d.items()}
    h, y = definition(ref, scale, post, norm, eps)
    ends, gs = ([h, y], [gh.double(), gy.double()]) if norm else ([h], [gh.double()])
    want = dict(zip(ref, torch.autograd.grad(ends, list(ref.values()), gs)))
    dev = {k: t.to("supa").requires_grad_() for k, t in d.items()}
    kw = dict(residual_scale=scale, post_norm=post, norm=norm, eps=eps)
    args = {k: dev.get(k) for k in NAMES[2:]}
    oh, oy = torch.supa.residual_norm(dev["x"], dev["residual"], **args, **kw)
    got = torch.autograd.grad([oh, oy] if norm else [oh], list(dev.values()), [g.to("supa") for g in (gh, gy)[: len(ends)]])
    assert oh.dtype == T[residual] and (norm is None) == (oy is None)
    from_h = gate is None and post is None and norm and residual != "f32" and params != "f32"
    rounded = torch.finfo(T[residual]).eps / 2 if from_h else 0.0
    m, extra = magnitudes(d, gh, gy, scale, post, norm, eps, rounded)
    check("h", oh.detach(), h.detach(), m, {})
    if norm:
        assert oy.dtype == T[x]
        check("y", oy.detach(), y.detach(), m, {})
    for k, g in zip(dev, got):
        assert g.dtype == d[k].dtype
        check(k, g, want[k], m, extra)
    # without gradients: the same bits
    with torch.no_grad():
        nh, ny = torch.supa.residual_norm(dev["x"], dev["residual"], **args, **kw)
    assert torch.equal(nh.cpu(), oh.detach().cpu()) and (norm is None or torch.equal(ny.cpu(), oy.detach().cpu()))
    # and again: sums in an order of their own
    oh, oy = torch.supa.residual_norm(dev["x"], dev["residual"], **args, **kw)
    again = torch.autograd.grad([oh, oy] if norm else [oh], list(dev.values()), [g.to("supa") for g in (gh, gy)[: len(ends)]])
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, again))


@pytest.mark.parametrize("use", ["h", "y", "x_only", "weight_only"])
def test_partial_gradients(use, no_fallback):
    """One of the two outputs used, or one of the inputs wanted."""
    d, gh, gy = make((3, 19, 300), "f32", "f32", "f32", "sample", "layer", "layer", 11)
    ref = {k: t.double().requires_grad_() for k, t in d.items()}
    dev = {k: t.to("supa") for k, t in d.items()}
    leaves = {"x_only": ["x"], "weight_only": ["weight"]}.get(use, list(d))
    if use == "h":
        leaves = [k for k in leaves if k not in ("weight", "bias")]
    for k in leaves:
        dev[k].requires_grad_()
    pick = {"h": [0], "y": [1]}.get(use, [0, 1])
    h = definition(ref, 1.0, "layer", "layer", 1e-6)
    o = torch.supa.residual_norm(dev["x"], dev["residual"], **{k: dev[k] for k in NAMES[2:]}, post_norm="layer",
                                 norm="layer")
    gs = (gh, gy)
    want = torch.autograd.grad([h[i] for i in pick], [ref[k] for k in leaves], [gs[i].double() for i in pick])
    got = torch.autograd.grad([o[i] for i in pick], [dev[k] for k in leaves], [gs[i].to("supa") for i in pick])
    m, extra = magnitudes(d, gh if 0 in pick else None, gy if 1 in pick else None, 1.0, "layer", "layer", 1e-6, 0.0)
    for k, a, b in zip(leaves, got, want):
        check(k, a, b, m, extra)


def test_gradient_against_differences(no_fallback):
    """Along a direction: the gradient's product with it against the central
    difference of the definition in float64 (step 1e-4: its error is of third
    order, 1e-8 of the terms, below float32's)."""
    d, gh, gy = make((4, 6, 257), "f32", "f32", "f32", "channel", "rms", "layer", 3)
    dev = {k: t.to("supa").requires_grad_() for k, t in d.items()}
    o = torch.supa.residual_norm(dev["x"], dev["residual"], **{k: dev.get(k) for k in NAMES[2:]}, residual_scale=0.5,
                                 post_norm="rms", norm="layer")
    got = torch.autograd.grad(list(o), list(dev.values()), [gh.to("supa"), gy.to("supa")])
    g = torch.Generator().manual_seed(4)

    def loss(v):
        h, y = definition(v, 0.5, "rms", "layer", 1e-6)
        return float((h * gh.double()).sum() + (y * gy.double()).sum())

    m, _ = magnitudes(d, gh, gy, 0.5, "rms", "layer", 1e-6, 0.0)
    for k, grad in zip(dev, got):
        way = torch.randn(d[k].shape, generator=g, dtype=torch.float64)
        step = 1e-4
        plus, minus = ({n: t.double() + (s * step * way if n == k else 0) for n, t in d.items()} for s in (1, -1))
        slope = (loss(plus) - loss(minus)) / (2 * step)
        tol = float((way.abs() * m[k]).sum()) * (K + 1e-7)
        assert abs(float((grad.double().cpu() * way).sum()) - slope) <= tol, k


def test_views_and_strides(no_fallback):
    """x a slice of a wider projection, residual heads-first, an expanded
    gradient; the same values as from contiguous tensors, bit for bit."""
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(2, 7, 700, generator=g).to("supa")
    res = torch.randn(2, 260, 7, generator=g).to("supa").transpose(1, 2)
    w = torch.randn(260, generator=g).to("supa").requires_grad_()
    x = wide[..., 13:273]
    outs = []
    for xi, ri in ((x, res), (x.contiguous(), res.contiguous())):
        xi, ri = xi.detach().requires_grad_(), ri.detach().requires_grad_()
        h, y = torch.supa.residual_norm(xi, ri, post_norm="rms", post_weight=w, weight=w)
        gr = torch.autograd.grad((h.sum() + y.sum()), [xi, ri, w])
        outs.append([t.detach().cpu() for t in (h, y, *gr)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    row = torch.randn(1, 260, generator=g).to("supa").expand(9, 260)  # every row the same memory
    h, y = torch.supa.residual_norm(row, row, weight=w.detach())
    assert torch.equal(h.cpu(), (row.cpu() * 2)) and torch.equal(y[0].cpu(), y[8].cpu())


def test_saved_tensors_come_back_otherwise(no_fallback):
    """Hooks that keep what the backward needs elsewhere give it back with other
    strides (a slice of a wider projection contiguous, a contiguous tensor as
    every second row): the same gradients, bit for bit; another shape or type
    raises."""
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(40, 700, generator=g).to("supa")
    w = torch.randn(260, generator=g).to("supa").requires_grad_()
    apart = lambda t: torch.stack((t, t), -2)[..., 0, :] if t.dim() > 1 else torch.stack((t, t), -1)[..., 0]  # noqa: E731

    def grads(unpack):
        x = wide[:, 13:273].detach().requires_grad_()
        r = wide[:, 300:560].detach().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
            h, y = torch.supa.residual_norm(x, r, post_norm="rms", post_weight=w, weight=w)
        return [t.cpu() for t in torch.autograd.grad(h.sum() + y.sum(), [x, r, w])]

    want = grads(lambda t: t)
    for unpack in (torch.Tensor.contiguous, apart, lambda t: t.cpu().to("supa")):
        assert all(torch.equal(a, b) for a, b in zip(grads(unpack), want))
    for unpack in (torch.Tensor.half, lambda t: t[:1], torch.Tensor.cpu):
        with pytest.raises(RuntimeError, match="saved tensor came back"):
            grads(unpack)


def test_changed_or_used_twice(no_fallback):
    """A saved tensor that was written since, and a second backward, raise."""
    x = torch.ones(4, 64, device="supa", requires_grad=True)
    w = torch.ones(64, device="supa", requires_grad=True)
    r = torch.ones(4, 64, device="supa")
    h, y = torch.supa.residual_norm(x, r, weight=w, gate=torch.ones(64, device="supa"))
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    h, y = torch.supa.residual_norm(x, r, weight=w, gate=torch.ones(64, device="supa"))
    r.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    h, y = torch.supa.residual_norm(x, r, weight=w)  # keeps h
    h.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_offsets_past_32_bits(no_fallback):
    """Rows that lie 2^30 elements apart: the same bits as from close ones."""
    g = torch.Generator().manual_seed(12)
    near = torch.randn(3, 300, generator=g).bfloat16().to("supa")
    room = torch.empty(2 ** 31 + 400, dtype=torch.bfloat16, device="supa")
    far = room.as_strided((3, 300), (2 ** 30, 1), 5)
    far.copy_(near)
    w = torch.randn(300, generator=g).bfloat16().to("supa").requires_grad_()
    outs = []
    for t in (near, far):
        x, r = t.detach().requires_grad_(), t.detach().requires_grad_()
        h, y = torch.supa.residual_norm(x, r, post_norm="layer", post_weight=w, weight=w)
        outs.append([o.detach().cpu() for o in (h, y, *torch.autograd.grad(h.sum() + y.sum(), [x, r, w]))])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_zero_nan_and_infinite_rows(no_fallback):
    d, gh, gy = make((6, 1000), "bf16", "bf16", "bf16", "channel", "rms", "rms", 9)
    dev = {k: t.to("supa") for k, t in d.items()}
    kw = {k: dev.get(k) for k in NAMES[2:]}
    clean = torch.supa.residual_norm(dev["x"], dev["residual"], post_norm="rms", norm="rms", **kw)
    x, r = d["x"].clone(), d["residual"].clone()
    x[1], r[1] = 0, 0
    x[2, 7] = math.nan
    r[3, 999] = math.inf
    h, y = (t.cpu().float() for t in torch.supa.residual_norm(x.to("supa"), r.to("supa"), post_norm="rms", norm="rms", **kw))
    assert (h[1] == 0).all() and (y[1] == 0).all()
    assert h[2].isnan().all() and y[2].isnan().all()
    assert torch.isinf(h[3, 999]) and y[3, 999].isnan() and (y[3, :999] == 0).all()
    for i in (0, 4, 5):
        assert torch.equal(h[i], clean[0][i].cpu().float()) and torch.equal(y[i], clean[1][i].cpu().float())


def test_no_rows(no_fallback):
    x = torch.empty(0, 5, 64, device="supa", requires_grad=True)
    w = torch.ones(64, device="supa", requires_grad=True)
    h, y = torch.supa.residual_norm(x, x.detach(), weight=w)
    assert h.shape == y.shape == (0, 5, 64)
    gx, gw = torch.autograd.grad(h.sum() + y.sum(), [x, w])
    assert gx.shape == x.shape and (gw == 0).all().item()


def test_on_another_stream(no_fallback):
    d, gh, gy = make((64, 33, 1024), "bf16", "bf16", "bf16", None, "rms", "rms", 21)
    dev = {k: t.to("supa") for k, t in d.items()}
    kw = {k: dev.get(k) for k in NAMES[2:]}
    want = [t.cpu() for t in torch.supa.residual_norm(dev["x"], dev["residual"], post_norm="rms", **kw)]
    s = torch.supa.Stream()
    s.wait_stream(torch.supa.current_stream())
    with torch.supa.stream(s):
        x = dev["x"] * 1  # produced on the stream, used there
        got = torch.supa.residual_norm(x, dev["residual"], post_norm="rms", **kw)
    s.synchronize()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_refusals(supa):
    f = torch.supa.residual_norm
    x = torch.ones(4, 8, device="supa")
    w = torch.ones(8, device="supa")
    bad = [
        (dict(x=x.cpu()), "supa"),
        (dict(residual=torch.ones(4, 9, device="supa")), "shape"),
        (dict(residual=x.cpu()), "expected supa"),
        (dict(x=x.double(), residual=x.double()), "float32, bfloat16 or float16"),
        (dict(residual=x.half()), "residual of x's dtype"),
        (dict(weight=w[:7]), "shape"),
        (dict(weight=w.half()), "weight of x's dtype"),
        (dict(bias=w), "not a layer norm"),
        (dict(post_weight=w), "without a post norm"),
        (dict(norm=None, weight=w), "without a norm"),
        (dict(norm="batch"), "expected norm"),
        (dict(gate=torch.ones(3, 8, device="supa")), "gate"),
        (dict(gate=torch.ones(4, 1, device="supa")), "gate"),
        (dict(eps=-1.0), "eps"),
        (dict(eps=math.nan), "eps"),
        (dict(x=torch.ones((), device="supa"), residual=torch.ones((), device="supa")), "last dim"),
        (dict(x=torch.ones(2, 16385, device="supa"), residual=torch.ones(2, 16385, device="supa")), "16384"),
    ]
    for kw, text in bad:
        args = {"x": x, "residual": x, **kw}
        with pytest.raises((RuntimeError, ValueError, NotImplementedError), match=text):
            f(args.pop("x"), args.pop("residual"), **args)
    h = x.half()
    with pytest.raises(RuntimeError, match="of one dtype"):
        f(h, h, weight=w, gate=w.half())
    with pytest.raises(RuntimeError, match="gate"):  # one value a position, not a sample
        f(torch.ones(2, 3, 8, device="supa"), torch.ones(2, 3, 8, device="supa"), gate=torch.ones(1, 3, 8, device="supa"))
    xg = x.clone().requires_grad_()
    y = f(xg, x)[1]
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum(), xg, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w, w)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(x, x, weight=dual)
        assert f(x, x, weight=w)[0].shape == x.shape
