"""Values of the transformer operators where the other tests do not look:
outputs that start as NaN (an element that is not written, or written as NaN,
fails), frequencies of narrower types, and more rows than one launch takes.

Tolerances are those derived in test_gpu_rotary.py, test_gpu_clip_grad.py and
test_gpu_residual_norm.py."""
import ctypes

import pytest
import torch

import torch_supa
from test_gpu_clip_grad import SPECS, as_params, grads_of, norm_of
from test_gpu_residual_norm import K
from test_gpu_rotary import CASES, T, inputs, turned
from test_transformer_args import BF16, F16, F32, I64, RotaryDesc, RotaryTensor, vp

pytestmark = pytest.mark.gpu

CODES = {"f32": F32, "bf16": BF16, "f16": F16}


def within(got, want, mag):
    fi = torch.finfo(got.dtype)
    tol = want.abs() * fi.eps / 2 + fi.tiny * fi.eps + 8 * 2.0 ** -24 * mag * (1 + fi.eps)
    return bool(((got.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c))
def test_rotary_writes_every_element(case, supa):
    """Outputs inside a buffer of NaN: all of theirs are written, nothing around them."""
    b, s, hq, hk, dim, rotary, t, layout, memory, start, scale = case
    lib = ctypes.CDLL(torch_supa.KERNELS_LIB)
    q, k, f = inputs(case)
    pos = start + torch.arange(s)
    angle = pos.double().view(1, s, 1).expand(b, s, 1) * f
    freq, dpos = f.cuda(), pos.cuda()
    for inverse in (0, 1):
        d = RotaryDesc(batch=b, seq=s, dim=dim, rotary=rotary, dtype=CODES[t], layout=int(layout == "interleaved"),
                       inverse=inverse, position_dtype=I64, scale=scale, frequencies=freq.data_ptr(),
                       positions=dpos.data_ptr())
        d.position_strides[1] = 1
        outs = []
        for x, desc in ((q, d.q), (k, d.k)):
            src = x.cuda()
            room = torch.full((src.numel() + 96,), float("nan"), dtype=T[t], device="cuda")
            out = room.as_strided(src.shape, src.stride(), 32)
            desc.data_in, desc.out, desc.heads = src.data_ptr(), out.data_ptr(), x.shape[2]
            for i in range(3):
                desc.in_strides[i], desc.out_strides[i] = src.stride(i), out.stride(i)
            outs.append((x, src, room, out))
        assert lib.supa_amd_rotary(ctypes.byref(d), vp(torch.cuda.current_stream().cuda_stream)) == 0
        torch.cuda.synchronize()
        for x, _, room, out in outs:
            assert within(out, *turned(x, angle, layout == "half", scale, inverse=bool(inverse)))
            assert room[:32].isnan().all() and room[out.numel() + 32:].isnan().all()


@pytest.mark.parametrize("p", [2.0, 1.0, float("inf")])
@pytest.mark.parametrize("spec", SPECS)
def test_clipped_values_are_numbers(spec, p, no_fallback):
    host = grads_of(SPECS[spec], 2)
    norm = norm_of(host, p)
    dev = [g.to("supa") for g in host]
    got = float(torch.supa.clip_grad_norm_(as_params(dev), 0.25 * norm, norm_type=p))
    assert abs(got - norm) <= norm * (2.0 ** -24 + 1e-12)
    c = 0.25 * norm / (norm + 1e-6)
    for a, b in zip(dev, host):
        fi, want = torch.finfo(b.dtype), b.double() * c
        assert ((a.double().cpu() - want).abs() <= want.abs() * (fi.eps / 2 + 3 * 2.0 ** -24) + fi.tiny * fi.eps).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_narrower_frequencies(dtype, no_fallback):
    """They are widened: the values of the float64 vector that they stand for, forward, gradient and in place."""
    case = (2, 19, 3, 1, 72, 48, "f32", "half", "bshd", 100, 1.25)
    q, k, f = inputs(case)
    f = f.to(dtype)
    angle = (100 + torch.arange(19)).double().view(1, 19, 1).expand(2, 19, 1) * f.double()
    dq, dk = q.to("supa").requires_grad_(), k.to("supa").requires_grad_()
    outs = []
    for v in (f.to("supa"), f.double().to("supa")):
        oq, ok = torch.supa.rotary_embedding(dq, dk, v, 100, scale=1.25)
        placed, _ = torch.supa.rotary_embedding_(q.to("supa"), None, v, 100, scale=1.25)
        outs.append([t.detach().cpu() for t in (oq, ok, *torch.autograd.grad([oq, ok], [dq, dk], [dq, dk]), placed)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    gq, gk = (turned(x, angle, True, 1.25, inverse=True) for x in (q, k))
    q, k = turned(q, angle, True, 1.25), turned(k, angle, True, 1.25)
    assert all(within(a, *w) for a, w in zip(outs[0], (q, k, gq, gk, q)))


@pytest.mark.parametrize("width", [1, 2])
def test_more_rows_than_a_launch(width, no_fallback):
    """2^27 narrow rows are one launch of the forward; those behind it, and at the border, are as in a short call."""
    border, rows, near = 2 ** 27, 2 ** 27 + 21, 6
    g = torch.Generator().manual_seed(13)
    pick = [slice(0, near), slice(border - near, border + near), slice(rows - near, rows)]
    n = 4 * near
    some = {k: torch.randn(n, width, generator=g).bfloat16() for k in ("x", "residual", "gh", "gy")}
    w = (1 + 0.1 * torch.randn(width, generator=g)).bfloat16()
    long = {}
    for k, v in some.items():
        long[k] = torch.zeros(rows, width, dtype=torch.bfloat16, device="supa")
        for at, part in zip(pick, v.to("supa").split([near, 2 * near, near])):
            long[k][at] = part

    def run(t, weight):
        t = {k: v.detach() for k, v in t.items()}
        x, r, weight = t["x"].requires_grad_(), t["residual"].requires_grad_(), weight.detach().requires_grad_()
        h, y = torch.supa.residual_norm(x, r, post_norm="rms", post_weight=weight, norm="rms", eps=1e-3)
        grads = torch.autograd.grad([h, y], [x, r, weight], [t["gh"], t["gy"]])
        return [v.detach() for v in (h, y, *grads)]

    *got, gw = run(long, w.to("supa"))
    *want, ww = run({k: v.to("supa") for k, v in some.items()}, w.to("supa"))
    for a, b in zip(got, want):
        assert torch.equal(torch.cat([a[at].cpu() for at in pick]), b.cpu())
    # the rows between hold zeros and add nothing to the weight's gradient
    x, wd = some["x"].double(), w.double()
    xn = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-3)
    h = (some["residual"].double() + xn * wd).requires_grad_()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-3)
    (dh,) = torch.autograd.grad(y, h, some["gy"].double())
    terms = (dh + some["gh"].double()) * xn
    # float32 on magnitudes: dh is of two terms that may cancel, each at most |gy| / sqrt(eps)
    mag = ((some["gh"].double().abs() + 2 * some["gy"].double().abs().amax(-1, keepdim=True) * 1e-3 ** -0.5) * xn.abs()).sum(0)
    tol = terms.sum(0).abs() * 2.0 ** -8 + K * mag * (1 + 2.0 ** -7)
    for v in (gw, ww):
        assert ((v.double().cpu() - terms.sum(0)).abs() <= tol).all()
