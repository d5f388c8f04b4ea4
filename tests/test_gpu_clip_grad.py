"""torch.supa.clip_grad_norm_ against float64 (CPU): the norm, the scaled
gradients, and what is left alone.

Tolerances, derived: the norm is summed in float64, so its float32 result is
off by its own half step (2^-24) and 1e-12; the factor rounds to float32
(2^-24) and the product to its type (eps / 2), after a float32 product
(2^-24)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def grads_of(spec, seed=0, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g, dtype=torch.float64) * scale).to(t) for s, t in spec]


def as_params(grads):
    ps = []
    for g in grads:
        p = torch.empty_like(g)
        p.grad = g
        ps.append(p)
    return ps


def norm_of(grads, p):
    v = torch.cat([g.double().reshape(-1) for g in grads])
    return float(torch.linalg.vector_norm(v, p)) if v.numel() else 0.0


F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
SPECS = {
    "one": [((1,), F32)],
    "odd": [((1023, 77), F32), ((1,), F32), ((0, 5), F32), ((4097,), F32), ((3, 5, 7), F32)],
    "mixed": [((129, 65), BF16), ((1000,), F32), ((33, 3), F16), ((64, 64), F64), ((0,), BF16), ((2049,), BF16)],
    "many": [((17 + i % 5, 31), F32 if i % 3 else BF16) for i in range(300)],
    "large": [((2048, 2048), F32), ((5504, 1024), BF16)],
    "empty": [((0,), F32), ((3, 0), BF16)],
}


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("spec", SPECS)
def test_clipped_and_not(spec, p, no_fallback):
    host = grads_of(SPECS[spec])
    norm = norm_of(host, p)
    for limit in (0.5 * norm, 10 * norm + 1):
        dev = [g.to("supa") for g in host]
        params = as_params(dev)
        got = torch.supa.clip_grad_norm_(params, limit, norm_type=p)
        wide = any(t == F64 for _, t in SPECS[spec])
        assert got.shape == () and got.dtype == (F64 if wide else F32)
        assert abs(float(got) - norm) <= norm * (2.0 ** -24 + 1e-12)
        c = min(1.0, limit / (norm + 1e-6))
        for a, b, q in zip(dev, host, params):
            assert q.grad is a
            if c == 1.0:
                assert torch.equal(a.cpu(), b)
                continue
            fi = torch.finfo(b.dtype)
            want = b.double() * c
            tol = want.abs() * (fi.eps / 2 + 3 * 2.0 ** -24) + fi.tiny * fi.eps
            assert not ((a.double().cpu() - want).abs() > tol).any()


def test_same_bits_each_time(no_fallback):
    host = grads_of(SPECS["mixed"] + SPECS["large"], 3)
    runs = []
    for _ in range(3):
        dev = [g.to("supa") for g in host]
        n = torch.supa.clip_grad_norm_(as_params(dev), 0.25)
        runs.append([n.cpu()] + [g.cpu() for g in dev])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


def test_float32_range(no_fallback):
    """Squares beyond float32's range, and below it."""
    for v in (1e25, 1e-30):
        dev = [torch.full((1000,), v, device="supa"), torch.full((24,), v, device="supa")]
        n = torch.supa.clip_grad_norm_(as_params(dev), 1.0)
        assert float(n) == pytest.approx(32 * v, rel=1e-6)
        want = min(1.0, 1.0 / (32 * v + 1e-6)) * v
        assert float(dev[0][5]) == pytest.approx(want, rel=1e-6)


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_nan_and_infinite_norms(p, no_fallback):
    host = grads_of([((100,), F32), ((3000,), BF16)], 5)
    host[1][77] = math.inf
    dev = [g.to("supa") for g in host]
    assert math.isinf(float(torch.supa.clip_grad_norm_(as_params(dev), 1.0, norm_type=p)))
    got = dev[1].cpu()
    assert got[77].isnan() and (got[:77] == 0).all() and (dev[0].cpu() == 0).all()
    host[0][3] = math.nan
    dev = [g.to("supa") for g in host]
    assert math.isnan(float(torch.supa.clip_grad_norm_(as_params(dev), 1.0, norm_type=p)))
    assert all(g.cpu().isnan().all() for g in dev)
    dev = [g.to("supa") for g in host]
    with pytest.raises(RuntimeError, match="non-finite"):
        torch.supa.clip_grad_norm_(as_params(dev), 1.0, norm_type=p, error_if_nonfinite=True)
    for a, b in zip(dev, host):  # nothing was scaled
        torch.testing.assert_close(a.cpu(), b, rtol=0, atol=0, equal_nan=True)
    fine = [g.to("supa") for g in grads_of([((100,), F32)], 6)]
    before = fine[0].cpu()
    n = torch.supa.clip_grad_norm_(as_params(fine), 1e-3, error_if_nonfinite=True)
    assert float(n) > 1e-3 and float((fine[0].cpu() / before).mean()) == pytest.approx(1e-3 / float(n), rel=1e-4)


def test_layouts(no_fallback):
    """Permuted, unaligned and strided gradients; neighbours in memory stay."""
    g = torch.Generator().manual_seed(8)
    base = torch.randn(64, 48, generator=g)
    big = torch.randn(9, 1001, generator=g)
    host = [base.t(), big.reshape(-1)[3:4004], torch.randn(40, 40, generator=g)[:, 3:30]]
    dbase, dbig, dslice = base.to("supa"), big.to("supa"), torch.randn(40, 40, generator=torch.Generator().manual_seed(9)).to("supa")
    keep = dslice.cpu()
    host[2] = keep[:, 3:30]
    dev = [dbase.t(), dbig.reshape(-1)[3:4004], dslice[:, 3:30]]
    ps = []
    for d in dev:
        p = torch.empty(d.shape, device="supa")
        p.grad = d
        ps.append(p)
    norm = norm_of(host, 2)
    n = torch.supa.clip_grad_norm_(ps, norm / 2)
    assert float(n) == pytest.approx(norm, rel=1e-6)
    for d, h in zip(dev, host):
        torch.testing.assert_close(d.cpu(), h * 0.5, rtol=4 * 2.0 ** -24 + 1e-6 / norm, atol=0)
    assert torch.equal(dslice.cpu()[:, :3], keep[:, :3]) and torch.equal(dslice.cpu()[:, 30:], keep[:, 30:])
    assert torch.equal(dbig.cpu().reshape(-1)[:3], big.reshape(-1)[:3]) and torch.equal(dbig.cpu().reshape(-1)[4004:], big.reshape(-1)[4004:])


def test_more_than_2_31_elements(no_fallback):
    """The last elements of a long tensor count and are scaled."""
    x = torch.zeros(2 ** 31 + 77, dtype=BF16, device="supa")
    x[-3:] = 4.0
    x[2 ** 31 - 1] = 1.0
    n = torch.supa.clip_grad_norm_(as_params([x]), 3.5)
    assert float(n) == 7.0
    # a factor of 3.5 / 7.000001, off from a half by 2^-22 of it: to the nearest bfloat16, a half
    assert (x[-3:].cpu() == 2.0).all() and float(x[2 ** 31 - 1]) == 0.5 and float(x[2 ** 31]) == 0.0


def test_columns_of_one_buffer(no_fallback):
    """Tensors that reach over each other's memory without sharing any of it; two
    that share some are refused with nothing written."""
    host = torch.randn(40, 30, generator=torch.Generator().manual_seed(4))
    dev = host.to("supa")
    parts = lambda t: [t[:, :7], t[:, 20:], t[:, 7:20]]  # noqa: E731
    norm = norm_of([host], 2)
    assert float(torch.supa.clip_grad_norm_(as_params(parts(dev)), norm / 2)) == pytest.approx(norm, rel=1e-6)
    torch.testing.assert_close(dev.cpu(), host * 0.5, rtol=4 * 2.0 ** -24 + 1e-6 / norm, atol=0)
    line = torch.ones(9, device="supa")
    assert float(torch.supa.clip_grad_norm_(as_params([line[::2], line[1::2]]), 1.0)) == 3.0
    before = dev.cpu()
    for pair in ([dev[:, :8], dev[:, 7:20]], [dev, dev[:, 3:9]], [dev[:, 3:9], dev[3]], [dev[:, 3:9], dev[:, 5:9].t()],
                 [dev[:20, :4], dev[19:, :4]]):
        with pytest.raises(RuntimeError, match="share memory"):
            torch.supa.clip_grad_norm_(as_params(pair), 0.1)
    assert torch.equal(dev.cpu(), before)


def test_argument_forms(no_fallback):
    p = torch.ones(3, device="supa")
    assert float(torch.supa.clip_grad_norm_(p, 1.0)) == 0.0  # no gradient
    assert float(torch.supa.clip_grad_norm_([], 1.0)) == 0.0
    p.grad = torch.full((3,), 2.0, device="supa")
    v = p.grad._version
    assert float(torch.supa.clip_grad_norm_(p, 1)) == pytest.approx(12 ** 0.5)
    assert p.grad._version > v
    assert float(torch.supa.clip_grad_norm_((q for q in [p]), 0.0, norm_type=float("inf"))) == pytest.approx(12 ** -0.5 * 2, rel=1e-5)
    assert (p.grad.cpu() == 0).all()


def test_refusals(supa):
    x = torch.ones(4, 4, device="supa")
    call = torch.ops.supa.clip_grad_norm_
    for grads, args, text in [
        ([x], (-1.0, 2.0, False), "max_norm"), ([x], (math.nan, 2.0, False), "max_norm"), ([x], (1.0, 3.0, False), "norm"),
        ([x, x], (1.0, 2.0, False), "share memory"), ([x[0], x.reshape(-1)[3:]], (1.0, 2.0, False), "share memory"),
        ([x[:, :2], x[:, :2]], (1.0, 2.0, False), "share memory"), ([x, x.cpu()], (1.0, 2.0, False), "supa"), ([x.long()], (1.0, 2.0, False), "floating"),
        ([x[:1].expand(4, 4)], (1.0, 2.0, False), None),
    ]:
        before = x.cpu()
        with pytest.raises((RuntimeError, NotImplementedError), match=text):
            call(grads, *args)
        assert torch.equal(x.cpu(), before)
