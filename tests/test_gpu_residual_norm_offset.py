"""torch.supa.residual_norm with layer norm on rows whose mean is large against
their deviation, in 16 bits: the rounding of h to its type moves the normalised
value by |mean| / deviation half steps there, so the gradients have to come from
h before its rounding, as y does.

Against the definition in float64, with the tolerances of
test_gpu_residual_norm.py for float32 arithmetic and one rounding of each
result, and nothing for a rounding of h."""
import pytest
import torch

from test_gpu_residual_norm import T, check, definition, magnitudes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("params", [True, False], ids=["weights", "no weights"])
@pytest.mark.parametrize("width", [520, 2047, 8200])
@pytest.mark.parametrize("t, mean, deviation", [("bf16", 8.0, 0.25), ("f16", 64.0, 0.25)])
def test_offset_rows(t, mean, deviation, width, params, no_fallback):
    g = torch.Generator().manual_seed(31)
    shape = (3, 11, width)
    rnd = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    d = {"x": (deviation * rnd(*shape)).to(T[t]), "residual": (mean + deviation * rnd(*shape)).to(T[t])}
    if params:
        d["weight"], d["bias"] = (1 + 0.1 * rnd(width)).to(T[t]), (0.1 * rnd(width)).to(T[t])
    eps = 1e-6
    ref = {k: v.double().requires_grad_() for k, v in d.items()}
    h, y = definition(ref, 1.0, None, "layer", eps)
    # a gradient that follows y, so that the mean of its product with the normalised value counts
    gh, gy = (0.1 * rnd(*shape)).to(T[t]), (y.detach() + 0.5 * rnd(*shape)).to(T[t])
    want = dict(zip(ref, torch.autograd.grad([h, y], list(ref.values()), [gh.double(), gy.double()])))
    dev = {k: v.to("supa").requires_grad_() for k, v in d.items()}
    oh, oy = torch.supa.residual_norm(dev["x"], dev["residual"], norm="layer", weight=dev.get("weight"),
                                      bias=dev.get("bias"), eps=eps)
    got = torch.autograd.grad([oh, oy], list(dev.values()), [gh.to("supa"), gy.to("supa")])
    m, _ = magnitudes(d, gh, gy, 1.0, None, "layer", eps, 0.0)
    check("h", oh.detach(), h.detach(), m, {})
    check("y", oy.detach(), y.detach(), m, {})
    for k, v in zip(dev, got):
        check(k, v, want[k], m, {})
