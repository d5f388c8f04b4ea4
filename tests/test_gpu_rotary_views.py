"""torch.supa.rotary_embedding on views whose strides do not tell their order of
dims: windows that slide over each other.  The outputs and
the gradients are those of the same values in contiguous tensors, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# shape and strides of [seq, heads, dim] or [batch, seq, heads, dim]: a dim before the head's has stride 1
WINDOWS = [
    ((5, 1, 16), (1, 16, 1)),
    ((1, 4, 2, 8), (64, 1, 16, 1)),
    ((6, 3, 8), (2, 1, 1)),
    ((6, 9, 8), (1, 1, 1)),
    ((2, 6, 9, 8), (1, 0, 1, 1)),
    ((3, 70, 5, 24), (500, 1, 60, 1)),
    ((2, 33, 4, 64), (1, 2, 3, 1)),
]


def window(shape, strides, dtype, seed):
    n = 1 + sum((a - 1) * b for a, b in zip(shape, strides)) + 3
    base = torch.randn(n, generator=torch.Generator().manual_seed(seed)).to(dtype).to("supa")
    return base.as_strided(shape, strides, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape, strides", WINDOWS, ids=str)
def test_windows(shape, strides, layout, dtype, no_fallback):
    f = torch.tensor([1.0, 0.3, 0.01], dtype=torch.float64, device="supa")

    def run(form):
        q, k, gq, gk = (form(window(shape, strides, dtype, seed)) for seed in range(4))
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        oq, ok = torch.supa.rotary_embedding(q, k, f, 11, layout=layout, scale=1.25)
        assert oq.stride(-1) == 1 and ok.stride(-1) == 1
        dq, dk = torch.autograd.grad([oq, ok], [q, k], [gq, gk])
        return [t.detach().cpu() for t in (oq, ok, dq, dk)]

    want = run(lambda t: t.contiguous())
    assert not any(t.isnan().any() for t in want)
    for a, b in zip(run(lambda t: t), want):
        assert torch.equal(a, b)


def test_windows_of_a_signal(no_fallback):
    """Every 16 neighbours of a signal, beside heads of their own memory."""
    f = torch.tensor([0.5] * 8, dtype=torch.float64, device="supa")
    signal = torch.randn(20, generator=torch.Generator().manual_seed(1)).to("supa")
    q, k = signal.as_strided((5, 1, 16), (1, 16, 1)), torch.ones(5, 2, 16, device="supa")
    got = torch.supa.rotary_embedding(q, k, f)
    want = torch.supa.rotary_embedding(q.contiguous(), k, f)
    assert got[0].shape == (5, 1, 16)
    assert torch.equal(got[0].cpu(), want[0].cpu()) and torch.equal(got[1].cpu(), want[1].cpu())
