"""The sines and cosines that torch.supa.rotary_embedding turns by, as its float32
outputs for the pair (1, 0), against float64: relative to their value, also next
to a zero (355 is 113 half turns less 3e-5).

Tolerance, derived: position times frequency and its turns are float64, off by
3 of 2^-53 (the reference's angle by one), 2^-50 of the angle in all.  The angle
left after whole quarter turns is rounded to float32, 2^-24 of it, which moves
its sine and cosine by no more than that of their value.  Sine and cosine of it
are within 4 units in the last place, 8 of 2^-24: 10 of 2^-24 with that
rounding and what is of second order."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_sine_and_cosine(layout, no_fallback):
    f = torch.tensor([1.0, 2.0, 0.75, 1e-2, 1e-4, 3.0], dtype=torch.float64)
    pos = torch.cat((torch.arange(-400, 3000), torch.tensor([710, 103993, 104348, 208341, 312689, 833719, 1146408]),
                     torch.randint(0, 10 ** 6, (2000,), generator=torch.Generator().manual_seed(2))))
    n, pairs = pos.numel(), f.numel()
    x = torch.zeros(n, 1, 2, pairs) if layout == "half" else torch.zeros(n, 1, pairs, 2)
    (x[:, :, 0] if layout == "half" else x[..., 0]).fill_(1.0)
    got, _ = torch.supa.rotary_embedding(x.flatten(-2).to("supa"), None, f.to("supa"), pos.to("supa"), layout=layout)
    got = got.double().cpu().view(x.shape)
    cos, sin = (got[:, 0, 0], got[:, 0, 1]) if layout == "half" else (got[:, 0, :, 0], got[:, 0, :, 1])
    angle = pos.double().unsqueeze(-1) * f
    for a, want in ((cos, angle.cos()), (sin, angle.sin())):
        assert ((a - want).abs() <= 10 * 2.0 ** -24 * want.abs() + 2.0 ** -50 * angle.abs()).all()
