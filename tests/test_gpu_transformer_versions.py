"""What the transformer operators write in place has a new version afterwards,
with gradients enabled, disabled and in inference mode; a backward that saved
the old value raises."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu

MODES = {"grad": contextlib.nullcontext, "no_grad": torch.no_grad, "inference": torch.inference_mode}


@pytest.mark.parametrize("mode", MODES)
def test_rotary_in_place(mode, no_fallback):
    f = torch.ones(4, dtype=torch.float64, device="supa")
    q, k = torch.ones(3, 2, 8, device="supa"), torch.ones(3, 1, 8, device="supa")
    w = torch.ones(8, device="supa", requires_grad=True)
    ends = [w * q, w * k]
    versions = [q._version, k._version]
    with MODES[mode]():
        torch.supa.rotary_embedding_(q, k, f)
    assert [q._version, k._version] == [v + 1 for v in versions]
    for end in ends:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            end.sum().backward()


@pytest.mark.parametrize("mode", MODES)
def test_clipping(mode, no_fallback):
    p, other = torch.ones(5, device="supa"), torch.ones(40, 30, device="supa")
    p.grad, other.grad = torch.full((5,), 2.0, device="supa"), torch.ones(40, 60, device="supa")[:, ::2]
    w = torch.ones((), device="supa", requires_grad=True)
    ends = [w * p.grad, w * other.grad]
    versions = [p.grad._version, other.grad._version]
    with MODES[mode]():
        torch.supa.clip_grad_norm_([p, other], 1.0)
    assert all(t.grad._version > v for t, v in zip((p, other), versions))
    for end in ends:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            end.sum().backward()


def test_inference_tensors(no_fallback):
    """They have no version and are written all the same."""
    f = torch.ones(4, dtype=torch.float64, device="supa")
    with torch.inference_mode():
        q = torch.ones(3, 2, 8, device="supa")
        torch.supa.rotary_embedding_(q, None, f)
        p = torch.ones(5, device="supa")
        p.grad = torch.full((5,), 2.0, device="supa")
        n = torch.supa.clip_grad_norm_(p, 1.0)
    assert q.is_inference() and not torch.equal(q.cpu(), torch.ones(3, 2, 8))
    assert float(n) == pytest.approx(20 ** 0.5) and float(p.grad[0]) == pytest.approx(2 / 20 ** 0.5, rel=1e-5)
