"""The operators on logits under torch.vmap (a loop over the samples) on tensors without memory: shapes, gradients, and
what is refused.  No GPU."""
import pytest
import torch

pytest.importorskip("torch_supa")

from test_transformer_meta import meta  # noqa: E402

pytestmark = pytest.mark.filterwarnings("ignore:There is a performance drop")
LONG = torch.int64


def test_shapes_and_gradients():
    x, i, t, e = meta(4, 3, 9, grad=True), meta(4, 3, 2, dtype=LONG), meta(4, 3, 2), meta(4, 3, 2, dtype=LONG)
    loss = torch.vmap(lambda *a: torch.supa.distillation_loss(*a))(x, i, t)
    assert loss.shape == (4,) and torch.autograd.grad(loss.sum(), x)[0].shape == x.shape
    assert torch.vmap(lambda a: torch.supa.distillation_loss(a, i[0], t[0], reduction="none"))(x).shape == (4, 3)
    loss, counts = torch.vmap(lambda *a: torch.supa.router_balance_loss(*a))(x, e)
    assert loss.shape == (4,) and counts.shape == (4, 9) and torch.autograd.grad(loss.sum(), x)[0].shape == x.shape
    out = torch.vmap(lambda a, h, n: torch.supa.adjust_logits(a, tokens=h, lengths=n, repetition=1.5))(
        x.detach()[:, 0], i[:, 0], meta(4, dtype=LONG))
    assert out.shape == (4, 9)


def test_in_place_is_refused():
    with pytest.raises(RuntimeError, match="Batching rule not implemented"):
        torch.vmap(lambda a: torch.supa.adjust_logits_(a))(meta(4, 3, 9))


def test_no_samples_are_refused():
    with pytest.raises(RuntimeError, match="size 0"):
        torch.vmap(lambda *a: torch.supa.distillation_loss(*a))(meta(0, 3, 9), meta(0, 3, 2, dtype=LONG), meta(0, 3, 2))
