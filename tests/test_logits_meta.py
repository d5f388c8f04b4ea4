"""The operators on logits on tensors without memory: shapes, types, gradients
and the calls that dispatch modes see.  No GPU."""
import pytest
import torch

pytest.importorskip("torch_supa")

from test_transformer_meta import Calls, meta  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LONG, INT = torch.int64, torch.int32


@pytest.mark.parametrize("dtype, teacher, index", [(F32, F32, LONG), (BF16, F16, INT), (F16, F32, LONG)])
@pytest.mark.parametrize("shape", [(9,), (3, 9), (2, 5, 9), (0, 9)], ids=str)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("rest", [False, True])
def test_distillation_loss(dtype, teacher, index, shape, reduction, rest):
    x = meta(*shape, dtype=dtype, grad=True)
    i, t = meta(*shape[:-1], 4, dtype=index), meta(*shape[:-1], 4, dtype=teacher)
    kw = {"reduction": reduction, "temperature": 2.0}
    if rest:
        kw["teacher_lse"] = meta(*shape[:-1])
    with Calls() as calls:
        loss = torch.supa.distillation_loss(x, i, t, **kw)
        assert loss.dtype == F32 and loss.shape == (shape[:-1] if reduction == "none" else ())
        (g,) = torch.autograd.grad(loss, x, torch.empty_like(loss))
    assert g.shape == x.shape and g.dtype == dtype and g.is_contiguous()
    assert calls.names == ["_distillation_loss_forward", "_distillation_loss_backward"]
    with Calls() as calls, torch.no_grad():
        assert not torch.supa.distillation_loss(x, i, t, **kw).requires_grad
    assert calls.names == ["distillation_loss"]


def test_no_gradient_of_the_gradient():
    x = meta(3, 9, grad=True)
    loss = torch.supa.distillation_loss(x, meta(3, 4, dtype=LONG), meta(3, 4))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(loss, x, create_graph=True)
    loss, _ = torch.supa.router_balance_loss(x, meta(3, 4, dtype=LONG))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(loss, x, create_graph=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("per_sequence, shape, counts", [(False, (7, 6), (6,)), (False, (6,), (6,)), (False, (2, 7, 6), (6,)),
                                                        (True, (2, 7, 6), (2, 6)), (True, (7, 6), (6,)),
                                                        (True, (3, 2, 7, 6), (3, 2, 6)), (True, (0, 7, 6), (0, 6))])
def test_router_balance_loss(dtype, per_sequence, shape, counts):
    x = meta(*shape, dtype=dtype, grad=True)
    e, m = meta(*shape[:-1], 2, dtype=LONG), meta(*shape[:-1], dtype=torch.bool)
    with Calls() as calls:
        loss, c = torch.supa.router_balance_loss(x, e, mask=m, scores="sigmoid", per_sequence=per_sequence)
        assert loss.shape == () and loss.dtype == F32 and c.shape == counts and c.dtype == LONG and not c.requires_grad
        (g,) = torch.autograd.grad(loss, x)
    assert g.shape == x.shape and g.dtype == dtype
    assert calls.names == ["_router_balance_loss_forward", "_router_balance_loss_backward"]
    with Calls() as calls, torch.no_grad():
        torch.supa.router_balance_loss(x, e)
    assert calls.names == ["router_balance_loss"]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_adjust_logits(dtype):
    x = meta(3, 70, dtype=dtype)
    kw = dict(tokens=meta(3, 5, dtype=INT), lengths=meta(3, dtype=LONG), prompt_lengths=meta(3, dtype=INT),
              repetition=meta(3), presence=0.5, frequency=meta(3), bias_tokens=meta(4, dtype=LONG), bias=meta(3, 4),
              allowed=meta(3, dtype=INT))
    with Calls() as calls:
        out = torch.supa.adjust_logits(x, **kw)
        assert out.shape == x.shape and out.dtype == dtype and out is not x
        assert torch.supa.adjust_logits_(x, **kw) is x
    assert calls.names == ["adjust_logits", "adjust_logits_"]
    assert torch.supa.adjust_logits(meta(70, 3).t()).is_contiguous()
    assert torch.supa.adjust_logits(meta(9), tokens=meta(5, dtype=LONG), lengths=meta(dtype=LONG)).shape == (9,)
    with torch.no_grad():  # a leaf under no_grad has no gradient to lose
        torch.supa.adjust_logits(meta(2, 9, grad=True))
