"""The transformer operators on tensors without memory: meta tensors and fake
supa tensors give the results' shapes, types and strides, with gradients, and
refuse what the device refuses; dispatch modes see every call, forward and
backward.  No GPU."""
import math
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

pytest.importorskip("torch_supa")

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64


class Calls(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "supa":
            self.names.append(func._opname)
        return func(*args, **(kwargs or {}))


def meta(*shape, dtype=F32, grad=False):
    return torch.empty(shape, dtype=dtype, device="meta", requires_grad=grad)


@pytest.mark.parametrize("x, residual, params", [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32)])
@pytest.mark.parametrize("gate", [None, (64,), (3, 1, 64), (3, 5, 64)], ids=str)
@pytest.mark.parametrize("norm", ["rms", "layer", None])
def test_residual_norm(x, residual, params, gate, norm):
    a, r = meta(3, 5, 64, dtype=x, grad=True), meta(3, 64, 5, dtype=residual).transpose(1, 2).requires_grad_()
    kw = {"post_norm": norm, "norm": norm}
    if gate:
        kw["gate"] = meta(*gate, dtype=params, grad=True)
    if norm:
        kw |= {n: meta(64, dtype=params, grad=True) for n in ("post_weight", "weight")}
    if norm == "layer":
        kw |= {n: meta(64, dtype=params, grad=True) for n in ("post_bias", "bias")}
    with Calls() as calls:
        h, y = torch.supa.residual_norm(a, r, **kw)
        assert h.shape == (3, 5, 64) and h.dtype == residual and h.is_contiguous() and h.device.type == "meta"
        assert (y is None) == (norm is None) and (y is None or (y.shape == (3, 5, 64) and y.dtype == x))
        leaves = [a, r] + [v for v in kw.values() if isinstance(v, torch.Tensor)]
        ends = [h] if y is None else [h, y]
        grads = torch.autograd.grad(ends, leaves, [torch.empty_like(t) for t in ends])
    assert [(g.shape, g.dtype) for g in grads] == [(v.shape, v.dtype) for v in leaves]
    assert calls.names == ["_residual_norm_forward", "_residual_norm_backward"]
    with Calls() as calls, torch.no_grad():
        torch.supa.residual_norm(a, r, **kw)
    assert calls.names == ["residual_norm"]


def test_rotary_embedding():
    f = meta(4, dtype=F64)
    q, k = meta(2, 3, 7, 12, dtype=BF16, grad=True), meta(2, 7, 3, 12, dtype=BF16).transpose(1, 2)[:, :, :1].requires_grad_()
    with Calls() as calls:
        oq, ok = torch.supa.rotary_embedding(q, k, f)
        assert oq.shape == q.shape and oq.stride() == q.stride() and ok.shape == k.shape and ok.stride(-1) == 1
        dq, dk = torch.autograd.grad([oq, ok], [q, k], [torch.empty_like(oq), torch.empty_like(ok)])
        assert dq.shape == q.shape and dk.shape == k.shape and dq.dtype == BF16
        p, none = torch.supa.rotary_embedding_(meta(3, 2, 8), None, f)
    assert calls.names == ["rotary_embedding", "rotary_embedding", "rotary_embedding_"]
    assert none is None and p.shape == (3, 2, 8)
    window = meta(20).as_strided((5, 1, 16), (1, 16, 1))  # the output's dims keep their order
    assert torch.supa.rotary_embedding(window, None, f)[0].is_contiguous()
    # function transforms reach the operator
    loss = lambda v: torch.supa.rotary_embedding(v, None, f)[0].sum()  # noqa: E731
    assert torch.func.grad(loss)(meta(3, 2, 8)).shape == (3, 2, 8)


def test_clip_grad_norm():
    with Calls() as calls:
        for types, want in (((F32, BF16), F32), ((F32, F64), F64)):
            n = torch.ops.supa.clip_grad_norm_([meta(3, 4, dtype=t) for t in types], 1.0, 2.0, False)
            assert n.shape == () and n.dtype == want and n.device.type == "meta"
    assert calls.names == ["clip_grad_norm_"] * 2


def test_fake_supa_tensors():
    """Nothing is launched and nothing allocated on the device."""
    with FakeTensorMode():
        x = torch.empty(4, 6, 8, dtype=BF16, device="supa:0")
        key, f = torch.empty(4, 1, 8, dtype=BF16, device="supa:0"), torch.empty(4, dtype=F64, device="supa:0")
        h, y = torch.supa.residual_norm(x, x, norm="layer", post_norm="rms")
        q, k = torch.supa.rotary_embedding(x, key, f)
        for t, shape in ((h, x.shape), (y, x.shape), (q, x.shape), (k, (4, 1, 8))):
            assert isinstance(t, FakeTensor) and t.shape == shape and t.device == torch.device("supa:0") and t.dtype == BF16
        assert torch.supa.rotary_embedding_(x, None, f)[0] is x
        n = torch.ops.supa.clip_grad_norm_([x, h], 1.0, math.inf, True)
        assert isinstance(n, FakeTensor) and n.shape == () and n.device == torch.device("supa:0")


def test_refusals():
    x, w = meta(4, 8), meta(8)
    for call, text in [
        (lambda: torch.supa.residual_norm(x, meta(4, 9)), "shape"),
        (lambda: torch.supa.residual_norm(x, x, weight=w.half()), "weight of x's dtype"),
        (lambda: torch.supa.residual_norm(x, x, gate=meta(3, 8)), "gate"),
        (lambda: torch.supa.rotary_embedding(x, None, w), "shape"),
        (lambda: torch.supa.rotary_embedding(meta(2, 4, 8), None, w), "rotate"),
        (lambda: torch.ops.supa.clip_grad_norm_([x], -1.0, 2.0, False), "max_norm"),
        (lambda: torch.ops.supa.clip_grad_norm_([x.long()], 1.0, 2.0, False), "floating"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_backward_arguments():
    """The gradients' own operator refuses tensors that do not fit together."""
    op = torch.ops.supa._residual_norm_backward
    g, x, w, stats = meta(4, 8), meta(4, 8), meta(8), meta(4, 4)
    base = dict(grad_h=g, grad_y=g, x=x, residual=x, h=None, stats=stats, gate=None, residual_scale=1.0, post_norm=0,
                post_weight=None, post_bias=None, norm=1, weight=w, bias=None, eps=1e-6, dtype=F32, residual_dtype=F32,
                output_mask=[True] * 7)
    out = op(**base)
    assert [None if t is None else tuple(t.shape) for t in out] == [(4, 8), (4, 8), None, None, None, (8,), None]
    for kw, text in [
        (dict(grad_h=None, grad_y=None), "expected a gradient"), (dict(grad_y=meta(4, 9)), "grad_y"),
        (dict(x=meta(4, 9)), "expected x"), (dict(residual=x.half()), "expected residual"), (dict(h=meta(3, 8)), "expected h"),
        (dict(stats=meta(4, 3)), "stats"), (dict(stats=stats.half()), "stats"), (dict(weight=meta(9)), "weight"),
        (dict(bias=w), "bias"), (dict(norm=3), "norm"), (dict(gate=meta(3, 8)), "gate"), (dict(dtype=F64), "float32, bfloat16"),
        (dict(dtype=BF16, residual_dtype=F16), "residual of x's dtype"), (dict(weight=torch.empty(8)), "weight is on"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            op(**{**base, **kw})


def test_numbers_that_require_a_gradient():
    """A learned scale would lose its gradient with its conversion to a number."""
    x, f, p = meta(4, 8, grad=True), meta(4, dtype=F64), torch.nn.Parameter(torch.tensor(0.5))
    calls = [lambda s: torch.supa.residual_norm(x, x, residual_scale=s), lambda s: torch.supa.residual_norm(x, x, eps=s),
             lambda s: torch.supa.rotary_embedding(meta(4, 1, 8, grad=True), None, f, scale=s)]
    for call in calls:
        with pytest.raises(TypeError, match="has no gradient"):
            call(p)
        assert call(p.detach())[0].requires_grad and call(0.5)[0].requires_grad
        with torch.no_grad(), warnings.catch_warnings():
            warnings.simplefilter("ignore")  # torch's own, of the conversion
            call(p)
