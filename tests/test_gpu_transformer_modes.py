"""The transformer operators under what stands above the device's kernels:
dispatch modes, fake tensors, function transforms and selective checkpointing.
Every result is the plain call's, bit for bit."""
import functools

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

from test_transformer_meta import Calls

pytestmark = pytest.mark.gpu


def rnd(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to("supa")


def inputs(grad=True):
    return [t.requires_grad_(grad) for t in (rnd(5, 7, 260, seed=1), rnd(5, 7, 260, seed=2), rnd(260, seed=3), rnd(260, seed=4))]


def block(x, r, gate, w):
    return torch.supa.residual_norm(x, r, gate=gate, post_norm="rms", post_weight=w, norm="layer", weight=w, bias=gate)


def gradients(leaves, ends):
    return [t.cpu() for t in torch.autograd.grad([e.sum() for e in ends] + [(e * e).sum() for e in ends], leaves)]


def test_dispatch_mode(no_fallback):
    leaves = inputs()
    plain = block(*leaves)
    want = gradients(leaves, plain)
    f, q = torch.ones(8, dtype=torch.float64, device="supa"), rnd(3, 2, 20).requires_grad_()
    with Calls() as calls:
        got = block(*leaves)
        again = gradients(leaves, got)
        o, _ = torch.supa.rotary_embedding(q, None, f)
        torch.autograd.grad(o.sum(), q)
        torch.supa.rotary_embedding_(q.detach().clone(), None, f)
        torch.ops.supa.clip_grad_norm_([o.detach()], 1.0, 2.0, False)
    assert calls.names == ["_residual_norm_forward", "_residual_norm_backward", "rotary_embedding", "rotary_embedding",
                           "rotary_embedding_", "clip_grad_norm_"]
    assert all(torch.equal(a.detach().cpu(), b.detach().cpu()) for a, b in zip(got, plain))
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_fake_tensors_with_gradients(supa):
    with FakeTensorMode():
        x, r = (torch.empty(5, 7, 260, device="supa", requires_grad=True) for _ in range(2))
        gate, w = (torch.empty(260, device="supa", requires_grad=True) for _ in range(2))
        h, y = block(x, r, gate, w)
        grads = torch.autograd.grad([h, y], [x, r, gate, w], [torch.empty_like(h), torch.empty_like(y)])
        assert all(isinstance(t, FakeTensor) and t.device.type == "supa" for t in (h, y, *grads))
        assert [g.shape for g in grads] == [x.shape, r.shape, gate.shape, w.shape]
        q = torch.empty(3, 2, 20, device="supa", requires_grad=True)
        o, _ = torch.supa.rotary_embedding(q, None, torch.empty(8, dtype=torch.float64, device="supa"))
        (g,) = torch.autograd.grad(o, q, torch.empty_like(o))
        assert isinstance(g, FakeTensor) and g.shape == q.shape


def test_function_transforms(no_fallback):
    f, q = torch.tensor([1.0, 0.1, 0.01], dtype=torch.float64, device="supa"), rnd(3, 2, 20, seed=5)

    def loss(v):
        o, _ = torch.supa.rotary_embedding(v, None, f, 4)
        return (o * o * o).sum()

    v = q.clone().requires_grad_()
    (want,) = torch.autograd.grad(loss(v), v)
    assert torch.equal(torch.func.grad(loss)(q).cpu(), want.cpu())
    out, back = torch.func.vjp(lambda v: torch.supa.rotary_embedding(v, None, f, 4)[0], q)
    assert torch.equal(back(torch.ones_like(out))[0].cpu(),
                       torch.autograd.grad(torch.supa.rotary_embedding(v, None, f, 4)[0].sum(), v)[0].cpu())
    # function transforms always ask for gradients of gradients, which residual_norm has not
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.func.grad(lambda x: torch.supa.residual_norm(x, x)[1].sum())(rnd(4, 64))


def test_selective_checkpointing(no_fallback):
    """A policy keeps the operator's outputs by name; the backward does not run it again."""
    leaves = inputs()
    want = gradients(leaves, block(*leaves))

    def policy(ctx, op, *args, **kwargs):
        kept = op is torch.ops.supa._residual_norm_forward.default
        return CheckpointPolicy.MUST_SAVE if kept else CheckpointPolicy.PREFER_RECOMPUTE

    outs = checkpoint(lambda *a: block(*(t * 1 for t in a)), *leaves, use_reentrant=False,
                      context_fn=functools.partial(create_selective_checkpoint_contexts, policy))
    with Calls() as calls:
        got = gradients(leaves, outs)
    assert calls.names == ["_residual_norm_backward"]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_backward_operator_refuses(supa):
    """Called by itself with tensors that do not fit together: an error before any launch."""
    x, w, stats = rnd(4, 8), rnd(8), rnd(4, 4)
    base = dict(grad_h=x, grad_y=x, x=x, residual=x, h=None, stats=stats, gate=None, residual_scale=1.0, post_norm=0,
                post_weight=None, post_bias=None, norm=1, weight=w, bias=None, eps=1e-6, dtype=torch.float32,
                residual_dtype=torch.float32, output_mask=[True] * 7)
    op = torch.ops.supa._residual_norm_backward
    for kw in (dict(grad_h=None, grad_y=None), dict(x=rnd(4, 9)), dict(residual=x.half()), dict(stats=None),
               dict(stats=rnd(3, 4)), dict(x=None), dict(residual=None), dict(x=x.cpu()), dict(weight=w.cpu()),
               dict(gate=rnd(3, 8)), dict(post_norm=2, x=None), dict(h=x, post_norm=1)):
        with pytest.raises(RuntimeError):
            op(**{**base, **kw})
