"""The operators on logits under what stands above and beside the device's
kernels: dispatch modes, fake tensors, function transforms, selective
checkpointing, other streams, two threads at once.  Every result is the plain
call's, bit for bit."""
import functools
import threading

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

from test_transformer_meta import Calls

pytestmark = pytest.mark.gpu


def inputs(seed=0, rows=9, vocab=3001, k=7, experts=20):
    g = torch.Generator().manual_seed(seed)
    d = {"x": torch.randn(rows, vocab, generator=g), "i": torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)]),
         "t": torch.randn(rows, k, generator=g), "r": torch.randn(rows, experts, generator=g)}
    d["lse"] = torch.logsumexp(d["t"], 1) + 0.3
    d["e"] = d["r"].topk(3).indices
    d["h"] = torch.randint(0, vocab, (rows, 50), generator=g)
    d = {n: v.to("supa") for n, v in d.items()}
    d["x"].requires_grad_()
    d["r"].requires_grad_()
    return d


def losses(d, x=None, r=None):
    a = torch.supa.distillation_loss(d["x"] if x is None else x, d["i"], d["t"], teacher_lse=d["lse"], temperature=1.3)
    b, counts = torch.supa.router_balance_loss(d["r"] if r is None else r, d["e"])
    return a, b, counts


def everything(d):
    a, b, counts = losses(d)
    gx, gr = torch.autograd.grad([a, b], [d["x"], d["r"]])
    y = torch.supa.adjust_logits(d["x"].detach(), tokens=d["h"], repetition=1.2, frequency=0.1)
    return [a.detach(), b.detach(), counts, gx, gr, y]


def same(a, b):
    return all(torch.equal(u.cpu(), v.cpu()) for u, v in zip(a, b, strict=True))


def test_dispatch_mode(no_fallback):
    d = inputs()
    want = everything(d)
    with Calls() as calls:
        got = everything(d)
        torch.supa.adjust_logits_(got[-1].clone())
    assert calls.names == ["_distillation_loss_forward", "_router_balance_loss_forward", "_router_balance_loss_backward",
                           "_distillation_loss_backward", "adjust_logits", "adjust_logits_"] or sorted(calls.names) == sorted(
        ["_distillation_loss_forward", "_router_balance_loss_forward", "_router_balance_loss_backward",
         "_distillation_loss_backward", "adjust_logits", "adjust_logits_"])
    assert same(got, want)


def test_fake_tensors_with_gradients(supa):
    with FakeTensorMode():
        x, r = torch.empty(4, 50, device="supa", requires_grad=True), torch.empty(4, 6, device="supa", requires_grad=True)
        i, t, e = (torch.empty(4, 3, dtype=k, device="supa") for k in (torch.int64, torch.float32, torch.int32))
        for reduction, shape in (("mean", ()), ("none", (4,))):
            loss = torch.supa.distillation_loss(x, i, t, reduction=reduction)
            (g,) = torch.autograd.grad(loss, x, torch.empty_like(loss))
            assert isinstance(g, FakeTensor) and g.shape == x.shape and loss.shape == shape and g.device.type == "supa"
        loss, counts = torch.supa.router_balance_loss(r, e)
        (g,) = torch.autograd.grad(loss, r)
        assert isinstance(g, FakeTensor) and g.shape == r.shape and counts.shape == (6,)
        assert torch.supa.adjust_logits(x.detach(), tokens=i).shape == x.shape


def test_function_transforms_are_refused(no_fallback):
    d = inputs()
    with pytest.raises(RuntimeError, match="create_graph"):  # they always ask for gradients of gradients
        torch.func.grad(lambda x: losses(d, x=x)[0])(d["x"].detach())
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: losses(d, x=x)[0], (d["x"].detach(),), (torch.ones_like(d["x"]),))


def test_selective_checkpointing(no_fallback):
    """A policy keeps the operator's outputs by name; the backward does not run it again."""
    d = inputs()
    want = torch.autograd.grad(losses(d)[0], d["x"])

    def policy(ctx, op, *args, **kwargs):
        kept = op is torch.ops.supa._distillation_loss_forward.default
        return CheckpointPolicy.MUST_SAVE if kept else CheckpointPolicy.PREFER_RECOMPUTE

    out = checkpoint(lambda x: losses(d, x=x * 1)[0], d["x"], use_reentrant=False,
                     context_fn=functools.partial(create_selective_checkpoint_contexts, policy))
    with Calls() as calls:
        got = torch.autograd.grad(out, d["x"])
    assert "_distillation_loss_forward" not in calls.names and "_distillation_loss_backward" in calls.names
    assert same(got, want)


def test_inference_mode(no_fallback):
    d = inputs()
    want = [t.detach() for t in losses(d)]
    with torch.inference_mode():
        assert same(losses(d), want)


def test_another_stream(no_fallback):
    """The calls run on the current stream, after the work that made their inputs there."""
    d = inputs()
    want = everything(d)
    s = torch.supa.Stream()
    for _ in range(3):
        s.wait_stream(torch.supa.current_stream())
        with torch.supa.stream(s):
            fresh = {n: v.detach().clone() for n, v in d.items()}
            fresh["x"].requires_grad_()
            fresh["r"].requires_grad_()
            got = everything(fresh)
        s.synchronize()
        assert same(got, want)


def test_two_threads_at_once(no_fallback):
    """Each on a stream of its own, with other inputs; nothing is shared between the calls."""
    ds = [inputs(1), inputs(2, rows=700, vocab=5000)]
    wants = [everything(d) for d in ds]
    torch.supa.synchronize()
    ok = [0, 0]

    def work(n):
        s = torch.supa.Stream()
        with torch.supa.stream(s):
            for _ in range(20):
                got = everything(ds[n])
                s.synchronize()
                ok[n] += same(got, wants[n])

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert ok == [20, 20]


def test_index_errors_are_reported_per_stream(supa):
    d = inputs()
    a, b = torch.supa.Stream(), torch.supa.Stream()
    bad = d["i"].clone()
    bad[0, 0] = 3001
    torch.supa.synchronize()
    with torch.no_grad():
        with torch.supa.stream(a):
            torch.supa.distillation_loss(d["x"], bad, d["t"])
        with torch.supa.stream(b):
            torch.supa.distillation_loss(d["x"], d["i"], d["t"]).item()  # another stream's error is not this one's
        with torch.supa.stream(a), pytest.raises(IndexError):
            torch.supa.distillation_loss(d["x"], d["i"], d["t"]).item()
    torch.supa.synchronize()


def test_backward_operators_refuse(supa):
    """Called by themselves with tensors that do not fit together: an error before any launch."""
    d = inputs()
    with torch.no_grad():
        loss, count, stats, pairs = torch.ops.supa._distillation_loss_forward(d["x"], d["i"], d["t"], None, 1.0, 1)
        base = dict(grad_loss=loss, logits=d["x"], count=count, stats=stats, pairs=pairs, temperature=1.0, reduction=1)
        op = torch.ops.supa._distillation_loss_backward
        op(**base)
        for kw in (dict(grad_loss=loss.half()), dict(grad_loss=d["t"]), dict(count=None), dict(stats=stats[:4]),
                   dict(pairs=pairs[:4]), dict(pairs=pairs.float()), dict(pairs=pairs[..., 0]), dict(reduction=0),
                   dict(reduction=5), dict(temperature=0.0), dict(stats=stats.cpu()), dict(logits=d["x"].long())):
            with pytest.raises(RuntimeError):
                op(**{**base, **kw})
        loss, counts, load, scale = torch.ops.supa._router_balance_loss_forward(d["r"], d["e"], None, 0, False)
        base = dict(grad_loss=loss, logits=d["r"], mask=None, load=load, scale=scale, k=3, scores=0, per_sequence=False)
        op = torch.ops.supa._router_balance_loss_backward
        op(**base)
        for kw in (dict(load=load[:5]), dict(scale=scale[:1]), dict(k=0), dict(k=21), dict(scores=2), dict(grad_loss=load),
                   dict(load=load.cpu()), dict(per_sequence=True, logits=d["r"][0]), dict(mask=load)):
            with pytest.raises(RuntimeError):
                op(**{**base, **kw})
