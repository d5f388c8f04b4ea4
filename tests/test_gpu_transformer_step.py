"""The transformer operators together, as a program uses them: training steps
of a small model (norms around gated residuals, rotary positions, a loss,
clipping, fused AdamW) with their gradients against the same model in float64,
and decoding token by token against the whole prompt.

The products between run wherever the device has them (this backend hands
matmul to the CPU)."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

B, S, W, HEADS, KV, DIM, VOCAB = 2, 12, 48, 4, 2, 12, 61


def parameters(seed):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s, scale=0.2, shift=0.0):
        return torch.randn(s, generator=g, dtype=torch.float64) * scale + shift

    return {"embed": rnd(VOCAB, W), "wq": rnd(W, HEADS * DIM), "wk": rnd(W, KV * DIM), "wv": rnd(W, KV * DIM),
            "wo": rnd(HEADS * DIM, W), "up": rnd(W, 2 * W), "down": rnd(2 * W, W), "out": rnd(W, VOCAB),
            "n0": rnd(W, shift=1.0), "p1": rnd(W, shift=1.0), "n1": rnd(W, shift=1.0), "g1": rnd(W, shift=0.5),
            "p2": rnd(W, shift=1.0), "pb2": rnd(W), "n2": rnd(W, shift=1.0), "b2": rnd(W), "g2": rnd(B, 1, W, shift=0.5)}


def plain_norm(v, kind, w, b=None):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w
    return v if b is None else v + b


def plain_residual_norm(x, r, gate, scale, post, pw, pb, norm, w, b):
    h = scale * r + gate * plain_norm(x, post, pw, pb)
    return h, plain_norm(h, norm, w, b)


def own_residual_norm(x, r, gate, scale, post, pw, pb, norm, w, b):
    return torch.supa.residual_norm(x, r, gate=gate, residual_scale=scale, post_norm=post, post_weight=pw, post_bias=pb,
                                    norm=norm, weight=w, bias=b)


def plain_rotary(x, f, scale):
    a = (torch.arange(x.shape[1], dtype=torch.float64)[:, None] * f)[:, None]
    c, s = a.cos() * scale, a.sin() * scale
    n = f.numel()
    u, v = x[..., :n], x[..., n: 2 * n]
    return torch.cat((u * c - v * s, v * c + u * s, x[..., 2 * n:]), -1)


def model(p, x0, f, scale, own):
    """Logits [B, S, VOCAB] of embedded tokens x0 [B, S, W]."""
    rn = own_residual_norm if own else plain_residual_norm
    zero = torch.zeros_like(x0)
    one = torch.ones(W, dtype=x0.dtype).to(x0.device)
    h, y = rn(zero, x0, one * 0, 1.0, "rms", one, None, "rms", p["n0"], None)
    q = (y @ p["wq"]).view(B, S, HEADS, DIM)
    k = (y @ p["wk"]).view(B, S, KV, DIM)
    v = (y @ p["wv"]).view(B, S, KV, DIM)
    if own:
        q, k = torch.supa.rotary_embedding(q, k, f, 0, scale=scale)
    else:
        q, k = plain_rotary(q, f, scale), plain_rotary(k, f, scale)
    outs = []
    mask = torch.full((S, S), -math.inf, dtype=x0.dtype).triu(1).to(x0.device)
    for i in range(HEADS):
        j = i * KV // HEADS
        scores = torch.matmul(q[:, :, i].contiguous(), k[:, :, j].transpose(1, 2).contiguous()) * (DIM ** -0.5) + mask
        outs.append(torch.matmul(F.softmax(scores, -1), v[:, :, j].contiguous()))
    x = torch.cat(outs, -1) @ p["wo"]
    h, y = rn(x, h, p["g1"], 1.0, "rms", p["p1"], None, "rms", p["n1"], None)
    x = F.silu(y @ p["up"]) @ p["down"]
    h, y = rn(x, h, p["g2"], 0.5, "layer", p["p2"], p["pb2"], "layer", p["n2"], p["b2"])
    return y @ p["out"]


def loss_of(p, tokens, f, scale, own):
    x0 = F.one_hot(tokens, VOCAB).to(p["embed"].dtype).to(p["embed"].device) @ p["embed"]
    logits = model(p, x0, f, scale, own)
    t = torch.roll(tokens, -1, 1).reshape(-1).to(p["embed"].device)
    return F.cross_entropy(logits.reshape(-1, VOCAB), t)


def test_training_steps(supa):
    """Gradients of each of three steps against float64 at the same
    parameters.  float32 throughout, some 40 operations deep, each off by at
    most 128 of 2^-24 of its magnitude: 3e-4 of a gradient's norm."""
    torch.supa.set_cpu_fallback_enabled(True)
    tokens = torch.randint(0, VOCAB, (B, S), generator=torch.Generator().manual_seed(3))
    freq, scale = torch.supa.rotary_frequencies(8, scaling="yarn", factor=2.0, original_length=32)
    leaves = {k: v.float().to("supa").requires_grad_() for k, v in parameters(1).items()}
    opt = torch.optim.AdamW(list(leaves.values()), lr=1e-2, fused=True)
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        loss_of(leaves, tokens, freq, scale, True).backward()
        ref = {k: v.detach().double().cpu().requires_grad_() for k, v in leaves.items()}
        loss_of(ref, tokens, freq.cpu(), scale, False).backward()
        norm = math.sqrt(sum(float((v.grad ** 2).sum()) for v in ref.values()))
        total = torch.supa.clip_grad_norm_(leaves.values(), norm / 3)
        assert abs(float(total) - norm) <= 3e-4 * norm
        for k, v in leaves.items():
            want = ref[k].grad / 3
            assert float((v.grad.double().cpu() - want).norm()) <= 3e-4 * float(want.norm()) + 1e-6 * norm, k
        before = leaves["wq"].detach().cpu()
        opt.step()
        assert not torch.equal(before, leaves["wq"].detach().cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_by_token(dtype, no_fallback):
    """A row's result does not depend on the rows beside it: single tokens
    give the prompt's bits, at their position, in place in a packed projection."""
    g = torch.Generator().manual_seed(9)
    width, hq, hk, dim = 4 * 128 + 5, 6, 2, 64
    x, r = (torch.randn(3, 7, width, generator=g).to(dtype).to("supa") for _ in range(2))
    w, gate = (torch.randn(width, generator=g).to(dtype).to("supa") for _ in range(2))
    qkv = torch.randn(3, 7, (hq + 2 * hk) * dim, generator=g).to(dtype).to("supa")
    f, _ = torch.supa.rotary_frequencies(48)

    def views(t):
        n = t.shape[1]
        return t[..., : hq * dim].view(-1, n, hq, dim), t[..., hq * dim: (hq + hk) * dim].view(-1, n, hk, dim)

    h, y = torch.supa.residual_norm(x, r, gate=gate, post_norm="rms", post_weight=w, weight=w)
    q, k = torch.supa.rotary_embedding(*views(qkv), f, 500)
    for t in range(7):
        ht, yt = torch.supa.residual_norm(x[:, t: t + 1], r[:, t: t + 1], gate=gate, post_norm="rms", post_weight=w,
                                          weight=w)
        assert torch.equal(ht.cpu(), h[:, t: t + 1].cpu()) and torch.equal(yt.cpu(), y[:, t: t + 1].cpu())
        step = qkv[:, t: t + 1].contiguous()
        at = torch.full((3, 1), 500 + t).to("supa")
        qt, kt = torch.supa.rotary_embedding_(*views(step), f, at)
        assert torch.equal(qt.cpu(), q[:, t: t + 1].cpu()) and torch.equal(kt.cpu(), k[:, t: t + 1].cpu())
