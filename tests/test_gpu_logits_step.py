"""The operators on logits together, as a program uses them: training steps of
a small mixture of experts against a teacher's stored logits (distillation beside
cross-entropy, the balance loss, clipping, fused AdamW) with their gradients against
the same model in float64; and decoding with penalties, biases and a grammar.

The products between run wherever the device has them (this backend hands
matmul to the CPU)."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

B, S, W, EXPERTS, K, VOCAB, TOP = 2, 16, 24, 6, 2, 97, 8


def parameters(seed):
    g = torch.Generator().manual_seed(seed)
    shapes = {"embed": (VOCAB, W), "router": (W, EXPERTS), "up": (EXPERTS, W, 2 * W), "down": (EXPERTS, 2 * W, W), "out": (W, VOCAB)}
    return {k: torch.randn(s, generator=g, dtype=torch.float64) * 0.3 for k, s in shapes.items()}


def plain_distillation(x, i, t, lse, tau):
    log_q = torch.log_softmax(x.reshape(-1, VOCAB) / tau, 1)
    i, t = i.reshape(-1, TOP), t.double().reshape(-1, TOP) / tau
    counted = (i >= 0).all(1)
    p = (t - lse.double().reshape(-1, 1)).exp()
    listed = torch.zeros_like(log_q, dtype=torch.bool).scatter(1, i.clamp(min=0), True)
    r = (1 - p.sum(1)).clamp(min=0)
    rest = torch.logsumexp(log_q.masked_fill(listed, -math.inf), 1)
    rows = (p * (p.log() - log_q.gather(1, i.clamp(min=0)))).sum(1) + torch.xlogy(r, r) - r * rest
    return rows[counted].mean()


def plain_balance(r, e, mask):
    p = torch.softmax(r, -1)[mask]
    counts = torch.bincount(e[mask].flatten(), minlength=EXPERTS)
    n = int(mask.sum())
    return (EXPERTS * counts / (K * n) * p.mean(0)).sum(), counts


def model(p, tokens, experts=None):
    """Student's logits, the router's and its choices (given, or its own)."""
    x = F.one_hot(tokens, VOCAB).to(p["embed"].dtype).to(p["embed"].device) @ p["embed"]
    r = x @ p["router"]
    if experts is None:
        experts = r.detach().cpu().topk(K, -1).indices
    gate = torch.softmax(r, -1) * F.one_hot(experts, EXPERTS).sum(-2).to(r.dtype).to(r.device)
    y = x
    for n in range(EXPERTS):
        y = y + gate[..., n: n + 1] * (F.silu(x @ p["up"][n]) @ p["down"][n])
    return y @ p["out"], r, experts


def test_training_steps(supa):
    """Gradients of each of three steps against float64 at the same parameters.  float32 throughout, some 40 operations
    deep, each off by at most 128 of 2^-24 of its magnitude: 3e-4 of a gradient's norm."""
    torch.supa.set_cpu_fallback_enabled(True)
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, VOCAB, (B, S), generator=g)
    teacher = torch.randn(B, S, VOCAB, generator=g) * 2
    tau = 1.5
    t, i = teacher.topk(TOP, -1)
    lse = torch.logsumexp(teacher / tau, -1)
    i[:, :3] = -1  # the prompt has no teacher
    mask = torch.ones(B, S, dtype=torch.bool)
    mask[1, 12:] = False  # padding
    targets = torch.roll(tokens, -1, 1)
    targets[~mask] = -100
    leaves = {k: v.float().to("supa").requires_grad_() for k, v in parameters(1).items()}
    opt = torch.optim.AdamW(list(leaves.values()), lr=1e-2, fused=True)
    dev = {k: v.to("supa") for k, v in dict(i=i, t=t, lse=lse, mask=mask, targets=targets.reshape(-1)).items()}
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        logits, r, experts = model(leaves, tokens)
        kd = torch.supa.distillation_loss(logits, dev["i"], dev["t"], teacher_lse=dev["lse"], temperature=tau)
        balance, counts = torch.supa.router_balance_loss(r, experts.to("supa"), mask=dev["mask"])
        (kd * tau ** 2 + 0.5 * F.cross_entropy(logits.reshape(-1, VOCAB), dev["targets"]) + 0.1 * balance).backward()
        ref = {k: v.detach().double().cpu().requires_grad_() for k, v in leaves.items()}
        x64, r64, _ = model(ref, tokens, experts)
        kd64 = plain_distillation(x64, i, t, lse, tau)
        balance64, counts64 = plain_balance(r64, experts, mask)
        (kd64 * tau ** 2 + 0.5 * F.cross_entropy(x64.reshape(-1, VOCAB), targets.reshape(-1)) + 0.1 * balance64).backward()
        assert torch.equal(counts.cpu(), counts64)
        assert abs(float(kd.detach()) - float(kd64.detach())) <= 3e-4 and abs(float(balance.detach()) - float(balance64.detach())) <= 3e-4
        norm = math.sqrt(sum(float((v.grad ** 2).sum()) for v in ref.values()))
        for k, v in leaves.items():
            assert float((v.grad.double().cpu() - ref[k].grad).norm()) <= 3e-4 * norm, k
        torch.supa.clip_grad_norm_(leaves.values(), norm)
        before = leaves["router"].detach().cpu()
        opt.step()
        assert not torch.equal(before, leaves["router"].detach().cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decoding(dtype, no_fallback):
    """Greedy decoding of a batch, token by token, in place, against the same rules in float64 on the same logits.  The
    logits are whole multiples of 1/4 and the penalties powers of two, so that nothing rounds and ties go to the lowest token."""
    g = torch.Generator().manual_seed(9)
    rows, vocab, steps, prompt = 5, 1000, 12, 7
    lengths = torch.full((rows,), prompt)
    history = torch.randint(0, vocab, (rows, prompt + steps), generator=g)
    prompts = lengths.clone()
    said = history.clone()
    bias_tokens, bias = torch.randint(0, vocab, (rows, 6), generator=g), torch.tensor([2.0, -1.0, 4.0, 0.5, -math.inf, 1.0]).expand(rows, 6).contiguous()
    dev = {k: v.to("supa") for k, v in dict(prompt_lengths=prompts, bias_tokens=bias_tokens, bias=bias).items()}
    for step in range(steps):
        logits = (torch.randn(rows, vocab, generator=g) * 8).round() / 4
        words = torch.randint(-(1 << 31), 1 << 31, (rows, (vocab + 31) // 32), generator=g).int()
        x = logits.to(dtype).to("supa")
        torch.supa.adjust_logits_(x, tokens=said.to("supa"), lengths=lengths.to("supa"), repetition=2.0, presence=0.5,
                                  frequency=0.25, allowed=words.to("supa"), **dev)
        probs = F.softmax(x, -1)
        picked = x.argmax(-1).cpu()
        want = logits.double()
        for r in range(rows):
            seen = torch.bincount(said[r, : lengths[r]], minlength=vocab) > 0
            count = torch.bincount(said[r, prompt: lengths[r]], minlength=vocab).double()
            v = torch.where(seen, torch.where(want[r] > 0, want[r] / 2, want[r] * 2), want[r]) - 0.25 * count - 0.5 * (count > 0)
            v = v.scatter_add(0, bias_tokens[r], bias[r].double())
            bits = (words[r].long()[:, None] >> torch.arange(32) & 1).bool().flatten()[:vocab]
            v[~bits] = -math.inf
            assert torch.equal(x[r].cpu().double(), v)
            best = int((v == v.max()).nonzero()[0])
            assert int(picked[r]) == best
            assert float(probs[r, best].float().cpu()) > 0 and not probs[r].cpu()[~bits].any()
            said[r, lengths[r]] = best
        lengths += 1
