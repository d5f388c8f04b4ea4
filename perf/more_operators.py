"""Performance cases of the operators on logits that stand beside the losses and
the softmax: distillation from a teacher's top logits, the balance loss of a
router with the counts of its experts, and the penalties, biases and grammar
masks that a server puts on logits before it draws from them.

``run`` computes them in plain torch operations, or (``own``) through the
framework's entry points ``torch.supa.distillation_loss``,
``torch.supa.router_balance_loss`` and ``torch.supa.adjust_logits``.
``prepare`` draws the inputs with torch's seeded generator on the GPU; for the
framework the same bytes are then copied into tensors of its device, where its
user's program has them.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # the answer of one short sample against a teacher's eight best tokens: latency
        dict(name="distill_sample", op="distill", batch=1, seq=24, vocab=32000, k=8, x="bf16", teacher="bf16",
             rest=False, temperature=1.0, reduction="mean", shifted=False, padded=0.0),
        # a training batch on the language-model loss's vocabulary, the teacher's 64 best tokens stored
        # beside the data; prompts are padded
        dict(name="distill_train", op="distill", batch=4, seq=1024, vocab=128256, k=64, x="bf16", teacher="bf16",
             rest=False, temperature=1.0, reduction="mean", shifted=False, padded=0.1),
        # a softened teacher whose other tokens count as one more class, odd sizes, float32, the last position of
        # each sequence cut off
        dict(name="distill_rest", op="distill", batch=3, seq=500, vocab=50257, k=20, x="f32", teacher="f32",
             rest=True, temperature=2.0, reduction="mean", shifted=True, padded=0.1),
        # a loss per token, weighted by the caller, float16 under a loss scale
        dict(name="distill_tokens", op="distill", batch=1, seq=2047, vocab=64001, k=100, x="f16", teacher="f32",
             rest=True, temperature=1.0, reduction="none", shifted=False, padded=0.0),
        # one sequence's tokens over eight experts
        dict(name="balance_small", op="balance", batch=1, seq=512, experts=8, k=2, x="f32", scores="softmax",
             masked=False, per_sequence=False),
        # a training batch over 64 experts
        dict(name="balance_train", op="balance", batch=8, seq=4096, experts=64, k=6, x="bf16", scores="softmax",
             masked=False, per_sequence=False),
        # sigmoid scores, a loss for each sequence, padded sequences of odd length, experts that fill no vector
        dict(name="balance_sequences", op="balance", batch=12, seq=2047, experts=161, k=6, x="f32", scores="sigmoid",
             masked=True, per_sequence=True),
        # the largest batch over 256 experts
        dict(name="balance_large", op="balance", batch=32, seq=8192, experts=256, k=8, x="f32", scores="softmax",
             masked=True, per_sequence=False),
        # one sequence's next token: penalties for what it has said
        dict(name="adjust_token", op="adjust", rows=1, vocab=32000, length=700, k=0, x="bf16", penalties=True,
             grammar=False),
        # a batch of decoding sequences on the language-model vocabulary, everything at once
        dict(name="adjust_batch", op="adjust", rows=64, vocab=128256, length=4096, k=32, x="bf16", penalties=True,
             grammar=True),
        # float32 logits of odd size under a grammar alone
        dict(name="adjust_grammar", op="adjust", rows=37, vocab=50257, length=0, k=300, x="f32", penalties=False,
             grammar=True),
        # the largest batch, long histories
        dict(name="adjust_large", op="adjust", rows=512, vocab=128256, length=32768, k=16, x="f32", penalties=True,
             grammar=True),
    ]


def _log(rng, lo, hi, odd=0.4):
    """A size from [lo, hi], uniform in its logarithm: of odd value for a
    share `odd` of the draws, else a multiple of 8 (where hi allows)."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < odd:
        n |= 1
    elif n >= 16:
        n -= n % 8
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["distill", "balance", "adjust"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "distill":
        vocab = _log(rng, 256, 262144)
        tokens = _log(rng, 4, max(4, min(65536, (1 << 28) // vocab)))
        batch = rng.choice([1, 2, 3, 4]) if tokens >= 16 else 1
        return dict(op=op, batch=batch, seq=max(2, tokens // batch), vocab=vocab, k=_log(rng, 1, 256), x=x,
                    teacher=rng.choice(["bf16", "f16", "f32"]), rest=rng.random() < 0.5,
                    temperature=rng.choice([1.0, 1.0, 2.0, 0.7]), reduction=rng.choice(["mean", "mean", "sum", "none"]),
                    shifted=rng.random() < 0.3, padded=rng.choice([0.0, 0.1, 0.5]))
    if op == "balance":
        experts = _log(rng, 4, 512)
        tokens = _log(rng, 64, min(262144, (1 << 26) // experts))
        batch = rng.choice([1, 2, 5, 8])
        return dict(op=op, batch=batch, seq=max(1, tokens // batch), experts=experts,
                    k=rng.choice([1, 2, 4, min(8, experts)]), x=x, scores=rng.choice(["softmax", "softmax", "sigmoid"]),
                    masked=rng.random() < 0.5, per_sequence=rng.random() < 0.4)
    vocab = _log(rng, 256, 262144)
    rows = _log(rng, 1, min(512, (1 << 25) // vocab))
    penalties = rng.random() < 0.8
    return dict(op=op, rows=rows, vocab=vocab, length=_log(rng, 1, 32768) if penalties else 0,
                k=rng.choice([0, _log(rng, 1, 300)]), x=x, penalties=penalties,
                grammar=rng.random() < 0.5 or not penalties)


# ------------------------------------------------------------------ inputs
def _distinct(g, rows, k, n):
    """k distinct indexes below n in each of `rows` rows, in no order: steps of random length from a random start."""
    steps = torch.randint(1, n // k + 1, (rows, k), generator=g, device="cuda")
    at = torch.randint(0, n, (rows, 1), generator=g, device="cuda") + steps.cumsum(1)
    return (at % n).gather(1, torch.rand((rows, k), generator=g, device="cuda").argsort(1))


def _distill_inputs(case, g):
    b, s, v, k = case["batch"], case["seq"], case["vocab"], min(case["k"], case["vocab"] // 2)
    n = b * s
    indices = _distinct(g, n, k, v)
    # a teacher's sorted logits: the best stand out, the others lie close together
    gaps = -torch.log1p(-torch.rand((n, k), generator=g, device="cuda")) * 2 / (1 + torch.arange(k, device="cuda"))
    teacher = (20 - gaps.cumsum(1)).to(DTYPES[case["teacher"]])
    # the student has learnt some of it
    logits = torch.randn((n, v), generator=g, device="cuda") * 2
    near = 8 + torch.randn((n, k), generator=g, device="cuda") + 0.5 * (teacher.float() - 20)
    logits = logits.scatter_(1, indices, near).to(DTYPES[case["x"]])
    src = dict(logits=logits.view(b, s, v))
    if case["rest"]:  # what the stored logits leave to the other tokens: 0.1 % to 20 %
        t = teacher.double() / case["temperature"]
        left = torch.rand((n,), generator=g, device="cuda").double() * 0.2 + 0.001
        src["teacher_lse"] = (torch.logsumexp(t, 1) - torch.log1p(-left)).float()
    if k > 4:  # some rows store fewer tokens
        short = torch.rand((n, 1), generator=g, device="cuda") < 0.1
        indices = torch.where(short & (torch.arange(k, device="cuda") >= k - 2), -1, indices)
    if case["padded"]:  # positions without a teacher: the prompt of each sequence
        prompt = (torch.rand((b, 1), generator=g, device="cuda") * 2 * case["padded"] * s).long()
        bare = (torch.arange(s, device="cuda") < prompt).view(n, 1)
        indices = torch.where(bare, -1, indices)
    src["indices"] = indices.view(b, s, k)
    src["teacher"] = teacher.view(b, s, k)
    tokens = b * (s - 1 if case["shifted"] else s)
    scale = 1024.0 if case["x"] == "f16" else 1.0
    if case["reduction"] == "none":
        shape = (b, s - 1 if case["shifted"] else s)
        src["upstream"] = scale / tokens * (0.5 + torch.rand(shape, generator=g, device="cuda"))
    else:
        src["upstream"] = torch.full((), scale / (tokens if case["reduction"] == "sum" else 1), device="cuda")
    return src


def _balance_inputs(case, g):
    b, s, e, k = case["batch"], case["seq"], case["experts"], case["k"]
    liked = torch.randn((e,), generator=g, device="cuda")  # some experts are chosen far more often
    logits = (torch.randn((b, s, e), generator=g, device="cuda") + 0.7 * liked).to(DTYPES[case["x"]])
    src = dict(logits=logits, experts=logits.float().topk(k, -1).indices.contiguous())
    if case["masked"]:
        length = (s * (0.5 + 0.5 * torch.rand((b, 1), generator=g, device="cuda"))).ceil()
        src["mask"] = torch.arange(s, device="cuda") < length
    # the loss's weight in the step; float16 under a loss scale
    src["upstream"] = torch.full((), 1024.0 if case["x"] == "f16" else 0.01, device="cuda")
    return src


def _adjust_inputs(case, g):
    n, v, length, k = case["rows"], case["vocab"], case["length"], min(case["k"], case["vocab"] // 2)
    src = dict(logits=(torch.randn((n, v), generator=g, device="cuda") * 4).to(DTYPES[case["x"]]))
    if case["penalties"]:
        # a text says few tokens often and many once
        src["tokens"] = (v * torch.rand((n, length), generator=g, device="cuda") ** 3).long().clamp_(max=v - 1)
        src["lengths"] = (length * (0.5 + 0.5 * torch.rand((n,), generator=g, device="cuda"))).ceil().long()
        src["prompt_lengths"] = (src["lengths"] * torch.rand((n,), generator=g, device="cuda")).long()
        src["repetition"] = 1 + 0.3 * torch.rand((n,), generator=g, device="cuda")
        src["presence"] = torch.rand((n,), generator=g, device="cuda")
        src["frequency"] = 0.5 * torch.rand((n,), generator=g, device="cuda")
    if k:
        src["bias_tokens"] = _distinct(g, n, k, v)
        src["bias"] = torch.randn((n, k), generator=g, device="cuda") * 5
    if case["grammar"]:  # bits of 32 tokens a word; every third sequence is free
        words = torch.randint(-(1 << 31), 1 << 31, (n, (v + 31) // 32), generator=g, device="cuda")
        src["allowed"] = torch.where(torch.arange(n, device="cuda")[:, None] % 3 == 2, -1, words).int()
    return src


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"distill": _distill_inputs, "balance": _balance_inputs, "adjust": _adjust_inputs}[case["op"]](case, g)


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-supa_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import torch_supa

    return torch_supa


def _to_supa(src):
    torch_supa = _framework()
    torch.cuda.synchronize()
    out = {}
    for k, v in src.items():
        out[k] = torch.empty(v.shape, dtype=v.dtype, device="supa")
        torch_supa._C.memcpy_d2d(out[k].data_ptr(), v.contiguous().data_ptr(), v.numel() * v.element_size())
    torch.supa.synchronize()
    return out


def _cut(case, src):
    """Without the last position of each sequence: views."""
    if not case["shifted"]:
        return src
    out = {k: v[:, :-1] for k, v in src.items() if k in ("logits", "indices", "teacher")}
    if "teacher_lse" in src:
        out["teacher_lse"] = src["teacher_lse"].view(case["batch"], case["seq"])[:, :-1]
    return {**src, **out}


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:  # the same bytes on the framework's device
        d = _to_supa(d)
    if case["op"] == "distill":
        if "teacher_lse" in d:
            d["teacher_lse"] = d["teacher_lse"].view(case["batch"], case["seq"])
        d = _cut(case, d)
    if own and case["op"] != "adjust":
        d["logits"] = d["logits"].detach().requires_grad_()
    return {"case": case, **d}


# --------------------------------------------------------- plain operators
def _plain_distill(state):
    case = state["case"]
    shape = state["logits"].shape
    v, k = shape[-1], state["indices"].shape[-1]
    x = state["logits"].float().reshape(-1, v) / case["temperature"]
    at = state["indices"].reshape(-1, k)
    there = at >= 0
    counted = there.any(1)
    # one less than nothing stored: an entry that is not there stands for the row's first, with no weight
    at = torch.where(there, at, at[:, :1].clamp(min=0))
    # the teacher's few numbers in 64 bits: what they leave to the rest is a difference of near values
    t = torch.where(there, state["teacher"].double().reshape(-1, k) / case["temperature"], -math.inf)
    if case["rest"]:
        lt = state["teacher_lse"].double().reshape(-1, 1)
    else:
        top = t.amax(1, keepdim=True)
        top = torch.where(counted[:, None], top, 0.0)
        lt = top + (t - top).exp().sum(1, keepdim=True).log()
    log_p = torch.where(there, t - lt, 0.0)
    p = torch.where(there, log_p.exp(), 0.0)
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(1, keepdim=True)
    log_q = x.gather(1, at) - m - total.log()
    loss = (p * (log_p - log_q)).sum(1)
    q = e / total
    q_top = q.gather(1, at)
    if case["rest"]:
        r = (1 - p.sum(1, keepdim=True)).clamp(min=0.0)
        left = e.scatter(1, at, 0.0).sum(1, keepdim=True)
        loss = loss + (r * (r.clamp(min=1e-300).log() - (left / total).log()))[:, 0]
        q = q * (1 - r * total / left).float()
    loss = torch.where(counted, loss, 0.0).float()
    g = state["upstream"].reshape(-1, 1) if case["reduction"] == "none" else state["upstream"]
    if case["reduction"] == "mean":
        g = g / counted.sum()
        loss = loss.sum() / counted.sum()
    elif case["reduction"] == "sum":
        loss = loss.sum()
    else:
        loss = loss.view(shape[:-1])
    grad = q.scatter(1, at, q_top).scatter_add(1, at, -p.float())
    grad = torch.where(counted[:, None], grad * (g / case["temperature"]), 0.0)
    return {"loss": loss, "logits": grad.to(state["logits"].dtype).view(shape)}


def _plain_balance(state):
    case = state["case"]
    x = state["logits"].float()
    b, s, e = x.shape
    if not case["per_sequence"]:
        x = x.reshape(1, b * s, e)
    ids = state["experts"].reshape(x.shape[0], -1)
    chosen = torch.ones_like(ids)
    tokens = torch.full((x.shape[0], 1), x.shape[1], device=x.device)
    on = None
    if case["masked"]:
        on = state["mask"].reshape(x.shape[0], -1, 1)
        tokens = on.sum(1)
        chosen = on.expand(-1, -1, case["k"]).reshape(ids.shape).long()
    counts = torch.zeros((x.shape[0], e), dtype=torch.int64, device=x.device).scatter_add_(1, ids, chosen)
    if case["scores"] == "softmax":
        w = (x - x.amax(-1, keepdim=True)).exp()
    else:
        w = 1 / (1 + (-x).exp())
    p = w / w.sum(-1, keepdim=True)
    p_on = p if on is None else p * on
    mean = p_on.sum(1) / tokens
    load = counts.float() * e / (case["k"] * tokens)
    loss = (load * mean).sum(1).mean()
    # the shares of a token's experts sum to one: a constant taken off the loads changes no gradient
    a = (load - 1)[:, None, :]
    d = p_on * (a - (p * a).sum(-1, keepdim=True))
    if case["scores"] == "sigmoid":
        d = d * (1 - w)
    grad = d * (state["upstream"] / (x.shape[0] * tokens))[:, :, None]
    shape = state["logits"].shape
    return {"loss": loss, "counts": counts if case["per_sequence"] else counts[0],
            "logits": grad.to(state["logits"].dtype).view(shape)}


def _allowed(words, vocab):
    bits = (words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return bits.reshape(words.shape[0], -1)[:, :vocab].bool()


def _plain_adjust(state):
    case = state["case"]
    x = state["logits"].float()
    if case["penalties"]:
        at = torch.arange(case["length"], device=x.device)
        said = at < state["lengths"][:, None]
        wrote = said & (at >= state["prompt_lengths"][:, None])
        zero = torch.zeros_like(x, dtype=torch.int32)
        seen = zero.scatter_add(1, state["tokens"], said.int()) > 0
        count = zero.scatter_add(1, state["tokens"], wrote.int()).float()
        rho = state["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rho, x * rho), x)
        x = x - state["frequency"][:, None] * count - state["presence"][:, None] * (count > 0)
    if "bias" in state:
        x = x.scatter_add(1, state["bias_tokens"], state["bias"])
    if case["grammar"]:
        x = torch.where(_allowed(state["allowed"], case["vocab"]), x, -math.inf)
    return x.to(state["logits"].dtype)


# ------------------------------------------------- the framework's entry points
def _own_distill(state):
    case = state["case"]
    loss = torch.supa.distillation_loss(
        state["logits"], state["indices"], state["teacher"], teacher_lse=state.get("teacher_lse"),
        temperature=case["temperature"], reduction=case["reduction"])
    grad, = torch.autograd.grad(loss, state["logits"], state["upstream"])
    return {"loss": loss.detach(), "logits": grad}


def _own_balance(state):
    case = state["case"]
    loss, counts = torch.supa.router_balance_loss(
        state["logits"], state["experts"], mask=state.get("mask"), scores=case["scores"],
        per_sequence=case["per_sequence"])
    grad, = torch.autograd.grad(loss, state["logits"], state["upstream"])
    return {"loss": loss.detach(), "counts": counts, "logits": grad}


def _own_adjust(state):
    penalties = {k: state[k] for k in ("tokens", "lengths", "prompt_lengths", "repetition", "presence", "frequency",
                                       "bias_tokens", "bias", "allowed") if k in state}
    return torch.supa.adjust_logits(state["logits"], **penalties)


def run(state):
    op = state["case"]["op"]
    if op == "distill":
        return _own_distill(state) if own else _plain_distill(state)
    if op == "balance":
        return _own_balance(state) if own else _plain_balance(state)
    return _own_adjust(state) if own else _plain_adjust(state)


# ------------------------------------------------------------ in 64 bits
def _exact_distill(case, src):
    """From the definition, with the gradient that torch's autograd takes of it in 64 bits, some rows at a time."""
    if "teacher_lse" in src:
        src["teacher_lse"] = src["teacher_lse"].view(case["batch"], case["seq"])
    src = _cut(case, src)
    shape = src["logits"].shape
    v, k = shape[-1], src["indices"].shape[-1]
    logits, ids, teacher = src["logits"].reshape(-1, v), src["indices"].reshape(-1, k), src["teacher"].reshape(-1, k)
    n = ids.shape[0]
    counted = (ids >= 0).any(1)
    up = src["upstream"].double()
    if case["reduction"] == "mean":
        up = up / counted.sum()
    up = up.reshape(-1).expand(n)
    losses, grads = [], []
    step = max(1, (1 << 27) // v)
    for i in range(0, n, step):
        x = logits[i: i + step].double().requires_grad_()
        at, on = ids[i: i + step], ids[i: i + step] >= 0
        hot = torch.zeros((at.shape[0], v + 1), dtype=torch.bool, device=x.device)
        hot.scatter_(1, torch.where(on, at, v), True)  # absent entries mark a column that is cut off
        hot = hot[:, :v]
        log_q = torch.log_softmax(x / case["temperature"], 1)
        z = (teacher[i: i + step].double() / case["temperature"]).masked_fill(~on, -math.inf)
        if case["rest"]:
            log_p = z - src["teacher_lse"].reshape(-1, 1)[i: i + step].double()
        else:
            log_p = torch.log_softmax(torch.where(counted[i: i + step, None], z, 0.0), 1)
        log_p = torch.where(on, log_p, 0.0)
        p = torch.where(on, log_p.exp(), 0.0)
        terms = p * (log_p - log_q.gather(1, at.clamp(min=0)))
        rows = torch.where(on, terms, 0.0).sum(1)
        if case["rest"]:
            r = (1 - p.sum(1)).clamp(min=0)
            rest = torch.logsumexp(log_q.masked_fill(hot, -math.inf), 1)
            rows = rows + torch.xlogy(r, r) - r * rest
        rows = torch.where(counted[i: i + step], rows, 0.0)
        grads.append(torch.autograd.grad(rows, x, up[i: i + step])[0])
        losses.append(rows.detach())
    loss = torch.cat(losses)
    loss = loss.view(shape[:-1]) if case["reduction"] == "none" else loss.sum()
    if case["reduction"] == "mean":
        loss = loss / counted.sum()
    return {"loss": loss, "logits": torch.cat(grads).view(shape)}


def _exact_balance(case, src):
    x = src["logits"].double().requires_grad_()
    b, s, e = x.shape
    on = src["mask"].double() if case["masked"] else torch.ones((b, s), dtype=torch.float64, device=x.device)
    p = torch.softmax(x, -1) if case["scores"] == "softmax" else torch.sigmoid(x)
    p = p / p.sum(-1, keepdim=True)
    hot = torch.zeros((b, s, e), dtype=torch.float64, device=x.device).scatter_(-1, src["experts"], 1.0)
    dims = (1,) if case["per_sequence"] else (0, 1)
    tokens = on.sum(dims)
    counts = (hot * on[..., None]).sum(dims)
    shares = (p * on[..., None]).sum(dims) / tokens[..., None]
    loss = (e * counts / (case["k"] * tokens[..., None]) * shares).sum(-1).mean()
    grad, = torch.autograd.grad(loss, x, src["upstream"].double())
    return {"loss": loss.detach(), "counts": None, "logits": grad}


def _exact_adjust(case, src):
    x = src["logits"].double()
    n, v = x.shape
    if case["penalties"]:
        rows = torch.arange(n, device=x.device)[:, None]
        at = torch.arange(case["length"], device=x.device)
        said = at < src["lengths"][:, None]
        wrote = said & (at >= src["prompt_lengths"][:, None])
        flat = rows * v + src["tokens"]
        seen = torch.bincount(flat[said], minlength=n * v).view(n, v) > 0
        count = torch.bincount(flat[wrote], minlength=n * v).view(n, v).double()
        rho = src["repetition"].double()[:, None].expand(n, v)
        x = torch.where(seen & (x > 0), x / rho, torch.where(seen, x * rho, x))
        x = x - count * src["frequency"].double()[:, None] - count.clamp(max=1) * src["presence"].double()[:, None]
    if "bias" in src:
        x = x + torch.zeros_like(x).scatter_add_(1, src["bias_tokens"], src["bias"].double())
    if case["grammar"]:
        x = x.masked_fill(~_allowed(src["allowed"], v), -math.inf)
    return x


def exact(case, seed):
    return {"distill": _exact_distill, "balance": _exact_balance, "adjust": _exact_adjust}[case["op"]](
        case, _inputs(case, seed))


# ------------------------------------------------------------ bookkeeping
def work(case):
    """Bytes that one pass cannot do without: each input read once and each
    output written once, for the forward and for the backward."""
    e = SIZE[case["x"]]
    if case["op"] == "distill":
        n = case["batch"] * (case["seq"] - 1 if case["shifted"] else case["seq"])
        n, k = round(n * (1 - case["padded"])), min(case["k"], case["vocab"] // 2)
        moved = n * case["vocab"] * e
        # the logits for the loss, again for the gradient, and the gradient, which has rows of zeros too
        zeros = (case["batch"] * (case["seq"] - case["shifted"]) - n) * case["vocab"] * e
        return {"bytes": 3 * moved + zeros + n * (k * (8 + SIZE[case["teacher"]]) + 8),
                "flops": n * case["vocab"] * 10}
    if case["op"] == "balance":
        n = case["batch"] * case["seq"]
        return {"bytes": n * (3 * case["experts"] * e + 8 * case["k"] + 2 * case["masked"]),
                "flops": n * case["experts"] * 20}
    n, v = case["rows"], case["vocab"]
    k = min(case["k"], v // 2)
    nbytes = n * (2 * v * e + 12 * k + (v + 31) // 32 * 4 * case["grammar"])
    if case["penalties"]:
        nbytes += n * (8 * case["length"] * 3 // 4 + 28)  # a history's mean length
    return {"bytes": nbytes, "flops": n * v * 6 + n * case["length"]}
