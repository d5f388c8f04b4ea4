"""Performance cases of the operators that stand between a transformer's matrix
products and in its optimizer step: the gated residual with the norms around
it, rotary positions, and the clipping of the global gradient norm.

``run`` computes them in plain torch operations, or (``own``) through the
framework's entry points ``torch.supa.residual_norm``,
``torch.supa.rotary_embedding`` / ``rotary_embedding_`` and
``torch.supa.clip_grad_norm_``.  ``prepare`` draws the inputs with torch's
seeded generator on the GPU; for the framework the same bytes are then copied
into tensors of its device, where its user's program has them.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
#: The limit of a clipped case falls by this factor a pass, so that every pass clips.
DECAY = 0.9999


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decoded sequence: norm after a block, gate, residual, next norm
        dict(name="norm_token", op="residual_norm", batch=1, seq=1, width=4096, x="bf16", residual="bf16",
             params="bf16", gate="channel", post="rms", norm="rms", scale=1.0, train=False),
        # a training batch of 8192 tokens, a learned gate per channel, RMS norms on both sides of the residual
        dict(name="norm_train", op="residual_norm", batch=4, seq=2048, width=4096, x="bf16", residual="bf16",
             params="bf16", gate="channel", post="rms", norm="rms", scale=1.0, train=True),
        # float32 training with LayerNorms and a gate per sample, on a width that is no multiple of anything
        dict(name="norm_ragged", op="residual_norm", batch=6, seq=1001, width=2047, x="f32", residual="f32",
             params="f32", gate="sample", post="layer", norm="layer", scale=0.5, train=True),
        # a wide model's add and norm: bf16 blocks on a float32 residual stream and float32 weights
        dict(name="norm_large", op="residual_norm", batch=8, seq=2048, width=8192, x="bf16", residual="f32",
             params="f32", gate="none", post="none", norm="rms", scale=1.0, train=True),
        # one decoding step of 64 sequences at far positions, in place in the packed projection
        dict(name="rotary_decode", op="rotary", batch=64, seq=1, heads=32, kv_heads=8, dim=128, rotary=128, x="bf16",
             layout="half", memory="packed", scaling="linear", start=250000, train=False),
        # a training batch with grouped heads
        dict(name="rotary_train", op="rotary", batch=4, seq=2048, heads=32, kv_heads=8, dim=128, rotary=128, x="bf16",
             layout="half", memory="bshd", scaling="none", start=0, train=True),
        # part of the head, neighbouring pairs, heads before positions in memory, float32
        dict(name="rotary_ragged", op="rotary", batch=3, seq=1021, heads=12, kv_heads=12, dim=72, rotary=36, x="f32",
             layout="interleaved", memory="bhsd", scaling="none", start=0, train=True),
        # the prompt of a long context, frequencies scaled with the attention's temperature
        dict(name="rotary_prompt", op="rotary", batch=1, seq=131072, heads=16, kv_heads=4, dim=128, rotary=128,
             x="bf16", layout="half", memory="bshd", scaling="yarn", start=0, train=False),
        # 24 small adapter matrices: the launches' latency
        dict(name="clip_adapters", op="clip", kind="adapters", layers=6, width=1024, hidden=16, x="f32", norm=2.0,
             clipped=True),
        # two blocks' bf16 gradients within the limit: the step of a settled training
        dict(name="clip_within", op="clip", kind="blocks", layers=2, width=2048, hidden=5504, x="bf16", norm=2.0,
             clipped=False),
        # bf16 matrices of odd sizes beside float32 vectors
        dict(name="clip_mixed", op="clip", kind="mixed", layers=3, width=1023, hidden=2749, x="bf16", norm=2.0,
             clipped=True),
        # six blocks' float32 gradients, 1.2 GB
        dict(name="clip_large", op="clip", kind="blocks", layers=6, width=2048, hidden=5504, x="f32", norm=2.0,
             clipped=True),
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
    op = rng.choice(["residual_norm", "rotary", "clip"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "residual_norm":
        width = _log(rng, 64, 16384)
        train = rng.random() < 0.6  # training sees batches of tokens, serving single ones too
        rows = _log(rng, 64 if train else 1, min(65536, (1 << 25) // width))
        batch = rng.choice([1, 2, 3, 4, 8]) if rows >= 64 else 1
        return dict(op=op, batch=batch, seq=max(1, rows // batch), width=width, x=x,
                    residual=rng.choice([x, x, "f32"]), params=rng.choice([x, x, "f32"]),
                    gate=rng.choice(["none", "channel", "sample", "full"]),
                    post=rng.choice(["none", "rms", "layer"]), norm=rng.choice(["rms", "rms", "layer", "none"]),
                    scale=rng.choice([1.0, 0.7071]), train=train)
    if op == "rotary":
        dim = rng.choice([64, 72, 80, 96, 128, 128, 192, 256])
        rotary = rng.choice([dim, dim, dim // 2, 2 * rng.randrange(1, dim // 2)])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 7])
        train = rng.random() < 0.5
        # a pass reads or writes an element of q or k at most four times, as often as the largest listed one
        tokens = _log(rng, 64 if train else 1, min(65536, (1 << 26) // (dim * (heads + kv_heads))))
        batch = rng.choice([1, 2, 4]) if tokens >= 64 else tokens
        memory = rng.choice(["bshd", "bhsd"] if train else ["bshd", "bhsd", "packed"])
        return dict(op=op, batch=batch, seq=max(1, tokens // batch), heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=rotary, x=x, layout=rng.choice(["half", "interleaved"]), memory=memory,
                    scaling=rng.choice(["none", "linear"] if memory == "packed" else ["none", "linear", "yarn"]),
                    start=rng.choice([0, 5000, 1000000]), train=train)
    width = _log(rng, 64, 2048)
    kind = rng.choice(["adapters", "blocks", "mixed"])
    return dict(op=op, kind=kind, layers=rng.choice([1, 2, 3, 4, 6]), width=width,
                hidden=_log(rng, 4, 64) if kind == "adapters" else width * 11 // 4, x=rng.choice(["f32", "bf16"]),
                norm=rng.choice([2.0, 2.0, 1.0, math.inf]), clipped=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[dtype])


def _norm_inputs(case, g):
    b, s, d = case["batch"], case["seq"], case["width"]
    p = case["params"]
    # a residual stream has a few channels far larger than the others
    loud = 2 * (1 + 20 * (torch.rand(d, generator=g, device="cuda") < 0.003).float())
    src = dict(x=_randn(g, (b, s, d), case["x"]),
               residual=(torch.randn((b, s, d), generator=g, device="cuda") * loud).to(DTYPES[case["residual"]]))
    if case["gate"] != "none":
        shape = {"channel": (d,), "sample": (b, 1, d), "full": (b, s, d)}[case["gate"]]
        src["gate"] = (0.5 + 0.3 * torch.randn(shape, generator=g, device="cuda")).to(DTYPES[p])
    for kind, w, bias in (("post", "post_weight", "post_bias"), ("norm", "weight", "bias")):
        if case[kind] != "none":
            src[w] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(DTYPES[p])
        if case[kind] == "layer":
            src[bias] = _randn(g, (d,), p, 0.1)
    if case["train"]:
        src["gh"] = _randn(g, (b, s, d), case["residual"])
        if case["norm"] != "none":
            src["gy"] = _randn(g, (b, s, d), case["x"])
    return src


def _frequencies(case):
    """The rotations' angular frequencies (float64) and the factor on the rotated values."""
    r = case["rotary"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    f = 10000.0 ** (-2 * i / r)
    if case["scaling"] == "linear":
        return f / 8, 1.0
    if case["scaling"] == "yarn":  # slow rotations interpolated by 16, fast ones kept, a ramp between
        turns = 8192 * f / (2 * math.pi)
        keep = ((torch.log(turns) - math.log(1.0)) / (math.log(32.0) - math.log(1.0))).clamp(0, 1)
        return f * keep + f / 16 * (1 - keep), 0.1 * math.log(16) + 1
    return f, 1.0


def _rotary_inputs(case, g):
    b, s, hq, hk, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
    f, _ = _frequencies(case)
    src = dict(frequencies=f)
    if case["seq"] == 1:  # every sequence of a decoding step has a length of its own
        src["positions"] = case["start"] + torch.randint(0, 4096, (b, 1), generator=g, device="cuda")
    else:
        src["positions"] = (case["start"] + torch.arange(s, device="cuda")).expand(b, s).contiguous()
    if case["memory"] == "packed":
        src["qkv"] = _randn(g, (b, s, (hq + 2 * hk) * d), case["x"])
        return src
    shape = (lambda h: (b, h, s, d)) if case["memory"] == "bhsd" else (lambda h: (b, s, h, d))
    for name, h in (("q", hq), ("k", hk)) + ((("gq", hq), ("gk", hk)) if case["train"] else ()):
        src[name] = _randn(g, shape(h), case["x"])
    return src


def _clip_shapes(case):
    """(shape, dtype) of each gradient."""
    w, h, x = case["width"], case["hidden"], case["x"]
    if case["kind"] == "adapters":
        return [((h, w), x), ((w, h), x)] * 2 * case["layers"]
    vec = "f32" if case["kind"] == "mixed" else x
    return ([((w, w), x)] * 4 + [((h, w), x)] * 2 + [((w, h), x)] + [((w,), vec)] * 2) * case["layers"]


def _clip_inputs(case, g):
    return {"g%d" % i: _randn(g, s, t, 1e-3) for i, (s, t) in enumerate(_clip_shapes(case))}


def _limit(case):
    """The largest norm allowed: half of what the gradients have, or ten times."""
    n = sum(math.prod(s) for s, _ in _clip_shapes(case))
    norm = 1e-3 * {2.0: math.sqrt(n), 1.0: 0.8 * n, math.inf: math.sqrt(2 * math.log(n))}[case["norm"]]
    return norm * (0.5 if case["clipped"] else 10.0)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"residual_norm": _norm_inputs, "rotary": _rotary_inputs, "clip": _clip_inputs}[case["op"]](case, g)


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
        torch_supa._C.memcpy_d2d(out[k].data_ptr(), v.data_ptr(), v.numel() * v.element_size())
    torch.supa.synchronize()
    return out


NORM_LEAVES = ("x", "residual", "gate", "post_weight", "post_bias", "weight", "bias")


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:  # the same bytes on the framework's device
        d = _to_supa(d)
    op = case["op"]
    if op == "clip":
        grads = [d["g%d" % i] for i in range(len(d))]
        params = [torch.empty_like(g) for g in grads]
        for p, g in zip(params, grads):
            p.grad = g
        return {"case": case, "params": params, "limit": _limit(case)}
    if op == "rotary":
        b, s, hq, hk, n = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
        if case["memory"] == "packed":
            qkv = d.pop("qkv")
            d["q"] = qkv[..., : hq * n].view(b, s, hq, n)
            d["k"] = qkv[..., hq * n: (hq + hk) * n].view(b, s, hk, n)
        elif case["memory"] == "bhsd":
            for k in ("q", "k", "gq", "gk"):
                if k in d:
                    d[k] = d[k].transpose(1, 2)
        d["factor"] = _frequencies(case)[1]
    if own and case["train"]:
        for k in ("q", "k") if op == "rotary" else NORM_LEAVES:
            if k in d:
                d[k] = d[k].requires_grad_()
    return {"case": case, **d}


# --------------------------------------------------------- plain operators
def _stats(v, kind):
    """Mean (0 for rms) and reciprocal deviation of each row."""
    m = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    return m, torch.rsqrt((v - m).square().mean(-1, keepdim=True) + EPS)


def _affine(n, w, b):
    n = n if w is None else n * w
    return n if b is None else n + b


def _norm_backward(g, n, r, w, kind):
    """Gradient of the rows that were normalised to n."""
    a = g if w is None else g * w
    centre = a.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return r * (a - centre - n * (a * n).mean(-1, keepdim=True))


def _plain_norm(state):
    case = state["case"]
    x, res, gate, pw, pb, w, b, gh, gy = (
        None if state.get(k) is None else state[k].float() for k in NORM_LEAVES + ("gh", "gy"))
    post, norm, scale = case["post"], case["norm"], case["scale"]
    u = x
    if post != "none":
        pm, pr = _stats(x, post)
        xn = (x - pm) * pr
        u = _affine(xn, pw, pb)
    h = res * scale + (u if gate is None else u * gate)
    out = {"h": h.to(state["residual"].dtype)}
    if norm != "none":
        m, r = _stats(h, norm)
        n = (h - m) * r
        out["y"] = _affine(n, w, b).to(state["x"].dtype)
    if not case["train"]:
        return out
    param = DTYPES[case["params"]]
    dh = gh
    if norm != "none":
        dh = dh + _norm_backward(gy, n, r, w, norm)
        out["weight"] = (gy * n).sum((0, 1)).to(param)
        if norm == "layer":
            out["bias"] = gy.sum((0, 1)).to(param)
    out["residual"] = (dh * scale).to(state["residual"].dtype)
    du = dh
    if gate is not None:
        out["gate"] = (dh * u).sum_to_size(gate.shape).to(param)
        du = dh * gate
    if post != "none":
        out["post_weight"] = (du * xn).sum((0, 1)).to(param)
        if post == "layer":
            out["post_bias"] = du.sum((0, 1)).to(param)
        du = _norm_backward(du, xn, pr, pw, post)
    out["x"] = du.to(state["x"].dtype)
    return out


def _rotate(x, c, s, case):
    """The rotation of x's pairs by the angles of cosine c and sine s (times the factor)."""
    r = case["rotary"]
    v = x[..., :r].float()
    if case["layout"] == "half":
        a, b = v[..., : r // 2], v[..., r // 2:]
        v = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = v[..., 0::2], v[..., 1::2]
        v = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((v.to(x.dtype), x[..., r:]), -1)


def _plain_rotary(state):
    case = state["case"]
    angle = (state["positions"].double().unsqueeze(-1) * state["frequencies"]).unsqueeze(2)  # far positions: 64 bits
    c, s = ((f(angle) * state["factor"]).float() for f in (torch.cos, torch.sin))
    q, k = (_rotate(state[n], c, s, case) for n in ("q", "k"))
    if case["memory"] == "packed":
        return {"q": state["q"].copy_(q), "k": state["k"].copy_(k)}
    if not case["train"]:
        return {"q": q, "k": k}
    return {"q": q, "k": k, "dq": _rotate(state["gq"], c, -s, case), "dk": _rotate(state["gk"], c, -s, case)}


def _plain_clip(state, limit):
    p = state["case"]["norm"]
    grads = [v.grad for v in state["params"]]
    if p == math.inf:
        norm = torch.stack([g.abs().max().float() for g in grads]).max()
    elif p == 2.0:
        norm = sum(g.float().square().sum(dtype=torch.float64) for g in grads).sqrt().float()
    else:
        norm = sum(g.float().abs().sum(dtype=torch.float64) for g in grads).float()
    c = (limit / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "grads": [g.copy_(g.float() * c) for g in grads]}


# ------------------------------------------------- the framework's entry points
def _own_norm(state):
    case = state["case"]
    kinds = {k: None if case[k] == "none" else case[k] for k in ("post", "norm")}
    h, y = torch.supa.residual_norm(
        state["x"], state["residual"], gate=state.get("gate"), residual_scale=case["scale"], post_norm=kinds["post"],
        post_weight=state.get("post_weight"), post_bias=state.get("post_bias"), norm=kinds["norm"],
        weight=state.get("weight"), bias=state.get("bias"), eps=EPS)
    out = {"h": h.detach()}
    if y is not None:
        out["y"] = y.detach()
    if not case["train"]:
        return out
    leaves = [k for k in NORM_LEAVES if k in state]
    ends = [(h, state["gh"])] if y is None else [(h, state["gh"]), (y, state["gy"])]
    grads = torch.autograd.grad([e[0] for e in ends], [state[k] for k in leaves], [e[1] for e in ends])
    out.update(zip(leaves, grads))
    return out


def _own_rotary(state):
    case = state["case"]
    if case["memory"] == "packed":
        torch.supa.rotary_embedding_(state["q"], state["k"], state["frequencies"], state["positions"],
                                     layout=case["layout"], scale=state["factor"])
        return {"q": state["q"], "k": state["k"]}
    q, k = torch.supa.rotary_embedding(state["q"], state["k"], state["frequencies"], state["positions"],
                                       layout=case["layout"], scale=state["factor"])
    if not case["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad([q, k], [state["q"], state["k"]], [state["gq"], state["gk"]])
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _own_clip(state, limit):
    norm = torch.supa.clip_grad_norm_(state["params"], limit, norm_type=state["case"]["norm"])
    return {"norm": norm, "grads": [v.grad for v in state["params"]]}


def run(state):
    op = state["case"]["op"]
    if op == "clip":
        limit = state["limit"]
        if state["case"]["clipped"]:
            state["limit"] = limit * DECAY
        return _own_clip(state, limit) if own else _plain_clip(state, limit)
    if op == "rotary":
        return _own_rotary(state) if own else _plain_rotary(state)
    return _own_norm(state) if own else _plain_norm(state)


# ------------------------------------------------------------ in 64 bits
def _exact_norm(case, src):
    """From the definition, with the gradients that torch's autograd takes of it in 64 bits."""
    v = {k: t.double() for k, t in src.items()}
    train = case["train"]
    leaves = [k for k in NORM_LEAVES if k in v]
    for k in leaves:
        v[k].requires_grad_(train)

    def normed(t, kind, w, b):
        if kind == "layer":
            t = t - t.mean(-1, keepdim=True)
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * v[w]
        return t + v[b] if kind == "layer" else t

    u = v["x"] if case["post"] == "none" else normed(v["x"], case["post"], "post_weight", "post_bias")
    h = case["scale"] * v["residual"] + u * v.get("gate", 1.0)
    ends, out = [h], {"h": h.detach()}
    if case["norm"] != "none":
        ends.append(normed(h, case["norm"], "weight", "bias"))
        out["y"] = ends[1].detach()
    if train:
        grads = torch.autograd.grad(ends, [v[k] for k in leaves], [v["gh"], v["gy"]][: len(ends)])
        out.update(zip(leaves, grads))
    return out


def _exact_rotary(case, src):
    """Each pair is a complex number, turned by its angle."""
    f, factor = _frequencies(case)
    angle = src["positions"].double()[:, :, None, None] * f
    turn = torch.polar(torch.full_like(angle, factor), angle)

    def turned(x, by):
        x = x.transpose(1, 2) if case["memory"] == "bhsd" else x
        r = case["rotary"]
        pairs = x[..., :r].double()
        pairs = pairs.unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else pairs.unflatten(-1, (r // 2, 2))
        got = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        got = got.transpose(-1, -2) if case["layout"] == "half" else got
        return torch.cat((got.flatten(-2), x[..., r:].double()), -1)

    if case["memory"] == "packed":
        hq, hk, n = case["heads"], case["kv_heads"], case["dim"]
        qkv = src["qkv"].unflatten(-1, (hq + 2 * hk, n))
        return {"q": turned(qkv[:, :, :hq], turn), "k": turned(qkv[:, :, hq: hq + hk], turn)}
    out = {"q": turned(src["q"], turn), "k": turned(src["k"], turn)}
    if case["train"]:
        out |= {"dq": turned(src["gq"], turn.conj()), "dk": turned(src["gk"], turn.conj())}
    return out


def _exact_clip(case, src):
    grads = [src["g%d" % i].double() for i in range(len(src))]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g, case["norm"]) for g in grads]), case["norm"])
    c = min(1.0, _limit(case) / (norm.item() + 1e-6))
    return {"norm": norm, "grads": [g * c for g in grads]}


def exact(case, seed):
    return {"residual_norm": _exact_norm, "rotary": _exact_rotary, "clip": _exact_clip}[case["op"]](
        case, _inputs(case, seed))


# ------------------------------------------------------------ bookkeeping
def work(case):
    """Bytes that one pass cannot do without: each input read once and each
    output written once, for the forward and for the backward."""
    e = SIZE[case["x"]]
    if case["op"] == "residual_norm":
        d = case["width"]
        n = case["batch"] * case["seq"] * d
        r, p = SIZE[case["residual"]], SIZE[case["params"]]
        has_y = case["norm"] != "none"
        gates = {"none": 0, "channel": d, "sample": case["batch"] * d, "full": n}[case["gate"]]
        vectors = sum({"none": 0, "rms": 1, "layer": 2}[case[k]] for k in ("post", "norm")) * d + gates
        nbytes = n * (e + 2 * r + e * has_y) + p * vectors
        if case["train"]:
            # in: gh, gy and what the gradients need of the forward; out: the gradients
            nbytes += n * (r + e * has_y) + n * (e + r) + 2 * p * vectors
            if case["gate"] != "none" or case["post"] != "none":
                nbytes += n * (e + r * has_y)
            elif has_y:
                nbytes += n * r
        return {"bytes": nbytes, "flops": n * (60 if case["train"] else 20)}
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv_heads"])
        moved = n * (case["rotary"] if case["memory"] == "packed" else case["dim"]) * e
        passes = 4 if case["train"] else 2
        return {"bytes": passes * moved + 8 * tokens + 4 * case["rotary"],
                "flops": n * case["rotary"] * 3 * passes // 2 + tokens * case["rotary"] * 20}
    moved = sum(math.prod(s) * SIZE[t] for s, t in _clip_shapes(case))
    n = sum(math.prod(s) for s, _ in _clip_shapes(case))
    # the norm's read, and where it clips the write (the gradients' second read is not counted)
    return {"bytes": moved * (2 if case["clipped"] else 1) + 4, "flops": n * (3 if case["clipped"] else 2)}
