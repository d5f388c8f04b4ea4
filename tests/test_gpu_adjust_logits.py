"""torch.supa.adjust_logits and adjust_logits_ against their definition in float64 (CPU).

Tolerances, derived (u = 2^-24): the repetition's quotient or product, the product of
frequency and count, two differences, the biases' sums (each addition) and their addition are
one rounding each, relative to what they form; so under 8 u plus one u per further bias of a token of the sum of
magnitudes, then the one rounding to the logits' type.  What no penalty, bias or mask
touches is returned bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def make(rows, vocab, length=0, m=0, grammar=False, x="f32", seed=0):
    g = torch.Generator().manual_seed(seed)
    d = {"logits": (torch.randn(rows, vocab, generator=g) * 4).to(T[x])}
    if length:
        d["tokens"] = (vocab * torch.rand(rows, length, generator=g) ** 2).long().clamp(max=vocab - 1)
        d["lengths"] = torch.randint(0, length + 1, (rows,), generator=g)
        d["prompt_lengths"] = torch.randint(0, length + 1, (rows,), generator=g)
        d["repetition"] = 0.8 + torch.rand(rows, generator=g)
        d["presence"] = torch.randn(rows, generator=g)
        d["frequency"] = torch.rand(rows, generator=g)
    if m:
        d["bias_tokens"] = torch.randint(0, vocab, (rows, m), generator=g)
        d["bias"] = torch.randn(rows, m, generator=g) * 5
    if grammar:
        d["allowed"] = torch.randint(-(1 << 31), 1 << 31, (rows, (vocab + 31) // 32), generator=g).int()
    return d


def definition(d):
    """float64 values, their tolerance before the last rounding, and where nothing applies."""
    x = d["logits"].double()
    rows, vocab = x.shape
    plain = torch.ones(rows, vocab, dtype=torch.bool)
    off = torch.zeros_like(x)

    def per_row(name, default):
        v = d.get(name, default)
        return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), float(torch.tensor(v)), dtype=torch.float64)

    if "tokens" in d:
        n = d["tokens"].shape[1]
        lengths = d.get("lengths", torch.full((rows,), n)).clamp(0, n)
        prompts = d.get("prompt_lengths", torch.zeros(rows, dtype=torch.int64))
        seen, count = torch.zeros(rows, vocab, dtype=torch.bool), torch.zeros(rows, vocab, dtype=torch.float64)
        for r in range(rows):
            t = d["tokens"][r, : lengths[r]].long()
            ok = (t >= 0) & (t < vocab)
            seen[r, t[ok]] = True
            wrote = ok & (torch.arange(len(t)) >= prompts[r])
            count[r] = torch.bincount(t[wrote], minlength=vocab)
        rho = per_row("repetition", 1.0)
        x = torch.where(seen, torch.where(x > 0, x / rho, x * rho), x)
        f, p = per_row("frequency", 0.0), per_row("presence", 0.0)
        off = off + torch.where(seen, 6 * U * (x.abs() + (f * count).abs() + p.abs()), 0.0)
        x = x - torch.where(count > 0, f * count + p, 0.0)
        plain &= ~seen
    if "bias" in d:
        bt, b = (v.expand(rows, -1) if v.dim() == 1 else v for v in (d["bias_tokens"], d["bias"]))
        bt = torch.where((bt >= 0) & (bt < vocab), bt.long(), vocab)
        add, size, times = (torch.zeros(rows, vocab + 1, dtype=torch.float64) for _ in range(3))
        add = add.scatter_add(1, bt, b.double())[:, :vocab]
        size = size.scatter_add(1, bt, b.double().abs())[:, :vocab]
        times = times.scatter_add(1, bt, torch.ones_like(b, dtype=torch.float64))[:, :vocab]
        off = off + torch.where(times > 0, (2 + times) * U * (x.abs() + size), 0.0)
        x = x + add
        plain &= times == 0
    if "allowed" in d:
        w = d["allowed"].expand(rows, -1) if d["allowed"].dim() == 1 else d["allowed"]
        bits = ((w.long()[:, :, None] >> torch.arange(32)) & 1).bool().reshape(rows, -1)[:, :vocab]
        x = torch.where(bits, x, -math.inf)
        off = torch.where(bits, off, 0.0)
    return x, off, plain


def to_supa(d):
    return {k: v.to("supa") if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def check(d):
    want, off, plain = definition(d)
    s = to_supa(d)
    x = s.pop("logits")
    kept = x.clone()
    out = torch.supa.adjust_logits(x, **s)
    assert torch.equal(x.cpu(), kept.cpu())
    assert torch.supa.adjust_logits_(x, **s) is x
    got, t = out.cpu(), d["logits"].dtype
    assert torch.equal(x.cpu(), got) and got.dtype == t
    fi = torch.finfo(t)
    finite = want.isfinite()
    assert torch.equal(got.double()[~finite], want[~finite])
    tol = (want.abs() + off) * fi.eps / 2 + fi.tiny * fi.eps + off
    err = (got.double() - want).abs()
    assert (err[finite] <= tol[finite]).all(), float((err[finite] / tol[finite]).max())
    same = plain & finite
    assert torch.equal(got[same], d["logits"][same])
    return got


SIZES = [
    # rows, vocab, length, m
    (1, 1, 1, 1), (1, 7, 3, 2), (3, 31, 40, 5), (2, 32, 100, 3), (5, 33, 1, 1), (4, 1000, 257, 30), (7, 1024, 1024, 300),
    (3, 4097, 5000, 1), (2, 8192, 700, 64), (2, 8193, 700, 64), (3, 16385, 64, 300), (1, 32000, 700, 10), (2, 50257, 3000, 300),
    (1, 128256, 20000, 1030), (70, 300, 33, 7),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("x", T)
def test_everything(size, x, no_fallback):
    check(make(*size, True, x, seed=sum(size)))


@pytest.mark.parametrize("x", T)
@pytest.mark.parametrize("rows, vocab", [(1, 5000), (33, 2001), (600, 800)], ids=str)
def test_each_alone(x, rows, vocab, no_fallback):
    check(make(rows, vocab, 100, 0, False, x))
    check(make(rows, vocab, 0, 9, False, x))
    check(make(rows, vocab, 0, 0, True, x))
    check(make(rows, vocab, 0, 9, True, x))
    check(make(rows, vocab, 100, 0, True, x))
    check(make(rows, vocab, 100, 9, False, x))
    check({"logits": make(rows, vocab, x=x)["logits"]})  # nothing: a copy


def test_numbers_and_defaults(no_fallback):
    d = make(4, 900, 60)
    tokens = {k: d[k] for k in ("logits", "tokens")}
    check(tokens | {"repetition": 1.3})
    check(tokens | {"presence": 0.7, "frequency": 0.2})
    check(tokens | {"frequency": -0.3, "lengths": d["lengths"].int()})
    check(tokens | {"repetition": d["repetition"], "prompt_lengths": d["prompt_lengths"].int(), "presence": 1.5})
    check(tokens)
    check(tokens | {"tokens": d["tokens"].int(), "repetition": 1.1})
    check(tokens | {"lengths": torch.tensor([0, 1000, -5, 60]), "prompt_lengths": torch.tensor([3, 2000, -4, 60]), "repetition": 2.0, "presence": 1.0})


@pytest.mark.parametrize("rows, vocab, length", [(3, 20011, 0), (2, 20011, 300), (2, 9000, 70000), (300, 2500, 40)], ids=str)
def test_a_bias_of_every_token(rows, vocab, length, no_fallback):
    """More biases than the hash table takes, each token once, in any order, or again and again."""
    d = make(rows, vocab, length, vocab, False, "bf16", 17)
    g = torch.Generator().manual_seed(1)
    d["bias_tokens"][0] = torch.randperm(vocab, generator=g)
    d["bias_tokens"][1, ::2] = d["bias_tokens"][1, 1::2][: (vocab + 1) // 2].repeat(2)[: (vocab + 1) // 2]
    got = check(d)
    s = to_supa(d)
    x = s.pop("logits")
    for _ in range(3):
        assert torch.equal(torch.supa.adjust_logits(x, **s).cpu(), got)
    d["bias_tokens"][-1] = vocab - 1
    check(d | {"bias_tokens": d["bias_tokens"].int()})


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_histories_end_anywhere(index, shift, no_fallback):
    """Every length about whole loads and whole rounds of them, rows at any alignment, tokens behind a row's length
    that would count."""
    near = [0, 1, 2, 3, 4, 5, 7, 8, 9, 255, 256, 257, 259, 511, 513, 1023, 1025, 2047, 2049, 4095, 4097, 4103]
    rows, vocab = len(near), 777
    d = make(rows, vocab, 4103 + shift, 0, False, seed=shift)
    d["lengths"] = torch.tensor(near)
    d["tokens"] = d["tokens"].to(index)
    if index == torch.int64:  # their lower halves are tokens
        d["tokens"][:, ::5] += 2 ** 32
        d["tokens"][:, 1::7] -= 2 ** 32
    check(d)
    d["prompt_lengths"] = (torch.tensor(near) - 2).clamp(min=0)
    d["tokens"] = torch.full_like(d["tokens"], 776)
    check(d)
    s = to_supa(d)
    x, history = s.pop("logits"), s.pop("tokens")
    wide = torch.full((rows, history.shape[1] + 3), 5, dtype=index, device="supa")
    wide[:, shift : shift + history.shape[1]] = history
    assert torch.equal(torch.supa.adjust_logits(x, tokens=wide[:, shift : shift + history.shape[1]], **s).cpu(), check(d))


def test_tokens_outside_are_passed_over(no_fallback):
    d = make(5, 200, 50, 20, False)
    d["tokens"][:, ::3] = -1
    d["tokens"][:, 1::7] = 200
    d["tokens"][2, 5] = 2 ** 40
    d["tokens"][3, 6] = -(2 ** 40)
    d["bias_tokens"][:, ::2] = -1
    d["bias_tokens"][1, 3], d["bias_tokens"][1, 5] = 200, 2 ** 33
    check(d)


def test_the_same_token_again(no_fallback):
    """A history of one token, and many biases of one: sums in the entries' order."""
    d = make(6, 3000, 2000, 500, False)
    d["tokens"][0] = 17
    d["tokens"][1] = 2999
    d["bias_tokens"][0] = 17
    d["bias_tokens"][1, 100:] = 5
    d["bias_tokens"][2, 1::2] = d["bias_tokens"][2, ::2]
    got = check(d)
    s = to_supa(d)
    x = s.pop("logits")
    for _ in range(3):
        assert torch.equal(torch.supa.adjust_logits(x, **s).cpu(), got)
    many = make(2, 100, 0, 3000, False)  # more entries than threads
    check(many)
    many["bias"][0, 5], many["bias"][1, 7] = math.inf, -math.inf
    check(many)


def test_biases_that_look_like_numbers_of_entries(no_fallback):
    d = make(1, 64, 0, 40, False)
    d["bias_tokens"] = (torch.arange(40) % 20)[None]
    d["bias"] = torch.arange(1, 41, dtype=torch.int32).view(torch.float32)[None].clone()
    d["logits"].zero_()
    got = check(d)
    assert torch.equal(got[0, :20].view(torch.int32), torch.tensor([(i + 1) + (i + 21) for i in range(20)], dtype=torch.int32))


def test_rows_shared(no_fallback):
    d = make(5, 700, 0, 11, True)
    d["bias_tokens"], d["bias"], d["allowed"] = d["bias_tokens"][0], d["bias"][0], d["allowed"][0]
    check(d)
    d["bias"] = make(5, 700, 0, 11)["bias"]
    check(d)


def test_one_row_without_a_batch(no_fallback):
    d = make(1, 1500, 90, 8, True, "bf16")
    want = check(d)[0]
    s = {k: (v[0] if v.dim() == 2 else v.reshape(())) for k, v in to_supa(d).items()}
    x = s.pop("logits")
    assert torch.equal(torch.supa.adjust_logits(x, **s).cpu(), want)
    assert torch.equal(torch.supa.adjust_logits_(x, **s).cpu(), want)


def test_nothing_allowed_and_special_values(no_fallback):
    d = make(4, 333, 40, 6, True)
    d["allowed"][1] = 0
    d["allowed"][2] = -1
    x = d["logits"]
    x[:, ::5] = -math.inf
    x[3, 1::5] = torch.finfo(torch.float32).min / 2
    got = check(d)
    assert (got[1] == -math.inf).all()
    x[0, 7] = math.nan
    x[0, 9] = math.inf
    d["allowed"][0] = -1
    d["bias_tokens"][0], d["tokens"][0] = 100, 11
    s = to_supa(d)
    got = torch.supa.adjust_logits(s.pop("logits"), **s).cpu()
    assert got[0, 7].isnan() and got[0, 9] == math.inf and got[0, 10] == -math.inf
    d["allowed"][0] = 0  # a NaN that is not allowed is not there
    s = to_supa(d)
    assert (torch.supa.adjust_logits(s.pop("logits"), **s).cpu()[0] == -math.inf).all()


def test_bits_past_the_vocabulary(no_fallback):
    d = make(3, 70, 0, 0, True)
    more = torch.cat([d["allowed"], torch.full((3, 4), -1, dtype=torch.int32)], 1)
    check(d | {"allowed": more})
    check(d | {"allowed": torch.cat([torch.full((3, 2), -1, dtype=torch.int32), d["allowed"]], 1)[:, 2:]})


@pytest.mark.parametrize("x", T)
def test_views(x, no_fallback):
    """Rows of a wider buffer: what lies beside them stays; odd distances, transposed inputs."""
    d = make(5, 1001, 30, 7, True, x)
    want = check(d)
    s = to_supa(d)
    logits = s.pop("logits")
    wide = torch.full((5, 1010), 7.0, dtype=logits.dtype, device="supa")
    wide[:, 4:1005] = logits
    assert torch.equal(torch.supa.adjust_logits(wide[:, 4:1005], **s).cpu(), want)
    torch.supa.adjust_logits_(wide[:, 4:1005], **s)
    got = wide.cpu()
    assert torch.equal(got[:, 4:1005], want) and (got[:, :4] == 7).all() and (got[:, 1005:] == 7).all()
    assert torch.equal(torch.supa.adjust_logits(logits.t().contiguous().t(), **s).cpu(), want)
    for k in ("tokens", "bias", "bias_tokens", "allowed"):
        v = s[k]
        s[k] = v.t().contiguous().t()
        assert torch.equal(torch.supa.adjust_logits(logits, **s).cpu(), want), k
        s[k] = torch.cat([v, v], 1)[:, : v.shape[1]]
        assert torch.equal(torch.supa.adjust_logits(logits, **s).cpu(), want), k
    s["repetition"] = torch.stack([s["repetition"]] * 2, 1)[:, 0]
    assert torch.equal(torch.supa.adjust_logits(logits, **s).cpu(), want)


def test_shared_memory_is_refused(no_fallback):
    buf = torch.zeros(4, 300, device="supa")
    logits = buf[:, :200]
    torch.supa.adjust_logits_(logits, bias_tokens=torch.zeros(4, 50, dtype=torch.int64, device="supa"), bias=buf[:, 200:250])
    with pytest.raises(RuntimeError, match="shares memory"):
        torch.supa.adjust_logits_(logits, bias_tokens=torch.zeros(4, 50, dtype=torch.int64, device="supa"), bias=buf[:, 180:230])
    torch.supa.adjust_logits(logits, bias_tokens=torch.zeros(4, 50, dtype=torch.int64, device="supa"), bias=buf[:, 180:230])


def test_empty(no_fallback):
    assert torch.supa.adjust_logits(torch.empty(0, 9, device="supa")).shape == (0, 9)
    torch.supa.adjust_logits_(torch.empty(0, 9, device="supa"))
    d = make(3, 50)
    s = d["logits"].to("supa")
    none = dict(tokens=torch.empty(3, 0, dtype=torch.int64, device="supa"), bias=torch.empty(3, 0, device="supa"),
                bias_tokens=torch.empty(3, 0, dtype=torch.int64, device="supa"), repetition=1.5)
    assert torch.equal(torch.supa.adjust_logits(s, **none).cpu(), d["logits"])


def test_versions(no_fallback):
    w = torch.ones(9, device="supa", requires_grad=True)
    for mode in (torch.no_grad, torch.enable_grad, torch.inference_mode):
        x = torch.ones(2, 9, device="supa")
        end, was = w * x, x._version
        with mode():
            torch.supa.adjust_logits_(x, allowed=torch.zeros(1, dtype=torch.int32, device="supa"))
        assert x._version == was + 1
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            end.sum().backward()
    with torch.inference_mode():
        x = torch.ones(2, 9, device="supa")
        torch.supa.adjust_logits_(x, allowed=torch.zeros(1, dtype=torch.int32, device="supa"))
    assert (x.cpu() == -math.inf).all()
