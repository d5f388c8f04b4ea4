"""The operators on logits without a GPU: what their C entry points refuse
before any launch, their workspace sizes, the Python layer's argument errors
and what the checks say of shapes, types and gradients (on meta tensors)."""
import ctypes
import math

import pytest
import torch

torch_supa = pytest.importorskip("torch_supa")

i64, i32, dbl, vp = ctypes.c_int64, ctypes.c_int32, ctypes.c_double, ctypes.c_void_p
EINVAL, EDTYPE, ELAYOUT, EWORKSPACE = -1, -2, -3, -4
F16, F32, F64, BF16, I64, I32 = 5, 6, 7, 15, 4, 3
FAKE = 256  # never dereferenced: the checks come first


class DistillDesc(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("rows", "vocab", "entries", "inner")] + [
        (n + "_strides", i64 * 2) for n in ("logits", "indices", "teacher", "lse")] + [
        (n, i32) for n in ("dtype", "teacher_dtype", "index_dtype", "reduction")] + [("temperature", dbl)] + [
        (n, vp) for n in ("logits", "indices", "teacher", "teacher_lse")]


class BalanceDesc(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("sequences", "tokens", "experts", "k")] + [
        (n, i32) for n in ("dtype", "index_dtype", "scores", "reserved")] + [(n, vp) for n in ("logits", "chosen", "mask")]


class AdjustDesc(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("rows", "vocab", "history", "biases", "in_stride", "out_stride", "tokens_stride",
                                   "bias_tokens_stride", "bias_stride", "allowed_stride")] + [
        (n, i32) for n in ("dtype", "token_dtype", "length_dtype", "prompt_dtype", "bias_token_dtype", "reserved")] + [
        (n, dbl) for n in ("repetition_value", "presence_value", "frequency_value")] + [
        (n, vp) for n in ("data_in", "out", "tokens", "lengths", "prompt_lengths", "repetition", "presence", "frequency",
                          "bias_tokens", "bias", "allowed")]


def made(desc, base, kw):
    d = desc(**base)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def distill_desc(**kw):
    return made(DistillDesc, dict(rows=4, vocab=64, entries=8, inner=4, logits_strides=(i64 * 2)(0, 64), dtype=BF16,
                                  teacher_dtype=F32, index_dtype=I64, reduction=1, temperature=1.0, logits=FAKE,
                                  indices=FAKE, teacher=FAKE), kw)


def balance_desc(**kw):
    return made(BalanceDesc, dict(sequences=2, tokens=10, experts=8, k=2, dtype=F32, index_dtype=I64, logits=FAKE,
                                  chosen=FAKE), kw)


def adjust_desc(**kw):
    return made(AdjustDesc, dict(rows=2, vocab=100, in_stride=100, out_stride=100, dtype=F32, repetition_value=1.0,
                                 data_in=FAKE, out=FAKE), kw)


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(torch_supa.KERNELS_LIB)
    L.supa_amd_distill_workspace_bytes.restype = i64
    L.supa_amd_balance_workspace_bytes.restype = i64
    return L


@pytest.mark.parametrize("kw, want", [
    (dict(rows=-1), EINVAL), (dict(vocab=0), EINVAL), (dict(entries=0), EINVAL), (dict(entries=1025), ELAYOUT),
    (dict(inner=0), EINVAL), (dict(rows=1 << 31), ELAYOUT), (dict(vocab=1 << 31), ELAYOUT), (dict(temperature=0.0), EINVAL),
    (dict(temperature=-1.0), EINVAL), (dict(temperature=math.nan), EINVAL), (dict(temperature=math.inf), EINVAL),
    (dict(reduction=3), EINVAL), (dict(dtype=F64), EDTYPE), (dict(teacher_dtype=I64), EDTYPE),
    (dict(index_dtype=F32), EDTYPE), (dict(logits=None), EINVAL), (dict(indices=None), EINVAL), (dict(teacher=None), EINVAL),
])
def test_distill_refuses(lib, kw, want):
    d = distill_desc(**kw)
    assert lib.supa_amd_distill_forward(ctypes.byref(d), vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), i64(1 << 20),
                                        None, None) == want
    if not kw.keys() & {"teacher", "indices"}:  # which the backward does not read
        assert lib.supa_amd_distill_backward(ctypes.byref(d), vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), None) == want


def test_distill_other_refusals(lib):
    fwd, bwd = lib.supa_amd_distill_forward, lib.supa_amd_distill_backward
    d = distill_desc()
    need = lib.supa_amd_distill_workspace_bytes(ctypes.byref(d))
    assert need >= 16 and lib.supa_amd_distill_workspace_bytes(ctypes.byref(distill_desc(vocab=0))) == EINVAL

    def forward(d=d, loss=FAKE, count=FAKE, stats=FAKE, ws=FAKE, size=need):
        return fwd(ctypes.byref(d), vp(loss), vp(count), vp(stats), None, vp(ws), i64(size), None, None)

    assert fwd(None, vp(FAKE), vp(FAKE), vp(FAKE), None, vp(FAKE), i64(need), None, None) == EINVAL
    assert forward(loss=None) == EINVAL and forward(count=None) == EINVAL and forward(stats=None) == EINVAL
    assert forward(ws=None) == EWORKSPACE and forward(size=need - 1) == EWORKSPACE and forward(ws=FAKE + 4) == EINVAL
    assert forward(distill_desc(rows=0, reduction=0)) == 0

    def back(d=d, grad=FAKE, count=FAKE, stats=FAKE, pairs=FAKE, out=FAKE):
        return bwd(ctypes.byref(d), vp(grad), vp(count), vp(stats), vp(pairs), vp(out), None)

    for name in ("grad", "count", "stats", "pairs", "out"):
        assert back(**{name: None}) == EINVAL, name
    assert back(pairs=FAKE + 4) == EINVAL
    assert back(distill_desc(rows=0)) == 0


@pytest.mark.parametrize("kw, want", [
    (dict(sequences=-1), EINVAL), (dict(tokens=-1), EINVAL), (dict(experts=0), EINVAL), (dict(k=0), EINVAL),
    (dict(experts=1025), ELAYOUT), (dict(k=9), ELAYOUT), (dict(sequences=1 << 16, tokens=1 << 16), ELAYOUT),
    (dict(scores=2), EINVAL), (dict(dtype=F64), EDTYPE), (dict(index_dtype=F32), EDTYPE), (dict(logits=None), EINVAL),
])
def test_balance_refuses(lib, kw, want):
    d = balance_desc(**kw)
    assert lib.supa_amd_balance_forward(ctypes.byref(d), vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), i64(1 << 24),
                                        None, None) == want
    assert lib.supa_amd_balance_backward(ctypes.byref(d), vp(FAKE), vp(FAKE), vp(FAKE), vp(FAKE), None) == want


def test_balance_takes_any_product_below_the_limit(lib):
    for sequences, tokens in ((3, (2 ** 31 - 1) // 3), (1, 2 ** 31 - 1), (2 ** 31 - 1, 1)):
        d = balance_desc(sequences=sequences, tokens=tokens)
        assert lib.supa_amd_balance_workspace_bytes(ctypes.byref(d)) > 0
        assert lib.supa_amd_balance_workspace_bytes(ctypes.byref(balance_desc(sequences=sequences, tokens=tokens + 1))) == ELAYOUT


def test_balance_other_refusals(lib):
    fwd, bwd = lib.supa_amd_balance_forward, lib.supa_amd_balance_backward
    d = balance_desc()
    need = lib.supa_amd_balance_workspace_bytes(ctypes.byref(d))
    assert need > 0 and lib.supa_amd_balance_workspace_bytes(ctypes.byref(balance_desc(k=0))) == EINVAL

    def forward(d=d, out=(FAKE,) * 4, ws=FAKE, size=need):
        return fwd(ctypes.byref(d), *map(vp, out), vp(ws), i64(size), None, None)

    for i in range(4):
        assert forward(out=[None if j == i else FAKE for j in range(4)]) == EINVAL
    assert forward(balance_desc(chosen=None)) == EINVAL and forward(balance_desc(sequences=0)) == EINVAL
    assert forward(ws=None) == EWORKSPACE and forward(size=need - 1) == EWORKSPACE and forward(ws=FAKE + 4) == EINVAL
    for i in range(4):
        assert bwd(ctypes.byref(d), *[vp(None if j == i else FAKE) for j in range(4)], None) == EINVAL
    assert bwd(ctypes.byref(balance_desc(tokens=0)), *[vp(FAKE)] * 4, None) == 0
    assert bwd(ctypes.byref(balance_desc(sequences=0)), *[vp(FAKE)] * 4, None) == 0


@pytest.mark.parametrize("kw, want", [
    (dict(rows=-1), EINVAL), (dict(vocab=0), EINVAL), (dict(history=-1), EINVAL), (dict(biases=-1), EINVAL),
    (dict(rows=1 << 31), ELAYOUT), (dict(vocab=1 << 29), ELAYOUT), (dict(history=1 << 31, tokens=FAKE), ELAYOUT),
    (dict(biases=1 << 31), ELAYOUT), (dict(dtype=F64), EDTYPE), (dict(history=3), EINVAL), (dict(biases=3), EINVAL),
    (dict(biases=3, bias_tokens=FAKE), EINVAL), (dict(history=3, tokens=FAKE, token_dtype=F32), EDTYPE),
    (dict(history=3, tokens=FAKE, token_dtype=I64, lengths=FAKE, length_dtype=F32), EDTYPE),
    (dict(history=3, tokens=FAKE, token_dtype=I64, prompt_lengths=FAKE, prompt_dtype=F32), EDTYPE),
    (dict(biases=3, bias_tokens=FAKE, bias=FAKE, bias_token_dtype=F32), EDTYPE), (dict(data_in=None), EINVAL),
    (dict(out=None), EINVAL), (dict(rows=0), 0),
])
def test_adjust_refuses(lib, kw, want):
    assert lib.supa_amd_adjust_logits(ctypes.byref(adjust_desc(**kw)), None) == want
    assert lib.supa_amd_adjust_logits(None, None) == EINVAL


def meta(*shape, dtype=torch.float32, grad=False):
    return torch.empty(shape, dtype=dtype, device="meta", requires_grad=grad)


LONG, INT, BOOL, BF = torch.int64, torch.int32, torch.bool, torch.bfloat16


@pytest.mark.parametrize("kw, match", [
    (dict(logits=meta(3, 9, dtype=torch.float64)), "float32, bfloat16"),
    (dict(logits=meta(3, 0)), "last dim"), (dict(logits=torch.ones(3, 9)), "on cpu|supa tensors|same device"),
    (dict(indices=meta(3, 2)), "int64 or int32"), (dict(indices=meta(2, 2, dtype=LONG)), "do not fit"),
    (dict(indices=meta(3, dtype=LONG)), "do not fit"), (dict(indices=meta(3, 0, dtype=LONG), teacher=meta(3, 0)), "1 to 1024"),
    (dict(indices=meta(3, 1025, dtype=LONG), teacher=meta(3, 1025)), "1 to 1024"),
    (dict(teacher=meta(3, 3)), "teacher_logits of"), (dict(teacher=meta(3, 2, dtype=LONG)), "teacher_logits of float32"),
    (dict(teacher=meta(3, 2, grad=True)), "no gradient"), (dict(teacher_lse=meta(3, grad=True)), "no gradient"),
    (dict(teacher_lse=meta(3, 1)), "teacher_lse"), (dict(teacher_lse=meta(3, dtype=LONG)), "teacher_lse"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=math.inf), "temperature"),
    (dict(temperature=math.nan), "temperature"), (dict(temperature=1e-39), "temperature"),
    (dict(reduction="batchmean"), "reduction"), (dict(reduction=1), "reduction"),
])
def test_distillation_loss_arguments(kw, match):
    a = {"logits": meta(3, 9), "indices": meta(3, 2, dtype=LONG), "teacher": meta(3, 2)} | kw
    x, i, t = (a.pop(n) for n in ("logits", "indices", "teacher"))
    with pytest.raises((RuntimeError, ValueError, NotImplementedError), match=match):
        torch.supa.distillation_loss(x, i, t, **a)


@pytest.mark.parametrize("kw, match", [
    (dict(logits=meta(3, 4, dtype=torch.float64)), "float32, bfloat16"), (dict(logits=meta(3, 0)), "1 to 1024 experts"),
    (dict(logits=meta(3, 1025)), "1 to 1024 experts"), (dict(experts=meta(3, 5, dtype=LONG)), "choices a token"),
    (dict(experts=meta(3, 0, dtype=LONG)), "choices a token"), (dict(experts=meta(dtype=LONG)), "scalar"),
    (dict(experts=meta(2, 2, dtype=LONG)), "do not fit"), (dict(experts=meta(3, 2)), "int64 or int32"),
    (dict(mask=meta(3)), "mask as bools"), (dict(mask=meta(3, 1, dtype=BOOL)), "mask as bools"),
    (dict(scores="tanh"), "scores"), (dict(logits=meta(4), experts=meta(2, dtype=LONG), per_sequence=True), "tokens, experts"),
])
def test_router_balance_loss_arguments(kw, match):
    a = {"logits": meta(3, 4), "experts": meta(3, 2, dtype=LONG)} | kw
    x, e = a.pop("logits"), a.pop("experts")
    with pytest.raises((RuntimeError, ValueError), match=match):
        torch.supa.router_balance_loss(x, e, **a)


@pytest.mark.parametrize("kw, match", [
    (dict(logits=meta(2, 3, 9)), "vocab"), (dict(logits=meta(2, 0)), "vocab"), (dict(logits=meta(2, 9, dtype=LONG)), "float32, bfloat16"),
    (dict(repetition=1.5), "need the tokens"), (dict(presence=meta(2)), "need the tokens"),
    (dict(lengths=meta(2, dtype=LONG)), "need the tokens"), (dict(tokens=meta(2, 5)), "int64 or int32 tokens"),
    (dict(tokens=meta(3, 5, dtype=LONG)), "tokens of shape"), (dict(tokens=meta(5, dtype=LONG)), "tokens of shape"),
    (dict(tokens=meta(2, 5, dtype=LONG), repetition=0.0), "repetition > 0"),
    (dict(tokens=meta(2, 5, dtype=LONG), repetition=math.nan), "repetition > 0"),
    (dict(tokens=meta(2, 5, dtype=LONG), repetition=1e-60), "repetition > 0"),  # as float32
    (dict(tokens=meta(2, 5, dtype=LONG), repetition=1e39), "repetition > 0"),
    (dict(tokens=meta(2, 5, dtype=LONG), presence=1e39), "finite penalties"),
    (dict(tokens=meta(2, 5, dtype=LONG), presence=math.inf), "finite"),
    (dict(tokens=meta(2, 5, dtype=LONG), lengths=meta(2)), "lengths of int64"),
    (dict(tokens=meta(2, 5, dtype=LONG), lengths=meta(3, dtype=LONG)), "lengths of shape"),
    (dict(tokens=meta(2, 5, dtype=LONG), repetition=meta(2, 1)), "repetition of shape"),
    (dict(tokens=meta(2, 5, dtype=LONG), frequency=meta(2, dtype=BF)), "frequency of float32"),
    (dict(bias=meta(2, 3)), "together"), (dict(bias_tokens=meta(2, 3, dtype=LONG)), "together"),
    (dict(bias_tokens=meta(2, 3, dtype=LONG), bias=meta(2, 4)), "tokens a row"),
    (dict(bias_tokens=meta(2, 3), bias=meta(2, 3)), "bias_tokens and a float32"),
    (dict(bias_tokens=meta(3, 3, dtype=LONG), bias=meta(3, 3)), "bias_tokens of shape"),
    (dict(allowed=meta(2, 1, dtype=LONG)), "int32 words"), (dict(allowed=meta(2, 0, dtype=INT)), "int32 words"),
    (dict(allowed=meta(3, 1, dtype=INT)), "allowed of shape"), (dict(logits=meta(2, 9, grad=True)), "no gradient"),
    (dict(bias_tokens=meta(3, dtype=LONG), bias=meta(3, grad=True)), "no gradient"),
])
def test_adjust_logits_arguments(kw, match):
    a = {"logits": meta(2, 9)} | kw
    x = a.pop("logits")
    for call in (torch.supa.adjust_logits, torch.supa.adjust_logits_):
        with pytest.raises(RuntimeError, match=match):
            call(x, **a)


def test_adjust_in_place_layouts():
    with pytest.raises(RuntimeError, match="contiguous"):
        torch.supa.adjust_logits_(meta(9, 2).t())
    with pytest.raises(RuntimeError, match="overlap"):
        torch.supa.adjust_logits_(meta(9).expand(2, 9))
    with pytest.raises(RuntimeError, match="overlap"):
        torch.supa.adjust_logits_(meta(20).as_strided((4, 9), (3, 1)))


def test_other_devices_have_no_kernel():
    with pytest.raises(NotImplementedError):
        torch.supa.distillation_loss(torch.ones(3, 9), torch.ones(3, 2, dtype=LONG), torch.ones(3, 2))
    with pytest.raises(NotImplementedError):
        torch.supa.router_balance_loss(torch.ones(3, 9), torch.ones(3, 2, dtype=LONG))
    with pytest.raises(NotImplementedError):
        torch.supa.adjust_logits(torch.ones(3, 9))


def test_operators_are_registered():
    for op in ("distillation_loss", "router_balance_loss", "adjust_logits", "adjust_logits_"):
        for key in ("PrivateUse1", "AutogradPrivateUse1", "Meta"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key("supa::" + op, key), (op, key)


def test_a_learned_temperature_is_refused():
    """It would get no gradient."""
    x, i, t = meta(4, 50), meta(4, 3, dtype=LONG), meta(4, 3)
    learned = torch.tensor(2.0, requires_grad=True)
    with pytest.raises(TypeError, match="temperature is a number"):
        torch.supa.distillation_loss(x, i, t, temperature=learned)
    with torch.no_grad():
        torch.supa.distillation_loss(x, i, t, temperature=learned)
    torch.supa.distillation_loss(x, i, t, temperature=torch.tensor(2.0))
