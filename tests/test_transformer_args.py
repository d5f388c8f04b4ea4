"""The transformer operators without a GPU: what their C entry points refuse
before any launch, their workspace sizes, the Python layer's argument errors,
and rotary_frequencies against its formulas."""
import ctypes
import math
import os

import pytest
import torch

torch_supa = pytest.importorskip("torch_supa")

i64, i32, dbl, vp = ctypes.c_int64, ctypes.c_int32, ctypes.c_double, ctypes.c_void_p
EINVAL, EDTYPE, ELAYOUT, EWORKSPACE = -1, -2, -3, -4
F16, F32, F64, BF16, I64 = 5, 6, 7, 15, 4
FAKE = 256  # never dereferenced: the checks come first


class NormDesc(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("rows", "width", "x_stride", "residual_stride", "gate_period")] + [
        (n, i32) for n in ("dtype", "residual_dtype", "param_dtype", "post_norm", "norm", "reserved")] + [
        (n, dbl) for n in ("residual_scale", "eps")] + [
        (n, vp) for n in ("x", "residual", "gate", "post_weight", "post_bias", "weight", "bias")]


class RotaryTensor(ctypes.Structure):
    _fields_ = [("data_in", vp), ("out", vp), ("heads", i64), ("in_strides", i64 * 3), ("out_strides", i64 * 3)]


class RotaryDesc(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("batch", "seq", "dim", "rotary")] + [
        (n, i32) for n in ("dtype", "layout", "inverse", "position_dtype")] + [
        ("scale", dbl), ("frequencies", vp), ("positions", vp), ("position_strides", i64 * 2), ("offset", i64),
        ("q", RotaryTensor), ("k", RotaryTensor)]


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(torch_supa.KERNELS_LIB)
    L.supa_amd_residual_norm_backward_workspace_bytes.restype = i64
    L.supa_amd_grad_norm_workspace_bytes.restype = i64
    return L


def norm_desc(**kw):
    d = NormDesc(rows=4, width=64, x_stride=64, residual_stride=64, gate_period=1, dtype=BF16, residual_dtype=BF16,
                 param_dtype=BF16, post_norm=0, norm=1, residual_scale=1.0, eps=1e-6, x=FAKE, residual=FAKE)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, want", [
    (dict(width=0), EINVAL), (dict(width=16385), ELAYOUT), (dict(rows=-1), EINVAL), (dict(rows=1 << 31), ELAYOUT),
    (dict(dtype=F64), EDTYPE), (dict(residual_dtype=F16), EDTYPE), (dict(param_dtype=F16), EDTYPE),
    (dict(norm=3), EINVAL), (dict(post_norm=-1), EINVAL), (dict(gate=FAKE, gate_period=3), EINVAL),
    (dict(gate=FAKE, gate_period=0), EINVAL), (dict(bias=FAKE), EINVAL), (dict(post_weight=FAKE), EINVAL),
    (dict(norm=0, weight=FAKE), EINVAL), (dict(x=None), EINVAL), (dict(residual=None), EINVAL),
    (dict(norm=0), EINVAL),  # y without a norm
])
def test_residual_norm_forward_refuses(lib, kw, want):
    d = norm_desc(**kw)
    assert lib.supa_amd_residual_norm_forward(ctypes.byref(d), vp(FAKE), vp(FAKE), None, None) == want


def test_residual_norm_other_refusals(lib):
    fwd, bwd = lib.supa_amd_residual_norm_forward, lib.supa_amd_residual_norm_backward
    d = norm_desc()
    assert fwd(None, vp(FAKE), vp(FAKE), None, None) == EINVAL
    assert fwd(ctypes.byref(d), None, vp(FAKE), None, None) == EINVAL
    assert fwd(ctypes.byref(d), vp(FAKE), None, None, None) == EINVAL  # no y
    assert fwd(ctypes.byref(norm_desc(rows=0)), None, None, None, None) == 0
    need = lib.supa_amd_residual_norm_backward_workspace_bytes(ctypes.byref(d))
    assert need > 0 and need % 4 == 0
    assert lib.supa_amd_residual_norm_backward_workspace_bytes(ctypes.byref(norm_desc(width=0))) == EINVAL
    assert lib.supa_amd_residual_norm_backward_workspace_bytes(ctypes.byref(norm_desc(rows=0))) == 0

    def back(desc=d, h=None, stats=FAKE, gate=None, pw=None, pb=None, w=None, b=None, ws=FAKE, size=need):
        return bwd(ctypes.byref(desc), vp(h), vp(FAKE), vp(FAKE), vp(stats), vp(FAKE), vp(FAKE), vp(gate), vp(pw), vp(pb),
                   vp(w), vp(b), vp(ws), i64(size), None)

    assert back(stats=FAKE + 8) == EINVAL and back(ws=FAKE + 2) == EINVAL  # alignment
    assert fwd(ctypes.byref(d), vp(FAKE), vp(FAKE), vp(FAKE + 4), None) == EINVAL
    assert back(ws=None) == EWORKSPACE and back(size=need - 1) == EWORKSPACE
    assert back(stats=None) == EINVAL and back(gate=FAKE) == EINVAL and back(pw=FAKE) == EINVAL
    assert back(b=FAKE) == EINVAL  # the bias of an RMS norm
    assert back(norm_desc(gate=FAKE, gate_period=4), h=FAKE) == EINVAL  # h alone does not do with a gate
    assert back(norm_desc(x=None)) == EINVAL and back(norm_desc(residual=None)) == EINVAL
    assert back(norm_desc(rows=0)) == EINVAL


def rotary_desc(**kw):
    d = RotaryDesc(batch=1, seq=4, dim=16, rotary=16, dtype=BF16, layout=0, position_dtype=I64, scale=1.0,
                   frequencies=FAKE)
    d.q = RotaryTensor(data_in=FAKE, out=FAKE, heads=2)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, want", [
    (dict(rotary=0), EINVAL), (dict(rotary=15), EINVAL), (dict(rotary=18), EINVAL), (dict(dim=0), EINVAL),
    (dict(batch=-1), EINVAL), (dict(layout=2), EINVAL), (dict(position_dtype=F32), EDTYPE), (dict(dtype=F64), EDTYPE),
    (dict(frequencies=None), EINVAL), (dict(q=RotaryTensor(data_in=FAKE, heads=2)), EINVAL),
    (dict(q=RotaryTensor(data_in=FAKE, out=FAKE, heads=-1)), EINVAL), (dict(dim=2048, rotary=1026), ELAYOUT),
    (dict(batch=1 << 16, seq=1 << 16), ELAYOUT), (dict(dim=1 << 24), ELAYOUT),
    (dict(q=RotaryTensor()), 0), (dict(seq=0), 0), (dict(batch=0), 0),  # nothing to do
])
def test_rotary_refuses(lib, kw, want):
    assert lib.supa_amd_rotary(ctypes.byref(rotary_desc(**kw)), None) == want
    assert lib.supa_amd_rotary(None, None) == EINVAL


def test_clip_refuses(lib):
    p = (vp * 2)(FAKE, FAKE)
    n = (i64 * 2)(1000, 70000)
    t = (i32 * 2)(BF16, F32)
    # 16 vectors for each of 256 threads: 32768 bf16, 16384 f32 elements a partial, and the norm
    need = lib.supa_amd_grad_norm_workspace_bytes(2, n, t)
    assert need == 8 * (1 + 1 + 5)
    assert lib.supa_amd_grad_norm_workspace_bytes(2, n, (i32 * 2)(BF16, I64)) == EDTYPE
    assert lib.supa_amd_grad_norm_workspace_bytes(2, (i64 * 2)(1, -1), t) == EINVAL
    clip = lib.supa_amd_clip_grad_norm

    def call(count=2, ptrs=p, numel=n, dtypes=t, order=2.0, limit=1.0, out=FAKE, out_type=F32, ws=FAKE, size=need):
        return clip(count, ptrs, numel, dtypes, dbl(order), dbl(limit), vp(out), out_type, vp(ws), i64(size), None)

    assert call(order=3.0) == EINVAL and call(limit=-1.0) == EINVAL and call(limit=math.nan) == EINVAL
    assert call(out=None) == EINVAL and call(out_type=BF16) == EDTYPE and call(count=-1) == EINVAL
    assert call(ptrs=(vp * 2)(FAKE, None)) == EINVAL and call(dtypes=(i32 * 2)(F32, I64)) == EDTYPE
    assert call(ws=FAKE + 4) == EINVAL and lib.supa_amd_grad_scale(2, p, n, t, dbl(1.0), vp(FAKE + 4), i64(8), None) == EINVAL
    assert call(ws=None) == EWORKSPACE and call(size=need - 1) == EWORKSPACE
    assert lib.supa_amd_grad_scale(2, p, n, t, dbl(-1.0), vp(FAKE), i64(8), None) == EINVAL
    assert lib.supa_amd_grad_scale(2, p, n, t, dbl(1.0), None, i64(8), None) == EWORKSPACE


def test_python_arguments():
    x = torch.ones(2, 3, 8)
    with pytest.raises(ValueError, match="layout"):
        torch.supa.rotary_embedding(x, None, torch.ones(4), layout="quarter")
    with pytest.raises(TypeError, match="positions"):
        torch.supa.rotary_embedding_(x, None, torch.ones(4), 0.5)
    with pytest.raises(ValueError, match="post_norm"):
        torch.supa.residual_norm(x, x, post_norm="batch")
    with pytest.raises(NotImplementedError):  # tensors of another device have no kernel
        torch.supa.residual_norm(x, x)
    p = torch.nn.Parameter(torch.ones(3))
    assert float(torch.supa.clip_grad_norm_([p], 1.0)) == 0.0  # no gradient
    p.grad = torch.ones(3)
    with pytest.raises(NotImplementedError):
        torch.supa.clip_grad_norm_([p], 1.0)


def test_rotary_frequencies():
    f, scale = torch.supa.rotary_frequencies(8, 500.0, device="cpu")
    assert f.dtype == torch.float64 and scale == 1.0
    want = [500.0 ** (-2 * i / 8) for i in range(4)]
    assert f.tolist() == pytest.approx(want, rel=1e-14)
    lin, s = torch.supa.rotary_frequencies(8, 500.0, scaling="linear", factor=4.0, device="cpu")
    assert lin.tolist() == pytest.approx([v / 4 for v in want], rel=1e-14) and s == 1.0
    ntk, _ = torch.supa.rotary_frequencies(8, 500.0, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0].item() == 1.0 and ntk[3].item() == pytest.approx(want[3] / 4, rel=1e-12)
    # turns over 4096 positions: pairs above `fast` kept, below `slow` divided, a line between
    sm, s = torch.supa.rotary_frequencies(64, scaling="smooth", factor=8.0, original_length=4096, device="cpu")
    base, _ = torch.supa.rotary_frequencies(64, device="cpu")
    for a, b in zip(sm.tolist(), base.tolist()):
        turns = 4096 * b / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        assert a == pytest.approx(b * keep + b / 8 * (1 - keep), rel=1e-12)
    assert s == 1.0 and sm[0] == base[0] and sm[-1].item() == pytest.approx(base[-1].item() / 8)
    ya, s = torch.supa.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    assert s == pytest.approx(0.1 * math.log(8.0) + 1)

    def index(turns):
        return 64 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))

    lo, hi = math.floor(index(32.0)), math.ceil(index(1.0))
    for i, (a, b) in enumerate(zip(ya.tolist(), base.tolist())):
        keep = 1 - min(1.0, max(0.0, (i - lo) / (hi - lo)))
        assert a == pytest.approx(b * keep + b / 8 * (1 - keep), rel=1e-12)


@pytest.mark.parametrize("args, kw", [
    ((7,), {}), ((0,), {}), ((8, 1.0), {}), ((8,), dict(scaling="other")), ((8,), dict(scaling="linear", factor=0.5)),
    ((8,), dict(scaling="smooth", factor=2.0)), ((8,), dict(scaling="yarn", factor=2.0, original_length=64, slow=9.0, fast=3.0)),
    ((2,), dict(scaling="ntk", factor=2.0)),
])
def test_rotary_frequencies_refuses(args, kw):
    with pytest.raises(ValueError):
        torch.supa.rotary_frequencies(*args, **kw)


def test_operators_are_registered():
    for op in ("residual_norm", "rotary_embedding", "rotary_embedding_", "clip_grad_norm_"):
        for key in ("PrivateUse1", "AutogradPrivateUse1"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key("supa::" + op, key), (op, key)
    assert os.path.exists(torch_supa.KERNELS_LIB)
