"""The transformer operators' C entry points through ctypes alone (device
memory from torch's HIP allocator): the values against float64, and a captured
run of all of them replayed with the program's own work between, every replay
against the eager calls."""
import ctypes

import pytest
import torch

from test_transformer_args import F32, BF16, I64, NormDesc, RotaryDesc, RotaryTensor, dbl, i32, i64, vp

import torch_supa

pytestmark = pytest.mark.gpu

ROWS, WIDTH, HEADS, DIM = 96, 1024, 8, 128


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(torch_supa.KERNELS_LIB)
    L.supa_amd_residual_norm_backward_workspace_bytes.restype = i64
    L.supa_amd_grad_norm_workspace_bytes.restype = i64
    return L


class Run:
    """Buffers of one pass: norm forward and backward, rotary positions in
    place, and the clipping of the gradients."""

    def __init__(self, lib, seed, norm=2):
        self.lib = lib
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
        shape = (ROWS, WIDTH)
        self.x, self.res, self.gh, self.gy = (self.rnd(*shape).bfloat16() for _ in range(4))
        self.gate, self.pw, self.w = (1 + 0.1 * self.rnd(WIDTH).bfloat16() for _ in range(3))
        self.h, self.y, self.gx, self.gres, self.q = (torch.empty_like(self.x) for _ in range(5))
        self.stats = torch.empty(ROWS, 4, device="cuda")
        self.grads = [torch.empty_like(self.gate) for _ in range(3)]
        self.total = torch.empty((), device="cuda")
        self.f = 10000.0 ** (-torch.arange(DIM // 2, dtype=torch.float64, device="cuda") * 2 / DIM)
        self.pos = torch.arange(1000, 1000 + ROWS, device="cuda")
        d = self.d = NormDesc(rows=ROWS, width=WIDTH, x_stride=WIDTH, residual_stride=WIDTH, gate_period=ROWS, dtype=BF16,
                              residual_dtype=BF16, param_dtype=BF16, post_norm=1, norm=norm, residual_scale=0.5, eps=1e-6)
        for name, t in dict(x=self.x, residual=self.res, gate=self.gate, post_weight=self.pw, weight=self.w).items():
            setattr(d, name, t.data_ptr())
        r = self.r = RotaryDesc(batch=1, seq=ROWS, dim=DIM, rotary=DIM, dtype=BF16, position_dtype=I64, scale=1.0,
                                frequencies=self.f.data_ptr(), positions=self.pos.data_ptr())
        r.position_strides[1] = 1
        r.q = RotaryTensor(data_in=self.q.data_ptr(), out=self.q.data_ptr(), heads=HEADS)
        for s in (r.q.in_strides, r.q.out_strides):
            s[0], s[1], s[2] = ROWS * WIDTH, WIDTH, DIM
        self.ws = torch.empty(lib.supa_amd_residual_norm_backward_workspace_bytes(ctypes.byref(d)), dtype=torch.uint8,
                              device="cuda")
        self.list = [self.gx, self.gres] + self.grads
        n = self.n = len(self.list)
        self.numel = (i64 * n)(*[t.numel() for t in self.list])
        self.types = (i32 * n)(*[BF16] * n)
        self.ptrs = (vp * n)(*[t.data_ptr() for t in self.list])
        self.clip_ws = torch.empty(lib.supa_amd_grad_norm_workspace_bytes(n, self.numel, self.types), dtype=torch.uint8,
                                   device="cuda")

    def launch(self):
        L, st = self.lib, vp(torch.cuda.current_stream().cuda_stream)
        p = lambda t: vp(t.data_ptr())  # noqa: E731
        rc = [L.supa_amd_residual_norm_forward(ctypes.byref(self.d), p(self.h), p(self.y), p(self.stats), st)]
        rc.append(L.supa_amd_residual_norm_backward(
            ctypes.byref(self.d), None, p(self.gh), p(self.gy), p(self.stats), p(self.gx), p(self.gres), p(self.grads[0]),
            p(self.grads[1]), None, p(self.grads[2]), None, p(self.ws), i64(self.ws.numel()), st))
        self.q.copy_(self.y)
        rc.append(L.supa_amd_rotary(ctypes.byref(self.r), st))
        rc.append(L.supa_amd_clip_grad_norm(self.n, self.ptrs, self.numel, self.types, dbl(2.0), dbl(1.0), p(self.total),
                                            F32, p(self.clip_ws), i64(self.clip_ws.numel()), st))
        assert rc == [0, 0, 0, 0], rc

    def outputs(self):
        torch.cuda.synchronize()
        return [t.cpu().clone() for t in [self.h, self.y, self.q, self.total] + self.list]


def test_values(lib):
    run = Run(lib, 1, norm=1)
    run.launch()
    h, y, q, total, *grads = run.outputs()
    x, res, gate, pw, w = (t.double().cpu().requires_grad_() for t in (run.x, run.res, run.gate, run.pw, run.w))

    def rms(v, weight):
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * weight

    eh = 0.5 * res + gate * rms(x, pw)
    ey = rms(eh, w)
    half = 2.0 ** -8
    # a rounding each (half a step of bf16), after float32
    assert ((h.double() - eh).abs() <= eh.abs() * half + 1e-5).all()
    assert ((y.double() - ey).abs() <= ey.abs() * half + 1e-5).all()
    v = y.double().view(ROWS, HEADS, 2, DIM // 2)
    turn = torch.polar(torch.ones((), dtype=torch.float64), (run.pos.cpu().double()[:, None] * run.f.cpu()))[:, None]
    z = torch.complex(v[:, :, 0], v[:, :, 1]) * turn
    eq = torch.stack((z.real, z.imag), 2).view(ROWS, WIDTH)
    assert ((q.double() - eq).abs() <= eq.abs() * half + 1e-5).all()
    want = torch.autograd.grad([eh, ey], [x, res, gate, pw, w], [run.gh.double().cpu(), run.gy.double().cpu()])
    norm = torch.sqrt(sum((g * g).sum() for g in want))
    # the norm of gradients rounded to bf16: no further off than their rounding
    assert abs(float(total) - float(norm)) <= float(norm) * half
    for g, e in zip(grads, want):
        e = e / (total.double() + 1e-6)
        # two roundings, and the sums' float32 (512 of 2^-24 of the largest column's magnitude)
        assert ((g.double() - e).abs() <= e.abs() * (2 * half + half * half) + 512 * 2.0 ** -24 * e.abs().max()).all()


def test_captured_and_replayed(lib):
    """Two graphs, each with its own buffers, and one workspace for both;
    eager work and synchronizations between the replays."""
    eager, a, b = Run(lib, 5), Run(lib, 5), Run(lib, 6)
    b.ws, b.clip_ws = a.ws, a.clip_ws  # graphs on one stream may share scratch memory
    for r in (eager, a, b):
        r.launch()  # nothing is loaded for the first time under capture
    torch.cuda.synchronize()
    graphs = []
    for r in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r.launch()
        graphs.append(g)
    for step in range(4):
        x = eager.rnd(ROWS, WIDTH).bfloat16()
        for r in (a, b, eager):
            r.x.copy_(x)
        for t in a.list + b.list + [a.h, b.h]:
            t.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        got_b = b.outputs()
        got_a = a.outputs()
        eager.launch()
        for u, v in zip(got_a, eager.outputs()):
            assert torch.equal(u, v), step
        b.launch()
        for u, v in zip(got_b, b.outputs()):
            assert torch.equal(u, v), step
