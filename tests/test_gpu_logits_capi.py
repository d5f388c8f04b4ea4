"""The C entry points of the operators on logits through ctypes alone (device
memory from torch's HIP allocator): the values against float64, and captured
runs of all of them replayed with the program's own work between, every replay
against the eager calls."""
import ctypes

import pytest
import torch

from test_logits_args import BF16, F32, I32, I64, AdjustDesc, BalanceDesc, DistillDesc, i64, vp

import torch_supa

pytestmark = pytest.mark.gpu

ROWS, VOCAB, K, EXPERTS, CHOSEN, HISTORY = 40, 5003, 12, 24, 3, 300


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(torch_supa.KERNELS_LIB)
    L.supa_amd_distill_workspace_bytes.restype = i64
    L.supa_amd_balance_workspace_bytes.restype = i64
    return L


class Run:
    """Buffers of one pass: both losses, their gradients, and adjusted logits in place."""

    def __init__(self, lib, seed, rest, rows=ROWS):
        self.lib, self.rest, self.rows = lib, rest, rows
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.rnd = rnd
        new = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        self.x = rnd(rows, VOCAB).bfloat16()
        self.ids = torch.rand(rows, VOCAB, generator=g, device="cuda").argsort(1)[:, :K].int().contiguous()
        self.t, self.lse, self.up = rnd(rows, K), new(rows).fill_(5.0), torch.full((), 2.0, device="cuda")
        self.loss, self.count, self.stats, self.pairs = new(1), new(1), new(rows, 8), new(rows, K, 2)
        self.gx = torch.empty_like(self.x)
        self.r = rnd(rows, EXPERTS)
        self.chosen = self.r.topk(CHOSEN).indices.contiguous()
        self.balance, self.counts, self.load, self.scale = new(1), new(EXPERTS, dtype=torch.int64), new(EXPERTS), new(2)
        self.gr = torch.empty_like(self.r)
        self.y = torch.empty_like(self.x)
        self.tokens = torch.randint(0, VOCAB, (rows, HISTORY), generator=g, device="cuda")
        self.bt, self.b = torch.randint(0, VOCAB, (9,), generator=g, device="cuda"), rnd(9)
        self.allowed = torch.randint(-(1 << 31), 1 << 31, (rows, (VOCAB + 31) // 32), generator=g, device="cuda").int()
        p = lambda t: t.data_ptr()  # noqa: E731
        self.d = DistillDesc(rows=rows, vocab=VOCAB, entries=K, inner=rows, dtype=BF16, teacher_dtype=F32, index_dtype=I32,
                             reduction=1, temperature=1.5, logits=p(self.x), indices=p(self.ids), teacher=p(self.t))
        self.d.logits_strides[1], self.d.indices_strides[1], self.d.teacher_strides[1], self.d.lse_strides[1] = VOCAB, K, K, 1
        if rest:
            self.d.teacher_lse = p(self.lse)
        self.bd = BalanceDesc(sequences=1, tokens=rows, experts=EXPERTS, k=CHOSEN, dtype=F32, index_dtype=I64,
                              logits=p(self.r), chosen=p(self.chosen))
        self.a = AdjustDesc(rows=rows, vocab=VOCAB, history=HISTORY, biases=9, in_stride=VOCAB, out_stride=VOCAB,
                            tokens_stride=HISTORY, allowed_stride=self.allowed.shape[1], dtype=BF16, token_dtype=I64,
                            bias_token_dtype=I64, repetition_value=1.25, presence_value=0.5, frequency_value=0.25,
                            data_in=p(self.y), out=p(self.y), tokens=p(self.tokens), bias_tokens=p(self.bt), bias=p(self.b),
                            allowed=p(self.allowed))
        self.ws = new(lib.supa_amd_distill_workspace_bytes(ctypes.byref(self.d)), dtype=torch.uint8)
        self.bws = new(lib.supa_amd_balance_workspace_bytes(ctypes.byref(self.bd)), dtype=torch.uint8)
        self.flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def launch(self):
        L, st, p, ref = self.lib, vp(torch.cuda.current_stream().cuda_stream), lambda t: vp(t.data_ptr()), ctypes.byref
        rc = [L.supa_amd_distill_forward(ref(self.d), p(self.loss), p(self.count), p(self.stats), p(self.pairs), p(self.ws),
                                         i64(self.ws.numel()), p(self.flag), st),
              L.supa_amd_distill_backward(ref(self.d), p(self.up), p(self.count), p(self.stats), p(self.pairs), p(self.gx), st),
              L.supa_amd_balance_forward(ref(self.bd), p(self.balance), p(self.counts), p(self.load), p(self.scale),
                                         p(self.bws), i64(self.bws.numel()), p(self.flag), st),
              L.supa_amd_balance_backward(ref(self.bd), p(self.up), p(self.load), p(self.scale), p(self.gr), st)]
        self.y.copy_(self.x)
        rc.append(L.supa_amd_adjust_logits(ref(self.a), st))
        assert rc == [0] * 5, rc

    def outputs(self):
        torch.cuda.synchronize()
        return [t.cpu().clone() for t in (self.loss, self.count, self.gx, self.balance, self.counts, self.gr, self.y, self.flag)]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows", [ROWS, 700])
def test_values(lib, rest, rows):
    run = Run(lib, 1, rest, rows)
    run.launch()
    loss, count, gx, balance, counts, gr, y, flag = run.outputs()
    assert float(count) == rows and int(flag) == 0
    x, ids, t = run.x.double().cpu().requires_grad_(), run.ids.long().cpu(), run.t.double().cpu() / 1.5
    log_q = torch.log_softmax(x / 1.5, 1)
    log_p = t - run.lse.double().cpu()[:, None] if rest else torch.log_softmax(t, 1)
    rows_ = (log_p.exp() * (log_p - log_q.gather(1, ids))).sum(1)
    if rest:
        r = 1 - log_p.exp().sum(1)
        rest_q = torch.logsumexp(log_q.scatter(1, ids, float("-inf")), 1)
        rows_ = rows_ + r * (r.log() - rest_q)
    want = rows_.mean()
    # as derived in test_gpu_distillation.py: (vocab / 64 + 128) of 2^-24, and what follows of it in the gradient
    s = (VOCAB / 64 + 128) * 2.0 ** -24
    assert abs(float(loss) - float(want.detach())) <= s + 2.0 ** -22 * float(want.detach())
    (wg,) = torch.autograd.grad(want * 2, x)
    assert ((gx.double() - wg).abs() <= wg.abs() * 2.0 ** -8 + 4 * s * 2 / rows).all()
    rr = run.r.double().cpu().requires_grad_()
    n = torch.bincount(run.chosen.cpu().flatten(), minlength=EXPERTS)
    assert torch.equal(counts, n)
    wb = (EXPERTS * n / (CHOSEN * rows) * torch.softmax(rr, 1).mean(0)).sum()
    assert abs(float(balance) - float(wb.detach())) <= 512 * 2.0 ** -24 * float(wb.detach())
    (wr,) = torch.autograd.grad(wb * 2, rr)
    assert ((gr.double() - wr).abs() <= 1024 * 2.0 ** -24 / rows * 4).all()
    v = run.x.double().cpu()
    c = torch.stack([torch.bincount(h, minlength=VOCAB) for h in run.tokens.cpu()]).double()
    v = torch.where(c > 0, torch.where(v > 0, v / 1.25, v * 1.25) - 0.25 * c - 0.5, v)
    v = v + torch.zeros(VOCAB, dtype=torch.float64).scatter_add(0, run.bt.cpu(), run.b.double().cpu())
    bits = (run.allowed.cpu().long()[:, :, None] >> torch.arange(32) & 1).bool().reshape(rows, -1)[:, :VOCAB]
    assert (y[~bits] == float("-inf")).all()
    assert ((y.double() - v).abs()[bits] <= (v.abs() * 2.0 ** -8 + 1e-5)[bits]).all()


@pytest.mark.parametrize("rest", [False, True])
def test_captured_and_replayed(lib, rest):
    """Two graphs, each with its own buffers, and one workspace for both;
    eager work and synchronizations between the replays."""
    eager, a, b = Run(lib, 5, rest), Run(lib, 5, rest), Run(lib, 6, rest)
    b.ws, b.bws = a.ws, a.bws  # graphs on one stream may share scratch memory
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
        x, route = eager.rnd(ROWS, VOCAB).bfloat16(), eager.rnd(ROWS, EXPERTS)
        for r in (a, b, eager):
            r.x.copy_(x)
            r.r.copy_(route)
            r.ids.copy_((eager.ids + step) % VOCAB)
        for r in (a, b):
            for t in (r.loss, r.gx, r.gr, r.balance, r.y, r.ws, r.bws):
                t.fill_(1)
            r.counts.fill_(-7)
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


def test_captured_long_ranges(lib):
    """A launch whose tables in LDS are the longest, captured without one before it in the process's other tests' sizes."""
    rows, vocab, history = 520, 33000, 70000
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, vocab, generator=g, device="cuda").bfloat16()
    outs = [torch.empty_like(x) for _ in range(2)]
    tokens = torch.randint(0, vocab, (rows, history), generator=g, device="cuda").int()
    bt, b = torch.randint(0, vocab, (rows, 16), generator=g, device="cuda"), torch.randn(rows, 16, generator=g, device="cuda")

    def desc(out, length):
        return AdjustDesc(rows=rows, vocab=vocab, history=length, biases=16, in_stride=vocab, out_stride=vocab, tokens_stride=history,
                          bias_tokens_stride=16, bias_stride=16, dtype=BF16, token_dtype=I32, bias_token_dtype=I64, repetition_value=1.5,
                          presence_value=0.25, frequency_value=0.125, data_in=x.data_ptr(), out=out.data_ptr(), tokens=tokens.data_ptr(),
                          bias_tokens=bt.data_ptr(), bias=b.data_ptr())

    for length in (65535, history):  # 16-bit and 32-bit counts
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert lib.supa_amd_adjust_logits(ctypes.byref(desc(outs[0], length)), vp(torch.cuda.current_stream().cuda_stream)) == 0
        assert lib.supa_amd_adjust_logits(ctypes.byref(desc(outs[1], length)), vp(torch.cuda.current_stream().cuda_stream)) == 0
        for _ in range(3):
            outs[0].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], outs[1])
        r = 517
        c = torch.bincount(tokens[r, :length].cpu(), minlength=vocab).double()
        v = x[r].double().cpu()
        v = torch.where(c > 0, torch.where(v > 0, v / 1.5, v * 1.5) - 0.125 * c - 0.25, v)
        v = v.scatter_add(0, bt[r].cpu(), b[r].double().cpu())
        assert ((outs[1][r].double().cpu() - v).abs() <= v.abs() * 2.0 ** -8 + 1e-5).all()


def test_out_of_range_sets_the_flag(lib):
    run = Run(lib, 3, False)
    run.ids[4, 5] = VOCAB
    run.launch()
    run.outputs()
    assert int(run.flag) == 3
    run.flag.zero_()
    run.ids[4, 5] = -1
    run.chosen[0, 0] = EXPERTS
    run.launch()
    assert int(run.outputs()[-1]) == 3
