"""torch.supa.distillation_loss where a token is listed twice: the loss is the sum over the pairs, each with its
own p log p, and the gradient (and what counts as listed) has the token once, with the sum of their p.

Values of a few tokens in closed form, float64.  The loss is off by under (vocab / 64 + 128) 2^-24, as derived in
test_gpu_distillation.py, the gradient by 300 of 2^-24 more of what it adds up (at most 2 here)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 2 * (3 * 129 + 300) * 2.0 ** -24


@pytest.mark.parametrize("rest", [False, True], ids=["listed", "rest"])
def test_pair_by_pair(rest, no_fallback):
    x = torch.tensor([[0.5, -1.0, 2.0, 0.0]])
    share = [0.25, 0.25, 0.5] if not rest else [0.25, 0.25, 0.375]  # of tokens 2, 2 and 0; 1/8 is the rest's
    t = torch.tensor([share], dtype=torch.float64).log().float()
    i = torch.tensor([[2, 2, 0]])
    q = torch.softmax(x.double(), 1)[0]
    p = t.double().exp()[0]
    lse = torch.zeros(1) if rest else None
    if not rest:
        p = p / p.sum()
    want = sum(float(p[k] * (p[k].log() - q[i[0, k]].log())) for k in range(3))
    grad = q.clone()
    if rest:
        r, q_rest = 1 - p.sum(), q[1] + q[3]
        want += float(r * (r.log() - q_rest.log()))
        grad[[1, 3]] -= r * q[[1, 3]] / q_rest
    grad[2] -= p[0] + p[1]
    grad[0] -= p[2]
    dx = x.to("supa").requires_grad_()
    loss = torch.supa.distillation_loss(dx, i.to("supa"), t.to("supa"), teacher_lse=None if lse is None else lse.to("supa"))
    (g,) = torch.autograd.grad(loss, dx)
    assert abs(float(loss.detach()) - want) <= TOL
    assert ((g[0].double().cpu() - grad).abs() <= TOL).all()
    # the divergence of the merged distribution is more by the two pairs' entropy, and has the same gradient
    merged = torch.supa.distillation_loss(dx, torch.tensor([[2, 0]], device="supa"), torch.tensor([[share[0] + share[1], share[2]]]).log().to("supa"),
                                          teacher_lse=None if lse is None else lse.to("supa"))
    (gm,) = torch.autograd.grad(merged, dx)
    assert abs(float(merged.detach()) - float(loss.detach()) - 0.5 * math.log(2)) <= 2 * TOL
    assert ((gm - g).abs().cpu() <= 2 * TOL).all()
