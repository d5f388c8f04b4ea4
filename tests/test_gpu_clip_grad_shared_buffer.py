"""torch.supa.clip_grad_norm_ on gradients that are pieces of one buffer: pieces
that reach over each other's memory without sharing any of it are clipped, what
lies between them stays, and pieces that share some are refused with nothing
written.

Tolerances: the norm's own half step (2^-24) beside its float64 sum; a factor of
one half less 1e-6 / norm of it, rounded to float32 (2^-24), the product to its
type (eps / 2)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16

APART = {
    "columns and a column": lambda m: [m[:, :7], m[:, 7]],
    "a column before columns": lambda m: [m[:, 8:], m[:, 7]],
    "columns, others transposed": lambda m: [m[:, :3], m[:, 3:9].t()],
    "every second row and a row between": lambda m: [m[::2], m[1:2]],
    "columns of rows that begin later": lambda m: [m[:22, :4], m[20:, 4:8]],
    "columns before, of rows that begin later": lambda m: [m[:22, 4:8], m[20:, :4]],
    "a slice and a block of a cube": lambda m: [m.view(8, 5, 30)[:, 0], m.view(8, 5, 30)[:, 1:, 2:]],
    "single elements": lambda m: [m[3, 4:5], m[3, 5], m[2:4, 6], m[2:4, :3]],
    "columns of two types": lambda m: [m[:, :10], m[:, 10:].view(BF16)],
}
SHARED = {
    "a column of the columns": lambda m: [m[:, :7], m[:, 6]],
    "transposed columns": lambda m: [m[:, :4], m[:, 3:9].t()],
    "a row of every second row": lambda m: [m[::2], m[2:3]],
    "a column more, of rows that begin later": lambda m: [m[:22, :5], m[20:, 4:8]],
    "a column more before": lambda m: [m[:22, 3:8], m[20:, :4]],
    "a slice and a block of a cube": lambda m: [m.view(8, 5, 30)[:, 1], m.view(8, 5, 30)[:, 1:, 2:]],
    "columns of two types": lambda m: [m[:, :11], m[:, 10:].view(BF16)],
    "an element of another's": lambda m: [m[3, 4:6], m[3, 5]],
}


def buffer():
    return torch.randn(40, 30, generator=torch.Generator().manual_seed(17))


def params(grads):
    ps = []
    for g in grads:
        p = torch.empty_like(g)
        p.grad = g
        ps.append(p)
    return ps


@pytest.mark.parametrize("pieces", APART)
def test_pieces_apart(pieces, no_fallback):
    if "types" in pieces:  # whole values of both types
        host = buffer()
        host[:, 10:] = torch.cat((buffer(), buffer().flip(0)), 1)[:, :40].to(BF16).view(torch.float32)
    else:
        host = buffer()
    dev = host.to("supa")
    parts, want = APART[pieces](dev), host.clone()
    before = [t.double() for t in APART[pieces](host)]
    norm = sum(float((t * t).sum()) for t in before) ** 0.5
    got = float(torch.supa.clip_grad_norm_(params(parts), norm / 2))
    assert abs(got - norm) <= norm * (2.0 ** -24 + 1e-12)
    for t, b in zip(parts, before):
        scaled = b * (0.5 * norm / (norm + 1e-6))
        tol = scaled.abs() * (torch.finfo(t.dtype).eps / 2 + 3 * 2.0 ** -24)
        assert ((t.double().cpu() - scaled).abs() <= tol).all()
    # the rest of the buffer is as it was
    for t in APART[pieces](want):
        t.zero_()
    after = dev.cpu()
    for t in APART[pieces](after):
        t.zero_()
    assert torch.equal(after, want)


@pytest.mark.parametrize("pieces", SHARED)
def test_pieces_that_share(pieces, no_fallback):
    dev = buffer().to("supa")
    before = dev.cpu()
    for parts in (SHARED[pieces](dev), SHARED[pieces](dev)[::-1]):
        with pytest.raises(RuntimeError, match="share memory"):
            torch.supa.clip_grad_norm_(params(parts), 0.1)
    assert torch.equal(dev.cpu(), before)
