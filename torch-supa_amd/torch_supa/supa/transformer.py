"""Operators of a transformer between its matrix products and in its optimizer
step, with no aten name: the gated residual with the norms around it, rotary
positions, and the clipping of the global gradient norm.

They run on the tensors' device, on its current stream, without waiting for
it; a wrong argument raises before anything is launched.
"""
from __future__ import annotations

import math

import torch

_residual_norm = torch.ops.supa.residual_norm.default
_rotary_embedding = torch.ops.supa.rotary_embedding.default
_rotary_embedding_ = torch.ops.supa.rotary_embedding_.default
_clip_grad_norm_ = torch.ops.supa.clip_grad_norm_.default

_NORMS = {None: 0, "none": 0, "rms": 1, "layer": 2}
_LAYOUTS = {"half": False, "interleaved": True}


def _norm_kind(name, value):
    try:
        return _NORMS[value]
    except (KeyError, TypeError):
        raise ValueError(f"residual_norm: expected {name} 'rms', 'layer' or None, got {value!r}") from None


def _number(name, value):
    """value; a tensor whose gradient would be lost with its conversion to a number raises."""
    if isinstance(value, torch.Tensor) and value.requires_grad and torch.is_grad_enabled():
        raise TypeError(f"{name} is a number and has no gradient, got a tensor that requires one")
    return value


def residual_norm(x, residual, *, gate=None, residual_scale=1.0, post_norm=None, post_weight=None, post_bias=None,
                  norm="rms", weight=None, bias=None, eps=1e-6):
    """Adds a block's output to the residual stream and normalises the sum for
    the next block, in one pass over memory (and one for the gradients)::

        u = post_norm(x)                        # x where post_norm is None
        h = residual_scale * residual + gate * u
        y = norm(h)                             # None where norm is None
        return h, y

    Norms run over the last dim (at most 16384 elements): ``"rms"`` is
    ``v / sqrt(mean(v^2) + eps) * weight``, ``"layer"`` is
    ``(v - mean(v)) / sqrt(var(v) + eps) * weight + bias``; weights default to
    ones, biases to zeros.

    x is float32, bfloat16 or float16, and y is of its dtype; residual has x's
    shape and its dtype or float32, and h is of residual's dtype.  gate, weights
    and biases are together of x's dtype or float32.  The gate's last dim is
    x's; its leading dims are x's first ones and then 1: ``[width]`` (one value
    a channel), ``[batch, 1, width]`` (one row a sample) or x's own shape.
    Statistics, products and the gradients' sums are float32, and y is the norm
    of h before h is rounded.

    Differentiable (once) in x, residual, gate, weights and biases;
    residual_scale and eps are numbers.
    """
    return _residual_norm(x, residual, gate, _number("residual_norm: residual_scale", residual_scale),
                          _norm_kind("post_norm", post_norm), post_weight, post_bias, _norm_kind("norm", norm), weight,
                          bias, _number("residual_norm: eps", eps))


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, slow=1.0,
                       fast=None, device="supa"):
    """The angular frequencies of `rotary_dim` / 2 pairs, ``base ** (-2 i / rotary_dim)``
    as a float64 vector on `device`, and the scale that goes with them:
    ``frequencies, scale = rotary_frequencies(...)``, both for rotary_embedding.

    scaling, for contexts `factor` times longer than the trained `original_length`:

    - ``"linear"``: every frequency divided by factor.
    - ``"ntk"``: the base times ``factor ** (r / (r - 2))``: the fastest pair is
      kept, the slowest divided by factor.
    - ``"smooth"``: pairs that turn fewer than `slow` times over original_length
      are divided by factor, those that turn more than `fast` (4) times kept, and
      between them the two are mixed linearly in the number of turns.
    - ``"yarn"``: the same between `slow` and `fast` (32) turns, linearly in the
      pair's index (between whole indexes); scale is ``0.1 ln(factor) + 1``.

    scale is 1 but for ``"yarn"``."""
    r = int(rotary_dim)
    if r < 2 or r % 2 or r != rotary_dim:
        raise ValueError(f"rotary_frequencies: expected an even rotary_dim >= 2, got {rotary_dim}")
    if scaling not in (None, "linear", "ntk", "smooth", "yarn"):
        raise ValueError("rotary_frequencies: expected scaling None, 'linear', 'ntk', 'smooth' or 'yarn', "
                         f"got {scaling!r}")
    if not base > 1 or not factor >= 1:
        raise ValueError(f"rotary_frequencies: expected base > 1 and factor >= 1, got {base} and {factor}")
    i = torch.arange(r // 2, dtype=torch.float64)
    if scaling == "ntk":
        if r == 2:
            raise ValueError("rotary_frequencies: 'ntk' needs more than one pair")
        base = base * factor ** (r / (r - 2))
    f = torch.pow(torch.tensor(float(base), dtype=torch.float64), -2.0 * i / r)
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling in ("smooth", "yarn"):
        fast = fast if fast is not None else (4.0 if scaling == "smooth" else 32.0)
        if original_length is None or not 0 < slow < fast:
            raise ValueError(f"rotary_frequencies: {scaling!r} needs original_length and 0 < slow < fast")
        if scaling == "smooth":
            keep = (original_length * f / (2 * math.pi) - slow) / (fast - slow)
        else:
            def index(turns):  # the pair (as a real number) that turns so often over original_length
                return r * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

            lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), r - 1)
            keep = 1 - (i - lo) / max(hi - lo, 1e-3)
            scale = 0.1 * math.log(factor) + 1.0
        keep = keep.clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f.to(device), scale


def _rotary_args(name, positions, layout):
    if layout not in _LAYOUTS:
        raise ValueError(f"{name}: expected layout 'half' or 'interleaved', got {layout!r}")
    if isinstance(positions, torch.Tensor):
        return positions, 0, _LAYOUTS[layout]
    if not isinstance(positions, int) or isinstance(positions, bool):
        raise TypeError(f"{name}: expected positions as a tensor or the first position as an int, got {positions!r}")
    return None, positions, _LAYOUTS[layout]


def rotary_embedding(q, k, frequencies, positions=0, *, layout="half", scale=1.0):
    """q and k (or None) with the first ``2 * len(frequencies)`` elements of
    every head turned in pairs by ``position * frequency`` and multiplied by
    scale; the elements after them are copied::

        (a, b) -> scale * (a cos - b sin, b cos + a sin)

    layout ``"half"`` pairs element i with i + len(frequencies),
    ``"interleaved"`` pairs 2i with 2i + 1.  q and k are ``[seq, heads, dim]`` or
    ``[batch, seq, heads, dim]`` of one dtype (float32, bfloat16, float16); their
    heads may differ in number, their strides are free (heads before
    positions: pass the transposed view).  frequencies is a vector (float64 as
    rotary_frequencies gives it, or narrower) of at most 512; positions an
    int64 or int32 tensor ``[seq]`` or ``[batch, seq]``, or the first of
    consecutive positions.

    Angles are formed in 64 bits; their sines and cosines are float32, within a
    few units in the last place, and so is the rotation, before the one rounding
    to q's dtype.  Differentiable in q and k.  Returns (q, k)."""
    at, offset, interleaved = _rotary_args("rotary_embedding", positions, layout)
    return _rotary_embedding(q, k, frequencies, at, offset, interleaved, _number("rotary_embedding: scale", scale), False)


def rotary_embedding_(q, k, frequencies, positions=0, *, layout="half", scale=1.0):
    """rotary_embedding in place, without gradients: q and k may be views of
    one projection (its heads contiguous in their last dim), and the elements
    that do not turn are not touched.  Returns (q, k)."""
    at, offset, interleaved = _rotary_args("rotary_embedding_", positions, layout)
    _rotary_embedding_(q, k, frequencies, at, offset, interleaved, scale, False)
    return q, k


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ in two passes over the gradients, or one
    where the norm is within max_norm: the norm (1, 2 or inf) of all gradients
    together, and every gradient times ``min(1, max_norm / (norm + 1e-6))``, in
    place.  Returns the norm as a float32 scalar (float64 where a gradient is).

    The sum is float64 and does not depend on timing.  The gradients are on one
    device, of float32, bfloat16, float16 or float64 in any mixture, and do not
    share memory (a parameter listed twice is an error; slices of one buffer may
    reach over each other); parameters without a gradient are left out.  A norm that is NaN makes every gradient NaN, one
    that is infinite makes them zero; error_if_nonfinite raises instead, before
    anything is scaled, and waits for the norm."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    return _clip_grad_norm_(grads, float(max_norm), float(norm_type), bool(error_if_nonfinite))
