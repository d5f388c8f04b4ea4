"""Operators on rows of logits with no aten name, beside the losses and the
softmax: distillation from a teacher's top logits, the balance loss of a
mixture's router, and what a server does to logits before it draws a token.

They run on the tensors' device, on its current stream, without waiting for
it; a wrong argument raises before anything is launched.
"""
from __future__ import annotations

import torch

from .transformer import _number

_distillation_loss = torch.ops.supa.distillation_loss.default
_router_balance_loss = torch.ops.supa.router_balance_loss.default
_adjust_logits = torch.ops.supa.adjust_logits.default
_adjust_logits_ = torch.ops.supa.adjust_logits_.default

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_SCORES = {"softmax": 0, "sigmoid": 1}


def _choice(name, value, choices):
    try:
        return choices[value]
    except (KeyError, TypeError):
        raise ValueError(f"{name}: expected {' or '.join(map(repr, choices))}, got {value!r}") from None


def distillation_loss(logits, indices, teacher_logits, *, teacher_lse=None, temperature=1.0, reduction="mean"):
    """The Kullback-Leibler divergence of a student from a teacher of whom each
    row stores the best tokens only, one read of the logits forward and one read
    and one write backward::

        q = softmax(logits / temperature)
        p = exp(teacher_logits / temperature - lse)
        loss = sum(p * (log(p) - log(q[indices])))

    temperature is a number.  logits are ``[..., vocab]`` of float32, bfloat16 or float16, indices (int64 or
    int32) and teacher_logits (any of the three types) ``[..., k]`` with k up to 1024;
    their order does not matter.  A pair with a negative index, or a teacher's
    logit of -inf, is not there: rows may store fewer than k.  A row without any has
    loss 0 and gradient 0, and does not count for the mean, which is NaN where no row
    counts.  A token that is listed twice is listed once for the student, and its gradient has the
    sum of its p; the loss adds up the pairs, each with its own log(p): it is less by p1 log(P / p1) + p2 log(P / p2)
    than that of one pair with P = p1 + p2.

    Without teacher_lse, lse is that of the row's own teacher_logits: p sums to 1 over
    the listed tokens.  teacher_lse (floats ``[...]``; float64 is taken as it is) is the
    log-sum-exp of all of the teacher's logits over temperature; the tokens that are not listed then are one more
    class, with r = 1 - sum(p) of the teacher's mass (at least 0)::

        loss += r * (log(r) - log(sum of q over the tokens that are not listed))

    The loss is float32: a scalar for reduction ``"mean"`` (over the rows that count) or
    ``"sum"``, ``[...]`` for ``"none"``.  It is not multiplied by temperature ** 2.
    Exponentials of the logits are summed in float32, in an order that the sizes and the alignment of a row fix, what depends on
    the listed pairs is float64.  Differentiable (once) in logits; the teacher is a constant.  An index of vocab
    and more, in a pair that is there, raises an IndexError when the stream is next waited for, as cross_entropy's
    targets do."""
    return _distillation_loss(logits, indices, teacher_logits, teacher_lse,
                              _number("distillation_loss: temperature", temperature),
                              _choice("distillation_loss: reduction", reduction, _REDUCTIONS))


def router_balance_loss(logits, experts, *, mask=None, scores="softmax", per_sequence=False):
    """The loss that keeps a mixture's experts equally busy, and how often each was
    chosen: ``loss, counts = router_balance_loss(...)``::

        p = softmax(logits)             # or sigmoid(logits) / sum(sigmoid(logits))
        load = counts * num_experts / (k * tokens)
        loss = sum(load * mean of p over the tokens)

    which is 1 for tokens spread evenly.  logits are the router's, ``[..., num_experts]``
    of float32, bfloat16 or float16 (at most 1024 experts); experts (int64 or int32)
    ``[..., k]`` those that each token was sent to, negative where one was dropped.
    mask (bools ``[...]``) is False for tokens that do not count, as padding; their gradient is 0.
    With per_sequence, logits are ``[..., tokens, num_experts]``, every sequence has a loss and counts
    of its own, and loss is the mean over the sequences with a counted token.  It is 0 where
    no token counts.

    loss is a float32 scalar, counts are int64: ``[num_experts]``, or ``[..., num_experts]`` for
    each sequence.  Sums are float32 within a workgroup and float64 from there on, in an order
    that only the sizes fix.  Differentiable (once) in logits, the counts being constants.  An expert of num_experts
    and more raises an IndexError when the stream is next waited for."""
    return _router_balance_loss(logits, experts, mask, _choice("router_balance_loss: scores", scores, _SCORES),
                                bool(per_sequence))


def _per_row(value, default):
    """(tensor, number) of a parameter that is either."""
    return (value, default) if isinstance(value, torch.Tensor) else (None, float(value))


def _adjust(op, logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias_tokens, bias, allowed):
    return op(logits, tokens, lengths, prompt_lengths, *_per_row(repetition, 1.0), *_per_row(presence, 0.0),
              *_per_row(frequency, 0.0), bias_tokens, bias, allowed)


def adjust_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0,
                  frequency=0.0, bias_tokens=None, bias=None, allowed=None):
    """Logits as they are before a token is drawn from them, in one pass::

        x / repetition if x > 0 else x * repetition     # tokens of the history
        x - frequency * count - presence * (count > 0)  # count: times behind the prompt
        x + bias                                        # at bias_tokens
        -inf                                            # tokens that are not allowed

    logits are ``[rows, vocab]`` or ``[vocab]`` of float32, bfloat16 or float16.  tokens (int64 or
    int32, ``[rows, n]``, for a single row ``[n]``) is the history: of each row the first ``lengths[row]``
    (all of them by default), of which the first ``prompt_lengths[row]`` (none) are the prompt.
    repetition, presence and frequency are numbers or float32 ``[rows]``.  bias_tokens and bias
    (float32) are ``[rows, m]``, or ``[m]`` for all rows; several biases of a token add up.  allowed is
    int32 ``[rows, words]``, or ``[words]`` for all rows: bit ``v % 32`` of word ``v // 32`` is set where token v may
    follow; a row that allows nothing is -inf throughout.  Tokens outside [0, vocab) are passed over.

    Everything is float32 and rounded once.  No gradient.  Returns new logits; adjust_logits_ works in place."""
    return _adjust(_adjust_logits, logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias_tokens,
                   bias, allowed)


def adjust_logits_(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0,
                   frequency=0.0, bias_tokens=None, bias=None, allowed=None):
    """adjust_logits in place, for logits whose rows are contiguous and share no memory with the
    other arguments.  Returns logits."""
    _adjust(_adjust_logits_, logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias_tokens,
            bias, allowed)
    return logits
