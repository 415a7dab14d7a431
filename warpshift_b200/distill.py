"""A student's loss against a teacher's record, and its gradient.

The record is what ``logits.top_logprobs`` gives for the teacher's logits: for every
position k token ids and their log-probabilities. With q the record's probabilities,
p = softmax(x / temperature) of the student's logits x and w a weight for each row,

    loss = w * sum_j q_j (log q_j - log p[id_j])

and with Q = sum_j q_j and g the gradient that comes in,

    d loss / d x_i = g w / temperature * (Q p_i - sum of q_j over the j with id_j = i).

``tail="drop"`` takes the record's probabilities as they are (Q < 1: what lies outside the record is left
out), ``tail="renormalize"`` divides them by their sum. Entries with an id outside [0, V) or a log-probability
of -inf carry no mass, a token that comes twice counts twice; a row whose weight is 0 is not even read.

``top_logprob_loss`` goes through autograd (``ws_distill_forward``, ``ws_distill_backward``): the logits are read
twice and the gradient is written once. Where the gradient that comes in is 1 for every row (weights carry all
scaling), ``top_logprob_loss_and_grad`` (``ws_distill_step``) gives both in one launch.
"""

from __future__ import annotations

from ctypes import byref

import torch

from warpshift_b200 import _lib
from warpshift_b200.logits import device_of, per_row, rows_of, stream_of


def _record(logits, ids, logprobs, weights, temperature, tail):
    """The library's view of a record, and the tensors that it points into."""
    if tail not in _lib.TAILS:
        raise ValueError(f"Unknown tail: {tail}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32, not {ids.dtype}")
    if logprobs.dtype != torch.float32:
        raise ValueError(f"logprobs must be float32, not {logprobs.dtype}")
    if logprobs.requires_grad or (weights is not None and weights.requires_grad):
        raise ValueError("the teacher's record and the weights are constants: detach them")
    if ids.shape != logprobs.shape or ids.dim() != logits.dim() or ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"ids {tuple(ids.shape)} and logprobs {tuple(logprobs.shape)} must be [..., k] with the rows of "
                         f"logits {tuple(logits.shape)}")
    k = ids.shape[-1]
    if not 1 <= k <= _lib.WS_TOP_MAX_K:
        raise ValueError(f"a record has {k} entries a row: 1 to {_lib.WS_TOP_MAX_K} are possible")
    if ids.device != logits.device or logprobs.device != logits.device:
        raise ValueError(f"the record is on {ids.device} and {logprobs.device}, the logits on {logits.device}")
    ids, logprobs = ids.contiguous(), logprobs.contiguous()
    if weights is not None:
        weights = per_row(weights, "weights", logits, (torch.float32,))
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be from 1e-6 to 1e6, not {temperature}")
    return _teacher(ids, logprobs, weights, temperature, tail), (ids, logprobs, weights)


def _teacher(ids, logprobs, weights, temperature, tail):
    return _lib.Teacher(ids.data_ptr(), logprobs.data_ptr(), None if weights is None else weights.data_ptr(), ids.shape[-1],
                        ids.dtype == torch.int32, _lib.TAILS[tail], temperature)


def _grad_like(logits: torch.Tensor, rows: _lib.Rows) -> torch.Tensor:
    """Room for the gradient. Rows that lie a little apart (a padded vocabulary) stay so: a gradient row on the same
    offset from a 16-byte boundary as its logits is written with the widest stores."""
    if logits.dim() == 2 and rows.vocab < rows.stride_inner <= rows.vocab + rows.vocab // 8:
        return logits.new_empty((rows.rows, rows.stride_inner))[:, : rows.vocab]
    return logits.new_empty(logits.shape)


def _backward(ctx, grad_loss):
    logits, ids, logprobs, weights, stats = ctx.saved_tensors
    # Anew from the saved tensors: hooks on them (offloading, say) may have put them elsewhere.
    rows = rows_of(logits)
    record = _teacher(ids, logprobs, weights, *ctx.settings)
    # One g for each row by the strides of the logits' two row dimensions; a sum's or a mean's gradient has strides of 0.
    if grad_loss.dtype != torch.float32:
        grad_loss = grad_loss.float()
    if logits.dim() == 2:
        outer, inner = 0, grad_loss.stride(0)
    elif all(s == 0 for s in grad_loss.stride()):
        outer = inner = 0
    else:
        grad_loss = grad_loss.contiguous()
        outer, inner = rows.inner, 1
    grad = _grad_like(logits, rows)
    out = rows_of(grad, "gradient")
    index = logits.get_device()
    _lib.check(_lib.load().ws_distill_backward(byref(rows), byref(record), stats.data_ptr(), grad_loss.data_ptr(), outer, inner,
                                               byref(out), index, stream_of(index)))
    if torch.is_grad_enabled():  # under create_graph
        grad = _Once.apply(grad, logits)
    return grad, None, None, None, None, None


class _Once(torch.autograd.Function):
    """A gradient that is not to be differentiated again, with respect to the logits it is a function of."""

    @staticmethod
    def forward(ctx, grad, logits):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("top_logprob_loss can be differentiated once")


class _TopLogprobLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, logprobs, weights, temperature, tail):
        rows = rows_of(logits)
        record, (ids, logprobs, weights) = _record(logits, ids, logprobs, weights, temperature, tail)
        index = device_of(logits)
        loss = logits.new_empty(logits.shape[:-1], dtype=torch.float32)
        stats = logits.new_empty((rows.rows, _lib.WS_DISTILL_STATS), dtype=torch.float32)
        _lib.check(_lib.load().ws_distill_forward(byref(rows), byref(record), loss.data_ptr(), stats.data_ptr(), index,
                                                  stream_of(index)))
        ctx.save_for_backward(logits, ids, logprobs, weights, stats)
        ctx.settings = temperature, tail
        return loss

    backward = staticmethod(_backward)


def top_logprob_loss(
    logits: torch.Tensor,
    ids: torch.Tensor,
    logprobs: torch.Tensor,
    *,
    weights: torch.Tensor | None = None,
    temperature: float = 1.0,
    tail: str = "drop",
) -> torch.Tensor:
    """The loss of every row of ``logits`` [..., V] against the record ``ids``, ``logprobs`` [..., k], as fp32 [...].

    ``logits``: bf16, fp16 or fp32; rows may lie apart (``logits[:, :-1]`` is read where it is). ``ids``: int64 or
    int32, ``logprobs``: fp32, k up to 256. ``weights`` [...] fp32: 0 for rows that do not count. Differentiable once, in
    ``logits`` alone; the gradient has their type. A token of the record whose logit is -inf makes its row's
    loss +inf; a row without any finite logit has no gradient.
    """
    return _TopLogprobLoss.apply(logits, ids, logprobs, weights, temperature, tail)


def top_logprob_loss_and_grad(
    logits: torch.Tensor,
    ids: torch.Tensor,
    logprobs: torch.Tensor,
    *,
    weights: torch.Tensor | None = None,
    temperature: float = 1.0,
    tail: str = "drop",
) -> tuple[torch.Tensor, torch.Tensor]:
    """``top_logprob_loss`` and the gradient of its sum with respect to ``logits``, in one launch.

    Arguments as there. For a training loop that goes on with ``hidden.backward(...)`` or ``logits.backward(grad)``
    and puts its scaling (a mean's 1/n, the rows that count) into ``weights``.
    """
    rows = rows_of(logits)
    record, keep = _record(logits, ids, logprobs, weights, temperature, tail)
    index = device_of(logits)
    loss = logits.new_empty(logits.shape[:-1], dtype=torch.float32)
    grad = _grad_like(logits, rows)
    out = rows_of(grad, "gradient")
    _lib.check(_lib.load().ws_distill_step(byref(rows), byref(record), loss.data_ptr(), byref(out), index, stream_of(index)))
    return loss, grad
