"""What a resident model answers with: operators on rows of logits.

``top_logprobs`` is a teacher's record of every position, its k largest
log-probabilities with their token ids; ``sample`` draws one token from every row.
Both read the logits from HBM once, in one launch of ``libwarpshift_b200.so``
(``include/warpshift_b200.h``: ``ws_top_logprobs``, ``ws_sample``), on the current
stream of the logits' device, without waiting for it and without a workspace, so
that they can be captured into a CUDA graph.

The reference leaves both to its serving engine and compares greedy tokens and
log-probabilities of a switched model with those of a natively loaded one on the
host (``scripts/validate.py:142-155``); ``verify.answer_record`` does that on the GPU.
"""

from __future__ import annotations

from ctypes import byref
from typing import NamedTuple

import torch

from warpshift_b200 import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # WS_DTYPE_*


class TopLogprobs(NamedTuple):
    """``ids`` [..., k] int64 and ``logprobs`` [..., k] fp32, largest first."""

    ids: torch.Tensor
    logprobs: torch.Tensor


class Sampled(NamedTuple):
    """``tokens`` [...] int64 and ``logprobs`` [...] fp32."""

    tokens: torch.Tensor
    logprobs: torch.Tensor


def rows_of(tensor: torch.Tensor, name: str = "logits") -> _lib.Rows:
    """The rows of ``tensor`` [..., V] for the library: no copy, whatever the leading strides,
    as long as the leading dimensions come down to two."""
    dtype = _DTYPES.get(tensor.dtype)
    if dtype is None:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, not {tensor.dtype}")
    shape, strides = tensor.shape, tensor.stride()
    if not shape:
        raise ValueError(f"{name} needs a dimension for the vocabulary")
    vocab = shape[-1]
    if not 1 <= vocab <= _lib.WS_MAX_VOCAB:
        raise ValueError(f"{name} has {vocab} elements a row: 1 to {_lib.WS_MAX_VOCAB} are possible")
    if vocab > 1 and strides[-1] != 1:
        raise ValueError(f"{name} must be contiguous in the last dimension")
    if len(shape) == 2:
        return _lib.Rows(tensor.data_ptr(), shape[0], shape[0] or 1, 0, strides[0], vocab, dtype, 0)
    rows = 1
    dims = []  # (size, stride) of the leading dimensions, those that continue one another joined
    for size, stride in zip(shape[:-1], strides[:-1]):
        rows *= size
        if size == 1:
            continue
        if dims and dims[-1][1] == size * stride:
            dims[-1] = (dims[-1][0] * size, stride)
        else:
            dims.append((size, stride))
    if rows == 0:
        dims = []
    if len(dims) > 2:
        raise ValueError(f"{name} has leading dimensions of more than two strides: make it contiguous")
    inner, stride_inner = dims[-1] if dims else (1, 0)
    stride_outer = dims[0][1] if len(dims) == 2 else 0
    return _lib.Rows(tensor.data_ptr(), rows, inner, stride_outer, stride_inner, vocab, dtype, 0)


def per_row(value: torch.Tensor, name: str, like: torch.Tensor, dtypes: tuple[torch.dtype, ...]) -> torch.Tensor:
    """Checks a tensor with one value for each row of ``like``; without gaps."""
    if value.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}, not {value.dtype}")
    if value.shape != like.shape[:-1]:
        raise ValueError(f"{name} has shape {tuple(value.shape)}: the rows have {tuple(like.shape[:-1])}")
    if value.device != like.device:
        raise ValueError(f"{name} is on {value.device}, the rows on {like.device}")
    return value if value.is_contiguous() else value.contiguous()


def device_of(tensor: torch.Tensor) -> int:
    """The index of the CUDA device of ``tensor``; there is no other path."""
    if not tensor.is_cuda:
        raise ValueError(f"logits must be on a CUDA device, not {tensor.device}")
    return tensor.get_device()


def stream_of(index: int) -> int:
    """The current stream of a CUDA device, as an address (``torch.cuda.current_stream`` without the Stream object,
    which takes 2 us: these calls are as short as 10)."""
    return torch._C._cuda_getCurrentRawStream(index)


def top_logprobs(logits: torch.Tensor, k: int, *, temperature: float = 1.0) -> TopLogprobs:
    """The ``k`` largest logits of every row as log-probabilities of ``softmax(logits / temperature)``.

    ``logits`` [..., V], bf16, fp16 or fp32, V up to 2^20; 1 <= k <= min(V, 256). Largest first; among
    equal logits the lowest id. Logits of -inf have no place in a record: where a row
    has fewer than k others, it ends with id -1 and log-probability -inf. A NaN logit is passed over and makes
    its row's log-probabilities NaN, as +inf does. No gradient flows through the result.
    """
    rows = rows_of(logits)
    if not 1 <= k <= min(rows.vocab, _lib.WS_TOP_MAX_K):
        raise ValueError(f"k is {k}: 1 to {min(rows.vocab, _lib.WS_TOP_MAX_K)} are possible")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be from 1e-6 to 1e6, not {temperature}")
    index = device_of(logits)
    shape = (*logits.shape[:-1], k)
    ids = logits.new_empty(shape, dtype=torch.int64)
    logprobs = logits.new_empty(shape, dtype=torch.float32)
    _lib.check(_lib.load().ws_top_logprobs(byref(rows), k, temperature, ids.data_ptr(), logprobs.data_ptr(), index, stream_of(index)))
    return TopLogprobs(ids, logprobs)


def sample(
    logits: torch.Tensor,
    uniform: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
) -> Sampled:
    """Draw one token from every row of ``logits`` [..., V] with the numbers ``uniform`` [...] (fp32, in [0, 1)).

    Each setting is one number or a tensor with a value for each row (fp32; ``top_k`` int32 or
    int64). With tokens ordered by logit (largest first, among equals the lowest id) and weights
    ``w = exp((x - max x) / temperature)``: ``top_k`` keeps the first that many (0: all), ``top_p`` of these the
    shortest run with at least that share of their weight, ``min_p`` of these the ones with ``w >= min_p``. The token
    drawn is the first one by id whose cumulative weight among those kept exceeds ``uniform`` times
    their total. The same inputs give the same tokens: borders are decided in 64-bit arithmetic. ``temperature`` 0 takes the
    largest logit.

    A row without a logit above -inf gives token -1. ``logprobs`` is the token's log-probability under
    ``softmax(logits / temperature)`` of the whole row (at temperature 1 where it is 0).
    """
    rows = rows_of(logits)
    uniform = per_row(uniform, "uniform", logits, (torch.float32,))
    keep = []  # tensors that the call reads

    def each(value, name, dtypes=(torch.float32,)):
        if isinstance(value, torch.Tensor):
            keep.append(per_row(value, name, logits, dtypes))
            return keep[-1].data_ptr(), 0
        return None, value

    temperature_each, temperature = each(temperature, "temperature")
    top_p_each, top_p = each(top_p, "top_p")
    min_p_each, min_p = each(min_p, "min_p")
    wide = isinstance(top_k, torch.Tensor) and top_k.dtype == torch.int64
    top_k_each, top_k = each(top_k, "top_k", (torch.int32, torch.int64))
    top_k = min(max(top_k, 0), _lib.WS_MAX_VOCAB)
    index = device_of(logits)
    settings = _lib.Sampling(temperature_each, top_p_each, min_p_each, top_k_each, top_k, temperature, top_p, min_p, wide)
    shape = logits.shape[:-1]
    tokens = logits.new_empty(shape, dtype=torch.int64)
    logprobs = logits.new_empty(shape, dtype=torch.float32)
    _lib.check(_lib.load().ws_sample(byref(rows), uniform.data_ptr(), byref(settings), tokens.data_ptr(), logprobs.data_ptr(),
                                     index, stream_of(index)))
    return Sampled(tokens, logprobs)
