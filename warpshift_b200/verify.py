"""Acceptance checks of a switched model, computed on the GPU.

``tensor_hashes``: per-tensor content hashes.

The reference's acceptance check (``scripts/validate.py:32-83``, the
``check_weights`` test loader) proves that a switched model equals a native load
by hashing every tensor with sha256 after copying it to the host in 64 MiB
pieces (``validate.py:50-56``). ``tensor_hashes`` gives the same per-tensor
verdict from one HBM-bound pass over the resident bytes: a 64-bit hash per
tensor (definition in ``include/warpshift_b200.h``), returned as 16 hex digits.
Equal bytes give equal hashes; any change of a tensor's bytes changes its hash
except with probability about 2^-64. It is a checksum against accidental
corruption, not a cryptographic digest.

``answer_record`` and ``compare_answers``: the reference's other check, that a switched
model's greedy tokens and log-probabilities equal those of a native load within 1e-3
(``validate.py:142-155``), on the logits themselves.
"""

from __future__ import annotations

import ctypes
from collections.abc import Mapping
from typing import Any

import torch

from warpshift_b200 import _lib
from warpshift_b200.logits import top_logprobs


def tensor_hashes(tensors: Mapping[str, torch.Tensor]) -> dict[str, str]:
    """Hash each CUDA tensor's bytes (row-major, as ``validate.py:51`` flattens them).

    Non-contiguous tensors are hashed through a contiguous copy. Raises
    ``ValueError`` for tensors that are not on a CUDA device.
    """
    lib = _lib.load()
    names = list(tensors)
    out: dict[str, str] = {}
    by_device: dict[int, list[str]] = {}
    for name in names:
        t = tensors[name]
        if t.device.type != "cuda":
            raise ValueError(f"tensor_hashes needs CUDA tensors; {name} is on {t.device}")
        by_device.setdefault(t.device.index, []).append(name)
    for device, group in by_device.items():
        keep = []
        ptrs = (ctypes.c_void_p * len(group))()
        sizes = (ctypes.c_uint64 * len(group))()
        for i, name in enumerate(group):
            t = tensors[name].detach()
            if not t.is_contiguous():
                t = t.contiguous()
            keep.append(t)
            ptrs[i] = t.data_ptr()
            sizes[i] = t.numel() * t.element_size()
        result = (ctypes.c_uint64 * len(group))()
        with torch.cuda.device(device):
            stream = torch.cuda.current_stream(device).cuda_stream
            _lib.check(lib.ws_tensor_hashes(ptrs, sizes, len(group), device, stream, result))
        for i, name in enumerate(group):
            out[name] = f"{result[i]:016x}"
    return {name: out[name] for name in names}


def answer_record(logits: torch.Tensor, k: int = 20) -> dict[str, Any]:
    """What the resident model answers with: the ``k`` top log-probabilities of every row of ``logits`` [..., V] and
    their token ids, the greedy token first, as lists (``json.dump`` takes them)."""
    top = top_logprobs(logits, k)
    return {"ids": top.ids.tolist(), "logprobs": top.logprobs.tolist()}


def compare_answers(expected: Mapping[str, Any], actual: Mapping[str, Any], atol: float = 1e-3) -> list[str]:
    """Where two records differ, one line a row; empty if they agree.

    Rows agree if their greedy tokens are equal and their log-probabilities lie within ``atol``, the largest against the
    largest and so on (tokens of nearly equal probability may change places).
    """
    ids = [torch.as_tensor(r["ids"], dtype=torch.int64) for r in (expected, actual)]
    logprobs = [torch.as_tensor(r["logprobs"], dtype=torch.float64) for r in (expected, actual)]
    if ids[0].shape != ids[1].shape or any(p.shape != ids[0].shape for p in logprobs):
        raise ValueError("Answer records have different shapes")
    k = ids[0].shape[-1]
    ids, logprobs = ([t.reshape(-1, k) for t in pair] for pair in (ids, logprobs))
    differences = []
    for row in range(ids[0].shape[0]):
        greedy = int(ids[0][row, 0]), int(ids[1][row, 0])
        if greedy[0] != greedy[1]:
            differences.append(f"row {row}: greedy token {greedy[1]}, expected {greedy[0]}")
        elif not torch.allclose(logprobs[1][row], logprobs[0][row], rtol=0, atol=atol):
            off = (logprobs[1][row] - logprobs[0][row]).abs().max().item()
            differences.append(f"row {row}: log-probabilities differ by up to {off:.3g}")
    return differences
