"""Inputs and error bounds shared by the tests of the operators on rows of logits."""

from __future__ import annotations

import numpy as np
import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def host(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().double().numpy()


def peaked(rows: int, vocab: int, dtype: torch.dtype, seed: int, device="cuda", scale: float = 1.5) -> torch.Tensor:
    """Rows like a language model's: noise, and a few tokens that stand out."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    n = min(vocab, 24)
    ids = torch.argsort(torch.rand(rows, min(vocab, 4096), generator=g), dim=1)[:, :n] * (vocab // min(vocab, 4096))
    x.scatter_(1, ids, 8 + 8 * torch.rand(rows, 1, generator=g) - 0.4 * torch.arange(n) + torch.rand(rows, n, generator=g))
    return x.to(dtype).to(device)


def sum_error(vocab: int) -> float:
    """Relative error of S = sum 2^(d c): the exponential's own 2^-22; its exponent's, three roundings of 2^-24 on at
    most 40 (terms below 2^-40 of the largest add up to less than 2^-20, and their error to nothing); and the additions, one
    rounding each on the longest chain (a thread's share of the row, then those of lanes, warps and blocks)."""
    return 2.0**-22 + 40 * 3 * 2.0**-24 * np.log(2) + (vocab / 256 + 64) * 2.0**-24


def logprob_bound(logp: np.ndarray, vocab: int) -> np.ndarray:
    """Absolute error of d - log S rounded to fp32: that of log S, and one rounding each of d, of log S and of the difference,
    none of which is larger than |logp| + log V."""
    return sum_error(vocab) + 3 * 2.0**-24 * (np.abs(logp) + np.log(vocab) + 1)


def grad_bound(row, ids, logprobs, weight, temperature, tail, grad_out, dtype) -> np.ndarray:
    """Absolute error of each element of a gradient row.

    Dense part a p_i: relative error of S, of the exponential, three roundings on the exponent |d| and six on factors.
    Record part b q_j, added up over equal ids: relative 2^-22 for the exponential and one rounding for each entry and
    factor. Then one rounding to the type, and what lies below its smallest step or fp32's smallest normal number."""
    row = row.astype(np.float64)
    there = (ids >= 0) & (ids < row.size) & (logprobs > -np.inf)
    if weight == 0 or not there.any() or not np.isfinite(row.max()):
        return np.zeros(row.shape)
    q = np.exp(logprobs[there].astype(np.float64))
    if tail == "renormalize":
        q = q / q.sum()
    d = np.where(np.isfinite(row), row - row.max(), 0.0) / temperature
    p = np.where(np.isfinite(row), np.exp(d), 0.0)
    p = p / p.sum()
    a = abs(weight * grad_out / temperature)
    bound = a * q.sum() * p * (sum_error(row.size) + 2.0**-22 + (3 * np.abs(d) + 6) * 2.0**-24)
    part = np.zeros(row.shape)
    np.add.at(part, ids[there], q)
    bound += a * part * (2.0**-22 + (ids.size + 6) * 2.0**-24)
    exact = a * np.abs(q.sum() * p - part)
    info = torch.finfo(dtype)
    step = info.smallest_normal * info.eps  # of the subnormal numbers
    return bound + (exact + bound) * info.eps / 2 + step + 2.0**-126
