"""The operators on rows of logits in NumPy, one row at a time, in 64 bits.

Written from the definitions, for the tests: ``top`` (largest log-probabilities),
``sample`` (one token from a uniform number) and ``distill`` (loss and gradient against
a teacher's record). A logit is whatever its type holds; NaN and infinities as documented in
``include/warpshift_b200.h``.
"""

from __future__ import annotations

import math

import numpy as np


def order(row: np.ndarray) -> np.ndarray:
    """Ids of the logits above -inf (and not NaN), by logit descending, then id ascending."""
    ids = np.nonzero(row > -np.inf)[0]
    return ids[np.lexsort((ids, -row[ids]))]


def log_softmax(row: np.ndarray, temperature: float) -> np.ndarray:
    row = row.astype(np.float64)
    if np.isnan(row).any() or (row == np.inf).any():
        return np.full(row.shape, np.nan)
    if not row.size or row.max() == -np.inf:
        return np.full(row.shape, -np.inf)
    z = (row - row.max()) / temperature
    return z - math.log(np.exp(z).sum())


def top(row: np.ndarray, k: int, temperature: float) -> tuple[np.ndarray, np.ndarray]:
    ids, logp = order(row)[:k], log_softmax(row, temperature)
    fill = np.nan if np.isnan(logp).any() else -np.inf
    return (np.concatenate([ids, np.full(k - ids.size, -1, np.int64)]),
            np.concatenate([logp[ids], np.full(k - ids.size, fill)]))


def sample(row: np.ndarray, uniform: float, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
           min_p: float = 0.0) -> tuple[int, float]:
    """Token and its log-probability; the settings as the fp32 numbers that the library gets."""
    row = row.astype(np.float64)
    temperature, top_p, min_p, uniform = (float(np.float32(v)) for v in (temperature, top_p, min_p, uniform))
    ids = order(row)
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    logp = log_softmax(row, temperature)
    if not ids.size:
        return -1, math.nan if np.isnan(row).any() else -math.inf
    best = row[ids[0]]
    with np.errstate(invalid="ignore"):
        weight = np.where(row[ids] == best, 1.0, np.exp((row[ids] - best) / temperature))
    if top_k > 0:
        ids, weight = ids[:top_k], weight[:top_k]
    if not top_p > 0:
        ids, weight = ids[:1], weight[:1]
    elif top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(weight)[:-1]])
        kept = before < top_p * weight.sum()
        ids, weight = ids[kept], weight[kept]
    if min_p > 0:
        kept = weight >= min(min_p, 1.0)
        ids, weight = ids[kept], weight[kept]
    by_id = np.argsort(ids)
    cumulative = np.cumsum(weight[by_id])
    at = np.nonzero(cumulative > uniform * cumulative[-1])[0]
    token = int(ids[by_id][at[0] if at.size else -1])
    return token, float(logp[token])


def distill(row: np.ndarray, ids: np.ndarray, logprobs: np.ndarray, weight: float = 1.0, temperature: float = 1.0,
            tail: str = "drop", grad_out: float = 1.0) -> tuple[float, np.ndarray]:
    """Loss of one row and its gradient with respect to the row."""
    row = row.astype(np.float64)
    grad = np.zeros(row.shape)
    there = (ids >= 0) & (ids < row.size) & (logprobs > -np.inf)
    ids, logq = ids[there], logprobs[there].astype(np.float64)
    if weight == 0 or not ids.size:
        return 0.0, grad
    if row.max() == -np.inf:
        return weight * math.inf, grad
    if tail == "renormalize":
        logq = logq - (math.log(np.exp(logq - logq.max()).sum()) + logq.max())
    q = np.exp(logq)
    logp = log_softmax(row, temperature)
    loss = weight * float(np.sum(q * (logq - logp[ids])))
    grad = q.sum() * np.exp(logp)
    np.subtract.at(grad, ids, q)
    return loss, grad * (weight * grad_out / temperature)
