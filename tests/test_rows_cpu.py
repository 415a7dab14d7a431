"""The operators on rows of logits without a GPU: the oracle's own properties, and every refusal."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import rows as oracle
from warpshift_b200 import _lib, distill, logits as ops, verify

RNG = np.random.default_rng(5)


# --------------------------------------------------------------------------- the oracle
def test_oracle_top_orders_by_logit_then_id() -> None:
    ids, logp = oracle.top(np.array([1.0, 3.0, -np.inf, 3.0, 2.0]), 5, 1.0)
    assert ids.tolist() == [1, 3, 4, 0, -1] and logp[-1] == -np.inf
    assert abs(np.exp(logp[:4]).sum() - 1) < 1e-15


def test_oracle_sample_takes_each_token_by_its_share() -> None:
    row = np.log(np.array([0.1, 0.2, 0.3, 0.4]))
    draw = lambda u, **p: oracle.sample(row, u, **p)[0]  # noqa: E731
    assert [draw(u) for u in (0.0, 0.0999, 0.1001, 0.2999, 0.3001, 0.5999, 0.6001, 0.9999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [draw(u, top_k=2) for u in (0.0, 0.42, 0.43, 0.99)] == [2, 2, 3, 3]
    assert {draw(u, top_p=0.39) for u in (0.0, 0.5, 0.99)} == {3}
    assert {draw(u, top_p=0.41) for u in (0.0, 0.99)} == {2, 3}
    assert {draw(u, min_p=0.49) for u in (0.0, 0.3, 0.99)} == {1, 2, 3}
    assert {draw(u, temperature=0.0) for u in (0.0, 0.5, 0.99)} == {3}
    assert oracle.sample(np.full(3, -np.inf), 0.5)[0] == -1


@pytest.mark.parametrize("tail", ["drop", "renormalize"])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
def test_oracle_gradient_against_differences(tail, temperature) -> None:
    row = RNG.standard_normal(40)
    ids = np.array([3, 3, 17, -1, 39, 50])
    logq = np.log(np.array([0.2, 0.1, 0.3, 0.1, 0.15, 0.1]))
    _, grad = oracle.distill(row, ids, logq, 0.7, temperature, tail, 1.3)
    h = 1e-5
    for i in range(40):
        step = np.zeros(40)
        step[i] = h
        up, down = (oracle.distill(row + s * step, ids, logq, 0.7, temperature, tail)[0] for s in (1, -1))
        assert abs(1.3 * (up - down) / (2 * h) - grad[i]) < 1e-8


def test_oracle_distill_against_autograd() -> None:
    x = torch.tensor(RNG.standard_normal(30), requires_grad=True)
    ids, logq = np.array([1, 5, 9]), np.log(np.array([0.5, 0.2, 0.1]))
    logp = torch.log_softmax(x / 2.0, 0)
    loss = (torch.tensor(np.exp(logq)) * (torch.tensor(logq) - logp[ids])).sum()
    loss.backward()
    want, grad = oracle.distill(x.detach().numpy(), ids, logq, 1.0, 2.0)
    assert abs(want - loss.item()) < 1e-14
    np.testing.assert_allclose(grad, x.grad.numpy(), atol=1e-15)


# --------------------------------------------------------------------------- refusals of the Python API
X = torch.zeros(2, 10)


@pytest.mark.parametrize("call", [
    lambda: ops.top_logprobs(X.double(), 1),
    lambda: ops.top_logprobs(X.long(), 1),
    lambda: ops.top_logprobs(torch.tensor(1.0), 1),
    lambda: ops.top_logprobs(X[:, :0], 1),
    lambda: ops.top_logprobs(X.t(), 1),
    lambda: ops.top_logprobs(X[:, ::2], 1),
    lambda: ops.top_logprobs(torch.zeros(1).expand(1, (1 << 20) + 1), 1),
    lambda: ops.top_logprobs(torch.zeros(4, 4, 4, 8)[::2, ::2, ::2], 1),
    lambda: ops.top_logprobs(X, 0),
    lambda: ops.top_logprobs(X, 11),
    lambda: ops.top_logprobs(torch.zeros(2, 1000), 257),
    lambda: ops.top_logprobs(X, 1, temperature=0.0),
    lambda: ops.top_logprobs(X, 1, temperature=-1.0),
    lambda: ops.top_logprobs(X, 1, temperature=math.nan),
    lambda: ops.top_logprobs(X, 1, temperature=math.inf),
    lambda: ops.sample(X, torch.zeros(3)),
    lambda: ops.sample(X, torch.zeros(2, 1)),
    lambda: ops.sample(X, torch.zeros(2).double()),
    lambda: ops.sample(X, torch.zeros(2), temperature=torch.ones(3)),
    lambda: ops.sample(X, torch.zeros(2), temperature=torch.ones(2, dtype=torch.float64)),
    lambda: ops.sample(X, torch.zeros(2), top_k=torch.ones(2)),
    lambda: ops.sample(X, torch.zeros(2), top_p=torch.ones(1)),
    lambda: ops.sample(X, torch.zeros(2), min_p=torch.tensor(0.1)),
    lambda: ops.sample(X.half().t(), torch.zeros(10)),
])
def test_python_refusals(call) -> None:
    with pytest.raises(ValueError):
        call()


IDS, LOGP = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)


@pytest.mark.parametrize("function", [distill.top_logprob_loss, distill.top_logprob_loss_and_grad])
@pytest.mark.parametrize("args,kwargs", [
    ((X.double(), IDS, LOGP), {}),
    ((X.t(), IDS, LOGP), {}),
    ((X, IDS.float(), LOGP), {}),
    ((X, IDS.short(), LOGP), {}),
    ((X, IDS, LOGP.half()), {}),
    ((X, IDS, LOGP[:, :2]), {}),
    ((X, IDS[:1], LOGP[:1]), {}),
    ((X, IDS[0], LOGP[0]), {}),
    ((X, IDS[:, :0], LOGP[:, :0]), {}),
    ((X, IDS[:, :1].expand(2, 257), LOGP[:, :1].expand(2, 257)), {}),
    ((X, IDS, LOGP.clone().requires_grad_(True)), {}),
    ((X, IDS, LOGP), {"weights": torch.ones(2, requires_grad=True)}),
    ((X, IDS, LOGP), {"weights": torch.ones(3)}),
    ((X, IDS, LOGP), {"weights": torch.ones(2).half()}),
    ((X, IDS, LOGP), {"tail": "lump"}),
    ((X, IDS, LOGP), {"temperature": 0.0}),
    ((X, IDS, LOGP), {"temperature": math.nan}),
])
def test_distill_refusals(function, args, kwargs) -> None:
    with pytest.raises(ValueError):
        function(*args, **kwargs)


def test_tensors_without_a_gpu_are_refused_last() -> None:
    for call in (lambda: ops.top_logprobs(X, 3), lambda: ops.sample(X, torch.zeros(2)),
                 lambda: distill.top_logprob_loss(X, IDS, LOGP), lambda: distill.top_logprob_loss_and_grad(X, IDS, LOGP),
                 lambda: verify.answer_record(X, 3)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


# --------------------------------------------------------------------------- refusals of the C ABI
def rows(**change) -> _lib.Rows:
    fields = {"data": 1 << 20, "rows": 2, "inner": 2, "stride_outer": 0, "stride_inner": 100, "vocab": 100, "dtype": 0, **change}
    return _lib.Rows(*(fields[n] for n in ("data", "rows", "inner", "stride_outer", "stride_inner", "vocab", "dtype")), 0)


BAD_ROWS = [{"data": None}, {"data": (1 << 20) + 1}, {"dtype": 2, "data": (1 << 20) + 2}, {"dtype": 3}, {"dtype": -1}, {"vocab": 0},
            {"vocab": (1 << 20) + 1}, {"rows": (1 << 27) + 1}, {"inner": 0}, {"stride_inner": -1}, {"stride_outer": -1}]


def teacher(**change) -> _lib.Teacher:
    fields = {"ids": 64, "logprobs": 64, "weights": None, "k": 4, "ids_are_int32": 0, "tail": 0, "temperature": 1.0, **change}
    return _lib.Teacher(*fields.values())


def all_calls(x, t=None, k=4, temperature=1.0, result=64, device=0, grad=None, stats=64, sampling=True):
    lib, t = _lib.load(), t or teacher()
    x_ref = ctypes.byref(x) if x is not None else None
    s = ctypes.byref(_lib.Sampling(temperature=1.0)) if sampling else None
    return {
        "top": lambda: lib.ws_top_logprobs(x_ref, k, temperature, result, 64, device, None),
        "sample": lambda: lib.ws_sample(x_ref, 64, s, result, None, device, None),
        "forward": lambda: lib.ws_distill_forward(x_ref, ctypes.byref(t), result, stats, device, None),
        "backward": lambda: lib.ws_distill_backward(x_ref, ctypes.byref(t), stats, result, 0, 0, ctypes.byref(grad or x), device, None),
        "step": lambda: lib.ws_distill_step(x_ref, ctypes.byref(t), result, ctypes.byref(grad or x), device, None),
    }


@pytest.mark.parametrize("change", BAD_ROWS)
def test_c_abi_refuses_bad_rows(change) -> None:
    for name, call in all_calls(rows(**change)).items():
        assert call() == _lib.WS_ERR_INVALID, name
        assert "logits" in _lib.last_error()
    calls = all_calls(rows(dtype=change.get("dtype", 0)), grad=rows(**change)) if change.get("dtype", 0) in (0, 1, 2) else {}
    for name in ("backward", "step"):
        if name in calls:
            assert calls[name]() == _lib.WS_ERR_INVALID, name


def test_c_abi_refuses_bad_arguments() -> None:
    x = rows()
    for k in (0, 101, 257):
        assert all_calls(x, k=k)["top"]() == _lib.WS_ERR_INVALID
    for t in (0.0, -1.0, math.nan, math.inf, 1e-7, 1e7):
        assert all_calls(x, temperature=t)["top"]() == _lib.WS_ERR_INVALID
        for name in ("forward", "backward", "step"):
            assert all_calls(x, teacher(temperature=t))[name]() == _lib.WS_ERR_INVALID
    for bad in ({"k": 0}, {"k": 257}, {"tail": 2}, {"tail": -1}, {"ids": None}, {"logprobs": None}):
        for name in ("forward", "backward", "step"):
            assert all_calls(x, teacher(**bad))[name]() == _lib.WS_ERR_INVALID, (bad, name)
    for name, call in all_calls(x, result=None).items():
        assert call() == _lib.WS_ERR_INVALID, name
    for name, call in all_calls(x, device=-1).items():
        assert call() == _lib.WS_ERR_INVALID, name
    assert all_calls(x, sampling=False)["sample"]() == _lib.WS_ERR_INVALID
    for stats in (None, 68):
        for name in ("forward", "backward"):
            assert all_calls(x, stats=stats)[name]() == _lib.WS_ERR_INVALID
    for other in (rows(rows=3), rows(vocab=99), rows(dtype=1)):
        for name in ("backward", "step"):
            assert all_calls(x, grad=other)[name]() == _lib.WS_ERR_INVALID
    lib = _lib.load()
    assert lib.ws_top_logprobs(None, 1, 1.0, 64, 64, 0, None) == _lib.WS_ERR_INVALID
    assert lib.ws_distill_forward(ctypes.byref(x), None, 64, 64, 0, None) == _lib.WS_ERR_INVALID


def test_c_abi_with_no_rows_does_nothing() -> None:
    for name, call in all_calls(rows(rows=0, data=None), result=None).items():
        assert call() == _lib.WS_OK, name


# --------------------------------------------------------------------------- answer records
def test_compare_answers() -> None:
    a = {"ids": [[5, 2], [7, 1]], "logprobs": [[-0.1, -3.0], [-0.5, -0.9]]}
    close = {"ids": [[5, 2], [7, 1]], "logprobs": [[-0.1005, -3.0], [-0.5, -0.9]]}
    swapped = {"ids": [[2, 5], [7, 3]], "logprobs": [[-0.1, -3.0], [-0.5, -0.902]]}
    assert verify.compare_answers(a, a) == [] and verify.compare_answers(a, close) == []
    got = verify.compare_answers(a, swapped)
    assert len(got) == 2 and "row 0: greedy token 2, expected 5" in got[0] and "row 1" in got[1] and "0.002" in got[1]
    assert verify.compare_answers(a, swapped, atol=0.01) == got[:1]
    assert verify.compare_answers(a, {"ids": a["ids"], "logprobs": [[-0.1, -3.0], [math.nan, -0.9]]})
    with pytest.raises(ValueError):
        verify.compare_answers(a, {"ids": [[5]], "logprobs": [[0.0]]})
