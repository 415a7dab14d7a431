"""Top log-probabilities and sampling against the oracle's 64-bit rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import rows as oracle
from tests.rows_helpers import TYPES, host, logprob_bound, peaked
from warpshift_b200 import logits as ops

pytestmark = pytest.mark.gpu


def check_top(x: torch.Tensor, k: int, temperature: float = 1.0) -> None:
    got = ops.top_logprobs(x, k, temperature=temperature)
    assert got.ids.shape == got.logprobs.shape == (*x.shape[:-1], k)
    assert got.ids.dtype == torch.int64 and got.logprobs.dtype == torch.float32
    v = x.shape[-1]
    for row, ids, logp in zip(host(x).reshape(-1, v), host(got.ids).reshape(-1, k), host(got.logprobs).reshape(-1, k)):
        want_ids, want = oracle.top(row, k, float(np.float32(temperature)))
        np.testing.assert_array_equal(ids, want_ids)
        np.testing.assert_array_equal(np.isnan(logp), np.isnan(want))
        fine = np.isfinite(want)
        np.testing.assert_array_equal(logp[~fine], want[~fine])
        assert (np.abs(logp[fine] - want[fine]) <= logprob_bound(want[fine], v)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 8, 3), (4, 257, 256), (3, 1000, 1), (2, 2047, 100),
                                          (2, 2049, 256), (3, 8191, 64), (2, 32000, 20), (7, 50257, 256), (2, 128256, 64)])
def test_top_logprobs(cuda_device, dtype, rows, vocab, k) -> None:
    check_top(peaked(rows, vocab, TYPES[dtype], seed=vocab + k), k)


@pytest.mark.parametrize("rows", [1, 2, 9, 40, 150, 400, 700])
def test_top_logprobs_by_number_of_rows(cuda_device, rows) -> None:
    check_top(peaked(rows, 5003, torch.bfloat16, seed=rows), 17, temperature=0.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [0.1, 1.3, 50.0])
def test_top_logprobs_at_a_temperature(cuda_device, dtype, temperature) -> None:
    check_top(peaked(3, 4099, TYPES[dtype], seed=5), 33, temperature)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["ascending", "descending", "constant", "two_values", "zeros", "steps"])
def test_top_logprobs_of_ordered_and_equal_logits(cuda_device, dtype, kind) -> None:
    v = 40000
    at = torch.arange(v, dtype=torch.float64)
    x = {"ascending": at / 1000, "descending": -at / 1000, "constant": torch.full((v,), 1.25), "two_values": (at % 97 == 0).double(),
         "zeros": torch.where(at % 2 == 0, 0.0, -0.0), "steps": torch.div(at, 3000, rounding_mode="floor")}[kind]
    check_top(x.to(TYPES[dtype]).to("cuda").expand(2, v), 256)
    check_top(x.to(TYPES[dtype]).to("cuda")[None], 5)


@pytest.mark.parametrize("dtype", TYPES)
def test_top_logprobs_with_masked_logits(cuda_device, dtype) -> None:
    t = TYPES[dtype]
    x = peaked(9, 3001, t, seed=2)
    x[0] = -torch.inf
    x[1, 5:] = -torch.inf
    x[2, :2990] = -torch.inf
    x[3] = torch.finfo(t).min
    x[4, 100:] = torch.finfo(t).min
    x[5, 77] = torch.nan
    x[6, 77] = torch.inf
    x[7] = torch.nan
    x[8, ::2] = -torch.inf
    check_top(x, 64)
    check_top(x, 256, temperature=2.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_stride_and_alignment(cuda_device, dtype) -> None:
    g = torch.Generator().manual_seed(1)
    buffer = torch.randn(40000, generator=g).to(TYPES[dtype]).to("cuda")
    for offset in range(0, 9):
        check_top(buffer[offset : offset + 3 * 1003].view(3, 1003), 9)
        check_top(buffer[offset : offset + 5 * 600].view(5, 600)[:, :523], 40)
    check_top(buffer[:36000].view(3, 4, 3000)[:, 1:], 6)          # rows with two strides
    check_top(buffer[:36000].view(3, 4, 3000)[::2, ::3], 6)
    check_top(buffer[:36000].view(2, 2, 3, 3000), 6)
    check_top(buffer[:777], 6)                                    # one row without a row dimension
    check_top(buffer[:777].expand(4, 777), 6)
    check_top(buffer[:36000].view(12, 3000)[:, ::3000], 1)        # one element a row
    empty = ops.top_logprobs(buffer.new_empty(0, 50), 4)
    assert empty.ids.shape == (0, 4)


# Long rows of a small batch go to clusters of 2, 4 and 8 blocks; many rows to one block each.
SPLITS = [(3, 70001), (40, 70001), (100, 40001), (160, 20001)]


@pytest.mark.parametrize("rows,vocab", SPLITS)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_top_logprobs_of_split_rows(cuda_device, dtype, rows, vocab) -> None:
    t = TYPES[dtype]
    x = peaked(rows, vocab, t, seed=rows)
    x[0] = -torch.inf
    x[1, 5:] = -torch.inf
    x[1, -3:] = 2.0
    x[2] = torch.finfo(t).min
    if rows > 9:
        at = torch.arange(vocab, device="cuda")
        x[3] = (at / 2000).to(t)
        x[4] = (-at / 2000).to(t)
        x[5] = 1.25
        x[6, vocab // 2 :] = -torch.inf
        x[7, 30000 % vocab] = torch.nan
        x[8, 30000 % vocab] = torch.inf
    check_top(x, 256)
    check_top(x[:9], 20, temperature=0.5)
    check_top(x[:9, 1:], 1)


def test_top_logprobs_of_the_longest_rows(cuda_device) -> None:
    x = peaked(2, 1 << 20, torch.float32, seed=3)
    check_top(x, 100)
    one_block = ops.top_logprobs(x[0].expand(200, 1 << 20), 100)
    assert torch.equal(one_block.ids, ops.top_logprobs(x[:1], 100).ids.expand(200, 100))
    with pytest.raises(ValueError):
        ops.top_logprobs(torch.zeros(1, device="cuda").expand((1 << 20) + 1), 1)


def test_rows_beyond_32_bits(cuda_device) -> None:
    """Rows whose offset passes 2^32 elements, and 2^32 bytes."""
    buffer = torch.empty((1 << 32) + 40000, dtype=torch.bfloat16, device="cuda")
    x = buffer.as_strided((3, 9001), ((1 << 31) + 9001, 1))
    x.copy_(peaked(3, 9001, torch.bfloat16, seed=1))
    check_top(x, 30)
    check_sample(x, torch.tensor([0.1, 0.5, 0.9], device="cuda"), top_p=0.9)


def settings(rows: int, seed: int) -> dict[str, torch.Tensor]:
    g = torch.Generator().manual_seed(seed)

    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (rows,), generator=g)].to("cuda")

    return {"temperature": pick([0.0, 0.01, 0.5, 1.0, 1.0, 3.0], torch.float32), "top_k": pick([0, 0, 1, 2, 30, 256, 257, 3000], torch.int64),
            "top_p": pick([1.0, 1.0, 0.0, 0.1, 0.6, 0.95, 0.9999], torch.float32), "min_p": pick([0.0, 0.0, 0.02, 0.3, 1.0], torch.float32)}


def check_sample(x: torch.Tensor, uniform: torch.Tensor, **params) -> None:
    got = ops.sample(x, uniform, **params)
    assert got.tokens.shape == got.logprobs.shape == x.shape[:-1]
    v = x.shape[-1]
    each = {n: host(p).reshape(-1) if isinstance(p, torch.Tensor) else None for n, p in params.items()}
    tokens, logps = host(got.tokens).reshape(-1), host(got.logprobs).reshape(-1)
    for r, (row, u) in enumerate(zip(host(x).reshape(-1, v), host(uniform).reshape(-1))):
        one = {n: params[n] if each[n] is None else each[n][r] for n in params}
        if "top_k" in one:
            one["top_k"] = int(one["top_k"])
        token, logp = oracle.sample(row, u, **one)
        assert tokens[r] == token, (r, one)
        if np.isfinite(logp):
            assert abs(logps[r] - logp) <= logprob_bound(np.array(logp), v), (r, one)
        else:
            np.testing.assert_equal(logps[r], logp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (20, 9), (60, 300), (60, 1025), (60, 5003), (24, 32000), (24, 128256)])
def test_sample_with_settings_of_each_row(cuda_device, dtype, rows, vocab) -> None:
    g = torch.Generator().manual_seed(rows * vocab)
    x = peaked(rows, vocab, TYPES[dtype], seed=vocab, scale=2.0)
    check_sample(x, torch.rand(rows, generator=g).to("cuda"), **settings(rows, vocab))


@pytest.mark.parametrize("rows", [1, 2, 9, 40, 150, 700])
def test_sample_by_number_of_rows(cuda_device, rows) -> None:
    g = torch.Generator().manual_seed(rows)
    x = peaked(rows, 3001, torch.float16, seed=rows)
    check_sample(x, torch.rand(rows, generator=g).to("cuda"), **settings(rows, rows))


PARAMS = [{}, {"temperature": 0.0}, {"temperature": 0.3}, {"top_k": 1}, {"top_k": 10}, {"top_k": 700}, {"top_p": 0.3}, {"top_p": 0.9},
          {"top_p": 0.999}, {"min_p": 0.1}, {"min_p": 1.0}, {"temperature": 1.7, "top_k": 50, "top_p": 0.9, "min_p": 0.03},
          {"temperature": 2.0, "top_k": 1500, "top_p": 0.95}]


@pytest.mark.parametrize("params", PARAMS)
@pytest.mark.parametrize("kind", ["peaked", "flat", "constant", "two_values", "ascending"])
def test_sample_over_distributions(cuda_device, params, kind) -> None:
    rows, v = 12, 6001
    g = torch.Generator().manual_seed(3)
    at = torch.arange(v, dtype=torch.float32).expand(rows, v)
    x = {"peaked": peaked(rows, v, torch.bfloat16, seed=1), "flat": torch.randn(rows, v, generator=g) * 0.1, "constant": torch.full((rows, v), -3.0),
         "two_values": (at % 5 == 0).float() * 3, "ascending": at / 500}[kind].to(torch.bfloat16).to("cuda")
    uniform = torch.cat([torch.tensor([0.0, 1 - 2.0**-24]), torch.rand(rows - 2, generator=g)]).to("cuda")
    check_sample(x, uniform, **params)
    check_sample(x.float(), uniform, **params)


@pytest.mark.parametrize("params", [{}, {"top_p": 0.5}, {"top_k": 3}, {"top_k": 400}, {"min_p": 0.5}, {"temperature": 0.0}])
@pytest.mark.parametrize("dtype", TYPES)
def test_sample_with_masked_logits(cuda_device, dtype, params) -> None:
    t = TYPES[dtype]
    x = peaked(9, 1501, t, seed=4)
    x[0] = -torch.inf
    x[1, 1:] = -torch.inf
    x[2, :1490] = -torch.inf
    x[3] = torch.finfo(t).min
    x[4, 10:] = torch.finfo(t).min
    x[5, 77] = torch.nan
    x[6, 77] = x[6, 1234] = torch.inf
    x[7] = torch.nan
    x[8, ::2] = -torch.inf
    for u in (0.0, 0.3, 0.7, 1 - 2.0**-24):
        check_sample(x, torch.full((9,), u, device="cuda"), **params)


@pytest.mark.parametrize("rows,vocab", SPLITS)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_sample_of_split_rows(cuda_device, dtype, rows, vocab) -> None:
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(rows)
    x = peaked(rows, vocab, t, seed=vocab, scale=2.0)
    if rows > 9:
        at = torch.arange(vocab, device="cuda")
        x[0] = -torch.inf
        x[1, 5:] = -torch.inf
        x[2] = torch.finfo(t).min
        x[3] = (at / 2000).to(t)
        x[4] = 1.25
        x[5, : vocab // 2] = -torch.inf
        x[6, 30000 % vocab] = torch.nan
        x[7, 30000 % vocab] = torch.inf
        x[8] = (at % 5 == 0).to(t)
        x[9] = torch.randn(vocab, generator=g).to(t)
        x[10] = torch.randn(vocab, generator=g).to(t) * 0.01
    uniform = torch.rand(rows, generator=g).to("cuda")
    uniform[0::7] = 0.0
    check_sample(x[:60], uniform[:60], **{n: p[:60] for n, p in settings(rows, vocab).items()})
    for params in ({}, {"top_p": 0.8}, {"top_k": 500, "top_p": 0.9}, {"top_k": 5000}, {"min_p": 0.2, "temperature": 1.5}, {"temperature": 0.0}):
        check_sample(x[:11], uniform[:11], **params)


def test_sample_of_the_longest_rows(cuda_device) -> None:
    x = peaked(1, 1 << 20, torch.float32, seed=3)
    u = torch.rand(200, generator=torch.Generator().manual_seed(1)).to("cuda")
    for params in ({}, {"top_p": 0.95}, {"top_k": 5000}):
        check_sample(x, u[:1], **params)
        many = ops.sample(x.expand(200, 1 << 20), u, **params).tokens  # a block for each row
        one = torch.cat([ops.sample(x, u[i : i + 1], **params).tokens for i in range(200)])  # eight for each
        assert torch.equal(many, one)


def test_sample_uniform_out_of_range_takes_the_ends(cuda_device) -> None:
    x = torch.zeros(4, 100, device="cuda")
    u = torch.tensor([-1.0, 1.0, torch.nan, torch.inf], device="cuda")
    assert ops.sample(x, u).tokens.tolist() == [0, 99, 0, 99]


def test_sample_draws_by_the_probabilities(cuda_device) -> None:
    """Equally spaced numbers give every token its share of them, give or take one."""
    n, v = 4096, 50
    x = peaked(1, v, torch.float32, seed=9, scale=1.0) * 0.3
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens = ops.sample(x.expand(n, v), u).tokens
    share = torch.bincount(tokens, minlength=v).double().cpu() / n
    assert (share - torch.softmax(x[0].double().cpu(), 0)).abs().max() <= 1.01 / n


def test_sample_any_stride(cuda_device) -> None:
    x = peaked(12, 4000, torch.bfloat16, seed=6)
    u = torch.rand(12, generator=torch.Generator().manual_seed(0)).to("cuda")
    check_sample(x[:, 3:2502], u, top_p=0.8)
    check_sample(x.view(3, 4, 4000)[:, 1:, 1:], u.view(3, 4)[:, 1:], top_k=torch.full((3, 3), 40, dtype=torch.int32, device="cuda"))
    check_sample(x[0], u[0])
    assert ops.sample(x[:0], u[:0]).tokens.shape == (0,)


def test_graph_replay_on_another_stream(cuda_device) -> None:
    """Captured once, replayed with new inputs in place; nothing is kept from the first call."""
    x, u = peaked(5, 3000, torch.bfloat16, seed=1), torch.rand(5, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.top_logprobs(x, 8), ops.sample(x, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        top, drawn = ops.top_logprobs(x, 8), ops.sample(x, u, top_p=0.9)
    for seed in (2, 3):
        x.copy_(peaked(5, 3000, torch.bfloat16, seed=seed))
        u.uniform_()
        graph.replay()
        want_top, want = ops.top_logprobs(x, 8), ops.sample(x, u, top_p=0.9)
        for a, b in zip((*top, *drawn), (*want_top, *want)):
            assert torch.equal(a, b)


def test_two_streams_at_once(cuda_device) -> None:
    xs = [peaked(64, 20011, torch.bfloat16, seed=s) for s in (1, 2)]
    u = torch.rand(64, device="cuda")
    want = [(ops.top_logprobs(x, 100), ops.sample(x, u, temperature=2.0)) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.top_logprobs(xs[i], 100), ops.sample(xs[i], u, temperature=2.0)))
    torch.cuda.synchronize()
    for i in range(2):
        for top, drawn in got[i]:
            for a, b in zip((*top, *drawn), (*want[i][0], *want[i][1])):
                assert torch.equal(a, b)


def test_answer_records_of_a_model_switched_there_and_back(cuda_device) -> None:
    """The acceptance check on answers: a model's record after a switch and a switch back equals the one before."""
    from warpshift_b200 import verify
    from warpshift_b200.delta import DeltaWeights

    g = torch.Generator().manual_seed(2)
    first = {"head": (torch.randn(5000, 128, generator=g) * 0.2).to(torch.bfloat16)}
    second = {"head": (first["head"].float() * (1 + 0.05 * torch.randn(5000, 128, generator=g))).to(torch.bfloat16).to("cuda")}
    hidden = torch.randn(6, 128, generator=g).to(torch.bfloat16).to("cuda")
    answers = lambda: verify.answer_record(hidden @ second["head"].t(), 10)  # noqa: E731
    before = answers()
    delta = DeltaWeights(first, second)
    delta.apply(reverse=True)
    other = answers()
    native = verify.answer_record(hidden @ first["head"].to("cuda").t(), 10)
    delta.apply(reverse=False)
    assert verify.compare_answers(native, other) == [] and verify.compare_answers(before, answers()) == []
    assert verify.compare_answers(before, other)


@pytest.mark.parametrize("temperature", [1e-38, 1e-30, 1e-6, 1e6, 1e30, float("inf")])
def test_sample_at_the_ends_of_temperature(cuda_device, temperature) -> None:
    g = torch.Generator().manual_seed(8)
    x = peaked(4, 3001, torch.float32, seed=8)
    x[1] = torch.finfo(torch.float32).max * (torch.rand(3001, generator=g) * 2 - 1).to("cuda")
    x[2] = torch.arange(3001, device="cuda") * 2.0**-20 + 1e4
    x[3] = torch.where(torch.arange(3001) % 7 == 0, 1e-40, 0.0).to("cuda")
    for u in (0.0, 0.2, 0.9):
        for params in ({}, {"top_p": 0.7}, {"top_k": 900}, {"min_p": 0.5}):
            check_sample(x[:3], torch.full((3,), u, device="cuda"), temperature=temperature, **params)
    # Logits below the smallest normal number still order the tokens.
    assert int(ops.sample(x[3:], torch.full((1,), 0.5, device="cuda"), temperature=0.0).tokens) == 0
    assert ops.top_logprobs(x[3:], 3).ids.tolist() == [[0, 7, 14]]
