"""The distillation loss and its gradient against the oracle's 64-bit rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import rows as oracle
from tests.rows_helpers import TYPES, grad_bound, host, peaked, sum_error
from warpshift_b200 import distill, logits as ops

pytestmark = pytest.mark.gpu


def record(rows: int, vocab: int, k: int, seed: int, spread: float = 3.0) -> tuple[torch.Tensor, torch.Tensor]:
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, vocab, (rows, k), generator=g)  # some come twice
    logprobs = torch.log_softmax(torch.randn(rows, k, generator=g) * spread, 1) - 0.05
    return ids.to("cuda"), logprobs.to("cuda")


def check(x, ids, logprobs, weights=None, temperature=1.0, tail="drop", grad_out=None, both=True) -> None:
    x = x.detach()
    v, k = x.shape[-1], ids.shape[-1]
    leaf = x.clone().requires_grad_(True) if x.is_contiguous() else x.requires_grad_(True)
    kw = {"weights": weights, "temperature": temperature, "tail": tail}
    loss = distill.top_logprob_loss(leaf, ids, logprobs, **kw)
    out = torch.ones_like(loss) if grad_out is None else grad_out
    (grad,) = torch.autograd.grad(loss, leaf, out)
    assert grad.dtype == x.dtype and grad.shape == x.shape and loss.dtype == torch.float32 and loss.shape == x.shape[:-1]
    compare(x, ids, logprobs, loss, grad, out, **kw)
    if both and grad_out is None:
        loss2, grad2 = distill.top_logprob_loss_and_grad(x, ids, logprobs, **kw)
        compare(x, ids, logprobs, loss2, grad2, out, **kw)


def compare(x, ids, logprobs, loss, grad, out, weights, temperature, tail) -> None:
    v, k = x.shape[-1], ids.shape[-1]
    t = float(np.float32(temperature))
    w = np.ones(loss.numel()) if weights is None else host(weights).reshape(-1)
    per_row = zip(host(x).reshape(-1, v), ids.cpu().numpy().reshape(-1, k), host(logprobs).reshape(-1, k), host(loss).reshape(-1),
                  host(grad).reshape(-1, v), w, host(out).reshape(-1))
    for r, (row, i, lp, got, got_grad, weight, g) in enumerate(per_row):
        want, want_grad = oracle.distill(row, i, lp, weight, t, tail, g)
        if np.isfinite(want):
            there = (i >= 0) & (i < v) & (lp > -np.inf)
            q = np.exp(lp[there])
            mass = 1.0 if tail == "renormalize" else q.sum()
            # log S once for each unit of mass, the sums over the record in 64 bits (1e-12 of their parts), one rounding of the loss
            # and one of the weight's product; 1 / temperature is rounded once.
            d = np.where(np.isfinite(row[i[there]]), np.abs(row[i[there]] - row.max()), 0.0) / t
            parts = (q * (np.abs(lp[there]) + d)).sum() / (q.sum() if tail == "renormalize" and q.size else 1.0)
            bound = abs(weight) * (mass * sum_error(v) + parts * (1e-12 + 2.0**-24)) + abs(want) * 2 * 2.0**-24 + 2.0**-126
            assert abs(got - want) <= bound, (r, got, want, bound)
        else:
            np.testing.assert_equal(got, want)
        bound = grad_bound(row, i, lp, weight, t, tail, g, x.dtype)
        off = np.abs(got_grad - want_grad)
        assert (off <= bound).all(), (r, int(np.argmax(off - bound)), off.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", ["drop", "renormalize"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (2, 2, 5), (3, 7, 3), (4, 64, 256), (5, 1000, 1), (3, 2049, 17), (3, 8193, 256),
                                          (2, 32000, 8), (3, 50257, 64), (2, 128256, 32)])
def test_loss_and_gradient(cuda_device, dtype, tail, rows, vocab, k) -> None:
    ids, logprobs = record(rows, vocab, k, seed=vocab + k)
    check(peaked(rows, vocab, TYPES[dtype], seed=vocab), ids, logprobs, tail=tail)


@pytest.mark.parametrize("rows", [1, 2, 9, 40, 150, 400, 700])
def test_by_number_of_rows(cuda_device, rows) -> None:
    ids, logprobs = record(rows, 5003, 20, seed=rows)
    check(peaked(rows, 5003, torch.bfloat16, seed=rows), ids, logprobs, temperature=1.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [0.25, 2.0, 20.0])
def test_temperatures_weights_and_incoming_gradients(cuda_device, dtype, temperature) -> None:
    rows, v = 24, 3001
    g = torch.Generator().manual_seed(7)
    ids, logprobs = record(rows, v, 40, seed=1)
    weights = torch.where(torch.rand(rows, generator=g) < 0.3, 0.0, torch.rand(rows, generator=g) * 2).to("cuda")
    x = peaked(rows, v, TYPES[dtype], seed=3)
    check(x, ids.int(), logprobs, weights=weights, temperature=temperature)
    check(x, ids, logprobs, weights=weights, temperature=temperature, tail="renormalize", grad_out=torch.randn(rows, generator=g).to("cuda"))
    check(x, ids, logprobs, grad_out=torch.randn(1, generator=g).to("cuda").expand(rows))
    check(x, ids, logprobs, grad_out=torch.randn(2 * rows, generator=g).to("cuda")[::2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", ["drop", "renormalize"])
def test_masks_and_records_with_gaps(cuda_device, dtype, tail) -> None:
    t = TYPES[dtype]
    rows, v, k = 10, 1503, 12
    ids, logprobs = record(rows, v, k, seed=11)
    x = peaked(rows, v, t, seed=12)
    ids[0] = -1                                    # a record of nothing
    logprobs[1, 3:] = -torch.inf
    ids[2, ::2] = torch.tensor([-1, v, -5, v + 7, 1 << 40, -(1 << 40)], device="cuda")
    ids[3] = 77                                    # one token k times
    x[4, ids[4]] = -torch.inf                      # tokens of the record are masked
    x[5] = -torch.inf                              # a row of nothing
    x[6] = torch.finfo(t).min
    x[7, 5:] = torch.finfo(t).min
    x[8, 7:] = -torch.inf
    ids[8] = ids[8] % 7
    logprobs[9] -= 100.0                           # a record far out in the teacher's tail
    check(x, ids, logprobs, tail=tail)


@pytest.mark.parametrize("rows,vocab", [(3, 70001), (40, 70001), (100, 40001), (160, 20001)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("tail", ["drop", "renormalize"])
def test_rows_split_over_blocks(cuda_device, dtype, rows, vocab, tail) -> None:
    """Long rows of a small batch go to clusters of 2, 4 and 8 blocks; many rows to one block each."""
    t = TYPES[dtype]
    ids, logprobs = record(rows, vocab, 200, seed=rows)
    x = peaked(rows, vocab, t, seed=vocab)
    weights = torch.ones(rows, device="cuda")
    weights[1] = 0
    if rows > 9:
        x[2] = -torch.inf
        x[3] = torch.finfo(t).min
        x[4, vocab // 3 :] = -torch.inf
        ids[4] %= vocab // 3
        x[5, ids[5, 0]] = -torch.inf
        ids[6] = -1
        ids[7] = 33333 % vocab
        ids[8, 100:] = ids[8, :100]
    check(x[:30], ids[:30], logprobs[:30], weights=weights[:30], tail=tail, temperature=0.8)
    if rows > 30:
        check(x, ids, logprobs, weights=weights, tail=tail, grad_out=torch.randn(rows, generator=torch.Generator().manual_seed(2)).to("cuda"))


def test_the_longest_rows(cuda_device) -> None:
    x = peaked(2, 1 << 20, torch.float32, seed=3)
    ids, logprobs = record(2, 1 << 20, 100, seed=4)
    check(x, ids, logprobs)
    loss, grad = distill.top_logprob_loss_and_grad(x[0].expand(200, 1 << 20), ids[0].expand(200, 100), logprobs[0].expand(200, 100))
    want, want_grad = distill.top_logprob_loss_and_grad(x[:1], ids[:1], logprobs[:1])
    torch.testing.assert_close(loss, want.expand(200), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(grad[[0, 77, 199]], want_grad.expand(3, 1 << 20), rtol=1e-4, atol=1e-9)


def test_rows_beyond_32_bits(cuda_device) -> None:
    buffer = torch.empty((1 << 32) + 40000, dtype=torch.bfloat16, device="cuda")
    x = buffer.as_strided((3, 9001), ((1 << 31) + 9001, 1))
    x.copy_(peaked(3, 9001, torch.bfloat16, seed=1))
    ids, logprobs = record(3, 9001, 20, seed=5)
    check(x, ids, logprobs)


def test_saved_tensors_may_be_kept_elsewhere(cuda_device) -> None:
    """Hooks on saved tensors (offloading to the host) give the backward pass other tensors than the forward pass had."""
    x = peaked(5, 3001, torch.bfloat16, seed=1).requires_grad_(True)
    ids, logprobs = record(5, 3001, 20, seed=2)
    with torch.autograd.graph.save_on_cpu():
        loss = distill.top_logprob_loss(x, ids, logprobs, weights=torch.full((5,), 0.5, device="cuda"))
    filler = torch.full((1 << 20,), 7.0, device="cuda")
    (grad,) = torch.autograd.grad(loss.sum(), x)
    del filler
    _, want = distill.top_logprob_loss_and_grad(x.detach(), ids, logprobs, weights=torch.full((5,), 0.5, device="cuda"))
    torch.testing.assert_close(grad, want, rtol=2.0**-7, atol=1e-8)


def test_backward_twice_and_changed_logits(cuda_device) -> None:
    x = peaked(4, 999, torch.float32, seed=1).requires_grad_(True)
    ids, logprobs = record(4, 999, 9, seed=2)
    loss = distill.top_logprob_loss(x, ids, logprobs)
    (first,) = torch.autograd.grad(loss.sum(), x, retain_graph=True)
    (second,) = torch.autograd.grad(loss.sum(), x, retain_graph=True)
    assert torch.equal(first, second)
    (grad,) = torch.autograd.grad(loss.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        grad.sum().backward()
    loss = distill.top_logprob_loss(x, ids, logprobs)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


def test_two_steps_on_two_streams(cuda_device) -> None:
    xs = [peaked(64, 20011, torch.bfloat16, seed=s) for s in (1, 2)]
    ids, logprobs = record(64, 20011, 30, seed=3)
    want = [distill.top_logprob_loss_and_grad(x, ids, logprobs) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(distill.top_logprob_loss_and_grad(xs[i], ids, logprobs))
    torch.cuda.synchronize()
    for i in range(2):
        for loss, grad in got[i]:
            assert torch.equal(loss, want[i][0]) and torch.equal(grad, want[i][1])


def test_rows_of_weight_zero_are_not_read(cuda_device) -> None:
    x = peaked(4, 999, torch.bfloat16, seed=1)
    ids, logprobs = record(4, 999, 5, seed=2)
    x[1], x[2, 10] = torch.nan, torch.inf
    logprobs[3] = torch.nan
    weights = torch.tensor([1.0, 0.0, 0.0, 0.0], device="cuda")
    loss, grad = distill.top_logprob_loss_and_grad(x, ids, logprobs, weights=weights)
    leaf = x.clone().requires_grad_(True)
    loss2 = distill.top_logprob_loss(leaf, ids, logprobs, weights=weights)
    loss2.sum().backward()
    for a, b in ((loss, grad), (loss2, leaf.grad)):
        assert a[0] > 0 and not a[1:].any() and b[0].any() and not b[1:].any()
        assert torch.isfinite(a).all() and torch.isfinite(b.float()).all()


def test_nan_and_inf_logits_show(cuda_device) -> None:
    x = peaked(3, 999, torch.float32, seed=1)
    ids, logprobs = record(3, 999, 5, seed=2)
    x[1, 500], x[2, 500] = torch.nan, torch.inf
    loss, grad = distill.top_logprob_loss_and_grad(x, ids, logprobs)
    assert torch.isfinite(loss[0]) and torch.isnan(loss[1:]).all()
    assert torch.isfinite(grad[0]).all() and torch.isnan(grad[1:]).any(1).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_any_stride_and_alignment(cuda_device, dtype) -> None:
    g = torch.Generator().manual_seed(1)
    buffer = torch.randn(40000, generator=g).to(TYPES[dtype]).to("cuda")
    for offset in (0, 1, 2, 3, 5, 8):
        ids, logprobs = record(3, 1003, 9, seed=offset)
        check(buffer[offset : offset + 3 * 1003].view(3, 1003), ids, logprobs)
        ids, logprobs = record(5, 523, 9, seed=offset)
        check(buffer[offset : offset + 5 * 600].view(5, 600)[:, :523], ids, logprobs)
        check(buffer[offset : offset + 5 * 530].view(5, 530)[:, 2:525], ids, logprobs)
    ids, logprobs = record(9, 3000, 9, seed=9)
    shifted = buffer[:36000].view(3, 4, 3000)[:, :-1]
    check(shifted, ids.view(3, 3, 9), logprobs.view(3, 3, 9))
    check(shifted, ids.view(3, 3, 9), logprobs.view(3, 3, 9), grad_out=torch.randn(3, 3, generator=g).to("cuda"))
    check(shifted, ids.view(3, 3, 9), logprobs.view(3, 3, 9), grad_out=torch.randn(3, 1, generator=g).to("cuda").expand(3, 3))
    check(buffer[:777], ids[0] % 777, logprobs[0])
    wide = torch.stack([ids, ids], 2)[..., 0]       # a record with gaps in memory
    check(buffer[:27000].view(9, 3000), wide, logprobs)
    loss, grad = distill.top_logprob_loss_and_grad(buffer.new_empty(0, 50), ids[:0], logprobs[:0])
    assert loss.shape == (0,) and grad.shape == (0, 50)


def test_shared_rows_add_up(cuda_device) -> None:
    """Logits broadcast over rows get the sum of the rows' gradients."""
    base = peaked(1, 2000, torch.float32, seed=5).requires_grad_(True)
    ids, logprobs = record(6, 2000, 10, seed=6)
    distill.top_logprob_loss(base.expand(6, 2000), ids, logprobs).sum().backward()
    one = peaked(1, 2000, torch.float32, seed=5).repeat(6, 1)
    _, grad = distill.top_logprob_loss_and_grad(one, ids, logprobs)
    torch.testing.assert_close(base.grad[0], grad.sum(0), rtol=1e-5, atol=1e-7)


def test_gradient_against_differences(cuda_device) -> None:
    """The loss of logits moved along a direction changes by the gradient's share of it: differences of the oracle's loss (64 bits)
    against the kernel's gradient."""
    x = peaked(4, 301, torch.float32, seed=8)
    ids, logprobs = record(4, 301, 7, seed=8)
    direction = np.random.default_rng(0).standard_normal((4, 301))
    for tail in ("drop", "renormalize"):
        _, grad = distill.top_logprob_loss_and_grad(x, ids, logprobs, temperature=1.5, tail=tail)
        for r in range(4):
            f = lambda e: oracle.distill(host(x)[r] + e * direction[r], ids[r].cpu().numpy(), host(logprobs)[r], 1.0, 1.5, tail)[0]  # noqa: B023, E731
            h = 1e-4  # the difference's own error: h^2 times a third derivative of order 10
            slope = (f(h) - f(-h)) / (2 * h)
            assert abs(slope - (host(grad)[r] * direction[r]).sum()) < 1e-5


def test_backward_in_a_graph(cuda_device) -> None:
    """A training step's forward and backward captured and replayed with new logits."""
    ids, logprobs = record(6, 4001, 16, seed=3)
    x = peaked(6, 4001, torch.bfloat16, seed=1).requires_grad_(True)
    g = torch.full((6,), 0.25, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(distill.top_logprob_loss(x, ids, logprobs), x, g)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = distill.top_logprob_loss(x, ids, logprobs)
        (grad,) = torch.autograd.grad(loss, x, g)
    loss, grad = loss.detach(), grad.detach()
    for seed in (4, 5):
        with torch.no_grad():
            x.copy_(peaked(6, 4001, torch.bfloat16, seed=seed))
        graph.replay()
        want, want_grad = distill.top_logprob_loss_and_grad(x.detach(), ids, logprobs, weights=g)
        assert torch.equal(loss * 0.25, want)
        compare(x, ids, logprobs, loss, grad, g, weights=None, temperature=1.0, tail="drop")
        compare(x, ids, logprobs, want, want_grad, torch.ones_like(g), weights=g, temperature=1.0, tail="drop")


def test_student_samples_teacher_scores_student_learns(cuda_device) -> None:
    """The operators in a row, as a round of on-policy distillation uses them."""
    rows, v, k = 16, 3000, 32
    hidden = torch.randn(rows, 64, generator=torch.Generator().manual_seed(0)).to("cuda")
    head = (torch.randn(v, 64, generator=torch.Generator().manual_seed(1)) * 0.3).to("cuda").requires_grad_(True)
    student = (hidden @ head.t()).to(torch.bfloat16)
    drawn = ops.sample(student.detach(), torch.rand(rows, device="cuda"), temperature=0.8, top_p=0.95)
    assert ((drawn.tokens >= 0) & (drawn.tokens < v)).all()
    teacher = peaked(rows, v, torch.bfloat16, seed=4)
    teacher.scatter_(1, drawn.tokens[:, None], 9.0)
    top = ops.top_logprobs(teacher, k, temperature=2.0)
    loss = distill.top_logprob_loss(student, top.ids, top.logprobs, temperature=2.0, tail="renormalize").mean()
    loss.backward()
    ids, lp = top.ids.cpu().numpy(), host(top.logprobs)
    s = host(student)
    want = np.stack([oracle.distill(s[r], ids[r], lp[r], 1.0, 2.0, "renormalize", 1 / rows)[1] for r in range(rows)])
    # Each element of the logits' gradient is rounded once to bf16 (2^-8 of it); the product adds rows of them up in fp32.
    reference = want.T @ host(hidden)
    room = (np.abs(want).T @ np.abs(host(hidden))) * (2.0**-8 + 2.0**-14)
    assert (np.abs(host(head.grad) - reference) <= room + 1e-9).all()
