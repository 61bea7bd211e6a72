"""GPU tests of the teacher's distribution: a softmax does not change when one
constant is added to all logits of a row.  The logits are multiples of 2^-6 up to
8 and the constants multiples of 2^-6 below 2^16, so that every sum is an FP32
number and the differences of a row's logits are the same numbers: losses and
gradients have to be the same bits.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _problem(rows, vocab, width, kind, most):
    import torch

    dtype = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
    gen = torch.Generator(device="cuda").manual_seed(rows + most)
    h = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
    e = (2.0 / math.sqrt(width) * torch.randn(vocab, width, generator=gen, device="cuda")).to(dtype)
    ids = torch.rand(rows, vocab, generator=gen, device="cuda").topk(most, 1).indices.sort(1).values
    logits = torch.randint(-512, 513, (rows, most), generator=gen, device="cuda").float() / 64
    logits[torch.rand(rows, most, generator=gen, device="cuda") < 0.05] = -math.inf
    logits[3] = -math.inf  # a row that says nothing
    offsets = (most * torch.arange(rows + 1, device="cuda")).int()
    grad = torch.rand(rows, generator=gen, device="cuda") - 0.3
    return h, e, offsets, ids.reshape(-1).int(), logits, grad, gen


def _step(mf, h, e, offsets, ids, logits, T, grad):
    import torch

    loss = mf.DenseLoss(e, h.shape[0], stream=torch.cuda.Stream())
    logits = logits.reshape(-1).contiguous()
    torch.cuda.synchronize()
    losses, lse = loss.distill(h, offsets, ids, logits, T)
    out = losses, lse, *loss.distill_backward(h, offsets, ids, logits, T, lse, grad)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("T", (1.0, 1.5, 0.01))
@pytest.mark.parametrize("rows,most", [(30, 64), (60, 64), (150, 64), (300, 5), (20, 700)])
def test_a_constant_added_to_a_rows_logits(mf, rows, most, T, kind):
    import torch

    h, e, offsets, ids, logits, grad, gen = _problem(rows, 1000, 72, kind, most)
    h *= T  # scores over T of a few units
    want = _step(mf, h, e, offsets, ids, logits, T, grad)
    assert bool(torch.isfinite(want[0]).all()) and float(want[0].abs().max()) > 0
    shift = torch.randint(-(1 << 22) + 513, (1 << 22) - 513, (rows, 1), generator=gen,
                          device="cuda").float() / 64
    shift[0], shift[1] = 10_000.0, -60_000.0
    moved = logits + shift
    assert torch.equal(moved - shift, logits) or bool(torch.isinf(logits).any())
    got = _step(mf, h, e, offsets, ids, moved, T, grad)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", (30, 60, 150))
def test_logits_far_apart(mf, rows):
    """Logits over T beyond FP32's range: the largest has all the weight, and the
    loss is the cross entropy of its id."""
    import torch

    h, e, offsets, ids, logits, grad, _ = _problem(rows, 1000, 72, "f16", 4)
    logits[:] = torch.tensor([-3e38, 3e38, -1.0, 2e38], device="cuda")
    T = 0.5
    losses, lse, dh, de = _step(mf, h, e, offsets, ids, logits, T, grad)
    hd, ed = h.double(), e.double()
    scores = hd @ ed.T / T
    at = ids.reshape(rows, 4)[:, 1].long()
    log_p = torch.log_softmax(scores, 1)
    want = -T * T * log_p[torch.arange(rows, device="cuda"), at]
    s_off = (76 * 2.0 ** -23 * (hd.abs() @ ed.abs().T) / T).amax(1)
    off = T * T * (2 * s_off + 1000 * 2.0 ** -24 + 2.0 ** -17 * (1 + scores.abs().amax(1)))
    assert bool(((losses.double() - want).abs() <= off).all())
    assert bool(torch.isfinite(dh).all()) and bool(torch.isfinite(de).all())
