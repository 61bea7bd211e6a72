"""GPU tests of the losses over a table with masked rows: a bias column (1 in
every hidden row) holds -inf, bfloat16's lowest value or -1e10 in the table rows that
no row may choose, so that whole walks begin with such scores.

Tolerances are those of test_gpu_loss.py: a score is off by at most (width + 4)
2^-23 sum |h e| over the unmasked columns, lse by that plus V 2^-24 plus 2^-20
(1 + |lse|), a loss by both; d adds one rounding (u |d|) and the products 2^-23
an addition, and the result is rounded once more.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

LOWEST = -3.3895313892515355e38  # bfloat16


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _problem(rows, vocab, width, kind, value, masked):
    """Hidden rows, table with `value` in column 0 of masked rows, and the same
    table in 64 bits with 0 there."""
    import torch

    dtype = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    h = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
    h[:, 0] = 1.0
    e = (2.0 / math.sqrt(width) * torch.randn(vocab, width, generator=gen, device="cuda")).to(dtype)
    e[:, 0] = 0.0
    clean = e.double()
    e[masked, 0] = value
    return h, e, clean, gen


class Exact:
    def __init__(self, h, clean, masked, T=1.0):
        import torch

        hd = h.double()
        width, vocab = h.shape[1], clean.shape[0]
        self.scores = hd @ clean.T / T
        self.scores[:, masked] = -math.inf
        self.s_off = ((width + 4) * 2.0 ** -23 * (hd.abs() @ clean.abs().T) / T).amax(1)
        self.lse = torch.logsumexp(self.scores, 1)
        self.lse_off = self.s_off + vocab * 2.0 ** -24 + 2.0 ** -20 * (1 + self.lse.abs())


def _near(got, want, off, what):
    import torch

    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))  # infinities, NaN
    bad = ~same & ~((got - want).abs() <= off)
    assert not bool(bad.any()), (what, torch.nonzero(bad)[:4].tolist(), got[bad][:4].tolist(),
                                 want[bad][:4].tolist())


VALUES = [("f16", -math.inf), ("bf16", -math.inf), ("bf16", LOWEST), ("bf16", -1e10)]
# the masked part: the first columns of every walk, all but a few in the middle, the end
MASKS = {"first": lambda v: slice(0, v // 2), "most": lambda v: [i for i in range(v) if i // 3 != v // 6],
         "last": lambda v: slice(v // 2, v)}


@pytest.mark.parametrize("kind,value", VALUES)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("rows", (1, 30, 64, 65, 300))
def test_masked_table_rows(mf, rows, mask, kind, value):
    import torch

    vocab, width = 4099, 72
    masked = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    masked[MASKS[mask](vocab)] = True
    h, e, clean, gen = _problem(rows, vocab, width, kind, value, masked)
    exact = Exact(h, clean, masked)
    open_ids = torch.nonzero(~masked)[:, 0]
    pick = torch.randint(0, open_ids.numel(), (rows,), generator=gen, device="cuda")
    targets = open_ids[pick].int()
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    inside[1::4] = True  # these ask for a masked id
    targets[inside] = torch.nonzero(masked)[:, 0][rows % 7].int()
    stream = torch.cuda.Stream()
    loss = mf.DenseLoss(e, rows, stream=stream)
    torch.cuda.synchronize()
    losses, lse = loss.cross_entropy(h, targets)
    torch.cuda.synchronize()
    _near(lse, exact.lse, exact.lse_off, "lse")
    at = exact.scores[torch.arange(rows, device="cuda"), targets.long()]
    want = exact.lse - at  # +inf where the target is masked
    if value != -math.inf:  # lse - value, which may be infinite too
        assert bool((losses[inside] > -0.99 * value).all())
        losses[inside] = math.inf
    _near(losses, want, exact.lse_off + exact.s_off + 18 * 2.0 ** -22 * (1 + at.abs() + exact.lse.abs()),
          "losses")


@pytest.mark.parametrize("kind,value", VALUES)
@pytest.mark.parametrize("rows", (30, 64, 65, 300))
def test_teacher_over_a_masked_table(mf, rows, kind, value):
    """Sets of unmasked ids, and in some rows a masked one: its loss is +inf (of
    a finite value T q of it, and q > 0.005 of four logits within a few units over
    T = 2), or what the others give where the teacher masks it too."""
    import torch

    vocab, width, T = 4099, 72, 2.0
    masked = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    masked[:3000] = True
    h, e, clean, gen = _problem(rows, vocab, width, kind, value, masked)
    exact = Exact(h, clean, masked, T)
    ids = torch.tensor([[2000 + r % 5, 3100, 3101 + r % 50, 4000] for r in range(rows)], device="cuda")
    logits = torch.randn(rows, 4, generator=gen, device="cuda")
    asked = torch.zeros(rows, dtype=torch.bool, device="cuda")
    asked[1::4] = True
    logits[~asked, 0] = -math.inf
    offsets = (4 * torch.arange(rows + 1, device="cuda")).int()
    stream = torch.cuda.Stream()
    loss = mf.DenseLoss(e, rows, stream=stream)
    torch.cuda.synchronize()
    losses, lse = loss.distill(h, offsets, ids.reshape(-1).int(), logits.reshape(-1), T)
    torch.cuda.synchronize()
    _near(lse, exact.lse, exact.lse_off, "lse")
    q = torch.softmax(logits.double() / T, 1)
    s = exact.scores.gather(1, ids)
    log_p = torch.where(q > 0, s - exact.lse[:, None], torch.zeros_like(s))
    want = T * T * (torch.special.xlogy(q, q) - q * log_p).sum(1)
    assert bool(torch.isinf(want[asked]).all()) and bool(torch.isfinite(want[~asked]).all())
    if value != -math.inf:  # the score is finite, and so may T^2 q times it be
        assert bool((losses[asked] > -0.01 * value).all())
        losses[asked] = math.inf
    size = torch.where(q > 0, q * (q.log().abs() + s.abs()), torch.zeros_like(s)).sum(1)
    off = T * T * (exact.s_off + exact.lse_off + 20 * 2.0 ** -22 * (1 + size + exact.lse.abs()))
    _near(losses, want, torch.where(asked, torch.zeros_like(off), off), "losses")


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("rows", (30, 64, 65, 300))
def test_rows_without_any_score(mf, rows, kind):
    """Every score -inf: lse -inf and a NaN loss; a NaN among them: both NaN."""
    import torch

    vocab, width = 700, 72
    masked = torch.ones(vocab, dtype=torch.bool, device="cuda")
    h, e, _, _ = _problem(rows, vocab, width, kind, -math.inf, masked)
    h[2, 1] = math.nan
    targets = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    losses, lse = loss.cross_entropy(h, targets)
    torch.cuda.synchronize()
    others = torch.arange(rows, device="cuda") != 2
    assert bool(torch.isnan(losses).all()) and math.isnan(float(lse[2]))
    assert bool((lse[others] == -math.inf).all())


@pytest.mark.parametrize("value", (LOWEST, -1e10))
@pytest.mark.parametrize("rows", (30, 64, 65, 300))
def test_gradients_over_a_masked_table(mf, rows, value):
    """A finite value masks: p is 0 there, and so are its gradients."""
    import torch

    vocab, width, u = 4099, 72, 2.0 ** -8
    masked = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    masked[:2500] = True
    h, e, clean, gen = _problem(rows, vocab, width, "bf16", value, masked)
    exact = Exact(h, clean, masked)
    targets = torch.randint(2500, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    grad = 0.5 + torch.rand(rows, generator=gen, device="cuda")
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    _, lse = loss.cross_entropy(h, targets)
    dh, de = loss.cross_entropy_backward(h, targets, lse, grad)
    torch.cuda.synchronize()
    hd, w = h.double(), grad.double()[:, None]
    p = (exact.scores - exact.lse[:, None]).exp()
    q = torch.nn.functional.one_hot(targets.long(), vocab).double()
    d = w * (p - q)
    d_off = ((exact.s_off + exact.lse_off)[:, None] * p * w + q * w * 2.0 ** -19) * (1 + u) \
        + u * d.abs() + float(grad.max()) * 2.0 ** -126
    d_off[:, masked] = 0  # an exponential of -inf is 0
    want_h, want_e = d @ clean, d.T @ hd
    off_h = d_off @ clean.abs() + (vocab + 4) * 2.0 ** -23 * (d.abs() @ clean.abs())
    off_e = d_off.T @ hd.abs() + (rows + 4) * 2.0 ** -23 * (d.abs().T @ hd.abs())
    # a hidden row carries a power of two of its weight, exact in bfloat16
    _near(dh, want_h, off_h * (1 + u) + u * want_h.abs() + 2.0 ** -134, "d_hidden")
    _near(de, want_e, off_e * (1 + u) + u * want_e.abs() + 2.0 ** -134, "d_embedding")
    assert not bool(de[masked].any())
