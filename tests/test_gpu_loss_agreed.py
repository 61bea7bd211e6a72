"""GPU tests of distillation where teacher and student are sure of the same id:
p and q are 1 - 1e-3 or so at scores of tens to hundreds, the loss and p - q are
small differences.

Tolerances.  Scores that are off by at most s = (width + 4) 2^-23 sum |h e| move p by
at most 2 p (1 - p) s and the loss by s sum |p - q|, as long as loss, lse and gradients
are made of the same ones.  Beyond that only roundings of numbers near 1 remain:
2^-20 relative of q, log q and exponentials, `steps` additions of 2^-24 in the
sum, and lse's rounding to FP32, 2^-24 |lse|, which the gradient sees.  d is rounded
once (u |d|; fp16 below its range by 2^-40 of the weight; up to 64 rows to two
16-bit numbers), the products add in FP32, the result is rounded once.
"""
from __future__ import annotations

import math

import pytest

from test_gpu_loss import Reference, _near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _dtype(kind):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16}[kind]


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("T", (1.0, 2.0))
@pytest.mark.parametrize("common", (0.0, 60.0, 400.0))
@pytest.mark.parametrize("rows,vocab,width", [(1, 700, 576), (20, 700, 576), (32, 900, 640),
                                              (25, 700, 1024), (48, 700, 576), (64, 3000, 328),
                                              (65, 700, 576), (300, 700, 576)])
def test_agreed_rows(mf, rows, vocab, width, common, T, kind):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows + width)
    half = width // 2
    e = torch.randn(vocab, width, generator=gen, device="cuda")
    e /= e[:, :half].norm(dim=1, keepdim=True)
    e[:, half:] = 1.0  # adds `common` to all scores
    sure = torch.randperm(vocab, generator=gen, device="cuda")[:rows]
    above = T * (10.0 + math.log(vocab) + 4.0 * torch.rand(rows, 1, generator=gen, device="cuda"))
    h = torch.empty(rows, width, device="cuda")
    h[:, :half] = above * e[sure, :half]
    h[:, half:] = T * common / (width - half)
    h, e = h.to(_dtype(kind)), e.to(_dtype(kind))
    ids = torch.stack([sure, (sure + 1) % vocab, (sure + 7) % vocab], 1).sort(1).values
    logits = torch.where(ids == sure[:, None], 8.0 * T, 0.0)
    offsets = (3 * torch.arange(rows + 1, device="cuda")).int()
    sets = (offsets, ids.reshape(-1).int(), logits.reshape(-1).contiguous())
    grad = 128 * (0.5 + torch.rand(rows, generator=gen, device="cuda"))
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    losses, lse = loss.distill(h, *sets, T)
    dh, de = loss.distill_backward(h, *sets, T, lse, grad)
    torch.cuda.synchronize()

    hd, ed, u = h.double(), e.double(), torch.finfo(h.dtype).eps / 2
    q = torch.zeros(rows, vocab, dtype=torch.float64, device="cuda")
    q.scatter_(1, ids, torch.softmax(logits.double() / T, 1))
    scores = hd @ ed.T / T
    lse64 = torch.logsumexp(scores, 1)
    log_p = scores - lse64[:, None]
    p = log_p.exp()
    want = T * T * (torch.special.xlogy(q, q) - q * log_p).sum(1)
    assert 1e-5 < float(want.min()) and float(want.max()) < 0.1 * T * T  # what the case says
    s_off = ((width + 4) * 2.0 ** -23 * (hd.abs() @ ed.abs().T) / T).amax(1)
    steps = vocab // 64 + 16
    size = torch.special.xlogy(q, q).abs().sum(1) + want / (T * T)
    off = T * T * (s_off * (p - q).abs().sum(1) + (2 * steps + 32) * 2.0 ** -24 + 2.0 ** -20 * size)
    _near(losses, want, off, "losses")

    w = T * grad.double()[:, None]
    d = w * (p - q)
    d_off = w * (2 * p * (1 - p) * s_off[:, None] + q * 2.0 ** -20
                 + p * (2.0 ** -24 * (1.5 * lse64.abs() + steps) + 2.0 ** -20)[:, None])
    tiny = float(w.max()) * (2.0 ** -40 if kind == "f16" else 2.0 ** -126)
    d_off = d_off * (1 + u) + u * d.abs() + tiny
    small = 2.0 ** -25 if kind == "f16" else 2.0 ** -134
    for got, want, bound, terms in (
            (dh, d @ ed, d_off @ ed.abs(), (vocab + 4) * 2.0 ** -23 * (d.abs() @ ed.abs())),
            (de, d.T @ hd, d_off.T @ hd.abs(), (rows + 4) * 2.0 ** -23 * (d.abs().T @ hd.abs()))):
        _near(got, want, (bound + terms) * (1 + u) + u * want.abs() + small, "gradients")


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("rows,vocab,width", [(1, 20_000, 64), (8, 20_000, 64), (64, 9000, 72),
                                              (16, 100_000, 64), (48, 40_000, 1024),
                                              (64, 40_000, 1024)])
def test_a_teacher_of_the_whole_vocabulary(mf, rows, vocab, width, kind):
    """More entries in a CTA's range than are listed at a time, more scores than its
    memory takes at once (width 1,024); some rows have few."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    h = torch.randn(rows, width, generator=gen, device="cuda").to(_dtype(kind))
    e = (2.0 / math.sqrt(width) * torch.randn(vocab, width, generator=gen, device="cuda")).to(
        _dtype(kind))
    keep = torch.ones(rows, vocab, dtype=torch.bool, device="cuda")
    keep[3::5] = torch.rand(rows, vocab, generator=gen, device="cuda")[3::5] < 0.01
    keep[4::9] = False
    offsets = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = keep.sum(1).cumsum(0)
    ids = torch.arange(vocab, device="cuda").expand(rows, vocab)[keep].int()
    logits = 3 * torch.randn(ids.numel(), generator=gen, device="cuda")
    logits[torch.rand(ids.numel(), generator=gen, device="cuda") < 0.05] = -math.inf
    sets, grad = (offsets, ids, logits), torch.rand(rows, generator=gen, device="cuda")
    ref = Reference(h, e, kind, sets=sets, temperature=1.5, grad=grad)
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    losses, lse = loss.distill(h, *sets, 1.5)
    dh, de = loss.distill_backward(h, *sets, 1.5, lse, grad)
    torch.cuda.synchronize()
    _near(lse, ref.lse, ref.lse_off, "lse")
    _near(losses, ref.losses, ref.losses_off, "losses")
    _near(dh, ref.d_hidden, ref.dh_off, "d_hidden")
    _near(de, ref.d_embedding, ref.de_off, "d_embedding")


@pytest.mark.parametrize("rows", (5, 40))
def test_sets_that_overlap_and_do_not_ascend(mf, rows):
    """Every row's offsets cover the same entries, in an order that only some rows
    find valid: the invalid ones give NaN and disturb no other row."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(7)
    vocab, width, n = 3000, 64, 4000
    h = torch.randn(rows, width, generator=gen, device="cuda").half()
    e = (torch.randn(vocab, width, generator=gen, device="cuda") / 8).half()
    ids = torch.randint(-5, vocab + 5, (n,), generator=gen, device="cuda", dtype=torch.int32)
    ids[:50] = torch.arange(50, device="cuda") * 60  # ascending
    logits = torch.randn(n, generator=gen, device="cuda")
    offsets = torch.full((rows + 1,), 0, dtype=torch.int32, device="cuda")
    offsets[1::2] = n        # rows 0, 2, ...: all entries; rows 1, 3, ...: decreasing
    offsets[rows - 1:] = torch.tensor([0, 50], device="cuda")  # the last: the ascending ones
    sets, grad = (offsets, ids, logits), torch.ones(rows, device="cuda")
    ref = Reference(h, e, "f16", sets=sets, grad=grad)
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    losses, lse = loss.distill(h, *sets)
    dh, de = loss.distill_backward(h, *sets, 1.0, lse, grad)
    torch.cuda.synchronize()
    assert bool(torch.isnan(losses[:-2]).all()) and bool(torch.isfinite(losses[-1]))
    _near(lse, ref.lse, ref.lse_off, "lse")
    _near(losses, ref.losses, ref.losses_off, "losses")
    _near(dh, ref.d_hidden, ref.dh_off, "d_hidden")
    _near(de, ref.d_embedding, ref.de_off, "d_embedding")


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("rows,width", [(7, 648), (33, 576), (48, 1024), (64, 576)])
def test_same_bits_whatever_the_workspace_held(mf, rows, width, kind):
    """Few rows of either loss, twice, over workspaces of NaN and of huge numbers."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    vocab = 9001
    h = torch.randn(rows, width, generator=gen, device="cuda").to(_dtype(kind))
    e = (2.0 / math.sqrt(width) * torch.randn(vocab, width, generator=gen, device="cuda")).to(
        _dtype(kind))
    t = torch.randint(-1, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    keep = torch.rand(rows, vocab, generator=gen, device="cuda") < 0.02
    offsets = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = keep.sum(1).cumsum(0)
    ids = torch.arange(vocab, device="cuda").expand(rows, vocab)[keep].int()
    sets = (offsets, ids, 2 * torch.randn(ids.numel(), generator=gen, device="cuda"))
    grad = torch.rand(rows, generator=gen, device="cuda") - 0.2
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    runs = []
    for fill in (0xFF, 0x7F):
        out = []
        for call in (lambda: loss.cross_entropy(h, t), lambda: loss.distill(h, *sets, 2.0),
                     lambda: loss.cross_entropy_backward(h, t, out[0][1], grad),
                     lambda: loss.distill_backward(h, *sets, 2.0, out[1][1], grad)):
            loss.workspace.fill_(fill)
            torch.cuda.synchronize()
            out.append(call())
            torch.cuda.synchronize()
        runs.append(out)
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            assert bool(torch.isfinite(x).all()) and torch.equal(x, y)
