"""GPU tests of the gradients of sure rows: 1 - p of the target between 1e-6 and
1e-2 at scores of tens to hundreds, where p - 1 is a difference of two numbers
that are nearly equal.

Tolerances.  u is half a step of the 16-bit type.  The truth is 1 - p =
sum over the others of exp(s - lse), so an error of x in the scores is one of
x (1 - p) in it.  lse is an FP32 number that lies within half a step of
score + loss, 2^-24 |lse|, and the loss within `steps` additions and a few
roundings of 1 (2^-24 each): absolute errors of p, and the only ones beside the
relative ones.  A score is off by at most (width + 4) 2^-23 sum |h e|, as
elsewhere.  d is rounded once (u |d|; fp16 below its range by 2^-40 of the
weight), the products add in FP32, and the result is rounded once.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _problem(rows, vocab, width, kind, common):
    """Rows parallel to their target's table row, 8 to 20 above the others, and a
    part of the width that adds `common` to all scores."""
    import torch

    dtype = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
    gen = torch.Generator(device="cuda").manual_seed(rows + width)
    half = width // 2
    e = torch.randn(vocab, width, generator=gen, device="cuda")
    e /= e[:, :half].norm(dim=1, keepdim=True)
    e[:, half:] = 1.0
    targets = torch.randperm(vocab, generator=gen, device="cuda")[:rows]
    # the others' scores have mean 0 and a standard deviation of above / sqrt(half)
    above = 8.0 + math.log(vocab) + 8.0 * torch.rand(rows, 1, generator=gen, device="cuda")
    h = torch.empty(rows, width, device="cuda")
    h[:, :half] = above * e[targets, :half]
    h[:, half:] = common / (width - half)
    return h.to(dtype), e.to(dtype), targets.int(), gen


SHAPES = [(7, 300, 576), (30, 700, 128), (33, 700, 576), (64, 700, 576), (100, 700, 576),
          (600, 1500, 576), (260, 1000, 1024)]


def _check(mf, h, e, targets, kind, grad):
    import torch

    rows, width = h.shape
    vocab = e.shape[0]
    hd, ed = h.double(), e.double()
    scores = hd @ ed.T
    lse64 = torch.logsumexp(scores, 1)
    at = torch.arange(rows, device="cuda")
    log_p = scores - lse64[:, None]
    p = log_p.exp()
    d = p.clone()
    d[at, targets.long()] = 0
    short = d.sum(1)  # 1 - p of the target, without the difference
    d[at, targets.long()] = -short
    d *= grad.double()[:, None]
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    losses, lse = loss.cross_entropy(h, targets)
    dh, de = loss.cross_entropy_backward(h, targets, lse, grad)
    torch.cuda.synchronize()
    u = torch.finfo(h.dtype).eps / 2
    s_off = (width + 4) * 2.0 ** -23 * (hd.abs() @ ed.abs().T).amax(1)
    steps = vocab // 64 + 16
    sure = 2.0 ** -24 * (lse64.abs() + 2 * steps)
    # the target's element, and the others'
    w = grad.double()[:, None]
    d_off = (2 * s_off + sure + 2.0 ** -20 * (1 + lse64.abs()))[:, None] * d.abs()
    d_off[at, targets.long()] += grad.double() * sure
    tiny = float(grad.max()) * (2.0 ** -40 if kind == "f16" else 2.0 ** -126)
    d_off = d_off * (1 + u) + u * d.abs() + tiny
    small = 2.0 ** -25 if kind == "f16" else 2.0 ** -134
    out = []
    for got, want, off, terms in (
            (dh, d @ ed, d_off @ ed.abs(), (vocab + 4) * 2.0 ** -23 * (d.abs() @ ed.abs())),
            (de, d.T @ hd, d_off.T @ hd.abs(), (rows + 4) * 2.0 ** -23 * (d.abs().T @ hd.abs()))):
        off = (off + terms) * (1 + u) + u * want.abs() + small
        out.append(((got.double() - want).abs() / off).max())
    loss_off = sure + 2 * s_off * short + 2.0 ** -20 * short
    out.append(((losses.double() + log_p[at, targets.long()]).abs() / loss_off).max())
    return [float(x) for x in out], short


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("common", (0.0, 60.0, 400.0))
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_sure_rows(mf, rows, vocab, width, common, kind):
    import torch

    h, e, targets, gen = _problem(rows, vocab, width, kind, common)
    grad = (0.5 + torch.rand(rows, generator=gen, device="cuda")) * 256
    worst, short = _check(mf, h, e, targets, kind, grad)
    assert 1e-7 < float(short.min()) and float(short.max()) < 1e-2  # the cases are what they say
    assert max(worst) <= 1, worst
