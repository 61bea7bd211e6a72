"""GPU tests of gradients over many pieces of the vocabulary: more pieces than
sets of d_hidden's sums, so that later pieces add to sums that earlier ones
wrote, and a short last piece that adds to only some of a set's splits.

A piece is at most 128 MiB of 16-bit d, at 16,384 rows 4,096 columns, and the sums
that are kept apart fill at most 128 MiB as well: at 16,384 x 512 those of four
pieces, at 12,000 x 1,400 those of one.

Tolerances: those of test_gpu_loss.py.  Scores are off by at most (width + 4)
2^-23 sum |h e|, lse by that plus V 2^-24 plus 2^-20 (1 + |lse|); d is rounded once
(u |d|, fp16 also by 2^-40 of the largest weight), the products add in FP32
(2^-23 an addition), the result is rounded once.
"""
from __future__ import annotations

import math

import pytest

from test_gpu_loss import Reference, _near

pytestmark = pytest.mark.gpu

# 7 pieces and 4 sets; 3 and 1; 5 and 4 of 2 splits; 12 and 11 of 2 splits, the last
# piece with one
SHAPES = [(16_384, 28_200, 512), (12_000, 16_000, 1400), (15_958, 16_450, 216),
          (16_392, 43_725, 88)]


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _problem(rows, vocab, width, kind):
    import torch

    dtype = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
    gen = torch.Generator(device="cuda").manual_seed(rows + width)
    h = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
    e = (2.0 / math.sqrt(width) * torch.randn(vocab, width, generator=gen, device="cuda")).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    t[torch.rand(rows, generator=gen, device="cuda") < 0.1] = -1
    grad = (0.5 + torch.rand(rows, generator=gen, device="cuda")) / 64
    return h, e, t, grad


def _step(loss, h, t, grad, **kw):
    import torch

    torch.cuda.synchronize()
    losses, lse = loss.cross_entropy(h, t)
    out = loss.cross_entropy_backward(h, t, lse, grad, **kw)
    torch.cuda.synchronize()
    return losses, lse, *out


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_more_pieces_than_sets_of_sums(mf, rows, vocab, width, kind):
    import torch

    h, e, t, grad = _problem(rows, vocab, width, kind)
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    _, lse, dh, de = _step(loss, h, t, grad)
    u = torch.finfo(h.dtype).eps / 2
    small = 2.0 ** -25 if kind == "f16" else 2.0 ** -134
    ed, ea = e.double(), e.double().abs()
    biggest = float(grad.max())
    tiny = biggest * (2.0 ** -40 if kind == "f16" else 2.0 ** -126)
    want_e = torch.zeros_like(ed)
    off_e = torch.zeros_like(ed)
    for r0 in range(0, rows, 1024):  # bounds and formulas, a part of the rows at a time
        part = slice(r0, min(rows, r0 + 1024))
        hd, tt = h[part].double(), t[part].long()
        has = tt >= 0
        w = torch.where(has, grad[part].double(), 0.0)[:, None]
        hd[~has] = 0
        scores = hd @ ed.T
        s_off = ((width + 4) * 2.0 ** -23 * (hd.abs() @ ea.T)).amax(1)
        lse64 = torch.logsumexp(scores, 1)
        lse_off = s_off + vocab * 2.0 ** -24 + 2.0 ** -20 * (1 + lse64.abs())
        assert bool(((lse[part].double() - lse64).abs() <= lse_off)[has].all())
        d = (scores - lse64[:, None]).exp()
        d_off = (s_off + lse_off)[:, None] * d * w
        at = torch.nonzero(has)[:, 0]
        d[at, tt[at]] -= 1
        d_off[at, tt[at]] += w[at, 0] * 2.0 ** -19
        d *= w
        d_off = d_off * (1 + u) + u * d.abs() + tiny * (w != 0)
        want = d @ ed
        off = (d_off @ ea + (vocab + 4) * 2.0 ** -23 * (d.abs() @ ea)) * (1 + u) \
            + u * want.abs() + small
        assert bool(((dh[part].double() - want).abs() <= off).all())
        want_e += d.T @ hd
        off_e += d_off.T @ hd.abs() + (rows + 4) * 2.0 ** -23 * (d.abs().T @ hd.abs())
        # below fp16's range a weighted hidden element is off by half its last step
        if kind == "f16":
            off_e += 2.0 ** -25 * (d.abs() / w.clamp(min=1e-30)).sum(0)[:, None] * biggest
    off_e = off_e * (1 + u) + u * want_e.abs() + small
    assert bool(((de.double() - want_e).abs() <= off_e).all())


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_same_bits_whatever_the_workspace_held(mf, rows, vocab, width, kind):
    """Also with one gradient alone: the other's products leave no trace."""
    import torch

    h, e, t, grad = _problem(rows, vocab, width, kind)
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    want = _step(loss, h, t, grad)
    for fill in (0xFF, 0x7F, 0x00):  # NaN, huge numbers, nothing
        loss.workspace.fill_(fill)
        got = _step(loss, h, t, grad)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    loss.workspace.fill_(0x7F)
    _, _, dh, none = _step(loss, h, t, grad, embedding_grad=False)
    assert none is None and torch.equal(dh, want[2])
    loss.workspace.fill_(0x7F)
    _, _, none, de = _step(loss, h, t, grad, hidden_grad=False)
    assert none is None and torch.equal(de, want[3])


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("distill", (False, True))
@pytest.mark.parametrize("rows,width", [(16, 648), (40, 72), (64, 136), (65, 72)])
def test_few_rows_over_several_pieces(mf, rows, width, distill, kind):
    """More vocabulary than a piece of one row tile holds (262,144 columns): score
    tiles of two segments, d in two halves and products share a launch."""
    import torch

    vocab = 300_000
    h, e, t, grad = _problem(rows, vocab, width, kind)
    if distill:
        gen = torch.Generator(device="cuda").manual_seed(width)
        ids = torch.randint(0, vocab, (rows, 40), generator=gen, device="cuda").sort(1).values
        keep = torch.ones_like(ids, dtype=torch.bool)
        keep[:, 1:] = ids[:, 1:] != ids[:, :-1]
        offsets = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = keep.sum(1).cumsum(0)
        ids = ids[keep].int()
        kw = dict(sets=(offsets, ids, 2 * torch.randn(ids.numel(), generator=gen, device="cuda")),
                  temperature=1.5)
    else:
        kw = dict(targets=t)
    ref = Reference(h, e, kind, grad=grad, **kw)
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    loss.workspace.fill_(0xFF)
    torch.cuda.synchronize()
    losses, lse = loss.distill(h, *kw["sets"], 1.5) if distill else loss.cross_entropy(h, t)
    torch.cuda.synchronize()
    loss.workspace.fill_(0xFF)
    torch.cuda.synchronize()
    dh, de = (loss.distill_backward(h, *kw["sets"], 1.5, lse, grad) if distill
              else loss.cross_entropy_backward(h, t, lse, grad))
    torch.cuda.synchronize()
    _near(lse, ref.lse, ref.lse_off, "lse")
    _near(losses, ref.losses, ref.losses_off, "losses")
    _near(dh, ref.d_hidden, ref.dh_off, "d_hidden")
    _near(de, ref.d_embedding, ref.de_off, "d_embedding")
