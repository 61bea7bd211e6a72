"""GPU tests of accuracies that the losses state beyond the formulas' bounds: up to
64 rows carry d as two 16-bit numbers, and scores are corrected for what the
tensor core's sums drop."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _dtype(kind):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16}[kind]


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("distill", (False, True))
@pytest.mark.parametrize("rows,width", [(1, 64), (5, 64), (32, 64), (33, 64), (64, 64), (1, 648),
                                        (7, 1024), (64, 648)])
def test_few_rows_round_the_result_alone(mf, rows, width, distill, kind):
    """A sum of two 16-bit numbers holds d to u^2 (fp16 to half the step of its
    smallest numbers, 2^-25 of 2^15 over the largest weight).  With scores of a few
    units (error (64 + 4) 2^-23 sum |h e|; wider rows hold zeros), what a gradient
    element is off by is its own rounding, u of it, and little more."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    vocab = 900
    h = torch.randn(rows, width, generator=gen, device="cuda").to(_dtype(kind))
    h[:, 64:] = 0  # products of the others add nothing and drop nothing
    e = (0.5 / 8 * torch.randn(vocab, width, generator=gen, device="cuda")).to(_dtype(kind))
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    grad = 256 * (0.5 + torch.rand(rows, generator=gen, device="cuda"))
    offsets = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    sets = (offsets, targets, torch.zeros(rows, device="cuda"))
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    if distill:
        _, lse = loss.distill(h, *sets)
        dh, de = loss.distill_backward(h, *sets, 1.0, lse, grad)
    else:
        _, lse = loss.cross_entropy(h, targets)
        dh, de = loss.cross_entropy_backward(h, targets, lse, grad)
    torch.cuda.synchronize()
    hd, ed, w = h.double(), e.double(), grad.double()[:, None]
    scores = hd @ ed.T
    p = torch.softmax(scores, 1)
    q = torch.nn.functional.one_hot(targets.long(), vocab).double()
    d, u = w * (p - q), torch.finfo(h.dtype).eps / 2
    # 64 products, and the score correction of the width, up to 3e-9 a product of |s|
    s_off = ((64 + 4) * 2.0 ** -23 * (hd.abs() @ ed.abs().T)
             + width * 3e-9 * scores.abs()).amax(1, keepdim=True)
    lse_off = s_off + vocab * 2.0 ** -24 + 2.0 ** -20 * (1 + torch.logsumexp(scores, 1, True).abs())
    tiny = float(grad.max()) * (2.0 ** -40 if kind == "f16" else 2.0 ** -126)
    d_off = w * ((s_off + lse_off) * p + q * 2.0 ** -19) + u * u * d.abs() + tiny
    small = 2.0 ** -25 if kind == "f16" else 2.0 ** -134
    for got, want, off, terms in (
            (dh, d @ ed, d_off @ ed.abs(), (vocab + 4) * 2.0 ** -23 * (d.abs() @ ed.abs())),
            (de, d.T @ hd, d_off.T @ hd.abs(), (rows + 4) * 2.0 ** -23 * (d.abs().T @ hd.abs()))):
        off = (off + terms) * (1 + u) + u * want.abs() + small
        assert bool(((got.double() - want).abs() <= off).all())


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("rows", (40, 300))
def test_scores_of_parallel_rows(mf, rows, kind):
    """Products of one sign lose the most (fp16 up to 6.1e-9 of the score a product);
    about 3e-9 a product is what the header leaves, on average over the rows (one
    row's lies within a few 4.5e-7 of that)."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    vocab, width = 500, 2048
    e = torch.randn(vocab, width, generator=gen, device="cuda").to(_dtype(kind))
    h = (e[torch.arange(rows, device="cuda") % vocab].float() / 8).to(_dtype(kind))
    none = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    _, lse = loss.cross_entropy(h, none)
    torch.cuda.synchronize()
    want = torch.logsumexp(h.double() @ e.double().T, 1)
    assert float(want.min()) > 200  # the parallel row's score alone
    off = float(((lse.double() - want) / want).mean().abs())
    assert off <= 3.3e-9 * width + 4 * 4.5e-7 / math.sqrt(rows), off / width


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("rows,width,products", [(3, 2048, 1024), (20, 2048, 1024),
                                                 (64, 1024, 512), (64, 2048, 2048),
                                                 (65, 2048, 2048)])
def test_few_rows_sum_scores_in_segments(mf, rows, width, products, kind):
    """The same in distillation, where up to 64 rows sum a score in two segments (as
    long as the hidden rows leave room beside the table's ring: not 64 of 2,048):
    what is left is that of half the products.  The gradients agree with it: of a row
    that is as sure as its teacher, the sum of d stays within lse's rounding and a
    few of numbers near 1."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    vocab = 500
    e = torch.randn(vocab, width, generator=gen, device="cuda")
    e[:, -64:] = 1.0  # shows the sum of d
    e = e.to(_dtype(kind))
    h = (e[:rows].float() / 8).to(_dtype(kind))
    sets = (torch.arange(rows + 1, dtype=torch.int32, device="cuda"),
            torch.arange(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda"))
    loss = mf.DenseLoss(e, rows, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    losses, lse = loss.distill(h, *sets)
    dh, _ = loss.distill_backward(h, *sets, 1.0, lse, torch.ones(rows, device="cuda"),
                                  embedding_grad=False)
    torch.cuda.synchronize()
    want = torch.logsumexp(h.double() @ e.double().T, 1)
    assert float(want.min()) > 100  # the parallel row's score alone: p and the loss are 1 and 0
    off = float(((lse.double() - want) / want).mean().abs())
    assert off <= 3.3e-9 * products + 4 * 4.5e-7 / math.sqrt(rows), off / products
    assert float(losses.abs().max()) <= 2.0 ** -20
    # d is p - 1 at the parallel row, which a clamp keeps at or below 0
    left = 1.5 * 2.0 ** -24 * want + 2.0 ** -20
    assert bool((dh[:, -64:].double().abs().amax(1) <= left * (1 + 2.0 ** -7)).all())


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("width", (1024, 2048))
@pytest.mark.parametrize("cosine", (0.5, 0.7, 0.9))
def test_scores_of_rows_that_lean(mf, cosine, width, kind):
    """The factor that scores are corrected by is between what rows at cosines of 0.5
    and 0.9 lose a product (fp16 2.4e-9 and 4.5e-9, bfloat16 1.1e-9 and 1.8e-9): on
    average over the rows a score is within 1.6e-9 a product, and its own deviation is
    4e-7 at most.  With one column, lse is the score."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(width)
    off = []
    for _ in range(4):  # the loss depends on where the score lies between powers of two
        e = (0.02 * torch.randn(1, width, generator=gen, device="cuda")).to(_dtype(kind))
        along = torch.nn.functional.normalize(e.float())
        x = torch.randn(1000, width, generator=gen, device="cuda")
        across = torch.nn.functional.normalize(x - (x @ along.T) * along)
        h = (math.sqrt(width) * (cosine * along + math.sqrt(1 - cosine ** 2) * across)).to(_dtype(kind))
        loss = mf.DenseLoss(e, 1000, stream=torch.cuda.Stream())
        none = torch.full((1000,), -1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        _, lse = loss.cross_entropy(h, none)
        torch.cuda.synchronize()
        want = (h.double() @ e.double().T)[:, 0]
        off.append((lse.double() - want) / want)
    assert abs(float(torch.cat(off).mean())) <= 1.6e-9 * width + 4 * 4e-7 / math.sqrt(4000)
