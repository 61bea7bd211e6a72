"""GPU tests of the losses over the tied table (include/mf_loss.h) against the
formulas in 64 bits.

Tolerances.  u is half a step of the 16-bit type (fp16 2^-11, bf16 2^-8).  A
score is a sum of `width` products, each exact in FP32, summed in FP32 by
additions that may truncate: off by at most width 2^-23 sum |h e|, the same
over T for s / T, plus two roundings.  exp, log and their arguments are good to
2^-20 relative of the term, so lse is off by at most the score's bound plus
V 2^-24 (the additions of the sum, each a rounding) plus 2^-20 (1 + |lse|).
p is then off by (score's bound + lse's bound) p.  d is rounded once
(u |d|, below fp16's smallest normal number by 2^-25 of it), the products add
in FP32 (2^-23 an addition), and the result is rounded once to the 16-bit
type.  Each bound is computed element by element below.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from helpers import INVALID, gpu_stream

pytestmark = pytest.mark.gpu

TYPES = ("f16", "bf16")


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _dtype(kind):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16}[kind]


def _half_step(kind):
    import torch

    return torch.finfo(_dtype(kind)).eps / 2


def _problem(seed, rows, vocab, width, kind, sharp=1.0):
    """Hidden rows and table; `sharp` scales the scores' spread."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, width, generator=gen, device="cuda").to(_dtype(kind))
    e = (sharp / math.sqrt(width) * torch.randn(vocab, width, generator=gen, device="cuda")).to(
        _dtype(kind))
    return h, e, gen


def _targets(gen, rows, vocab, ignored):
    import torch

    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    return torch.where(torch.rand(rows, generator=gen, device="cuda") < ignored, -1, t).int()


def _sets(gen, rows, vocab, most, empty=0.1, masked=0.05):
    """Ragged ascending sets: some empty, some entries at -inf."""
    import torch

    most = min(most, vocab)
    ids = torch.rand(rows, vocab, generator=gen, device="cuda").topk(most, 1).indices.sort(1).values
    length = torch.randint(1, most + 1, (rows, 1), generator=gen, device="cuda")
    keep = torch.rand(rows, most, generator=gen, device="cuda").argsort(1) < length
    keep &= torch.rand(rows, 1, generator=gen, device="cuda") >= empty
    logits = 2.0 * torch.randn(rows, most, generator=gen, device="cuda")
    logits[torch.rand(rows, most, generator=gen, device="cuda") < masked] = -math.inf
    offsets = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = keep.sum(1).cumsum(0)
    return offsets, ids[keep].int(), logits[keep]


def _wanted(h, vocab, targets=None, sets=None, temperature=1.0):
    """(q [rows, vocab] in 64 bits, rows with a target, invalid rows)."""
    import torch

    rows = h.shape[0]
    q = torch.zeros(rows, vocab, dtype=torch.float64, device="cuda")
    invalid = torch.zeros(rows, dtype=torch.bool, device="cuda")
    if targets is not None:
        has = (targets >= 0) & (targets < vocab)
        invalid = ~has & (targets != -1)
        at = torch.nonzero(has)[:, 0]
        q[at, targets[at].long()] = 1.0
        return q, has, invalid
    offsets, ids, logits = sets
    has = torch.zeros_like(invalid)
    off = offsets.tolist()
    for r in range(rows):
        a, b = off[r], off[r + 1]
        if a < 0 or b < a or b > ids.numel():
            invalid[r] = True
            continue
        i, t = ids[a:b].long(), logits[a:b].double()
        if i.numel() and (bool((i[1:] <= i[:-1]).any()) or int(i.min()) < 0 or int(i.max()) >= vocab
                          or bool(torch.isnan(t).any()) or bool((t == math.inf).any())):
            invalid[r] = True
        elif bool((t > -math.inf).any()):
            has[r] = True
            q[r, i] = torch.softmax(t / temperature, 0)
    return q, has, invalid


class Reference:
    """Losses, lse and gradients in 64 bits with an error bound for each."""

    def __init__(self, h, e, kind, targets=None, sets=None, temperature=1.0, grad=None):
        import torch

        T, u = temperature, _half_step(kind)
        hd, ed = h.double(), e.double()
        rows, width = h.shape
        vocab = e.shape[0]
        q, has, invalid = _wanted(h, vocab, targets, sets, T)
        scores = hd @ ed.T / T
        s_off = ((width + 4) * 2.0 ** -23 * (hd.abs() @ ed.abs().T) / T).amax(1)
        self.lse = torch.logsumexp(scores, 1)
        self.lse_off = s_off + vocab * 2.0 ** -24 + 2.0 ** -20 * (1 + self.lse.abs())
        log_p = scores - self.lse[:, None]
        cross = (torch.special.xlogy(q, q) - q * log_p).sum(1)
        self.losses = torch.where(has, T * T * cross, torch.zeros_like(cross))
        self.losses[invalid] = math.nan
        # q's own logarithms and weights: 2^-20 relative of |log q| + |s| + |lse|
        size = (q * (torch.special.xlogy((q > 0).double(), q).abs() + scores.abs())).sum(1)
        terms = q.count_nonzero(1)
        self.losses_off = T * T * (s_off + self.lse_off
                                   + (terms + 16) * 2.0 ** -22 * (1 + size + self.lse.abs()))
        if grad is None:
            return
        w = torch.where(has, grad.double(), torch.zeros_like(self.lse)) * T
        p = log_p.exp()
        d = w[:, None] * (p - q)
        d[w == 0] = 0
        hz, = (torch.where((w == 0)[:, None], torch.zeros_like(hd), hd),)
        self.d_hidden, self.d_embedding = d @ ed, d.T @ hz
        biggest = float(w.abs().max())
        # d as it enters the products: p's own error, then one rounding; fp16
        # holds d / (largest weight) times 2^15
        d_off = (s_off + self.lse_off)[:, None] * p * w.abs()[:, None] \
            + q * w.abs()[:, None] * 2.0 ** -19
        # an exponential below 2^-126, FP32's smallest normal number, may come out
        # as 0 (p <= 2^-126 is then off by all of itself): for bf16, whose range is
        # FP32's, that is the floor of d; fp16's own 2^-25 2^-15 lies far above it
        tiny = biggest * 2.0 ** -40 if kind == "f16" else biggest * 2.0 ** -126
        d_off = d_off * (1 + u) + u * d.abs() + tiny * (w != 0)[:, None]
        # a hidden row carries its weight's power of two: exact but below fp16's range
        h_off = (2.0 ** -25 if kind == "f16" else 2.0 ** -133) * (
            1 if float(w.abs()[w != 0].min() if bool((w != 0).any()) else 1) < biggest / 2 else 0)
        self.dh_off = d_off @ ed.abs() + (vocab + 4) * 2.0 ** -23 * (d.abs() @ ed.abs())
        self.de_off = d_off.T @ hz.abs() + (rows + 4) * 2.0 ** -23 * (d.abs().T @ hz.abs()) \
            + h_off * biggest
        small = 2.0 ** -25 if kind == "f16" else 2.0 ** -134
        self.dh_off = self.dh_off * (1 + u) + u * self.d_hidden.abs() + small
        self.de_off = self.de_off * (1 + u) + u * self.d_embedding.abs() + small


def _near(got, want, off, what):
    import torch

    got = got.double()
    bad = torch.isnan(want) != torch.isnan(got)
    assert not bool(bad.any()), f"{what}: NaN where none belongs, or none where one does"
    fine = ~torch.isnan(want)
    over = ((got - want).abs() - off)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, (
        f"{what}: off by {float((got - want).abs()[fine].max()):.3g}, "
        f"beyond the bound by {float(over.max()):.3g} "
        f"at {torch.nonzero((got - want).abs() > off)[:4].tolist()}")


def _forward(mf, h, e, targets=None, sets=None, temperature=1.0):
    import torch

    loss = mf.DenseLoss(e, h.shape[0], stream=gpu_stream())
    out = (loss.cross_entropy(h, targets) if targets is not None
           else loss.distill(h, *sets, temperature))
    torch.cuda.synchronize()
    return loss, out


def _backward(mf, loss, h, lse, grad, targets=None, sets=None, temperature=1.0, **kw):
    import torch

    torch.cuda.synchronize()
    out = (loss.cross_entropy_backward(h, targets, lse, grad, **kw) if targets is not None
           else loss.distill_backward(h, *sets, temperature, lse, grad, **kw))
    torch.cuda.synchronize()
    return out


def _check(mf, h, e, kind, grad, targets=None, sets=None, temperature=1.0):
    ref = Reference(h, e, kind, targets, sets, temperature, grad)
    loss, (losses, lse) = _forward(mf, h, e, targets, sets, temperature)
    _near(lse, ref.lse, ref.lse_off, "lse")
    _near(losses, ref.losses, ref.losses_off, "losses")
    dh, de = _backward(mf, loss, h, lse, grad, targets, sets, temperature)
    assert dh.dtype == h.dtype and de.dtype == e.dtype
    _near(dh, ref.d_hidden, ref.dh_off, "d_hidden")
    _near(de, ref.d_embedding, ref.de_off, "d_embedding")
    return ref, loss, losses, lse, dh, de


# rows, vocabulary, width: single values, tile edges on both sides, odd ones
SHAPES = [(1, 1, 8), (1, 17, 64), (2, 300, 72), (3, 8, 576), (63, 127, 64), (64, 128, 128),
          (65, 129, 136), (127, 255, 576), (128, 256, 192), (129, 257, 200), (255, 511, 328),
          (256, 512, 576), (257, 513, 584), (300, 4099, 64), (520, 1000, 1024), (1, 5000, 2048),
          (16, 95, 8), (17, 4800, 640), (32, 20_011, 576), (31, 45_000, 200), (33, 600, 576)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_cross_entropy(mf, rows, vocab, width, kind):
    import torch

    h, e, gen = _problem(rows + vocab, rows, vocab, width, kind, 2.0)
    targets = _targets(gen, rows, vocab, 0.2 if rows > 1 else 0.0)
    grad = 0.5 + torch.rand(rows, generator=gen, device="cuda")
    _check(mf, h, e, kind, grad, targets=targets)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("most,temperature", [(1, 1.0), (40, 2.0), (700, 0.7)])
@pytest.mark.parametrize("rows,vocab,width", [s for s in SHAPES if s[1] <= 1000 or s[0] in (17, 32)])
def test_distill(mf, rows, vocab, width, most, temperature, kind):
    import torch

    h, e, gen = _problem(rows + vocab + most, rows, vocab, width, kind, 2.0)
    sets = _sets(gen, rows, vocab, most, empty=0.1 if rows > 1 else 0.0)
    grad = torch.rand(rows, generator=gen, device="cuda") - 0.3  # weights of both signs
    _check(mf, h, e, kind, grad, sets=sets, temperature=temperature)


@pytest.mark.parametrize("kind", TYPES)
def test_several_pieces(mf, kind):
    """More vocabulary than one piece of d holds (8,192 rows: 16,384 columns),
    the last piece a ragged one."""
    import torch

    rows, vocab, width = 8192, 33_000, 64
    h, e, gen = _problem(5, rows, vocab, width, kind, 2.0)
    targets = _targets(gen, rows, vocab, 0.1)
    grad = (0.5 + torch.rand(rows, generator=gen, device="cuda")) / 64
    _check(mf, h, e, kind, grad, targets=targets)


@pytest.mark.parametrize("kind", TYPES)
def test_wide_and_long(mf, kind):
    """The table of the benchmark (49,152 x 576) with a batch that is no
    multiple of anything, and a teacher set over several thousand ids."""
    import torch

    h, e, gen = _problem(8, 333, 49_152, 576, kind, 3.0)
    grad = torch.rand(333, generator=gen, device="cuda")
    _check(mf, h, e, kind, grad, targets=_targets(gen, 333, 49_152, 0.1))
    _check(mf, h, e, kind, grad, sets=_sets(gen, 333, 49_152, 5000), temperature=1.5)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (100, 25))
def test_confident_rows(mf, kind, rows):
    """Scores far apart: p is 0 or 1 to the last bit in many places, and lse is
    far from 0 on both sides."""
    import torch

    h, e, gen = _problem(11, rows, 700, 128, kind, 60.0)
    targets = _targets(gen, rows, 700, 0.1)
    right = (h.float() @ e.float().T).argmax(1).int()
    targets[:rows // 2] = right[:rows // 2]  # some are right
    _check(mf, h, e, kind, torch.ones(rows, device="cuda"), targets=targets)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (100, 25))
def test_scores_of_hundreds_of_millions(mf, kind, rows):
    """Scores of 3.5e8, whose errors are beyond an exponential's range: losses and
    gradients stay finite and within the formulas' bounds, a sure row's loss is 0."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(21)
    e = (100.0 * torch.randn(700, 576, generator=gen, device="cuda").sign()).to(_dtype(kind))
    right = torch.randint(0, 700, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    h = (e[right.long()] * 60).contiguous()
    targets = _targets(gen, rows, 700, 0.1)
    targets[:rows // 2] = right[:rows // 2]
    _, _, losses, _, _, _ = _check(mf, h, e, kind, torch.full((rows,), 1e-3, device="cuda"),
                                   targets=targets)
    assert not bool(losses[:rows // 2].any())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (100, 25))
def test_sure_rows_lose_no_less_than_nothing(mf, kind, rows):
    """A loss is lse's distance from a score that it contains, however far the
    rounding of scores of 1,000 goes."""
    import torch

    h, e, gen = _problem(22, rows, 3000, 576, kind, 2.0)
    right = torch.randint(0, 3000, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    h = (e[right.long()].float() * 400).to(_dtype(kind))
    loss, (losses, lse) = _forward(mf, h, e, right)
    # e^(-loss) is a share of a sum of at least its own term: a few roundings of 1
    assert float(losses.min()) >= -2.0 ** -20


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (300, 64, 30))
def test_one_target_for_all_rows(mf, kind, rows):
    import torch

    h, e, _ = _problem(23, rows, 5000, 128, kind, 2.0)
    _check(mf, h, e, kind, torch.ones(rows, device="cuda"),
           targets=torch.full((rows,), 4999, device="cuda", dtype=torch.int32))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", (1.0, 1e-6, 4096.0))
@pytest.mark.parametrize("rows", (200, 30))
def test_weights_over_a_wide_range(mf, kind, scale, rows):
    """Weights from 1 down to 2^-12, zeros and negative ones among them."""
    import torch

    h, e, gen = _problem(12, rows, 900, 96, kind, 2.0)
    grad = scale * torch.exp2(-12 * torch.rand(rows, generator=gen, device="cuda"))
    grad[::7] = 0
    grad[::5] *= -1
    ref, _, _, _, dh, _ = _check(mf, h, e, kind, grad, targets=_targets(gen, rows, 900, 0.1))
    assert not bool(dh[::7].any())


def _poisoned(kind, rows):
    """Rows that do not take part hold NaN and infinities."""
    h, e, gen = _problem(13, rows, 500, 64, kind, 2.0)
    clean = h.clone()
    h[3:9] = math.nan
    h[20::10] = math.inf
    return h, clean, e, gen


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (150, 28))
def test_masked_rows_hold_anything(mf, kind, rows):
    import torch

    h, clean, e, gen = _poisoned(kind, rows)
    bad = ~torch.isfinite(h).all(1)
    targets = _targets(gen, rows, 500, 0.0)
    targets[bad] = -1
    targets[torch.nonzero(bad)[0, 0]] = 700     # invalid
    grad = torch.ones(rows, device="cuda")
    grad[3:9] = math.nan                        # of masked rows: not read
    live = torch.where(bad, torch.zeros_like(grad), grad)
    targets[4], grad[4] = 17, 0.0               # a target, but no weight
    ref = Reference(clean, e, kind, targets, None, 1.0, live)
    loss, (losses, lse) = _forward(mf, h, e, targets)
    assert math.isnan(float(losses[3])) and math.isnan(float(losses[4]))
    rest = torch.arange(rows, device="cuda") > 4
    _near(losses[rest], ref.losses[rest], ref.losses_off[rest], "losses")
    dh, de = _backward(mf, loss, h, lse, grad, targets)
    assert not bool(dh[bad].any())
    _near(dh, ref.d_hidden, ref.dh_off, "d_hidden")
    _near(de, ref.d_embedding, ref.de_off, "d_embedding")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,bad", [(140, 77), (19, 8)])
def test_non_finite_rows_stay_their_own(mf, kind, rows, bad):
    """A NaN hidden row that takes part: its loss and gradient are NaN, the
    other rows' are not."""
    import torch

    h, e, gen = _problem(14, rows, 300, 64, kind, 2.0)
    targets = _targets(gen, rows, 300, 0.0)
    grad = torch.ones(rows, device="cuda")
    ref = Reference(h, e, kind, targets, None, 1.0, grad)
    h[bad, 5] = math.nan
    loss, (losses, lse) = _forward(mf, h, e, targets)
    others = torch.arange(rows, device="cuda") != bad
    assert math.isnan(float(losses[bad])) and math.isnan(float(lse[bad]))
    _near(losses[others], ref.losses[others], ref.losses_off[others], "losses")
    dh, de = _backward(mf, loss, h, lse, grad, targets)
    assert bool(torch.isnan(dh[bad]).all()) and bool(torch.isnan(de).all())
    _near(dh[others], ref.d_hidden[others], ref.dh_off[others], "d_hidden")


@pytest.mark.parametrize("rows", (40, 20))
def test_infinite_weight_spoils_its_own_row(mf, rows):
    import torch

    h, e, gen = _problem(15, rows, 300, 64, "f16", 2.0)
    targets = _targets(gen, rows, 300, 0.0)
    grad = torch.ones(rows, device="cuda")
    ref = Reference(h, e, "f16", targets, None, 1.0, grad)
    grad[9] = math.inf
    loss, (_, lse) = _forward(mf, h, e, targets)
    dh, de = _backward(mf, loss, h, lse, grad, targets)
    others = torch.arange(rows, device="cuda") != 9
    assert not bool(torch.isfinite(dh[9]).any()) and not bool(torch.isfinite(de).all())
    _near(dh[others], ref.d_hidden[others], ref.dh_off[others], "d_hidden")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (70, 7))
def test_nothing_takes_part(mf, kind, rows):
    """Every row ignored, or every weight 0: losses and gradients are 0."""
    import torch

    h, e, gen = _problem(16, rows, 300, 64, kind)
    none = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    loss, (losses, lse) = _forward(mf, h, e, none)
    assert not bool(losses.any())
    for targets, grad in ((none, torch.ones(rows, device="cuda")),
                          (_targets(gen, rows, 300, 0.0), torch.zeros(rows, device="cuda"))):
        dh, de = _backward(mf, loss, h, lse, grad, targets)
        assert not bool(dh.any()) and not bool(de.any())


@pytest.mark.parametrize("kind", TYPES)
def test_rows_of_a_teacher_that_say_nothing_or_wrong(mf, kind):
    """Empty sets, sets of -inf, repeated, unsorted and foreign ids, NaN and
    +inf logits, offsets that decrease or point past the entries."""
    import torch

    rows, vocab = 12, 200
    h, e, gen = _problem(17, rows, vocab, 64, kind, 2.0)
    row_ids = [[1, 5, 150], [], [7, 9], [4, 4], [9, 3], [-1, 3], [3, 200], [0, 199], [2], [8, 60],
               [130, 140], [10]]
    logits = [[1.0, -2.0, 0.5], [], [-math.inf] * 2, [1.0, 2.0], [1.0, 2.0], [0.0, 0.0],
              [0.0, 0.0], [-math.inf, 3.0], [math.nan], [math.inf, 0.0], [50.0, -80.0], [1.0]]
    off = np.cumsum([0] + [len(r) for r in row_ids])
    sets = (torch.tensor(off, dtype=torch.int32, device="cuda"),
            torch.tensor(sum(row_ids, []), dtype=torch.int32, device="cuda"),
            torch.tensor(sum(logits, []), dtype=torch.float32, device="cuda"))
    grad = torch.ones(rows, device="cuda")
    _, _, losses, _, dh, _ = _check(mf, h, e, kind, grad, sets=sets, temperature=1.5)
    invalid = [3, 4, 5, 6, 8, 9]
    assert bool(torch.isnan(losses[invalid]).all())
    assert not bool(dh[invalid + [1, 2]].any()) and losses[1] == 0 and losses[2] == 0
    bad = sets[0].clone()
    bad[5], bad[12] = 2, 1000
    _, _, losses, _, _, _ = _check(mf, h, e, kind, grad, sets=(bad, *sets[1:]))
    assert math.isnan(float(losses[4])) and math.isnan(float(losses[11]))


@pytest.mark.parametrize("kind", TYPES)
def test_no_entries_at_all(mf, kind):
    import torch

    h, e, _ = _problem(18, 5, 100, 64, kind)
    sets = (torch.zeros(6, dtype=torch.int32, device="cuda"),
            torch.empty(0, dtype=torch.int32, device="cuda"),
            torch.empty(0, dtype=torch.float32, device="cuda"))
    _check(mf, h, e, kind, torch.ones(5, device="cuda"), sets=sets)


def test_distillation_of_one_sure_token_is_cross_entropy(mf):
    import torch

    h, e, gen = _problem(19, 90, 400, 64, "f16", 2.0)
    targets = _targets(gen, 90, 400, 0.0)
    sets = (torch.arange(91, dtype=torch.int32, device="cuda"), targets,
            torch.zeros(90, device="cuda"))
    grad = torch.rand(90, generator=gen, device="cuda")
    _, (a, lse_a) = _forward(mf, h, e, targets)
    loss, (b, lse_b) = _forward(mf, h, e, None, sets)
    # the target's score is summed with rounding to nearest in one and by the
    # tensor core in the other: both lie within the formula's bounds
    ref = Reference(h, e, "f16", targets)
    for lse, losses in ((lse_a, a), (lse_b, b)):
        _near(lse, ref.lse, ref.lse_off, "lse")
        _near(losses, ref.losses, ref.losses_off, "losses")
    x = _backward(mf, loss, h, lse_a, grad, targets)
    y = _backward(mf, loss, h, lse_a, grad, None, sets)
    u = _half_step("f16")
    for i, j in zip(x, y):  # p - 1 and p - exp(0 - log 1) round alike up to a last bit
        torch.testing.assert_close(i, j, rtol=4 * u, atol=4 * u * float(i.abs().max()))


@pytest.mark.parametrize("distill", (False, True))
def test_gradient_against_differences(mf, distill):
    """Central differences of the operator's own losses.  Along a step x of
    one side the row's loss is smooth, with a third derivative of at most 2
    (max_v |ds_v / T|)^3 T^2 (third cumulant of a bounded variable), so the
    difference quotient is off by a sixth of it, plus the losses' own bound."""
    import torch

    rows, vocab, width, T = 40, 150, 64, 2.0 if distill else 1.0
    h, e, gen = _problem(20, rows, vocab, width, "f16", 1.0)
    targets = None if distill else _targets(gen, rows, vocab, 0.0)
    sets = _sets(gen, rows, vocab, 20, empty=0.0, masked=0.0) if distill else None
    grad = torch.ones(rows, device="cuda")
    ref = Reference(h, e, "f16", targets, sets, T, grad)
    loss, (_, lse) = _forward(mf, h, e, targets, sets, T)
    dh, de = _backward(mf, loss, h, lse, grad, targets, sets, T)
    for side in ("hidden", "table"):
        base, g, off = (h, dh, ref.dh_off) if side == "hidden" else (e, de, ref.de_off)
        step = torch.randint(-1, 2, base.shape, generator=gen, device="cuda").to(base.dtype)
        step *= 2.0 ** -4 if side == "hidden" else 2.0 ** -7
        up, down = base + step, base - step
        moved = (up.double() - down.double()) / 2   # as rounded
        a = _forward(mf, *((up, e) if side == "hidden" else (h, up)), targets, sets, T)[1][0]
        b = _forward(mf, *((down, e) if side == "hidden" else (h, down)), targets, sets, T)[1][0]
        got = (a.double() - b.double()).sum() / 2
        mid = (up.double() + down.double()) / 2 - base.double()  # a shift of the midpoint
        ds = (moved @ e.double().T if side == "hidden" else h.double() @ moved.T) / T
        shift = (mid @ e.double().T if side == "hidden" else h.double() @ mid.T) / T
        room = (T * T * (2 * ds.abs().amax(1) ** 3 / 6
                         + 2 * ds.abs().amax(1) * shift.abs().amax(1)
                         )).sum() + ref.losses_off.sum() + (off * moved.abs()).sum()
        want = (g.double() * moved).sum()
        assert abs(float(got - want)) <= float(room), (side, float(got), float(want), float(room))
        assert float(room) < 0.3 * float(want.abs() + ref.losses.abs().sum() * 0.02) + 1.0


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (130, 21))
def test_one_gradient_alone(mf, kind, rows):
    import torch

    h, e, gen = _problem(21, rows, 700, 72, kind)
    targets = _targets(gen, rows, 700, 0.1)
    grad = torch.rand(rows, generator=gen, device="cuda")
    loss, (_, lse) = _forward(mf, h, e, targets)
    dh, de = _backward(mf, loss, h, lse, grad, targets)
    a, none = _backward(mf, loss, h, lse, grad, targets, embedding_grad=False)
    assert none is None and torch.equal(a, dh)
    none, b = _backward(mf, loss, h, lse, grad, targets, hidden_grad=False)
    assert none is None and torch.equal(b, de)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", (600, 32))
def test_same_bits_every_time_and_nothing_kept(mf, kind, rows):
    """Two runs give the same bits, whatever the workspace held before."""
    import torch

    h, e, gen = _problem(22, rows, 5000, 96, kind)
    sets = _sets(gen, rows, 5000, 60)
    grad = torch.rand(rows, generator=gen, device="cuda")
    loss, first = _forward(mf, h, e, None, sets, 2.0)
    g1 = _backward(mf, loss, h, first[1], grad, None, sets, 2.0)
    loss.workspace.fill_(0xFF)
    torch.cuda.synchronize()
    second = loss.distill(h, *sets, 2.0)
    torch.cuda.synchronize()
    loss.workspace.fill_(0x7F)
    g2 = _backward(mf, loss, h, second[1], grad, None, sets, 2.0)
    for x, y in zip((*first, *g1), (*second, *g2)):
        assert torch.equal(x, y)


def test_outputs_end_where_they_end(mf):
    """Nothing is written behind the outputs' and the workspace's last bytes."""
    import torch

    for rows, vocab, width, kind in ((5, 33, 72, "f16"), (130, 1001, 200, "bf16")):
        h, e, gen = _problem(23, rows, vocab, width, kind)
        targets = _targets(gen, rows, vocab, 0.2)
        guard = 64

        def padded(n, dtype):
            return torch.full((n + guard,), 7, dtype=dtype, device="cuda")

        need = mf.dense_loss_backward_workspace_bytes(rows, width, vocab)
        ws = padded(need, torch.uint8)
        losses, lse = padded(rows, torch.float32), padded(rows, torch.float32)
        dh, de = padded(rows * width, h.dtype), padded(vocab * width, h.dtype)
        grad = torch.rand(rows, generator=gen, device="cuda")
        s = gpu_stream()
        f = getattr(mf, "dense_xent_" + kind)
        fwd = mf.dense_loss_workspace_bytes(rows, width, vocab)
        ws2 = padded(fwd, torch.uint8)
        torch.cuda.synchronize()
        assert f(h, e, targets, losses[:rows], lse[:rows], ws2[:fwd], rows, width, vocab, s).ok()
        f = getattr(mf, "dense_xent_backward_" + kind)
        assert f(h, e, targets, lse[:rows], grad, dh[:rows * width], de[:vocab * width], ws[:need],
                 rows, width, vocab, s).ok()
        torch.cuda.synchronize()
        for t, n in ((ws, need), (ws2, fwd), (losses, rows), (lse, rows), (dh, rows * width),
                     (de, vocab * width)):
            assert bool((t[n:] == 7).all())


@pytest.mark.parametrize("distill", (False, True))
def test_captured_and_replayed(mf, distill):
    """A training step in a CUDA graph, replayed on new inputs in the same
    buffers; two graphs that share the workspace run one after the other."""
    import torch

    rows, vocab, width, kind = 200, 3000, 64, "f16"
    h, e, gen = _problem(24, rows, vocab, width, kind)
    h2, _, _ = _problem(25, rows, vocab, width, kind)
    targets = _targets(gen, rows, vocab, 0.1)
    sets = _sets(gen, rows, vocab, 30)
    grad = torch.rand(rows, generator=gen, device="cuda")
    kw = dict(sets=sets, temperature=2.0) if distill else dict(targets=targets)
    want = []
    for x in (h, h2):
        loss, out = _forward(mf, x, e, **kw)
        want.append([t.clone() for t in (*out, *_backward(mf, loss, x, out[1], grad, **kw))])
    stream = torch.cuda.Stream()
    loss = mf.DenseLoss(e, rows, stream=stream)
    x, source = h.clone(), h.clone()
    torch.cuda.synchronize()
    graphs = []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            if k == 0:
                x.copy_(source)  # the first kernel comes after a copy node
            if distill:
                out = loss.distill(x, *sets, 2.0)
                out = (*out, *loss.distill_backward(x, *sets, 2.0, out[1], grad))
            else:
                out = loss.cross_entropy(x, targets)
                out = (*out, *loss.cross_entropy_backward(x, targets, out[1], grad))
        graphs.append((g, out))
    for k, new in enumerate((h, h2, h)):
        source.copy_(new)
        torch.cuda.synchronize()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want[k % 2]):
                assert torch.equal(a, b)


def test_two_streams_at_once(mf):
    """Two objects, each with a workspace of its own, on two streams."""
    import torch

    problems = []
    for k in range(2):
        h, e, gen = _problem(30 + k, 700, 6000, 128, "bf16")
        targets = _targets(gen, 700, 6000, 0.1)
        grad = torch.rand(700, generator=gen, device="cuda")
        loss, (losses, lse) = _forward(mf, h, e, targets)
        want = (losses, lse, *_backward(mf, loss, h, lse, grad, targets))
        problems.append((h, targets, grad, mf.DenseLoss(e, 700, stream=torch.cuda.Stream()), want))
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for h, targets, grad, loss, _ in problems:
            losses, lse = loss.cross_entropy(h, targets)
            got.append((losses, lse, *loss.cross_entropy_backward(h, targets, lse, grad)))
    torch.cuda.synchronize()
    for k, out in enumerate(got):
        for a, b in zip(out, problems[k % 2][4]):
            assert torch.equal(a, b)


def test_scores_of_the_heads_choices(mf):
    """The head answers, the loss scores the answer, and a teacher's candidate
    sets train it: dense head ids (and a ragged batch's, with an empty row) go
    in as targets, the ragged batch itself as a teacher's sets."""
    import torch

    from market_sim_b200 import synth

    rows, vocab, width = 96, 4096, 576
    h = torch.from_numpy(synth.hidden_states(3, rows)).cuda()
    e = torch.from_numpy(synth.embedding(3, vocab=vocab)).cuda()
    off, ids = synth.ragged_batch(3, rows=rows, kmax=200, vocab=vocab, sort_ids=True)
    off[1] = 0  # row 0 has no candidate, row 1 has both rows' many
    ids[:off[2]] = np.arange(off[2])
    off, ids = torch.from_numpy(off).cuda(), torch.from_numpy(ids).cuda()
    stream = gpu_stream()
    chosen = torch.empty(rows, dtype=torch.int32, device="cuda")
    best = torch.empty(rows, dtype=torch.float32, device="cuda")
    ws = torch.zeros(mf.dense_workspace_bytes(rows), dtype=torch.uint8, device="cuda")
    loss = mf.DenseLoss(e, rows, stream=stream)
    torch.cuda.synchronize()
    assert mf.dense_head_f16(h, e, None, chosen, best, ws, rows, width, vocab, 0, stream).ok()
    losses, lse = loss.cross_entropy(h, chosen)
    torch.cuda.synchronize()
    ref = Reference(h, e, "f16", chosen)
    _near(losses, ref.losses, ref.losses_off, "losses")
    # the winning score the head reports is the one the loss subtracts
    torch.testing.assert_close(lse - losses, best, rtol=0, atol=2e-6 + 2.0 ** -22 * 20)
    ragged = mf.RaggedHead(e, rows, stream=stream)
    picked, scores = ragged(h, off, ids)
    losses, lse = loss.cross_entropy(h, picked)
    torch.cuda.synchronize()
    assert picked[0] == INVALID - 2 ** 32 and losses[0] == 0
    ref = Reference(h, e, "f16", picked)
    _near(losses, ref.losses, ref.losses_off, "losses")
    sets = (off, ids, torch.randn(ids.numel(), device="cuda"))
    _check(mf, h, e, "f16", torch.ones(rows, device="cuda"), sets=sets, temperature=2.0)


def test_current_stream_is_used_and_checked(mf):
    import torch

    h, e, gen = _problem(41, 10, 100, 64, "f16")
    targets = _targets(gen, 10, 100, 0.0)
    loss = mf.DenseLoss(e, 10)
    with pytest.raises(RuntimeError):
        loss.cross_entropy(h, targets)  # the legacy default stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        losses, _ = loss.cross_entropy(h, targets)
    torch.cuda.synchronize()
    ref = Reference(h, e, "f16", targets)
    _near(losses, ref.losses, ref.losses_off, "losses")


@pytest.mark.parametrize("kind", TYPES)
def test_one_object_for_batches_of_every_size(mf, kind):
    """One workspace, batches that grow and shrink over it."""
    import torch

    _, e, _ = _problem(50, 1, 1500, 96, kind)
    stream = gpu_stream()
    loss = mf.DenseLoss(e, 900, stream=stream)
    for rows in (900, 1, 65, 64, 257, 32, 33, 600, 256):
        h, _, gen = _problem(51 + rows, rows, 1, 96, kind)
        targets = _targets(gen, rows, 1500, 0.1)
        sets = _sets(gen, rows, 1500, 30)
        grad = torch.rand(rows, generator=gen, device="cuda")
        torch.cuda.synchronize()
        for kw in (dict(targets=targets), dict(sets=sets, temperature=2.0)):
            ref = Reference(h, e, kind, grad=grad, **kw)
            losses, lse = (loss.cross_entropy(h, targets) if "targets" in kw
                           else loss.distill(h, *sets, 2.0))
            torch.cuda.synchronize()
            _near(losses, ref.losses, ref.losses_off, "losses")
            dh, de = _backward(mf, loss, h, lse, grad, **kw)
            _near(dh, ref.d_hidden, ref.dh_off, "d_hidden")
            _near(de, ref.d_embedding, ref.de_off, "d_embedding")


def test_outputs_that_are_only_16_byte_aligned(mf):
    """Inputs and gradients that start 16 bytes into their memory."""
    import torch

    for rows, vocab, width in ((20, 700, 96), (150, 700, 96)):
        h, e, gen = _problem(60, rows, vocab, width, "f16")
        targets = _targets(gen, rows, vocab, 0.1)
        grad = torch.rand(rows, generator=gen, device="cuda")

        def shifted(t):
            out = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")[8:].view(t.shape)
            out.copy_(t)
            return out

        want_loss, (_, lse) = _forward(mf, h, e, targets)
        want = _backward(mf, want_loss, h, lse, grad, targets)
        h2, e2 = shifted(h), shifted(e)
        loss, (_, lse2) = _forward(mf, h2, e2, targets)
        assert torch.equal(lse, lse2)
        got = _backward(mf, loss, h2, lse2, grad, targets, d_hidden=shifted(h),
                        d_embedding=shifted(e))
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
