"""CPU checks of the losses' entry points (include/mf_loss.h): bad metadata is
rejected on the host before any CUDA call (the pointers here are never
dereferenced)."""
from __future__ import annotations

import ctypes

import pytest

STREAM = 0xDEAD00
ROWS, HIDDEN, VOCAB, ENTRIES = 4, 64, 1000, 10
KINDS = ("f16", "bf16")


@pytest.fixture(scope="module")
def lib():
    from market_sim_b200 import build

    build.build()
    from market_sim_b200 import _lib

    return _lib.lib


@pytest.fixture(scope="module")
def E():
    from market_sim_b200.head import ErrorCode

    return ErrorCode


def _xent(lib, kind, backward, rows=ROWS, width=HIDDEN, vocab=VOCAB, stream=STREAM, **change):
    """One call with good arguments but for `change`: name -> (address, bytes)."""
    r, v = (min(x, 1 << 25) for x in (rows, vocab))
    ws = (lib.mf_dense_loss_backward_workspace_bytes if backward
          else lib.mf_dense_loss_workspace_bytes)(rows, width, vocab) or 1 << 40
    sizes = dict(hidden=r * width * 2, embedding=v * width * 2, targets=r * 4)
    if backward:
        sizes.update(lse=r * 4, grad_losses=r * 4, d_hidden=r * width * 2,
                     d_embedding=v * width * 2)
    else:
        sizes.update(losses=r * 4, lse=r * 4)
    sizes["workspace"] = ws
    args = []
    for i, (name, n) in enumerate(sizes.items()):
        at, n = change.pop(name, (1 << (44 + i), n))
        args += [ctypes.c_void_p(at), n]
    assert not change
    f = getattr(lib, f"mf_dense_xent_{'backward_' if backward else ''}{kind}")
    return f(*args, rows, width, vocab, ctypes.c_void_p(stream)).code


def _distill(lib, kind, backward, rows=ROWS, width=HIDDEN, vocab=VOCAB, temperature=1.0,
             stream=STREAM, **change):
    ws = (lib.mf_dense_loss_backward_workspace_bytes if backward
          else lib.mf_dense_loss_workspace_bytes)(rows, width, vocab) or 1 << 40
    sizes = dict(hidden=rows * width * 2, embedding=vocab * width * 2, offsets=(rows + 1) * 4,
                 ids=ENTRIES * 4, teacher_logits=ENTRIES * 4, temperature=None)
    if backward:
        sizes.update(lse=rows * 4, grad_losses=rows * 4, d_hidden=rows * width * 2,
                     d_embedding=vocab * width * 2)
    else:
        sizes.update(losses=rows * 4, lse=rows * 4)
    sizes["workspace"] = ws
    args = []
    for i, (name, n) in enumerate(sizes.items()):
        if n is None:
            args.append(temperature)
            continue
        at, n = change.pop(name, (1 << (44 + i), n))
        args += [ctypes.c_void_p(at), n]
    assert not change
    f = getattr(lib, f"mf_dense_distill_{'backward_' if backward else ''}{kind}")
    return f(*args, rows, width, vocab, ctypes.c_void_p(stream)).code


CALLS = [(c, k, b) for c in (_xent, _distill) for k in KINDS for b in (False, True)]
IDS = [f"{c.__name__[1:]}-{k}-{'backward' if b else 'forward'}" for c, k, b in CALLS]


@pytest.mark.parametrize("call,kind,backward", CALLS, ids=IDS)
def test_sizes(lib, E, call, kind, backward):
    assert call(lib, kind, backward, rows=0) == E.invalid_argument
    assert call(lib, kind, backward, vocab=0) == E.invalid_argument
    assert call(lib, kind, backward, width=0) == E.invalid_argument
    assert call(lib, kind, backward, stream=0) == E.invalid_argument
    assert call(lib, kind, backward, width=60) == E.resource_limit  # a multiple of 8
    assert call(lib, kind, backward, width=8200) == E.resource_limit
    assert call(lib, kind, backward, rows=(1 << 16) + 1) == E.resource_limit
    assert call(lib, kind, backward, vocab=(1 << 24) + 1) == E.resource_limit


@pytest.mark.parametrize("call,kind,backward", CALLS, ids=IDS)
def test_buffers(lib, E, call, kind, backward):
    distill = call is _distill
    at = 1 << 60  # clear of the good buffers
    sixteen = ["hidden", "embedding"] + (["d_hidden", "d_embedding"] if backward else [])
    sizes = dict(hidden=ROWS * HIDDEN * 2, embedding=VOCAB * HIDDEN * 2,
                 d_hidden=ROWS * HIDDEN * 2, d_embedding=VOCAB * HIDDEN * 2)
    for name in sixteen:
        assert call(lib, kind, backward, **{name: (at + 8, sizes[name])}) == E.invalid_argument
        assert call(lib, kind, backward, **{name: (at, sizes[name] - 2)}) == E.invalid_argument
    rowwise = ["lse", "grad_losses"] if backward else ["losses", "lse"]
    for name in rowwise:
        assert call(lib, kind, backward, **{name: (at + 2, ROWS * 4)}) == E.invalid_argument
        assert call(lib, kind, backward, **{name: (0, ROWS * 4)}) == E.invalid_argument
        assert call(lib, kind, backward, **{name: (at, ROWS * 4 + 4)}) == E.invalid_argument
    rows_of = "offsets" if distill else "targets"
    n = (ROWS + (1 if distill else 0)) * 4
    assert call(lib, kind, backward, **{rows_of: (at, n - 4)}) == E.invalid_argument
    assert call(lib, kind, backward, **{rows_of: (at + 1, n)}) == E.invalid_argument
    need = (lib.mf_dense_loss_backward_workspace_bytes if backward
            else lib.mf_dense_loss_workspace_bytes)(ROWS, HIDDEN, VOCAB)
    assert call(lib, kind, backward, workspace=(at, need - 1)) == E.invalid_argument
    for off in (8, 16, 32, 128):  # the workspace starts on 256 bytes
        assert call(lib, kind, backward, workspace=(at + off, need)) == E.invalid_argument
    # an output or the workspace that overlaps another buffer, by its last bytes
    out = "lse" if not backward else "d_hidden"
    size = ROWS * 4 if not backward else ROWS * HIDDEN * 2
    assert call(lib, kind, backward, **{out: ((1 << 44) + 16, size)}) == E.invalid_argument
    assert call(lib, kind, backward, workspace=((1 << 45) - need + 16, need)) == E.invalid_argument
    if backward:
        both = {"d_hidden": (0, 0), "d_embedding": (0, 0)}
        assert call(lib, kind, True, **both) == E.invalid_argument


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("backward", (False, True))
def test_distill_only(lib, E, kind, backward):
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-30, 1e30):
        assert _distill(lib, kind, backward, temperature=t) == E.invalid_argument
    at = 1 << 60
    assert _distill(lib, kind, backward, ids=(at, ENTRIES * 4 + 4)) == E.invalid_argument
    assert _distill(lib, kind, backward, ids=(0, ENTRIES * 4)) == E.invalid_argument
    assert _distill(lib, kind, backward, teacher_logits=(at + 2, ENTRIES * 4)) \
        == E.invalid_argument
    big = ((1 << 31) - 1023) * 4  # one entry too many
    assert _distill(lib, kind, backward, ids=(1 << 55, big), teacher_logits=(1 << 56, big)) \
        == E.resource_limit


def test_workspace_bytes(lib):
    f, b = lib.mf_dense_loss_workspace_bytes, lib.mf_dense_loss_backward_workspace_bytes
    for bad in ((0, 64, 8), (8, 0, 8), (8, 64, 0), (8, 65, 8), ((1 << 16) + 1, 64, 8),
                (8, 64, (1 << 24) + 1), (8, 8200, 8)):
        assert f(*bad) == 0 and b(*bad) == 0
    for rows in (1, 100, 8192, 1 << 16):
        for vocab in (1, 1000, 49152):
            assert 0 < f(rows, 576, vocab) <= 4096 + rows * 3300
            # two pieces of d, the copy of the rows, FP32 sums of d_hidden
            pieces = 2 * (128 << 20)
            sums = max(128 << 20, rows * 576 * 4)
            assert rows * 576 * 6 < b(rows, 576, vocab) <= pieces + sums + rows * 576 * 2 + 4096 + rows * 24


def test_a_workspace_holds_every_smaller_batch(lib):
    """A user keeps one workspace for the largest batch."""
    f, b = lib.mf_dense_loss_workspace_bytes, lib.mf_dense_loss_backward_workspace_bytes
    steps = [1, 2, 16, 31, 32, 33, 63, 64, 65, 100, 255, 256, 257, 300, 511, 512, 513, 700, 768,
             1000, 1024, 1025, 2000, 4096, 5000, 8192, 20_000, 65_536]
    for width, vocab in ((576, 49152), (64, 300), (1024, 20_000), (8, 1)):
        for g in (f, b):
            sizes = [g(r, width, vocab) for r in steps]
            assert sizes == sorted(sizes)


def test_class_checks_before_the_call():
    """DenseLoss refuses tensors of another type, shape, layout or place."""
    torch = pytest.importorskip("torch")
    from market_sim_b200 import head

    table = torch.zeros(40, 16, dtype=torch.float16)
    loss = head.DenseLoss(table, 4)
    hidden, targets = torch.zeros(3, 16, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        loss.cross_entropy(torch.zeros(5, 16, dtype=torch.float16), targets)  # max_rows
    with pytest.raises(ValueError):
        loss.cross_entropy(hidden.bfloat16(), targets)
    with pytest.raises(ValueError):
        loss.cross_entropy(hidden, targets.long())
    with pytest.raises(ValueError):
        loss.cross_entropy(torch.zeros(3, 32, dtype=torch.float16)[:, ::2], targets)
    with pytest.raises(ValueError):
        loss.distill(hidden, torch.zeros(3, dtype=torch.int32), targets, torch.zeros(3))
    with pytest.raises(ValueError):
        head.DenseLoss(table.float(), 4)
    with pytest.raises(ValueError):
        head.DenseLoss(torch.zeros(40, 12, dtype=torch.float16), 4)
    with pytest.raises(RuntimeError):
        head.DenseLoss(table, 4, backward=False).cross_entropy_backward(
            hidden, targets, torch.zeros(3), torch.zeros(3))


def test_class_refuses_host_memory():
    """A table and batch that agree with each other, but not on a GPU."""
    torch = pytest.importorskip("torch")
    from market_sim_b200 import head

    loss = head.DenseLoss(torch.zeros(40, 16, dtype=torch.float16), 4)
    launched = []
    loss._launch = lambda *a: launched.append(a)
    hidden, targets = torch.zeros(3, 16, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="not on a GPU"):
        loss.cross_entropy(hidden, targets, losses=torch.zeros(3), lse=torch.zeros(3))
    with pytest.raises(ValueError, match="not on a GPU"):
        loss.cross_entropy_backward(hidden, targets, torch.zeros(3), torch.zeros(3),
                                    d_hidden=torch.zeros_like(hidden), embedding_grad=False)
    assert not launched


def test_workspace_of_few_wide_rows(lib):
    """Up to 32 rows keep a plane of sums for each CTA, where their kernel takes the
    width (up to 640): the sums stay within 128 MiB, or 4 bytes an element."""
    b = lib.mf_dense_loss_backward_workspace_bytes
    for width in (8, 576, 640, 648, 1024, 4096, 8192):
        for rows in (1, 31, 32, 33, 64, 300):
            for vocab in (1, 1000, 49152, 1 << 24):
                # d of all the vocabulary, up to 64 rows in two halves
                whole = 2 * max(rows, 2 * min(rows, 64)) * ((vocab + 255) // 256 * 256)
                pieces = min(whole, 2 * (128 << 20))
                sums = max(128 << 20, rows * width * 4)
                assert b(rows, width, vocab) <= pieces + sums + rows * width * 2 + 4096 + rows * 24, \
                    (width, rows, vocab)
    # no planes above 640: 32 rows need what the tile engine needs for one row more than 31
    assert b(32, 640, 1000) > 148 * 32 * 640 * 4
    assert b(32, 648, 1000) < 148 * 32 * 648 * 4 // 4
    assert b(32, 8192, 1000) < 32 << 20
