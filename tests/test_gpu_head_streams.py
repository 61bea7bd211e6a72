"""GPU tests of RaggedHead's memory: made on one stream, called on another and
dropped while its calls are queued."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROWS, VOCAB, WIDTH = 64, 3000, 576
LONG = 40_000_000  # clocks: about 20 ms


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _batch():
    import torch

    from market_sim_b200 import synth

    h = torch.from_numpy(synth.hidden_states(5, ROWS)).cuda()
    e = torch.from_numpy(synth.embedding(5, vocab=VOCAB)).cuda()
    off, ids = synth.ragged_batch(5, rows=ROWS, kmax=900, vocab=VOCAB)
    return e, h, torch.from_numpy(off).cuda(), torch.from_numpy(ids).cuda()


def _dirty(nbytes):
    """Memory of that size on the current stream that holds no zeros, given back."""
    import torch

    t = torch.full((nbytes,), 0x5A, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    del t


@pytest.fixture(scope="module")
def answers(mf):
    import torch

    e, h, off, ids = _batch()
    stream = torch.cuda.Stream()
    head = mf.RaggedHead(e, ROWS, stream=stream)
    torch.cuda.synchronize()
    out = head(h, off, ids)
    torch.cuda.synchronize()
    ids_np, off_np = ids.cpu().numpy(), off.cpu().numpy()
    for r in range(ROWS):  # each answer is one of its row's candidates
        assert int(out[0][r]) in ids_np[off_np[r]:off_np[r + 1]]
    return [t.clone() for t in out]


@pytest.mark.parametrize("given", (True, False))
def test_made_behind_queued_work(mf, answers, given):
    """The constructor's stream is busy, so its zeros would come late."""
    import torch

    e, h, off, ids = _batch()
    side = torch.cuda.Stream()
    nbytes = mf.head_workspace_bytes(ROWS)
    _dirty(nbytes)
    with torch.cuda.stream(side):
        _dirty(nbytes)
    torch.cuda.synchronize()
    torch.cuda._sleep(LONG)
    head = mf.RaggedHead(e, ROWS, stream=side if given else None)
    with torch.cuda.stream(side):
        got = head(h, off, ids)
    torch.cuda.synchronize()
    for a, b in zip(got, answers):
        assert torch.equal(a, b)


@pytest.mark.parametrize("given", (True, False))
def test_dropped_while_a_call_is_queued(mf, answers, given):
    import torch

    e, h, off, ids = _batch()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    head = mf.RaggedHead(e, ROWS, stream=side if given else None)
    nbytes = head.workspace.numel()
    out = (torch.empty(ROWS, dtype=torch.int32, device="cuda"),
           torch.empty(ROWS, dtype=torch.float32, device="cuda"))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        head(h, off, ids, *out)
    del head
    fresh = torch.empty(nbytes, dtype=torch.uint8, device="cuda").fill_(0x33)
    torch.cuda.synchronize()
    assert bool((fresh == 0x33).all())
    for a, b in zip(out, answers):
        assert torch.equal(a, b)


def test_outputs_made_while_their_memory_is_in_use(mf, answers):
    """Outputs are written on the object's stream, so they are not taken from
    memory that the current stream still uses; a reader on the current stream
    may drop them before it has read them."""
    import torch

    e, h, off, ids = _batch()
    side = torch.cuda.Stream()
    head = mf.RaggedHead(e, ROWS, stream=side)
    kept = torch.zeros(ROWS, dtype=torch.int32, device="cuda")
    source = torch.full((ROWS,), 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    used = torch.empty(ROWS, dtype=torch.int32, device="cuda")
    used.copy_(source)
    torch.cuda._sleep(LONG)
    kept.copy_(used)
    del used
    picked, scores = head(h, off, ids)
    torch.cuda.synchronize()
    assert bool((kept == 7).all()) and torch.equal(picked, answers[0])
    torch.cuda._sleep(LONG)
    kept.copy_(picked)
    del picked, scores
    with torch.cuda.stream(side):
        for _ in range(8):
            torch.empty(ROWS, dtype=torch.int32, device="cuda").fill_(-5)
    torch.cuda.synchronize()
    assert torch.equal(kept, answers[0])
