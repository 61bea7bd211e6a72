"""GPU tests of whose memory an object's workspace is: the object is made on one
stream, called on another and dropped while its calls are queued."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

ROWS, VOCAB, WIDTH = 300, 4000, 64
LONG = 40_000_000  # clocks: about 20 ms


@pytest.fixture(scope="module")
def mf(cuda):
    from market_sim_b200 import head

    return head


def _batch():
    import torch

    gen = torch.Generator(device="cuda").manual_seed(3)
    e = (torch.randn(VOCAB, WIDTH, generator=gen, device="cuda") / 8).half()
    h = torch.randn(ROWS, WIDTH, generator=gen, device="cuda").half()
    targets = torch.randint(0, VOCAB, (ROWS,), generator=gen, device="cuda", dtype=torch.int32)
    grad = torch.rand(ROWS, generator=gen, device="cuda")
    return e, h, targets, grad


def _owner(tensor):
    """Handle of the stream whose memory a tensor lies in."""
    import torch

    at = tensor.data_ptr()
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= at < s["address"] + s["total_size"]:
            return s["stream"]
    raise AssertionError("not of the allocator")


def _step(loss, h, targets, grad, out):
    losses, lse = loss.cross_entropy(h, targets, losses=out[0], lse=out[1])
    loss.cross_entropy_backward(h, targets, lse, grad, d_hidden=out[2], d_embedding=out[3])


def _outputs(e, h):
    import torch

    return (torch.empty(ROWS, device="cuda"), torch.empty(ROWS, device="cuda"),
            torch.empty_like(h), torch.empty_like(e))


@pytest.mark.parametrize("backward", (False, True))
def test_workspace_belongs_to_the_stream_that_was_given(mf, backward):
    import torch

    e = _batch()[0]
    for stream, handle in ((s := torch.cuda.Stream(), s.cuda_stream),
                           (c := mf.CudaStream.create(), c.handle()),
                           (s.cuda_stream, s.cuda_stream)):
        loss = mf.DenseLoss(e, ROWS, stream=stream, backward=backward)
        assert _owner(loss.workspace) == handle


@pytest.mark.parametrize("given", (True, False))
def test_dropped_while_its_calls_are_queued(mf, given):
    """The next tensors of the constructor's stream, of the workspace's size, are
    filled at once; the queued calls neither see nor spoil them."""
    import torch

    e, h, targets, grad = _batch()
    side = torch.cuda.Stream()
    want = _outputs(e, h)
    torch.cuda.synchronize()
    loss = mf.DenseLoss(e, ROWS, stream=side)
    _step(loss, h, targets, grad, want)
    torch.cuda.synchronize()
    del loss
    got = _outputs(e, h)
    torch.cuda.synchronize()
    loss = mf.DenseLoss(e, ROWS, stream=side if given else None)
    nbytes = loss.workspace.numel()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        _step(loss, h, targets, grad, got)
    del loss
    fresh = [torch.empty(nbytes, dtype=torch.uint8, device="cuda").fill_(k) for k in (17, 23)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for t, k in zip(fresh, (17, 23)):
        assert bool((t == k).all())


@pytest.mark.parametrize("given", (True, False))
def test_made_from_memory_that_is_still_in_use(mf, given):
    """The constructor's stream has work queued on memory of the workspace's size
    that was just given back: the calls on the other stream leave it alone."""
    import torch

    e, h, targets, grad = _batch()
    side = torch.cuda.Stream()
    want, got = _outputs(e, h), _outputs(e, h)
    torch.cuda.synchronize()
    loss = mf.DenseLoss(e, ROWS, stream=side)
    nbytes = loss.workspace.numel()
    _step(loss, h, targets, grad, want)
    torch.cuda.synchronize()
    del loss
    kept = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
    source = torch.full((nbytes,), 9, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(2):
        used = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        used.copy_(source)
        torch.cuda._sleep(LONG)
        kept.copy_(used)
        del used
        loss = mf.DenseLoss(e, ROWS, stream=side if given else None)
        with torch.cuda.stream(side):
            _step(loss, h, targets, grad, got)
        del loss
        torch.cuda.synchronize()
        assert bool((kept == 9).all())
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_one_object_on_two_streams_then_dropped(mf):
    """Without a stream of its own: calls on one stream after the other."""
    import torch

    e, h, targets, grad = _batch()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    want, a, b = _outputs(e, h), _outputs(e, h), _outputs(e, h)
    torch.cuda.synchronize()
    loss = mf.DenseLoss(e, ROWS, stream=first)
    _step(loss, h, targets, grad, want)
    torch.cuda.synchronize()
    loss = mf.DenseLoss(e, ROWS)
    nbytes = loss.workspace.numel()
    with torch.cuda.stream(first):
        _step(loss, h, targets, grad, a)
    second.wait_stream(first)
    with torch.cuda.stream(second):
        torch.cuda._sleep(LONG)
        _step(loss, h, targets, grad, b)
    del loss
    fresh = torch.empty(nbytes, dtype=torch.uint8, device="cuda").fill_(5)
    torch.cuda.synchronize()
    assert bool((fresh == 5).all())
    for got in (a, b):
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_made_and_called_in_a_capture(mf):
    """Without a stream of its own, inside a capture: nothing there waits."""
    import torch

    e, h, targets, grad = _batch()
    want, got = _outputs(e, h), _outputs(e, h)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    loss = mf.DenseLoss(e, ROWS, stream=stream)
    _step(loss, h, targets, grad, want)
    torch.cuda.synchronize()
    outside = mf.DenseLoss(e, ROWS)
    graphs = []
    for inside in (False, True):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            obj = mf.DenseLoss(e, ROWS) if inside else outside
            _step(obj, h, targets, grad, got)
        graphs.append((g, obj))
    for g, _ in graphs:
        for t in got:
            t.fill_(0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
