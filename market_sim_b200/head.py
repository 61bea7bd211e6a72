"""Host-side mirror of the reference's ``marketforge::cuda`` head interface.

Same names, argument meaning and error behaviour as
``include/marketforge/cuda/greedy.hpp`` (plus the boundary types of
``device_buffer.hpp`` / ``cuda_stream.hpp`` / ``core/status.hpp``), calling
the CUDA kernels through the C-ABI in ``include/mf_head.h``.  Buffers may be
:class:`DeviceBuffer` objects or CUDA ``torch.Tensor`` s (their byte size is
``numel * element_size``); streams may be :class:`CudaStream`,
``torch.cuda.Stream`` or a raw ``cudaStream_t`` integer.
"""
from __future__ import annotations

import ctypes
import enum
from dataclasses import dataclass
from typing import Optional, Union

from ._lib import lib

INVALID_TOKEN_ID = 0xFFFFFFFF
"""``restricted_greedy_invalid_token_id`` (greedy.hpp:11-12)."""


class ErrorCode(enum.IntEnum):
    """``marketforge::ErrorCode`` (include/marketforge/core/status.hpp:7-31)."""

    ok = 0
    invalid_argument = 1
    unsupported_dtype = 2
    invalid_shape = 3
    invalid_model = 4
    arithmetic_overflow = 5
    invalid_alignment = 6
    allocation_failed = 7
    insufficient_memory = 8
    insufficient_resources = 9
    io_error = 10
    invalid_format = 11
    invalid_utf8 = 12
    invalid_json = 13
    duplicate_key = 14
    resource_limit = 15
    truncated_data = 16
    invalid_tensor = 17
    missing_tensor = 18
    unexpected_tensor = 19
    hash_mismatch = 20
    cuda_backend_failure = 21
    cuda_runtime_failure = 22


@dataclass(frozen=True)
class Status:
    """``marketforge::Status`` (status.hpp:33-49)."""

    code: ErrorCode = ErrorCode.ok
    detail: int = 0

    def ok(self) -> bool:
        return self.code == ErrorCode.ok

    @staticmethod
    def success() -> "Status":
        return Status()

    @staticmethod
    def failure(code: ErrorCode, detail: int = 0) -> "Status":
        return Status(ErrorCode(code), detail)


def _status(s) -> Status:
    return Status(ErrorCode(s.code), int(s.detail))


class CudaStream:
    """``marketforge::cuda::CudaStream`` (cuda_stream.hpp:19-41): a
    non-blocking stream (src/cuda/cuda_stream.cu:13)."""

    def __init__(self, stream=None):
        import torch

        self._stream = stream if stream is not None else torch.cuda.Stream()

    @staticmethod
    def create() -> "CudaStream":
        return CudaStream()

    def handle(self) -> int:
        return int(self._stream.cuda_stream)

    @property
    def torch_stream(self):
        return self._stream

    def synchronize(self) -> Status:
        self._stream.synchronize()
        return Status.success()


class DeviceBuffer:
    """``marketforge::cuda::DeviceBuffer`` (device_buffer.hpp:20-56): an exact
    byte-sized device allocation (torch's caching allocator underneath)."""

    def __init__(self, tensor=None):
        self._t = tensor

    @staticmethod
    def allocate(byte_count: int) -> "DeviceBuffer":
        import torch

        if byte_count == 0:
            return DeviceBuffer()
        return DeviceBuffer(torch.empty(int(byte_count), dtype=torch.uint8, device="cuda"))

    def size_bytes(self) -> int:
        return 0 if self._t is None else self._t.numel() * self._t.element_size()

    def address(self) -> int:
        return 0 if self._t is None else int(self._t.data_ptr())

    @property
    def tensor(self):
        return self._t

    def view(self, dtype):
        return self._t.view(dtype)

    def copy_from_host_async(self, source, byte_count: int, offset: int, stream) -> Status:
        return _copy(self, source, byte_count, offset, stream, to_device=True)

    def copy_to_host_async(self, destination, byte_count: int, offset: int, stream) -> Status:
        return _copy(self, destination, byte_count, offset, stream, to_device=False)


def _copy(buf: DeviceBuffer, host, byte_count, offset, stream, to_device) -> Status:
    # src/cuda/device_buffer.cu:13-31 validation order
    import torch

    h = _stream_handle(stream)
    if h == 0 or (byte_count != 0 and host is None):
        return Status.failure(ErrorCode.invalid_argument)
    if offset + byte_count > buf.size_bytes():
        return Status.failure(ErrorCode.invalid_argument)
    if byte_count == 0:
        return Status.success()
    host_t = host if isinstance(host, torch.Tensor) else torch.from_numpy(host)
    host_bytes = host_t.reshape(-1).view(torch.uint8)[:byte_count]
    dev = buf.tensor[offset:offset + byte_count]
    with torch.cuda.stream(_torch_stream(stream)):
        if to_device:
            dev.copy_(host_bytes, non_blocking=True)
        else:
            host_bytes.copy_(dev, non_blocking=True)
    return Status.success()


Buffer = Union[DeviceBuffer, "torch.Tensor", None]  # noqa: F821


def _addr(b: Buffer) -> int:
    if b is None:
        return 0
    if isinstance(b, DeviceBuffer):
        return b.address()
    return int(b.data_ptr())


def _size(b: Buffer) -> int:
    if b is None:
        return 0
    if isinstance(b, DeviceBuffer):
        return b.size_bytes()
    return b.numel() * b.element_size()


def _stream_handle(s) -> int:
    if s is None:
        return 0
    if isinstance(s, CudaStream):
        return s.handle()
    if isinstance(s, int):
        return s
    return int(s.cuda_stream)


def _torch_stream(s):
    import torch

    if isinstance(s, CudaStream):
        return s.torch_stream
    if isinstance(s, int):
        return torch.cuda.ExternalStream(s)
    return s


def _made_on(stream, device, make):
    """``make()``'s tensor, from the memory of ``stream`` (None: the current
    stream).  A stream's memory is handed on in that stream's order, so nothing
    made for one stream is first written, or still in use, on another."""
    import torch

    if stream is None or device.type != "cuda":
        return make()
    with torch.cuda.device(device), torch.cuda.stream(_torch_stream(stream)):
        return make()


def _outputs_on(stream, device, *makes):
    """Outputs for the caller from the memory of ``stream``, which writes them; a
    caller on another current stream may read them there and drop them.  None
    stands for an output that is given."""
    import torch

    def made():
        return [make and make() for make in makes]

    if stream is None or device.type != "cuda":
        return made()
    current = torch.cuda.current_stream(device)
    if current.cuda_stream == _stream_handle(stream):
        return made()
    out = _made_on(stream, device, made)
    for t in out:
        if t is not None:
            t.record_stream(current)
    return out


class _Workspace:
    """A workspace that outlives its calls on the streams that use it.

    With a ``stream`` it belongs to that stream.  Without one it is made on the
    current stream, which the constructor waits for (work queued there may
    still use the memory, and fills it), and every stream that a call uses it
    on is made known to the allocator, which then holds the memory back from
    others until that stream's work is done.
    """

    def __init__(self, make, device, stream):
        import torch

        self.tensor = _made_on(stream, device, make)
        self._seen = None  # a stream was given: its memory, its order
        if stream is None and device.type == "cuda":
            self._seen, self._torch = set(), torch
            with torch.cuda.device(device):
                if not torch.cuda.is_current_stream_capturing():
                    torch.cuda.current_stream().synchronize()

    def used_on(self, stream) -> None:
        """Before a call on ``stream`` (where the constructor got none)."""
        if self._seen is not None:
            handle = _stream_handle(stream)
            if handle not in self._seen:
                self.tensor.record_stream(_torch_stream(stream))
                self._seen.add(handle)


def _pb(b: Buffer):
    return ctypes.c_void_p(_addr(b) or None), ctypes.c_uint64(_size(b))


def _sp(s):
    h = _stream_handle(s)
    return ctypes.c_void_p(h or None)


# ---- reference-signature functions (greedy.hpp:17-49) ----------------------

def greedy_select_f16(logits: Buffer, token_ids: Buffer, rows: int, vocabulary_size: int,
                      stream) -> Status:
    """greedy.hpp:17-21: argmax per row of fp16 logits[rows, V]."""
    return _status(lib.mf_greedy_select_f16(*_pb(logits), *_pb(token_ids), rows,
                                            vocabulary_size, _sp(stream)))


def restricted_greedy_select_f16(logits: Buffer, allowed_token_ids: Buffer,
                                 allowed_token_counts: Buffer, token_ids: Buffer, rows: int,
                                 vocabulary_size: int, maximum_allowed_tokens: int,
                                 stream) -> Status:
    """greedy.hpp:29-33: masked argmax over a padded candidate table."""
    return _status(lib.mf_restricted_greedy_select_f16(
        *_pb(logits), *_pb(allowed_token_ids), *_pb(allowed_token_counts), *_pb(token_ids),
        rows, vocabulary_size, maximum_allowed_tokens, _sp(stream)))


def restricted_output_head_f16(hidden: Buffer, embedding: Buffer, allowed_token_ids: Buffer,
                               allowed_token_counts: Buffer, token_ids: Buffer, rows: int,
                               hidden_size: int, vocabulary_size: int,
                               maximum_allowed_tokens: int, stream) -> Status:
    """greedy.hpp:43-49: fused tied projection + restricted argmax."""
    return _status(lib.mf_restricted_output_head_f16(
        *_pb(hidden), *_pb(embedding), *_pb(allowed_token_ids), *_pb(allowed_token_counts),
        *_pb(token_ids), rows, hidden_size, vocabulary_size, maximum_allowed_tokens,
        _sp(stream)))


# ---- ragged CSR head and device DFA (new batched launch path) -------------

def head_workspace_bytes(rows: int) -> int:
    return int(lib.mf_head_workspace_bytes(rows))


def dfa_workspace_bytes(batch: int) -> int:
    return int(lib.mf_dfa_workspace_bytes(batch))


def restricted_output_head_csr_f16(hidden: Buffer, embedding: Buffer, offsets: Buffer,
                                   ids: Buffer, token_ids: Buffer, scores: Optional[Buffer],
                                   workspace: Buffer, rows: int, hidden_size: int,
                                   vocabulary_size: int, stream) -> Status:
    """Ragged head: row r's candidates are ids[offsets[r]:offsets[r+1]]."""
    return _status(lib.mf_head_restricted_csr_f16(
        *_pb(hidden), *_pb(embedding), *_pb(offsets), *_pb(ids), *_pb(token_ids), *_pb(scores),
        *_pb(workspace), rows, hidden_size, vocabulary_size, _sp(stream)))


LAUNCH_OVERLAP_PREVIOUS = 1
"""``restricted_output_head_csr_f16_ex`` flag: the launch may overlap the tail
of the previous kernel on the stream, which must not write this call's
inputs (consecutive head calls on independent batches)."""


def restricted_output_head_csr_f16_ex(hidden: Buffer, embedding: Buffer, offsets: Buffer,
                                      ids: Buffer, token_ids: Buffer, scores: Optional[Buffer],
                                      workspace: Buffer, rows: int, hidden_size: int,
                                      vocabulary_size: int, launch_flags: int, stream) -> Status:
    """``restricted_output_head_csr_f16`` with launch options
    (``LAUNCH_OVERLAP_PREVIOUS``)."""
    return _status(lib.mf_head_restricted_csr_f16_ex(
        *_pb(hidden), *_pb(embedding), *_pb(offsets), *_pb(ids), *_pb(token_ids), *_pb(scores),
        *_pb(workspace), rows, hidden_size, vocabulary_size, launch_flags, _sp(stream)))


def restricted_output_head_csr_u16ids_f16_ex(hidden: Buffer, embedding: Buffer, offsets: Buffer,
                                             ids: Buffer, token_ids: Buffer,
                                             scores: Optional[Buffer], workspace: Buffer, rows: int,
                                             hidden_size: int, vocabulary_size: int,
                                             launch_flags: int, stream) -> Status:
    """``restricted_output_head_csr_f16_ex`` with the candidate ids as uint16
    (vocabularies of at most 65,536 ids): half the bytes to move per batch."""
    return _status(lib.mf_head_restricted_csr_u16ids_f16_ex(
        *_pb(hidden), *_pb(embedding), *_pb(offsets), *_pb(ids), *_pb(token_ids), *_pb(scores),
        *_pb(workspace), rows, hidden_size, vocabulary_size, launch_flags, _sp(stream)))


NOALLOC_MAX_ROWS = 65536
"""Largest batch ``restricted_output_head_csr_f16_noalloc`` accepts."""


def restricted_output_head_csr_f16_noalloc(hidden: Buffer, embedding: Buffer, offsets: Buffer,
                                           ids: Buffer, token_ids: Buffer,
                                           scores: Optional[Buffer], rows: int, hidden_size: int,
                                           vocabulary_size: int, stream) -> Status:
    """The ragged head without a workspace argument, for callers that cannot
    allocate device memory: the library keeps a fixed scratch array per GPU
    (up to NOALLOC_MAX_ROWS rows).  Calls sharing a device must not overlap
    on the GPU; make the first call on a device before any stream capture."""
    return _status(lib.mf_head_restricted_csr_f16_noalloc(
        *_pb(hidden), *_pb(embedding), *_pb(offsets), *_pb(ids), *_pb(token_ids), *_pb(scores),
        rows, hidden_size, vocabulary_size, _sp(stream)))


def restricted_output_head_csr_rmsnorm_f16(hidden: Buffer, gamma: Buffer, eps: float,
                                           embedding: Buffer, offsets: Buffer, ids: Buffer,
                                           token_ids: Buffer, scores: Optional[Buffer],
                                           workspace: Buffer, rows: int, hidden_size: int,
                                           vocabulary_size: int, stream) -> Status:
    """Ragged head with the final RMSNorm fused in front (hidden = the last
    layer's un-normalised rows, gamma = the norm weight)."""
    return _status(lib.mf_head_restricted_csr_rmsnorm_f16(
        *_pb(hidden), *_pb(gamma), float(eps), *_pb(embedding), *_pb(offsets), *_pb(ids),
        *_pb(token_ids), *_pb(scores), *_pb(workspace), rows, hidden_size, vocabulary_size,
        _sp(stream)))


def dfa_head_step_f16(hidden: Buffer, embedding: Buffer, state_offsets: Buffer,
                      arc_tokens: Buffer, arc_next: Buffer, states_in: Buffer,
                      states_out: Buffer, tokens: Buffer, scores: Optional[Buffer],
                      workspace: Buffer, batch: int, num_states: int, hidden_size: int,
                      vocabulary_size: int, stream) -> Status:
    """One device step: allowed-set lookup, restricted head, DFA advance."""
    return _status(lib.mf_dfa_head_step_f16(
        *_pb(hidden), *_pb(embedding), *_pb(state_offsets), *_pb(arc_tokens), *_pb(arc_next),
        *_pb(states_in), *_pb(states_out), *_pb(tokens), *_pb(scores), *_pb(workspace),
        batch, num_states, hidden_size, vocabulary_size, _sp(stream)))


def dfa_head_step_rmsnorm_f16(hidden: Buffer, gamma: Buffer, eps: float, embedding: Buffer,
                              state_offsets: Buffer, arc_tokens: Buffer, arc_next: Buffer,
                              states_in: Buffer, states_out: Buffer, tokens: Buffer,
                              scores: Optional[Buffer], workspace: Buffer, batch: int,
                              num_states: int, hidden_size: int, vocabulary_size: int,
                              stream) -> Status:
    """One device step with the final RMSNorm fused in front (hidden = the
    last layer's un-normalised rows, gamma = the norm weight)."""
    return _status(lib.mf_dfa_head_step_rmsnorm_f16(
        *_pb(hidden), *_pb(gamma), float(eps), *_pb(embedding), *_pb(state_offsets),
        *_pb(arc_tokens), *_pb(arc_next), *_pb(states_in), *_pb(states_out), *_pb(tokens),
        *_pb(scores), *_pb(workspace), batch, num_states, hidden_size, vocabulary_size,
        _sp(stream)))


def dfa_decode_f16(hidden: Buffer, embedding: Buffer, state_offsets: Buffer, arc_tokens: Buffer,
                   arc_next: Buffer, state_trace: Buffer, token_trace: Buffer,
                   score_trace: Optional[Buffer], workspace: Buffer, steps: int, batch: int,
                   num_states: int, hidden_size: int, vocabulary_size: int, stream) -> Status:
    """``steps`` DFA head steps back to back, no host synchronisation."""
    return _status(lib.mf_dfa_decode_f16(
        *_pb(hidden), *_pb(embedding), *_pb(state_offsets), *_pb(arc_tokens), *_pb(arc_next),
        *_pb(state_trace), *_pb(token_trace), *_pb(score_trace), *_pb(workspace), steps, batch,
        num_states, hidden_size, vocabulary_size, _sp(stream)))


# ---- dense full-vocabulary head (tcgen05) ---------------------------------

def dense_workspace_bytes(rows: int) -> int:
    return int(lib.mf_dense_workspace_bytes(rows))


def dense_head_f16(hidden: Buffer, embedding: Buffer, keys: Optional[Buffer],
                   token_ids: Optional[Buffer], scores: Optional[Buffer], workspace: Buffer,
                   rows: int, hidden_size: int, vocab_rows: int, vocab_begin: int,
                   stream) -> Status:
    """Full-vocabulary greedy head over one vocabulary shard (replaces
    linear_f16 + greedy_select_f16): packed keys and/or ids and scores."""
    return _status(lib.mf_dense_head_f16(
        *_pb(hidden), *_pb(embedding), *_pb(keys), *_pb(token_ids), *_pb(scores),
        *_pb(workspace), rows, hidden_size, vocab_rows, vocab_begin, _sp(stream)))


def dense_head_f16_ex(hidden: Buffer, embedding: Buffer, keys: Optional[Buffer],
                      token_ids: Optional[Buffer], scores: Optional[Buffer], workspace: Buffer,
                      rows: int, hidden_size: int, vocab_rows: int, vocab_begin: int,
                      launch_flags: int, stream) -> Status:
    """``dense_head_f16`` with launch options (``LAUNCH_OVERLAP_PREVIOUS``)."""
    return _status(lib.mf_dense_head_f16_ex(
        *_pb(hidden), *_pb(embedding), *_pb(keys), *_pb(token_ids), *_pb(scores),
        *_pb(workspace), rows, hidden_size, vocab_rows, vocab_begin, launch_flags, _sp(stream)))


def decode_keys(keys: Buffer, token_ids: Buffer, scores: Optional[Buffer], rows: int,
                stream) -> Status:
    """Packed keys (after a cross-shard max) -> ids and scores."""
    return _status(lib.mf_decode_keys(*_pb(keys), *_pb(token_ids), *_pb(scores), rows,
                                      _sp(stream)))


IPC_HANDLE_BYTES = 64


def exchange_bytes(rows: int, world: int) -> int:
    """Bytes of one rank's exchange buffer for ``dense_head_sharded_f16``."""
    return int(lib.mf_exchange_bytes(rows, world))


def exchange_broken(buffer) -> int:
    """1 once a sharded call on this rank's exchange buffer (a device tensor
    or address) gave up on a peer or saw a peer fail, else 0.  A broken
    buffer gives every row the sentinel until new buffers are made.  Reads
    the word synchronously."""
    ptr = buffer.data_ptr() if hasattr(buffer, "data_ptr") else int(buffer)
    out = ctypes.c_uint32()
    st = _status(lib.mf_exchange_broken(ctypes.c_void_p(ptr), ctypes.byref(out)))
    if not st.ok():
        raise RuntimeError(f"mf_exchange_broken failed: {st}")
    return int(out.value)


def dense_head_sharded_f16(hidden: Buffer, embedding: Buffer, keys: Optional[Buffer],
                           token_ids: Optional[Buffer], scores: Optional[Buffer],
                           workspace: Buffer, rows: int, hidden_size: int, vocab_rows: int,
                           vocab_begin: int, exchange, stream, launch_flags: int = 0) -> Status:
    """Vocabulary shards on several GPUs merged inside the dense kernel: every
    rank calls this on its own shard (``vocab_begin`` = the shard's first id)
    and gets the global ids / scores / keys.  ``exchange`` is a
    ``VocabShardExchange`` (or any object with ``ptrs``, ``nbytes``,
    ``world`` and ``rank``)."""
    arr = (ctypes.c_void_p * len(exchange.ptrs))(*exchange.ptrs)
    return _status(lib.mf_dense_head_sharded_f16(
        *_pb(hidden), *_pb(embedding), *_pb(keys), *_pb(token_ids), *_pb(scores),
        *_pb(workspace), rows, hidden_size, vocab_rows, vocab_begin, arr, exchange.nbytes,
        exchange.world, exchange.rank, launch_flags, _sp(stream)))


class VocabShardExchange:
    """The exchange buffers of ``dense_head_sharded_f16``: this rank allocates
    its own (``mf_exchange_alloc``), the 64-byte CUDA IPC handles are
    all-gathered (``all_gather(bytes) -> list[bytes]``, by default
    ``torch.distributed.all_gather_object`` on ``group``) and every peer's
    buffer is mapped here (``mf_exchange_open_peer``).  One process per GPU;
    the current device must be this rank's GPU."""

    def __init__(self, rows: int, world: int = None, rank: int = None, group=None,
                 all_gather=None):
        if world is None or rank is None:
            import torch.distributed as dist

            world, rank = dist.get_world_size(group), dist.get_rank(group)
        if all_gather is None:
            import torch.distributed as dist

            def all_gather(b: bytes):
                out = [None] * world
                dist.all_gather_object(out, b, group=group)
                return out
        self.world, self.rank, self.rows = int(world), int(rank), int(rows)
        self.nbytes = exchange_bytes(rows, world)
        own, handle = ctypes.c_void_p(), ctypes.create_string_buffer(IPC_HANDLE_BYTES)
        st = _status(lib.mf_exchange_alloc(ctypes.byref(own), self.nbytes, handle))
        if not st.ok():
            raise RuntimeError(f"mf_exchange_alloc failed: {st}")
        self._own = own.value
        self._opened = []
        handles = all_gather(handle.raw)
        ptrs = []
        try:
            for q, h in enumerate(handles):
                if q == self.rank:
                    ptrs.append(self._own)
                    continue
                peer = ctypes.c_void_p()
                st = _status(lib.mf_exchange_open_peer(ctypes.create_string_buffer(h, len(h)),
                                                       ctypes.byref(peer)))
                if not st.ok():
                    raise RuntimeError(f"mf_exchange_open_peer({q}) failed: {st}")
                self._opened.append(peer.value)
                ptrs.append(peer.value)
        except Exception:
            self.close()
            raise
        self.ptrs = ptrs

    def close(self) -> None:
        for p in self._opened:
            lib.mf_exchange_close_peer(p)
        self._opened = []
        if self._own:
            lib.mf_exchange_free(self._own)
            self._own = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


KEY_SIGN_FLIP = 1 << 63
"""XOR with this maps the unsigned key order onto signed int64 order, so a
signed MAX all-reduce (NCCL / torch.distributed) merges keys correctly."""


class RaggedHead:
    """Owns the workspace for repeated ragged-head calls on one stream.

    ``embedding`` stays resident; each ``__call__`` takes a batch of hidden
    rows and its CSR allowed sets (device tensors) and returns
    ``(token_ids, scores)`` device tensors, which are made (from the stream's
    memory, 25 us of host time where it is not the current one) unless given.
    Without a ``stream`` the constructor waits for the work queued on the
    current stream.
    """

    def __init__(self, embedding, max_rows: int, stream=None):
        import torch

        self.embedding = embedding
        self.vocab, self.hidden_size = int(embedding.shape[0]), int(embedding.shape[1])
        self.max_rows = int(max_rows)
        self._memory = _Workspace(
            lambda: torch.zeros(head_workspace_bytes(self.max_rows), dtype=torch.uint8,
                                device=embedding.device), embedding.device, stream)
        self.workspace = self._memory.tensor
        self.stream = stream

    def __call__(self, hidden, offsets, ids, out_ids=None, out_scores=None):
        import torch

        rows = int(hidden.shape[0])
        if rows > self.max_rows:
            raise ValueError(f"batch of {rows} rows exceeds max_rows={self.max_rows}")
        if out_ids is None or out_scores is None:
            device = hidden.device
            ids_made, scores_made = _outputs_on(
                self.stream, device,
                None if out_ids is not None else
                lambda: torch.empty(rows, dtype=torch.int32, device=device),
                None if out_scores is not None else
                lambda: torch.empty(rows, dtype=torch.float32, device=device))
            out_ids = ids_made if out_ids is None else out_ids
            out_scores = scores_made if out_scores is None else out_scores
        ws = self.workspace[: head_workspace_bytes(rows)]
        stream = self.stream
        if stream is None:
            stream = torch.cuda.current_stream()
            self._memory.used_on(stream)
        st = restricted_output_head_csr_f16(hidden, self.embedding, offsets, ids, out_ids,
                                            out_scores, ws, rows, self.hidden_size, self.vocab,
                                            stream)
        if not st.ok():
            raise RuntimeError(f"restricted head failed: {st}")
        return out_ids, out_scores


# ---- losses over the tied table (include/mf_loss.h) ------------------------

def dense_loss_workspace_bytes(rows: int, hidden_size: int, vocab: int) -> int:
    """Workspace of the forward calls; 0 for sizes outside the limits."""
    return int(lib.mf_dense_loss_workspace_bytes(rows, hidden_size, vocab))


def dense_loss_backward_workspace_bytes(rows: int, hidden_size: int, vocab: int) -> int:
    """Workspace of the backward calls; 0 for sizes outside the limits."""
    return int(lib.mf_dense_loss_backward_workspace_bytes(rows, hidden_size, vocab))


def _xent(f, hidden, embedding, targets, losses, lse, workspace, rows, hidden_size, vocab, stream):
    return _status(f(*_pb(hidden), *_pb(embedding), *_pb(targets), *_pb(losses), *_pb(lse),
                     *_pb(workspace), rows, hidden_size, vocab, _sp(stream)))


def dense_xent_f16(hidden: Buffer, embedding: Buffer, targets: Buffer, losses: Buffer, lse: Buffer,
                   workspace: Buffer, rows: int, hidden_size: int, vocab: int, stream) -> Status:
    """Softmax cross entropy of each row's target over the whole vocabulary:
    losses[r] = lse[r] - score(r, targets[r]).  INVALID_TOKEN_ID rows are
    ignored (loss 0)."""
    return _xent(lib.mf_dense_xent_f16, hidden, embedding, targets, losses, lse, workspace, rows,
                 hidden_size, vocab, stream)


def dense_xent_bf16(hidden: Buffer, embedding: Buffer, targets: Buffer, losses: Buffer, lse: Buffer,
                    workspace: Buffer, rows: int, hidden_size: int, vocab: int, stream) -> Status:
    """``dense_xent_f16`` on bfloat16 hidden rows and table."""
    return _xent(lib.mf_dense_xent_bf16, hidden, embedding, targets, losses, lse, workspace, rows,
                 hidden_size, vocab, stream)


def _xent_backward(f, hidden, embedding, targets, lse, grad_losses, d_hidden, d_embedding,
                   workspace, rows, hidden_size, vocab, stream):
    return _status(f(*_pb(hidden), *_pb(embedding), *_pb(targets), *_pb(lse), *_pb(grad_losses),
                     *_pb(d_hidden), *_pb(d_embedding), *_pb(workspace), rows, hidden_size, vocab,
                     _sp(stream)))


def dense_xent_backward_f16(hidden: Buffer, embedding: Buffer, targets: Buffer, lse: Buffer,
                            grad_losses: Buffer, d_hidden: Optional[Buffer],
                            d_embedding: Optional[Buffer], workspace: Buffer, rows: int,
                            hidden_size: int, vocab: int, stream) -> Status:
    """Gradients of sum(grad_losses * losses) of ``dense_xent_f16`` (either
    output may be None)."""
    return _xent_backward(lib.mf_dense_xent_backward_f16, hidden, embedding, targets, lse,
                          grad_losses, d_hidden, d_embedding, workspace, rows, hidden_size, vocab,
                          stream)


def dense_xent_backward_bf16(hidden: Buffer, embedding: Buffer, targets: Buffer, lse: Buffer,
                             grad_losses: Buffer, d_hidden: Optional[Buffer],
                             d_embedding: Optional[Buffer], workspace: Buffer, rows: int,
                             hidden_size: int, vocab: int, stream) -> Status:
    """``dense_xent_backward_f16`` on bfloat16 hidden rows and table."""
    return _xent_backward(lib.mf_dense_xent_backward_bf16, hidden, embedding, targets, lse,
                          grad_losses, d_hidden, d_embedding, workspace, rows, hidden_size, vocab,
                          stream)


def _distill(f, hidden, embedding, offsets, ids, teacher_logits, temperature, losses, lse,
             workspace, rows, hidden_size, vocab, stream):
    return _status(f(*_pb(hidden), *_pb(embedding), *_pb(offsets), *_pb(ids), *_pb(teacher_logits),
                     float(temperature), *_pb(losses), *_pb(lse), *_pb(workspace), rows,
                     hidden_size, vocab, _sp(stream)))


def dense_distill_f16(hidden: Buffer, embedding: Buffer, offsets: Buffer, ids: Optional[Buffer],
                      teacher_logits: Optional[Buffer], temperature: float, losses: Buffer,
                      lse: Buffer, workspace: Buffer, rows: int, hidden_size: int, vocab: int,
                      stream) -> Status:
    """Distillation from a teacher's top logits: row r's entries are
    [offsets[r], offsets[r+1]) of ids (ascending) and teacher_logits;
    losses[r] = T^2 KL(teacher over its set || student over the vocabulary)."""
    return _distill(lib.mf_dense_distill_f16, hidden, embedding, offsets, ids, teacher_logits,
                    temperature, losses, lse, workspace, rows, hidden_size, vocab, stream)


def dense_distill_bf16(hidden: Buffer, embedding: Buffer, offsets: Buffer, ids: Optional[Buffer],
                       teacher_logits: Optional[Buffer], temperature: float, losses: Buffer,
                       lse: Buffer, workspace: Buffer, rows: int, hidden_size: int, vocab: int,
                       stream) -> Status:
    """``dense_distill_f16`` on bfloat16 hidden rows and table."""
    return _distill(lib.mf_dense_distill_bf16, hidden, embedding, offsets, ids, teacher_logits,
                    temperature, losses, lse, workspace, rows, hidden_size, vocab, stream)


def _distill_backward(f, hidden, embedding, offsets, ids, teacher_logits, temperature, lse,
                      grad_losses, d_hidden, d_embedding, workspace, rows, hidden_size, vocab,
                      stream):
    return _status(f(*_pb(hidden), *_pb(embedding), *_pb(offsets), *_pb(ids), *_pb(teacher_logits),
                     float(temperature), *_pb(lse), *_pb(grad_losses), *_pb(d_hidden),
                     *_pb(d_embedding), *_pb(workspace), rows, hidden_size, vocab, _sp(stream)))


def dense_distill_backward_f16(hidden: Buffer, embedding: Buffer, offsets: Buffer,
                               ids: Optional[Buffer], teacher_logits: Optional[Buffer],
                               temperature: float, lse: Buffer, grad_losses: Buffer,
                               d_hidden: Optional[Buffer], d_embedding: Optional[Buffer],
                               workspace: Buffer, rows: int, hidden_size: int, vocab: int,
                               stream) -> Status:
    """Gradients of sum(grad_losses * losses) of ``dense_distill_f16`` (either
    output may be None)."""
    return _distill_backward(lib.mf_dense_distill_backward_f16, hidden, embedding, offsets, ids,
                             teacher_logits, temperature, lse, grad_losses, d_hidden, d_embedding,
                             workspace, rows, hidden_size, vocab, stream)


def dense_distill_backward_bf16(hidden: Buffer, embedding: Buffer, offsets: Buffer,
                                ids: Optional[Buffer], teacher_logits: Optional[Buffer],
                                temperature: float, lse: Buffer, grad_losses: Buffer,
                                d_hidden: Optional[Buffer], d_embedding: Optional[Buffer],
                                workspace: Buffer, rows: int, hidden_size: int, vocab: int,
                                stream) -> Status:
    """``dense_distill_backward_f16`` on bfloat16 hidden rows and table."""
    return _distill_backward(lib.mf_dense_distill_backward_bf16, hidden, embedding, offsets, ids,
                             teacher_logits, temperature, lse, grad_losses, d_hidden, d_embedding,
                             workspace, rows, hidden_size, vocab, stream)


class DenseLoss:
    """Owns the workspace for repeated loss calls on one stream.

    ``embedding`` (fp16 or bfloat16 [vocab, hidden_size], contiguous) stays
    resident and is read in place, so an optimizer may update it between
    calls.  Forward methods return ``(losses, lse)``, backward methods
    ``(d_hidden, d_embedding)``; outputs are allocated unless given, and a
    gradient is left out (None) with ``hidden_grad=False`` /
    ``embedding_grad=False``.  With ``backward=False`` only the forward
    workspace is kept.  ``stream`` defaults to the current stream, which must
    not be the legacy default stream; without one the constructor waits for the
    work queued on the current stream.  The workspace is safe on every stream
    that calls use, and the object may be dropped while they run.  The caller
    orders what was made on another stream before the call
    (``Stream.wait_stream``), keeps its memory until the call is done
    (``Tensor.record_stream``), as for any tensor used on another stream than
    its own, and keeps the object for as long as a graph captured from its
    calls is replayed.  Calls of one object share its workspace: they must not
    overlap on the GPU.
    """

    def __init__(self, embedding, max_rows: int, stream=None, backward: bool = True):
        import torch

        kinds = {torch.float16: "f16", torch.bfloat16: "bf16"}
        if embedding.dtype not in kinds or embedding.dim() != 2 or not embedding.is_contiguous():
            raise ValueError("the table is a contiguous fp16 or bfloat16 [vocab, hidden_size]")
        self.embedding = embedding
        self.vocab, self.hidden_size = int(embedding.shape[0]), int(embedding.shape[1])
        self.max_rows, self.stream = int(max_rows), stream
        sizes = (self.max_rows, self.hidden_size, self.vocab)
        nbytes = dense_loss_workspace_bytes(*sizes)
        if nbytes == 0:
            raise ValueError(f"rows, hidden_size, vocab = {sizes} are outside the limits")
        if backward:
            nbytes = max(nbytes, dense_loss_backward_workspace_bytes(*sizes))
        self._backward, self._torch = backward, torch
        self._i32, self._f32, self._kind = torch.int32, torch.float32, embedding.dtype
        self._device, self._index = embedding.device, embedding.get_device()
        self._table_shape = (self.vocab, self.hidden_size)
        self._table_bytes, self._workspace_bytes = self.vocab * self.hidden_size * 2, nbytes
        kind = kinds[embedding.dtype]
        self._functions = {n: getattr(lib, f"mf_dense_{n}_{kind}")
                           for n in ("xent", "xent_backward", "distill", "distill_backward")}
        self._memory = _Workspace(
            lambda: torch.empty(nbytes, dtype=torch.uint8, device=self._device), self._device, stream)
        self.workspace = self._memory.tensor

    def _on(self):
        """The stream of the call, as torch knows it."""
        if self.stream is None:
            return self._torch.cuda.current_stream(self._device)
        return _torch_stream(self.stream)

    def _wrong(self, name, t, dtype, shape):
        return ValueError(f"{name}: a contiguous {dtype} tensor of shape {shape} on {self._device} "
                          f"is wanted, not {t.dtype} {tuple(t.shape)} on {t.device}")

    def _in(self, args, name, t, dtype, shape, nbytes):
        """Checks an input and appends its address and bytes."""
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self._index \
                or not t.is_contiguous():
            raise self._wrong(name, t, dtype, shape)
        args += (t.data_ptr(), nbytes)

    def _out(self, args, name, t, dtype, shape, nbytes):
        """The same for an output, which is made if it is not given: from the
        memory of the stream that writes it."""
        if t is None:
            torch = self._torch
            with torch.cuda.device(self._device), torch.cuda.stream(self._on()):
                t = torch.empty(shape, dtype=dtype, device=self._device)
        self._in(args, name, t, dtype, shape, nbytes)
        return t

    def _begin(self, hidden):
        """Rows, the shape and bytes of a float or int32 per row, and the call's
        arguments so far."""
        rows = hidden.shape[0]
        if rows > self.max_rows:
            raise ValueError(f"batch of {rows} rows exceeds max_rows={self.max_rows}")
        args, width, kind = [], self.hidden_size, self._kind
        self._in(args, "hidden", hidden, kind, (rows, width), rows * width * 2)
        self._in(args, "embedding", self.embedding, kind, self._table_shape, self._table_bytes)
        return rows, (rows,), rows * 4, args

    def _sets(self, args, rows, offsets, ids, teacher_logits, temperature):
        n = ids.numel()
        self._in(args, "offsets", offsets, self._i32, (rows + 1,), rows * 4 + 4)
        self._in(args, "ids", ids, self._i32, (n,), n * 4)
        self._in(args, "teacher_logits", teacher_logits, self._f32, (n,), n * 4)
        args.append(float(temperature))

    def _call(self, name, args, rows):
        if self._index < 0:
            raise ValueError(f"the table and its batches lie on {self._device}, not on a GPU")
        if self._torch.cuda.current_device() != self._index:
            with self._torch.cuda.device(self._device):
                code = self._launch(name, args, rows)
        else:
            code = self._launch(name, args, rows)
        if code.code:
            raise RuntimeError(f"mf_dense_{name} failed: {_status(code)}")

    def _launch(self, name, args, rows):
        stream = self.stream
        if stream is None:
            stream = self._torch.cuda.current_stream(self._device)
            self._memory.used_on(stream)
        ws = self.workspace
        return self._functions[name](*args, ws.data_ptr(), self._workspace_bytes, rows,
                                     self.hidden_size, self.vocab, _stream_handle(stream))

    def _losses(self, args, shape, nbytes, losses, lse):
        losses = self._out(args, "losses", losses, self._f32, shape, nbytes)
        return losses, self._out(args, "lse", lse, self._f32, shape, nbytes)

    def cross_entropy(self, hidden, targets, losses=None, lse=None):
        """targets int32 [rows]; -1 (``INVALID_TOKEN_ID``) ignores a row."""
        rows, shape, nbytes, args = self._begin(hidden)
        self._in(args, "targets", targets, self._i32, shape, nbytes)
        out = self._losses(args, shape, nbytes, losses, lse)
        self._call("xent", args, rows)
        return out

    def distill(self, hidden, offsets, ids, teacher_logits, temperature=1.0, losses=None,
                lse=None):
        """The teacher's top logits as CSR: offsets int32 [rows + 1], ids int32
        (ascending within a row) and teacher_logits float32 [entries]."""
        rows, shape, nbytes, args = self._begin(hidden)
        self._sets(args, rows, offsets, ids, teacher_logits, temperature)
        out = self._losses(args, shape, nbytes, losses, lse)
        self._call("distill", args, rows)
        return out

    def _gradients(self, args, rows, lse, grad_losses, d_hidden, d_embedding, hidden_grad,
                   embedding_grad):
        if not self._backward:
            raise RuntimeError("this DenseLoss was made with backward=False")
        shape, nbytes, width = (rows,), rows * 4, self.hidden_size
        self._in(args, "lse", lse, self._f32, shape, nbytes)
        self._in(args, "grad_losses", grad_losses, self._f32, shape, nbytes)
        if hidden_grad:
            d_hidden = self._out(args, "d_hidden", d_hidden, self._kind, (rows, width),
                                 rows * width * 2)
        else:
            d_hidden = None
            args += (0, 0)
        if embedding_grad:
            d_embedding = self._out(args, "d_embedding", d_embedding, self._kind,
                                    self._table_shape, self._table_bytes)
        else:
            d_embedding = None
            args += (0, 0)
        return d_hidden, d_embedding

    def cross_entropy_backward(self, hidden, targets, lse, grad_losses, d_hidden=None,
                               d_embedding=None, hidden_grad=True, embedding_grad=True):
        """Gradients of ``(grad_losses * losses).sum()``; ``lse`` as
        ``cross_entropy`` returned it."""
        rows, shape, nbytes, args = self._begin(hidden)
        self._in(args, "targets", targets, self._i32, shape, nbytes)
        out = self._gradients(args, rows, lse, grad_losses, d_hidden, d_embedding, hidden_grad,
                              embedding_grad)
        self._call("xent_backward", args, rows)
        return out

    def distill_backward(self, hidden, offsets, ids, teacher_logits, temperature, lse, grad_losses,
                         d_hidden=None, d_embedding=None, hidden_grad=True, embedding_grad=True):
        """Gradients of ``(grad_losses * losses).sum()``; ``lse`` as ``distill``
        returned it with the same temperature."""
        rows, _, _, args = self._begin(hidden)
        self._sets(args, rows, offsets, ids, teacher_logits, temperature)
        out = self._gradients(args, rows, lse, grad_losses, d_hidden, d_embedding, hidden_grad,
                              embedding_grad)
        self._call("distill_backward", args, rows)
        return out


class HostPipeline:
    """Restricted head over batches that live in host memory (native
    ``mf_pipeline_*``): each ``submit`` copies one batch (hidden rows, CSR
    offsets, CSR ids) from pinned host memory to the device, runs the ragged
    head and copies ids and scores back into pinned host memory, in order on
    the stream of the next of ``depth`` slots (each slot has its own device
    buffers and workspace), so batches on different slots overlap.  Host
    tensors must stay untouched until ``wait(ticket)`` returns.
    """

    def __init__(self, embedding, max_rows: int, max_ids: int, depth: int = 6, device=None):
        self.embedding = embedding  # keeps the device table alive
        self.vocab, self.hidden_size = int(embedding.shape[0]), int(embedding.shape[1])
        self._p = ctypes.c_void_p()
        self._ticket = ctypes.c_uint64()
        self._ticket_ref = ctypes.byref(self._ticket)
        st = _status(lib.mf_pipeline_create(ctypes.byref(self._p), *_pb(embedding), self.vocab,
                                            self.hidden_size, int(max_rows), int(max_ids),
                                            int(depth)))
        if not st.ok():
            raise RuntimeError(f"mf_pipeline_create failed: {st}")

    def depth(self) -> int:
        """Number of slots (batches in flight)."""
        return int(lib.mf_pipeline_depth(self._p))

    def stream(self, slot: int) -> int:
        """cudaStream_t of slot ``slot`` (copy in, head, copy out in order)."""
        return int(lib.mf_pipeline_stream(self._p, slot) or 0)

    def submit(self, hidden, offsets, ids, out_ids, out_scores=None) -> int:
        """hidden fp16 [rows, H], offsets int32 [rows + 1], ids int32 [total],
        out_ids int32 [rows], out_scores float32 [rows] or None: pinned host
        tensors.  Returns the batch's ticket."""
        return self.submit_ptrs(hidden.data_ptr(), hidden.shape[0], offsets.data_ptr(),
                                ids.data_ptr(), ids.shape[0], out_ids.data_ptr(),
                                out_scores.data_ptr() if out_scores is not None else None)

    def submit_ptrs(self, hidden: int, rows: int, offsets: int, ids: int, total_ids: int,
                    out_ids: int, out_scores) -> int:
        """``submit`` with raw host addresses (for callers that keep their own
        pinned buffers)."""
        s = lib.mf_pipeline_submit(self._p, hidden, rows, offsets, ids or None, total_ids,
                                   out_ids, out_scores, self._ticket_ref)
        if s.code:
            raise RuntimeError(f"mf_pipeline_submit failed: {_status(s)}")
        return self._ticket.value

    @staticmethod
    def pack(hidden, offsets, ids, u16_ids: bool = False):
        """One pinned uint8 host buffer holding hidden fp16 [rows, H], offsets
        int32 [rows + 1] and ids int32 [total] back to back (the layout of
        ``submit_packed``); with ``u16_ids`` the ids as uint16 (the layout of
        ``submit_packed(..., u16_ids=True)``, vocabularies of at most 65,536)."""
        import numpy as np
        import torch

        if u16_ids:
            a = np.asarray(ids)
            if a.size and (a.min() < 0 or a.max() > 0xFFFF):
                raise ValueError("ids outside [0, 65535] do not fit uint16")
            ids = torch.from_numpy(a.astype(np.uint16).view(np.int16))
        parts = [torch.as_tensor(x).contiguous().view(torch.uint8).reshape(-1)
                 for x in (hidden, offsets, ids)]
        buf = torch.empty(sum(p.numel() for p in parts), dtype=torch.uint8).pin_memory()
        at = 0
        for part in parts:
            buf[at:at + part.numel()] = part
            at += part.numel()
        return buf

    def submit_packed_ptrs(self, batch: int, batch_bytes: int, rows: int, total_ids: int,
                           out: int, u16_ids: bool = False) -> int:
        """One packed batch (see ``pack``) at host address ``batch``; ``out``
        receives ids u32 [rows] then scores f32 [rows].  One H2D and one D2H
        copy per batch."""
        f = lib.mf_pipeline_submit_packed_u16ids if u16_ids else lib.mf_pipeline_submit_packed
        s = f(self._p, batch, batch_bytes, rows, total_ids, out, self._ticket_ref)
        if s.code:
            raise RuntimeError(f"mf_pipeline_submit_packed failed: {_status(s)}")
        return self._ticket.value

    def submit_packed(self, batch, rows: int, total_ids: int, out, u16_ids: bool = False) -> int:
        """``batch`` from ``pack`` (with the same ``u16_ids``); ``out`` a pinned
        host tensor of 8 * rows bytes."""
        return self.submit_packed_ptrs(batch.data_ptr(), batch.numel() * batch.element_size(),
                                       rows, total_ids, out.data_ptr(), u16_ids)

    def wait(self, ticket: int) -> None:
        st = _status(lib.mf_pipeline_wait(self._p, ticket))
        if not st.ok():
            raise RuntimeError(f"mf_pipeline_wait failed: {st}")

    def synchronize(self) -> None:
        st = _status(lib.mf_pipeline_synchronize(self._p))
        if not st.ok():
            raise RuntimeError(f"mf_pipeline_synchronize failed: {st}")

    def close(self) -> None:
        if self._p:
            lib.mf_pipeline_destroy(self._p)
            self._p = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
