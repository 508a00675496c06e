"""Beam search over constrained rows: selection, reordering of per-beam state, back-trace.

The engine says which tokens a row may take; these functions decode with beams under it.  A
batch holds `groups` requests of `beams` beams; row r = group * beams + beam.  One step:

    got = beam_select(logits, scores, mask=mask, finished=finished, end_token=eos)
    beam_reorder(caches, got.beams, lengths=written, dim=2)     # the model's per-beam state
    tokens_trace[t], beams_trace[t] = got.tokens, got.beams
    scores, finished = got.scores, got.finished
    ...
    texts = beam_sequences(tokens_trace[:t], beams_trace[:t])

`Engine.beam_select` does the first under the masks of the engine's slots, read in place (the
logits are not written), and `Engine.reorder` moves the slots' constraint states.  Kernels and
C entry points: csrc/beams.cu, include/xgraph_b200.h.  The reference has no counterpart.

Every function takes `stream` (a raw cudaStream_t as int, 0 = the default stream, as the engine's
methods do, whatever torch's current stream is: under `torch.cuda.stream(s)` give
`stream=s.cuda_stream`), enqueues its kernels there and does not wait; tensors are on one GPU and
stay valid until the stream has passed the call.  Captured into a CUDA graph (stream = the
capturing stream), a call keeps its own workspace in the graph's memory.  No gradient goes
through these functions: results need none, whether or not the inputs do.
"""

from __future__ import annotations

import ctypes
import struct
from collections.abc import Sequence
from contextlib import nullcontext
from typing import NamedTuple

MAX_BEAMS = 64
MAX_CANDIDATES = 128
MAX_BEAM_VOCAB = 1 << 20
_INT32 = (1 << 31) - 1

# XgRowTensor: data, then rows, row_stride, size[4], stride[4], dims, element_bytes, position_dim, reserved
_ADDRESS, _ROW_LAYOUT = struct.Struct("<q"), struct.Struct("<qq4q4q4i")

_torch = None
_lib = None
_call_errors = None
_get_device = _get_stream = None  # the current device, and its current raw stream
_dtypes: dict = {}
_workspaces: dict[tuple, int] = {}  # bytes a selection of these sizes needs


class BeamCandidates(NamedTuple):
    """The best continuations of each group, best first: [groups, candidates] scores float32,
    the beam each goes on from (int32), its token (int32), and whether it has ended (bool).
    Places that no continuation fills hold -inf, -1, -1 and False."""

    scores: object
    beams: object
    tokens: object
    finished: object


def _load():
    """torch and the library, at the first call (this module imports without either)."""
    global _torch, _lib, _call_errors, _get_device, _get_stream
    if _lib is None:
        import torch

        from .engine import _check, load_library

        _call_errors, _torch = _check, torch
        _get_device, _get_stream = torch.cuda.current_device, torch._C._cuda_getCurrentRawStream
        _dtypes.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        _lib = load_library()  # last: another thread's first call may see it and go on
    return _torch


def _placed(device: int, stream: int):
    """The context in which a call's kernels run on `device` and what it allocates belongs to
    `stream`; None where that is the current state."""
    if _get_device() == device and _get_stream(device) == stream:
        return None
    return _torch.cuda.stream(_torch.cuda.ExternalStream(stream, device=device) if stream
                              else _torch.cuda.default_stream(device))


def _table(tensor, name: str, shape, dtype, device):
    """A contiguous tensor of this shape and type on `device`; its address."""
    if not isinstance(tensor, _torch.Tensor) or tensor.dtype != dtype or tensor.device != device:
        raise ValueError(f"{name} must be a {str(dtype).removeprefix('torch.')} tensor on {device}")
    if tensor.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(tensor.shape)}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return tensor.data_ptr()


def _check_sizes(groups: int, beams: int, vocab: int = 1, candidates: int = 1, steps: int = 0) -> None:
    """The limits, before a size reaches the C entry points, which take the low 32 bits of it."""
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"a group holds 1 to {MAX_BEAMS} beams, got {beams}")
    if not 1 <= candidates <= MAX_CANDIDATES:
        raise ValueError(f"candidates must be between 1 and {MAX_CANDIDATES}, got {candidates}")
    if not 1 <= vocab <= MAX_BEAM_VOCAB:
        raise ValueError(f"the vocabulary must hold 1 to {MAX_BEAM_VOCAB} tokens, got {vocab}")
    if groups > _INT32 or steps > _INT32:
        raise ValueError(f"too many {'groups' if groups > _INT32 else 'steps'}")


def beam_select(logits, scores, *, mask=None, finished=None, candidates: int | None = None, vocab: int | None = None,
                end_token: int | None = None, renormalize: bool = True, stream: int = 0) -> BeamCandidates:
    """The `candidates` best continuations of each group (default: as many as beams).

    logits [groups * beams, columns] (float32, bfloat16 or float16; unit column stride, any row
    stride) and scores [groups, beams] (float32, each beam's log-probability so far).
    Continuing beam b with token v scores scores[b] + logits[v] - log(sum of exp(logits)), the
    sum over the tokens that b may take (renormalize) or over the whole vocabulary (the
    model's own probabilities).  A token may be taken when it is below `vocab` (default: every
    column), its bit is set in `mask` (int32 words [groups * beams, >= ceil(vocab / 32)], bit i
    of word w = token 32 w + i, as Engine.mask holds them) and its logit is not -inf.

    `finished` (bool [groups, beams]) marks beams that have ended: each offers one
    continuation, end_token, at its own score.  A continuation has ended when its beam had or
    its token is end_token.  Order: the score in 64 bits, equal scores by the lower (beam,
    token); of unequal logits that 64 bits score alike, either may be offered first.  The scores
    returned are within half a float32 unit in the last place, plus 1e-6, of the exact ones, and
    their last bits may differ with the batch that a row is in.
    A beam of score -inf is empty (start a search with scores [0, -inf, ...]); a beam
    of NaN or +inf score, or whose logits hold a NaN or +inf that counts, offers nothing, and
    so does one that may take no token.  At most MAX_BEAMS beams, MAX_CANDIDATES candidates and
    MAX_BEAM_VOCAB tokens.
    """
    _load()
    return _select(None, logits, None, scores, mask, finished, candidates, vocab, end_token, renormalize, stream)


def _select(engine, logits, slots, scores, mask, finished, candidates, vocab, end_token, renormalize, stream):
    torch = _torch
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() != 2:
        raise ValueError("logits must be a 2-D tensor on the GPU")
    dtype = _dtypes.get(logits.dtype)
    if dtype is None:
        raise ValueError("logits must be float32, bfloat16 or float16")
    rows, columns = logits.shape
    row_stride, unit = logits.stride()
    if unit != 1 and columns > 1 and rows:
        raise ValueError("logits need one contiguous row per beam")
    if not isinstance(scores, torch.Tensor) or scores.dim() != 2:
        raise ValueError("scores must be [groups, beams]")
    device = logits.device
    groups, beams = scores.shape
    scores_at = _table(scores, "scores", (groups, beams), torch.float32, device)
    if groups * beams != rows:
        raise ValueError(f"logits need one row per beam: {groups} x {beams} beams, {rows} rows")
    if row_stride < columns:
        if rows > 1:
            raise ValueError("logits rows overlap")
        row_stride = columns
    if vocab is None:
        vocab = columns
    elif not 1 <= vocab <= columns:
        raise ValueError(f"vocab must be between 1 and the {columns} columns, got {vocab}")
    wanted = beams if candidates is None else int(candidates)
    _check_sizes(groups, beams, vocab, wanted)
    mask_at, mask_stride = None, 0
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.int32 or mask.device != device or mask.dim() != 2:
            raise ValueError(f"mask must be a 2-D int32 tensor on {device}")
        words = (vocab + 31) // 32
        if mask.shape[0] != rows or mask.shape[1] < words:
            raise ValueError(f"mask must have {rows} rows of at least {words} words, got {list(mask.shape)}")
        if mask.stride(1) != 1 and words > 1:
            raise ValueError("mask needs one contiguous row per beam")
        mask_at, mask_stride = mask.data_ptr(), mask.stride(0) if rows > 1 else words
        if mask_stride < words:
            raise ValueError("mask rows overlap")
    finished_at = None
    if finished is not None:
        if end_token is None:
            raise ValueError("finished beams need end_token, the token they go on with")
        finished_at = _table(finished, "finished", (groups, beams), torch.bool, device)
    if end_token is not None and not 0 <= end_token < vocab:
        raise ValueError(f"end_token must be a token below {vocab}, got {end_token}")
    index = device.index
    if engine is None:
        call, head = _lib.xg_beam_select, (logits.data_ptr(), dtype, groups, beams, vocab, row_stride, scores_at,
                                           mask_at, mask_stride)
    else:
        call, head = _lib.xg_engine_beam_select, (engine, logits.data_ptr(), dtype, groups, beams, vocab, row_stride,
                                                  slots, scores_at)
    rest = (finished_at, wanted, -1 if end_token is None else end_token, 1 if renormalize else 0)
    sizes = (index, groups, beams, vocab, dtype, wanted)
    placed = _placed(index, stream)
    if placed is None:
        return _launch_select(call, head, rest, sizes, device, stream)
    with placed:
        return _launch_select(call, head, rest, sizes, device, stream)


def _launch_select(call, head, rest, sizes, device, stream):
    size = _workspaces.get(sizes)
    if size is None:
        out = ctypes.c_int64()
        _call_errors(_lib.xg_beam_workspace(*sizes[1:], ctypes.byref(out)))
        if len(_workspaces) > 4096:
            _workspaces.clear()
        size = _workspaces[sizes] = out.value
    torch, groups, wanted = _torch, sizes[1], sizes[5]
    empty, shape, strides = torch.empty_strided, (groups, wanted), (wanted, 1)
    workspace = empty((size,), (1,), dtype=torch.uint8, device=device)
    scores = empty(shape, strides, dtype=torch.float32, device=device)
    beams = empty(shape, strides, dtype=torch.int32, device=device)
    tokens = empty(shape, strides, dtype=torch.int32, device=device)
    finished = empty(shape, strides, dtype=torch.bool, device=device)
    rc = call(*head, *rest, scores.data_ptr(), beams.data_ptr(), tokens.data_ptr(), finished.data_ptr(),
              workspace.data_ptr(), size, stream)
    if rc:
        _call_errors(rc)
    return BeamCandidates(scores, beams, tokens, finished)


def beam_reorder(tensors, beams, *, lengths=None, dim: int | Sequence[int] | None = None, rows=None,
                 stream: int = 0) -> None:
    """Per-beam state after a selection: in every tensor, row (group, b) takes what row (group,
    beams[group, b]) held, in place and in one launch (64 tensors each).

    tensors: one tensor or a sequence, each with the beams' rows as its first dimension (all
    with the same number of rows), up to four more dimensions, any type of 1 to 16 bytes and
    any non-overlapping strides that leave at most two strided dimensions outside a contiguous
    run.  beams [groups, beams] int32; an entry outside [0, beams) (a place that no
    continuation filled) leaves its row as it is.  rows [groups, beams] int32 (distinct) names
    the tensors' rows of the beams, for example engine slots; default: row group * beams + b.

    With lengths [groups] int32 only the positions below lengths[group] of dimension `dim` of
    each tensor move (one dimension for all or one per tensor), such as the written part of a
    cache; everything else keeps its value.  Tensors must not share memory, also not with
    beams, lengths and rows; those without elements are left out.
    """
    torch = _load()
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not isinstance(beams, torch.Tensor) or beams.dim() != 2 or not beams.is_cuda:
        raise ValueError("beams must be a [groups, beams] tensor on the GPU")
    device = beams.device
    groups, per_group = beams.shape
    beams_at = _table(beams, "beams", (groups, per_group), torch.int32, device)
    lengths_at = rows_at = None
    if lengths is not None:
        lengths_at = _table(lengths, "lengths", (groups,), torch.int32, device)
        if dim is None:
            raise ValueError("lengths need dim, the dimension they count")
    elif dim is not None:
        raise ValueError("dim goes with lengths")
    if rows is not None:
        rows_at = _table(rows, "rows", (groups, per_group), torch.int32, device)
    if not tensors:
        return
    _check_sizes(groups, per_group)
    if dim is not None and not isinstance(dim, int):
        dim = list(dim)
        if len(dim) != len(tensors):
            raise ValueError("dim needs one entry per tensor")
    records, count = _row_tensors(tensors, dim, device)
    if rows is None and count != groups * per_group:
        raise ValueError(f"the tensors need {groups * per_group} rows, one per beam, got {count}")
    with _placed(device.index, stream) or nullcontext():
        _call_errors(_lib.xg_beam_reorder(records, len(tensors), beams_at, groups, per_group, lengths_at, rows_at,
                                          stream))


def _row_tensors(tensors, dim, device) -> tuple[bytes, int]:
    """XgRowTensor records of the tensors, which must not share memory, and the first's rows."""
    kind, first = _torch.Tensor, tensors[0]
    if not isinstance(first, kind):
        raise ValueError("tensors must be torch tensors")
    shape, dtype, index = first.shape, first.dtype, device.index
    # one shape and type for all, without gaps, as a model's layers have: one layout serves
    if not isinstance(dim, list) and set(map(type, tensors)) == {kind} and all(
            [t.is_contiguous() and t.shape == shape and t.dtype == dtype and t.get_device() == index
             and not t.requires_grad for t in tensors]):
        layout, size, _ = _layout(first, dim, device)
        places = [t.data_ptr() for t in tensors]
        if len(places) > 1 and size:
            order = sorted(places)
            if min([b - a for a, b in zip(order, order[1:])]) < size:
                raise ValueError("the tensors share memory")
        return b"".join([_ADDRESS.pack(at) + layout for at in places]), shape[0]
    records, spans = [], []
    for k, tensor in enumerate(tensors):
        if not isinstance(tensor, kind):
            raise ValueError("tensors must be torch tensors")
        layout, size, dense = _layout(tensor, dim[k] if isinstance(dim, list) else dim, device)
        records.append(_ADDRESS.pack(tensor.data_ptr()) + layout)
        spans.append((tensor.data_ptr(), size, dense))
    _check_apart(spans)
    return b"".join(records), shape[0]


def _layout(tensor, dim, device) -> tuple[bytes, int, bool]:
    """What tensors of this layout share: their record after the address, the bytes from the
    first element to the last, and whether those are all the tensor's."""
    if tensor.device != device:
        raise ValueError(f"the tensors must be on {device}")
    if tensor.dim() < 1 or tensor.dim() > 5:
        raise ValueError("a tensor needs its rows as the first of 1 to 5 dimensions")
    size = tensor.element_size()
    if size not in (1, 2, 4, 8, 16) or tensor.layout != _torch.strided:
        raise ValueError(f"{tensor.dtype} tensors cannot be reordered")
    if tensor.is_neg() or tensor.is_conj() or tensor.requires_grad:
        raise ValueError("tensors that are lazily negated or conjugated, or need gradients, cannot be reordered")
    count = tensor.dim() - 1
    position = -1
    if dim is not None:
        position = dim if dim >= 0 else dim + tensor.dim()
        if not 1 <= position <= count:
            raise ValueError(f"dim must be one of a tensor's dimensions after its rows, got {dim}")
        position -= 1
    shape, strides = tensor.shape, tensor.stride()
    pad = (0,) * (4 - count)
    layout = _ROW_LAYOUT.pack(shape[0], strides[0], *shape[1:], *pad, *strides[1:], *pad, count, size, position, 0)
    if tensor.numel() == 0:
        return layout, 0, True
    elements = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    return layout, elements * size, elements == tensor.numel()


def _check_apart(spans):
    """Refuse tensors that share memory: two that begin at one place, or one that begins inside
    another without gaps.  (Interleaved ones, whose gaps hold each other, are apart.)"""
    filled, start = -1, -1  # the end of the dense tensors so far, and the last one's begin
    for at, size, dense in sorted(spans):
        if size and (at == start or at < filled):
            raise ValueError("the tensors share memory")
        if size:
            start = at
            if dense:
                filled = max(filled, at + size)


def beam_sequences(tokens, beams, *, lengths=None, pad_token: int = -1, stream: int = 0):
    """The token sequences that a search wrote: [groups, beams, steps] int32.

    tokens and beams [steps, groups, beams] int32 (unit stride over beams, any over steps and
    groups) hold each step's selected tokens and the beams they continued (beam_select's
    outputs, one step after another).  Sequence k of a group ends in place k of its last step,
    lengths[group] - 1 (lengths int32 [groups], clamped to [0, steps]; default: steps), and is
    read back from there; `pad_token` fills the positions from lengths[group] on and those
    before an entry of beams outside [0, beams).
    """
    torch = _load()
    for name, trace in (("tokens", tokens), ("beams", beams)):
        if not isinstance(trace, torch.Tensor) or not trace.is_cuda or trace.dtype != torch.int32 or trace.dim() != 3:
            raise ValueError(f"{name} must be a 3-D int32 tensor on the GPU")
        if trace.numel() and trace.shape[2] > 1 and trace.stride(2) != 1:
            raise ValueError(f"{name} must have unit stride over the beams")
    if tokens.shape != beams.shape or tokens.device != beams.device:
        raise ValueError("tokens and beams must have the same shape and device")
    steps, groups, per_group = tokens.shape
    _check_sizes(groups, per_group, steps=steps)
    device = tokens.device
    lengths_at = None if lengths is None else _table(lengths, "lengths", (groups,), torch.int32, device)
    if not -(1 << 31) <= pad_token < 1 << 31:
        raise ValueError(f"pad_token must be an int32, got {pad_token}")
    with _placed(device.index, stream) or nullcontext():
        out = torch.empty_strided((groups, per_group, steps), (per_group * steps, steps, 1), dtype=torch.int32,
                                  device=device)
        _call_errors(_lib.xg_beam_sequences(
            tokens.data_ptr(), tokens.stride(0), tokens.stride(1), beams.data_ptr(), beams.stride(0), beams.stride(1),
            steps, groups, per_group, lengths_at, pad_token, out.data_ptr(), stream))
    return out
