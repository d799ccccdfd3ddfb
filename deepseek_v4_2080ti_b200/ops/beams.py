"""Beam search on the device (csrc/kernels/beam_select.cu, beam_reorder.cu): which continuations of a request's beams are kept, and the beams'
states in their new order.

    scores, parents, tokens = beams.select(logits, scores)               # a step of the search, [requests, beams]
    beams.reorder([states, tails], parents, slots)                       # recurrent states; tables; the last pages of the beams' caches

The same selection grows a drafted tree (``ops.tree``): the beams are its newest nodes, the candidates the nodes that it gets next."""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import _lib
from .attention import _at, _current, _index, _status, _stream

MAX_BEAMS, MAX_CANDIDATES, MAX_VOCAB = 128, 128, 1 << 29          # (places of a row's tiles fit 32 bits)
MAX_STATES = 16                          # tensors of one launch
TILE = 8192                              # logits that a block looks at together
NUM_SMS = 148
# SelectCall, ReorderCall and ReorderState in ops.h, packed
_SELECT = struct.Struct("@iiPqPPPPPPPP10i0P")
_REORDER, _STATE = struct.Struct("@iiPPPP4i"), struct.Struct("@Pqqqii")
_REORDER_BYTES = _REORDER.size + MAX_STATES * _STATE.size
_REST = [b"\0" * ((MAX_STATES - i) * _STATE.size) for i in range(MAX_STATES + 1)]
_typed = False


def _kernels() -> ctypes.CDLL:
    global _typed
    lib = _lib.lib()
    if not _typed:
        for f in (lib.b200_beam_select, lib.b200_beam_reorder):
            f.argtypes = [ctypes.c_char_p]
        _typed = True
    return lib


def _parts(rows: int, vocab: int) -> tuple[int, int]:
    """Parts that a row is read in, and tiles of each."""
    tiles = -(-vocab // TILE)
    per = max(1, min(tiles, rows * tiles // (3 * NUM_SMS)))
    return -(-tiles // per), per


def select(logits: torch.Tensor, scores: torch.Tensor, n: int | None = None, finished: torch.Tensor | None = None,
           pad_token: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``n`` best continuations (default: as many as beams) of every request: ``scores[b, w] + log_softmax(logits[b, w])`` over all beams w and
    tokens, best first, of equals the lowest beam and token first (of one beam by the logits, also where 64 bits do not tell the sums apart).
    logits fp32 or bf16 [B, W, V] (tokens side by side; a whole vocabulary), scores fp32 [B, W].  Returns fp32 scores, int32 parents (beams) and int32 tokens, [B, n] each.

    A beam with ``finished`` (bool [B, W]) offers itself alone, with ``pad_token`` and its score as it is.  Tokens with a logit of -inf and beams with a
    score of -inf are not offered, nor are beams whose score or logits hold NaN or +inf; where fewer than n are left the rest is -inf, -1, -1.
    Scores are off by their rounding to 32 bits and 4.5e-7 + 5.1e-8 (log2 V + 2) at most (1.4e-6 at 248320 tokens); where candidates of different
    beams lie closer together than that their order is taken from sums to 2^-30, in 64 bits."""
    dev, shape = logits.get_device(), logits.shape
    if dev < 0 or len(shape) != 3 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits: fp32 or bf16 [requests, beams, vocabulary] on a GPU expected, got {logits.dtype} {list(shape)} on {logits.device}")
    if _current() != dev:
        with torch.cuda.device(dev):
            return select(logits, scores, n, finished, pad_token)
    b, w, v = shape
    n = w if n is None else int(n)
    if not 0 < w <= MAX_BEAMS or not 0 < n <= MAX_CANDIDATES or not 0 < v <= MAX_VOCAB:
        raise ValueError(f"{n} of {w} beams and {v} tokens: 1 to {MAX_BEAMS} beams, 1 to {MAX_CANDIDATES} candidates and 1 to {MAX_VOCAB} tokens expected")
    if not 0 <= pad_token < v:
        raise ValueError(f"pad_token {pad_token} of a vocabulary of {v}")
    sb, row, one = logits.stride()
    if w == 1:
        row = sb
    if v > 1 and one != 1 or b > 1 and sb != w * row or b * w > 1 and row < v:
        raise ValueError(f"logits: tokens side by side, rows one distance apart, expected; got strides {list(logits.stride())} of {list(shape)}")
    if scores.dtype is not torch.float32 or scores.shape != (b, w) or scores.get_device() != dev or not scores.is_contiguous():
        raise ValueError(f"scores: contiguous fp32 [{b}, {w}] on cuda:{dev} expected, got {scores.dtype} {list(scores.shape)} on {scores.device}")
    if finished is not None and (finished.dtype is not torch.bool or finished.shape != (b, w) or finished.get_device() != dev or not finished.is_contiguous()):
        raise ValueError(f"finished: contiguous bool [{b}, {w}] on cuda:{dev} expected, got {finished.dtype} {list(finished.shape)} on {finished.device}")
    if b * w > 65535:
        raise ValueError(f"{b} requests of {w} beams: 65535 rows at most")
    out_scores = scores.new_empty(b, n)
    parents = torch.empty(b, n, dtype=torch.int32, device=logits.device)
    tokens = torch.empty_like(parents)
    if b == 0:
        return out_scores, parents, tokens
    parts, tiles = _parts(b * w, v)
    size = logits.element_size()
    vectors = logits.data_ptr() % 16 == 0 and row * size % 16 == 0 and v * size % 16 == 0
    lists = torch.empty(b * w * parts * (n + 2), dtype=torch.int64, device=logits.device)      # and two doubles a part
    rc = _kernels().b200_beam_select(_SELECT.pack(
        _SELECT.size, b, logits.data_ptr(), row, scores.data_ptr(), _at(finished), lists.data_ptr() + 16 * b * w * parts, lists.data_ptr(),
        out_scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(), _stream(dev), w, v, n, parts, tiles, size == 2, pad_token, vectors, 0, 0))
    _lib.check(rc, "beam_select", 2)
    return out_scores, parents, tokens


@functools.lru_cache(maxsize=256)
def _state(shape: tuple, stride: tuple, size: int, dim: int) -> tuple[int, tuple[int, int, int, int], int]:
    """Checks the sizes of a tensor of states (elements of ``size`` bytes); its slots, bytes from part to part before the axis, from slot to slot and
    of a slot, number of such parts, and the low bits of all three."""
    if not 0 <= dim < len(shape) or min(shape) < 1:
        raise ValueError(f"states: slots along axis {dim} expected, got {list(shape)}")
    inner = 1
    for d in range(len(shape) - 1, dim, -1):
        if shape[d] != 1 and stride[d] != inner:
            raise ValueError(f"states: contiguous behind axis {dim} expected, got strides {list(stride)} of {list(shape)}")
        inner *= shape[d]
    outer, step = 1, 0
    for d in range(dim - 1, -1, -1):
        if shape[d] != 1:
            if outer > 1 and stride[d] != outer * step:
                raise ValueError(f"states: one distance between all parts before axis {dim} expected, got strides {list(stride)} of {list(shape)}")
            step = step if outer > 1 else stride[d]
            outer *= shape[d]
    slots = shape[dim]
    if slots > 1 and stride[dim] < inner or outer > 1 and step < inner:
        raise ValueError(f"states: slots that lie apart expected, got strides {list(stride)} of {list(shape)}")
    step, slot, inner = step * size, stride[dim] * size if slots > 1 else 0, inner * size
    return slots, (step, slot, inner, outer), (step | slot | inner) & 15


def reorder(states, parents: torch.Tensor, slots: torch.Tensor | None = None, dim: int = 0) -> None:
    """In place, for all beams of a request at once: the state of beam w becomes that of beam ``parents[b, w]``.

    ``states``: a tensor or several of any type, their slots along axis ``dim``, everything behind it contiguous ([slots, layers, ..] with dim 0, caches
    [layers, pages, ..] with dim 1), none of them part of another.  parents int32 [B, W], as ``select`` returns them; a beam whose parent is itself, or none (-1), stays as it
    is.  ``slots`` int32 [B, W]: where the beams' states are, all of them different (default: slot b W + w); a beam whose slot is not there is
    neither read nor written.  Other slots stay as they are."""
    dev = parents.get_device()
    if dev < 0 or parents.dim() != 2:
        raise ValueError(f"parents: int32 [requests, beams] on a GPU expected, got {list(parents.shape)} on {parents.device}")
    if _current() != dev:
        with torch.cuda.device(dev):
            return reorder(states, parents, slots, dim)
    b, w = parents.shape
    _index(parents, (b, w), dev, "parents")
    if slots is not None:
        _index(slots, (b, w), dev, "slots")
    if not 0 < w <= MAX_BEAMS:
        raise ValueError(f"{w} beams: 1 to {MAX_BEAMS} expected")
    states = [states] if isinstance(states, torch.Tensor) else states
    packed, n_slots = {}, None
    for x in states:
        n, sizes, low = _state(x.shape, x.stride(), x.element_size(), dim)
        at = x.data_ptr()
        if x.get_device() != dev or n_slots is not None and n != n_slots or at in packed:
            raise ValueError(f"states: different tensors of one number of slots on cuda:{dev} expected, got {list(x.shape)} on {x.device}")
        n_slots = n
        packed[at] = _STATE.pack(at, *sizes, (at | low) & 15 == 0)
    if n_slots is None:
        raise ValueError("states: a tensor or several expected")
    if slots is None and b * w > n_slots:
        raise ValueError(f"{b} requests of {w} beams in {n_slots} slots")
    if b == 0:
        return
    _lib.check_indices(slots, -2 ** 31, n_slots, 4)         # (a bad slot becomes a negative one)
    packed = list(packed.values())
    for i in range(0, len(packed), MAX_STATES):
        some = packed[i:i + MAX_STATES]
        call = _REORDER.pack(_REORDER_BYTES, b, parents.data_ptr(), _at(slots), _status(dev), _stream(dev), w, n_slots, len(some), 0)
        _lib.check(_kernels().b200_beam_reorder(call + b"".join(some) + _REST[len(some)]), "beam_reorder")
