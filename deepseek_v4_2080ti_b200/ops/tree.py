"""Trees of drafted tokens (csrc/kernels/tree.cu): what their rows need before the target's pass, and what is kept of them after it.

Sequence b's tree is the rows ``q_start[b] .. q_start[b] + q_len[b] - 1`` of a step's batch, node 0 first: the token that the target chose
last, then the drafts.  ``parents[t]`` is the node of its own tree that row t continues, before it in the order; -1: the context.

    positions, mask = tree.layout(parents, q_start, q_len, kv_len, max_nodes)       # once a step, before the layers
    ... attention.decode_tree(q, .., mask, q_start, q_len, kv_len, ..) in every layer, keys and values of node i appended at kv_len - q_len + i
    path, count, emitted = tree.accept(tokens, parents, predicted, q_start, q_len, max_path, kv_len, block_table, [k_cache, v_cache])

``predicted[t]``: the token that the target puts behind row t, its best one or one drawn by ``sampling.sample`` - either way the tokens that
come out are distributed as without drafts.  The context grows by ``count``: kv_len - q_len + count keys are valid after it."""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import _lib
from .attention import MAX_TREE, _at, _current, _index, _stream

MAX_PATH = 256                           # longest path that is kept
MAX_CACHES = 16
# TreeLayoutCall, AcceptCall and AcceptCache in ops.h, packed
_LAYOUT, _CALL, _CACHE = struct.Struct("@ii7Pii"), struct.Struct("@ii10PP6i"), struct.Struct("@Pqiiii")
_CALL_BYTES = _CALL.size + MAX_CACHES * _CACHE.size
_REST = [b"\0" * ((MAX_CACHES - i) * _CACHE.size) for i in range(MAX_CACHES + 1)]
_typed = False


def _kernels() -> ctypes.CDLL:
    global _typed
    lib = _lib.lib()
    if not _typed:
        for f in (lib.b200_tree_layout, lib.b200_tree_accept):
            f.argtypes = [ctypes.c_char_p]
        _typed = True
    return lib


def layout(parents: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor, kv_len: torch.Tensor, max_nodes: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``positions`` int32 [T] - the context's length and the row's depth in its tree - and ``mask`` int32 [T, words] of the node itself and
    those that it continues, for ``attention.decode_tree``.  parents int32 [T], q_start / q_len / kv_len (the tree's rows among the keys) int32
    [B]; ``max_nodes`` (host) is at least the longest of ``q_len``.  A parent that does not lie before its child counts as the context.
    Rows of no sequence: position 0 and an empty mask."""
    dev = parents.get_device()
    if dev < 0 or parents.dim() != 1:
        raise ValueError(f"parents: int32 [T] on a GPU expected, got {list(parents.shape)} on {parents.device}")
    if _current() != dev:
        with torch.cuda.device(dev):
            return layout(parents, q_start, q_len, kv_len, max_nodes)
    t, b = parents.shape[0], q_len.shape[0] if q_len.dim() == 1 else -1
    _index(parents, (t,), dev, "parents")
    _index(q_start, (b,), dev, "q_start")
    _index(q_len, (b,), dev, "q_len")
    _index(kv_len, (b,), dev, "kv_len")
    if not 1 <= max_nodes <= MAX_TREE:
        raise ValueError(f"trees of {max_nodes} nodes: 1 to {MAX_TREE} expected")
    words = (int(max_nodes) + 31) // 32
    positions, mask = parents.new_empty(t), parents.new_empty(t, words)
    if t:
        rc = _kernels().b200_tree_layout(_LAYOUT.pack(
            _LAYOUT.size, b, parents.data_ptr(), q_start.data_ptr(), q_len.data_ptr(), kv_len.data_ptr(), positions.data_ptr(), mask.data_ptr(), _stream(dev),
            t, words))
        _lib.check(rc, "tree_layout")
    return positions, mask


@functools.lru_cache(maxsize=256)
def _cache(shape: tuple, stride: tuple, size: int) -> tuple[int, int, int, int, int, int, int]:
    """Checks a cache's sizes (elements of ``size`` bytes); layers, pages, heads, page size, bytes of a row, of a layer, and the low bits of both."""
    if len(shape) < 4 or min(shape, default=0) < 1:
        raise ValueError(f"caches: [layers, pages, heads, page size, ..] expected, got {list(shape)}")
    layers, nb, heads, bs = shape[:4]
    inner = 1
    for d in range(len(shape) - 1, 0, -1):
        if stride[d] != inner and shape[d] != 1:
            raise ValueError(f"caches: contiguous layers expected, got strides {list(stride)} of {list(shape)}")
        inner *= shape[d]
    if layers > 1 and stride[0] < inner:
        raise ValueError(f"caches: layers that lie apart expected, got strides {list(stride)} of {list(shape)}")
    row, step = inner // (nb * heads * bs) * size, stride[0] * size if layers > 1 else 0
    return layers, nb, heads, bs, row, step, (row | step) & 15


def _caches(caches, dev: int):
    """Checks the caches; (pages, page size, packed)."""
    if not 0 < len(caches) <= MAX_CACHES:
        raise ValueError(f"{len(caches)} caches: 1 to {MAX_CACHES} expected")
    if len({c.data_ptr() for c in caches}) < len(caches):
        raise ValueError("caches: a tensor that is there twice would move twice")
    pages = None
    packed = []
    for c in caches:
        layers, nb, heads, bs, row, step, low = _cache(c.shape, c.stride(), c.element_size())
        at = c.data_ptr()
        if c.get_device() != dev or pages is not None and pages != (nb, bs):
            raise ValueError(f"caches: on cuda:{dev}, of as many pages and rows of them each, expected; got {list(c.shape)} on {c.device}")
        pages = nb, bs
        low |= at & 15
        if low & 3:
            raise ValueError(f"caches: rows of a multiple of 4 bytes on 4-byte boundaries expected, got {row} bytes")
        packed.append(_CACHE.pack(at, step, layers, heads, row, 4 if low else 16))
    return nb, bs, b"".join(packed)


def _check_pages(path, q_len, kv_len, block_table, nb: int, bs: int) -> None:
    """Debug mode: reports pages that are not there, or keys behind the table, where a row of a path lies or would go.  Nothing is replaced."""
    if not _lib.bounds_checks_on():
        return
    b, most = path.shape
    to = torch.arange(most, device=path.device)
    first = (kv_len.long() - q_len)[:, None]
    moves = (path > to) & (first >= 0)
    keys = torch.stack([first + path, first + to.expand(b, most)], -1)         # [B, max_path, from and to]
    pages = block_table.long().gather(1, (keys // bs).clamp(0, block_table.shape[1] - 1).view(b, -1)).view(keys.shape)
    pages = torch.where(keys < block_table.shape[1] * bs, pages, -1)
    _lib.check_indices(torch.where(moves[..., None], pages, 0).to(torch.int32), 0, nb, 8)


def accept(tokens, parents, predicted, q_start, q_len, max_path: int, kv_len=None, block_table=None, caches=()):
    """The path that the target agrees with: from node 0 to the child whose token is the one predicted at its parent (of several the first),
    as long as there is one, ``max_path`` nodes at most.  tokens / parents / predicted int32 [T], q_start / q_len int32 [B]; negative tokens and
    predictions agree with nothing, nor do nodes behind the first 1024.

    Returns ``path`` int32 [B, max_path] (nodes, node 0 first), ``count`` int32 [B] and ``emitted`` int32 [B, max_path]: the tokens that the target puts
    behind the path's nodes - the drafts it agrees with, then one of its own; -1 behind ``count``.  A sequence of no rows has a count of 0.

    ``caches``: a list of tensors [layers, pages, heads, page size, ..] of any type, rows of a multiple of 4 bytes, layers contiguous (a single layer:
    ``cache[None]``; keys, values, scales of quantised rows); with them kv_len [B] and block_table int32 [B, pages], as in
    ``attention.decode_tree``.  The path's rows move in place from kv_len - q_len + path[i] to kv_len - q_len + i; rows in pages outside the
    cache stay where they are, which the debug mode reports.  No cache is part of another, and no two sequences have the page of a row that moves."""
    dev = tokens.get_device()
    if dev < 0 or tokens.dim() != 1:
        raise ValueError(f"tokens: int32 [T] on a GPU expected, got {list(tokens.shape)} on {tokens.device}")
    if _current() != dev:
        with torch.cuda.device(dev):
            return accept(tokens, parents, predicted, q_start, q_len, max_path, kv_len, block_table, caches)
    t, b = tokens.shape[0], q_len.shape[0] if q_len.dim() == 1 else -1
    _index(tokens, (t,), dev, "tokens")
    _index(parents, (t,), dev, "parents")
    _index(predicted, (t,), dev, "predicted")
    _index(q_start, (b,), dev, "q_start")
    _index(q_len, (b,), dev, "q_len")
    if not 1 <= max_path <= MAX_PATH or b > 65535:
        raise ValueError(f"{b} paths of {max_path} nodes: 65535 at most, of 1 to {MAX_PATH} nodes")
    if isinstance(caches, torch.Tensor):                     # (its layers would be taken for caches, their pages for layers)
        raise ValueError(f"caches: a list of tensors expected, got one of {list(caches.shape)}")
    caches = list(caches)
    nb, bs, width, packed = 0, 0, 0, b""
    if caches:
        nb, bs, packed = _caches(caches, dev)
        if kv_len is None or block_table is None or block_table.dim() != 2 or block_table.shape[1] < 1:
            raise ValueError("caches come with kv_len [B] and block_table [B, pages]")
        width = block_table.shape[1]
        _index(kv_len, (b,), dev, "kv_len")
        _index(block_table, (b, width), dev, "block_table")
    path, emitted, count = tokens.new_empty(b, max_path), tokens.new_empty(b, max_path), tokens.new_empty(b)
    if b:
        call = _CALL.pack(_CALL_BYTES, b, tokens.data_ptr(), parents.data_ptr(), predicted.data_ptr(), q_start.data_ptr(), q_len.data_ptr(), _at(kv_len),
                          _at(block_table), path.data_ptr(), count.data_ptr(), emitted.data_ptr(), _stream(dev), t, int(max_path), width, nb, bs, len(caches))
        _lib.check(_kernels().b200_tree_accept(call + packed + _REST[len(caches)]), "tree_accept")
        if caches:
            _check_pages(path, q_len, kv_len, block_table, nb, bs)
    return path, count, emitted
