"""GQA attention over a paged KV cache (head_dim 128): fused q/k norm + partial RoPE + cache
append, tcgen05 flash prefill, split-context decode.  Cache layout:
``[num_blocks, kv_heads, block_size, 128]`` bf16, zero-initialised.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct

import torch

from . import _lib

_f = ctypes.c_float
D = 128


def rope_inv_freq(rot: int, theta: float, device) -> torch.Tensor:
    return (1.0 / (theta ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))).float().to(device)


def qk_norm_rope_append(q_src, q_off, q_head_stride, gate_in_q, k_src, k_off, v_src, v_off, q_gamma, k_gamma,
                        unit_offset, eps, inv_freq, rot, positions, slots, k_cache, v_cache, n_q_heads, n_kv_heads,
                        mscale: float = 1.0):
    """Normalise + rotate q and k, split the q||gate layout, and write K/V rows into the paged cache.

    ``*_src`` are 2-D bf16 tensors (often the same fused-projection output) addressed as
    ``src[t, off + head * stride + d]``. Returns (q [T, Hq, 128], gate [T, Hq, 128] or None).
    """
    t = q_src.shape[0]
    bs = k_cache.shape[2]
    _lib.check_indices(slots, 0, k_cache.shape[0] * bs, 2)
    q_out = torch.empty(t, n_q_heads, D, dtype=torch.bfloat16, device=q_src.device)
    gate_out = torch.empty_like(q_out) if gate_in_q else None
    rc = _lib.lib().b200_qk_norm_rope_append(
        _lib.ptr(q_src), q_src.stride(0), q_off, q_head_stride, int(gate_in_q),
        _lib.ptr(k_src), k_src.stride(0), k_off, _lib.ptr(v_src), v_src.stride(0), v_off,
        _lib.ptr(q_gamma), _lib.ptr(k_gamma), int(unit_offset), _f(eps), _lib.ptr(inv_freq), rot, _f(mscale),
        _lib.ptr(positions), _lib.ptr(slots), _lib.ptr(q_out), _lib.ptr(gate_out), _lib.ptr(k_cache),
        _lib.ptr(v_cache), bs, t, n_q_heads, n_kv_heads, _lib.stream())
    _lib.check(rc, "qk_norm_rope_append")
    return q_out, gate_out


def qk_sumsq(proj: torch.Tensor, q_off: int, q_width: int, k_off: int, k_width: int) -> torch.Tensor:
    """fp32 [T, 2]: sums of squares of the q and k column ranges of each projection row."""
    t = proj.shape[0]
    out = torch.empty(t, 2, dtype=torch.float32, device=proj.device)
    rc = _lib.lib().b200_qk_sumsq(_lib.ptr(proj), proj.stride(0), q_off, q_width, k_off, k_width, _lib.ptr(out), t, _lib.stream())
    _lib.check(rc, "qk_sumsq")
    return out


def qk_fullnorm_rope_append(proj, q_off, k_off, v_off, q_gamma, k_gamma, row_ss, q_full_width, k_full_width, eps, inv_freq,
                            rot, positions, slots, k_cache, v_cache, n_q_heads, n_kv_heads):
    """MiniMax-style attention prologue: RMSNorm whose statistic spans the whole q / k projection row (``row_ss`` holds
    the rows' sums of squares over all ranks), per-(head, dim) gamma, half-split partial RoPE, paged K/V append."""
    t = proj.shape[0]
    bs = k_cache.shape[2]
    q_out = torch.empty(t, n_q_heads, D, dtype=torch.bfloat16, device=proj.device)
    rc = _lib.lib().b200_qk_fullnorm_rope_append(
        _lib.ptr(proj), proj.stride(0), q_off, _lib.ptr(proj), proj.stride(0), k_off, _lib.ptr(proj), proj.stride(0), v_off,
        _lib.ptr(q_gamma), _lib.ptr(k_gamma), _lib.ptr(row_ss), q_full_width, k_full_width, _f(eps), _lib.ptr(inv_freq), rot,
        _lib.ptr(positions), _lib.ptr(slots), _lib.ptr(q_out), _lib.ptr(k_cache), _lib.ptr(v_cache), bs, t, n_q_heads,
        n_kv_heads, _lib.stream())
    _lib.check(rc, "qk_fullnorm_rope_append")
    return q_out


def prefill(q, k_cache, v_cache, block_table, q_start, q_len, kv_len, max_q_len, gate=None, scale=None, window: int = 0,
            sinks: int = 0):
    """Causal attention of new query rows against the paged cache (which already holds their K/V).

    q: [T, Hq, 128]; block_table [B, max_blocks] int32; q_start/q_len/kv_len [B] int32 device tensors.
    """
    t, hq, d = q.shape
    assert d == D
    nb, hkv, bs, _ = k_cache.shape
    _lib.check_indices(block_table, 0, nb, 3)
    out = torch.empty_like(q)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    rc = _lib.lib().b200_gqa_prefill_ex(
        _lib.ptr(q), _lib.ptr(k_cache), _lib.ptr(v_cache), _lib.ptr(out), _lib.ptr(gate), _lib.ptr(block_table),
        _lib.ptr(q_start), _lib.ptr(q_len), _lib.ptr(kv_len), block_table.shape[0], int(max_q_len), t,
        block_table.shape[1], nb, bs, hq, hkv, _f(scale), int(window), int(sinks), _lib.ptr(_lib.status_word(q.device)),
        _lib.stream())
    _lib.check(rc, "gqa_prefill")
    return out


_dec_ws: dict[int, torch.Tensor] = {}
_outgrown: list[torch.Tensor] = []      # smaller workspaces stay alive: captured graphs hold their addresses


def decode(q, k_cache, v_cache, block_table, kv_len, gate=None, scale=None, splits: int | None = None,
           max_kv_len: int | None = None, window: int = 0, sinks: int = 0):
    """One query row per sequence. q: [B, Hq, 128].  ``window`` > 0: only the first ``sinks`` and the last ``window``
    keys of each sequence are visible (sliding window with attention sinks)."""
    b, hq, d = q.shape
    nb, hkv, bs, _ = k_cache.shape
    _lib.check_indices(block_table, 0, nb, 3)
    out = torch.empty_like(q)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if splits is None:
        ctx = max_kv_len if max_kv_len is not None else block_table.shape[1] * bs
        splits = max(1, min(64, (2 * 148) // max(1, b * hkv), (ctx + 255) // 256))
    ws = None
    if splits > 1:
        need = b * hq * splits * (D + 2)
        dev = q.device.index or 0
        ws = _dec_ws.get(dev)
        if ws is None or ws.numel() < need:
            if ws is not None:
                _outgrown.append(ws)
            ws = torch.empty(max(need, 1 << 20), dtype=torch.float32, device=q.device)
            _dec_ws[dev] = ws
    rc = _lib.lib().b200_gqa_decode_ex(_lib.ptr(q), _lib.ptr(k_cache), _lib.ptr(v_cache), _lib.ptr(out), _lib.ptr(gate),
                                       _lib.ptr(block_table), _lib.ptr(kv_len), _lib.ptr(ws), b, block_table.shape[1],
                                       bs, hq, hkv, splits, _f(scale), int(window), int(sinks), _lib.stream())
    _lib.check(rc, "gqa_decode", 2 if splits > 1 else 1)
    return out


# ---------------------------------------------------------------- quantised KV cache
KV8_FORMATS = {"fp8": 1, "int8_per_token_head": 2, "turboquant_k8v4": 3}


class Kv8Cache:
    """Quantised paged cache of one attention layer set: ``fmt`` "fp8" = E4M3 keys and values, "int8_per_token_head" =
    INT8, "turboquant_k8v4" = E4M3 keys + 4-bit affine values.  ``k`` uint8 [L, num_blocks, Hkv, bs, 128], ``v`` the
    same (64 bytes per row for 4-bit values), one fp32 scale per (block, head, row) in ``k_scale`` / ``v_scale``
    [L, num_blocks, Hkv, bs] and, for 4-bit values, the row minimum in ``v_min``.  Rows reach it through a bf16
    staging cache (the fused norm + RoPE kernel writes there) and ``kv8_quantize``."""

    def __init__(self, fmt: str, layers: int, num_blocks: int, hkv: int, block_size: int, device):
        self.fmt = KV8_FORMATS[fmt]
        self.k = torch.zeros(layers, num_blocks, hkv, block_size, D, dtype=torch.uint8, device=device)
        self.v = torch.zeros(layers, num_blocks, hkv, block_size, D // 2 if self.fmt == 3 else D, dtype=torch.uint8,
                             device=device)
        self.k_scale = torch.zeros(layers, num_blocks, hkv, block_size, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)
        self.v_min = torch.zeros_like(self.k_scale) if self.fmt == 3 else None

    def layer(self, idx: int):
        """(k, v, k_scale, v_scale, v_min) views of one layer."""
        return self.k[idx], self.v[idx], self.k_scale[idx], self.v_scale[idx], None if self.v_min is None else self.v_min[idx]

    def nbytes(self) -> int:
        return self.k.numel() + self.v.numel() + 4 * self.k_scale.numel() * (3 if self.fmt == 3 else 2)


def kv8_quantize(fmt: int, stage_k, stage_v, src_slots, dst_slots, k8, v8, k_scale, v_scale, v_min=None):
    """Quantise staged rows ``src_slots`` (bf16 [nb_s, Hkv, bs_s, 128]) into rows ``dst_slots`` of the cache."""
    rc = _lib.lib().b200_kv8_quantize(_lib.ptr(stage_k), _lib.ptr(stage_v), _lib.ptr(src_slots), _lib.ptr(dst_slots),
                                      _lib.ptr(k8), _lib.ptr(v8), _lib.ptr(k_scale), _lib.ptr(v_scale), _lib.ptr(v_min),
                                      stage_k.shape[2], k8.shape[2], src_slots.numel(), k8.shape[1], int(fmt), _lib.stream())
    _lib.check(rc, "kv8_quantize")


def kv8_dequantize(fmt: int, k8, v8, k_scale, v_scale, block_table_row, n_tokens: int, stage_k, stage_v, v_min=None):
    """Dequantise the first ``n_tokens`` positions of one sequence into the staging caches (blocks 0, 1, 2, ...)."""
    if n_tokens <= 0:
        return
    assert stage_k.shape[2] == k8.shape[2] and stage_k.shape[0] * stage_k.shape[2] >= n_tokens
    rc = _lib.lib().b200_kv8_dequantize(_lib.ptr(k8), _lib.ptr(v8), _lib.ptr(k_scale), _lib.ptr(v_scale), _lib.ptr(v_min),
                                        _lib.ptr(block_table_row), _lib.ptr(stage_k), _lib.ptr(stage_v), k8.shape[2],
                                        int(n_tokens), k8.shape[1], int(fmt), _lib.stream())
    _lib.check(rc, "kv8_dequantize")


def decode_kv8(fmt: int, q, k8, v8, k_scale, v_scale, block_table, kv_len, gate=None, scale=None, splits: int | None = None,
               max_kv_len: int | None = None, window: int = 0, sinks: int = 0, v_min=None):
    """``decode`` over a quantised cache; rows are dequantised in registers."""
    b, hq, d = q.shape
    nb, hkv, bs, _ = k8.shape
    out = torch.empty_like(q)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if splits is None:
        ctx = max_kv_len if max_kv_len is not None else block_table.shape[1] * bs
        splits = max(1, min(64, (2 * 148) // max(1, b * hkv), (ctx + 255) // 256))
    ws = None
    if splits > 1:
        need = b * hq * splits * (D + 2)
        dev = q.device.index or 0
        ws = _dec_ws.get(dev)
        if ws is None or ws.numel() < need:
            if ws is not None:
                _outgrown.append(ws)
            ws = torch.empty(max(need, 1 << 20), dtype=torch.float32, device=q.device)
            _dec_ws[dev] = ws
    rc = _lib.lib().b200_gqa_decode_kv8(int(fmt), _lib.ptr(q), _lib.ptr(k8), _lib.ptr(v8), _lib.ptr(k_scale),
                                        _lib.ptr(v_scale), _lib.ptr(v_min), _lib.ptr(out), _lib.ptr(gate), _lib.ptr(block_table),
                                        _lib.ptr(kv_len), _lib.ptr(ws), b, block_table.shape[1], bs, hq, hkv, splits,
                                        _f(scale), int(window), int(sinks), _lib.stream())
    _lib.check(rc, "gqa_decode_kv8", 2 if splits > 1 else 1)
    return out


# ---------------------------------------------------------------- several rotary axes, spans of keys, shared pages
NUM_SMS = 148
SCALE = 1.0 / math.sqrt(D)
ROW_TILE, KEY_TILE = 256, 128            # (token, head) rows and keys of a tile in attn_spans.cu
MAX_TREE = 1024                          # nodes of a drafted tree


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


_I32, _BF16, _F32 = torch.int32, torch.bfloat16, torch.float32


def _index(t, shape, dev: int, what: str) -> None:
    if t.dtype is not _I32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous int32 {list(shape)} on cuda:{dev} expected, got {t.dtype} {list(t.shape)} on {t.device}")


def _like(t, shape, dev: int, what: str) -> None:
    if t.dtype is not _BF16 or t.shape != shape or t.get_device() != dev or not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{what}: contiguous bf16 {list(shape)} on cuda:{dev}, 16-byte aligned, expected; got {t.dtype} {list(t.shape)} on {t.device}")


def _caches(k_cache, v_cache, dev: int):
    """Shape of a pair of caches."""
    shape = k_cache.shape
    if len(shape) != 4 or shape[3] != D or k_cache.dtype is not _BF16 or k_cache.get_device() != dev or not k_cache.is_contiguous() or k_cache.data_ptr() % 16:
        raise ValueError("caches: contiguous bf16 [pages, kv heads, page size, 128] on the device of the rows, 16-byte aligned, expected")
    _like(v_cache, shape, dev, "v_cache")
    return shape


_LEAST, _MOST = 2.0 ** -100, 2.0 ** 100


def _scores(scale, cap) -> float:
    """Checks scale and cap; the scale.  The kernels hold both and scale / cap in 32 bits: a cap that became zero there would be none, and
    scores times an infinite factor NaN."""
    scale = SCALE if scale is None else float(scale)
    if not _LEAST <= scale <= _MOST or cap and not (_LEAST <= cap <= _MOST and _LEAST <= scale / cap <= _MOST):
        raise ValueError(f"scale {scale}, cap {cap}: a positive scale and a cap that is positive, or 0 for none, both and their ratio "
                         f"between 2^-100 and 2^100, expected")
    return scale


def _paged(q, k_cache, v_cache, block_table, kv_len, gate, out, scale, cap):
    """Checks what the calls over spans have in common; (device, rows, Hq, pages, Hkv, page size, sequences, table width, scale, out)."""
    dev, rows = q.get_device(), q.shape
    if dev < 0 or len(rows) != 3 or rows[2] != D or q.dtype is not _BF16 or not q.is_contiguous() or q.data_ptr() % 16:
        raise ValueError(f"q: contiguous bf16 [T, Hq, 128] on a GPU, 16-byte aligned, expected; got {q.dtype} {list(rows)} on {q.device}")
    t, hq, _ = rows
    nb, hkv, bs, _ = _caches(k_cache, v_cache, dev)
    if nb < 1 or hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError(f"{hq} query heads over {hkv} key/value heads in {nb} pages")
    if bs not in (16, 32, 64, 128, 256):
        raise ValueError(f"page size {bs}: 16, 32, 64, 128 or 256 expected")
    table = block_table.shape
    if len(table) != 2 or table[1] < 1:
        raise ValueError("block_table: int32 [sequences, pages] expected")
    b, width = table
    _index(block_table, table, dev, "block_table")
    _index(kv_len, (b,), dev, "kv_len")
    if gate is not None:
        _like(gate, rows, dev, "gate")
    if out is None:
        out = torch.empty_like(q)
    else:
        _like(out, rows, dev, "out")
    return dev, t, hq, nb, hkv, bs, b, width, _scores(scale, cap), out


# The kernels' arguments as one block each (AxesAppendCall and SpansCall in ops.h), packed: a third of what 33 arguments cost one by one.
_AXES_CALL, _SPANS_CALL = struct.Struct("@ii13P16iff64s"), struct.Struct("@ii17P11iff0P")
_typed = False


def _kernels() -> ctypes.CDLL:
    """The kernel library with the parameter types of the calls below, which take a block."""
    global _typed
    lib = _lib.lib()
    if not _typed:
        for f in (lib.b200_qk_norm_rope_axes_append, lib.b200_attn_spans, lib.b200_attn_shared, lib.b200_attn_own_rows, lib.b200_attn_tree):
            f.argtypes = [ctypes.c_char_p]
        _typed = True
    return lib


def _rows(x, t: int, dev: int, what: str) -> int:
    """Checks a tensor of rows; their distance."""
    shape, (ld, one) = x.shape, x.stride() if x.dim() == 2 else (0, 0)
    if one != 1 or shape[0] != t or ld % 4 or x.dtype is not _BF16 or x.get_device() != dev or x.data_ptr() % 8:
        raise ValueError(f"{what}: bf16 rows [{t}, ..] on cuda:{dev}, 8-byte aligned, expected; got {x.dtype} {list(shape)} on {x.device}")
    return ld


def _at(t):
    return 0 if t is None else t.data_ptr()


# (looked up at the call: a torch without CUDA has neither, and the oracles below serve the host runtime)
def _current() -> int:
    return torch._C._cuda_getDevice()


def _stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


def _status(dev: int) -> int:
    t = _lib._status.get(dev)
    return (_lib.status_word(dev) if t is None else t).data_ptr()


class PairAxes(tuple):
    """Axis of every rotary pair, with the table that the kernel takes (laid out once: 1.2 us a call for 64 pairs otherwise)."""

    def __new__(cls, axes):
        self = super().__new__(cls, axes)
        self.table = bytes(self)                            # (axes outside 0 .. 255: ValueError)
        self.n_axes = max(self.table, default=0) + 1
        return self


@functools.lru_cache(maxsize=64)
def _pair_axes(sections: tuple, interleaved: bool) -> PairAxes:
    _need(sections and min(sections) >= 0 and 0 < sum(sections) <= D // 2, f"sections {sections}: 1 to {D // 2} pairs in all expected")
    if not interleaved:
        return PairAxes(a for a, n in enumerate(sections) for _ in range(n))
    axes = [0] * sum(sections)
    for a, n in enumerate(sections[1:], 1):
        _need(n == 0 or a + len(sections) * (n - 1) < len(axes), f"sections {sections}: axis {a} is too long to take turns")
        axes[a:a + len(sections) * n:len(sections)] = [a] * n
    return PairAxes(axes)


def rotary_axes(sections, interleaved: bool = False) -> PairAxes:
    """Axis of every rotary pair from the number of pairs of each axis: one block per axis, or - ``interleaved`` - the axes in
    turn (T H W T H W ..), where pairs that no other axis claims stay on the first."""
    return _pair_axes(tuple(int(n) for n in sections), bool(interleaved))


def qk_norm_rope_axes_append(q_src, q_off, q_head_stride, gate_in_q, k_src, k_off, v_src, v_off, q_gamma, k_gamma,
                             unit_offset, eps, inv_freq, axes, positions, slots, k_cache, v_cache, n_q_heads, n_kv_heads,
                             mscale: float = 1.0):
    """``qk_norm_rope_append`` with rotary positions of several axes: pair i turns by ``positions[axes[i], t] * inv_freq[i]``.

    ``axes`` from ``rotary_axes`` (a multiple of 4 pairs); ``positions`` int32 [axes, T]; ``slots`` int32 [T], distinct; rows
    with a negative slot are not cached.  Returns (q [T, Hq, 128], gate [T, Hq, 128] or None).
    """
    dev = q_src.get_device()
    if dev < 0:
        raise ValueError(f"q_src: rows on a GPU expected, got {q_src.device}")
    if _current() != dev:
        with torch.cuda.device(dev):
            return qk_norm_rope_axes_append(q_src, q_off, q_head_stride, gate_in_q, k_src, k_off, v_src, v_off, q_gamma, k_gamma, unit_offset, eps,
                                            inv_freq, axes, positions, slots, k_cache, v_cache, n_q_heads, n_kv_heads, mscale)
    t = q_src.shape[0]
    ldq = _rows(q_src, t, dev, "q_src")
    ldk = ldq if k_src is q_src else _rows(k_src, t, dev, "k_src")
    ldv = ldq if v_src is q_src else _rows(v_src, t, dev, "v_src")
    kv = n_kv_heads * D
    if (q_off % 4 or k_off % 4 or v_off % 4 or q_head_stride % 4 or min(q_off, k_off, v_off, q_head_stride) < 0 or n_q_heads < 1 or n_kv_heads < 1 or
            q_off + (n_q_heads - 1) * q_head_stride + (2 * D if gate_in_q else D) > q_src.shape[1] or k_off + kv > k_src.shape[1] or
            v_off + kv > v_src.shape[1]):
        raise ValueError(f"{n_q_heads} / {n_kv_heads} heads from columns {q_off} (every {q_head_stride}), {k_off}, {v_off}: multiples of 4 inside the rows expected")
    nb, hkv, bs, _ = _caches(k_cache, v_cache, dev)
    if hkv != n_kv_heads:
        raise ValueError(f"caches of {hkv} heads, {n_kv_heads} in the rows")
    for g in (q_gamma, k_gamma):
        if g is not None and (g.dtype is not _BF16 or g.numel() != D or not g.is_contiguous() or g.get_device() != dev or g.data_ptr() % 8):
            raise ValueError("gammas: bf16 [128] on the device of the rows, 8-byte aligned, expected")
    if type(axes) is not PairAxes:
        axes = PairAxes(axes)
    n, n_axes = len(axes), positions.shape[0]
    if n % 4 or not 0 < n <= D // 2 or n_axes < axes.n_axes:
        raise ValueError(f"axes: 4, 8 .. {D // 2} pairs, each with a row of positions, expected")
    if inv_freq.dtype is not _F32 or inv_freq.numel() != n or not inv_freq.is_contiguous() or inv_freq.get_device() != dev:
        raise ValueError("inv_freq: fp32, one per pair, on the device of the rows expected")
    _index(positions, (n_axes, t), dev, "positions")
    _index(slots, (t,), dev, "slots")
    q_out = q_src.new_empty(t, n_q_heads, D)
    gate_out = torch.empty_like(q_out) if gate_in_q else None
    if t == 0:
        return q_out, gate_out
    _lib.check_indices(slots, -2 ** 31, nb * bs, 2)         # (a bad slot becomes a negative one)
    rc = _kernels().b200_qk_norm_rope_axes_append(_AXES_CALL.pack(
        _AXES_CALL.size, t, q_src.data_ptr(), k_src.data_ptr(), v_src.data_ptr(), _at(q_gamma), _at(k_gamma), inv_freq.data_ptr(), positions.data_ptr(),
        slots.data_ptr(), q_out.data_ptr(), _at(gate_out), k_cache.data_ptr(), v_cache.data_ptr(), _stream(dev), ldq, q_off, q_head_stride, gate_in_q,
        ldk, k_off, ldv, v_off, unit_offset, 2 * n, n_axes, t, nb, bs, n_q_heads, n_kv_heads, eps, mscale, axes.table))
    _lib.check(rc, "qk_norm_rope_axes_append")
    return q_out, gate_out


def visible_spans(kv_len: int, documents=None, blocks=(), window: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """``lo``, ``hi`` int32 [kv_len] (host) of the positions of one sequence: causal within each of ``documents`` (lengths that add
    up to ``kv_len``), not further back than ``window`` keys, and inside a block ``(first, end)`` - an image, a prefix - up to
    the block's end (the furthest of them, where blocks overlap).  A block lies in one document."""
    pos = torch.arange(kv_len)
    lo, hi = torch.zeros_like(pos), pos + 1
    if documents is not None:
        lengths = torch.as_tensor(documents, dtype=torch.long).reshape(-1)
        _need(int(lengths.sum()) == kv_len and bool((lengths >= 0).all()), f"documents of {int(lengths.sum())} tokens in a context of {kv_len}")
        ends = torch.repeat_interleave(lengths.cumsum(0), lengths)
        lo = torch.repeat_interleave(lengths.cumsum(0) - lengths, lengths)
    if window > 0:
        lo = torch.maximum(lo, pos + 1 - window)
    for first, end in blocks:
        _need(0 <= first <= end <= kv_len, f"block ({first}, {end}) in a context of {kv_len}")
        _need(documents is None or first == end or end <= int(ends[first]), f"block ({first}, {end}) reaches into another document")
        hi[first:end].clamp_(min=end)
    return lo.to(torch.int32), hi.to(torch.int32)


def _seen_pages(t, width, bs, kv_len, q_start, q_len, lo, hi):
    """bool [B, width]: pages with a key that some row of the sequence sees (arguments as in ``prefill_spans``)."""
    row = torch.arange(t, device=kv_len.device)
    kv, first, n = (x.long()[:, None] for x in (kv_len, q_start, q_len))
    begin = torch.zeros_like(row) if lo is None else lo.long().clamp(min=0)
    end = torch.minimum(row - first + kv - n + 1 if hi is None else hi.long(), kv.clamp(max=width * bs))
    seen = ((first >= 0) & (row >= first) & (row < first + n) & (begin < end)).long()        # [B, T]
    edge = torch.zeros(kv.shape[0], width + 1, dtype=torch.long, device=row.device)
    edge.scatter_add_(1, (begin // bs).clamp(max=width).expand_as(seen), seen)
    edge.scatter_add_(1, ((end - 1) // bs + 1).clamp(0, width), -seen)
    return edge[:, :width].cumsum(1) > 0


def _check_pages(block_table, nb, bs, kv_len, rows=None) -> None:
    """Debug mode: -1 stands for a page that is not there, which only keys that no row sees may lie in.  ``rows``: T, q_start, q_len, lo, hi
    of prompt rows, else every key of a sequence is seen."""
    if not _lib.bounds_checks_on():
        return
    width = block_table.shape[1]
    if rows is None:
        seen = torch.arange(width, device=kv_len.device) * bs < kv_len[:, None]
    else:
        t, q_start, q_len, lo, hi = rows
        seen = _seen_pages(t, width, bs, kv_len, q_start, q_len, lo, hi)
    block_table.masked_fill_(seen & (block_table == -1), -2)
    _lib.check_indices(block_table, 0, nb, 3, keep=-1)


def _row_splits(b: int, t: int, g: int, hkv: int, max_q_len: int, max_kv_len: int) -> int:
    """Items that the keys of a row tile are cut into: as many as there are SMs for, of two key tiles at least."""
    tiles = hkv * min(b * -(-max_q_len * g // ROW_TILE), t * g // ROW_TILE + b)
    return max(1, min(NUM_SMS // tiles, -(-max_kv_len // KEY_TILE) // 2))


def prefill_spans(q, k_cache, v_cache, block_table, q_start, q_len, kv_len, max_q_len, lo=None, hi=None, gate=None, scale=None,
                  cap: float = 0.0, max_kv_len: int | None = None, splits: int | None = None, out=None):
    """Attention of new rows against the paged cache (which already holds their keys and values), every row over a span of keys
    of its own: row t sees ``lo[t] <= j < min(hi[t], kv_len)`` of its sequence - documents in one context, blocks that see each
    other, prefixes, windows (``visible_spans``).  Without ``lo`` the span begins at 0, without ``hi`` it is causal.
    ``cap`` > 0: a score s becomes cap tanh(s / cap).  A row that sees nothing is 0; a key outside a row's span has no part in
    it, whatever the cache holds there.

    q: [T, Hq, 128]; block_table [B, max_blocks], q_start / q_len / kv_len [B], lo / hi [T]: int32 device tensors.  Rows of no
    sequence are not written (``out``: where to write, ``q`` itself if it is not needed any more).  Entries of ``block_table`` for
    pages that no row sees are not followed; a page outside the cache that a row does see reads as keys and values of zero.
    ``max_q_len`` (host) is at least the longest of ``q_len``; ``max_kv_len`` bounds the contexts, for the choice of ``splits`` (items
    a row's keys are cut into).
    """
    dev, t, hq, nb, hkv, bs, b, width, scale, out = _paged(q, k_cache, v_cache, block_table, kv_len, gate, out, scale, cap)
    if _current() != dev:
        with torch.cuda.device(dev):
            return prefill_spans(q, k_cache, v_cache, block_table, q_start, q_len, kv_len, max_q_len, lo, hi, gate, scale, cap, max_kv_len, splits, out)
    _index(q_start, (b,), dev, "q_start")
    _index(q_len, (b,), dev, "q_len")
    if lo is not None:
        _index(lo, (t,), dev, "lo")
    if hi is not None:
        _index(hi, (t,), dev, "hi")
    max_q_len = min(int(max_q_len), t)
    if t == 0 or b == 0 or max_q_len <= 0:
        return out
    if splits is None:
        splits = _row_splits(b, t, hq // hkv, hkv, max_q_len, max_kv_len if max_kv_len is not None else width * bs)
    if not 1 <= splits <= 1024:
        raise ValueError(f"{splits} splits")
    ws = q.new_empty(splits * t * hq * (D + 2), dtype=_F32) if splits > 1 else None
    _check_pages(block_table, nb, bs, kv_len, (t, q_start, q_len, lo, hi))
    rc = _kernels().b200_attn_spans(_SPANS_CALL.pack(
        _SPANS_CALL.size, b, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), _at(gate), block_table.data_ptr(), kv_len.data_ptr(),
        q_start.data_ptr(), q_len.data_ptr(), _at(lo), _at(hi), 0, 0, 0, _at(ws), _status(dev), _stream(dev), 0, max_q_len, t, width, nb, bs, hq, hkv,
        splits, 1, 0, scale, cap))
    _lib.check(rc, "prefill_spans", 2 if splits > 1 else 1)
    return out


def _check_tree_pages(block_table, nb, bs, kv_len, q_start, q_len, lo, mask) -> None:
    """``_check_pages`` for a tree's rows: keys of the context that some row sees, and nodes that some row has the bit of."""
    if not _lib.bounds_checks_on():
        return
    (t, words), width = mask.shape, block_table.shape[1]
    kv, start, n = (x.long()[:, None] for x in (kv_len, q_start, q_len))
    row, first = torch.arange(t, device=mask.device), kv - n
    mine = (start >= 0) & (row >= start) & (row < start + n)                                    # [B, T]: a negative q_start is no sequence
    context = torch.where(mine, first, 0).sum(0)                                                # (a row is one sequence's at most)
    seen = _seen_pages(t, width, bs, kv_len, q_start, q_len, lo, context)
    nodes = ((mask[..., None] >> torch.arange(32, dtype=torch.int32, device=mask.device)) & 1).reshape(t, -1)
    node = torch.arange(32 * words, device=mask.device)
    if lo is not None:
        nodes = nodes * (context[:, None] + node >= lo[:, None])
    key = first + node                                                                          # [B, nodes]
    bits = (mine.float() @ nodes.float() > 0) & (key >= 0) & (key < kv.clamp(max=width * bs))
    seen = seen.long().scatter_add(1, (key // bs).clamp(0, width - 1), bits.long()) > 0
    block_table.masked_fill_(seen & (block_table == -1), -2)
    _lib.check_indices(block_table, 0, nb, 3, keep=-1)


def decode_tree(q, k_cache, v_cache, block_table, mask, q_start, q_len, kv_len, max_q_len, lo=None, gate=None, scale=None, cap: float = 0.0,
                max_kv_len: int | None = None, splits: int | None = None, out=None):
    """Attention of the rows of drafted trees - tokens that continue one context in several ways, verified in one pass - against the paged
    cache, which already holds their keys and values: node i of sequence b, row ``q_start[b] + i``, is the key at ``kv_len[b] - q_len[b] + i``.
    A row sees the context before its tree and the nodes whose bits are set in its ``mask``: int32 [T, words], bit i % 32 of word i / 32 for
    node i - itself and the nodes that it continues, as ``tree.layout`` gives it, or any others; with ``lo`` only keys from ``lo[t]`` on.
    Bits of nodes that a sequence does not have count for nothing.  A row that sees nothing is 0; a key that a row does not see has no part
    in it, whatever the cache holds there.

    The other arguments, pages and rows of no sequence as in ``prefill_spans``.  The keys that a row tile sees are cut
    into ``splits`` items by how many there are; ``max_kv_len`` only bounds their number, so that a bound far above the contexts costs no more
    than the items' join."""
    dev, t, hq, nb, hkv, bs, b, width, scale, out = _paged(q, k_cache, v_cache, block_table, kv_len, gate, out, scale, cap)
    if _current() != dev:
        with torch.cuda.device(dev):
            return decode_tree(q, k_cache, v_cache, block_table, mask, q_start, q_len, kv_len, max_q_len, lo, gate, scale, cap, max_kv_len, splits, out)
    _index(q_start, (b,), dev, "q_start")
    _index(q_len, (b,), dev, "q_len")
    if lo is not None:
        _index(lo, (t,), dev, "lo")
    max_q_len = min(int(max_q_len), t)
    if mask.dim() != 2 or not 0 < mask.shape[1] <= MAX_TREE // 32:
        raise ValueError(f"mask {list(mask.shape)}: int32 [T, words] with 1 to {MAX_TREE // 32} words expected")
    words = mask.shape[1]
    _index(mask, (t, words), dev, "mask")
    if max_q_len > 32 * words:
        raise ValueError(f"trees of {max_q_len} rows, masks of {32 * words} nodes")
    if t == 0 or b == 0 or max_q_len <= 0:
        return out
    if splits is None:
        splits = _row_splits(b, t, hq // hkv, hkv, max_q_len, max_kv_len if max_kv_len is not None else width * bs)
    if not 1 <= splits <= 1024:
        raise ValueError(f"{splits} splits")
    ws = q.new_empty(splits * t * hq * (D + 2), dtype=_F32) if splits > 1 else None
    _check_tree_pages(block_table, nb, bs, kv_len, q_start, q_len, lo, mask)
    rc = _kernels().b200_attn_tree(_SPANS_CALL.pack(
        _SPANS_CALL.size, b, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), _at(gate), block_table.data_ptr(), kv_len.data_ptr(),
        q_start.data_ptr(), q_len.data_ptr(), _at(lo), 0, 0, 0, mask.data_ptr(), _at(ws), _status(dev), _stream(dev), 0, max_q_len, t, width, nb, bs, hq,
        hkv, splits, 1, words, scale, cap))
    _lib.check(rc, "decode_tree", 2 if splits > 1 else 1)
    return out


def shared_groups(pages, block_size: int) -> tuple[list[int], list[int]]:
    """``group_start``, ``shared_len`` for ``decode_shared`` from the page lists of the sequences, in batch order: runs of neighbours that
    share their common leading pages (a sequence alone shares nothing), cut where that saves the most reads of pages - documents behind one
    system page are groups of their own, the page alone is shared where there is no more."""
    pages = [[int(x) for x in row] for row in pages]
    common = [next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b))) for a, b in zip(pages, pages[1:])]   # of neighbours
    # Cuts to consider: where neighbours share equally much several times in a row, the first and the last of them (one in between can move to an
    # end and lose nothing).
    at = [0] + [b for b in range(1, len(pages)) if b in (1, len(pages) - 1) or common[b - 2] != common[b - 1] or common[b] != common[b - 1]] + [len(pages)]
    least = [min(common[a:b - 1], default=math.inf) for a, b in zip(at, at[1:])]              # within the stretches between them
    best = [(0, 0, 0)]                                     # of the sequences up to a cut: pages saved, the last group's cut, what it shares
    for e in range(1, len(at)):
        top, n = (-1, 0, 0), math.inf
        for b in range(e - 1, -1, -1):
            n = min(n, least[b], common[at[b + 1] - 1] if b + 1 < e else math.inf)
            if n == 0 and top[0] >= 0:                     # nothing in common from here on
                break
            saved, shares = (best[b][0] + (at[e] - 1 - at[b]) * n, n) if at[e] - at[b] > 1 else (best[b][0], 0)
            if saved >= top[0]:                            # (of equals, the fewest groups)
                top = (saved, b, shares)
        best.append(top)
    start, shared, e = [len(pages)], [], len(at) - 1
    while e > 0 and pages:
        _, b, n = best[e]
        firsts = [at[b]] if n else range(at[e] - 1, at[b] - 1, -1)
        start += firsts
        shared += [n * block_size] * len(firsts)
        e = b
    return start[::-1], shared[::-1]


def _shared_splits(rows: int, groups: int, g: int, hkv: int, tiles: int, own_keys: int) -> int:
    """Items the shared keys are cut into.  A tile of 128 keys takes an SM about 2 us for a row tile of more than 128 (row, head) pairs and
    half of it for a smaller one, which is cut half as often; a sequence's own keys come at 40 KB an SM and us, on the SMs
    that are left.  Cut as finely as fills the GPU where the shared keys are most of the work (64 rows on 32768 keys: 4 / 9 / 18 / 36 items
    121 / 93 / 108 / 128 us), and by their share of it where they are not (16 rows on 1024 keys, 2000 own ones each: 1 / 4 / 18 items
    38 / 50 / 58 us)."""
    if groups == 0:
        return 1
    per_group = max(1, rows * g // groups)
    whole, rest = divmod(per_group, ROW_TILE)
    full = groups * hkv * (whole + (rest > ROW_TILE // 2))               # row tiles of the two kinds
    half = groups * hkv * (0 < rest <= ROW_TILE // 2)
    work, own_work = (2 * full + half) * tiles * 1.0, rows * hkv * own_keys * (4 * D / 40e3)
    sms = NUM_SMS if 2 * work >= own_work else NUM_SMS * work / (work + own_work)
    splits = int(sms / (full + half / 2))
    if full * splits + half * ((splits + 1) // 2) > sms:
        splits -= 1
    return max(1, min(64, splits, -(-tiles // 2)))


def decode_shared(q, k_cache, v_cache, block_table, kv_len, group_start, shared_len, gate=None, scale=None, cap: float = 0.0,
                  max_shared: int | None = None, max_kv_len: int | None = None, splits: int | None = None, out=None):
    """``decode`` (one query row per sequence) where groups of sequences hold the same leading pages, as a prefix cache hands them
    out: those keys are read and multiplied once for the whole group.

    q: [B, Hq, 128]; group_start int32 [groups + 1], shared_len int32 [groups] (device; ``shared_groups``): the rows
    group_start[g] .. group_start[g + 1] - 1 of ``block_table`` begin with the same pages, whose first shared_len[g] keys they have
    in common (keys at ``kv_len`` and beyond stay unseen); rows of no group are on their own.  ``cap`` as in ``prefill_spans``;
    ``max_shared`` / ``max_kv_len`` bound the lengths, for the choice of ``splits`` (of the shared keys) and of the blocks that share a
    sequence's own keys, by their difference: own keys far beyond it (of a row in no group, or without ``max_shared``) are right, but one
    block's work for each kv head.  A sequence with ``kv_len`` 0 gives 0.  Pages outside the cache as in ``prefill_spans``.  The weights of
    the softmax are rounded to bf16, as in ``prefill``; ``decode`` keeps them in 32 bits."""
    dev, t, hq, nb, hkv, bs, b, width, scale, out = _paged(q, k_cache, v_cache, block_table, kv_len, gate, out, scale, cap)
    if _current() != dev:
        with torch.cuda.device(dev):
            return decode_shared(q, k_cache, v_cache, block_table, kv_len, group_start, shared_len, gate, scale, cap, max_shared, max_kv_len, splits, out)
    if b != t or shared_len.dim() != 1:
        raise ValueError(f"{t} rows for {b} sequences, shared lengths {list(shared_len.shape)}: a row per sequence and a length per group expected")
    n = shared_len.shape[0]
    _index(shared_len, (n,), dev, "shared_len")
    _index(group_start, (n + 1,), dev, "group_start")
    if b == 0:
        return out
    longest = max_kv_len if max_kv_len is not None else width * bs
    common = 0 if n == 0 else longest if max_shared is None else min(longest, max(0, int(max_shared)))
    g = hq // hkv
    own_keys = longest - common
    if splits is None:
        splits = _shared_splits(b, n, g, hkv, -(-common // KEY_TILE), own_keys)
    if not 1 <= splits <= 64:
        raise ValueError(f"{splits} splits")
    # Blocks that share a sequence's own keys: a cluster is slow to launch (32 sequences of 128 keys: 32 us alone, 39 / 53 / 108 us with 2 / 4 / 8
    # blocks), so that it pays only where sequences and kv heads leave SMs idle (2 of 16000 keys: 331 us alone, 172 / 90 / 64 us).
    blocks, cluster = b * hkv * -(-g // 16), 1
    while cluster < 8 and cluster * blocks <= NUM_SMS and own_keys > 256 * cluster:
        cluster *= 2
    lib = _kernels()
    _check_pages(block_table, nb, bs, kv_len)
    ws = q.new_empty(splits * b * hq * (D + 2), dtype=_F32) if n else None
    call = _SPANS_CALL.pack(
        _SPANS_CALL.size, b, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), _at(gate), block_table.data_ptr(), kv_len.data_ptr(),
        0, 0, 0, 0, group_start.data_ptr(), shared_len.data_ptr(), 0, _at(ws), _status(dev), _stream(dev), n, 1, t, width, nb, bs, hq, hkv, splits, cluster,
        0, scale, cap)
    if n:
        _lib.check(lib.b200_attn_shared(call), "decode_shared")
    _lib.check(lib.b200_attn_own_rows(call), "decode_shared")
    return out


# ---------------------------------------------------------------- fp32 oracles
def rope_ref(x, positions, inv_freq, rot):
    """Half-split rotation over the first ``rot`` dims. x: [T, H, D] fp32."""
    half = rot // 2
    ang = positions.double()[:, None] * inv_freq.double()[None, :]
    cos, sin = ang.cos().float()[:, None, :], ang.sin().float()[:, None, :]
    a, b = x[..., :half], x[..., half:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def attention_ref(q, k, v, causal_offset: int, gate=None, scale=None):
    """q [Tq, Hq, D], k/v [Tk, Hkv, D] fp32; query i sees keys <= causal_offset + i."""
    tq, hq, d = q.shape
    tk, hkv, _ = k.shape
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    kk = k.float().repeat_interleave(g, 1)
    vv = v.float().repeat_interleave(g, 1)
    s = torch.einsum("qhd,khd->hqk", q.float(), kk) * scale
    mask = torch.arange(tk, device=q.device)[None, :] > (causal_offset + torch.arange(tq, device=q.device))[:, None]
    s = s.masked_fill(mask[None], float("-inf"))
    o = torch.einsum("hqk,khd->qhd", s.softmax(-1), vv)
    if gate is not None:
        o = o * torch.sigmoid(gate.float())
    return o
