"""Attention over spans and shared pages where something else went wrong: an error that another kernel has reported, pages that are not there,
values that are not finite under weights of zero, and what the debug mode says of them.  Bounds as in ``test_spans_gpu``."""
import math

import pytest
import torch

from test_spans_gpu import DEV, NAN, _i32, close, oracle, pages, rand, run_spans

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


def _modules():
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    return _lib, attention


@pytest.mark.parametrize("code", [4, 2])
def test_an_error_of_another_kernel_changes_no_result(code):
    """The error word is the device's, and stays set until the host has read it: calls meanwhile do all their work."""
    lib, a = _modules()
    torch.manual_seed(11)
    n, new, hq, hkv, bs = 900, 300, 10, 2, 64
    k, v = rand(n, hkv, 128), rand(n, hkv, 128)
    kc, vc, table = pages([(k, v)], bs)
    q, at = rand(new, hq, 128), torch.arange(n - new, n, device=DEV)
    want, bound = oracle(q, k, v, torch.zeros_like(at), at + 1, SCALE)
    lib.check_status()
    lib.status_word(q.device).fill_(code)
    got = [a.prefill_spans(q, kc, vc, table, _i32([0]), _i32([new]), _i32([n]), new, splits=s, out=torch.full_like(q, 7.0)) for s in (1, 4)]
    rows = q[-5:].contiguous()
    got.append(a.decode_shared(rows, kc, vc, table.repeat(5, 1), _i32([n - 4 + i for i in range(5)]), _i32([0, 5]), _i32([640]), splits=3))
    torch.cuda.synchronize()
    with pytest.raises(lib.KernelError, match=lib.ERR_NAMES[code]):
        lib.check_status()
    lib.check_status()
    close(got[0], want, bound)
    close(got[1], want, bound)
    close(got[2], want[-5:], bound[-5:])


@pytest.mark.parametrize("bad", [-1, 1 << 20])
@pytest.mark.parametrize("shared", [0, 192])
@pytest.mark.parametrize("cap", [0.0, 6.0])
def test_pages_that_are_not_there_read_as_zeros(bad, shared, cap):
    """A page outside the cache among the keys that a row sees: keys and values of zero, in every call alike."""
    lib, a = _modules()
    torch.manual_seed(12)
    n, hq, hkv, bs = 500, 6, 2, 64
    k, v = rand(n, hkv, 128), rand(n, hkv, 128)
    kc, vc, table = pages([(k, v)], bs)
    for page in (1, 4, 7):                                 # one that may be shared, one of its own, the last
        table[0, page] = bad
        k[page * bs:(page + 1) * bs] = 0
        v[page * bs:(page + 1) * bs] = 0
    lens = [n, n - 1, n - 77]
    q = rand(3, hq, 128)
    zero = _i32([0, 0, 0])
    want, bound = oracle(q, k, v, zero, _i32(lens), SCALE, cap)
    out = a.decode_shared(q, kc, vc, table.repeat(3, 1), _i32(lens), _i32([0, 3]), _i32([shared]), cap=cap)
    rows = a.prefill_spans(q, kc, vc, table, _i32([0]), _i32([3]), _i32([n]), 3, zero, _i32(lens), cap=cap)
    alone = a.decode_shared(q, kc, vc, table.repeat(3, 1), _i32(lens), _i32([0]), _i32([]), cap=cap)
    torch.cuda.synchronize()
    lib.check_status()
    for got in (rows, out, alone):
        close(got, want, bound)


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("masked", [False, True])
def test_values_that_are_not_finite_under_weights_of_zero(splits, masked):
    """0 x NaN is NaN, in a masked tile as in a whole one: rows that see the key, and no others."""
    def poke(seqs):
        k, v = seqs[0]
        k[:, :, 0] = 0                                     # scores of three keys lie 300 x 8 / sqrt(128) under what they would be: weights below 2^-250
        k[[20, 150, 290], :, 0] = -300
        v[20, :, 3] = NAN                                  # a whole tile of causal rows
        v[150, :, 5] = NAN
        v[290, 0, 7] = NAN                                 # the last tile, masked in any case

    def spans(i, n, kv):
        if not masked:
            return None
        lo = torch.zeros(n, dtype=torch.long)
        lo[::3] = 140
        lo[1::3] = 295
        return lo, torch.arange(kv - n, kv) + 1

    import test_spans_gpu
    made = test_spans_gpu.rand

    def eights(*shape, scale=1.0):                         # queries with 8 in the first place
        x = made(*shape, scale=scale)
        if len(shape) == 3 and shape[1] == 4:
            x[..., 0] = 8
        return x
    test_spans_gpu.rand = eights
    try:
        run_spans([(40, 300)], 4, 2, 64, spans, splits=splits)
        out = run_spans([(40, 300)], 4, 2, 64, spans, splits=splits, poke=poke)
    finally:
        test_spans_gpu.rand = made
    assert out.isnan().any() and not out.isnan().all()


@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("hq,splits", [(4, 2), (4, 1), (24, 2)])
def test_a_part_of_the_keys_that_weighs_nothing_keeps_its_nan(where, hq, splits):
    """A sequence's parts - items of the shared keys, warps of its own - are joined by the formula also where one weighs 2^-250: 0 x NaN is NaN."""
    lib, a = _modules()
    torch.manual_seed(16)
    n, common, hkv, bs = 256 + 64, 256, 2, 64
    k, v = rand(n, hkv, 128), rand(n, hkv, 128)
    k[..., 0] = 0
    low, bad = (slice(0, 256), 130) if where == "shared" else (slice(256 + 16, 256 + 32), 256 + 20)
    k[low, :, 0] = -300                                    # every key of the part
    v[bad, :, 9] = NAN
    kc, vc, table = pages([(k, v)], bs)
    q = rand(3, hq, 128)
    q[..., 0] = 8
    lens = [n, n - 3, n - 12]
    args = kc, vc, table.repeat(3, 1), _i32(lens), _i32([0, 3]), _i32([common])
    out = a.decode_shared(q, *args, splits=splits)
    torch.cuda.synchronize()
    lib.check_status()
    want, bound = oracle(q, k, v, _i32([0, 0, 0]), _i32(lens), SCALE)
    assert want[..., 9].isnan().all() and want.isnan().sum() == 3 * hq
    close(out, want, bound)


def test_debug_mode_reports_missing_pages_that_a_row_sees(monkeypatch):
    """-1 stands for a page that is not there: allowed where no row looks, reported where one does, with its place in the table."""
    lib, a = _modules()
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    torch.manual_seed(13)
    n, new, hq, hkv, bs = 700, 30, 4, 2, 64
    k, v = rand(n, hkv, 128), rand(n, hkv, 128)
    kc, vc, table = pages([(k, v)], bs, table_width=14)
    q = rand(new, hq, 128)
    lo, hi = (x[n - new:].to(DEV) for x in a.visible_spans(n, window=200))
    args = _i32([0]), _i32([new]), _i32([n]), new
    unseen = list(range((n - new - 199) // bs)) + [11, 12, 13]
    for page in range(14):
        odd = table.clone()
        odd[0, page] = -1
        a.prefill_spans(q, kc, vc, odd, *args, lo, hi)
        if page in unseen:
            lib.check_status()
        else:
            with pytest.raises(lib.KernelError, match=f"page table at element {page} "):
                lib.check_status()
        odd = table.repeat(2, 1)
        odd[1, page] = -1
        kv = [n, 5 * bs + 1]
        got = a.decode_shared(q[:2].contiguous(), kc, vc, odd, _i32(kv), _i32([0, 2]), _i32([128]))
        if page > 5:
            lib.check_status()
            close(got, *oracle(q[:2], k, v, _i32([0, 0]), _i32(kv), SCALE))
        else:
            with pytest.raises(lib.KernelError, match=f"page table at element {14 + page} "):
                lib.check_status()
    lib.check_status()


@pytest.mark.parametrize("kv", [1, 64, 65, 300])
def test_debug_mode_decodes_tables_with_pages_that_are_not_there(monkeypatch, kv):
    """Decoding rows over tables that end in -1, as a scheduler keeps them, against sums in 64 bits."""
    lib, a = _modules()
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    torch.manual_seed(14)
    hq, hkv, bs = 10, 2, 64
    seqs = [(rand(n, hkv, 128), rand(n, hkv, 128)) for n in (kv, 200, 0)]
    kc, vc, table = pages(seqs, bs, table_width=8)
    for i, (k, _) in enumerate(seqs):
        table[i, -(-k.shape[0] // bs):] = -1
    before = table.clone()
    q, gate = rand(3, hq, 128), rand(3, hq, 128)
    for groups in ([0], [0, 2]):
        out = a.decode_shared(q, kc, vc, table, _i32([kv, 200, 0]), _i32(groups), _i32([0] * (len(groups) - 1)), gate=gate)
        lib.check_status()
        assert torch.equal(table, before) and not out[2].any()
        for i in range(2):
            close(out[i:i + 1], *oracle(q[i:i + 1], *seqs[i], _i32([0]), _i32([seqs[i][0].shape[0]]), SCALE, gate=gate[i:i + 1]))


@pytest.mark.parametrize("t", [1, 37, 300])
def test_guard_bands_around_the_rows_and_gates_of_an_append(monkeypatch, t):
    """Nothing is written beside the queries and gates that an append gives, nor beside the caches."""
    from deepseek_v4_2080ti_b200.utils import canary
    lib, a = _modules()
    torch.manual_seed(15)
    hq, hkv, bs, kept = 5, 1, 32, []

    def guarded(x, *shape, **kw):
        kept.append(canary.empty(*(shape or x.shape), dtype=x.dtype, device=x.device, name="rows"))
        return kept[-1]
    with canary.enabled(True):
        monkeypatch.setattr(torch.Tensor, "new_empty", guarded)
        monkeypatch.setattr(torch, "empty_like", guarded)
        kc, vc = (canary.zeros(12, hkv, bs, 128, dtype=torch.bfloat16, device=DEV, name="cache") for _ in range(2))
        src = rand(t, hq * 256 + 2 * hkv * 128)
        q, gate = a.qk_norm_rope_axes_append(src, 0, 256, True, src, hq * 256, src, (2 * hq + hkv) * 128, None, None, True, 1e-6,
                                             a.rope_inv_freq(32, 1e6, DEV), a.rotary_axes((6, 5, 5), True), _i32(torch.zeros(3, t)),
                                             _i32(torch.randperm(12 * bs)[:t]), kc, vc, hq, hkv)
        torch.cuda.synchronize()
        monkeypatch.undo()
        lib.check_status()
        assert len(kept) == 2 and q is kept[0] and gate is kept[1]
        assert torch.equal(gate, src[:, :hq * 256].view(t, hq, 256)[..., 128:])
        canary.assert_clean()


def test_scales_and_caps_that_32_bits_do_not_hold_are_refused():
    _, a = _modules()
    k, v = rand(40, 2, 128), rand(40, 2, 128)
    kc, vc, table = pages([(k, v)], 64)
    q = rand(1, 4, 128)
    for kw in ({"cap": 1e-50}, {"cap": 1e-40}, {"cap": 3e38}, {"cap": 1e300}, {"scale": 1e-50}, {"scale": 1e300}, {"scale": 1e25, "cap": 1e-25}):
        with pytest.raises(ValueError):
            a.prefill_spans(q, kc, vc, table, _i32([0]), _i32([1]), _i32([40]), 1, **kw)
        with pytest.raises(ValueError):
            a.decode_shared(q, kc, vc, table, _i32([40]), _i32([0, 1]), _i32([0]), **kw)
