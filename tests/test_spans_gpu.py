"""Rows with spans of keys of their own, and one row per sequence over shared pages, against plain sums in 64 bits.

Bounds.  The kernels round the weights p of a row to bf16 (each off by 2^-8 of itself at most) before they multiply values,
and the result once more: |error| <= 2^-8 A + 2^-8 |o| with A = sum p |v| / sum p, and as much again times 2^-4 for everything
in 32 bits (products, exponentials, sums: below 2^-12 of A at these sizes, and the second order of the two roundings).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def oracle(q, k, v, lo, hi, scale, cap=0.0, gate=None):
    """q [T, Hq, 128], k / v [n, Hkv, 128], lo / hi [T]; every row over the keys it sees and no others.  (result, bound)"""
    t, hq, _ = q.shape
    n, hkv, _ = k.shape
    j = torch.arange(n, device=q.device)
    seen = (j >= lo[:, None]) & (j < hi[:, None])
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mean = torch.zeros_like(out)
    for h in range(hq):
        kh, vh = k[:, h * hkv // hq].double(), v[:, h * hkv // hq].double()
        for a in range(0, t, 64):
            s = q[a:a + 64, h].double() @ kh.t() * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            see = seen[a:a + 64]
            s = torch.where(see, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            l = p.sum(-1, keepdim=True)
            l = torch.where(see.any(-1, keepdim=True), l, 1.0)
            pv = torch.where(see[..., None], p[..., None] * vh[None], 0.0)
            out[a:a + 64, h] = pv.sum(1) / l
            mean[a:a + 64, h] = pv.abs().sum(1) / l
    g = 1.0 if gate is None else torch.sigmoid(gate.double())
    return out * g, (mean + out.abs()) * g * 2.0 ** -8 * (1 + 2.0 ** -4)


def close(got, want, bound):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    fine = want.isfinite()
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or over.max().item() <= 1e-30, f"off by {over.max().item():.3e} more than the bound"


def pages(seqs, bs, spare=2, fill=NAN, seed=0, table_width=None):
    """Caches and block table of sequences [(k [n, Hkv, 128], v)]; what belongs to none of them is ``fill``."""
    hkv = seqs[0][0].shape[1]
    counts = [(k.shape[0] + bs - 1) // bs for k, _ in seqs]
    total = sum(counts) + spare
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(total, generator=g).to(DEV)
    kc = torch.full((total, hkv, bs, 128), fill, dtype=torch.bfloat16, device=DEV)
    vc = torch.full_like(kc, fill)
    table = torch.full((len(seqs), max(max(counts), 1) if table_width is None else table_width), total - 1 if spare else 0, device=DEV)
    at = 0
    for i, (k, v) in enumerate(seqs):
        table[i, :counts[i]] = perm[at:at + counts[i]]
        at += counts[i]
        j = torch.arange(k.shape[0], device=DEV)
        kc[table[i, j // bs], :, j % bs] = k
        vc[table[i, j // bs], :, j % bs] = v
    return kc, vc, _i32(table)


def rand(*shape, scale=1.0):
    return (torch.randn(*shape, device=DEV) * scale).bfloat16()


def run_spans(lens, hq, hkv, bs, spans, cap=0.0, gate=False, splits=None, q_scale=1.5, fill=NAN, poke=None, scale=None):
    """``lens`` [(new, kv)]; ``spans(i, new, kv)`` -> (lo, hi) or None.  Checks every row."""
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    torch.manual_seed(sum(n + 7 * k for n, k in lens) + hq)
    seqs = [(rand(kv, hkv, 128), rand(kv, hkv, 128)) for _, kv in lens]
    if poke:
        poke(seqs)
    kc, vc, table = pages(seqs, bs, fill=fill)
    total = sum(n for n, _ in lens)
    q = rand(total, hq, 128, scale=q_scale)
    g = rand(total, hq, 128) if gate else None
    starts = [sum(n for n, _ in lens[:i]) for i in range(len(lens))]
    parts = [spans(i, n, kv) for i, (n, kv) in enumerate(lens)]
    lo = hi = None
    if parts[0] is not None:
        lo, hi = (torch.cat([p[c].to(DEV).to(torch.int32) for p in parts]) for c in (0, 1))
    out = attention.prefill_spans(q, kc, vc, table, _i32(starts), _i32([n for n, _ in lens]), _i32([k for _, k in lens]), max(n for n, _ in lens),
                                  lo, hi, gate=g, cap=cap, splits=splits, scale=scale, max_kv_len=max(k for _, k in lens))
    torch.cuda.synchronize()
    _lib.check_status()
    for i, (n, kv) in enumerate(lens):
        r = slice(starts[i], starts[i] + n)
        pos = torch.arange(kv - n, kv, device=DEV)
        l, h = (torch.zeros_like(pos), pos + 1) if lo is None else (lo[r].long(), hi[r].long().clamp(max=kv))
        want, bound = oracle(q[r], *seqs[i], l, h, 1 / math.sqrt(128) if scale is None else scale, cap, None if g is None else g[r])
        close(out[r], want, bound)
    return out


def causal(i, n, kv):
    return None


def documents(lengths):
    def spans(i, n, kv):
        from deepseek_v4_2080ti_b200.ops import attention
        lo, hi = attention.visible_spans(kv, lengths[i])
        return lo[kv - n:], hi[kv - n:]
    return spans


def ragged(i, n, kv):
    """Spans of every kind, some empty, some beyond the context."""
    g = torch.Generator().manual_seed(n * 31 + kv)
    a = torch.randint(-3, kv + 3, (n,), generator=g)
    b = torch.randint(-3, kv + 40, (n,), generator=g)
    return a.clamp(min=0), torch.where(torch.rand(n, generator=g) < 0.2, a.clamp(min=0), b)


@pytest.mark.parametrize("lens,hq,hkv,bs", [
    ([(1, 1)], 1, 1, 64), ([(1, 129)], 5, 1, 16), ([(128, 128)], 2, 1, 64), ([(129, 129)], 2, 2, 32), ([(77, 300)], 4, 2, 128),
    ([(300, 300)], 8, 8, 256), ([(52, 1000)], 10, 2, 64), ([(51, 640)], 5, 1, 64), ([(1, 4000), (3, 5), (200, 200)], 16, 2, 64)])
@pytest.mark.parametrize("gate,cap", [(False, 0.0), (True, 5.0)])
def test_causal_rows(lens, hq, hkv, bs, gate, cap):
    run_spans(lens, hq, hkv, bs, causal, cap=cap, gate=gate)


@pytest.mark.parametrize("splits", [1, 2, 5, 40])
@pytest.mark.parametrize("lens,hq,hkv", [([(40, 700)], 5, 1), ([(300, 900), (9, 1)], 4, 4), ([(2, 2500), (130, 260)], 12, 2)])
def test_keys_cut_into_items(lens, hq, hkv, splits):
    lens = [(min(n, k), k) for n, k in lens]
    run_spans(lens, hq, hkv, 64, causal, splits=splits, gate=True)


@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_documents(splits, cap):
    run_spans([(700, 700), (150, 420)], 6, 2, 64, documents([[1, 127, 128, 3, 300, 0, 141], [400, 20]]), cap=cap, splits=splits)


@pytest.mark.parametrize("splits", [None, 1, 4])
@pytest.mark.parametrize("lens", [[(200, 333)], [(1, 1), (130, 600), (17, 40)]])
def test_ragged_and_empty_spans(lens, splits):
    out = run_spans(lens, 4, 2, 32, ragged, splits=splits, gate=True)
    assert out.isfinite().all()


def test_blocks_that_see_each_other_and_windows():
    from deepseek_v4_2080ti_b200.ops import attention
    lo, hi = attention.visible_spans(900, blocks=[(10, 410), (500, 501), (600, 900)], window=450)
    run_spans([(777, 900)], 5, 1, 64, lambda i, n, kv: (lo[kv - n:], hi[kv - n:]))


@pytest.mark.parametrize("splits", [1, 3])
def test_values_that_are_not_finite(splits):
    """A document's infinities and NaN reach its own rows - as the formula has it - and no others."""
    def poke(seqs):
        k, v = seqs[0]
        v[5, :, 3] = NAN                  # first document
        v[140, 0, :] = math.inf           # second: one kv head
        v[141, 0, 7] = -math.inf
        k[300, 1, :] = NAN                # third: a key
        v[420, :, 100] = math.inf         # fourth: its last ten rows
    run_spans([(430, 430)], 4, 2, 64, documents([[100, 120, 130, 80]]), poke=poke, splits=splits)

    def first_keys(i, n, kv):
        lo = torch.zeros(n, dtype=torch.long)
        return lo, torch.full((n,), 419)
    run_spans([(90, 430)], 4, 2, 64, first_keys, poke=lambda s: (s[0][0][419:].fill_(NAN), s[0][1][419:].fill_(math.inf)), splits=splits)


def test_scores_far_apart():
    """Maxima that grow by more than any rescale step from tile to tile, and rows whose first tiles weigh nothing."""
    def poke(seqs):
        k, _ = seqs[0]
        k *= torch.linspace(0.1, 6.0, k.shape[0], device=DEV)[:, None, None].bfloat16()
    run_spans([(140, 1500)], 2, 1, 64, causal, q_scale=6.0, poke=poke)
    run_spans([(140, 1500)], 2, 1, 64, causal, q_scale=6.0, poke=poke, cap=50.0)
    run_spans([(30, 1500)], 2, 1, 64, causal, q_scale=6.0, poke=poke, cap=3.0, splits=1)


def test_rows_of_no_sequence_stay():
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    torch.manual_seed(3)
    k, v = rand(300, 2, 128), rand(300, 2, 128)
    kc, vc, table = pages([(k, v)], 64)
    q = rand(50, 4, 128)
    for splits in (1, 3):
        out = torch.full_like(q, 7.0)
        got = attention.prefill_spans(q, kc, vc, table, _i32([10]), _i32([20]), _i32([300]), 20, out=out, splits=splits)
        torch.cuda.synchronize()
        _lib.check_status()
        assert got is out and bool((out[:10] == 7.0).all()) and bool((out[30:] == 7.0).all())
        pos = torch.arange(280, 300, device=DEV)
        close(out[10:30], *oracle(q[10:30], k, v, torch.zeros_like(pos), pos + 1, 1 / math.sqrt(128)))


# ------------------------------------------------------------------------------------------------ shared pages
def run_shared(groups, hq, hkv, bs, cap=0.0, gate=False, splits=None, alone=0, lens_below=False, poke=None):
    """``groups`` [(shared keys in whole pages or not, [own keys])]; ``alone``: rows behind them that belong to no group."""
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    torch.manual_seed(len(groups) * 100 + hq + bs)
    seqs, rows, start, shared = [], [], [0], []
    for n, own in groups:
        pk, pv = rand(n, hkv, 128), rand(n, hkv, 128)
        rows += [(torch.cat([pk, rand(m, hkv, 128)]), torch.cat([pv, rand(m, hkv, 128)])) for m in own]
        start.append(len(rows))
        shared.append(n)
    rows += [(rand(50 + 90 * i, hkv, 128), rand(50 + 90 * i, hkv, 128)) for i in range(alone)]
    if poke:
        poke(rows)
    kc, vc, table = pages(rows, bs)                       # every sequence has pages of its own ..
    for g, n in enumerate(shared):                        # .. but a group's leading ones are its first row's
        table[start[g]:start[g + 1], :n // bs] = table[start[g], :n // bs].clone()
    kv = [k.shape[0] for k, _ in rows]
    if lens_below:                                        # sequences that have not reached the end of what their pages share
        kv[0] = max(1, shared[0] // 2)
        kv[1] = 0
    q = rand(len(rows), hq, 128, scale=1.5)
    g = rand(len(rows), hq, 128) if gate else None
    out = attention.decode_shared(q, kc, vc, table, _i32(kv), _i32(start), _i32(shared), gate=g, cap=cap, splits=splits,
                                  max_shared=max(shared, default=0), max_kv_len=max(kv))
    torch.cuda.synchronize()
    _lib.check_status()
    for b, (k, v) in enumerate(rows):
        want, bound = oracle(q[b:b + 1], k, v, _i32([0]), _i32([kv[b]]), 1 / math.sqrt(128), cap, None if g is None else g[b:b + 1])
        close(out[b:b + 1], want, bound)
    return out


@pytest.mark.parametrize("groups,hq,hkv,bs", [
    ([(64, [1, 1])], 5, 1, 64), ([(640, [40, 3, 200])], 40, 8, 64), ([(256, [5] * 30)], 10, 2, 16), ([(384, [1] * 64)], 5, 1, 128),
    ([(512, [7] * 60)], 6, 1, 256), ([(0, [30, 40]), (128, [2] * 9), (320, [600])], 4, 4, 64), ([(1024, [130, 129])], 1, 1, 32)])
@pytest.mark.parametrize("gate,cap", [(False, 0.0), (True, 8.0)])
def test_shared_pages(groups, hq, hkv, bs, gate, cap):
    run_shared(groups, hq, hkv, bs, cap=cap, gate=gate)


@pytest.mark.parametrize("splits", [1, 2, 7, 64])
def test_shared_pages_cut_into_items(splits):
    run_shared([(900 // 64 * 64, [10, 700, 64]), (192, [1] * 6)], 8, 2, 64, splits=splits, gate=True, alone=3)


def test_rows_of_no_group_and_short_rows():
    run_shared([(320, [9, 9, 33])], 6, 2, 64, alone=2, lens_below=True)
    run_shared([], 6, 2, 64, alone=4)


def test_values_that_are_not_finite_in_one_sequence():
    def poke(rows):
        rows[1][1][700, :, 5] = NAN
        rows[2][1][705, 0, 6] = math.inf
    run_shared([(640, [70, 70, 70])], 4, 2, 64, poke=poke)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (8, 1), (9, 1), (24, 2), (17, 1), (40, 1)])
def test_head_counts(hq, hkv):
    """One, a group of 8, two, and more heads of a kv head than a block takes."""
    run_shared([(128, [1, 130, 64]), (64, [300])], hq, hkv, 32, alone=2, gate=True)
    run_spans([(20, 150), (3, 3)], hq, hkv, 32, causal)


@pytest.mark.parametrize("own", [15, 16, 17, 500, 2100, 9000])
def test_long_own_contexts(own):
    run_shared([(64, [own, 1]), (0, [own])], 6, 2, 16, cap=20.0)


def test_results_do_not_depend_on_the_memory_s_pace():
    """Several items a block, loads that finish late and in any order (another stream keeps the memory busy): the same bits every time."""
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    torch.manual_seed(5)
    b, hq, hkv, bs, shared, own = 40, 40, 8, 64, 4096, 200
    total = shared // bs + b * 4
    kc, vc = rand(total, hkv, bs, 128), rand(total, hkv, bs, 128)
    table = torch.zeros(b, shared // bs + 4, dtype=torch.long, device=DEV)
    table[:, :shared // bs] = torch.arange(shared // bs, device=DEV)
    table[:, shared // bs:] = shared // bs + torch.arange(b * 4, device=DEV).view(b, 4)
    q, table, kv = rand(b, hq, 128), _i32(table), _i32([shared + own] * b)
    rows = rand(1200, hq, 128)
    side, big = torch.cuda.Stream(), torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    want = None
    for i in range(60):
        if i:
            with torch.cuda.stream(side):
                big[:1 << 27].copy_(big[1 << 27:])
        got = (attention.decode_shared(q, kc, vc, table, kv, _i32([0, b]), _i32([shared]), max_shared=shared, max_kv_len=shared + own, splits=12),
               attention.prefill_spans(rows, kc, vc, table[:1].contiguous(), _i32([0]), _i32([1200]), _i32([shared + own]), 1200, splits=1))
        torch.cuda.synchronize()
        _lib.check_status()
        if want is None:
            want = got
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
