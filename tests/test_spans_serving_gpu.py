"""The calls over several axes, spans and shared pages together and under the conditions of a server: a picture that several questions
share, captured steps whose lengths change between replays, two streams, caches larger than 32-bit offsets, odd tables and limits."""
import math

import pytest
import torch

from test_spans_gpu import DEV, NAN, _i32, causal, close, oracle, pages, rand, run_shared, run_spans

pytestmark = pytest.mark.gpu
HQ, HKV, BS = 10, 2, 64
SECTIONS = (6, 5, 5)


def _attention():
    from deepseek_v4_2080ti_b200.ops import attention
    return attention


class Layer:
    """One attention layer's projections of given rows: q and gate per head, keys, values."""

    def __init__(self, n_pages):
        a = _attention()
        self.kc = torch.full((n_pages, HKV, BS, 128), NAN, dtype=torch.bfloat16, device=DEV)
        self.vc = torch.full_like(self.kc, NAN)
        self.qg, self.kg = rand(128, scale=0.2), rand(128, scale=0.2)
        self.inv, self.axes = a.rope_inv_freq(2 * sum(SECTIONS), 1e6, DEV), a.rotary_axes(SECTIONS, True)

    def append(self, src, positions, slots):
        return _attention().qk_norm_rope_axes_append(src, 0, 256, True, src, HQ * 256, src, HQ * 256 + HKV * 128, self.qg, self.kg, True, 1e-6,
                                                     self.inv, self.axes, positions, slots, self.kc, self.vc, HQ, HKV)

    def check_append(self, src, positions, slots, q):
        """Bound: one rounding to bf16 and 32-bit arithmetic below 2^-16 of a pair before it."""
        h, rot = sum(SECTIONS), 2 * sum(SECTIONS)
        ang = torch.stack([positions[a].double() * self.inv[i].double() for i, a in enumerate(self.axes)], -1)[:, None]

        def want(x, gamma):
            x = x.double()
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (gamma.double() + 1)
            a, b = x[..., :h], x[..., h:rot]
            y = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), x[..., rot:]], -1)
            pair = torch.cat([torch.maximum(a.abs(), b.abs())] * 2 + [x[..., rot:].abs()], -1)
            return y, y.abs() * 2.0 ** -8 + pair * 2.0 ** -16
        t, live = src.shape[0], slots >= 0
        at = slots[live].long()
        close(q, *want(src[:, :HQ * 256].view(t, HQ, 256)[..., :128], self.qg))
        close(self.kc[at // BS, :, at % BS], *(x[live] for x in want(src[:, HQ * 256:HQ * 256 + HKV * 128].reshape(t, HKV, 128), self.kg)))

    def keys(self, table_row, n):
        j = torch.arange(n, device=DEV)
        rows = table_row.long()[j // BS]
        return self.kc[rows, :, j % BS], self.vc[rows, :, j % BS]


def _src(t):
    return rand(t, HQ * 256 + 2 * HKV * 128, scale=1.5)


def test_a_picture_and_the_questions_about_it():
    """Text, a picture whose patches see each other, text; then questions that share its whole pages, each read in one ragged batch; then
    decoding steps.  Every call's rows against sums in 64 bits over what the cache holds."""
    from deepseek_v4_2080ti_b200.ops import _lib
    a = _attention()
    torch.manual_seed(1)
    layer, text, side, tail = Layer(40), 90, 12, 60
    n = text + side * side + tail
    i = torch.arange(side * side)
    pos = torch.cat([torch.arange(text).repeat(3, 1), torch.stack([torch.zeros_like(i), i // side, i % side]) + text,
                     (torch.arange(tail) + text + side).repeat(3, 1)], 1)
    lo, hi = a.visible_spans(n, blocks=[(text, text + side * side)])
    first = torch.randperm(40)[:5].tolist()
    table = _i32([first])
    slots = _i32([first[j // BS] * BS + j % BS for j in range(n)])
    src, positions = _src(n), _i32(pos)
    q, gate = layer.append(src, positions, slots)
    layer.check_append(src, positions, slots, q)
    out = a.prefill_spans(q, layer.kc, layer.vc, table, _i32([0]), _i32([n]), _i32([n]), n, _i32(lo), _i32(hi), gate=gate, max_kv_len=n)
    close(out, *oracle(q, *layer.keys(table[0], n), _i32(lo), _i32(hi), 1 / math.sqrt(128), gate=gate))

    # questions: the prompt's four whole pages are shared, its rest and the question are every sequence's own
    common, lens = n // BS * BS, [n + 7, n + 1, n + 130, n + 64]
    free = [x for x in range(40) if x not in first]
    lists = []
    for length in lens:
        need = -(-(length + 4) // BS) - common // BS
        lists.append(first[:common // BS] + free[:need])
        free = free[need:]
    width = max(map(len, lists))
    table = _i32([row + [0] * (width - len(row)) for row in lists])
    new = [length - common for length in lens]
    starts = [sum(new[:b]) for b in range(4)]
    p = torch.cat([torch.cat([pos[:, common:], (torch.arange(length - n) + int(pos.max()) + 1).repeat(3, 1)], 1) for length in lens], 1)
    slots = _i32([lists[b][j // BS] * BS + j % BS for b in range(4) for j in range(common, lens[b])])
    src, positions = _src(sum(new)), _i32(p)
    q, gate = layer.append(src, positions, slots)
    layer.check_append(src, positions, slots, q)
    out = a.prefill_spans(q, layer.kc, layer.vc, table, _i32(starts), _i32(new), _i32(lens), max(new), gate=gate, max_kv_len=max(lens))
    for b in range(4):
        r, at = slice(starts[b], starts[b] + new[b]), torch.arange(common, lens[b], device=DEV)
        close(out[r], *oracle(q[r], *layer.keys(table[b], lens[b]), torch.zeros_like(at), at + 1, 1 / math.sqrt(128), gate=gate[r]))

    start, shared = a.shared_groups(lists, BS)
    assert (start, shared) == ([0, 4], [common])
    for step in range(3):
        slots = _i32([lists[b][lens[b] // BS] * BS + lens[b] % BS for b in range(4)])
        positions, src = _i32([[x - n + int(pos.max()) + 1 for x in lens]] * 3), _src(4)
        lens = [x + 1 for x in lens]
        q, gate = layer.append(src, positions, slots)
        layer.check_append(src, positions, slots, q)
        out = a.decode_shared(q, layer.kc, layer.vc, table, _i32(lens), _i32(start), _i32(shared), gate=gate, cap=20.0 if step == 2 else 0.0,
                              max_shared=common, max_kv_len=max(lens))
        for b in range(4):
            close(out[b:b + 1], *oracle(q[b:b + 1], *layer.keys(table[b], lens[b]), _i32([0]), _i32(lens[b:b + 1]), 1 / math.sqrt(128),
                                        20.0 if step == 2 else 0.0, gate[b:b + 1]))
    torch.cuda.synchronize()
    _lib.check_status()


def _captured(fn):
    """``fn`` captured, after a warm-up on a side stream, with its outputs."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_captured_steps_with_other_lengths_rows_and_groups():
    """Two captured steps (append and decoding; a ragged portion of prompt rows), replayed in turn over changed lengths, tables, groups and
    spans, idle rows among them: the bits of eager calls, and those within their bounds."""
    from deepseek_v4_2080ti_b200.ops import _lib
    a = _attention()
    torch.manual_seed(2)
    layer, b, width, t = Layer(64), 6, 10, 150
    layer.kc.copy_(rand(*layer.kc.shape))
    layer.vc.copy_(rand(*layer.vc.shape))
    src, positions, slots = _src(b), _i32(torch.zeros(3, b)), _i32([-1] * b)
    table, kv, start, shared = _i32(torch.zeros(b, width)), _i32([0] * b), _i32([0, 0, 0]), _i32([0, 0])
    rows, gates = rand(t, HQ, 128), rand(t, HQ, 128)
    q_start, q_len, lens, lo, hi = _i32([0] * b), _i32([0] * b), _i32([0] * b), _i32([0] * t), _i32([0] * t)
    out_rows = torch.zeros_like(rows)

    def decode():
        q, gate = layer.append(src, positions, slots)
        return q, gate, a.decode_shared(q, layer.kc, layer.vc, table, kv, start, shared, gate=gate, max_shared=300, max_kv_len=width * BS, splits=3)

    def prompt():
        return a.prefill_spans(rows, layer.kc, layer.vc, table, q_start, q_len, lens, t, lo, hi, gate=gates, splits=4, out=out_rows)
    g1, got1 = _captured(decode)
    g2, got2 = _captured(prompt)
    for trial in range(4):
        g = torch.Generator().manual_seed(trial)
        perm = torch.randperm(64, generator=g)
        tb = torch.stack([torch.cat([perm[:5], perm[5 + 5 * i:10 + 5 * i]]) for i in range(b)])           # five pages in common, five of their own
        table.copy_(tb)
        n = torch.randint(321, width * BS, (b,), generator=g)
        n[trial] = 0                                       # idle
        kv.copy_(n)
        slots.copy_(torch.where(n > 0, tb[torch.arange(b), (n - 1).clamp(min=0) // BS] * BS + (n - 1) % BS, -1))
        positions.copy_(n.repeat(3, 1))
        start.copy_(torch.tensor([[0, 6, 6], [0, 2, 6], [1, 4, 6], [0, 0, 5]][trial]))
        shared.copy_(torch.tensor([[300, 0], [320, 64], [17, 300], [300, 256]][trial]))
        src.copy_(_src(b))
        m = torch.randint(0, 25, (b,), generator=g)
        q_len.copy_(m)
        q_start.copy_(m.cumsum(0) - m)
        lens.copy_(n)
        lo.copy_(torch.randint(0, 400, (t,), generator=g))
        hi.copy_(torch.randint(0, 700, (t,), generator=g))
        rows.copy_(rand(t, HQ, 128))
        out_rows.fill_(5.0)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in got1] + [got2.clone()]
        out_rows.fill_(5.0)
        q, gate, out = decode()
        for x, y in zip(replayed, (q, gate, out, prompt())):
            assert torch.equal(x, y)
        torch.cuda.synchronize()
        _lib.check_status()
        layer.check_append(src, positions, slots, q)
        for i in range(b):
            r = slice(int(q_start[i]), int(q_start[i] + q_len[i]))
            if n[i] == 0:
                assert not out[i].any() and not out_rows[r].any()
                continue
            k, v = layer.keys(table[i], int(n[i]))
            close(out[i:i + 1], *oracle(q[i:i + 1], k, v, _i32([0]), _i32([int(n[i])]), 1 / math.sqrt(128), gate=gate[i:i + 1]))
            close(out_rows[r], *oracle(rows[r], k, v, lo[r].long(), hi[r].long().clamp(max=int(n[i])), 1 / math.sqrt(128), gate=gates[r]))
        assert bool((out_rows[int(m.sum()):] == 5.0).all())


def test_two_streams_at_once():
    from deepseek_v4_2080ti_b200.ops import _lib
    a = _attention()
    torch.manual_seed(3)
    b, n = 12, 640
    kc, vc = rand(200, HKV, BS, 128), rand(200, HKV, BS, 128)
    table = torch.randint(0, 200, (b, 10), device=DEV, dtype=torch.int32)
    table[:, :4] = table[0, :4].clone()
    q, rows, kv = rand(b, HQ, 128), rand(700, HQ, 128), _i32([n] * b)
    group, shared, zero, many, full = _i32([0, b]), _i32([256]), _i32([0]), _i32([600]), _i32([n])
    first = table[:1].contiguous()

    def one():
        return a.decode_shared(q, kc, vc, table, kv, group, shared, max_shared=256, max_kv_len=n, splits=2)

    def two():
        return a.prefill_spans(rows, kc, vc, first, zero, many, full, 600, splits=3, out=torch.zeros_like(rows))
    want = one(), two()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = ([], [])
    for _ in range(25):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((one, two)[i]())
    torch.cuda.synchronize()
    _lib.check_status()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("cap,q_scale", [(30.0, 1.5), (5.0, 1.5), (2.0, 0.5), (1.0, 3.0), (0.01, 1.0), (1e-6, 1.0), (1e6, 1.0), (1e9, 0.5)])
def test_scores_on_every_side_of_a_cap(cap, q_scale):
    """Far below the cap, around half of it, around it, beyond; caps whose powers leave 32 bits.  Whole tiles and masked ones."""
    run_spans([(150, 700), (20, 20)], 4, 2, 64, causal, cap=cap, q_scale=q_scale, splits=1)


@pytest.mark.parametrize("cap", [5.0, 1.0, 0.01, 1e6, 1e9])
def test_shared_and_own_scores_on_every_side_of_a_cap(cap):
    run_shared([(192, [70, 5, 300]), (64, [33, 1])], 6, 2, 64, cap=cap, gate=True, alone=1)


@pytest.mark.parametrize("n,hq,hkv", [(57, 8, 8), (64, 16, 8), (128, 8, 8)])
def test_many_sequences(n, hq, hkv):
    """More (sequence, kv head) pairs than blocks of the larger form run at once."""
    run_shared([(64, [1 + 13 * i % 90 for i in range(n - 9)])], hq, hkv, 32, alone=9, gate=True)


def test_a_portion_beside_single_rows():
    """The longest portion would leave most row tiles empty; and portions in any order, empty ones among them."""
    run_spans([(1, 70)] * 40 + [(700, 900)] + [(1, 3), (2, 2)], 4, 1, 64, causal, gate=True)
    run_spans([(500, 500)] + [(1, 129)] * 5 + [(300, 310)], 10, 2, 16, causal, splits=2)


@pytest.mark.parametrize("splits", [1, 3])
def test_infinite_scores_under_a_cap(splits):
    """Keys with an infinity give the cap or its negative, also where a row sees nothing else."""
    def poke(seqs):
        seqs[0][0][[0, 5, 64, 300], :, 3] = math.inf
        seqs[1][0][:, :, 9] = -math.inf
    run_spans([(400, 400), (30, 200)], 4, 2, 64, causal, cap=4.0, splits=splits, poke=poke)


@pytest.mark.parametrize("splits", [1, 3])
def test_spans_at_the_ends_of_32_bits(splits):
    """Ends below zero and behind every context: nothing, and everything, is seen."""
    low, high = -2 ** 31, 2 ** 31 - 1

    def spans(i, n, kv):
        ends = [(0, low), (0, high), (high, high), (low, high), (low, low), (0, -1), (5, 200), (high, low)]
        lo, hi = zip(*(ends[j % 8] for j in range(n)))
        return torch.tensor(lo), torch.tensor(hi)
    run_spans([(40, 300), (9, 129)], 4, 2, 64, spans, splits=splits)


def test_pages_that_no_row_sees_are_not_followed():
    """Entries before a window's first key and behind the last one: pages that were given back, or none."""
    from deepseek_v4_2080ti_b200.ops import _lib
    a = _attention()
    torch.manual_seed(4)
    n, new = 700, 30
    k, v = rand(n, HKV, 128), rand(n, HKV, 128)
    for bs in (16, 64):
        kc, vc, table = pages([(k, v)], bs, table_width=n // bs + 4)
        lo, hi = (x[n - new:].to(DEV) for x in a.visible_spans(n, window=200))
        for bad in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
            odd = table.clone()
            odd[:, :(n - new - 199) // bs] = bad
            odd[:, n // bs + 1:] = bad
            q = rand(new, HQ, 128)
            out = a.prefill_spans(q, kc, vc, odd, _i32([0]), _i32([new]), _i32([n]), new, lo, hi)
            torch.cuda.synchronize()
            _lib.check_status()
            close(out, *oracle(q, k, v, lo.long(), hi.long(), 1 / math.sqrt(128)))


def test_debug_mode(monkeypatch):
    """With index checks on: tables with -1 for pages that are not there and negative slots pass; a page beyond the cache is reported, and
    the kernels have run on what took its place."""
    from deepseek_v4_2080ti_b200.ops import _lib
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    a = _attention()
    torch.manual_seed(8)
    n, new = 400, 20
    k, v = rand(n, HKV, 128), rand(n, HKV, 128)
    kc, vc, table = pages([(k, v)], BS)
    lo, hi = (x[n - new:].to(DEV) for x in a.visible_spans(n, window=100))
    q = rand(new, HQ, 128)
    want, bound = oracle(q, k, v, lo.long(), hi.long(), 1 / math.sqrt(128))
    table[0, :4] = -1
    args = _i32([0]), _i32([new]), _i32([n]), new, lo, hi
    close(a.prefill_spans(q, kc, vc, table, *args), want, bound)
    layer = Layer(2)
    src, slots = _src(3), _i32([-7, 5, -1])
    rows, _ = layer.append(src, _i32(torch.zeros(3, 3)), slots)
    layer.check_append(src, _i32(torch.zeros(3, 3)), slots, rows)
    assert slots.tolist() == [-7, 5, -1]
    _lib.check_status()
    table[0, 0] = kc.shape[0] + 3
    close(a.prefill_spans(q, kc, vc, table, *args), want, bound)
    with pytest.raises(_lib.KernelError, match="index out of range"):
        _lib.check_status()
    one = a.decode_shared(q[:1].contiguous(), kc, vc, table.clamp(min=0), _i32([n]), _i32([0, 1]), _i32([0]))
    _lib.check_status()
    assert one.shape == (1, HQ, 128)


def test_guard_bands(monkeypatch):
    """Nothing is written beside caches, results and workspaces: bands around all of them stay as they are."""
    from deepseek_v4_2080ti_b200.ops import _lib
    from deepseek_v4_2080ti_b200.utils import canary
    a = _attention()
    torch.manual_seed(9)

    kept = []                                              # (a buffer's bands are looked at while it lives)

    def guarded(t, *shape, dtype=None):
        kept.append(canary.empty(*shape, dtype=dtype or t.dtype, device=t.device, name="workspace"))
        return kept[-1]

    def empty_like(t):
        return guarded(t, *t.shape)
    with canary.enabled(True):
        monkeypatch.setattr(torch.Tensor, "new_empty", guarded)
        layer = Layer(1)
        layer.kc, layer.vc = (canary.zeros(12, HKV, BS, 128, dtype=torch.bfloat16, device=DEV, name="cache") for _ in range(2))
        for t in (1, 37, 300):
            layer.append(_src(t), _i32(torch.randint(0, 99, (3, t))), _i32(torch.randperm(12 * BS)[:t]))
        table = _i32(torch.arange(12).view(1, 12).repeat(40, 1))
        for lens in ([1], [300], [7, 128, 200], [1] * 39 + [150]):
            starts, total = [sum(lens[:b]) for b in range(len(lens))], sum(lens)
            q = guarded(layer.kc, total, HQ, 128).normal_()
            out = empty_like(q)
            for splits in (1, 3):
                a.prefill_spans(q, layer.kc, layer.vc, table[:len(lens)].contiguous(), _i32(starts), _i32(lens), _i32([12 * BS - b for b in range(len(lens))]),
                                max(lens), gate=q, splits=splits, out=out)
        for b in (1, 3, 40):
            q = guarded(layer.kc, b, HQ, 128).normal_()
            for splits in (1, 5):
                a.decode_shared(q, layer.kc, layer.vc, table[:b].contiguous(), _i32([12 * BS - i for i in range(b)]), _i32([0, b // 2, b]), _i32([300, 512]),
                                gate=q, splits=splits, out=empty_like(q))
        torch.cuda.synchronize()
        monkeypatch.undo()
        _lib.check_status()
        assert canary.live_buffers() >= len(kept)
        canary.assert_clean()


def test_in_place():
    """Rows whose results take the queries' place."""
    a = _attention()
    torch.manual_seed(6)
    k, v = rand(500, HKV, 128), rand(500, HKV, 128)
    kc, vc, table = pages([(k, v)] * 3, BS)
    q, gate = rand(3, HQ, 128), rand(3, HQ, 128)
    table[1:, :4] = table[0, :4].clone()
    args = kc, vc, table, _i32([500, 420, 300]), _i32([0, 3]), _i32([256])
    want, out = a.decode_shared(q, *args, gate=gate), q.clone()
    assert a.decode_shared(out, *args, gate=gate, out=out) is out and torch.equal(out, want)
    rows = rand(300, HQ, 128)
    for splits in (1, 4):
        args = kc, vc, table[:1].contiguous(), _i32([0]), _i32([300]), _i32([500]), 300
        want, out = a.prefill_spans(rows, *args, splits=splits), rows.clone()
        assert a.prefill_spans(out, *args, splits=splits, out=out) is out and torch.equal(out, want)


def test_caches_beyond_32_bit_offsets():
    """The last pages of caches of 2.3 G elements: append, prompt rows and a decoding row."""
    from deepseek_v4_2080ti_b200.ops import _lib
    a = _attention()
    torch.manual_seed(7)
    n_pages, n = 140000, 150
    kc = torch.zeros(n_pages, HKV, BS, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    assert kc.numel() > 2 ** 31
    last = [n_pages - 1, n_pages - 3, n_pages - 2]
    src = _src(n)
    slots = _i32([last[j // BS] * BS + j % BS for j in range(n)])
    layer = Layer(1)
    layer.kc, layer.vc = kc, vc
    positions = _i32(torch.arange(n).repeat(3, 1))
    q, gate = layer.append(src, positions, slots)
    layer.check_append(src, positions, slots, q)
    table = _i32([last])
    at = torch.arange(n, device=DEV)
    k, v = layer.keys(table[0], n)
    assert torch.equal(v, src[:, -HKV * 128:].view(n, HKV, 128))
    vc[last[1], 0, 3, 7] = math.inf                        # (rows that see it add it themselves, from its place in the cache)
    k, v = layer.keys(table[0], n)
    out = a.prefill_spans(q, kc, vc, table, _i32([0]), _i32([n]), _i32([n]), n, gate=gate)
    close(out, *oracle(q, k, v, torch.zeros_like(at), at + 1, 1 / math.sqrt(128), gate=gate))
    two = table.repeat(2, 1)
    out = a.decode_shared(q[-2:].contiguous(), kc, vc, two, _i32([n, n - 1]), _i32([0, 2]), _i32([64]))
    torch.cuda.synchronize()
    _lib.check_status()
    close(out, *oracle(q[-2:], k, v, _i32([0, 0]), _i32([n, n - 1]), 1 / math.sqrt(128)))


def test_tensors_off_their_alignment_are_refused():
    a = _attention()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)

    def off(*s, by=1):
        return torch.zeros(math.prod(s) + by, dtype=torch.bfloat16, device=DEV)[by:].view(*s)
    good = {"q": off(2, 4, 128, by=8), "k_cache": off(3, 2, 64, 128, by=8), "v_cache": off(3, 2, 64, 128, by=8), "block_table": i(2, 3), "kv_len": i(2)}
    for name, shape in (("q", (2, 4, 128)), ("k_cache", (3, 2, 64, 128)), ("v_cache", (3, 2, 64, 128)), ("gate", (2, 4, 128)), ("out", (2, 4, 128))):
        with pytest.raises(ValueError):
            a.prefill_spans(**good | {name: off(*shape)}, q_start=i(2), q_len=i(2), max_q_len=1)
        for groups in (0, 1):
            with pytest.raises(ValueError):
                a.decode_shared(**good | {name: off(*shape, by=4)}, group_start=i(groups + 1), shared_len=i(groups))
    src = off(2, 1024, by=4)
    rope = dict(q_src=src, q_off=0, q_head_stride=128, gate_in_q=False, k_src=src, k_off=512, v_src=src, v_off=768, q_gamma=off(128, by=4), k_gamma=None,
                unit_offset=True, eps=1e-6, inv_freq=torch.ones(16, device=DEV), axes=a.rotary_axes((8, 4, 4)), positions=i(3, 2), slots=i(2) - 1,
                k_cache=good["k_cache"], v_cache=good["v_cache"], n_q_heads=4, n_kv_heads=2)
    a.qk_norm_rope_axes_append(**rope)
    for change in ({"q_src": off(2, 1024)}, {"v_src": off(2, 1024, by=2)}, {"q_gamma": off(128)}, {"k_gamma": off(128, by=2)}, {"v_cache": off(3, 2, 64, 128)}):
        with pytest.raises(ValueError):
            a.qk_norm_rope_axes_append(**rope | change)
