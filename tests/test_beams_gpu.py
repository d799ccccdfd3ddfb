"""Beam search: the selection over beams and vocabulary, and states that follow the beams, against plain statements in 64 bits.

Bound of the scores: one rounding to 32 bits (2^-24 of the value) of a total that is off by as much as the logarithm of a sum of exponentials in 32
bits.  2^t with t = x log2 e - k: t is rounded (2^-24 of it) and log2 e is (2^-26 of it); sum p |t| is log2 V + 1 at most (p = 2^t / sum, whose entropy is
log2 V at most); the exponentials are off by 2^-22, three sums of four terms by 2^-24 each.  Parents, tokens and moved states are exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def oracle(logits, scores, n, finished=None, pad=0):
    b, w, v = logits.shape
    out = torch.full((b, n), -math.inf, dtype=torch.float64, device=DEV)
    parents, tokens = _i32([[-1] * n] * b), _i32([[-1] * n] * b)
    for r in range(b):
        total = scores[r].double()[:, None] + torch.log_softmax(logits[r].double(), -1)
        dead = ~scores[r].isfinite() | (logits[r].double().amax(-1) == math.inf)
        total = torch.where(dead[:, None] | total.isnan(), -math.inf, total)
        if finished is not None:
            total[finished[r]] = -math.inf
            total[finished[r], pad] = torch.where(dead & ~scores[r].isfinite(), -math.inf, scores[r].double())[finished[r]]
        x, order = total.reshape(-1).sort(descending=True, stable=True)
        m = min(n, int((x > -math.inf).sum()))
        out[r, :m], parents[r, :m], tokens[r, :m] = x[:m], (order[:m] // v).int(), (order[:m] % v).int()
    return out, parents, tokens


def check(logits, scores, n=None, finished=None, pad=0):
    from deepseek_v4_2080ti_b200.ops import beams
    got = beams.select(logits, scores, n, finished, pad)
    want = oracle(logits, scores, scores.shape[1] if n is None else n, finished, pad)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    fine = want[0].isfinite()
    assert torch.equal(fine, got[0].isfinite()) and bool((got[0][~fine] == -math.inf).all())
    off = (got[0].double() - want[0]).abs()[fine]
    assert bool((off <= want[0].abs()[fine] * 2.0 ** -24 + 2.0 ** -22 + 3 * 2.0 ** -24 + (math.log2(logits.shape[-1]) + 1) * math.log(2) * (2.0 ** -24 + 2.0 ** -26)).all()), off.max()
    return got


def random_logits(b, w, v, dtype=torch.float32, seed=0, scale=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed + b * 7 + w * 3 + v)
    return (torch.randn(b, w, v, generator=g, device=DEV) * scale).to(dtype), -torch.rand(b, w, generator=g, device=DEV) * 8


@pytest.mark.parametrize("v", [1, 2, 31, 32, 33, 1000, 8191, 8192, 8193, 16388, 51001, 248320])
@pytest.mark.parametrize("b,w,n", [(1, 1, 1), (1, 4, 8), (3, 5, 7), (2, 16, 16)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(b, w, v, n, dtype):
    check(*random_logits(b, w, v, dtype), n)


@pytest.mark.parametrize("b,w,n", [(1, 128, 128), (40, 3, 1), (2, 1, 128), (1, 33, 100), (7, 12, 64), (700, 4, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_beams_and_candidates(b, w, n, dtype):
    check(*random_logits(b, w, 9001, dtype), n)


@pytest.mark.parametrize("n", [1, 16, 128])
@pytest.mark.parametrize("level", [0.0, -0.0, 3.25, -3.4028234663852886e38, 1e30, 40000.0])
def test_ties(n, level):
    """Equal logits, in whole rows and in some beams only, equal beams: the lowest beam and token first."""
    for w, v in ((1, 300), (3, 20000), (20, 9000), (128, 8200)):
        logits = torch.full((2, w, v), level, device=DEV)
        scores = torch.zeros(2, w, device=DEV) - 1
        check(logits, scores, n)
        logits[:, ::2, 5:v // 2] = -math.inf
        logits[1, -1, ::3] = -math.inf
        check(logits, scores, n)
    logits, _ = random_logits(2, 6, 30000, torch.bfloat16, scale=0.3)
    logits[:, 3] = logits[:, 1]
    check(logits, torch.zeros(2, 6, device=DEV), n)
    coarse = (logits.float() * 2).round()
    check(coarse, torch.zeros(2, 6, device=DEV), n)
    check(torch.where(coarse == 0, -0.0, coarse), torch.zeros(2, 6, device=DEV), n)


@pytest.mark.parametrize("order", ["rising", "falling", "steps"])
@pytest.mark.parametrize("n", [3, 128])
def test_orders_in_memory(order, n):
    x = torch.linspace(-20, 20, 100000, device=DEV)
    x = {"rising": x, "falling": x.flip(0), "steps": (x * 4).floor()}[order]
    check(x.expand(2, 3, -1).contiguous(), torch.tensor([[0.0, -1e-9, -30], [-2, -2, -2]], device=DEV), n)


def test_allowed_tokens_only():
    """Constrained decoding: all other tokens at -inf, or at the type's lowest value; fewer allowed ones than candidates."""
    logits, scores = random_logits(3, 4, 40001)
    keep = torch.zeros_like(logits, dtype=torch.bool)
    keep[..., [0, 77, 8192, 40000]] = True
    keep[1, 2] = False
    for fill in (-math.inf, torch.finfo(torch.float32).min):
        check(torch.where(keep, logits, fill), scores, 8)
        check(torch.where(keep, logits, fill), scores, 40)
    check(torch.where(keep, logits, torch.finfo(torch.bfloat16).min).bfloat16(), scores, 40)
    mixed = torch.where(keep, logits, torch.finfo(torch.float32).min)
    mixed[..., ::2] = -math.inf
    check(mixed, scores, 40)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_finished_beams_and_beams_that_have_come_to_nothing(dtype):
    logits, scores = random_logits(6, 5, 3001, dtype)
    finished = torch.zeros(6, 5, dtype=torch.bool, device=DEV)
    finished[0, 2] = finished[1, :] = finished[2, 0] = finished[4, 1] = True
    scores[3, 1:] = -math.inf
    scores[2, 0] = 0.0
    scores[4, 1] = -math.inf                               # at its end and nothing worth
    scores[5] = -math.inf
    logits[1] = NAN                                        # rows that nobody looks at
    logits[3, 2] = NAN
    check(logits, scores, 5, finished, 2)
    check(logits, scores, 11, finished, 3000)
    scores[0, 1], scores[0, 3], scores[0, 4] = NAN, math.inf, -math.inf
    check(logits, scores, 11, finished, 0)


def test_rows_that_are_not_finite():
    """NaN or +inf among the logits: the beam offers nothing, the others are as without it."""
    logits, scores = random_logits(4, 4, 20001)
    logits[0, 1, 19999] = NAN
    logits[1, 0, 3] = math.inf
    logits[1, 2, 8192] = math.inf
    logits[2, 3] = -math.inf
    logits[3, 0, 5], logits[3, 1, 20000], logits[3, 2, 100], logits[3, 3, 0] = NAN, math.inf, NAN, math.inf
    check(logits, scores, 8)


def test_large_logits_and_scores():
    logits, scores = random_logits(4, 4, 12345)
    check(logits * 1e3, scores, 16)
    check(logits * 1e6 + 1e7, scores, 16)
    check(logits * 1e30, scores, 16)
    check(logits + 32768 * 2, scores * 1e6, 16)
    check(logits * 1e-3 - 70000, scores * 1e-6, 16)
    logits[:, ::2] += 1e5                                  # rows far from one another
    check(logits, scores, 16)


def test_candidates_closer_than_32_bits():
    """Beams whose totals differ by less than sums in 32 bits are off."""
    logits, _ = random_logits(1, 1, 30000)
    logits = logits.expand(8, 12, -1).contiguous()
    logits[:, :, 1:20000] = logits[:, :, 1:20000].flip(-1)
    perm = torch.stack([torch.randperm(30000, device=DEV) for _ in range(12)])
    shuffled = torch.stack([logits[0, i][perm[i]] for i in range(12)])[None].expand(8, -1, -1).contiguous()
    scores = (-torch.arange(12, device=DEV) * 2.0 ** -22).expand(8, 12).contiguous() - 3
    check(shuffled, scores, 100)


def test_a_long_row():
    """More tiles than parts, offsets beyond 32 bits of bytes."""
    from deepseek_v4_2080ti_b200.ops import beams
    v = (1 << 29) + (1 << 28)
    big = torch.full((2, v), -8.0, dtype=torch.bfloat16, device=DEV)
    at = [5, 8191, 8192, 1 << 28, (1 << 29) - 1]
    for i, t in enumerate(at):
        big[1, t] = 10 - i
    row = big[1:2, :1 << 29][None]
    score, parents, tokens = beams.select(row, torch.zeros(1, 1, device=DEV), 7)
    others = [t for t in range(7) if t not in at][:2]
    assert tokens.tolist() == [at + others] and parents.tolist() == [[0] * 7]
    z = math.log(sum(math.exp(10 - i) for i in range(5)) + ((1 << 29) - 5) * math.exp(-8))
    assert all(abs(x - (l - z)) < 1e-5 * abs(l - z) + 1e-6 for x, l in zip(score[0].tolist(), [10, 9, 8, 7, 6, -8, -8]))
    with pytest.raises(ValueError):
        beams.select(big[None], torch.zeros(1, 2, device=DEV))


def test_strides():
    """Rows of a longer buffer, a slice of the vocabulary off 16 bytes, one beam of several."""
    base, scores = random_logits(3, 4, 5000)
    for view in (base[..., :4001], base[..., 1:4097], base[..., 8:4008], base.bfloat16()[..., 8:4008], base.bfloat16()[..., 3:]):
        check(view, scores, 9)
    check(base[:, 2:3, :], scores[:, 2:3].contiguous(), 4)
    check(base[1:2, :, :], scores[1:2], 4)


def test_captured_and_on_two_streams():
    from deepseek_v4_2080ti_b200.ops import beams
    logits, scores = random_logits(4, 6, 33333)
    fixed, s = logits.clone(), scores.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        beams.select(fixed, s, 12)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beams.select(fixed, s, 12)
    for seed in range(3):
        x, y = random_logits(4, 6, 33333, seed=seed)
        fixed.copy_(x)
        s.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = beams.select(x, y, 12)
        torch.cuda.synchronize()
        want = oracle(x, y, 12)
        for r in (got, other):
            assert torch.equal(r[1], want[1]) and torch.equal(r[2], want[2])


# ---------------------------------------------------------------- states
def moved(x, parents, slots, dim):
    w = parents.shape[1]
    y = x.clone()
    for row, s in zip(parents.tolist(), slots.tolist()):
        for i, p in enumerate(row):
            if 0 <= p < w and 0 <= s[i] < x.shape[dim] and 0 <= s[p] < x.shape[dim]:
                y.select(dim, s[i]).copy_(x.select(dim, s[p]))
    return y


def check_reorder(states, parents, slots=None, dim=0):
    from deepseek_v4_2080ti_b200.ops import _lib, beams
    b, w = parents.shape
    where = slots if slots is not None else torch.arange(b * w, device=DEV).view(b, w)
    want = [moved(x, parents, where, dim) for x in states]
    beams.reorder(states, parents, slots, dim)
    torch.cuda.synchronize()
    _lib.check_status()
    assert all(torch.equal(x, y) for x, y in zip(states, want))


def filled(*shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV).to(dtype) if dtype.is_floating_point else torch.randint(0, 200, shape, device=DEV).to(dtype)


@pytest.mark.parametrize("b,w", [(1, 1), (1, 2), (3, 4), (2, 31), (1, 33), (2, 100), (1, 128)])
@pytest.mark.parametrize("inner", [4, 1000, 4096, 70004])
def test_reorder(b, w, inner):
    g = torch.Generator(device=DEV).manual_seed(b + w + inner)
    parents = torch.randint(-1, w, (b, w), generator=g, device=DEV).int()
    slots = torch.randperm(b * w + 3, generator=g, device=DEV)[:b * w].view(b, w).int()
    check_reorder([filled(b * w + 3, inner), filled(b * w + 3, 3, 8, dtype=torch.bfloat16)], parents, slots)
    check_reorder([filled(b * w + 3, inner)], parents)


@pytest.mark.parametrize("kind", ["cycle", "swap", "chain", "one", "own"])
def test_parents_of_every_shape(kind):
    w = 16
    i = torch.arange(w, device=DEV)
    parents = {"cycle": (i + 1) % w, "swap": i ^ 1, "chain": (i - 1).clamp(min=0), "one": torch.full_like(i, 7), "own": i}[kind]
    check_reorder([filled(2 * w, 5, 64, 33), filled(2 * w, 7, dtype=torch.uint8)], parents.expand(2, w).int().contiguous())


def test_axes_types_and_strides():
    parents, slots = _i32([[2, 0, 0], [1, 1, -1]]), _i32([[5, 1, 3], [0, 6, 2]])
    check_reorder([filled(4, 9, 2, 16, 128, dtype=torch.bfloat16), filled(4, 9, 3, dtype=torch.int32), filled(2, 9, 5, dtype=torch.uint8),
                   filled(3, 9, 1, dtype=torch.float64), filled(1, 9, dtype=torch.int16)], parents, slots, 1)
    wide = filled(9, 6, 64)
    kept = wide[:, 4:].clone()
    check_reorder([wide[:, :4]], parents, slots)           # one layer's share of longer slots
    assert torch.equal(wide[:, 4:], kept)
    layers = filled(8, 9, 64)
    kept = layers[1::2].clone()
    check_reorder([layers[::2]], parents, slots, 1)
    assert torch.equal(layers[1::2], kept)
    check_reorder([filled(9, 24, dtype=torch.uint8)[:, 1:]], parents, slots)
    check_reorder([filled(9, 64) for _ in range(35)], parents, slots)          # more tensors than a launch takes


def test_slots_that_are_not_there():
    parents = _i32([[1, 2, 0, 1]])
    check_reorder([filled(6, 100), filled(6, 3, dtype=torch.uint8)], parents, _i32([[0, 9, 2, 3]]))
    check_reorder([filled(6, 100), filled(6, 3, dtype=torch.uint8)], parents, _i32([[-1, 4, 2, 2 ** 31 - 1]]))
    check_reorder([filled(6, 100)], _i32([[7, -5, 0, 2 ** 31 - 1]]), _i32([[5, 4, 3, 2]]))


def test_debug_mode_leaves_slots_that_are_not_there_alone(monkeypatch):
    from deepseek_v4_2080ti_b200.ops import _lib, beams
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    check_reorder([filled(6, 100)], _i32([[1, 2, 0, 1]]), _i32([[0, -1, 2, 3]]))              # idle ones are no error
    x = filled(6, 100)
    want = moved(x, _i32([[1, 0, 0, 2]]), _i32([[0, 6, 2, 3]]), 0)
    beams.reorder(x, _i32([[1, 0, 0, 2]]), _i32([[0, 6, 2, 3]]))
    with pytest.raises(_lib.KernelError):
        _lib.check_status()
    assert torch.equal(x, want)


def test_nothing_beside_the_states_is_touched():
    """Slots within a larger buffer: what lies before, between and behind them stays, for copies of 16 bytes and of one."""
    parents = _i32([[3, 0, 1, 1, 4, 2]])
    for width, dtype in ((4096, torch.float32), (70000, torch.uint8), (333, torch.bfloat16)):
        room = filled(3, 10, width + 64, dtype=dtype)
        for a, b in ((0, width), (16, width + 16), (64, width + 64)):
            was = room.clone()
            check_reorder([room[:, 2:8, a:b]], parents, dim=1)
            was[:, 2:8, a:b] = room[:, 2:8, a:b]
            assert torch.equal(room, was)


@pytest.mark.parametrize("n", [1, 5, 128])
def test_many_steps_of_one_search(n):
    """The same inputs give the same answer every time, whatever ran before and beside it."""
    from deepseek_v4_2080ti_b200.ops import beams
    x, y = random_logits(5, 7, 20011, torch.bfloat16)
    first = beams.select(x, y, n)
    for i in range(30):
        beams.select(*random_logits(1 + i % 3, 4, 9000, seed=i), 3 + i)
        assert all(torch.equal(a, b) for a, b in zip(first, beams.select(x, y, n)))


def test_large_states():
    """Offsets beyond 32 bits, more items than blocks."""
    x = torch.empty(10, 260 << 20, dtype=torch.int16, device=DEV)
    for i in range(10):
        x[i] = i
    from deepseek_v4_2080ti_b200.ops import beams
    beams.reorder(x, _i32([[1, 0, 0, 2, 9, 4, 5, 7, 7, 3]]))
    want = [1, 0, 0, 2, 9, 4, 5, 7, 7, 3]
    assert all(bool((x[i] == want[i]).all()) for i in range(10))


@pytest.mark.parametrize("v", [1, 2, 33, 9000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forced_tokens_of_beams_with_equal_scores(v, dtype):
    """One token allowed: a beam's total is its score, whatever the logit, so that beams of equal scores - ended ones among them - are equal."""
    g = torch.Generator(device=DEV).manual_seed(v)
    logits, _ = random_logits(40, 6, v, dtype)
    keep = torch.randint(0, v, (40, 6, 1), generator=g, device=DEV)
    logits = torch.full_like(logits, -math.inf).scatter_(2, keep, logits.gather(2, keep))
    logits[30:] *= 20000.0
    scores = -torch.randint(0, 3, (40, 6), generator=g, device=DEV).float() / 3
    finished = torch.rand(40, 6, generator=g, device=DEV) < 0.3
    for n in (1, 4, 9):
        check(logits, scores, n)
        check(logits, scores, n, finished, v // 2)


def test_the_last_place_between_more_candidates_of_one_beam():
    """Behind beam 1's best lie the two best of beam 0, 2^-29 apart, and beam 1's second, 2^-28 above both: whether sums in 32 bits see it above,
    between or below them, it is the second (sums to 2^-30 do see it)."""
    g = torch.Generator(device=DEV).manual_seed(31)
    b, v = 512, 200
    logits = -torch.rand(b, 2, v, generator=g, device=DEV)
    logits[:, :, 40] = 0.02
    logits[:, 0, 50] = torch.nextafter(torch.tensor(0.02), torch.tensor(0.0)).item()
    logits[:, 1, 90] = 1.0
    best = torch.log_softmax(logits.double(), -1)[:, :, 40]
    scores = torch.stack([torch.zeros(b, device=DEV), (best[:, 0] - best[:, 1] + 2.0 ** -28).float()], 1)
    for n in (2, 3, 4):
        parents, tokens = check(logits, scores, n)[1:]
        assert bool((parents[:, :2] == 1).all() and (tokens[:, 1] == 40).all())


# ---------------------------------------------------------------- together
def test_beam_search_finds_what_an_exhaustive_search_of_the_beams_finds():
    """Three steps of a search whose model is a recurrent state: the states follow the beams, so that the scores are those of whole sequences."""
    from deepseek_v4_2080ti_b200.ops import beams
    g = torch.Generator(device=DEV).manual_seed(4)
    b, w, v, d = 3, 5, 700, 64
    emb, head, mix = (torch.randn(*s, generator=g, device=DEV) for s in ((v, d), (d, v), (d, d)))
    mix /= math.sqrt(d)
    advance = lambda state, token: torch.tanh(state @ mix + emb[token])
    slots = torch.randperm(b * w, generator=g, device=DEV).view(b, w).int()
    states = torch.zeros(b * w, d, device=DEV)
    states[slots.long()] = advance(torch.zeros(b, 1, d, device=DEV), torch.randint(0, v, (b, 1), generator=g, device=DEV)).expand(b, w, d)
    start = states[slots[:, 0].long()].clone()
    scores = torch.full((b, w), -math.inf, device=DEV)
    scores[:, 0] = 0
    history = torch.zeros(b * w, 3, dtype=torch.int32, device=DEV)
    for step in range(3):
        scores, parents, tokens = beams.select(states[slots.long()] @ head, scores)
        beams.reorder([states, history], parents, slots)
        history[slots.reshape(-1).long(), step] = tokens.reshape(-1)
        states[slots.long()] = advance(states[slots.long()], tokens.long())
    # every beam's tokens, from the start on
    for r in range(b):
        assert len({tuple(history[slots[r, i]].tolist()) for i in range(w)}) == w
        for i in range(w):
            state, total = start[r], 0.0
            for t in history[slots[r, i].long()].long():
                total += torch.log_softmax((state[None] @ head)[0].double(), -1)[t].item()
                state = advance(state[None], t[None])[0]
            assert abs(total - scores[r, i].item()) < 1e-3 and torch.allclose(state, states[slots[r, i].long()], atol=1e-4)
