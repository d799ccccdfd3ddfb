"""Drafted trees: attention of their rows, positions and masks, the accepted path; and the three of them as a decoder uses them.  Bounds of the
attention as in ``test_spans_gpu``; everything else is exact."""
import math
import random

import pytest
import torch

from test_spans_gpu import DEV, NAN, _i32, close, pages, rand

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


def _modules():
    from deepseek_v4_2080ti_b200.ops import _lib, attention, tree
    return _lib, attention, tree


def chain_of(parents, i):
    out = [i]
    while 0 <= parents[i] < i:
        i = parents[i]
        out.append(i)
    return out[::-1]


def random_tree(n, width, rng):
    return [-1] + [max(0, i - 1 - rng.randint(0, width)) for i in range(1, n)] if n else []


def bits(nodes, words):
    x = sum(1 << i for i in set(nodes))
    return [((x >> (32 * w) & 0xFFFFFFFF) + 2 ** 31) % 2 ** 32 - 2 ** 31 for w in range(words)]


def oracle(q, k, v, seen, cap=0.0, gate=None, scale=SCALE):
    """q [T, Hq, 128], k / v [n, Hkv, 128], seen [T, n] -> (result, bound)."""
    hq, hkv = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    mean = torch.zeros_like(out)
    for h in range(hq):
        kh, vh = k[:, h * hkv // hq].double(), v[:, h * hkv // hq].double()
        for a in range(0, q.shape[0], 64):
            see = seen[a:a + 64]
            s = torch.where(see[..., None], q[a:a + 64, h].double()[:, None] * torch.where(see[..., None], kh, 0.0), 0.0).sum(-1) * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            s = torch.where(see, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            l = torch.where(see.any(-1, keepdim=True), p.sum(-1, keepdim=True), 1.0)
            pv = torch.where(see[..., None], p[..., None] * vh[None], 0.0)
            out[a:a + 64, h] = pv.sum(1) / l
            mean[a:a + 64, h] = pv.abs().sum(1) / l
    g = 1.0 if gate is None else torch.sigmoid(gate.double())
    return out * g, (mean + out.abs()) * g * 2.0 ** -8 * (1 + 2.0 ** -4)


def run_tree(lens, hq, hkv, bs=64, width=2, cap=0.0, gate=False, splits=None, window=0, masks=None, words=None, poke=None, q_scale=1.5, scale=None):
    """``lens``: [(nodes, context)].  ``masks(i, node)`` -> nodes that a row sees (default: its ancestors and itself)."""
    lib, attention, _ = _modules()
    torch.manual_seed(sum(n * 3 + c for n, c in lens) + hq)
    rng = random.Random(len(lens) + lens[0][0])
    trees = [random_tree(n, width, rng) for n, _ in lens]
    see = masks or (lambda i, node: chain_of(trees[i], node))
    words = words or (max(n for n, _ in lens) + 31) // 32
    seqs = [(rand(n + c, hkv, 128), rand(n + c, hkv, 128)) for n, c in lens]
    if poke:
        poke(seqs)
    kc, vc, table = pages(seqs, bs)
    total = sum(n for n, _ in lens)
    q, g = rand(total, hq, 128, scale=q_scale), rand(total, hq, 128) if gate else None
    starts = [sum(n for n, _ in lens[:i]) for i in range(len(lens))]
    mask = _i32([bits(see(i, x), words) for i, (n, _) in enumerate(lens) for x in range(n)])
    depth = [len(chain_of(trees[i], x)) - 1 for i, (n, _) in enumerate(lens) for x in range(n)]
    lo = _i32([max(0, c + depth[starts[i] + x] + 1 - window) for i, (n, c) in enumerate(lens) for x in range(n)]) if window else None
    out = attention.decode_tree(q, kc, vc, table, mask, _i32(starts), _i32([n for n, _ in lens]), _i32([n + c for n, c in lens]),
                                max(n for n, _ in lens), lo=lo, gate=g, cap=cap, splits=splits, scale=scale, max_kv_len=max(n + c for n, c in lens))
    torch.cuda.synchronize()
    lib.check_status()
    for i, (n, c) in enumerate(lens):
        seen = torch.zeros(n, n + c, dtype=torch.bool)
        seen[:, :c] = True
        for x in range(n):
            seen[x, [c + y for y in see(i, x) if y < n]] = True
            if lo is not None:
                seen[x, :int(lo[starts[i] + x])] = False
        r = slice(starts[i], starts[i] + n)
        close(out[r], *oracle(q[r], *seqs[i], seen.to(DEV), cap, None if g is None else g[r], SCALE if scale is None else scale))
    return out


@pytest.mark.parametrize("lens,hq,hkv,bs", [
    ([(1, 0)], 1, 1, 64), ([(1, 128)], 5, 1, 16), ([(7, 350)], 40, 8, 64), ([(5, 1), (3, 127), (1, 129)], 4, 2, 32), ([(26, 600)], 10, 2, 64),
    ([(64, 65)], 8, 8, 128), ([(61, 300), (17, 31), (40, 700)], 6, 1, 256), ([(130, 126)], 2, 1, 64), ([(33, 95), (250, 40)], 4, 4, 16)])
@pytest.mark.parametrize("gate,cap", [(False, 0.0), (True, 6.0)])
def test_ancestors(lens, hq, hkv, bs, gate, cap):
    run_tree(lens, hq, hkv, bs, gate=gate, cap=cap)


@pytest.mark.parametrize("width", [0, 1, 40])
@pytest.mark.parametrize("splits", [1, 2, 5, 30])
def test_chains_wide_trees_and_keys_cut_into_items(width, splits):
    run_tree([(40, 700), (9, 1), (70, 1290)], 6, 2, width=width, splits=splits, gate=True)


@pytest.mark.parametrize("n", [31, 32, 33, 63, 65, 127, 129])
@pytest.mark.parametrize("context", [0, 1, 63, 64, 97, 128])
def test_trees_that_begin_anywhere_in_a_tile(n, context):
    run_tree([(n, context)], 2, 1, width=5)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_any_masks(splits, cap):
    """Rows that see no node, all of them, nodes behind them, more bits than there are nodes; without a context a row may see nothing."""
    rng = random.Random(5)
    pick = {}

    def masks(i, node):
        kind = (node + i) % 5
        return pick.setdefault((i, node), {0: [], 1: list(range(96)), 2: [95, 70]}.get(kind) or [x for x in range(96) if rng.random() < 0.3] * (kind > 2))
    out = run_tree([(50, 0), (70, 333), (20, 0)], 4, 2, masks=masks, words=3, splits=splits, cap=cap)
    assert bool((out[0] == 0).all()) and out.isfinite().all()


@pytest.mark.parametrize("cap", [0.0, 8.0])
def test_windows(cap):
    run_tree([(30, 900), (12, 100), (40, 513)], 4, 2, window=200, cap=cap, width=1)


def test_the_longest_tree():
    run_tree([(1024, 77)], 1, 1, width=3)


@pytest.mark.parametrize("splits", [1, 2])
def test_values_that_are_not_finite(splits):
    """A node's NaN and infinities reach those that continue it and no others; the context's reach everyone."""
    def poke(seqs):
        k, v = seqs[0]
        v[200 + 3, :, 5] = math.inf
        v[200 + 8, 0, 7] = NAN
        k[200 + 11, 1, :] = NAN
        seqs[1][1][4, :, 9] = NAN
        k[200 + 20, :, :] = math.inf
    run_tree([(30, 200), (4, 60)], 4, 2, width=3, poke=poke, splits=splits)


def test_scores_far_apart():
    def poke(seqs):
        seqs[0][0].mul_(torch.linspace(0.1, 6.0, seqs[0][0].shape[0], device=DEV)[:, None, None].bfloat16())
    run_tree([(60, 900)], 2, 1, q_scale=6.0, poke=poke)
    run_tree([(60, 900)], 2, 1, q_scale=6.0, poke=poke, cap=50.0)


def test_in_place_and_beside_the_rows():
    """Results over the queries, within a larger buffer; gates and a cap; nothing else is written."""
    lib, attention, tree = _modules()
    torch.manual_seed(9)
    k, v = rand(700, 2, 128), rand(700, 2, 128)
    kc, vc, table = pages([(k, v)], 32)
    parents = random_tree(45, 3, random.Random(1))
    args = (kc, vc, table, tree.layout(_i32(parents), _i32([0]), _i32([45]), _i32([700]), 45)[1], _i32([0]), _i32([45]), _i32([700]), 45)
    for splits in (1, 4):
        room = rand(60, 6, 128)
        gate, was = rand(45, 6, 128), room.clone()
        want = attention.decode_tree(room[7:52].clone(), *args, gate=gate, cap=9.0, splits=splits)
        q = room[7:52]
        assert attention.decode_tree(q, *args, gate=gate, cap=9.0, splits=splits, out=q) is q
        assert torch.equal(q, want) and torch.equal(room[:7], was[:7]) and torch.equal(room[52:], was[52:])
    lib.check_status()


def test_rows_of_no_sequence_stay_and_pages_that_are_not_there(monkeypatch):
    lib, attention, _ = _modules()
    torch.manual_seed(3)
    k, v = rand(300, 2, 128), rand(300, 2, 128)
    kc, vc, table = pages([(k, v)], 64, table_width=7)
    table[0, 5:] = -1                                      # behind the sequence
    q, mask = rand(50, 4, 128), _i32([[1 << i] for i in range(31)] + [[0]] * 19)
    seen = torch.zeros(20, 300, dtype=torch.bool, device=DEV)
    seen[:, :280] = True
    seen[torch.arange(20), 280 + torch.arange(20)] = True
    mask = torch.roll(mask, 10, 0)
    want, bound = oracle(q[10:30], k, v, seen)
    for debug in "01":
        monkeypatch.setenv("B200_BOUNDS_CHECK", debug)
        for splits in (1, 3):
            out = torch.full_like(q, 7.0)
            got = attention.decode_tree(q, kc, vc, table, mask, _i32([10]), _i32([20]), _i32([300]), 20, out=out, splits=splits)
            torch.cuda.synchronize()
            lib.check_status()
            assert got is out and bool((out[:10] == 7).all()) and bool((out[30:] == 7).all())
            close(out[10:30], want, bound)
    table[0, 2] = -1                                       # a page of the context: zeros, and a report in the debug mode
    k[128:192] = 0
    v[128:192] = 0
    monkeypatch.setenv("B200_BOUNDS_CHECK", "0")
    out = attention.decode_tree(q, kc, vc, table.clone(), mask, _i32([10]), _i32([20]), _i32([300]), 20)
    close(out[10:30], *oracle(q[10:30], k, v, seen))
    lib.check_status()
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    attention.decode_tree(q, kc, vc, table.clone(), mask, _i32([10]), _i32([20]), _i32([300]), 20)
    with pytest.raises(lib.KernelError):
        lib.check_status()


def test_a_captured_call_in_the_debug_mode(monkeypatch):
    lib, attention, _ = _modules()
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    torch.manual_seed(5)
    k, v = rand(300, 2, 128), rand(300, 2, 128)
    kc, vc, table = pages([(k, v)], 64)
    args = (rand(20, 4, 128), kc, vc, table, _i32([[1 << i] for i in range(20)]), _i32([0]), _i32([20]), _i32([300]), 20)
    want = attention.decode_tree(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention.decode_tree(*args)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    lib.check_status()
    assert torch.equal(got, want)


# ---------------------------------------------------------------- positions and masks
@pytest.mark.parametrize("sizes,width", [([1], 0), ([7], 2), ([61] * 40, 8), ([1, 0, 250, 33], 1), ([1024, 5], 0), ([64, 300, 2], 1000)])
def test_layout(sizes, width):
    lib, _, tree = _modules()
    rng = random.Random(sum(sizes))
    trees = [random_tree(n, width, rng) for n in sizes]
    starts, kv = [2 + sum(sizes[:i]) + 3 * i for i in range(len(sizes))], [n + rng.randint(0, 5000) for n in sizes]       # rows of nobody between them
    total = starts[-1] + sizes[-1] + 4
    words = (max(sizes) + 31) // 32
    parents, where, mask = [17] * total, [0] * total, [[0] * words for _ in range(total)]
    for s, n, t, k in zip(starts, sizes, trees, kv):
        for i in range(n):
            parents[s + i] = t[i]
            where[s + i] = k - n + len(chain_of(t, i)) - 1
            mask[s + i] = bits(chain_of(t, i), words)
    got = tree.layout(_i32(parents), _i32(starts), _i32(sizes), _i32(kv), max(sizes))
    assert got[0].tolist() == where and got[1].tolist() == mask


def test_layout_of_parents_that_make_no_tree():
    """A parent that does not lie before its child is the context: nothing turns in circles or leaves the batch."""
    _, _, tree = _modules()
    parents = [5, 1, 9, -7, 3, 2 ** 31 - 1, -2 ** 31, 6]
    where, mask = tree.layout(_i32(parents), _i32([0]), _i32([8]), _i32([108]), 8)
    assert where.tolist() == [100, 100, 100, 100, 101, 100, 100, 101]
    assert mask[:, 0].tolist() == [1, 2, 4, 8, 24, 32, 64, 192]
    where, mask = tree.layout(_i32(parents), _i32([-3, 6, 50]), _i32([5, 9, 9]), _i32([108, 20, 20]), 9)      # rows that are not there
    assert where.tolist() == [0] * 6 + [11, 11] and mask[:, 0].tolist() == [0] * 6 + [1, 2]


# ---------------------------------------------------------------- the accepted path
def accept_oracle(tokens, parents, predicted, most):
    path = [0] if tokens else []
    while path and len(path) < most:
        c = path[-1]
        child = [x for x in range(c + 1, len(tokens)) if parents[x] == c and tokens[x] == predicted[c] >= 0]
        if not child:
            break
        path.append(child[0])
    return path


@pytest.mark.parametrize("sizes,width,most", [([1], 0, 1), ([7], 2, 8), ([61, 1, 0, 40, 64], 6, 9), ([30] * 70, 1, 40), ([300, 20], 0, 256), ([1024], 3, 5)])
@pytest.mark.parametrize("bs,layers,heads", [(16, 1, 1), (64, 3, 4)])
def test_accept(sizes, width, most, bs, layers, heads):
    lib, _, tree = _modules()
    rng = random.Random(sum(sizes) + most)
    trees = [random_tree(n, width, rng) for n in sizes]
    tokens = [[rng.randint(0, 3) for _ in range(n)] for n in sizes]            # (few tokens: siblings that hold the same one)
    predicted = []
    for t, n in zip(trees, sizes):
        p = [rng.randint(0, 3) for _ in range(n)]
        for i in range(1, n):
            if rng.random() < 0.9:
                p[t[i]] = tokens[len(predicted)][i]
        predicted.append(p)
    starts, contexts = [sum(sizes[:i]) + i for i in range(len(sizes))], [rng.randint(0, 150) for _ in sizes]
    flat = lambda x: _i32([y for row in x for y in row + [0]])
    counts = [-(-(c + n) // bs) for c, n in zip(contexts, sizes)]
    nb = sum(counts) + 1
    order = list(range(nb))
    rng.shuffle(order)
    table = torch.full((len(sizes), max(counts + [1])), -1, dtype=torch.int32)
    for i, c in enumerate(counts):
        table[i, :c] = torch.tensor(order[sum(counts[:i]):sum(counts[:i + 1])], dtype=torch.int32)
    k = torch.randn(layers, nb, heads, bs, 128, device=DEV).bfloat16()
    scale = torch.randn(layers, nb, heads, bs, device=DEV)
    codes = torch.randint(0, 255, (2 * layers, nb, 2 * heads, bs, 64), device=DEV, dtype=torch.uint8)[::2]     # layers apart, other heads
    odd = torch.randint(0, 255, (1, nb, 1, bs, 20), device=DEV, dtype=torch.uint8)
    room = torch.randn(layers + 2, nb, heads, bs, 128, device=DEV).bfloat16()                                # layers of a larger cache
    caches = [k, k.flip(0).contiguous(), scale, codes, odd, room[1:-1]]
    beside = [(codes._base[1::2], codes._base[1::2].clone()), (room[0], room[0].clone()), (room[-1], room[-1].clone())]
    wanted = [c.clone() for c in caches]
    paths = [accept_oracle(tokens[i], trees[i], predicted[i], most) for i in range(len(sizes))]
    for b, path in enumerate(paths):
        for i, node in enumerate(path):
            src, dst = contexts[b] + node, contexts[b] + i
            for c, w in zip(caches, wanted):
                w[:, table[b, dst // bs], :, dst % bs] = c[:, table[b, src // bs], :, src % bs]
    path, count, emitted = tree.accept(flat(tokens), flat(trees), flat(predicted), _i32(starts), _i32(sizes), most,
                                       _i32([c + n for c, n in zip(contexts, sizes)]), table.to(DEV), caches)
    torch.cuda.synchronize()
    assert count.tolist() == [len(p) for p in paths]
    assert path.tolist() == [p + [-1] * (most - len(p)) for p in paths]
    assert emitted.tolist() == [[predicted[b][x] for x in p] + [-1] * (most - len(p)) for b, p in enumerate(paths)]
    for c, w in [*zip(caches, wanted), *beside]:
        assert torch.equal(c, w)
    alone = tree.accept(flat(tokens), flat(trees), flat(predicted), _i32(starts), _i32(sizes), most)
    assert all(torch.equal(x, y) for x, y in zip(alone, (path, count, emitted)))


def test_accept_of_what_makes_no_tree():
    """Negative tokens and predictions agree with nothing, parents that do not lie before their child have no children; pages that are not there
    keep their rows."""
    _, _, tree = _modules()
    path, count, emitted = tree.accept(_i32([4, -1, 4, 4]), _i32([-1, 0, 3, 0]), _i32([-1, 4, 4, 4]), _i32([0]), _i32([4]), 4)
    assert path.tolist() == [[0, -1, -1, -1]] and count.tolist() == [1] and emitted.tolist() == [[-1, -1, -1, -1]]
    tokens, parents, predicted = _i32([9, 1, 2, 3, 2]), _i32([-1, 0, 0, 0, 3]), _i32([3, 0, 0, 2, 8])
    cache = torch.arange(6 * 16, device=DEV, dtype=torch.float32).view(1, 6, 1, 16).clone()
    was = cache.clone()
    for table in ([[-1]], [[6]], [[2 ** 30]]):
        out = tree.accept(tokens, parents, predicted, _i32([0]), _i32([5]), 4, _i32([10]), _i32(table), [cache])
        assert out[0].tolist() == [[0, 3, 4, -1]] and out[2].tolist() == [[3, 2, 8, -1]] and torch.equal(cache, was)
    tree.accept(tokens, parents, predicted, _i32([0]), _i32([5]), 4, _i32([2]), _i32([[0]]), [cache])            # fewer keys than nodes
    assert torch.equal(cache, was)
    out = tree.accept(tokens, parents, predicted, _i32([0, -2, 3, 7]), _i32([5, 3, 9, 2]), 4)                    # rows that are not there
    assert out[1].tolist() == [3, 0, 1, 0]


# ---------------------------------------------------------------- together
def test_a_step_of_a_decoder_with_a_drafted_tree():
    """Keys and values of a tree's nodes appended in the tree's order, attended to, the accepted path kept: the cache is then the one of a decoder
    that has seen the accepted tokens one after the other, and so is the last node's attention."""
    lib, attention, tree = _modules()
    torch.manual_seed(8)
    layers, hq, hkv, bs, context, vocab = 2, 10, 2, 16, 75, 50
    emb_k, emb_v = rand(layers, vocab, hkv, 128), rand(layers, vocab, hkv, 128)
    emb_q = rand(vocab, hq, 128)
    prompt = torch.randint(0, vocab, (context,), device=DEV)
    tokens = [11, 7, 3, 7, 20, 21, 3, 40]
    parents = [-1, 0, 0, 1, 1, 3, 3, 6]
    accepted = [0, 1, 3, 6]                                 # 11 7 7 3
    predicted = [7, 7, 0, 3, 0, 0, 9, 0]
    n, nb = len(tokens), 9
    table = _i32([[4, 8, 0, 2, 7, 1]])
    k, v = (torch.zeros(layers, nb, hkv, bs, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def append(where, toks):
        where, toks = torch.as_tensor(where, device=DEV), torch.as_tensor(toks, device=DEV)
        for c, e in ((k, emb_k), (v, emb_v)):
            c[:, table[0, where // bs].long(), :, where % bs] = e[:, toks].transpose(0, 1)
    append(torch.arange(context), prompt)
    where, mask = tree.layout(_i32(parents), _i32([0]), _i32([n]), _i32([context + n]), n)
    assert where.tolist() == [context + len(chain_of(parents, i)) - 1 for i in range(n)]
    append(torch.arange(context, context + n), tokens)
    rows = attention.decode_tree(emb_q[torch.tensor(tokens)].contiguous(), k[1], v[1], table, mask, _i32([0]), _i32([n]), _i32([context + n]), n)
    path, count, emitted = tree.accept(_i32(tokens), _i32(parents), _i32(predicted), _i32([0]), _i32([n]), 6, _i32([context + n]), table, [k, v])
    assert path.tolist() == [accepted + [-1, -1]] and count.tolist() == [4] and emitted.tolist() == [[7, 7, 3, 9, -1, -1]]
    kept = [c.clone() for c in (k, v)]
    append(torch.arange(context, context + 4), [11, 7, 7, 3])                  # as without drafts
    assert torch.equal(k, kept[0]) and torch.equal(v, kept[1])
    ids = torch.cat([prompt, torch.tensor([11, 7, 7, 3], device=DEV)])
    seen = torch.tril(torch.ones(4, context + 4, dtype=torch.bool, device=DEV), context)
    want, bound = oracle(emb_q[ids[-4:]], emb_k[1, ids], emb_v[1, ids], seen)
    close(rows[torch.tensor(accepted)], want, bound)
    lib.check_status()


def test_captured_steps_and_two_streams():
    """One graph of the three calls, replayed on other trees, beside the same calls on another stream."""
    _, attention, tree = _modules()
    torch.manual_seed(2)
    rng = random.Random(2)
    b, n, hq, hkv, bs, nb = 3, 20, 8, 2, 32, 40
    k, v = rand(1, nb, hkv, bs, 128), rand(1, nb, hkv, bs, 128)
    first = k.clone(), v.clone()
    table = torch.randperm(nb, device=DEV)[:b * 10].view(b, 10).int()
    start, size = _i32([0, n, 2 * n]), _i32([n] * b)

    def inputs():
        sizes = [rng.randint(1, n) for _ in range(b)]
        trees = [random_tree(n, 2, rng) for _ in range(b)]
        return (_i32([x for t in trees for x in t]), _i32(sizes), _i32([s + rng.randint(0, 250) for s in sizes]),
                torch.randint(0, 3, (b * n,), device=DEV).int(), torch.randint(0, 3, (b * n,), device=DEV).int(), rand(b * n, hq, 128))
    fixed = inputs()

    def step(x, caches, splits=None):
        parents, lens, kv, tokens, predicted, q = x
        where, mask = tree.layout(parents, start, lens, kv, n)
        out = attention.decode_tree(q, caches[0][0], caches[1][0], table, mask, start, lens, kv, n, out=torch.zeros_like(q), splits=splits)
        return (where, mask, out, *tree.accept(tokens, parents, predicted, start, lens, 6, kv, table, caches))
    for splits in (1, 4):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(fixed, [k, v], splits)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(fixed, [k, v], splits)
        for _ in range(4):
            new = inputs()
            for x, y in zip(fixed, new):
                x.copy_(y)
            k.copy_(first[0])
            v.copy_(first[1])
            mine = [c.clone() for c in first]
            torch.cuda.synchronize()
            graph.replay()
            with torch.cuda.stream(side):
                want = step(new, mine, splits)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
            assert torch.equal(k, mine[0]) and torch.equal(v, mine[1])
