"""Faults of the calls over drafted trees and beams that were found after they had run, each with the test that shows it."""
import math
import random

import pytest
import torch

from test_beams_gpu import check, random_logits
from test_spans_gpu import DEV, _i32, close, pages, rand
from test_trees_gpu import bits, chain_of, oracle, random_tree

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- key ranges of tree attention
def tree_inputs(lens, hq, hkv, bs=64, wide=None, window=0, seed=0):
    """``lens``: [(nodes, context)].  (arguments of ``decode_tree`` up to max_q_len, lo, (sequences, rows' sets of keys))."""
    torch.manual_seed(seed + sum(n + c for n, c in lens))
    rng = random.Random(seed)
    seqs = [(rand(n + c, hkv, 128), rand(n + c, hkv, 128)) for n, c in lens]
    kc, vc, table = pages(seqs, bs, table_width=wide)
    total, most = sum(n for n, _ in lens), max(n for n, _ in lens)
    starts = [sum(n for n, _ in lens[:i]) for i in range(len(lens))]
    mask, lo, seen = [], [], []
    for n, c in lens:
        parents = random_tree(n, 3, rng)
        see = torch.zeros(n, n + c, dtype=torch.bool)
        see[:, :c] = True
        for x in range(n):
            chain = chain_of(parents, x)
            mask.append(bits(chain, (most + 31) // 32))
            lo.append(max(0, c + len(chain) - window) if window else 0)
            see[x, [c + y for y in chain]] = True
            see[x, :lo[-1]] = False
        seen.append(see.to(DEV))
    q = rand(total, hq, 128, scale=1.5)
    args = (q, kc, vc, table, _i32(mask), _i32(starts), _i32([n for n, _ in lens]), _i32([n + c for n, c in lens]), most)
    return args, _i32(lo) if window else None, (seqs, seen, starts)


@pytest.mark.parametrize("lens,window", [([(16, 4000)], 0), ([(9, 700), (30, 2500), (4, 60)], 0), ([(16, 9000)], 1000), ([(12, 5000), (7, 3)], 300)])
def test_key_ranges_follow_the_keys_and_not_the_bound(lens, window):
    """A row tile's keys are cut into ``splits`` items by how many there are, so that a bound that is far above them - a captured step's, the
    table's - leaves the work where it is: the same bits as with the longest context itself."""
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    args, lo, (seqs, seen, starts) = tree_inputs(lens, 10, 2, wide=512, window=window)
    most = max(n + c for n, c in lens)
    for splits in (2, 6, 18):
        outs = [attention.decode_tree(*args, lo=lo, splits=splits, max_kv_len=bound) for bound in (most, 4 * most, 131072, None)]
        assert all(torch.equal(x, outs[0]) for x in outs[1:])
        for i, (n, _) in enumerate(lens):
            r = slice(starts[i], starts[i] + n)
            close(outs[0][r], *oracle(args[0][r], *seqs[i], seen[i]))
    outs = [attention.decode_tree(*args, lo=lo, max_kv_len=bound) for bound in (131072, None)]      # and as many items as either bound gives
    for i, (n, _) in enumerate(lens):
        r = slice(starts[i], starts[i] + n)
        for x in outs:
            close(x[r], *oracle(args[0][r], *seqs[i], seen[i]))
    _lib.check_status()


def test_a_captured_step_is_cut_as_the_contexts_that_it_meets():
    """One graph for contexts of 40 to 7000 keys: at every replay the bits of a call that knows the longest of them."""
    from deepseek_v4_2080ti_b200.ops import attention
    args, _, _ = tree_inputs([(16, 7000), (16, 5000)], 10, 2)
    kv = args[7].clone()
    call = lambda bound: attention.decode_tree(*args[:7], kv, 16, splits=9, max_kv_len=bound)
    call(7016)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(None)
    for lens in ([7016, 5016], [1500, 40], [56, 3000], [16, 16]):
        kv.copy_(_i32(lens))
        graph.replay()
        want = call(max(lens))
        torch.cuda.synchronize()
        assert torch.equal(got, want)


# ---------------------------------------------------------------- what lets candidates into the join of beam selection
def alone(logits, scores, w, n):
    """The selection over one beam of every request: the scores that sums of the first pass give."""
    from deepseek_v4_2080ti_b200.ops import beams
    return beams.select(logits[:, w:w + 1], scores[:, w:w + 1].contiguous(), n)


@pytest.mark.parametrize("w,n", [(8, 64), (20, 40), (4, 128), (13, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_first_step_of_a_search(w, n, dtype):
    """One beam of several offers tokens, as at a search's first step: its candidates are picked from its own lists, and none of them is so near to
    another beam's that its row would be summed again - the bits of the same beam alone."""
    for live in range(0, w, 3):
        logits, scores = random_logits(1, w, 248320, dtype, seed=live)
        scores[:, :live] = scores[:, live + 1:] = -math.inf
        scores[:, live] = 0
        got = check(logits, scores, n)
        one = alone(logits, scores, live, n)
        assert torch.equal(got[0], one[0]) and torch.equal(got[2], one[2]) and bool((got[1] == live).all())


@pytest.mark.parametrize("w,n", [(8, 64), (20, 40), (4, 128), (3, 100)])
def test_a_beam_far_ahead_of_the_others(w, n):
    """All candidates come from one beam, more of them above what a sample of all lists gives as a bound than are ordered at once: the bits of that
    beam alone."""
    for ahead in range(0, w, 3):
        logits, scores = random_logits(1, w, 248320, seed=ahead)
        scores[:] = -1000 - torch.arange(w, device=DEV)
        scores[:, ahead] = 0
        got = check(logits, scores, n)
        one = alone(logits, scores, ahead, n)
        assert torch.equal(got[0], one[0]) and torch.equal(got[2], one[2]) and bool((got[1] == ahead).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_some_beams_far_ahead(dtype):
    """Two or three beams share all places, beams at their end among them; equal logits by the thousand; several requests."""
    for b, w, n in ((1, 16, 128), (2, 10, 128), (3, 6, 100), (1, 40, 64)):
        logits, scores = random_logits(b, w, 248320, dtype, seed=n)
        scores[:, 3:] -= 1000
        finished = torch.zeros(b, w, dtype=torch.bool, device=DEV)
        finished[:, -1] = finished[-1, 1] = True
        scores[0, -1] = -3.0
        check(logits, scores, n, finished, 17)
        check((logits.float() * 0.5).round().to(dtype), scores.round(), n, finished, 17)


# ---------------------------------------------------------------- order within a beam
@pytest.mark.parametrize("w", [1, 3])
def test_logits_that_sums_in_64_bits_do_not_tell_apart(w):
    """Of one beam the larger logit is first, also where both totals are the same number: fewer candidates are the first of more."""
    from deepseek_v4_2080ti_b200.ops import beams
    logits = -1 - torch.rand(4, w, 300, generator=torch.Generator(device=DEV).manual_seed(w), device=DEV)
    logits[:, 0, [3, 50, 7, 200]] = torch.tensor([0.0, 1e-30, -1e-30, 2e-20], device=DEV)
    scores = torch.zeros(4, w, device=DEV)
    scores[:, 1:] = -50
    for n in (1, 2, 3, 4):
        assert beams.select(logits, scores, n)[2].tolist() == [[200, 50, 3, 7][:n]] * 4
    equal = logits[:, :1].expand(4, 3, 300).contiguous()
    got = beams.select(equal, torch.zeros(4, 3, device=DEV), 12)
    assert got[1].tolist() == [[0] * 4 + [1] * 4 + [2] * 4] * 4 and got[2].tolist() == [[200, 50, 3, 7] * 3] * 4


@pytest.mark.parametrize("w,v,n", [(1, 9000, 8), (3, 5000, 20), (20, 9000, 128), (4, 248320, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", [torch.finfo(torch.float32).min, -1e30])
def test_scores_that_outweigh_the_logits(w, v, n, dtype, score):
    """Beams at the type's lowest value, whose totals are all one number: of equals the lowest beam, and of its tokens the best."""
    from deepseek_v4_2080ti_b200.ops import beams
    logits, scores = random_logits(2, w, v, dtype)
    scores[:] = score
    best = logits[:, 0].float().sort(descending=True, stable=True).indices[:, :n].int()
    got = beams.select(logits, scores, n)
    assert bool((got[0] == score).all() and (got[1] == 0).all()) and torch.equal(got[2], best)


# ---------------------------------------------------------------- what the debug mode says of pages
def test_idle_sequences_in_the_debug_mode(monkeypatch):
    """A sequence whose q_start is negative is none: its empty table is no error and stays as it is, whatever its lengths are."""
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    args, _, (seqs, seen, _) = tree_inputs([(20, 300)], 4, 2, wide=9)
    q, kc, vc, table, mask = args[:5]
    table = torch.cat([torch.full_like(table, -1), table, torch.full_like(table, -1)])
    table[1, 5:] = -1
    kept = table.clone()
    for debug in "01":
        monkeypatch.setenv("B200_BOUNDS_CHECK", debug)
        for splits in (1, 3):
            out = attention.decode_tree(q, kc, vc, table, mask, _i32([-3, 0, -1]), _i32([30, 20, 5]), _i32([900, 320, 40]), 20, splits=splits)
            _lib.check_status()
            assert torch.equal(table, kept)
            close(out, *oracle(q, *seqs[0], seen[0]))


def test_nodes_below_lo_in_the_debug_mode(monkeypatch):
    """A page of nodes that no row's span reaches back to may be missing; where one does it is reported."""
    from deepseek_v4_2080ti_b200.ops import _lib, attention
    args, _, (seqs, seen, _) = tree_inputs([(20, 60)], 4, 2, wide=3)       # nodes at the keys 60 to 79, pages of 64
    table, lo = args[3], _i32([64] * 20)
    table[0, 0] = table[0, 2] = -1
    kept = table.clone()
    seen[0][:, :64] = False
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    out = attention.decode_tree(*args, lo=lo)
    _lib.check_status()
    assert torch.equal(table, kept)
    close(out, *oracle(args[0], *seqs[0], seen[0]))
    lo[3] = 60
    attention.decode_tree(*args, lo=lo)
    with pytest.raises(_lib.KernelError):
        _lib.check_status()


# ---------------------------------------------------------------- accepted paths in the debug mode
def accept_inputs():
    """Three sequences of one cache: a path of rows that move, an idle one, one whose path is its first node."""
    tokens, parents, predicted = _i32([9, 1, 2, 3, 2, 5, 6]), _i32([-1, 0, 0, 0, 3, -1, 0]), _i32([3, 0, 0, 2, 8, 4, 4])
    cache = torch.arange(8 * 16, device=DEV, dtype=torch.float32).view(1, 8, 1, 16).clone()
    return (tokens, parents, predicted, _i32([0, -1, 5]), _i32([5, 3, 2]), 4, _i32([37, 20, 40])), cache


def test_pages_that_are_not_there_are_reported_by_accept(monkeypatch):
    """Rows of the path that lie in pages outside the cache stay where they are; the debug mode says so, whichever page it is, and says nothing
    of pages that no row of a path lies in.  The table is left as it is."""
    from deepseek_v4_2080ti_b200.ops import _lib, tree
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    args, cache = accept_inputs()                          # sequence 0: keys 32 .. 36 are the tree, 35 -> 33 and 36 -> 34
    for row, bad in (([0, 1, 2], False), ([-1, 99, 2], False), ([0, 1, -1], True), ([0, 1, 8], True), ([0, 1, -2 ** 31], True), ([0, 1, 2 ** 31 - 1], True)):
        table = _i32([row, [-1, -1, -1], [-1, -1, -1]])
        was, kept = cache.clone(), table.clone()
        got = tree.accept(*args, table, [cache])
        assert got[0].tolist() == [[0, 3, 4, -1], [-1] * 4, [0] + [-1] * 3]
        if bad:
            with pytest.raises(_lib.KernelError):
                _lib.check_status()
            assert torch.equal(cache, was)
        else:
            _lib.check_status()
            was[0, 2, 0, 1], was[0, 2, 0, 2] = was[0, 2, 0, 3].clone(), was[0, 2, 0, 4].clone()
            assert torch.equal(cache, was)
        assert torch.equal(table, kept)


def test_a_captured_accept_in_the_debug_mode(monkeypatch):
    from deepseek_v4_2080ti_b200.ops import _lib, tree
    monkeypatch.setenv("B200_BOUNDS_CHECK", "1")
    args, cache = accept_inputs()
    table = _i32([[0, 1, 2], [-1] * 3, [-1] * 3])
    tree.accept(*args, table, [cache.clone()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tree.accept(*args, table, [cache])
    graph.replay()
    torch.cuda.synchronize()
    _lib.check_status()
    assert got[1].tolist() == [3, 0, 1]
    table[0, 2] = 70
    graph.replay()
    with pytest.raises(_lib.KernelError):
        _lib.check_status()


def test_a_tensor_in_the_place_of_a_list_of_caches_is_refused():
    """Its layers would be taken for caches, and their pages for layers: rows of other keys would move."""
    from deepseek_v4_2080ti_b200.ops import tree
    args, _ = accept_inputs()
    cache = torch.arange(2 * 3 * 2 * 16 * 4, device=DEV, dtype=torch.float32).view(2, 3, 2, 16, 4)
    was, table = cache.clone(), _i32([[0, 1, 2], [-1] * 3, [-1] * 3])
    with pytest.raises(ValueError):
        tree.accept(*args, table, cache)
    assert torch.equal(cache, was)
    tree.accept(*args, table, (cache,))
    assert not torch.equal(cache, was)
