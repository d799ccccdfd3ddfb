"""Plans of the calls over spans and shared pages, on the host: spans of blocks that overlap, groups of sequences, limits of scale and cap, pages
that a row sees, and a torch without CUDA."""
import math
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from deepseek_v4_2080ti_b200.ops import attention


@pytest.mark.parametrize("blocks", [[(0, 8), (2, 4)], [(1, 9), (3, 7), (4, 5)], [(0, 4), (2, 7)], [(5, 5), (2, 6), (2, 3)]])
def test_blocks_that_overlap_see_to_the_furthest_end(blocks):
    """In any order: a position sees up to the furthest end of the blocks that it lies in."""
    want = [max([j + 1] + [e for f, e in blocks if f <= j < e]) for j in range(10)]
    for order in (blocks, blocks[::-1], sorted(blocks)):
        lo, hi = attention.visible_spans(10, blocks=order)
        assert hi.tolist() == want and lo.tolist() == [0] * 10


def test_blocks_stay_in_their_document():
    lo, hi = attention.visible_spans(7, [3, 0, 4], blocks=[(0, 3), (4, 7), (3, 3), (7, 7)])
    assert lo.tolist() == [0, 0, 0, 3, 3, 3, 3] and hi.tolist() == [3, 3, 3, 4, 7, 7, 7]
    for bad in ((1, 5), (0, 7), (2, 4)):
        with pytest.raises(ValueError, match="document"):
            attention.visible_spans(7, [3, 0, 4], blocks=[bad])
    assert attention.visible_spans(7, [0, 7, 0], blocks=[(1, 7)])[1].tolist() == [1, 7, 7, 7, 7, 7, 7]


def _saved(pages, start, shared, block_size):
    """Pages that need not be read again, after a look at the plan itself."""
    assert start[0] == 0 and start[-1] == len(pages) and len(shared) == len(start) - 1 and all(a < b for a, b in zip(start, start[1:]))
    saved = 0
    for a, b, n in zip(start, start[1:], shared):
        assert n % block_size == 0 and (b - a > 1 or n == 0)
        n //= block_size
        assert all(row[:n] == pages[a][:n] and len(row) >= n for row in pages[a:b])
        saved += (b - a - 1) * n
    return saved


def _best(pages):
    """The most that any cut of the sequences into runs of neighbours saves: all cuts, one by one."""
    n, best = len(pages), 0
    for cuts in range(1 << max(0, n - 1)):
        edges = [0] + [i + 1 for i in range(n - 1) if cuts >> i & 1] + [n]
        total = 0
        for a, b in zip(edges, edges[1:]):
            common = 0
            while all(len(row) > common and row[common] == pages[a][common] for row in pages[a:b]):
                common += 1
            total += (b - a - 1) * common
        best = max(best, total)
    return best


def test_a_system_page_before_several_documents():
    a, b = [9] + list(range(100, 120)), [9] + list(range(200, 220))
    assert attention.shared_groups([a + [i] for i in range(4)] + [b + [10 + i] for i in range(4)], 64) == ([0, 4, 8], [21 * 64] * 2)
    for at in (0, 3, 6):                                   # one that has nothing but the first page in common
        rows = [a + [i] for i in range(6)]
        rows.insert(at, [9, 5000])
        start, shared = attention.shared_groups(rows, 16)
        assert _saved(rows, start, shared, 16) == _best(rows)
    assert attention.shared_groups([[9, i] for i in range(5)], 32) == ([0, 5], [32])         # the page alone is still shared
    assert attention.shared_groups([[i] for i in range(4)] + [[], []], 32) == ([0, 1, 2, 3, 4, 5, 6], [0] * 6)


def test_groups_save_the_most():
    rng = random.Random(1)
    for trial in range(150):
        n = rng.randint(1, 9)
        pages = [[rng.randint(0, 1) * 10 ** i for i in range(rng.randint(0, 7))] for _ in range(n)]
        if trial % 2:
            pages.sort()
        start, shared = attention.shared_groups(pages, 16)
        assert _saved(pages, start, shared, 16) == _best(pages), pages


def test_scales_and_caps_that_32_bits_do_not_hold():
    """A cap that becomes zero in 32 bits would be none at all, one beyond them infinite."""
    for scale, cap in ((None, 0.0), (0.1, 30.0), (1.0, 1e-6), (0.0884, 1e9), (2.0 ** -100, 0.0), (2.0 ** 100, 1.0), (1.0, 2.0 ** 100)):
        assert attention._scores(scale, cap) == 1 / math.sqrt(128) if scale is None else scale
    for scale, cap in ((None, 1e-50), (None, 1e-40), (None, 3e38), (None, 1e300), (1e-50, 0.0), (1e300, 0.0), (1e25, 1e-25), (1e-25, 1e25), (0.0, 0.0),
                       (-1.0, 0.0), (math.nan, 0.0), (math.inf, 0.0), (None, -1.0), (None, math.inf), (None, math.nan)):
        with pytest.raises(ValueError):
            attention._scores(scale, cap)


def test_pages_that_a_row_sees():
    rng = random.Random(2)
    for trial in range(60):
        bs, width, b = rng.choice((16, 32)), rng.randint(1, 6), rng.randint(1, 4)
        q_len = [rng.randint(0, 9) for _ in range(b)]
        q_start, t = [], rng.randint(0, 3)
        for n in q_len:
            q_start.append(t)
            t += n + rng.randint(0, 2)
        kv = [rng.randint(0, width * bs + 20) for _ in range(b)]
        lo = [rng.randint(-5, width * bs + 5) for _ in range(t)] if trial % 3 else None
        hi = [rng.choice((rng.randint(-5, width * bs + 50), 2 ** 31 - 1, -2 ** 31)) for _ in range(t)] if trial % 2 else None
        want = [[False] * width for _ in range(b)]
        for i in range(b):
            for r in range(q_start[i], q_start[i] + q_len[i]):
                first = max(0, lo[r]) if lo else 0
                end = hi[r] if hi else kv[i] - q_len[i] + r - q_start[i] + 1
                for j in range(first, min(end, kv[i], width * bs)):
                    want[i][j // bs] = True
        ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32)
        got = attention._seen_pages(t, width, bs, ints(kv), ints(q_start), ints(q_len), ints(lo), ints(hi))
        assert got.tolist() == want


def test_the_module_loads_where_torch_has_no_cuda():
    """The host reference runtime takes its fp32 oracles from this module; a torch built without CUDA lacks these entry points."""
    code = ("import torch\n"
            "for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream', '_cuda_setDevice', '_cuda_getDeviceCount'):\n"
            "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
            "import deepseek_v4_2080ti_b200.models.reference_cpu.qwen_hybrid_ref\n"
            "from deepseek_v4_2080ti_b200.ops import attention\n"
            "assert attention.rotary_axes((2, 1, 1), True) == (0, 1, 2, 0)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
