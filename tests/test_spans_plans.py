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
