"""Host side of the calls over drafted trees and beams: refusals, without a device and on one."""
import pytest
import torch

from deepseek_v4_2080ti_b200.ops import attention, beams, tree

Z = torch.zeros
I32 = torch.int32


def test_host_tensors_are_refused():
    one = Z(2, dtype=I32)
    with pytest.raises(ValueError):
        tree.layout(one, one, one, one, 4)
    with pytest.raises(ValueError):
        tree.accept(one, one, one, one, one, 4)
    with pytest.raises(ValueError):
        beams.select(Z(1, 2, 30), Z(1, 2))
    with pytest.raises(ValueError):
        beams.reorder(Z(4, 8), Z(1, 2, dtype=I32))
    c = Z(3, 2, 64, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention.decode_tree(Z(2, 4, 128, dtype=torch.bfloat16), c, c, Z(1, 3, dtype=I32), Z(2, 1, dtype=I32), *(Z(1, dtype=I32),) * 3, 2)


def test_parts_of_a_row():
    """Every logit in a part, and no more parts than the kernel that joins them takes."""
    for v in (1, 8192, 8193, 51001, 248320, beams.MAX_VOCAB):
        for rows in (1, 4, 128, 512, 65535):
            parts, tiles = beams._parts(rows, v)
            assert parts * tiles * beams.TILE >= v > (parts - 1) * tiles * beams.TILE
            assert parts * min(rows, beams.MAX_BEAMS) + beams.MAX_BEAMS <= 8192
            assert parts * tiles * beams.TILE < 2 ** 31             # places are numbers of 32 bits


def seen_and_missing(monkeypatch, table, mask, q_start, q_len, kv_len, lo=None, bs=16):
    """The table after the debug mode's look at it, without the scan that reports (-2) and replaces what it has marked."""
    from deepseek_v4_2080ti_b200.ops import _lib
    monkeypatch.setattr(_lib, "bounds_checks_on", lambda: True)
    monkeypatch.setattr(_lib, "check_indices", lambda *a, **k: None)
    i = lambda x: torch.tensor(x, dtype=I32)
    table = i(table)
    attention._check_tree_pages(table, 8, bs, i(kv_len), i(q_start), i(q_len), None if lo is None else i(lo), i(mask))
    return table.tolist()


def test_idle_sequences_claim_no_rows_in_the_debug_mode(monkeypatch):
    """A negative q_start is no sequence, whatever its lengths: its table is not looked at, and rows of others see their own context."""
    mask = [[1], [3], [5]]
    for table in ([[0, 1, -1], [-1, -1, -1]], [[0, -1, -1], [-1, -1, -1]]):
        found = seen_and_missing(monkeypatch, table, mask, [0, -1], [3, 5], [20, 200])
        assert found == [[x if x >= 0 or i > 1 else -2 for i, x in enumerate(table[0])], [-1, -1, -1]]
    # an idle one before and after, and one that begins behind the rows
    assert seen_and_missing(monkeypatch, [[-1] * 3, [4, 5, -1], [-1] * 3, [-1] * 3], mask, [-3, 0, -1, 3], [4, 3, 3, 4], [40, 32, 48, 40]) == [[-1] * 3, [4, 5, -1], [-1] * 3, [-1] * 3]
    # two sequences, each row with the context of its own
    assert seen_and_missing(monkeypatch, [[0, -1, -1], [1, 2, -1]], [[1], [3], [1]], [0, 2], [2, 1], [10, 40]) == [[0, -1, -1], [1, 2, -2]]


def test_nodes_below_lo_are_not_seen_in_the_debug_mode(monkeypatch):
    """A node's key counts only for rows that have its bit and whose span reaches back to it."""
    mask, args = [[1], [3], [7], [15]], ([0], [4], [18])               # nodes at the keys 14 to 17
    assert seen_and_missing(monkeypatch, [[-1, 3, -1]], mask, *args, lo=[16, 16, 16, 16]) == [[-1, 3, -1]]
    assert seen_and_missing(monkeypatch, [[-1, 3, -1]], mask, *args, lo=[16, 15, 16, 16]) == [[-2, 3, -1]]
    assert seen_and_missing(monkeypatch, [[-1, -1, -1]], [[1], [2], [4], [3]], *args, lo=[18, 16, 16, 16]) == [[-1, -2, -1]]
    assert seen_and_missing(monkeypatch, [[-1, -1, -1]], [[1], [2], [3], [3]], *args, lo=[18, 16, 16, 16]) == [[-1, -1, -1]]
    assert seen_and_missing(monkeypatch, [[-1, -1, -1]], mask, *args) == [[-2, -2, -1]]


@pytest.mark.gpu
def test_refusals_on_a_device():
    i = lambda *s: Z(*s, dtype=I32, device="cuda")
    f = lambda *s: Z(*s, device="cuda")
    c = lambda *s: Z(*s, dtype=torch.bfloat16, device="cuda")
    good = dict(q=c(6, 4, 128), k_cache=c(3, 2, 64, 128), v_cache=c(3, 2, 64, 128), block_table=i(2, 3), mask=i(6, 1), q_start=i(2), q_len=i(2), kv_len=i(2),
                max_q_len=3)
    attention.decode_tree(**good)
    for change in ({"mask": i(6)}, {"mask": i(5, 1)}, {"mask": i(6, 0)}, {"mask": i(6, 33)}, {"mask": i(6, 2)[:, :1]}, {"mask": i(6, 1).long()}, {"lo": i(5)},
                   {"q_len": i(3)}, {"splits": 0}, {"splits": 2000}, {"cap": -1.0}, {"q": c(40, 4, 128), "mask": i(40, 1), "max_q_len": 40}, {"gate": c(6, 4, 64)}):
        with pytest.raises(ValueError):
            attention.decode_tree(**good | change)
    good = dict(parents=i(6), q_start=i(2), q_len=i(2), kv_len=i(2), max_nodes=3)
    tree.layout(**good)
    for change in ({"parents": i(6).long()}, {"parents": i(12)[::2]}, {"q_start": i(3)}, {"kv_len": i(2).float()}, {"q_len": i(2, 1)}, {"max_nodes": 0},
                   {"max_nodes": 1025}):
        with pytest.raises(ValueError):
            tree.layout(**good | change)
    k = c(2, 3, 2, 64, 128)
    good = dict(tokens=i(6), parents=i(6), predicted=i(6), q_start=i(2), q_len=i(2), max_path=4, kv_len=i(2), block_table=i(2, 3), caches=[k])
    tree.accept(**good)
    for change in ({"tokens": i(6).long()}, {"parents": i(5)}, {"predicted": i(7)}, {"q_len": i(3)}, {"max_path": 0}, {"max_path": 257}, {"kv_len": None},
                   {"kv_len": i(3)}, {"block_table": i(3, 3)}, {"block_table": None}, {"caches": [k] * 17}, {"caches": [k.cpu()]}, {"caches": [k[0]]},
                   {"caches": [k, c(2, 4, 2, 64, 128)]}, {"caches": [k.transpose(2, 3)]}, {"caches": [k, k]}, {"caches": [c(2, 3, 2, 64, 127)]},
                   {"caches": [k[:, :, :1]]}):
        with pytest.raises(ValueError):
            tree.accept(**good | change)
    good = dict(logits=f(2, 3, 50), scores=f(2, 3))
    beams.select(**good)
    for change in ({"logits": f(6, 50)}, {"logits": f(2, 3, 50).half()}, {"logits": f(2, 3, 100)[..., ::2]}, {"logits": f(2, 4, 50)[:, :3]},
                   {"logits": f(3, 2, 50).transpose(0, 1)}, {"logits": f(2, 3, 50)[:, :1].expand(2, 3, 50)}, {"logits": f(2, 3, 0)}, {"scores": f(2, 4)},
                   {"scores": f(2, 3).double()}, {"scores": f(3, 2).t()}, {"n": 0}, {"n": 129}, {"finished": f(2, 3)}, {"pad_token": 50}, {"pad_token": -1},
                   {"logits": f(1, 129, 5), "scores": f(1, 129)}):
        with pytest.raises(ValueError):
            beams.select(**good | change)
    good = dict(states=[f(6, 8), f(6, 3)], parents=i(2, 3))
    beams.reorder(**good)
    for change in ({"parents": i(6)}, {"parents": i(2, 3).long()}, {"parents": i(3, 3)}, {"slots": i(2, 4)}, {"states": [f(6, 8), f(7, 8)]}, {"states": []},
                   {"states": f(6, 8, 2)[:, ::2]}, {"states": f(6, 0)}, {"states": f(1, 8).expand(6, 8)}, {"dim": 2}, {"dim": -1},
                   {"states": f(6, 8).cpu()}, {"states": f(3, 4, 6, 8)[:, :3], "dim": 2}, {"parents": i(1, 129), "states": f(200, 4)}):
        with pytest.raises(ValueError):
            beams.reorder(**good | change)


@pytest.mark.gpu
def test_nothing_to_do():
    i = lambda *s: Z(*s, dtype=I32, device="cuda")
    c = lambda *s: Z(*s, dtype=torch.bfloat16, device="cuda")
    assert attention.decode_tree(c(0, 4, 128), c(3, 2, 64, 128), c(3, 2, 64, 128), i(1, 3), i(0, 1), i(1), i(1), i(1), 0).shape == (0, 4, 128)
    assert [x.shape for x in tree.layout(i(0), i(2), i(2), i(2), 40)] == [(0,), (0, 2)]
    assert tree.layout(i(3), i(0), i(0), i(0), 4)[0].tolist() == [0, 0, 0]
    assert [x.shape for x in tree.accept(i(3), i(3), i(3), i(0), i(0), 4)] == [(0, 4), (0,), (0, 4)]
    assert tree.accept(i(0), i(0), i(0), i(2), i(2), 4)[1].tolist() == [0, 0]
    assert [x.shape for x in beams.select(Z(0, 3, 50, device="cuda"), Z(0, 3, device="cuda"), 4)] == [(0, 4)] * 3
    beams.reorder(c(4, 8), i(0, 3))
