"""Host side of the calls over spans and shared pages: helpers and refusals, without a device."""
import pytest
import torch

from deepseek_v4_2080ti_b200.models.qwen4_exp_components import mrope_cos_sin
from deepseek_v4_2080ti_b200.ops import attention


@pytest.mark.parametrize("sections", [(6, 5, 5), (12, 10, 10), (24, 20, 20), (8, 4, 4), (32, 0, 0)])
def test_interleaved_axes_are_those_of_the_tensor_statement(sections):
    axes = attention.rotary_axes(sections, True)
    rot = 2 * sum(sections)
    pos = torch.tensor([3, 700, 90000])[:, None, None]
    cos, _ = mrope_cos_sin(pos, rot, 1e4, sections)
    want = torch.tensor([float(pos[a]) for a in axes]) * (1.0 / (1e4 ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot)))
    assert torch.equal(cos[0, 0, :rot // 2], want.cos())


def test_axes_in_blocks_and_refusals():
    assert attention.rotary_axes((2, 1, 3)) == (0, 0, 1, 2, 2, 2)
    assert attention.rotary_axes((2, 1, 1), True) == (0, 1, 2, 0)
    for bad in ((), (0, 0), (-1, 5), (40, 30)):
        with pytest.raises(ValueError):
            attention.rotary_axes(bad)
    with pytest.raises(ValueError):
        attention.rotary_axes((16, 24, 24), True)


def test_visible_spans():
    lo, hi = attention.visible_spans(7, [3, 0, 4])
    assert lo.tolist() == [0, 0, 0, 3, 3, 3, 3] and hi.tolist() == [1, 2, 3, 4, 5, 6, 7]
    lo, hi = attention.visible_spans(6, blocks=[(1, 4)], window=2)
    assert lo.tolist() == [0, 0, 1, 2, 3, 4] and hi.tolist() == [1, 4, 4, 4, 5, 6]
    assert attention.visible_spans(0)[0].numel() == 0
    for kw in ({"documents": [3, 3]}, {"documents": [-1, 8]}, {"blocks": [(4, 3)]}, {"blocks": [(0, 8)]}):
        with pytest.raises(ValueError):
            attention.visible_spans(7, **kw)


def test_shared_groups():
    pages = [[5, 6, 7], [5, 6, 9, 2], [5, 6], [8], [3, 4], [3, 1], []]
    assert attention.shared_groups(pages, 64) == ([0, 3, 4, 6, 7], [128, 0, 64, 0])
    assert attention.shared_groups([], 64) == ([0], [])
    assert attention.shared_groups([[1, 2], [1, 2]], 16) == ([0, 2], [32])


def _args(**change):
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype)
    a = {"q": z(2, 4, 128, dtype=torch.bfloat16), "k_cache": z(3, 2, 64, 128, dtype=torch.bfloat16), "v_cache": z(3, 2, 64, 128, dtype=torch.bfloat16),
         "block_table": z(2, 3), "kv_len": z(2)}
    return a | change


def test_host_tensors_and_wrong_shapes_are_refused():
    """Nothing of these reaches a device; the checks name what they expect."""
    z = torch.zeros
    spans = {"q_start": z(2, dtype=torch.int32), "q_len": z(2, dtype=torch.int32), "max_q_len": 1}
    for change in ({}, {"q": z(2, 4, 64, dtype=torch.bfloat16)}, {"q": z(2, 4, 128)}, {"k_cache": z(3, 2, 64, 128)}):
        with pytest.raises(ValueError):
            attention.prefill_spans(**_args(**change), **spans)
        with pytest.raises(ValueError):
            attention.decode_shared(**_args(**change), group_start=z(2, dtype=torch.int32), shared_len=z(1, dtype=torch.int32))
    src = z(2, 8 * 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention.qk_norm_rope_axes_append(src, 0, 128, False, src, 512, src, 768, None, None, True, 1e-6, z(16), attention.rotary_axes((8, 4, 4)),
                                           z(3, 2, dtype=torch.int32), z(2, dtype=torch.int32), _args()["k_cache"], _args()["v_cache"], 4, 2)


@pytest.mark.gpu
def test_refusals_on_a_device():
    dev = lambda d: {k: v.cuda() for k, v in d.items()}
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    spans = {"q_start": i(2), "q_len": i(2), "max_q_len": 1}
    shared = {"group_start": i(2), "shared_len": i(1)}
    c = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    bad = [{"q": c(2, 3, 128)}, {"k_cache": c(3, 2, 48, 128), "v_cache": c(3, 2, 48, 128)}, {"v_cache": c(3, 2, 32, 128)}, {"kv_len": i(3)},
           {"block_table": i(2, 6)[:, ::2]}, {"q": c(2, 8, 128)[:, ::2]}, {"scale": 0.0}, {"scale": float("nan")}, {"cap": -1.0}, {"cap": float("inf")},
           {"gate": c(2, 4, 64)}, {"out": c(1, 4, 128)}, {"kv_len": torch.zeros(2, dtype=torch.int64, device="cuda")}]
    for change in bad:
        with pytest.raises(ValueError):
            attention.prefill_spans(**dev(_args()) | spans | change)
        with pytest.raises(ValueError):
            attention.decode_shared(**dev(_args()) | shared | change)
    for change in ({"lo": i(3)}, {"hi": i(2).long()}, {"q_start": i(1)}, {"splits": 0}, {"splits": 5000}):
        with pytest.raises(ValueError):
            attention.prefill_spans(**dev(_args()) | spans | change)
    for change in ({"group_start": i(1)}, {"shared_len": i(2)}, {"splits": 65}, {"block_table": i(3, 3), "kv_len": i(3)}):
        with pytest.raises(ValueError):
            attention.decode_shared(**dev(_args()) | shared | change)
    src, kc = c(2, 1024), c(3, 2, 64, 128)
    good = dict(q_src=src, q_off=0, q_head_stride=128, gate_in_q=False, k_src=src, k_off=512, v_src=src, v_off=768, q_gamma=None, k_gamma=None,
                unit_offset=True, eps=1e-6, inv_freq=torch.ones(16, device="cuda"), axes=attention.rotary_axes((8, 4, 4)), positions=i(3, 2),
                slots=i(2) - 1, k_cache=kc, v_cache=c(3, 2, 64, 128), n_q_heads=4, n_kv_heads=2)
    attention.qk_norm_rope_axes_append(**good)
    for change in ({"positions": i(2, 2)}, {"positions": i(3, 3)}, {"slots": i(3)}, {"inv_freq": torch.ones(8, device="cuda")}, {"axes": (0, 1, 2)},
                   {"q_off": 2}, {"v_off": 800}, {"q_head_stride": 304}, {"n_kv_heads": 1}, {"q_gamma": c(64)}, {"k_src": src.float()},
                   {"v_cache": c(3, 2, 32, 128)}, {"axes": (-1,) * 16}):
        with pytest.raises(ValueError):
            attention.qk_norm_rope_axes_append(**good | change)


@pytest.mark.gpu
def test_nothing_to_do():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    c = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    kc = c(3, 2, 64, 128)
    assert attention.prefill_spans(c(0, 4, 128), kc, kc, i(1, 3), i(1), i(1), i(1), 0).shape == (0, 4, 128)
    assert attention.decode_shared(c(0, 4, 128), kc, kc, i(0, 3), i(0), i(1), i(0)).shape == (0, 4, 128)
    out = attention.decode_shared(c(2, 4, 128) + 1, kc, kc, i(2, 3), i(2), i(1), i(0))           # contexts of no keys
    assert bool((out == 0).all())
    src = c(0, 1024)
    q, gate = attention.qk_norm_rope_axes_append(src, 0, 128, False, src, 512, src, 768, None, None, True, 1e-6, torch.ones(16, device="cuda"),
                                                 attention.rotary_axes((8, 4, 4)), i(3, 0), i(0), kc, kc, 4, 2)
    assert q.shape == (0, 4, 128) and gate is None
