"""Norm, rotation by positions of several axes and append, against the same in 64 bits.

Bound: one rounding to bf16 (2^-8 of the value) and 32-bit arithmetic before it - norm, cosine and sine to 2^-20, one product and
one sum each - which is below 2^-16 of the larger of a pair's normalised values."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(t, hq, hkv, sections, interleaved, gate, bs, norm="unit", split=False, far=0, seed=0, mscale=1.0, pad=0, axes=3):
    from deepseek_v4_2080ti_b200.ops import attention
    torch.manual_seed(seed + t)
    rot = 2 * sum(sections)
    per = 256 if gate else 128
    qw, kw = hq * per, hkv * 128
    src = (torch.randn(t, qw + 2 * kw + pad, device=DEV) * 2).bfloat16()
    if split:                                              # three tensors, rows further apart than they are wide
        q_src, k_src, v_src = (torch.randn(t, w + 12, device=DEV).bfloat16()[:, :w + 4] for w in (qw, kw, kw))
        ko = vo = 4
        qo = 4
    else:
        q_src = k_src = v_src = src
        qo, ko, vo = 0, qw, qw + kw
    g = lambda: None if norm is None else (torch.randn(128, device=DEV) * 0.2 + (norm == "plain")).bfloat16()
    qg, kg = g(), g()
    pos = torch.randint(0, 50, (axes, t), device=DEV, dtype=torch.int32) + far
    pages = (t + bs - 1) // bs + 2
    slots = torch.randperm(pages * bs, device=DEV)[:t].to(torch.int32)
    slots = torch.where(torch.arange(t, device=DEV) % 7 == 3, -1 - slots, slots).to(torch.int32)
    kc = torch.full((pages, hkv, bs, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    vc = torch.full_like(kc, 3.0)
    inv = attention.rope_inv_freq(rot, 1e7, DEV)
    table = attention.rotary_axes(sections, interleaved)
    q, gate_out = attention.qk_norm_rope_axes_append(q_src, qo, per, gate, k_src, ko, v_src, vo, qg, kg, norm == "unit", 1e-6, inv, table, pos,
                                                     slots, kc, vc, hq, hkv, mscale=mscale)
    torch.cuda.synchronize()

    def prep(x, gamma):
        x = x.double()
        if gamma is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (gamma.double() + (norm == "unit"))
        h = rot // 2
        y = x.clone()
        for i, a in enumerate(table):
            ang = pos[a].double() * inv[i].double()
            c, s = (ang.cos() * mscale)[:, None], (ang.sin() * mscale)[:, None]
            y[..., i] = x[..., i] * c - x[..., i + h] * s
            y[..., i + h] = x[..., i + h] * c + x[..., i] * s
        m = x.abs()
        pair = torch.cat([torch.maximum(m[..., :h], m[..., h:rot])] * 2 + [m[..., rot:]], -1)
        return y, y.abs() * 2.0 ** -8 + pair * 2.0 ** -16 * max(1.0, mscale)

    def close(got, want):
        over = (got.double() - want[0]).abs() - want[1]
        assert over.numel() == 0 or over.max().item() <= 0.0, over.max().item()
    heads = q_src[:, qo:qo + qw].reshape(t, hq, per)
    close(q, prep(heads[..., :128], qg))
    assert gate_out is None if not gate else torch.equal(gate_out, heads[..., 128:])
    live = slots >= 0
    at = slots[live].long()
    key, val = k_src[:, ko:ko + kw].reshape(t, hkv, 128), v_src[:, vo:vo + kw].reshape(t, hkv, 128)
    close(kc[at // bs, :, at % bs], tuple(x[live] for x in prep(key, kg)))
    assert torch.equal(vc[at // bs, :, at % bs], val[live])
    rest = torch.ones(pages * bs, dtype=torch.bool, device=DEV)
    rest[at] = False
    for c in (kc, vc):
        assert bool((c.transpose(1, 2).reshape(pages * bs, hkv, 128)[rest] == 3.0).all())


@pytest.mark.parametrize("t", [1, 2, 5, 37, 300])
@pytest.mark.parametrize("hq,hkv,sections,interleaved,gate,bs", [
    (40, 8, (6, 5, 5), True, True, 64), (5, 1, (16, 24, 24), False, False, 16), (48, 8, (24, 20, 20), True, False, 64),
    (1, 1, (4, 0, 0), False, True, 32), (8, 8, (4, 4, 4), True, False, 24), (28, 4, (12, 10, 10), True, False, 128)])
def test_rows(t, hq, hkv, sections, interleaved, gate, bs):
    _case(t, hq, hkv, sections, interleaved, gate, bs)


def test_layouts_norms_and_far_positions():
    _case(33, 6, 2, (8, 4, 4), True, True, 64, norm="plain", split=True)
    _case(33, 6, 2, (8, 4, 4), False, False, 64, norm=None, split=True, mscale=1.25)
    _case(33, 6, 2, (32, 0, 0), False, False, 64, far=10_000_000)
    _case(33, 6, 2, (20, 20, 8, 8), False, True, 64, far=-25, axes=4, pad=20)
    _case(9, 6, 2, (64,), False, False, 64, far=2_000_000_000, axes=1)


def test_equal_axes_give_the_one_axis_kernel():
    """Text counts on all axes at once: the same bits as the kernel with one axis."""
    from deepseek_v4_2080ti_b200.ops import attention
    torch.manual_seed(1)
    t, hq, hkv, bs = 77, 10, 2, 64
    src = torch.randn(t, (2 * hq + 2 * hkv) * 128, device=DEV).bfloat16()
    qg, kg = ((torch.randn(128, device=DEV) * 0.1).bfloat16() for _ in range(2))
    pos = torch.arange(5000, 5000 + t, dtype=torch.int32, device=DEV)
    slots = torch.randperm(t, device=DEV).to(torch.int32)
    inv = attention.rope_inv_freq(64, 1e6, DEV)
    got = []
    for several in (False, True):
        kc, vc = (torch.zeros(2, hkv, bs, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        args = (src, 0, 256, True, src, 2 * hq * 128, src, (2 * hq + hkv) * 128, qg, kg, True, 1e-6, inv)
        tail = (slots, kc, vc, hq, hkv)
        q, gate = attention.qk_norm_rope_axes_append(*args, attention.rotary_axes((12, 10, 10), True), pos.expand(3, t).contiguous(), *tail) if several \
            else attention.qk_norm_rope_append(*args, 64, pos, *tail)
        got.append((q, gate, kc, vc))
    for a, b in zip(*got):
        assert (a.double() - b.double()).abs().max().item() <= 2.0 ** -7 * a.abs().max().item()
        assert (a != b).float().mean().item() < 1e-3       # (a value on the border between two bf16 numbers)
