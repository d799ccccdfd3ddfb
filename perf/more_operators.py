"""The operators that carry several continuations of one context - drafted trees and beams - as they are timed.

``tree``: ``attention.decode_tree`` - rows of a drafted tree over a paged cache: the context, and the ancestors of every row.

``layout``: ``tree.layout`` - positions and masks of a tree's rows from the parents that the drafter hands over.

``accept``: ``tree.accept`` - the path that the target agrees with; its rows of every layer's cache move up behind the context.

``select``: ``beams.select`` - the best continuations over the beams of a request and the vocabulary.

``reorder``: ``beams.reorder`` - the beams' states follow the beams that were chosen.

Caches are bf16 pages [layers, pages, kv heads, page size, 128]; head counts, layers, vocabularies and recurrent states are those of this
framework's configurations (40 / 8 heads with an output gate, 48 / 8; 16 attention and 48 recurrent layers; 248320, 200064, 129280
tokens) and generic ones.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
D = 128


# ------------------------------------------------------------------------------------------------ cases
def _tree(name, batch, nodes, context, hq, hkv, width=4, cap=0.0, gate=False, bs=64, ragged=False, window=0):
    return {"name": name, "kind": "tree", "batch": batch, "nodes": nodes, "context": context, "hq": hq, "hkv": hkv, "width": width,
            "cap": cap, "gate": gate, "bs": bs, "ragged": ragged, "window": window}


def _layout(name, batch, nodes, context, width=4, ragged=False):
    return {"name": name, "kind": "layout", "batch": batch, "nodes": nodes, "context": context, "width": width, "ragged": ragged}


def _accept(name, batch, nodes, context, layers, hkv, taken, width=4, bs=64, ragged=False):
    return {"name": name, "kind": "accept", "batch": batch, "nodes": nodes, "context": context, "layers": layers, "hkv": hkv, "taken": taken,
            "width": width, "bs": bs, "ragged": ragged}


def _select(name, requests, beams, vocab, n, dtype="float32", finished=False, first=False):
    return {"name": name, "kind": "select", "requests": requests, "beams": beams, "vocab": vocab, "n": n, "dtype": dtype,
            "finished": finished, "first": first}


def _reorder(name, requests, beams, what, layers, size, idle=False):
    return {"name": name, "kind": "reorder", "requests": requests, "beams": beams, "what": what, "layers": layers, "size": size, "idle": idle}


def listed():
    return [
        _tree("tree_1x7", 1, 7, 350, 40, 8, width=2, gate=True),                            # one user, a small tree after a short prompt
        _tree("tree_9x26_ragged", 9, 26, 3100, 48, 8, cap=30.0, bs=32, ragged=True),        # a few users, trees of several sizes
        _tree("tree_32x64", 32, 64, 8192, 40, 8, width=8, gate=True),                       # the benchmark's decode batch on its prompt, wide trees
        _layout("layout_1x7", 1, 7, 350, width=2),                                          # once per step of the smallest tree
        _layout("layout_64x61_ragged", 64, 61, 9000, width=8, ragged=True),                 # once per step of a busy server
        _accept("accept_1x7", 1, 7, 350, 16, 8, 3, width=2),                                # three drafts kept in 16 layers of one sequence
        _accept("accept_64x61_ragged", 64, 61, 700, 16, 8, 6, width=8, ragged=True),        # and for a busy server
        _select("select_1x4", 1, 4, 248320, 8),                                             # one user's four beams, twice as many candidates
        _select("select_9x7_odd", 9, 7, 51001, 13, dtype="bfloat16"),                       # trees that grow by 13 nodes, odd sizes, ties
        _select("select_64x8", 64, 8, 248320, 16, finished=True),                           # many users, some of their beams at their end
        _reorder("reorder_pages_1x4", 1, 4, "pages", 16, 8),                                # the beams' last pages in 16 layers
        _reorder("reorder_states_4x4", 4, 4, "states", 48, 32),                             # their recurrent states in 48 layers
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((40, 8), (48, 8), (32, 8), (28, 4), (16, 16), (16, 2), (5, 1))


def draw(rng):
    kind = rng.choice(("tree", "tree", "layout", "accept", "select", "select", "reorder"))
    ragged, width = rng.random() < 0.5, rng.choice((0, 1, 2, 4, 8, 30))
    if kind == "tree":
        batch, nodes = _log(rng, 1, 32), _log(rng, 1, 130)
        hq, hkv = rng.choice(HEADS)
        most = 32 * 64 * 8192 * 40 // (batch * nodes * hq) * 10 // 14               # the work of the largest listed one, ragged or not
        context = min(_log(rng, 16, 30000), max(16, most), 260000 // batch)
        return _tree("", batch, nodes, context, hq, hkv, width, rng.choice((0.0, 0.0, 20.0, 50.0)), rng.random() < 0.5,
                     rng.choice((16, 32, 64, 64, 128)), ragged, rng.choice((0, 0, 0, 512)))
    if kind == "layout":
        return _layout("", _log(rng, 1, 64), _log(rng, 1, 250), _log(rng, 1, 100000), width, ragged)
    if kind == "accept":
        return _accept("", _log(rng, 1, 64), _log(rng, 1, 130), _log(rng, 1, 1000), rng.choice((1, 3, 16)), rng.choice((8, 4, 1)),
                       rng.randint(0, 8), width, rng.choice((16, 32, 64, 128)), ragged)
    if kind == "select":
        requests, beams = _log(rng, 1, 64), _log(rng, 1, 20)
        vocab = min(_log(rng, 300, 250000), 64 * 8 * 248320 // (requests * beams))
        return _select("", requests, beams, vocab, rng.choice((beams, 2 * beams, _log(rng, 1, 64))), rng.choice(("float32", "float32", "bfloat16")),
                       rng.random() < 0.3, rng.random() < 0.2)
    what = rng.choice(("pages", "states", "rows"))
    requests, beams = _log(rng, 1, 12), _log(rng, 1, 20)
    layers = _log(rng, 1, max(1, min(48, 48 * 16 // (requests * beams))))
    return _reorder("", requests, beams, what, layers, {"pages": rng.choice((2, 4, 8)), "states": rng.choice((4, 16, 32)), "rows": _log(rng, 1, 30000)}[what],
                    rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, *more):
    g = torch.Generator(device=DEV)
    g.manual_seed(sum(m * 8191 ** (i + 1) for i, m in enumerate(more)) + int(seed) * 1_000_003)
    return g


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def _ragged(n, i, on):
    """Length of sequence ``i`` of nominally ``n``: 60 to 140 of 100 parts of it."""
    return max(1, n * (60 + (i * 37) % 81) // 100) if on else n


def _lengths(case):
    """Rows of every sequence's tree, and its keys with them."""
    rows = [_ragged(case["nodes"], i, case["ragged"]) for i in range(case["batch"])]
    return rows, [n + _ragged(case["context"], 2 * i + 1, case["ragged"]) for i, n in enumerate(rows)]


def _trees(case, g):
    """A tree for every sequence: each node continues one of the ``width`` + 1 nodes before it (0: a chain), the first one the context."""
    rows, keys = _lengths(case)
    most = max(rows)
    node = torch.arange(most, device=DEV)
    back = (torch.rand(len(rows), most, generator=g, device=DEV) * (case["width"] + 1)).long()
    parent = (node - 1 - back).clamp(min=0)
    parent[:, 0] = -1
    there = node < torch.tensor(rows, device=DEV)[:, None]
    start = [sum(rows[:i]) for i in range(len(rows))]
    return {"rows": rows, "keys": keys, "most": most, "parents": parent[there].to(torch.int32), "q_start": _i32(start), "q_len": _i32(rows), "kv_len": _i32(keys)}


def _table(g, lengths, bs):
    """Page table of sequences of these lengths, -1 behind their pages, and the number of pages."""
    counts = torch.tensor([(n + bs - 1) // bs for n in lengths], device=DEV)
    total = int(counts.sum()) + 2
    there = torch.arange(int(counts.max()), device=DEV) < counts[:, None]
    table = torch.full(there.shape, -1, dtype=torch.int32, device=DEV)
    table[there] = torch.randperm(total, generator=g, device=DEV)[:total - 2].to(torch.int32)
    return table, total


def _tree_inputs(case, seed):
    g = _gen(seed, 1, case["nodes"])
    s = _trees(case, g)
    hq, hkv, bs, t = case["hq"], case["hkv"], case["bs"], sum(s["rows"])
    s["table"], pages = _table(g, s["keys"], bs)
    s["k"] = torch.randn(pages, hkv, bs, D, generator=g, device=DEV, dtype=torch.bfloat16)
    s["v"] = torch.randn(pages, hkv, bs, D, generator=g, device=DEV, dtype=torch.bfloat16)
    u = torch.randn(hkv, D, generator=g, device=DEV)                     # every sequence's first key is one that many rows look at
    s["k"][s["table"][:, 0].long(), :, 0] += u.bfloat16()
    weight = torch.linspace(0.0, 0.6, hq, device=DEV)[None, :, None]
    s["q"] = (torch.randn(t, hq, D, generator=g, device=DEV) * 1.5 + weight * u.repeat_interleave(hq // hkv, 0)).bfloat16()
    s["gate"] = torch.randn(t, hq, D, generator=g, device=DEV).bfloat16() if case["gate"] else None
    where, mask = _run_layout(s | {"case": case}, plain=True)            # a user's program has them from its layout, once for all layers
    s["mask"] = mask
    s["lo"] = (where - case["window"] + 1).clamp(min=0).to(torch.int32) if case["window"] else None
    return s


def _layout_inputs(case, seed):
    return _trees(case, _gen(seed, 2, case["nodes"]))


def _accept_inputs(case, seed):
    """Drafts of which the target agrees with the first ``taken`` on the way to a sequence's last node."""
    g = _gen(seed, 3, case["nodes"])
    s = _trees(case, g)
    t, layers = sum(s["rows"]), case["layers"]
    s["table"], pages = _table(g, s["keys"], case["bs"])
    s["tokens"] = torch.randint(0, 5000, (t,), generator=g, device=DEV).to(torch.int32)
    parents, there = _padded(s["parents"], s), _there(s)
    seen = _ancestors(parents, there)
    last = seen[torch.arange(len(s["rows"]), device=DEV), s["q_len"].long() - 1]
    agreed = last & (seen.sum(-1) - 1 <= case["taken"]) & (parents >= 0)
    predicted = torch.randint(0, 5000, there.shape, generator=g, device=DEV)
    predicted.scatter_(1, torch.where(agreed, parents, there.shape[1] - 1), torch.where(agreed, _padded(s["tokens"], s), predicted[:, -1:]))
    s["predicted"] = predicted[there].to(torch.int32)
    s["caches"] = [torch.randn(layers, pages, case["hkv"], case["bs"], D, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    s["max_path"] = case["taken"] + 3
    return s


def _select_inputs(case, seed):
    g = _gen(seed, 4, case["beams"])
    b, w, v = case["requests"], case["beams"], case["vocab"]
    logits = torch.randn(b, w, v, generator=g, device=DEV) * 2.5
    likely = torch.randint(0, v, (b, w, 40), generator=g, device=DEV)   # and some tokens that stand out
    logits.scatter_reduce_(2, likely, torch.rand(b, w, 40, generator=g, device=DEV) * 12 + 4, "amax")
    scores = -torch.rand(b, w, generator=g, device=DEV) * 6 - 10
    if case["first"]:                                                    # a request begins with one beam
        scores[:, 1:] = -math.inf
        scores[:, 0] = 0
    finished = torch.rand(b, w, generator=g, device=DEV) < 0.2 if case["finished"] else None
    return {"logits": logits.to(getattr(torch, case["dtype"])), "scores": scores, "finished": finished, "pad": 1}


def _states(case):
    """Shapes, types and slot axis of the tensors whose slots follow the beams; 0 in the place of the number of slots."""
    n, size = case["layers"], case["size"]
    if case["what"] == "pages":
        return [((n, 0, size, 64, D), torch.bfloat16)] * 2, 1
    if case["what"] == "states":                                         # recurrent state and convolution tail of every layer
        return [((0, n, size, D, D), torch.float32), ((0, n, 3, size * 2 * D), torch.bfloat16)], 0
    return [((0, n, size), torch.bfloat16), ((0, size), torch.int32)], 0        # rows of any length, tables


def _reorder_inputs(case, seed):
    g = _gen(seed, 5, case["beams"])
    b, w = case["requests"], case["beams"]
    parents = torch.randint(0, w, (b, w), generator=g, device=DEV)
    if case["idle"]:                                                     # beams that have come to nothing
        parents = torch.where(torch.rand(b, w, generator=g, device=DEV) < 0.2, -1, parents)
    slots = torch.randperm(b * w + 2, generator=g, device=DEV)[:b * w].view(b, w)
    shapes, dim = _states(case)
    states = [torch.randint(0, 30000, tuple(x or b * w + 2 for x in shape), generator=g, device=DEV, dtype=dtype) if dtype == torch.int32 else
              torch.randn(tuple(x or b * w + 2 for x in shape), generator=g, device=DEV, dtype=dtype) for shape, dtype in shapes]
    return {"states": states, "dim": dim, "parents": parents.to(torch.int32), "slots": slots.to(torch.int32)}


INPUTS = {"tree": _tree_inputs, "layout": _layout_inputs, "accept": _accept_inputs, "select": _select_inputs, "reorder": _reorder_inputs}


@torch.no_grad()
def prepare(case, seed):
    return {"case": case} | INPUTS[case["kind"]](case, seed)


# ------------------------------------------------------------------------------------------------ one pass
@torch.no_grad()
def run(state):
    return {"tree": _run_tree, "layout": _run_layout, "accept": _run_accept, "select": _run_select, "reorder": _run_reorder}[state["case"]["kind"]](state)


def _there(s):
    """[B, most]: nodes that a sequence has."""
    return torch.arange(s["most"], device=DEV) < s["q_len"][:, None]


def _rows_at(s):
    """[B, most]: row of every node."""
    return (s["q_start"][:, None] + torch.arange(s["most"], device=DEV)).clamp(max=s["parents"].shape[0] - 1)


def _padded(x, s):
    return torch.where(_there(s), x[_rows_at(s)].long(), -1)


def _ancestors(parents, there):
    """[B, n, n]: node j is node i or one that it continues, by steps of twice the length each."""
    n = parents.shape[1]
    node = torch.arange(n, device=DEV)
    seen = ((node == parents[..., None]) | (node == node[:, None])).float() * there[..., None]
    for _ in range(max(1, (n - 1).bit_length())):
        seen = (seen @ seen > 0).float()
    return seen > 0


def _run_layout(s, plain=False):
    if own and not plain:
        from deepseek_v4_2080ti_b200.ops import tree
        return tree.layout(s["parents"], s["q_start"], s["q_len"], s["kv_len"], s["most"])
    there = _there(s)
    seen = _ancestors(_padded(s["parents"], s), there)
    where = (s["kv_len"] - s["q_len"])[:, None] + seen.sum(-1) - 1
    words = (s["most"] + 31) // 32
    bits = torch.nn.functional.pad(seen.long(), (0, 32 * words - s["most"])).unflatten(-1, (words, 32))
    mask = (bits << torch.arange(32, device=DEV)).sum(-1)
    mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask)
    return where[there].to(torch.int32), mask[there].to(torch.int32)


def _run_tree(s):
    c = s["case"]
    if own:
        from deepseek_v4_2080ti_b200.ops import attention
        return attention.decode_tree(s["q"], s["k"], s["v"], s["table"], s["mask"], s["q_start"], s["q_len"], s["kv_len"], s["most"],
                                     lo=s["lo"], gate=s["gate"], cap=c["cap"], max_kv_len=max(s["keys"]))
    hkv, g, n, b = c["hkv"], c["hq"] // c["hkv"], s["most"], c["batch"]
    at, there = _rows_at(s), _there(s)
    keys = s["table"].shape[1] * c["bs"]
    lay = lambda cache: cache[s["table"].clamp(min=0)].transpose(1, 2).reshape(b * hkv, keys, D).float()
    q = s["q"][at].float().view(b, n, hkv, g, D).permute(0, 2, 3, 1, 4).reshape(b * hkv, g * n, D)
    x = (q @ lay(s["k"]).transpose(1, 2)) / math.sqrt(D)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    j = torch.arange(keys, device=DEV)
    node = j - (s["kv_len"] - s["q_len"])[:, None]                       # [B, keys]: node of a key, below 0 in the context
    word = s["mask"][at].gather(2, (node.clamp(0, n - 1) // 32)[:, None].expand(b, n, keys))
    in_tree = (word >> (node.clamp(0, n - 1) % 32)[:, None].int()) & 1 > 0
    seen = torch.where((node < 0)[:, None], torch.ones_like(in_tree), in_tree & (node < s["q_len"][:, None])[:, None])
    if s["lo"] is not None:
        seen &= j >= s["lo"][at][..., None]
    x = x.view(b, hkv, g, n, keys).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    o = (p.view(b * hkv, g * n, keys) @ lay(s["v"])).view(b, hkv, g, n, D) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, c["hq"], D)[there]
    return (o if s["gate"] is None else o * torch.sigmoid(s["gate"].float())).bfloat16()


def _run_accept(s):
    c = s["case"]
    if own:
        from deepseek_v4_2080ti_b200.ops import tree
        path, count, emitted = tree.accept(s["tokens"], s["parents"], s["predicted"], s["q_start"], s["q_len"], s["max_path"], s["kv_len"], s["table"],
                                           s["caches"])
        return {"path": path, "count": count, "emitted": emitted, "k": s["caches"][0], "v": s["caches"][1]}
    there = _there(s)
    n, most = s["most"], s["max_path"]
    tokens, parents, predicted = (_padded(s[x], s) for x in ("tokens", "parents", "predicted"))
    agrees = there & (parents >= 0) & (tokens == predicted.gather(1, parents.clamp(min=0)))
    node = torch.arange(n, device=DEV)
    earlier = agrees[:, None] & (parents[:, None] == parents[..., None]) & (node < node[:, None])        # a sibling before it that agrees too
    agrees &= ~earlier.any(-1)
    agrees[:, 0] = there[:, 0]
    seen = _ancestors(parents, there)
    depth = seen.sum(-1) - 1
    taken = there & ~(seen & ~agrees[:, None]).any(-1) & (depth < most)
    count = taken.sum(-1)
    path = torch.full((c["batch"], most + 1), -1, dtype=torch.long, device=DEV)
    path.scatter_(1, torch.where(taken, depth, most), torch.where(taken, node, -1))
    path = path[:, :most]
    emitted = torch.where(path >= 0, predicted.gather(1, path.clamp(min=0)), -1)
    seq, i = (path >= 0).nonzero(as_tuple=True)
    first = (s["kv_len"] - s["q_len"]).long()[seq]
    src, dst, bs = first + path[seq, i], first + i, c["bs"]
    page = lambda pos: s["table"][seq, pos // bs].long()
    for cache in s["caches"]:
        cache[:, page(dst), :, dst % bs] = cache[:, page(src), :, src % bs]
    return {"path": path.to(torch.int32), "count": count.to(torch.int32), "emitted": emitted.to(torch.int32), "k": s["caches"][0], "v": s["caches"][1]}


def _run_select(s):
    c, n = s["case"], s["case"]["n"]
    if own:
        from deepseek_v4_2080ti_b200.ops import beams
        return beams.select(s["logits"], s["scores"], n, finished=s["finished"], pad_token=s["pad"])
    b, w, v = s["logits"].shape
    x = s["logits"].double()                                             # (borders between beams lie closer than 32 bits tell apart)
    x -= x.amax(-1, keepdim=True)
    x -= x.exp().sum(-1, keepdim=True).log()
    x += s["scores"].double()[..., None]
    if s["finished"] is not None:
        pad = (torch.arange(v, device=DEV) == s["pad"]) & s["finished"][..., None]
        x = torch.where(s["finished"][..., None], torch.where(pad, s["scores"].double()[..., None], -math.inf), x)
    x = x.view(b, w * v)
    n_of = min(n, w * v)
    least = torch.topk(x, n_of).values[:, -1:]
    above, equal = x > least, x == least
    chosen = above | (equal & (equal.cumsum(-1) <= n_of - above.sum(-1, keepdim=True)))  # of equals the first ones
    flat = chosen.nonzero()[:, 1].view(b, n_of)
    score, order = x.gather(1, flat).sort(dim=-1, descending=True, stable=True)
    flat = torch.where(score > -math.inf, flat.gather(1, order), -1)
    pad_to = (0, n - n_of)
    out = lambda t, fill, dtype: torch.nn.functional.pad(t, pad_to, value=fill).to(dtype)
    return (out(score, -math.inf, torch.float32), out(torch.where(flat >= 0, flat // v, -1), -1, torch.int32),
            out(torch.where(flat >= 0, flat % v, -1), -1, torch.int32))


def _run_reorder(s):
    if own:
        from deepseek_v4_2080ti_b200.ops import beams
        beams.reorder(s["states"], s["parents"], s["slots"], dim=s["dim"])
        return list(s["states"])
    w = s["parents"].shape[1]
    parents = torch.where(s["parents"] >= 0, s["parents"], torch.arange(w, device=DEV)).long()
    to, source = s["slots"].reshape(-1).long(), s["slots"].gather(1, parents).reshape(-1).long()
    return [x.index_copy_(s["dim"], to, x.index_select(s["dim"], source)) for x in s["states"]]


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    kind = case["kind"]
    if kind == "select":
        rows = case["requests"] * case["beams"]
        if case["first"]:
            rows = case["requests"]
        elif case["finished"]:
            rows = rows * 0.8
        return {"bytes": rows * case["vocab"] * (4 if case["dtype"] == "float32" else 2) + case["requests"] * case["n"] * 12, "flops": rows * case["vocab"] * 4.0}
    if kind == "reorder":
        b, w = case["requests"], case["beams"]
        keep = 0.8 if case["idle"] else 1.0
        moved = w * keep * (1 - 1 / w)                                   # beams that continue another one, and the others that some beam continues
        wanted = w * (1 - (1 - keep * (1 - 1 / w) / max(1, w - 1)) ** (w - 1)) if w > 1 else 0.0
        size = sum(math.prod(x or 1 for x in shape) * dtype.itemsize for shape, dtype in _states(case)[0])
        return {"bytes": b * (moved + wanted) * size + b * w * 8, "flops": 0}
    rows, keys = _lengths(case)
    if kind == "layout":
        return {"bytes": sum(rows) * (8 + 4 * ((max(rows) + 31) // 32)) + 12 * len(rows), "flops": 0}
    if kind == "accept":
        kept = sum(min(case["taken"], max(0, n - 1)) for n in rows)
        return {"bytes": kept * case["layers"] * case["hkv"] * D * 2 * 2 * 2 + sum(rows) * 12, "flops": 0}
    hq, hkv = case["hq"], case["hkv"]
    context = [k - n if not case["window"] else min(k - n, case["window"]) for k, n in zip(keys, rows)]
    return {"bytes": sum(n + c for n, c in zip(rows, context)) * 2 * hkv * D * 2 + sum(rows) * (hq * D * 2 * (3 if case["gate"] else 2) + 4 * ((max(rows) + 31) // 32)),
            "flops": 4.0 * D * hq * sum(n * (c + 1) for n, c in zip(rows, context))}


# ------------------------------------------------------------------------------------------------ 64-bit statement
def _chains(s):
    """For every row the nodes from its tree's first one down to it, and the sequence that it belongs to, walked one by one."""
    parents, out = s["parents"].tolist(), []
    for b, n in enumerate(s["rows"]):
        base = sum(s["rows"][:b])
        mine = []
        for i in range(n):
            up = parents[base + i]
            mine.append((mine[up] if up >= 0 else []) + [i])
        out.append(mine)
    return out


def _exact_tree(case, seed):
    s = _tree_inputs(case, seed)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    g, at = case["hq"] // case["hkv"], 0
    for b, chains in enumerate(_chains(s)):
        n, kv = s["rows"][b], s["keys"][b]
        hidden = torch.ones(n, kv, dtype=torch.bool)
        hidden[:, :kv - n] = False
        for i, chain in enumerate(chains):
            hidden[i, [kv - n + x for x in chain]] = False
            if case["window"]:
                hidden[i, :max(0, kv - n + len(chain) - case["window"])] = True
        hidden = hidden.to(DEV)
        j = torch.arange(kv, device=DEV)
        page = s["table"][b].long()[j // case["bs"]]
        for h in range(case["hkv"]):
            k, v = (s[c][page, h, j % case["bs"]].double() for c in "kv")
            x = torch.einsum("tgd,kd->gtk", s["q"][at:at + n, h * g:(h + 1) * g].double(), k) * D ** -0.5
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            w = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, h * g:(h + 1) * g] = torch.einsum("gtk,kd->tgd", w, v)
        at += n
    return out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].double()))


def _exact_layout(case, seed):
    s = _layout_inputs(case, seed)
    words = (s["most"] + 31) // 32
    where, mask = [], []
    for b, chains in enumerate(_chains(s)):
        for chain in chains:
            where.append(s["keys"][b] - s["rows"][b] + len(chain) - 1)
            bits = sum(1 << x for x in chain)
            mask.append([((bits >> (32 * w) & 0xFFFFFFFF) + 2 ** 31) % 2 ** 32 - 2 ** 31 for w in range(words)])
    return _i32(where), _i32(mask)


def _exact_accept(case, seed):
    s = _accept_inputs(case, seed)
    tokens, parents, predicted = (s[x].tolist() for x in ("tokens", "parents", "predicted"))
    paths, counts, emitted, at = [], [], [], 0
    for n in s["rows"]:
        path = [0]
        while len(path) < s["max_path"]:
            c = path[-1]
            child = [x for x in range(c + 1, n) if parents[at + x] == c and tokens[at + x] == predicted[at + c]]
            if not child:
                break
            path.append(child[0])
        fill = [-1] * (s["max_path"] - len(path))
        paths.append(path + fill)
        counts.append(len(path))
        emitted.append([predicted[at + x] for x in path] + fill)
        at += n
    return {"path": _i32(paths), "count": _i32(counts), "emitted": _i32(emitted), "k": None, "v": None}


def _exact_select(case, seed):
    s, n = _select_inputs(case, seed), case["n"]
    b, w, v = s["logits"].shape
    scores = torch.full((b, n), -math.inf, dtype=torch.float64, device=DEV)
    parents, tokens = (torch.full((b, n), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    for r in range(b):
        total = torch.log_softmax(s["logits"][r].double(), -1) + s["scores"][r].double()[:, None]
        for i in range(w):
            if s["finished"] is not None and bool(s["finished"][r, i]):
                total[i] = -math.inf
                total[i, s["pad"]] = s["scores"][r, i].double()
        value, index = torch.sort(total.reshape(-1), descending=True, stable=True)
        m = min(n, int((value > -math.inf).sum()))
        scores[r, :m], parents[r, :m], tokens[r, :m] = value[:m], (index[:m] // v).int(), (index[:m] % v).int()
    return scores, parents, tokens


@torch.no_grad()
def exact(case, seed):
    if case["kind"] == "reorder":                                        # (nothing is computed)
        return None
    return {"tree": _exact_tree, "layout": _exact_layout, "accept": _exact_accept, "select": _exact_select}[case["kind"]](case, seed)
