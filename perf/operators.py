"""The attention operators for requests over shared prompts of documents and images, as they are timed.

``append``: ``attention.qk_norm_rope_axes_append`` - norm of queries and keys, rotation by positions with three axes (time,
height, width), keys and values to their pages.

``spans``: ``attention.prefill_spans`` - prompt rows that each see a span of keys of their own: packed documents, blocks of an
image that see each other, windows, plain causal rows after a context; scores capped by a tanh or not.

``shared``: ``attention.decode_shared`` - one row per sequence, groups of sequences that hold the same leading pages.

All over bf16 pages [pages, kv heads, page size, 128].  Head counts are those of this framework's configurations (40 / 8 with
an output gate, 48 / 8) and generic ones.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
D, EPS, THETA = 128, 1e-6, 1e7


# ------------------------------------------------------------------------------------------------ cases
def _append(name, tokens, hq, hkv, sections, interleaved=True, gate=False, layout="text", bs=64, padded=False):
    return {"name": name, "kind": "append", "tokens": tokens, "hq": hq, "hkv": hkv, "sections": ",".join(map(str, sections)),
            "interleaved": interleaved, "gate": gate, "layout": layout, "bs": bs, "padded": padded}


def _spans(name, batch, new, past, hq, hkv, layout, cap=0.0, gate=False, bs=64, ragged=False):
    return {"name": name, "kind": "spans", "batch": batch, "new": new, "past": past, "hq": hq, "hkv": hkv, "layout": layout,
            "cap": cap, "gate": gate, "bs": bs, "ragged": ragged}


def _shared(name, batch, groups, prefix, tail, hq, hkv, cap=0.0, gate=False, bs=64, ragged=False):
    return {"name": name, "kind": "shared", "batch": batch, "groups": groups, "prefix": prefix, "tail": tail, "hq": hq, "hkv": hkv,
            "cap": cap, "gate": gate, "bs": bs, "ragged": ragged}


def listed():
    return [
        _append("axes_1", 1, 40, 8, (6, 5, 5), gate=True),                                  # decoding one sequence
        _append("axes_batch_37", 37, 48, 8, (24, 20, 20), padded=True),                     # a captured decode batch with idle rows
        _append("axes_image_1369", 1369, 28, 4, (16, 24, 24), interleaved=False, layout="image"),   # an image of 37 x 37 patches
        _append("axes_prompt_8192", 8192, 40, 8, (12, 10, 10), gate=True, layout="mixed"),  # a whole prompt portion, text and images
        _spans("spans_verify_9", 4, 9, 1500, 40, 8, "causal", gate=True, ragged=True),      # a few rows each after a context
        _spans("spans_image_1025", 1, 1025, 333, 32, 8, "image", bs=16),                    # an image behind some text, its patches see each other
        _spans("spans_documents_4000", 1, 4000, 0, 48, 8, "documents", cap=30.0),           # documents packed into one portion, capped
        _spans("spans_prompt_8192", 1, 8192, 0, 40, 8, "causal", gate=True),                # the benchmark's prompt
        _shared("shared_3x700", 3, 1, 700, 40, 40, 8, gate=True),                           # a few questions on a short page
        _shared("shared_24x5000_groups", 24, 5, 5000, 300, 48, 8, cap=50.0, ragged=True, bs=32),    # several documents at once, ragged
        _shared("shared_32x8192", 32, 1, 8192, 128, 40, 8, gate=True),                      # the benchmark's decode batch on its prompt
        _shared("shared_64x32768", 64, 1, 32768, 500, 40, 8, gate=True, ragged=True),       # a busy server on one long document
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((40, 8), (48, 8), (32, 8), (28, 4), (16, 16), (16, 2), (5, 1))


def draw(rng):
    kind = rng.choice(("append", "spans", "shared"))
    hq, hkv = rng.choice(HEADS)
    bs, gate = rng.choice((16, 32, 64, 64, 128)), rng.random() < 0.5
    if kind == "append":
        sections = rng.choice(((6, 5, 5), (12, 10, 10), (16, 24, 24), (24, 20, 20), (8, 4, 4), (32, 0, 0)))
        interleaved = rng.random() < 0.5 and sections[1] <= sections[0]          # taking turns needs axes of about one length
        return _append("", _log(rng, 1, 8192), hq, hkv, sections, interleaved, gate, rng.choice(("text", "image", "mixed")), bs, rng.random() < 0.3)
    cap = rng.choice((0.0, 0.0, 20.0, 50.0))
    if kind == "spans":
        batch = rng.choice((1, 1, 2, 3, 7))
        new = _log(rng, 1, 8000 // batch)
        past = rng.choice((0, 0, _log(rng, 16, 8000 // batch)))
        if (new + past) * new * batch > 8192 * 8192 // 2:               # the work of the listed prompt at most
            past = 0
        return _spans("", batch, new, past, hq, hkv, rng.choice(("causal", "documents", "image", "window")), cap, gate, bs, rng.random() < 0.5)
    batch = _log(rng, 2, 64)
    prefix = _log(rng, 64, 32768)
    tail = _log(rng, 1, max(2, min(1000, 32000 // batch)))
    return _shared("", batch, rng.randint(1, max(1, min(6, batch // 2))), prefix, tail, hq, hkv, cap, gate, bs, rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, *more):
    g = torch.Generator(device=DEV)
    n = int(seed) * 1_000_003
    for m in more:
        n = n * 8191 + m
    g.manual_seed(n % (1 << 62))
    return g


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def _share(n, parts, i):
    return (n * (i + 1)) // parts - (n * i) // parts


def _ragged(n, i, on):
    """Length of sequence ``i`` of nominally ``n``: 60 to 140 of 100 parts of it."""
    return max(1, n * (60 + (i * 37) % 81) // 100) if on else n


def _axes(case):
    """Axis of every rotary pair: blocks of ``sections`` pairs, or time, height, width in turn while they last."""
    sec = [int(x) for x in case["sections"].split(",")]
    if not case["interleaved"]:
        return sec, [a for a, n in enumerate(sec) for _ in range(n)]
    axis = [0] * sum(sec)
    for a in (1, 2):
        for j in range(sec[a]):
            axis[a + 3 * j] = a
    return sec, axis


def _append_inputs(case, seed):
    g = _gen(seed, 1)
    t, hq, hkv, bs = case["tokens"], case["hq"], case["hkv"], case["bs"]
    rot = 2 * sum(_axes(case)[0])
    width = hq * D * (2 if case["gate"] else 1) + 2 * hkv * D
    src = (torch.randn(t, width, generator=g, device=DEV) * 1.5).bfloat16()
    gamma = lambda: (torch.randn(D, generator=g, device=DEV) * 0.1).bfloat16()
    # text counts on all axes at once, an image stands still in time while its patches count rows and columns
    start = int(torch.randint(0, 100_000, (1,), generator=g, device=DEV))
    n = torch.arange(t, device=DEV)
    text = (n + start).expand(3, t)
    side = max(1, math.isqrt(t if case["layout"] == "image" else 900))
    image = torch.stack([torch.zeros_like(n), n // side, n % side]) + start
    pos = {"text": text, "image": image, "mixed": torch.where(n // 1000 % 2 == 1, image + n // 1000 * 1000, text)}[case["layout"]]
    pages = (t + bs - 1) // bs
    perm = torch.randperm(pages + 2, generator=g, device=DEV)[:pages]
    slots = perm[n // bs] * bs + n % bs
    if case["padded"]:
        slots = torch.where(n % 5 == 4, -1, slots)                   # rows of a captured batch without a request
    inv = (1.0 / (THETA ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))).float().to(DEV)
    return {"src": src, "q_gamma": gamma(), "k_gamma": gamma(), "inv": inv, "pos": pos.to(torch.int32).contiguous(),
            "slots": slots.to(torch.int32), "pages": pages + 2}


def _span_lengths(case):
    """(new rows, context with them) of every sequence."""
    return [(_ragged(case["new"], i, case["ragged"]), _ragged(case["new"], i, case["ragged"]) + _ragged(case["past"], 2 * i + 1, case["ragged"]))
            for i in range(case["batch"])] if case["past"] else \
           [(_ragged(case["new"], i, case["ragged"]),) * 2 for i in range(case["batch"])]


def _span_rows(case):
    """int64 lo, hi [rows]: the keys that every row sees."""
    lo, hi = [], []
    for i, (new, kv) in enumerate(_span_lengths(case)):
        p = torch.arange(kv - new, kv)
        l, h = torch.zeros_like(p), p + 1
        if case["layout"] == "documents":                            # documents of 200 to 900 tokens, each on its own
            ends, at, k = [], 0, i
            while at < kv:
                at += 200 + (k * 331) % 701
                ends.append(at)
                k += 1
            l = torch.tensor([0] + ends)[torch.bucketize(p, torch.tensor(ends), right=True)]
        elif case["layout"] == "image":                              # blocks of 900 see all of themselves, 100 rows of text between them
            block = p % 1000
            h = torch.where(block < 900, torch.clamp(p - block + 900, max=kv), h)
        elif case["layout"] == "window":
            l = torch.clamp(p - 511, min=0)
        lo.append(l)
        hi.append(h)
    return torch.cat(lo), torch.cat(hi)


def _pool(g, lengths, hkv, bs, first, table=None, pool=None):
    """Pages with the keys and values of sequences of ``lengths`` and their table; ``first`` marks the keys that many rows look at."""
    counts = [(n + bs - 1) // bs for n in lengths]
    total = sum(counts) + 2
    u = torch.randn(hkv, D, generator=g, device=DEV)
    k = torch.randn(total, hkv, bs, D, generator=g, device=DEV).bfloat16()
    v = torch.randn(total, hkv, bs, D, generator=g, device=DEV).bfloat16()
    perm = torch.randperm(total, generator=g, device=DEV)
    table = torch.zeros(len(lengths), max(counts), dtype=torch.long, device=DEV)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = perm[at:at + c]
        at += c
        for j in first[i]:
            k[table[i, j // bs], :, j % bs] += u.bfloat16()
    return k, v, table, u


def _queries(g, rows, hq, u):
    """Rows that look at the marked keys, some heads more than others."""
    q = torch.randn(rows, hq, D, generator=g, device=DEV) * 1.5
    w = torch.linspace(0.0, 0.6, hq, device=DEV)
    return (q + w[None, :, None] * u.repeat_interleave(hq // u.shape[0], 0)[None]).bfloat16()


def _spans_inputs(case, seed):
    g = _gen(seed, 2)
    lens = _span_lengths(case)
    lo, hi = _span_rows(case)
    ends = [0]
    for new, _ in lens:
        ends.append(ends[-1] + new)
    first = [sorted(set(lo[a:b].tolist())) if case["layout"] == "documents" else [0] for a, b in zip(ends, ends[1:])]
    k, v, table, u = _pool(g, [kv for _, kv in lens], case["hkv"], case["bs"], first)
    q = _queries(g, ends[-1], case["hq"], u)
    gate = torch.randn(q.shape, generator=g, device=DEV).bfloat16() if case["gate"] else None
    return {"q": q, "k": k, "v": v, "table": _i32(table), "gate": gate, "lo": _i32(lo), "hi": _i32(hi), "q_start": _i32(ends[:-1]),
            "q_len": _i32([n for n, _ in lens]), "kv_len": _i32([kv for _, kv in lens])}


def _group_lengths(case):
    """[(shared keys, [keys of every sequence])] of the groups."""
    out, row = [], 0
    for i in range(case["groups"]):
        shared = _ragged(case["prefix"], i, case["ragged"])
        n = _share(case["batch"], case["groups"], i)
        out.append((shared, [shared + _ragged(case["tail"], row + j, case["ragged"]) for j in range(n)]))
        row += n
    return out


def _shared_inputs(case, seed):
    g = _gen(seed, 3)
    bs = case["bs"]
    groups = _group_lengths(case)
    own_len, shared_rows, starts = [], [], [0]
    for i, (shared, lens) in enumerate(groups):
        whole = shared // bs                                         # whole pages are shared; the rest of the prefix is every sequence's own
        shared_rows.append(whole * bs)
        own_len += [n - whole * bs for n in lens]
        starts.append(starts[-1] + len(lens))
    lengths = [n for n in shared_rows if n] + own_len
    n_pre = len(lengths) - len(own_len)
    k, v, table, u = _pool(g, lengths, case["hkv"], bs, [[0]] * n_pre + [[]] * len(own_len))
    kv = [n for _, lens in groups for n in lens]
    wide = max((n + bs - 1) // bs for n in kv)
    full = torch.zeros(len(kv), wide, dtype=torch.long, device=DEV)
    pre = 0
    for i, shared in enumerate(shared_rows):
        w = shared // bs
        for b in range(starts[i], starts[i + 1]):
            full[b, :w] = table[pre, :w]
            c = (own_len[b] + bs - 1) // bs
            full[b, w:w + c] = table[n_pre + b, :c]
        pre += shared > 0
    q = _queries(g, len(kv), case["hq"], u)
    gate = torch.randn(q.shape, generator=g, device=DEV).bfloat16() if case["gate"] else None
    return {"q": q, "k": k, "v": v, "table": _i32(full), "gate": gate, "kv_len": _i32(kv), "group_start": _i32(starts), "shared_len": _i32(shared_rows)}


INPUTS = {"append": _append_inputs, "spans": _spans_inputs, "shared": _shared_inputs}


def prepare(case, seed):
    s = {"case": case} | INPUTS[case["kind"]](case, seed)
    if case["kind"] == "append":
        s["k"] = torch.zeros(s["pages"], case["hkv"], case["bs"], D, dtype=torch.bfloat16, device=DEV)
        s["v"] = torch.zeros_like(s["k"])
    elif case["kind"] == "spans":                                    # a scheduler knows its portions' lengths
        s["lens"] = _span_lengths(case)
    else:
        s["kv_host"] = [n for _, lens in _group_lengths(case) for n in lens]
        s["shared_host"] = [n // case["bs"] * case["bs"] for n, _ in _group_lengths(case)]
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"append": _run_append, "spans": _run_spans, "shared": _run_shared}[state["case"]["kind"]](state)


def _offsets(case):
    """Columns of a projection row: q (with its gate behind every head), k, v."""
    qw = case["hq"] * D * (2 if case["gate"] else 1)
    return qw, qw + case["hkv"] * D


def _run_append(s):
    c = s["case"]
    ko, vo = _offsets(c)
    if own:
        from deepseek_v4_2080ti_b200.ops import attention
        axes = attention.rotary_axes([int(x) for x in c["sections"].split(",")], c["interleaved"])
        q, gate = attention.qk_norm_rope_axes_append(
            s["src"], 0, D * (2 if c["gate"] else 1), c["gate"], s["src"], ko, s["src"], vo, s["q_gamma"], s["k_gamma"], True, EPS,
            s["inv"], axes, s["pos"], s["slots"], s["k"], s["v"], c["hq"], c["hkv"])
        return {"q": q, "gate": gate, "k": s["k"], "v": s["v"]}
    t, hq, hkv, bs = c["tokens"], c["hq"], c["hkv"], c["bs"]
    src = s["src"].float()
    qg = src[:, :ko].view(t, hq, -1)
    axis = torch.tensor(_axes(c)[1], device=DEV)
    ang = s["pos"].double()[axis].t() * s["inv"].double()            # [T, rot / 2]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def prep(x, gamma):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + gamma.float())
        h = cos.shape[-1]
        a, b = x[..., :h], x[..., h:2 * h]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1).bfloat16()
    q = prep(qg[..., :D], s["q_gamma"])
    gate = qg[..., D:].bfloat16() if c["gate"] else None
    key = prep(src[:, ko:vo].view(t, hkv, D), s["k_gamma"])
    live = s["slots"] >= 0
    at = s["slots"][live].long()
    s["k"][at // bs, :, at % bs] = key[live]
    s["v"][at // bs, :, at % bs] = src[:, vo:].view(t, hkv, D).bfloat16()[live]
    return {"q": q, "gate": gate, "k": s["k"], "v": s["v"]}


def _context(s, row, n):
    """fp32 keys and values [Hkv, n, 128] of the sequence in table row ``row``."""
    pages = s["table"][row, :(n + s["case"]["bs"] - 1) // s["case"]["bs"]].long()
    take = lambda c: c[pages].transpose(0, 1).reshape(c.shape[1], -1, D)[:, :n].float()
    return take(s["k"]), take(s["v"])


def _attend(q, k, v, seen, cap):
    """q [r, Hq, 128], k / v [Hkv, n, 128], seen [r, n] -> [r, Hq, 128]; a row that sees nothing is zero."""
    r, hq, _ = q.shape
    hkv = k.shape[0]
    q = q.view(r, hkv, hq // hkv, D).permute(1, 2, 0, 3).reshape(hkv, -1, D)       # [Hkv, G r, 128]
    x = (q @ k.transpose(1, 2)) / math.sqrt(D)
    if cap:
        x = cap * torch.tanh(x / cap)
    x = x.view(hkv, -1, r, k.shape[1]).masked_fill(~seen, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    o = (p.view(hkv, -1, k.shape[1]) @ v).view(hkv, -1, r, D) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(2, 0, 1, 3).reshape(r, hq, D)


def _gated(o, gate):
    return (o if gate is None else o * torch.sigmoid(gate.float())).bfloat16()


def _run_spans(s):
    c = s["case"]
    if own:
        from deepseek_v4_2080ti_b200.ops import attention
        return attention.prefill_spans(s["q"], s["k"], s["v"], s["table"], s["q_start"], s["q_len"], s["kv_len"], max(n for n, _ in s["lens"]),
                                       s["lo"], s["hi"], gate=s["gate"], cap=c["cap"], max_kv_len=max(n for _, n in s["lens"]))
    out, at = [], 0
    for i, (new, kv) in enumerate(s["lens"]):
        k, v = _context(s, i, kv)
        j = torch.arange(kv, device=DEV)
        for a in range(at, at + new, 1024):
            b = min(a + 1024, at + new)
            seen = (j >= s["lo"][a:b, None]) & (j < s["hi"][a:b, None])
            out.append(_attend(s["q"][a:b].float(), k, v, seen, c["cap"]))
        at += new
    return _gated(torch.cat(out), s["gate"])


def _run_shared(s):
    c = s["case"]
    if own:
        from deepseek_v4_2080ti_b200.ops import attention
        return attention.decode_shared(s["q"], s["k"], s["v"], s["table"], s["kv_len"], s["group_start"], s["shared_len"], gate=s["gate"],
                                       cap=c["cap"], max_shared=max(s["shared_host"]), max_kv_len=max(s["kv_host"]))
    out = []
    for b, n in enumerate(s["kv_host"]):
        k, v = _context(s, b, n)
        out.append(_attend(s["q"][b:b + 1].float(), k, v, torch.ones(1, n, dtype=torch.bool, device=DEV), c["cap"]))
    return _gated(torch.cat(out), s["gate"])


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    hq, hkv = case["hq"], case["hkv"]
    kv_row = 2 * hkv * D * 2
    if case["kind"] == "append":
        t = case["tokens"]
        row = (hq * (2 if case["gate"] else 1) + 2 * hkv) * D * 2
        return {"bytes": t * (2 * row + 4 * 4), "flops": t * (hq + hkv) * D * 8.0}
    rows_bytes = hq * D * 2 * (3 if case["gate"] else 2)
    if case["kind"] == "spans":
        lo, hi = _span_rows(case)
        seen, at = 0, 0
        for new, kv in _span_lengths(case):                          # keys that some row of the sequence sees
            edge = torch.zeros(kv + 1, dtype=torch.long)
            edge.index_add_(0, lo[at:at + new], torch.ones(new, dtype=torch.long))
            edge.index_add_(0, hi[at:at + new], -torch.ones(new, dtype=torch.long))
            seen += int((edge.cumsum(0) > 0).sum())
            at += new
        return {"bytes": lo.numel() * (rows_bytes + 8) + seen * kv_row, "flops": 4.0 * D * hq * float((hi - lo).sum())}
    b = flops = 0.0
    for shared, lens in _group_lengths(case):
        whole = shared // case["bs"] * case["bs"]
        b += whole * kv_row + sum(n - whole for n in lens) * kv_row + len(lens) * rows_bytes
        flops += 4.0 * D * hq * sum(lens)
    return {"bytes": b, "flops": flops}


# ------------------------------------------------------------------------------------------------ 64-bit statement
def _exact_append(case, seed):
    x = _append_inputs(case, seed)
    t, hq, hkv, bs = case["tokens"], case["hq"], case["hkv"], case["bs"]
    heads = x["src"].double().view(t, -1, D)
    per = 2 if case["gate"] else 1
    q, gate = heads[:, :per * hq:per], (heads[:, 1:2 * hq:2] if case["gate"] else None)
    key, val = heads[:, per * hq:per * hq + hkv], heads[:, per * hq + hkv:]
    phase = torch.stack([x["pos"][a].double() * x["inv"][i].double() for i, a in enumerate(_axes(case)[1])], -1)
    turn = torch.polar(torch.ones_like(phase), phase)[:, None]
    half = phase.shape[-1]

    def prep(y, gamma):
        y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * (gamma.double() + 1)
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
        return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)
    kc = torch.zeros(x["pages"] * bs, hkv, D, dtype=torch.float64, device=DEV)
    vc = torch.zeros_like(kc)
    live = (x["slots"] >= 0).nonzero()[:, 0]
    kc[x["slots"][live].long()] = prep(key, x["k_gamma"])[live]
    vc[x["slots"][live].long()] = val[live]
    lay = lambda y: y.view(x["pages"], bs, hkv, D).transpose(1, 2)
    return {"q": prep(q, x["q_gamma"]), "gate": gate, "k": lay(kc), "v": lay(vc)}


def _exact_rows(q, k, v, lo, hi, cap, gate):
    """q [r, 128] of one head, k / v [n, 128]; every row by itself over the keys [lo, hi)."""
    x = torch.einsum("rd,nd->rn", q, k) * D ** -0.5
    if cap:
        x = torch.tanh(x / cap) * cap
    j = torch.arange(k.shape[0], device=DEV)
    hidden = (j[None] < lo[:, None]) | (j[None] >= hi[:, None])
    x[hidden] = -math.inf
    w = torch.softmax(x, -1)
    w[hi <= lo] = 0
    o = torch.einsum("rn,nd->rd", w, v)
    return o if gate is None else o / (1 + torch.exp(-gate))


def _exact_spans(case, seed):
    x = _spans_inputs(case, seed)
    out = torch.empty(x["q"].shape, dtype=torch.float64, device=DEV)
    rep, at = case["hq"] // case["hkv"], 0
    for i, (new, kv) in enumerate(_span_lengths(case)):
        j = torch.arange(kv, device=DEV)
        page = x["table"][i].long()[j // case["bs"]]
        for h in range(case["hq"]):
            k, v = (x[c][page, h // rep, j % case["bs"]].double() for c in "kv")
            for a in range(at, at + new, 4096):
                rows = slice(a, min(a + 4096, at + new))
                out[rows, h] = _exact_rows(x["q"][rows, h].double(), k, v, x["lo"][rows], x["hi"][rows], case["cap"],
                                           None if x["gate"] is None else x["gate"][rows, h].double())
        at += new
    return out


def _exact_shared(case, seed):
    x = _shared_inputs(case, seed)
    out = torch.empty(x["q"].shape, dtype=torch.float64, device=DEV)
    rep = case["hq"] // case["hkv"]
    lens = [n for _, g in _group_lengths(case) for n in g]
    for b, n in enumerate(lens):
        j = torch.arange(n, device=DEV)
        page = x["table"][b].long()[j // case["bs"]]
        for h in range(case["hkv"]):
            k, v = (x[c][page, h, j % case["bs"]].double() for c in "kv")
            r = slice(h * rep, (h + 1) * rep)
            zero = torch.zeros(rep, dtype=torch.long, device=DEV)
            out[b, r] = _exact_rows(x["q"][b, r].double(), k, v, zero, zero + n, case["cap"], None if x["gate"] is None else x["gate"][b, r].double())
    return out


@torch.no_grad()
def exact(case, seed):
    return {"append": _exact_append, "spans": _exact_spans, "shared": _exact_shared}[case["kind"]](case, seed)
