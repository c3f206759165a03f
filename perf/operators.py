"""Cases, inputs, plain forms and exact values of the attention-block operators:

* ``rope``    rotary positions of the query and key heads of a packed batch
* ``append``  new tokens' keys (rotated) and values into a paged cache, queries rotated on the way
* ``scored``  packed variable-length attention with capped scores, a bias by distance, windows, prefix and document masks
* ``paged``   attention of a chunk of new tokens (one or many) over the paged cache

``own = False`` computes the plain form with elementary torch operations in 32 bits, ``own = True`` calls the library's
operators through its C ABI. Head layouts are those of the repository's named configurations.
"""
import ctypes
import math
import random

import torch

own = False

HALF, INTERLEAVED = 0, 1
NONE, LINEAR, NTK, BANDS, YARN = 0, 1, 2, 3, 4
THETA = 1.0e6        # of the decoder configuration
ORIGINAL = 2048      # its trained length: what the scalings stretch
LOW, HIGH = 1.0, 4.0           # BANDS: wavelengths in units of the trained length
FAST, SLOW = 32.0, 1.0         # YARN: rotations over the trained length
# (query heads, key-value heads, head_dim) of the named configurations, and a small grouped layout of the tests
LAYOUTS = [(12, 12, 32), (16, 16, 64), (12, 12, 64), (28, 4, 128), (4, 2, 64), (16, 4, 96)]


def _rope_case(name, seqs, lo, hi, lens, layout, rot, pairs, scaling, factor, start, explicit, inverse=False):
    return {"name": name, "op": "rope", "seqs": seqs, "lo": lo, "hi": hi, "lens": lens, "heads": layout[0], "kv_heads": layout[1],
            "dim": layout[2], "rot": rot, "pairs": pairs, "scaling": scaling, "factor": factor, "start": start,
            "explicit": explicit, "inverse": inverse}


def _append_case(name, seqs, lo, hi, lens, old, page, by_head, layout, rot, pairs, scaling, factor):
    return {"name": name, "op": "append", "seqs": seqs, "lo": lo, "hi": hi, "lens": lens, "old": old, "page": page,
            "by_head": by_head, "heads": layout[0], "kv_heads": layout[1], "dim": layout[2], "rot": rot, "pairs": pairs,
            "scaling": scaling, "factor": factor}


def _scored_case(name, seqs, lo, hi, lens, layout, causal=False, left=-1, right=-1, cap=0.0, slopes=False, radius=0, prefix=False,
                 docs=0):
    return {"name": name, "op": "scored", "seqs": seqs, "lo": lo, "hi": hi, "lens": lens, "heads": layout[0],
            "kv_heads": layout[1], "dim": layout[2], "causal": causal, "left": left, "right": right, "cap": cap,
            "slopes": slopes, "radius": radius, "prefix": prefix, "docs": docs}


def _paged_case(name, seqs, lo, hi, kv_lo, kv_hi, lens, page, by_head, layout, left=-1, cap=0.0, slopes=False):
    return {"name": name, "op": "paged", "seqs": seqs, "lo": lo, "hi": hi, "kv_lo": kv_lo, "kv_hi": kv_hi, "lens": lens,
            "page": page, "by_head": by_head, "heads": layout[0], "kv_heads": layout[1], "dim": layout[2], "left": left,
            "cap": cap, "slopes": slopes}


def listed():
    return [
        # one short query through the decoder: latency
        _rope_case("rope_query", 1, 24, 24, 1, (28, 4, 128), 128, HALF, NONE, 1.0, 0, False),
        # an indexing batch at full context, long-context scaling, part of the head, interleaved pairs
        _rope_case("rope_batch", 16, 512, 2048, 2, (28, 4, 128), 64, INTERLEAVED, YARN, 16.0, 0, False),
        # explicit far positions, whole head, the rotation taken back (the gradient, or cached keys that move)
        _rope_case("rope_far_inverse", 7, 300, 1500, 3, (16, 16, 64), 64, HALF, BANDS, 8.0, 900_001, True, True),
        # one token for each of 48 sequences: a serving step
        _append_case("append_step", 48, 1, 1, 4, 4000, 16, False, (28, 4, 128), 128, HALF, NONE, 1.0),
        # chunks of long documents
        _append_case("append_chunk", 16, 100, 1024, 5, 3000, 64, True, (28, 4, 128), 128, HALF, LINEAR, 4.0),
        # one short query through an encoder with a linear distance bias: latency
        _scored_case("scored_query", 1, 24, 24, 6, (12, 12, 64), slopes=True),
        # an indexing batch through the same kind of encoder
        _scored_case("scored_batch", 192, 8, 512, 7, (16, 16, 64), slopes=True),
        # a decoder with capped scores and a local layer at its longest context
        _scored_case("scored_cap_window", 8, 600, 2048, 8, (28, 4, 128), causal=True, left=1023, cap=50.0),
        # documents packed into long rows, a bias table by clamped distance, padding tokens between them
        _scored_case("scored_docs", 4, 2500, 4096, 9, (12, 12, 32), radius=128, docs=12),
        # one token over a short cache: latency
        _paged_case("paged_query", 1, 1, 1, 700, 700, 10, 16, False, (28, 4, 128)),
        # one token for each of 64 sequences
        _paged_case("paged_step", 64, 1, 1, 64, 8192, 11, 16, False, (28, 4, 128)),
        # chunks of new tokens over long caches, capped, in pages stored head by head
        _paged_case("paged_chunk", 6, 200, 512, 2000, 6144, 12, 64, True, (28, 4, 128), cap=50.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "scored", "scored", "paged", "paged"])
    lens = rng.randrange(1 << 30)
    layout = rng.choice(LAYOUTS)
    heads, kv, dim = layout
    rot = dim if rng.random() < 0.5 else rng.choice([dim // 2, dim // 4])
    pairs, scaling = rng.choice([HALF, INTERLEAVED]), rng.choice([NONE, LINEAR, NTK, BANDS, YARN])
    factor = 1.0 if scaling == NONE else rng.choice([2.0, 4.0, 8.0, 16.0])
    if op == "rope":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(2048, 16384 // seqs))
        c = _rope_case("", seqs, max(1, hi // 8), hi, lens, layout, rot, pairs, scaling, factor, rng.choice([0, 5, 70_000]),
                       rng.random() < 0.4, rng.random() < 0.3)
    elif op == "append":
        seqs = _log_int(rng, 1, 64)
        hi = 1 if rng.random() < 0.4 else _log_int(rng, 1, min(1024, 8192 // seqs))
        c = _append_case("", seqs, max(1, hi // 8), hi, lens, _log_int(rng, 1, 4000), rng.choice([8, 16, 24, 32, 64, 128]),
                         rng.random() < 0.5, layout, rot, pairs, scaling, factor)
    elif op == "scored":
        hi = _log_int(rng, 8, 4096)
        most = max(1, int(700e6 / (heads * hi * hi)))
        seqs = _log_int(rng, 1, min(192, most))
        kind = rng.choice(["slopes", "table", "cap", "prefix", "docs", "window"])
        causal = kind == "prefix" or rng.random() < 0.4
        left = _log_int(rng, 16, 1024) if kind == "window" or rng.random() < 0.25 else -1
        right = left if left >= 0 and not causal else -1
        c = _scored_case("", seqs, max(1, hi // 16), hi, lens, layout, causal, left, right,
                         rng.choice([20.0, 30.0, 50.0]) if kind == "cap" or rng.random() < 0.2 else 0.0, kind == "slopes",
                         _log_int(rng, 8, 512) if kind == "table" else 0, kind == "prefix", rng.randrange(2, 20) if kind == "docs" else 0)
    else:
        hi = 1 if rng.random() < 0.4 else _log_int(rng, 1, 512)
        kv_hi = max(hi, _log_int(rng, 16, 8192))
        most = max(1, min(int(600e6 / (heads * hi * kv_hi)), int(200e6 / (kv * dim * kv_hi))))
        seqs = _log_int(rng, 1, min(64, most))
        c = _paged_case("", seqs, max(1, hi // 8), hi, max(1, kv_hi // 64), kv_hi, lens, rng.choice([8, 16, 24, 32, 64, 128]),
                        rng.random() < 0.5, layout, _log_int(rng, 16, 4096) if rng.random() < 0.3 else -1,
                        rng.choice([30.0, 50.0]) if rng.random() < 0.3 else 0.0, rng.random() < 0.3)
    del c["name"]
    return c


# -- lengths: of the case, not of the seed ---------------------------------------------------
def _lens(case):
    """New tokens of each sequence, and its keys in all where there is a cache; the first sequence has the longest of both."""
    rng = random.Random(case["lens"])
    new = [case["hi"]] + [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]
    if case["op"] == "append":
        return new, [n + rng.randrange(case["old"] + 1) for n in new]
    if case["op"] == "paged":
        return new, [max(n, k) for n, k in zip(new, [case["kv_hi"]] + [_log_int(rng, case["kv_lo"], case["kv_hi"]) for _ in new[1:]])]
    return new, None


def _doc_ids(case):
    """Runs of one id, a run of padding (-1) between some of them; one list for each sequence."""
    rng = random.Random(case["lens"] + 1)
    rows = []
    for n in _lens(case)[0]:
        row, d = [], 0
        while len(row) < n:
            row += [d] * _log_int(rng, max(1, n // (4 * case["docs"])), max(2, 2 * n // case["docs"]))
            row += [-1] * (rng.random() < 0.3) * rng.randrange(1, 9)
            d += 1
        rows.append(row[:n])
    return rows


def _prefixes(case):
    rng = random.Random(case["lens"] + 2)
    return [rng.randrange(n // 2 + 1) for n in _lens(case)[0]]


def _pairs(case):
    """(query, key) pairs that are visible, over all sequences."""
    new, kv = _lens(case)
    total = 0
    docs = _doc_ids(case) if case.get("docs") else None
    prefix = _prefixes(case) if case.get("prefix") else None
    for s, n in enumerate(new):
        k = kv[s] if kv else n
        i = torch.arange(n, dtype=torch.int64) + (k - n)
        last = i if case.get("causal", True) else (i + case["right"] if case["right"] >= 0 else torch.full_like(i, k - 1))
        first = i - case["left"] if case["left"] >= 0 else torch.zeros_like(i)
        last, first = last.clamp(max=k - 1), first.clamp(min=0)
        if docs:
            d = torch.tensor(docs[s])
            # tokens of the same document form one run
            start = torch.cat([torch.tensor([True]), d[1:] != d[:-1]]).cumsum(0) - 1
            size = torch.bincount(start)
            end = size.cumsum(0)
            first, last = torch.maximum(first, (end - size)[start]), torch.minimum(last, end[start] - 1)
            total += int(((last - first + 1).clamp(min=0) * (d >= 0)).sum())
        else:
            seen = (last - first + 1).clamp(min=0)
            if prefix:
                seen = seen + torch.minimum(first, torch.tensor(prefix[s])) + (prefix[s] - 1 - last).clamp(min=0)
            total += int(seen.sum())
    return total


def work(case):
    new, kv = _lens(case)
    tokens, heads, kvh, dim = sum(new), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        n = tokens * (heads + kvh)
        return {"bytes": 4 * n * dim, "flops": 3 * n * case["rot"]}
    if case["op"] == "append":
        n = tokens * (heads + 2 * kvh)
        return {"bytes": 4 * n * dim, "flops": 3 * tokens * (heads + kvh) * case["rot"]}
    flops = 4 * dim * heads * _pairs(case)
    if case["op"] == "scored":
        return {"bytes": 2 * tokens * dim * (2 * heads + 2 * kvh), "flops": flops}
    left = case["left"]
    seen = sum(k if left < 0 else min(k, left + n) for n, k in zip(new, kv))
    return {"bytes": 2 * dim * (2 * tokens * heads + 2 * seen * kvh), "flops": flops}


# -- inputs ---------------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    new, kv = _lens(case)
    heads, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = {"case": case, "tokens": tokens, "longest": max(new), "cu": _ints(cu)}
    # projections of normalised states: queries wider than keys, as trained heads have them
    x = torch.randn(tokens, heads + 2 * kvh, dim, generator=g, device="cuda")
    x[:, :heads] *= 2.0
    if case.get("cap"):
        x[:, :heads] *= 4.0  # scores that reach into the cap
    s["qkv"] = x.view(tokens, -1).to(torch.bfloat16)
    if case["op"] == "rope":
        jump = torch.randint(0, 4, (tokens,), generator=g, device="cuda") if case["explicit"] else None
        start = torch.randint(case["start"], case["start"] + 2048, (len(new),), generator=g, device="cuda") if case["start"] else None
        s["start"] = None if start is None else start.to(torch.int32)
        s["positions"] = None
        if case["explicit"]:  # positions with gaps, as a packed prompt with removed spans has them
            s["positions"] = (jump.cumsum(0) + case["start"]).to(torch.int32)
            s["start"] = None
    if kv:
        s["kv_lens"], s["most_keys"] = _ints(kv), max(kv)
        page = case["page"]
        used = [-(-k // page) for k in kv]
        n_pages = sum(used) + 3
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(new), max(used)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(used):
            table[i, :n] = order[at:at + n]
            at += n
        s["table"] = table
        shape = (n_pages, kvh, page, dim) if case["by_head"] else (n_pages, page, kvh, dim)
        s["k"] = torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)
        s["v"] = torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)
        if case["op"] == "paged":
            s["q"] = s.pop("qkv")[:, :heads * dim].contiguous()
    if case.get("slopes"):
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")
    if case.get("radius"):
        s["bias"] = torch.randn(heads, 2 * case["radius"] + 1, generator=g, device="cuda") * 2.0
    if case.get("docs"):
        s["docs"] = _ints([d for row in _doc_ids(case) for d in row])
    if case.get("prefix"):
        s["prefix"] = _ints(_prefixes(case))
    return s


# -- plain forms ------------------------------------------------------------------------------
def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and the factor on cos and sin."""
    r = case["rot"]
    i = torch.arange(0, r, 2, dtype=torch.float64, device="cuda")
    f, mode = case["factor"], case["scaling"]
    theta = THETA * f ** (r / (r - 2.0)) if mode == NTK else THETA
    w = theta ** (-i / r)
    if mode == LINEAR:
        return w / f, 1.0
    if mode == BANDS:
        turns = ORIGINAL * w / (2 * math.pi)  # rotations over the trained length
        keep = ((turns - LOW) / (HIGH - LOW)).clamp(0, 1)
        return w * keep + w / f * (1 - keep), 1.0
    if mode == YARN:
        at = lambda turns: r * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        lo, hi = max(0.0, math.floor(at(FAST))), min(r - 1.0, math.ceil(at(SLOW)))
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return w * (1 - ramp) + w / f * ramp, 0.1 * math.log(f) + 1.0
    return w, 1.0


def _rotate(x, positions, case, inverse=False):
    """x [tokens, heads, dim] in 32 bits."""
    w, m = _frequencies(case)
    a = positions.double()[:, None] * w
    cos, sin = (a.cos() * m).float()[:, None], (a.sin() * m).float()[:, None]
    sin = -sin if inverse else sin
    r = case["rot"]
    head, rest = x[..., :r], x[..., r:]
    if case["pairs"] == HALF:
        u, v = head[..., :r // 2], head[..., r // 2:]
        y = torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
    else:
        u, v = head[..., 0::2], head[..., 1::2]
        y = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _sequence_of(s):
    """Sequence of each token, and its place in it."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    return seq, t - s["cu"].long()[seq]


def _slots(s, seq, pos):
    """Index of each (sequence, position) in a cache laid out as [pages, page, ...]: page and place in it."""
    page = s["case"]["page"]
    return s["table"].long()[seq, pos // page].clamp(min=0), pos % page


def _by_token(s, name):
    return s[name].transpose(1, 2) if s["case"]["by_head"] else s[name]


def _attend(q, k, v, qpos, kpos, seen, s, heads, kvh):
    """q [b, n, heads, d], k and v [b, m, kvh, d] in 32 bits; seen [b, n, m]: what there is to see. [b, n, heads, d]."""
    case = s["case"]
    b, n, _, d = q.shape
    m, grp = k.shape[1], heads // kvh
    qg = q.view(b, n, kvh, grp, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, grp * n, d)
    x = torch.matmul(qg, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d)).view(b, heads, n, m)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    dist = kpos[:, None, :] - qpos[:, :, None]  # [b, n, m]
    if case["slopes"]:
        x.sub_(s["slopes"][:, None, None] * dist.abs().float()[:, None])
    if case.get("radius"):
        r = case["radius"]
        x.add_(s["bias"][:, dist.clamp(-r, r) + r].transpose(0, 1))
    right = 0 if case.get("causal", True) else case["right"]
    near = torch.ones_like(dist, dtype=torch.bool)
    if right >= 0:
        near &= dist <= right
    if case["left"] >= 0:
        near &= dist >= -case["left"]
    if case.get("prefix"):
        near |= kpos[:, None, :] < s["prefix"].long()[:, None, None]
    x.masked_fill_(~(near & seen)[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, kvh, grp * n, m), v.transpose(1, 2)).view(b, heads, n, d)
    return torch.where(total > 0, o / total, torch.zeros_like(o)).transpose(1, 2)


def _plain(s):
    case = s["case"]
    heads, kvh, dim, t = case["heads"], case["kv_heads"], case["dim"], s["tokens"]
    seq, place = _sequence_of(s)
    if case["op"] == "rope":
        x = s["qkv"].view(t, heads + 2 * kvh, dim)[:, :heads + kvh].float()
        pos = s["positions"] if s["positions"] is not None else place + (s["start"].long()[seq] if s["start"] is not None else 0)
        return _rotate(x, pos, case, case["inverse"]).to(torch.bfloat16).view(t, -1)
    if case["op"] == "append":
        x = s["qkv"].view(t, heads + 2 * kvh, dim).float()
        new = s["cu"].long().diff()
        pos = place + (s["kv_lens"].long() - new)[seq]
        turned = _rotate(x[:, :heads + kvh], pos, case).to(torch.bfloat16)
        at, off = _slots(s, seq, pos)
        _by_token(s, "k")[at, off] = turned[:, heads:]
        _by_token(s, "v")[at, off] = s["qkv"].view(t, heads + 2 * kvh, dim)[:, heads + kvh:]
        return [turned[:, :heads].reshape(t, -1), s["k"], s["v"]]
    n = s["longest"]
    cu = s["cu"].long()
    new = cu.diff()
    rows = (cu[:-1, None] + torch.arange(n, device="cuda")).clamp(max=t - 1)  # [seqs, n]
    there = torch.arange(n, device="cuda") < new[:, None]
    if case["op"] == "scored":
        x = s["qkv"].float().view(t, heads + 2 * kvh, dim)[rows]
        pos = torch.arange(n, device="cuda").expand(len(new), n)
        seen = there[:, None, :].expand(-1, n, -1)
        if case["docs"]:
            d = s["docs"][rows]
            seen = seen & (d[:, :, None] == d[:, None, :]) & (d[:, :, None] >= 0)
        o = _attend(x[:, :, :heads], x[:, :, heads:heads + kvh], x[:, :, heads + kvh:], pos, pos, seen, s, heads, kvh)
    else:
        m = s["most_keys"]
        kpos = torch.arange(m, device="cuda").expand(len(new), m)
        at, off = _slots(s, torch.arange(len(new), device="cuda")[:, None], kpos)
        inside = kpos < s["kv_lens"].long()[:, None]
        k, v = (torch.where(inside[:, :, None, None], _by_token(s, name)[at, off].float(), 0.0) for name in ("k", "v"))
        qpos = (s["kv_lens"].long() - new)[:, None] + torch.arange(n, device="cuda")
        o = _attend(s["q"].float().view(t, heads, dim)[rows], k, v, qpos, kpos, inside[:, None, :], s, heads, kvh)
    return o[there].to(torch.bfloat16).reshape(t, heads * dim)


# -- the library's operators --------------------------------------------------------------------
def _rope_desc(_lib, case, inverse=False):
    low, high = (FAST, SLOW) if case["scaling"] == YARN else (LOW, HIGH)
    return _lib.RopeDesc(rot_dim=case["rot"], layout=case["pairs"], scaling=case["scaling"], original_max_pos=ORIGINAL, theta=THETA,
                         factor=case["factor"], low=low, high=high, magnitude=0.0, inverse=int(inverse))


def _cache(_lib, s):
    case, k = s["case"], s["k"]
    by_head = case["by_head"]
    return _lib.KvCache(k=k.data_ptr(), v=s["v"].data_ptr(), page_table=s["table"].data_ptr(), n_pages=k.shape[0],
                        page_size=case["page"], n_kv_heads=case["kv_heads"], head_dim=case["dim"],
                        table_stride=s["table"].shape[1], page_stride=k.stride(0), token_stride=k.stride(2 if by_head else 1),
                        head_stride=k.stride(1 if by_head else 2))


def _options(_lib, s):
    case = s["case"]
    ptr = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    return _lib.AttnOpts(scale=0.0, cap=case["cap"], causal=int(case.get("causal", True)), window_left=case["left"],
                         window_right=case.get("right", -1), bias_radius=case.get("radius", 0), slopes=ptr("slopes"),
                         bias=ptr("bias"), prefix_lens=ptr("prefix"), doc_ids=ptr("docs"))


def _workspace(lib, s):
    """The attention operators' scratch memory."""
    case = s["case"]
    n = lib.b200emb_attention_workspace_bytes(case["seqs"], s["tokens"], case["heads"], case["kv_heads"], case["dim"])
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _kept(s, name, make):
    """Descriptors and scratch memory, which a program makes once and keeps with its buffers."""
    if name not in s:
        s[name] = make()
    return s[name]


def _own(s):
    from infinity_b200 import _lib

    lib, case = _lib.load(), s["case"]
    heads, kvh, dim, t, seqs = case["heads"], case["kv_heads"], case["dim"], s["tokens"], case["seqs"]
    stream = torch.cuda.current_stream().cuda_stream
    ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    cu = s["cu"].data_ptr()
    ref = ctypes.byref
    width = (heads + 2 * kvh) * dim
    if case["op"] == "rope":
        out = torch.empty(t, (heads + kvh) * dim, dtype=torch.bfloat16, device="cuda")
        _lib.check(lib.b200emb_op_rope(s["qkv"].data_ptr(), width, out.data_ptr(), (heads + kvh) * dim, ptr(s["positions"]), cu,
                                       ptr(s["start"]), seqs, t, heads + kvh, dim,
                                       ref(_kept(s, "rope", lambda: _rope_desc(_lib, case, case["inverse"]))), stream))
        return out
    out = torch.empty(t, heads * dim, dtype=torch.bfloat16, device="cuda")
    if case["op"] == "append":
        _lib.check(lib.b200emb_op_kv_append(s["qkv"].data_ptr(), width, cu, s["kv_lens"].data_ptr(), seqs, t, heads,
                                            ref(_kept(s, "rope", lambda: _rope_desc(_lib, case))), out.data_ptr(), heads * dim,
                                            ref(_kept(s, "cache", lambda: _cache(_lib, s))), stream))
        return [out, s["k"], s["v"]]
    ws = _kept(s, "workspace", lambda: _workspace(lib, s))
    options = _kept(s, "options", lambda: _options(_lib, s))
    if case["op"] == "scored":
        q = s["qkv"].data_ptr()
        k, v = q + 2 * heads * dim, q + 2 * (heads + kvh) * dim
        _lib.check(lib.b200emb_op_attention_scored(q, width, k, width, v, width, out.data_ptr(), heads * dim, cu, seqs, t, heads, kvh,
                                                   dim, ref(options), ws.data_ptr(), ws.numel(), stream))
    else:
        _lib.check(lib.b200emb_op_attention_paged(s["q"].data_ptr(), heads * dim, out.data_ptr(), heads * dim, cu,
                                                  s["kv_lens"].data_ptr(), seqs, t, heads,
                                                  ref(_kept(s, "cache", lambda: _cache(_lib, s))), ref(options),
                                                  ws.data_ptr(), ws.numel(), stream))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# -- exact values: from the definitions, sequence by sequence, in 64 bits -------------------------
def _exact_rotated(x, pos, case, sign):
    """x [heads, dim] rows of one token set [n, heads, dim], positions [n] -> rotated, float64."""
    r, f, mode = case["rot"], case["factor"], case["scaling"]
    y = x.clone()
    for p in range(r // 2):
        w = THETA ** (-2.0 * p / r)
        m = 1.0
        if mode == LINEAR:
            w = w / f
        elif mode == NTK:
            w = (THETA * f ** (r / (r - 2.0))) ** (-2.0 * p / r)
        elif mode == BANDS:
            length = 2 * math.pi / w
            if length > ORIGINAL / LOW:
                w = w / f
            elif length > ORIGINAL / HIGH:
                mix = (ORIGINAL / length - LOW) / (HIGH - LOW)
                w = (1 - mix) * w / f + mix * w
        elif mode == YARN:
            edge = [r * math.log(ORIGINAL / (n * 2 * math.pi)) / (2 * math.log(THETA)) for n in (FAST, SLOW)]
            lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
            up = min(1.0, max(0.0, (p - lo) / max(hi - lo, 1e-3)))
            w, m = w / f * up + w * (1 - up), 0.1 * math.log(f) + 1.0
        a = pos.double() * w
        c, d = (a.cos() * m)[:, None], (a.sin() * m * sign)[:, None]
        i, j = (p, p + r // 2) if case["pairs"] == HALF else (2 * p, 2 * p + 1)
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * d, x[..., j] * c + x[..., i] * d
    return y


def exact(case, seed):
    s = prepare(case, seed)
    heads, kvh, dim, t = case["heads"], case["kv_heads"], case["dim"], s["tokens"]
    new, kv = _lens(case)
    cu = s["cu"].tolist()
    if case["op"] in ("rope", "append"):
        x = s["qkv"].double().view(t, -1, dim)
        if case["op"] == "rope" and s["positions"] is not None:
            pos = s["positions"]
        else:
            first = [k - n for n, k in zip(new, kv)] if kv else s["start"].tolist() if s["start"] is not None else [0] * len(new)
            pos = torch.cat([torch.arange(n, device="cuda") + f for n, f in zip(new, first)])
        sign = -1.0 if case.get("inverse") else 1.0
        y = _exact_rotated(x[:, :heads + kvh], pos, case, sign)
        if case["op"] == "rope":
            return y.reshape(t, -1)
        k, v, page = s["k"].double(), s["v"].double(), case["page"]
        for i in range(len(new)):
            p = pos[cu[i]:cu[i + 1]]
            at, off = s["table"][i].long()[p // page], p % page
            if case["by_head"]:
                k[at, :, off], v[at, :, off] = y[cu[i]:cu[i + 1], heads:], x[cu[i]:cu[i + 1], heads + kvh:]
            else:
                k[at, off], v[at, off] = y[cu[i]:cu[i + 1], heads:], x[cu[i]:cu[i + 1], heads + kvh:]
        return [y[:, :heads].reshape(t, -1), k, v]
    out = torch.zeros(t, heads, dim, dtype=torch.float64, device="cuda")
    docs = _doc_ids(case) if case.get("docs") else None
    prefix = _prefixes(case) if case.get("prefix") else None
    for i, n in enumerate(new):
        rows = slice(cu[i], cu[i + 1])
        if case["op"] == "scored":
            x = s["qkv"][rows].double().view(n, -1, dim)
            q, k, v, m = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:], n
        else:
            m, page = kv[i], case["page"]
            pages = s["table"][i, :-(-m // page)].long()
            both = []
            for name in ("k", "v"):
                c = s[name][pages].double()
                both.append((c.transpose(1, 2) if case["by_head"] else c).reshape(-1, kvh, dim)[:m])
            q, (k, v) = s["q"][rows].double().view(n, heads, dim), both
        qi = torch.arange(m - n, m, device="cuda")[:, None]
        kj = torch.arange(m, device="cuda")[None, :]
        ok = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if case.get("causal", True):
            ok &= kj <= qi
        elif case["right"] >= 0:
            ok &= kj - qi <= case["right"]
        if case["left"] >= 0:
            ok &= qi - kj <= case["left"]
        if prefix:
            ok |= kj < prefix[i]
        if docs:
            d = _ints(docs[i])
            ok &= (d[:, None] == d[None, :]) & (d >= 0)[:, None]
        for h in range(heads):
            x = q[:, h] @ k[:, h * kvh // heads].T / math.sqrt(dim)
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            if case["slopes"]:
                x = x - 2.0 ** (-8.0 * (h + 1) / heads) * (kj - qi).abs().double()
            if case.get("radius"):
                r = case["radius"]
                x = x + s["bias"][h].double()[(kj - qi).clamp(-r, r) + r]
            some = ok.any(1)
            x = torch.where(ok, x, -math.inf)
            x = torch.where(some[:, None], x, 0.0)
            out[rows, h] = torch.where(some[:, None], torch.softmax(x, 1) @ v[:, h * kvh // heads], 0.0)
    return out.reshape(t, heads * dim)
