"""Operators over paged key/value caches: rotation by positions that are given per token, rows of new tokens into pages, attention of a
chunk of new tokens of every sequence over its pages, and eviction of the rows that received the least attention.

A case is a dict of plain values.  Every sequence s of a case has `cached` rows already and brings `new` tokens, both spread over the
case's ranges by the sequence's number; its rows lie in pages that are scattered over the pool.  `run` computes the operators in their plain
form - sums, products and exponentials of 32 bits by torch, padded to the longest sequence - or, where `own` is true, through the
framework's calls."""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decode step of 32 sequences: the queries of a layer, turned by the position that each sequence has reached
        {"name": "rotary_32", "kind": "rotary", "dt": "bf16", "tokens": 32, "heads": 32, "dim": 128, "axes": 1, "halves": False},
        # a clip of video: time, height and width of every patch, pairs in halves, keys and values beside the queries in a row
        {"name": "rotary_video_8192", "kind": "rotary", "dt": "f16", "tokens": 8192, "heads": 16, "dim": 128, "axes": 3, "halves": True},
        # one token of each of 96 sequences into the pages of a layer that is kept in 32 bits
        {"name": "append_96", "kind": "append", "dt": "f32", "kv_heads": 8, "dim": 64, "vdim": 64, "page": 16, "sequences": 96, "chunks": 0,
         "new": "1-1", "cached": "5-900", "mass": False},
        # prompts of seven sequences behind what they have, whose attention weight is going to be summed
        {"name": "append_prompts", "kind": "append", "dt": "bf16", "kv_heads": 8, "dim": 128, "vdim": 128, "page": 64, "sequences": 7, "chunks": 7,
         "new": "600-1700", "cached": "0-3000", "mass": True},
        # one token of one sequence, heads as Phi-3 has them: all latency
        {"name": "decode_one_1000", "kind": "attend", "dt": "f16", "heads": 32, "kv_heads": 32, "dim": 96, "vdim": 96, "page": 16, "sequences": 1, "chunks": 0,
         "new": "1-1", "cached": "1000-1000", "window": 0, "first": 0, "sink": False, "mass": False},
        # a batch in generation, from short sequences to long ones
        {"name": "decode_64", "kind": "attend", "dt": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128, "page": 64, "sequences": 64, "chunks": 0,
         "new": "1-1", "cached": "100-8000", "window": 0, "first": 0, "sink": False, "mass": False},
        # generation over a book, with the weights summed for an eviction to come
        {"name": "decode_131000_mass", "kind": "attend", "dt": "f16", "heads": 64, "kv_heads": 8, "dim": 128, "vdim": 128, "page": 256, "sequences": 1, "chunks": 0,
         "new": "1-1", "cached": "131000-131000", "window": 0, "first": 0, "sink": False, "mass": True},
        # a prompt into an empty cache
        {"name": "prompt_4096", "kind": "attend", "dt": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128, "page": 128, "sequences": 1, "chunks": 1,
         "new": "4096-4096", "cached": "0-0", "window": 0, "first": 0, "sink": False, "mass": False},
        # two prompts among sequences in generation, 32-bit weights and cache, heads as Whisper has them, a window with its first tokens and sinks
        {"name": "mixed_window_f32", "kind": "attend", "dt": "f32", "heads": 6, "kv_heads": 6, "dim": 64, "vdim": 64, "page": 32, "sequences": 9, "chunks": 2,
         "new": "101-300", "cached": "0-1500", "window": 500, "first": 4, "sink": True, "mass": False},
        # a piece of a long prompt, heads of Phi-2's width, with the weights summed
        {"name": "chunk_777_mass", "kind": "attend", "dt": "f16", "heads": 32, "kv_heads": 8, "dim": 80, "vdim": 80, "page": 32, "sequences": 1, "chunks": 1,
         "new": "777-777", "cached": "20000-20000", "window": 0, "first": 0, "sink": False, "mass": True},
        # one sequence at the end of its budget, a kv head per head
        {"name": "evict_2048", "kind": "evict", "dt": "f16", "kv_heads": 32, "dim": 96, "vdim": 96, "page": 16, "sequences": 1, "cached": "2048-2048", "keep": 1000,
         "first": 4, "recent": 256},
        # a batch of long sequences cut to a quarter
        {"name": "evict_16", "kind": "evict", "dt": "bf16", "kv_heads": 8, "dim": 128, "vdim": 128, "page": 64, "sequences": 16, "cached": "9000-16000", "keep": 4096,
         "first": 4, "recent": 512},
    ]


def _spread(rng, lo, hi):
    """A whole number between the two, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(lo, hi):
    """A range as a plain value."""
    return "%d-%d" % (lo, hi)


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "attend", "evict"])
    dt = rng.choice(["f16", "bf16", "bf16", "f16", "f32"])
    if kind == "rotary":
        return {"kind": kind, "dt": dt, "tokens": _spread(rng, 1, 8192), "heads": rng.choice([6, 8, 16, 32]), "dim": rng.choice([64, 80, 96, 128]),
                "axes": rng.choice([1, 2, 3, 4]), "halves": rng.random() < 0.5}
    dim = rng.choice([64, 80, 96, 128])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "evict":
        long = _spread(rng, 64, 16000)
        keep = _spread(rng, 16, max(16, long // 2))
        return {"kind": kind, "dt": dt, "kv_heads": rng.choice([1, 2, 6, 8]), "dim": dim, "vdim": rng.choice([dim, 64]), "page": page,
                "sequences": _spread(rng, 1, 16), "cached": _text(rng.randint(1, long), long), "keep": keep, "first": rng.randint(0, 8),
                "recent": rng.randint(0, keep - 8)}
    kv = rng.choice([1, 2, 6, 8])
    if kind == "append":
        chunks = rng.choice([0, 1, 4])
        new = _spread(rng, 2, 1700)
        return {"kind": kind, "dt": dt, "kv_heads": kv, "dim": dim, "vdim": rng.choice([dim, 64]), "page": page, "sequences": chunks + _spread(rng, 1, 96),
                "chunks": chunks, "new": _text(max(1, new // 2), new), "cached": _text(0, _spread(rng, 1, 3000)), "mass": rng.random() < 0.5}
    form = rng.choice(["decode", "decode", "chunk", "chunk", "mixed"])
    group = rng.choice([1, 2, 4, 7, 8]) if kv < 6 else rng.choice([1, 2, 4])
    if form == "decode":
        sequences = _spread(rng, 1, 64)
        new, chunks, cached = 1, 0, _spread(rng, 1, min(131000, 400000 // (sequences * kv)))
    elif form == "chunk":
        sequences = chunks = 1
        new = _spread(rng, 2, 4096)
        cached = _spread(rng, 1, max(1, min(20000, 8 * 10 ** 6 // (new * max(1, kv * group // 8)) - new)))
    else:
        chunks = rng.choice([1, 2])
        sequences, new, cached = chunks + _spread(rng, 1, 20), _spread(rng, 2, 300), _spread(rng, 1, 1500)
    wide = rng.random() < 0.3
    if form == "chunk" and dt == "f32" and new * (cached + new) > 4 * 10 ** 6:
        dt = rng.choice(["f16", "bf16"])             # long prompts run in 16 bits
    return {"kind": kind, "dt": dt, "heads": kv * group, "kv_heads": kv, "dim": dim, "vdim": dim, "page": page, "sequences": sequences, "chunks": chunks,
            "new": _text(max(1, new // 2), new), "cached": _text(rng.randint(0, cached), cached), "window": _spread(rng, 1, 4000) if wide else 0,
            "first": rng.choice([0, 1, 4]) if wide else 0, "sink": rng.random() < 0.3, "mass": rng.random() < 0.3}


# ---------------------------------------------------------------------------------------- sizes
def _range(text):
    lo, hi = text.split("-")
    return int(lo), int(hi)


def _place(i, lo, hi):
    """A number between the two that goes by the sequence's; the first one has the largest."""
    return hi - (i * 2654435761 % (1 << 32)) * (hi - lo + 1) // (1 << 32)


def _lengths(case):
    """Tokens that each sequence brings, and rows that it has with them."""
    n = case["sequences"]
    cached = [_place(i, *_range(case["cached"])) for i in range(n)]
    if case["kind"] == "evict":
        return [0] * n, cached
    new = [_place(i, *_range(case["new"])) if i < case["chunks"] else 1 for i in range(n)]
    return new, [a + b for a, b in zip(cached, new)]


def _sections(case):
    """Pairs that go by each axis: the first axis has the fewest."""
    pairs, n = case["dim"] // 2, case["axes"]
    per = 3 * pairs // (3 * n - 1) if n > 1 else 0
    return [pairs - per * (n - 1)] + [per] * (n - 1)


def work(case):
    e = 4 if case["dt"] == "f32" else 2
    if case["kind"] == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * e + 4 * case["tokens"] * case["axes"], "flops": 3 * n}
    new, rows = _lengths(case)
    G, width = case["kv_heads"], case["dim"] + case["vdim"]
    if case["kind"] == "append":
        return {"bytes": sum(new) * G * (2 * width * e + (4 if case["mass"] else 0)), "flops": 0}
    if case["kind"] == "evict":
        kept = [min(L, case["keep"]) for L in rows]
        return {"bytes": sum(G * (4 * L + k * (2 * width * e + 4)) for L, k in zip(rows, kept)), "flops": 0}
    H, window, first = case["heads"], case["window"], case["first"]
    pairs = seen = 0
    for n, L in zip(new, rows):
        at = np.arange(L - n, L, dtype=np.int64)
        low = np.maximum(at - window + 1, 0) if window else np.zeros_like(at)
        pairs += int((at - low + 1 + np.minimum(low, first)).sum())
        seen += L - int(low[0]) + min(int(low[0]), first)
    extra = 8 * G * seen if case["mass"] else 0
    return {"bytes": sum(new) * H * width * e + G * seen * width * e + extra, "flops": 2 * H * width * pairs}


# ---------------------------------------------------------------------------------------- inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rotary_inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    T, H, D, axes, pairs = case["tokens"], case["heads"], case["dim"], case["axes"], case["dim"] // 2
    # queries of a row that holds a quarter as many keys and values behind them
    x = torch.randn(T, (H + 2 * max(1, H // 4)) * D, generator=g, device="cuda").to(_TYPES[case["dt"]])
    if axes == 1:
        positions = torch.randint(0, 131072, (1, T), generator=g, device="cuda", dtype=torch.int32)
    else:                                        # a grid of patches, behind a text of its own length
        side, start = 16, int(torch.randint(0, 5000, (1,), generator=g, device="cuda"))
        at = torch.arange(T, device="cuda")
        grid = [at // (side * side), at // side % side, at % side, at // 7][:axes]
        positions = (start + torch.stack(grid)).to(torch.int32)
    freqs = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
    value = freqs.float()
    return x, positions, torch.stack([value, (freqs - value.double()).float()])


def _pool(g, shape, dt):
    """Random pages, a part at a time: what torch draws is of 32 bits."""
    out = torch.empty(shape, dtype=dt, device="cuda")
    for part in out.chunk(8):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda", dtype=dt))
    return out


def _pages(case, rows, order):
    """[sequences, pages of the longest] of page ids; behind a sequence's last page its row names pages of others."""
    R = case["page"]
    need = [-(-L // R) for L in rows]
    total, most = sum(need), max(1, max(need))
    ids = list(range(total + 3))
    order.shuffle(ids)
    table, at = [], 0
    for n in need:
        own_pages = ids[at:at + n]
        at += n
        table.append(own_pages + [ids[(at + j) % len(ids)] for j in range(most - n)])
    return _ints(table), total + 3


def _cache_inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    new, rows = _lengths(case)
    G, R, dt = case["kv_heads"], case["page"], _TYPES[case["dt"]]
    table, pages = _pages(case, rows, random.Random(seed))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return g, {"keys": _pool(g, (pages, G, R, case["dim"]), dt), "values": _pool(g, (pages, G, R, case["vdim"]), dt), "table": table, "starts": _ints(starts),
               "lengths": _ints(rows), "most": max(rows), "most_new": max(new)}


def _mass(g, case, table):
    """Sums of attention weights so far: a few rows have most of it, some have none."""
    shape = (case["sequences"], case["kv_heads"], table.shape[1] * case["page"])
    u = torch.rand(shape, generator=g, device="cuda")
    return torch.where(u < 0.02, torch.zeros_like(u), u ** 8)


def _inputs(case, seed):
    if case["kind"] == "rotary":
        x, positions, freqs = _rotary_inputs(case, seed)
        return {"x": x, "positions": positions, "freqs": freqs, "out": torch.empty(case["tokens"], case["heads"], case["dim"], dtype=x.dtype, device="cuda")}
    g, s = _cache_inputs(case, seed)
    dt, T = _TYPES[case["dt"]], int(s["starts"][-1])
    if case["kind"] == "append":
        # keys as the rotation leaves them, values where the projection has them: behind queries and keys
        s["k"] = torch.randn(T, case["kv_heads"] * case["dim"], generator=g, device="cuda").to(dt)
        s["v"] = torch.randn(T, 64 + case["kv_heads"] * case["vdim"], generator=g, device="cuda").to(dt)
        s["mass"] = _mass(g, case, s["table"]) if case["mass"] else None
    elif case["kind"] == "attend":
        s["q"] = (1.5 * torch.randn(T, case["heads"], case["dim"], generator=g, device="cuda")).to(dt)
        s["sink"] = torch.randn(case["heads"], generator=g, device="cuda") if case["sink"] else None
        s["mass"] = _mass(g, case, s["table"]) if case["mass"] else None
        s["out"] = torch.empty(T, case["heads"] * case["vdim"], dtype=dt, device="cuda")
    else:
        s["mass"] = _mass(g, case, s["table"])
        kept = [min(L, case["keep"]) for L in s["lengths"].tolist()]
        table, pages = _pages(case, kept, random.Random(seed + 1))
        s["kept"] = tuple(torch.from_numpy(np.concatenate(p)).cuda() for p in ([np.full(n, i) for i, n in enumerate(kept)], [np.arange(n) for n in kept]))
        s["into"] = {"keys": torch.zeros((pages,) + s["keys"].shape[1:], dtype=dt, device="cuda"),
                     "values": torch.zeros((pages,) + s["values"].shape[1:], dtype=dt, device="cuda"), "table": table,
                     "lengths": torch.zeros_like(s["lengths"]), "mass": torch.zeros(case["sequences"], case["kv_heads"], table.shape[1] * case["page"], device="cuda")}
    return s


_device = None


def _dev():
    global _device
    if _device is None:
        from ratchet_b200 import Device
        _device = Device(0)
    return _device


def _buffer(t):
    from ratchet_b200 import capi
    dt = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16, torch.int32: capi.I32}[t.dtype]
    return None if t is None else _dev().wrap(dt, t.shape, t.data_ptr())


def _handles(case, s):
    """What a program over the framework keeps: its buffers, and the cache that names them."""
    from ratchet_b200 import PagedCache
    wrap = lambda names: {n: _buffer(s[n]) for n in names if s.get(n) is not None}  # noqa: E731
    h = wrap(["x", "positions", "freqs", "out", "k", "v", "q", "sink"])
    if case["kind"] != "rotary":
        h["cache"] = PagedCache(**wrap(["keys", "values", "table", "starts", "lengths", "mass"]))
    if case["kind"] == "evict":
        h["into"] = PagedCache(**{n: _buffer(t) for n, t in s["into"].items()})
    return h


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if own:
        s["own"] = _handles(case, s)
    return s


# ---------------------------------------------------------------------------------------- one pass
def run(s):
    return {"rotary": _rotary, "append": _append, "attend": _attend, "evict": _evict}[s["case"]["kind"]](s)


def _rotary(s):
    c = s["case"]
    if own:
        h = s["own"]
        _dev().rotary_axes(h["x"], c["heads"], c["dim"], h["freqs"], h["positions"], _sections(c), halves=c["halves"], out=h["out"])
        return {"out": s["out"]}
    T, H, D = c["tokens"], c["heads"], c["dim"]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), torch.tensor(_sections(c), device="cuda"), output_size=D // 2)
    freqs = s["freqs"].double()
    angle = s["positions"][axis].T.double() * (freqs[0] + freqs[1])              # [tokens, pairs]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s["x"][:, :H * D].float().view(T, H, D)
    u, v = (x[..., :D // 2], x[..., D // 2:]) if c["halves"] else (x[..., ::2], x[..., 1::2])
    y = u * cos - v * sin, v * cos + u * sin
    s["out"].copy_(torch.cat(y, -1) if c["halves"] else torch.stack(y, -1).flatten(-2))
    return {"out": s["out"]}


def _where(s):
    """Sequence and row of every new token."""
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    T = s["k"].shape[0] if "k" in s else s["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new, output_size=T)
    return seq, torch.arange(T, device="cuda") - s["starts"][:-1].long()[seq] + (s["lengths"].long() - new)[seq]


def _append(s):
    c = s["case"]
    if own:
        h = s["own"]
        _dev().paged_append(h["k"], h["v"], h["cache"], v_col=64)
    else:
        G, R = c["kv_heads"], c["page"]
        seq, row = _where(s)
        page, at = s["table"].long()[seq, row // R], row % R
        s["keys"][page, :, at] = s["k"].view(-1, G, c["dim"])
        s["values"][page, :, at] = s["v"][:, 64:].view(-1, G, c["vdim"])
        if c["mass"]:
            s["mass"][seq, :, row] = 0.0
    return {"keys": s["keys"], "values": s["values"], **({"mass": s["mass"]} if c["mass"] else {})}


def _rows(pages, table, most):
    """[sequences, kv heads, rows, features] of the paged rows, in 32 bits."""
    x = pages[table.long()]                                              # [sequences, pages, kv heads, rows of a page, features]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :most].float()


def _attend(s):
    c = s["case"]
    scale = c["dim"] ** -0.5
    if own:
        h = s["own"]
        _dev().paged_attention(h["q"], h["cache"], scale, sink=h.get("sink"), window=c["window"], first=c["first"], out=h["out"])
        return {"out": s["out"], **({"mass": s["mass"]} if c["mass"] else {})}
    G, S, N, L = c["kv_heads"], c["sequences"], s["most_new"], s["most"]
    T, H = s["q"].shape[:2]
    seq, row = _where(s)
    place = torch.arange(T, device="cuda") - s["starts"].long()[seq]
    q = s["q"].new_zeros((S, N, H, c["dim"]), dtype=torch.float32)
    q[seq, place] = s["q"].float()
    at = torch.full((S, N), -1, device="cuda")
    at[seq, place] = row
    q = q.view(S, N, G, H // G, -1).permute(0, 2, 3, 1, 4)               # [sequences, kv heads, heads of a group, tokens, features]
    z = torch.matmul(q.flatten(2, 3), _rows(s["keys"], s["table"], L).transpose(-1, -2)).view(S, G, H // G, N, L) * scale
    j = torch.arange(L, device="cuda")
    seen = j <= at[..., None]
    if c["window"]:
        seen &= (j > at[..., None] - c["window"]) | (j < c["first"])
    z.masked_fill_(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    if c["sink"]:
        sink = s["sink"].view(G, H // G, 1, 1)
        top = torch.maximum(top, sink)
    top = top.masked_fill(at[:, None, None, :, None] < 0, 0.0)
    p = z.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + (sink - top).exp()
    p /= total.masked_fill(at[:, None, None, :, None] < 0, 1.0)
    v = _rows(s["values"], s["table"], L)
    o = torch.matmul(p.flatten(2, 3), v).view(S, G, H // G, N, -1).permute(0, 3, 1, 2, 4).flatten(2)
    s["out"].copy_(o[seq, place])
    if not c["mass"]:
        return {"out": s["out"]}
    s["mass"][:, :, :L] += p.sum((2, 3))
    return {"out": s["out"], "mass": s["mass"]}


def _moved(into):
    return {n: into[n] for n in ("keys", "values", "mass", "lengths")}


def _evict(s):
    c, into = s["case"], s["into"]
    if own:
        h = s["own"]
        _dev().paged_evict(h["cache"], h["into"], c["keep"], first=c["first"], recent=c["recent"])
        return _moved(into)
    R, G, K = c["page"], c["kv_heads"], min(c["keep"], s["most"])
    L = s["lengths"].long()
    j = torch.arange(s["most"], device="cuda")
    m = s["mass"][:, :, :s["most"]]
    stays = (j < c["first"]) | (j >= L[:, None] - c["recent"]) | (L[:, None] <= K)
    m = m.masked_fill(stays[:, None], math.inf).masked_fill((j >= L[:, None])[:, None], -math.inf)
    kept = m.sort(dim=-1, descending=True, stable=True).indices[:, :, :K]
    kept = kept.masked_fill(torch.arange(K, device="cuda") >= L[:, None, None], s["most"]).sort(-1).values      # what a short sequence lacks goes behind
    seq, to = s["kept"]                                                  # every row that is kept: its sequence and its new place
    src, seq, to, head = kept[seq, :, to], seq[:, None], to[:, None], torch.arange(G, device="cuda")
    page, new = s["table"].long()[seq, src // R], into["table"].long()[seq, to // R]
    into["keys"][new, head, to % R] = s["keys"][page, head, src % R]
    into["values"][new, head, to % R] = s["values"][page, head, src % R]
    into["mass"][seq, head, to] = s["mass"][seq, head, src]
    into["lengths"].copy_(L.clamp(max=c["keep"]))
    return _moved(into)


# ---------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    return {"rotary": _rotary_exact, "append": _append_exact, "attend": _attend_exact, "evict": _evict_exact}[case["kind"]](case, seed)


def _rotary_exact(case, seed):
    x, positions, freqs = _rotary_inputs(case, seed)
    T, H, D = case["tokens"], case["heads"], case["dim"]
    y = x[:, :H * D].double().reshape(T, H, D).clone()
    f = freqs.double().sum(0)
    i = 0
    for axis, pairs in enumerate(_sections(case)):
        for k in range(i, i + pairs):
            a, b = (k, k + D // 2) if case["halves"] else (2 * k, 2 * k + 1)
            turn = torch.polar(torch.ones(T, dtype=torch.float64, device="cuda"), positions[axis].double() * f[k])
            z = torch.complex(y[..., a].clone(), y[..., b].clone()) * turn[:, None]
            y[..., a], y[..., b] = z.real, z.imag
        i += pairs
    return {"out": y}


def _append_exact(case, seed):
    s = _inputs(case, seed)
    new, rows = _lengths(case)
    keys, values, table, R, t = s["keys"].double(), s["values"].double(), s["table"].tolist(), case["page"], 0
    mass = s["mass"].double() if case["mass"] else None
    for i, (n, L) in enumerate(zip(new, rows)):
        at = L - n
        while at < L:                           # a page at a time
            m = min(L - at, R - at % R)
            p, o = table[i][at // R], at % R
            keys[p, :, o:o + m] = s["k"][t:t + m].double().reshape(m, case["kv_heads"], -1).transpose(0, 1)
            values[p, :, o:o + m] = s["v"][t:t + m, 64:].double().reshape(m, case["kv_heads"], -1).transpose(0, 1)
            at, t = at + m, t + m
        if mass is not None:
            mass[i, :, L - n:L] = 0
    return {"keys": keys, "values": values, **({} if mass is None else {"mass": mass})}


def _attend_exact(case, seed):
    s = _inputs(case, seed)
    new, rows = _lengths(case)
    G, per, R, table = case["kv_heads"], case["heads"] // case["kv_heads"], case["page"], s["table"].tolist()
    out = torch.empty(s["q"].shape[0], case["heads"], case["vdim"], dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if case["mass"] else None
    t = 0
    for i, (n, L) in enumerate(zip(new, rows)):
        pages = torch.tensor(table[i][:-(-L // R)], device="cuda")
        at, j = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
        hidden = j > at
        if case["window"]:
            hidden = hidden | ((at - j >= case["window"]) & (j >= case["first"]))
        for g in range(G):
            k = s["keys"][pages, g].reshape(-1, case["dim"])[:L].double()
            v = s["values"][pages, g].reshape(-1, case["vdim"])[:L].double()
            for h in range(g * per, g * per + per):
                z = (s["q"][t:t + n, h].double() @ k.T) / math.sqrt(case["dim"])
                z[hidden] = -math.inf
                if case["sink"]:
                    z = torch.cat([z, s["sink"][h].double().expand(n, 1)], 1)
                w = torch.softmax(z, 1)[:, :L]
                out[t:t + n, h] = w @ v
                if mass is not None:
                    mass[i, g, :L] += w.sum(0)
        t += n
    return {"out": out.flatten(1), **({} if mass is None else {"mass": mass})}


def _evict_exact(case, seed):
    s = _inputs(case, seed)
    _, rows = _lengths(case)
    R, into = case["page"], s["into"]
    keys, values, mass = into["keys"].double(), into["values"].double(), into["mass"].double()
    lengths = []
    for i, L in enumerate(rows):
        weights = s["mass"][i, :, :L].cpu().numpy()
        n = min(L, case["keep"])
        lengths.append(n)
        for g in range(case["kv_heads"]):
            if n == L:
                kept = np.arange(L)
            else:
                first, last = min(case["first"], n), L - min(case["recent"], n)
                middle = np.arange(first, last)
                best = middle[np.lexsort((middle, -weights[g, middle]))][:n - first - (L - last)]
                kept = np.concatenate([np.arange(first), np.sort(best), np.arange(last, L)])
            src, dst = torch.from_numpy(kept).cuda(), torch.arange(n, device="cuda")
            a, b = s["table"][i].long()[src // R], into["table"][i].long()[dst // R]
            keys[b, g, dst % R] = s["keys"][a, g, src % R].double()
            values[b, g, dst % R] = s["values"][a, g, src % R].double()
            mass[i, g, :n] = s["mass"][i, g, src].double()
    return {"keys": keys, "values": values, "mass": mass, "lengths": torch.tensor(lengths, dtype=torch.float64)}
