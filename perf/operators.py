"""Timed cases of the paged INT8 key/value cache and of the attention that reads it (cactus_amd/paged.py).

Three operators, each with a plain form in elementary torch operations and the framework's own calls (`own`):
  append   one step's q / k / v rows: per-head RMS norm, rotation, quantization into the pages, then the touched
           tokens read back as halves (kv_append, kv_read)
  paged    attention over the paged cache, one token or a chunk per sequence, full or window + sinks (attention)
  ragged   FP16 attention of whole prompts packed one behind the other, full or window + sinks (attention_ragged)

A page holds `page` tokens of one sequence: int8 [pages, kv_heads, page, head_dim] with one float32 scale per page and
kv head.  Token j of a sequence is visible to position p when j <= p and, with a window, p - j <= window or j < sink.
"""
import math
import random

import torch

own = False

EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------ cases

def _append(name, batch, shape, page, past, new, salt, theta=1e6, norm=True):
    heads, kv_heads, head_dim = shape
    return {"name": name, "op": "append", "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "past_low": past[0], "past_high": past[1], "new_low": new[0], "new_high": new[1],
            "salt": salt, "theta": theta, "norm": norm}


def _paged(name, batch, shape, page, past, new, salt, window=0, sink=0):
    heads, kv_heads, head_dim = shape
    return {"name": name, "op": "paged", "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "past_low": past[0], "past_high": past[1], "new_low": new[0], "new_high": new[1],
            "salt": salt, "window": window, "sink": sink}


def _ragged(name, batch, shape, new, salt, window=0, sink=0):
    heads, kv_heads, head_dim = shape
    return {"name": name, "op": "ragged", "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "new_low": new[0], "new_high": new[1], "salt": salt, "window": window, "sink": sink}


# (query heads, kv heads, head_dim) of the decoder shapes that the repository's benchmark and tests use
QWEN3, LFM2, GEMMA, WIDE = (16, 8, 128), (32, 8, 64), (4, 1, 256), (32, 8, 128)


def listed():
    return [
        # one sequence generating a token: latency is all there is
        _append("append 1 token", 1, QWEN3, 16, (515, 515), (1, 1), 1),
        # a full decode batch, every sequence at its own position
        _append("append 256 tokens", 256, QWEN3, 64, (300, 700), (1, 1), 2),
        # prompts of odd lengths admitted together, from position 0
        _append("append prompts", 7, LFM2, 32, (0, 0), (500, 1900), 3),
        # later prompt chunks that begin inside a page whose earlier tokens are requantized; far positions
        _append("append chunks", 5, GEMMA, 128, (1000, 30000), (100, 256), 4, theta=1e4),
        # decode of one conversation
        _paged("decode 1 x 4k", 1, QWEN3, 16, (4090, 4090), (1, 1), 5),
        # decode of a full batch
        _paged("decode 256 x 512", 256, QWEN3, 64, (300, 700), (1, 1), 6),
        # decode of a few long documents
        _paged("decode 4 x 32k", 4, WIDE, 64, (30011, 32766), (1, 1), 7),
        # decode of a layer with a sliding window and the first tokens kept
        _paged("decode window", 64, GEMMA, 32, (2000, 8000), (1, 1), 8, window=508, sink=4),
        # prompt chunks against what the cache already holds
        _paged("chunk on 4k", 3, QWEN3, 16, (3500, 4100), (131, 256), 9),
        # short prompts admitted together
        _ragged("prompts short", 24, LFM2, (17, 300), 10),
        # one long prompt
        _ragged("prompt 4k", 1, QWEN3, (4096, 4096), 11),
        # long prompts of a sliding-window layer
        _ragged("prompts window", 3, GEMMA, (4001, 8190), 12, window=508, sink=4),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    shapes = [QWEN3, LFM2, GEMMA, WIDE, (8, 8, 128), (12, 4, 64), (9, 3, 64), (20, 4, 128), (8, 2, 256), (32, 2, 64)]
    limit = max(_cost(c) for c in listed())
    while True:
        op, shape, salt = rng.choice(["append", "paged", "ragged"]), rng.choice(shapes), rng.randrange(1 << 20)
        batch = _log(rng, 1, 256)
        page = rng.choice([16, 32, 64, 128])
        top = max(1, _log(rng, 1, 8192) // batch)
        new = rng.choice([(1, 1), (max(0, top // 3), top)])
        past_high = _log(rng, 1, 32768)
        past = (rng.randrange(past_high + 1), past_high)
        window, sink = rng.choice([(0, 0), (_log(rng, 1, 4096), 0), (_log(rng, 16, 1024), rng.choice([1, 4, 17, 64]))])
        if op == "append":
            case = _append("", batch, shape, page, past, new, salt, rng.choice([1e4, 1e6]), rng.random() < 0.6)
        elif op == "paged":
            case = _paged("", batch, shape, page, past, new, salt, window, sink)
        else:
            top = _log(rng, 1, 8192)
            batch = min(batch, max(1, 16384 // top))
            case = _ragged("", batch, shape, (max(1, top // 3), top), salt, window, sink)
        del case["name"]
        # what the plain forms hold: padded scores, and the gathered cache in float32
        news, pasts = _lengths(case)
        longest = max(n + p for n, p in zip(news, pasts))
        scores = batch * shape[0] * max(news) * longest if op != "append" else 0
        held = batch * shape[1] * shape[2] * longest
        if _cost(case) <= limit and scores <= 600e6 and held <= 400e6:
            return case


def _lengths(case):
    """(new tokens, tokens before them) of every sequence; at least one new token in all."""
    r = random.Random(case["salt"])
    news = [r.randint(case["new_low"], case["new_high"]) for _ in range(case["batch"])]
    pasts = [r.randint(case.get("past_low", 0), case.get("past_high", 0)) for _ in range(case["batch"])]
    if not sum(news):
        news[0] = 1
    return news, pasts


def _seen(case, position):
    """How many keys a query at `position` sees."""
    if not case["window"]:
        return position + 1
    first = max(0, position - case["window"])
    return position + 1 - first + min(first, case["sink"])


def work(case):
    news, pasts = _lengths(case)
    tokens, Hq, Hkv, D = sum(news), case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        page = case["page"]
        back = sum(p % page + n for n, p in zip(news, pasts))
        touched = sum((p + n + page - 1) // page - p // page for n, p in zip(news, pasts))
        moved = tokens * (Hq + 2 * Hkv) * D * 2 + tokens * Hq * D * 2 + tokens * 2 * Hkv * D   # rows in, q out, int8 out
        moved += back * 2 * Hkv * D * 3                                                      # int8 in, halves out
        return {"bytes": moved + touched * 2 * Hkv * 4 * 3, "flops": tokens * (Hq + Hkv) * D * 8 + back * 2 * Hkv * D}
    pairs = keys = scales = 0
    for n, p in zip(news, pasts):
        if not n:
            continue
        if case["window"]:
            w, s = case["window"], case["sink"]
            pairs += sum(_seen(case, p + i) for i in range(n))
            first = max(0, p - w)
            read = p + n - first + min(first, s)
        else:
            pairs += n * p + n * (n + 1) // 2
            read = p + n
        keys += read
        scales += (read + case["page"] - 1) // case["page"] if case["op"] == "paged" else 0
    one = 1 if case["op"] == "paged" else 2
    return {"bytes": tokens * Hq * D * 4 + keys * 2 * Hkv * D * one + scales * 2 * Hkv * 4,
            "flops": 4 * pairs * Hq * D}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 5e14)


# ------------------------------------------------------------------------------------------------------------ inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lengths):
    total, out = 0, [0]
    for n in lengths:
        total += n
        out.append(total)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    news, pasts = _lengths(case)
    tokens, Hq, Hkv, D = sum(news), case["heads"], case["kv_heads"], case["head_dim"]
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=gen)                           # noqa: E731
    s = {"case": case, "cu": _ints(_offsets(news)), "longest_new": max(news), "one_each": max(news) == min(news) == 1}
    # the rows of a fused q/k/v projection; the attention's q (and the prompts' k) come out of the rotation as
    # tensors of their own
    fused = normal(tokens, (Hq + 2 * Hkv) * D).half()
    s["q"] = fused[:, :Hq * D].unflatten(1, (Hq, D))
    s["k"] = fused[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
    s["v"] = fused[:, (Hq + Hkv) * D:].unflatten(1, (Hkv, D))
    if case["op"] != "append":
        s["q"] = (s["q"] * 1.5).contiguous()
        s["k"] = s["k"].contiguous()
    if case["op"] == "ragged":
        return s
    if case["op"] == "append" and case["norm"]:
        s["q_weight"] = (1 + 0.1 * normal(D)).half()
        s["k_weight"] = (1 + 0.1 * normal(D)).half()
    # pages in no particular order, a few of them nobody's; entries past a sequence's last page are -1
    page = case["page"]
    used = [(n + p + page - 1) // page for n, p in zip(news, pasts)]
    total = sum(used) + 3
    width = max(used) + 1
    order = torch.randperm(total, device="cuda", generator=gen).int()
    at = torch.arange(width, device="cuda")[None] + torch.tensor(_offsets(used)[:-1], device="cuda")[:, None]
    here = torch.arange(width, device="cuda")[None] < _ints(used)[:, None]
    s["nobodys"] = order[total - 1].long()
    s["tables"] = torch.where(here, order[at.clamp_max(total - 1)], -1).int().contiguous()
    pages = lambda: (normal(total, Hkv, page, D) * 32).round_().clamp_(-127, 127).to(torch.int8)       # noqa: E731
    scales = lambda: 0.01 + 0.03 * torch.rand((total, Hkv), device="cuda", generator=gen)              # noqa: E731
    s["kv"] = (pages(), pages(), scales(), scales())
    s["past"] = _ints(pasts)
    s["context"] = _ints([n + p for n, p in zip(news, pasts)])
    s["longest"] = max(n + p for n, p in zip(news, pasts))
    if case["op"] == "append":
        s["read_from"] = _ints([p // page * page for p in pasts])
        back = [p % page + n for n, p in zip(news, pasts)]
        s["read_cu"] = _ints(_offsets(back))
        s["read_rows"] = sum(back)
    return s


# --------------------------------------------------------------------------------------------------------------- run

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"append": _plain_append, "paged": _plain_paged, "ragged": _plain_ragged}[op](state)


def _own(s, op):
    from cactus_amd import paged
    c = s["case"]
    if op == "append":
        q = paged.kv_append(s["k"], s["v"], s["kv"], s["tables"], s["past"], c["theta"],
                            cu_seqlens=None if s["one_each"] else s["cu"], q=s["q"], q_weight=s.get("q_weight"),
                            k_weight=s.get("k_weight"), eps=EPS)
        k, v = paged.kv_read(s["kv"], s["tables"], s["read_from"], s["read_cu"], s["read_rows"])
        return {"q": q, "k": k, "v": v, "k_scales": s["kv"][2], "v_scales": s["kv"][3]}
    if op == "paged":
        return paged.attention(s["q"], s["kv"], s["tables"], s["context"], cu_seqlens=None if s["one_each"] else s["cu"],
                               max_context=s["longest"], window=c["window"], sink=c["sink"])
    return paged.attention_ragged(s["q"], s["k"], s["v"], s["cu"], window=c["window"], sink=c["sink"])


def _owners(cu, rows):
    """The sequence of every packed row, and the row's place in it."""
    counts = (cu[1:] - cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=cu.device), counts, output_size=rows)
    return seq, torch.arange(rows, device=cu.device) - cu[:-1].long()[seq]


def _normed(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    c = s["case"]
    page, D = c["page"], c["head_dim"]
    k_pages, v_pages, k_scales, v_scales = s["kv"]
    tables, past = s["tables"].clamp_min(0).long(), s["past"].long()
    seq, i = _owners(s["cu"], s["q"].shape[0])
    pos = past[seq] + i
    freq = c["theta"] ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    angle = pos[:, None, None].double() * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotated(_normed(s["q"], s.get("q_weight")), cos, sin).half()
    k = _rotated(_normed(s["k"], s.get("k_weight")), cos, sin)
    pid, slot = tables[seq, pos // page], pos % page
    first = tables.gather(1, (past // page)[:, None])[:, 0]         # the page a sequence's first new token falls into
    held = past % page                                              # tokens it already holds
    writes = s["cu"][1:] > s["cu"][:-1]
    for x, pages, scales in ((k, k_pages, k_scales), (s["v"].float(), v_pages, v_scales)):
        grown = torch.zeros_like(scales)
        old = torch.where((held > 0)[:, None], scales[first], 0.0)
        grown.index_reduce_(0, first, torch.where(writes[:, None], old, 0.0), "amax")
        peak = torch.zeros_like(scales).index_reduce_(0, pid, x.abs().amax(-1), "amax")
        grown = torch.maximum(grown, (peak / 127).clamp_min(1e-10))
        was = pages[first].float()
        again = torch.round(was * (old / grown[first])[:, :, None, None])
        keep = writes[:, None, None, None] & (torch.arange(page, device="cuda") < held[:, None])[:, None, :, None]
        # a sequence without new tokens writes into a page of nobody's
        pages[torch.where(writes, first, s["nobodys"])] = torch.where(keep, again, was).to(torch.int8)
        pages[pid, :, slot] = torch.round(x / grown[pid][:, :, None]).clamp(-127, 127).to(torch.int8)
        scales[pid] = grown[pid]
    seq, i = _owners(s["read_cu"], s["read_rows"])
    pos = s["read_from"].long()[seq] + i
    pid, slot = tables[seq, pos // page], pos % page
    k = (k_pages[pid, :, slot].float() * k_scales[pid][:, :, None]).half()
    v = (v_pages[pid, :, slot].float() * v_scales[pid][:, :, None]).half()
    return {"q": q, "k": k, "v": v, "k_scales": k_scales, "v_scales": v_scales}


def _visible(case, pos, keys):
    """[.., queries, keys]: which keys a position sees."""
    j = torch.arange(keys, device="cuda")
    pos = pos[..., None]
    seen = j <= pos
    if case["window"]:
        seen &= (pos - j <= case["window"]) | (j < case["sink"])
    return seen


def _softmaxed(q, k, v, seen):
    """q [B, Hkv, g, n, D] (float), k / v [B, Hkv, L, D], seen [B, n, L] -> [B, Hkv, g, n, D]."""
    B, Hkv, g, n, D = q.shape
    scores = torch.matmul(q.reshape(B, Hkv, g * n, D) * D ** -0.5, k.transpose(-1, -2)).reshape(B, Hkv, g, n, -1)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.reshape(B, Hkv, g * n, -1), v).reshape(B, Hkv, g, n, D)
    return out / torch.where(total > 0, total, 1.0)


def _plain_paged(s):
    c = s["case"]
    Hq, Hkv, D, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    k_pages, v_pages, k_scales, v_scales = s["kv"]
    B, n = c["batch"], s["longest_new"]
    tables = s["tables"][:, :(s["longest"] + page - 1) // page].clamp_min(0).long()
    L = tables.shape[1] * page
    cached = lambda pages, scales: (pages[tables].float() * scales[tables][..., None, None]).transpose(1, 2).reshape(B, Hkv, L, D)  # noqa: E731
    rows = (s["cu"][:-1].long()[:, None] + torch.arange(n, device="cuda")).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[rows].reshape(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    pos = s["context"].long()[:, None] - (s["cu"][1:] - s["cu"][:-1]).long()[:, None] + torch.arange(n, device="cuda")
    out = _softmaxed(q, cached(k_pages, k_scales), cached(v_pages, v_scales), _visible(c, pos, L))
    seq, i = _owners(s["cu"], s["q"].shape[0])
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[seq, i].half()


def _plain_ragged(s):
    c = s["case"]
    Hq, Hkv, D = c["heads"], c["kv_heads"], c["head_dim"]
    B, n = c["batch"], s["longest_new"]
    rows = (s["cu"][:-1].long()[:, None] + torch.arange(n, device="cuda")).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[rows].reshape(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    k, v = s["k"].float()[rows].transpose(1, 2), s["v"].float()[rows].transpose(1, 2)
    pos = torch.arange(n, device="cuda").expand(B, n)
    out = _softmaxed(q, k, v, _visible(c, pos, n))
    seq, i = _owners(s["cu"], s["q"].shape[0])
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[seq, i].half()


# ------------------------------------------------------------------------------------------------------------- exact

def exact(case, seed):
    """The definitions in 64 bits, one sequence at a time."""
    s = prepare(case, seed)
    news, pasts = _lengths(case)
    if case["op"] == "append":
        return _exact_append(case, s, news, pasts)
    Hq, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    outs, start = [], 0
    for b, (n, p) in enumerate(zip(news, pasts)):
        rows = slice(start, start + n)
        start += n
        if not n:
            continue
        if case["op"] == "paged":
            pages = s["tables"][b, :(n + p + case["page"] - 1) // case["page"]].long()
            k, v = ((x[pages].double() * y[pages].double()[:, :, None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :n + p]
                    for x, y in ((s["kv"][0], s["kv"][2]), (s["kv"][1], s["kv"][3])))
        else:
            k, v = s["k"][rows].double().permute(1, 0, 2), s["v"][rows].double().permute(1, 0, 2)
        out = torch.empty((n, Hq, D), dtype=torch.float64, device="cuda")
        far = torch.arange(p, p + n, device="cuda")[:, None] - torch.arange(n + p, device="cuda")[None]
        hidden = far < 0
        if case["window"]:
            hidden |= (far > case["window"]) & (torch.arange(n + p, device="cuda") >= case["sink"])
        for h in range(Hq):
            one = s["q"][rows, h].double() @ k[h * Hkv // Hq].T / math.sqrt(D)
            one[hidden] = -math.inf
            out[:, h] = torch.softmax(one, -1) @ v[h * Hkv // Hq]
        outs.append(out)
    return torch.cat(outs)


def _exact_append(case, s, news, pasts):
    page, D, half = case["page"], case["head_dim"], case["head_dim"] // 2
    stores = [(s["kv"][0].double(), s["kv"][2].double()), (s["kv"][1].double(), s["kv"][3].double())]
    freq = torch.tensor([case["theta"] ** (-2.0 * i / D) for i in range(half)], dtype=torch.float64, device="cuda")
    qs, back, start = [], ([], []), 0
    for b, (n, p) in enumerate(zip(news, pasts)):
        rows = slice(start, start + n)
        start += n
        turn = torch.polar(torch.ones((n, half), dtype=torch.float64, device="cuda"),
                           torch.arange(p, p + n, dtype=torch.float64, device="cuda")[:, None] * freq)[:, None]

        def turned(x, weight):
            x = x.double()
            if weight is not None:
                x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * weight.double()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        qs.append(turned(s["q"][rows], s.get("q_weight")))
        fresh = (turned(s["k"][rows], s.get("k_weight")), s["v"][rows].double())
        ids = s["tables"][b].tolist()
        for j in range(p // page, (p + n + page - 1) // page):
            low, high = max(p, j * page), min(p + n, (j + 1) * page)
            if high <= low:
                continue
            for (values, scales), x in zip(stores, fresh):
                x = x[low - p:high - p].transpose(0, 1)
                old = scales[ids[j]] if low > j * page else torch.zeros_like(scales[ids[j]])
                new = torch.maximum(old, x.abs().amax((1, 2)) / 127).clamp_min(1e-10)
                held = values[ids[j], :, :low - j * page]
                values[ids[j], :, :low - j * page] = torch.round(held * (old / new)[:, None, None])
                values[ids[j], :, low - j * page:high - j * page] = torch.round(x / new[:, None, None])
                scales[ids[j]] = new
        low = p // page * page
        at = torch.arange(low, p + n, device="cuda")
        pid = s["tables"][b].long()[at // page]
        for out, (values, scales) in zip(back, stores):
            out.append(values[pid, :, at % page] * scales[pid][:, :, None])
    return {"q": torch.cat(qs), "k": torch.cat(back[0]), "v": torch.cat(back[1]), "k_scales": stores[0][1],
            "v_scales": stores[1][1]}
