"""Measured cases of the paged KV-cache operators.

Four operators a serving loop runs around a paged cache:

* ``attention`` -- one new token per row over a paged KV cache (grouped heads,
  optional sliding window with a few first tokens that stay visible);
* ``append``    -- rotary positions on the new rows' q and k, and k / v written
  into their pages;
* ``copy``      -- page copies over every layer (forking and compacting);
* ``beam``      -- beam search's selection over beams and vocabulary and the
  reordering of the beams' page tables that follows it.

``run`` computes an operator with elementary torch operations (``own`` false)
or with the calls a user makes of this package (``own`` true).
"""

from __future__ import annotations

import math
import sys

import torch

own = False


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    return [
        # a chat that has just begun, alone on the GPU: pure latency
        attention("attend one short", 1, 9, 3, 64, 16, 200, 200),
        # a few long contexts of very different lengths
        attention("attend few ragged", 8, 24, 8, 128, 64, 1024, 8192),
        # a full serving batch, the largest read of the cache
        attention("attend full batch", 64, 24, 8, 128, 64, 1024, 8192, out="bf16"),
        # one document of 131071 tokens: the split over the length does it all
        attention("attend one long", 1, 24, 8, 128, 128, 131071, 131071),
        # streaming batch: a window and four first tokens, older pages freed
        attention("attend window", 48, 15, 5, 64, 32, 1, 8000, window=1024, sinks=4),
        # fp32 cache, every head its own keys, a page size that is no power of two
        attention("attend fp32 odd page", 6, 12, 12, 64, 24, 17, 1003, cache="f32"),
        # one decode step's new tokens
        append("append step", 64, 64, 24, 8, 128, 128, "half", 64),
        # prompts of a prefill, half of each head rotated, neighbouring pairs
        append("append prompts", 12001, 7, 24, 8, 128, 64, "interleaved", 16),
        # beams that part inside a page: the filled rows of a few pages, all layers
        copy("fork beams", 56, 96, 8, 64, 128, 24, "partial"),
        # a fragmented pool moved together: whole pages, all layers
        copy("compact pool", 60, 900, 3, 64, 64, 420, "whole"),
        # one request with four beams
        beam("beams of one request", 1, 4, 49152, 16, 64),
        # sixteen requests with eight beams each over a large vocabulary
        beam("beams of a batch", 16, 8, 128256, 130, 64),
    ]


def attention(name, rows, heads, kv_heads, dim, page, len_min, len_max, window=0,
              sinks=0, cache="bf16", out="f32"):
    c = dict(op="attention", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim,
             page=page, len_min=len_min, len_max=len_max, window=window, sinks=sinks,
             cache=cache, out=out)
    return dict(c, name=name) if name else c


def append(name, rows, seqs, heads, kv_heads, dim, rotary, pairs, page, cache="bf16"):
    c = dict(op="append", rows=rows, seqs=seqs, heads=heads, kv_heads=kv_heads,
             dim=dim, rotary=rotary, pairs=pairs, page=page, cache=cache)
    return dict(c, name=name) if name else c


def copy(name, planes, pages, kv_heads, page, dim, copies, fill, cache="bf16"):
    c = dict(op="copy", planes=planes, pages=pages, kv_heads=kv_heads, page=page,
             dim=dim, copies=copies, fill=fill, cache=cache)
    return dict(c, name=name) if name else c


def beam(name, groups, beams, vocab, columns, page):
    c = dict(op="beam", groups=groups, beams=beams, vocab=vocab, columns=columns,
             page=page)
    return dict(c, name=name) if name else c


def _spread(rng, low, high):
    """A whole number, uniform over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low),
                                                             math.log(high)))))))


HEADS = [(9, 3, 64), (15, 5, 64), (32, 32, 64), (12, 12, 64), (24, 8, 128),
         (16, 2, 128), (8, 1, 128), (6, 2, 96)]


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "copy", "beam"])
    if op == "attention":
        heads, kv_heads, dim = rng.choice(HEADS)
        cache = rng.choice(["bf16", "bf16", "bf16", "f32"])
        size = kv_heads * dim * 2 * (2 if cache == "bf16" else 4)
        rows = _spread(rng, 1, 64)
        len_max = _spread(rng, 1, max(1, min(131071, (1 << 30) // (size * rows))))
        len_min = rng.choice([0, 1, len_max // 8, len_max])
        window = rng.choice([0, 0, 0, _spread(rng, 1, 4096)])
        return attention("", rows, heads, kv_heads, dim,
                         rng.choice([16, 32, 64, 64, 128, 20]), len_min, len_max, window,
                         rng.choice([0, 1, 4, 4, 33]) if window else 0, cache,
                         rng.choice(["f32", "bf16"]))
    if op == "append":
        heads, kv_heads, dim = rng.choice(HEADS)
        rows = _spread(rng, 1, 12000)
        return append("", rows, rng.choice([1, max(1, rows // 100), rows]), heads,
                      kv_heads, dim, rng.choice([dim, dim, dim // 2]),
                      rng.choice(["half", "interleaved"]), rng.choice([16, 32, 64, 20]),
                      rng.choice(["bf16", "bf16", "f32"]))
    if op == "copy":
        kv_heads, dim = rng.choice([(3, 64), (5, 64), (8, 128), (1, 128)])
        page = rng.choice([16, 32, 64, 20])
        planes = rng.choice([2, 24, 56, 60])
        most = (1 << 31) // (planes * kv_heads * page * dim * 2)
        pages = _spread(rng, 4, max(4, min(2000, most)))
        return copy("", planes, pages, kv_heads, page, dim, rng.randint(1, pages // 2),
                    rng.choice(["partial", "whole"]))
    return beam("", _spread(rng, 1, 16), _spread(rng, 1, 8),
                _spread(rng, 1000, 128256), _spread(rng, 2, 130), rng.choice([16, 64]))


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _lens(case):
    """Row lengths, spread evenly over [len_min, len_max]."""
    n, lo, hi = case["rows"], case["len_min"], case["len_max"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _live(case, length):
    """Keys that a row of this length attends."""
    if not case["window"]:
        return length
    return min(length, min(case["sinks"], length) + case["window"]) \
        if length > case["window"] else length


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    h = torch.Generator().manual_seed(int(seed))
    make = {"attention": _prepare_attention, "append": _prepare_append,
            "copy": _prepare_copy, "beam": _prepare_beam}[case["op"]]
    state = dict(make(case, g, h), case=case)
    if own and "table" in state and "k" in state:
        # the cache handle that a serving program builds once beside its pages
        state["kv"] = _package().PagedKV(state["k"], state["v"], state["table"])
    return state


kernels = None


def _package():
    """This package's kernels, imported once."""
    global kernels
    if kernels is None:
        sys.path.insert(0, "triton-llm_b200")
        import triton_llm.kernels
        kernels = triton_llm.kernels
    return kernels


def _normal(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)


def _prepare_attention(c, g, h):
    R, P, D, dt = c["rows"], c["page"], c["dim"], DTYPES[c["cache"]]
    lens = torch.tensor(_lens(c))[torch.randperm(R, generator=h)]
    columns = max(1, -(-int(lens.max()) // P))
    first = torch.arange(columns)[None, :] * P
    end = lens[:, None]
    needed = first < end
    if c["window"]:   # pages that hold no visible key have been freed
        needed &= (first < c["sinks"]) | (first + P > end - c["window"])
    n = int(needed.sum())
    table = torch.full((R, columns), -1, dtype=torch.int32)
    table[needed] = torch.randperm(n + 2, generator=h)[:n].int()
    out_dt = DTYPES[c["out"]]
    return dict(
        k=_normal(g, n + 2, c["kv_heads"], P, D, dtype=dt),
        v=_normal(g, n + 2, c["kv_heads"], P, D, dtype=dt),
        q=_normal(g, R, c["heads"], D), table=table.cuda(), lens=lens.int().cuda(),
        max_len=int(lens.max()), keys=int(lens.sum()),
        out=torch.empty(R, c["heads"], D, dtype=out_dt, device="cuda"))


def _rope_tables(positions, rotary):
    """cos and sin of each position and pair, wavelengths stretched for a long
    context: slow pairs by a factor of 8, fast ones not, a ramp between."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    freq = 500000.0 ** (-2 * i / rotary)
    turns = 8192 * freq / (2 * math.pi)
    keep = ((turns - 1) / 3).clamp(0, 1)
    freq = freq * (keep + (1 - keep) / 8)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _prepare_append(c, g, h):
    R, S, P, D, dt = c["rows"], c["seqs"], c["page"], c["dim"], DTYPES[c["cache"]]
    # S sequences take R / S new tokens each (the last one the rest), after
    # some that they hold already
    each = max(1, R // S)
    seq = (torch.arange(R) // each).clamp(max=S - 1)
    held = torch.randint(0, 300, (S,), generator=h)
    start = torch.arange(S) * each
    pos = held[seq] + torch.arange(R) - start[seq]
    columns = int(pos.max()) // P + 1
    tail = torch.zeros(S, dtype=torch.long).scatter_reduce_(0, seq, pos, "amax")
    # pages of tokens held before the new ones are elsewhere in the pool
    col = torch.arange(columns)[None, :]
    needed = (col <= (tail // P)[:, None]) & (col >= (held // P)[:, None])
    n = int(needed.sum())
    table = torch.full((S, columns), -1, dtype=torch.int32)
    table[needed] = torch.randperm(n + 1, generator=h)[:n].int()
    cos, sin = _rope_tables(int(pos.max()) + 1, c["rotary"])
    return dict(
        k=_normal(g, n + 1, c["kv_heads"], P, D, dtype=dt),
        v=_normal(g, n + 1, c["kv_heads"], P, D, dtype=dt),
        qkv=_normal(g, R, (c["heads"] + 2 * c["kv_heads"]) * D),
        q_out=torch.empty(R, c["heads"], D, device="cuda"),
        table=table.cuda(), seq=seq.int().cuda(), pos=pos.int().cuda(), cos=cos, sin=sin)


def _parents(copies):
    return copies - copies // 4


def _prepare_copy(c, g, h):
    N, n, P = c["pages"], c["copies"], c["page"]
    perm = torch.randperm(N, generator=h)
    src, dst = perm[:n], perm[N - n:]
    if c["fill"] == "partial":      # several beams may come from the same page
        src = src[torch.randint(0, _parents(n), (n,), generator=h)]
    own_page = torch.rand(n, generator=h) < 0.1     # a beam that stays where it is
    src, dst = torch.where(own_page, dst, src), dst
    fill = torch.randint(1, P + 1, (n,), generator=h) if c["fill"] == "partial" \
        else torch.full((n,), P)
    return dict(
        arena=_normal(g, c["planes"], N, c["kv_heads"], P, c["dim"],
                      dtype=DTYPES[c["cache"]]),
        src=src.int().cuda(), dst=dst.int().cuda(), fill=fill.int().cuda())


def _prepare_beam(c, g, h):
    G, W, V, C, P = c["groups"], c["beams"], c["vocab"], c["columns"], c["page"]
    scores = -(torch.rand(G, W, generator=h) * 20 + 5).sort(dim=1)[0]
    done = torch.rand(G, W, generator=h) < 0.1
    length = torch.randint(1, (C - 1) * P, (G,), generator=h)
    # full pages before the last are shared by a group's beams
    table = torch.randperm(G * W * C, generator=h).int().view(G, W, C)
    shared = torch.arange(C)[None, :] < (length // (2 * P))[:, None]
    table = torch.where(shared[:, None, :], table[:, :1], table)
    return dict(
        # a language model's logits: mostly noise, a few tokens stand out
        logits=_normal(g, G * W, V, scale=2.5), scores=scores.cuda(),
        done=done.int().cuda(), pad=V - 1,
        table=table.reshape(G * W, C).contiguous().cuda(),
        lens=length.int().repeat_interleave(W).cuda(),
        out=dict(scores=torch.empty(G, W, device="cuda"),
                 parents=torch.empty(G, W, dtype=torch.int32, device="cuda"),
                 tokens=torch.empty(G, W, dtype=torch.int32, device="cuda"),
                 table=torch.empty(G * W, C, dtype=torch.int32, device="cuda"),
                 src=torch.empty(G * W, dtype=torch.int32, device="cuda"),
                 dst=torch.empty(G * W, dtype=torch.int32, device="cuda"),
                 fill=torch.empty(G * W, dtype=torch.int32, device="cuda")))


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "append": _own_append, "copy": _own_copy,
                "beam": _own_beam}[op](state)
    return {"attention": _plain_attention, "append": _plain_append, "copy": _plain_copy,
            "beam": _plain_beam}[op](state)


def _own_attention(s):
    c = s["case"]
    return _package().paged_attention(
        s["kv"], s["q"], s["lens"], s["out"], max_len=s["max_len"], keys_hint=s["keys"],
        window=c["window"], sinks=c["sinks"])


def _own_append(s):
    c = s["case"]
    _package().paged_append(s["kv"], s["qkv"], s["pos"], s["q_out"], s["cos"], s["sin"],
                            n_head=c["heads"], row_seq=s["seq"],
                            interleaved=c["pairs"] == "interleaved")
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_copy(s):
    _package().page_copy(s["arena"], s["src"], s["dst"], s["fill"])
    return s["arena"]


def _own_beam(s):
    c, o = s["case"], s["out"]
    k = _package()
    k.beam_select(s["logits"], s["scores"], o["scores"], o["parents"], o["tokens"],
                  done=s["done"], pad_token=s["pad"])
    k.beam_reorder(o["parents"], s["lens"], s["table"], o["table"], o["src"], o["dst"],
                   o["fill"], page_size=c["page"])
    return o


def _visible(c, position, length):
    seen = position < length
    if c["window"]:
        seen = seen & ((position < c["sinks"]) | (position >= length - c["window"]))
    return seen


def _plain_attention(s):
    c = s["case"]
    R, H, K, D = c["rows"], c["heads"], c["kv_heads"], c["dim"]
    page = s["table"].clamp(min=0).long()
    S = page.shape[1] * c["page"]
    k = s["k"][page].float().permute(0, 2, 1, 3, 4).reshape(R, K, S, D)
    v = s["v"][page].float().permute(0, 2, 1, 3, 4).reshape(R, K, S, D)
    q = s["q"].view(R, K, H // K, D) / math.sqrt(D)
    seen = _visible(c, torch.arange(S, device="cuda")[None, :], s["lens"][:, None])
    score = (q @ k.transpose(2, 3)).masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = (score - top).exp()
    total = p.sum(dim=-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    return out.reshape(R, H, D).to(s["out"].dtype)


def _plain_rotate(x, cos, sin, pairs):
    r = 2 * cos.shape[-1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if pairs == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_append(s):
    c = s["case"]
    R, H, K, D, P = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    rows = s["qkv"].view(R, H + 2 * K, D)
    pos = s["pos"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _plain_rotate(rows[:, :H], cos, sin, c["pairs"])
    k = _plain_rotate(rows[:, H:H + K], cos, sin, c["pairs"])
    page, slot = s["table"][s["seq"].long(), pos // P].long(), pos % P
    s["k"][page, :, slot] = k.to(s["k"].dtype)
    s["v"][page, :, slot] = rows[:, H + K:].to(s["v"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_copy(s):
    a, src, dst = s["arena"], s["src"].long(), s["dst"].long()
    filled = torch.arange(a.shape[3], device="cuda")[None, :] < s["fill"][:, None]
    a[:, dst] = torch.where(filled[None, :, None, :, None], a[:, src], a[:, dst])
    return a


def _plain_beam(s):
    c = s["case"]
    G, W, V, C, P = c["groups"], c["beams"], c["vocab"], c["columns"], c["page"]
    x = s["logits"].view(G, W, V)
    top = x.amax(dim=-1, keepdim=True)
    norm = top + (x - top).exp().sum(dim=-1, keepdim=True).log()
    score = s["scores"][:, :, None] + (x - norm)
    # a finished beam proposes itself alone
    pad = torch.arange(V, device="cuda") == s["pad"]
    kept = torch.where(pad, s["scores"][:, :, None], -math.inf)
    score = torch.where(s["done"][:, :, None] != 0, kept, score).view(G, W * V)
    best, index = score.sort(dim=-1, descending=True, stable=True)
    best, index = best[:, :W].contiguous(), index[:, :W]
    parents, tokens = (index // V).int(), (index % V).int()
    # page tables: a beam takes its parent's pages; in the page that is partly
    # filled the first child keeps the parent's, the others copy it into the
    # pages of beams that end here
    length = s["lens"].view(G, W)[:, 0].long()
    column, fill = length // P, length % P
    old = s["table"].view(G, W, C)
    up = parents.long()
    child_of = up[:, :, None] == torch.arange(W, device="cuda")
    first = (child_of & (child_of.cumsum(dim=1) == 1)).any(dim=2)
    ends = ~child_of.any(dim=1)
    free = (ends[:, None, :] & ~first[:, :, None]
            & ((~first).cumsum(dim=1)[:, :, None] == ends.cumsum(dim=1)[:, None, :]))
    target = torch.where(first, up, free.int().argmax(dim=2))
    last = old.gather(2, column[:, None, None].expand(G, W, 1))[:, :, 0]
    src, dst = last.gather(1, up), last.gather(1, target)
    part = (fill > 0)[:, None]
    at = torch.arange(C, device="cuda")[None, None, :]
    moved = old.gather(1, up[:, :, None].expand(G, W, C))
    table = torch.where(at < column[:, None, None], moved, old)
    table = torch.where((at == column[:, None, None]) & part[:, :, None],
                        dst[:, :, None], table)
    fills = torch.where(part, fill[:, None], 0).expand(G, W)
    return {"scores": best, "parents": parents, "tokens": tokens,
            "table": table.reshape(G * W, C),
            "src": torch.where(part, src, -1).reshape(-1).int(),
            "dst": torch.where(part, dst, -1).reshape(-1).int(),
            "fill": fills.reshape(-1).int()}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append,
            "copy": lambda s: None, "beam": _exact_beam}[case["op"]](s)


def _exact_attention(s):
    c = s["case"]
    out = torch.zeros(c["rows"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    share = c["heads"] // c["kv_heads"]
    lens, table = s["lens"].tolist(), s["table"].long()
    for r, length in enumerate(lens):
        at = [j for j in range(length) if not c["window"] or j < c["sinks"]
              or j >= length - c["window"]]
        if not at:
            continue
        at = torch.tensor(at, device="cuda")
        page, slot = table[r, at // c["page"]], at % c["page"]
        k = s["k"][page, :, slot].double()           # (keys, kv_heads, dim)
        v = s["v"][page, :, slot].double()
        for j in range(c["kv_heads"]):
            q = s["q"][r, j * share:(j + 1) * share].double()
            logit = torch.einsum("gd,nd->gn", q, k[:, j]) / c["dim"] ** 0.5
            weight = torch.exp(logit - torch.logsumexp(logit, dim=1, keepdim=True))
            out[r, j * share:(j + 1) * share] = torch.einsum("gn,nd->gd", weight, v[:, j])
    return out


def _exact_append(s):
    c = s["case"]
    H, K, D, P, r = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rotary"]
    x = s["qkv"].double().view(c["rows"], H + 2 * K, D).clone()
    pos = s["pos"].long()
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None, :]
    i = torch.arange(r // 2, device="cuda")
    a, b = (i, i + r // 2) if c["pairs"] == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(x[:, :H + K, a], x[:, :H + K, b]) * turn
    x[:, :H + K, a], x[:, :H + K, b] = z.real, z.imag
    k, v = s["k"].double(), s["v"].double()
    page, slot = s["table"][s["seq"].long(), pos // P].long(), pos % P
    k[page, :, slot], v[page, :, slot] = x[:, H:H + K], x[:, H + K:]
    return {"q": x[:, :H].contiguous(), "k": k, "v": v}


def _exact_beam(s):
    c = s["case"]
    G, W, V = c["groups"], c["beams"], c["vocab"]
    best = []
    for g in range(G):
        found = []
        for b in range(W):
            base = s["scores"][g, b].double()
            if int(s["done"][g, b]):
                found.append(base[None])
                continue
            row = s["logits"][g * W + b].double()
            found.append(base + row.topk(min(W, V))[0] - torch.logsumexp(row, dim=0))
        best.append(torch.cat(found).sort(descending=True)[0][:W])
    return {"scores": torch.stack(best), "parents": None, "tokens": None, "table": None,
            "src": None, "dst": None, "fill": None}


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "attention":
        size = 2 if c["cache"] == "bf16" else 4
        keys = sum(_live(c, n) for n in _lens(c))
        row = c["heads"] * c["dim"]
        return {"bytes": 2.0 * keys * c["kv_heads"] * c["dim"] * size
                + c["rows"] * row * (4 + (2 if c["out"] == "bf16" else 4)),
                "flops": 4.0 * keys * row}
    if c["op"] == "append":
        size = 2 if c["cache"] == "bf16" else 4
        q, kv = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        return {"bytes": float(c["rows"] * (4 * (q + 2 * kv) + 4 * q + 2 * size * kv
                                            + 4 * c["rotary"] + 8)),
                "flops": 3.0 * c["rows"] * (c["heads"] + c["kv_heads"]) * c["rotary"]}
    if c["op"] == "copy":
        size = 2 if c["cache"] == "bf16" else 4
        rows = c["page"] if c["fill"] == "whole" else (c["page"] + 1) / 2
        n, m = c["copies"], _parents(c["copies"])
        # pages read: all, or as many as n draws out of m parents name
        read = n if c["fill"] == "whole" else m * (1 - (1 - 1 / m) ** n)
        page = rows * c["kv_heads"] * c["dim"] * size
        return {"bytes": 0.9 * (n + read) * page * c["planes"], "flops": 0.0}
    n = c["groups"] * c["beams"]
    return {"bytes": 4.0 * n * c["vocab"] + 8.0 * n * c["columns"] + 40.0 * n,
            "flops": 4.0 * n * c["vocab"]}
