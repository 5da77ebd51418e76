"""Timed cases of the operators of a serving loop over a paged cache: attention of chunks of new tokens whose scores are
capped, biased by distance or limited to a window, verification of drafted tokens, the rows of accepted ones moved to where they belong, and
pages reserved and given back.

A case is one call as a serving program makes it (pages: the reservation in front of a step and the return behind it).  `run` computes
it in plain torch operations, or, where `own` is true, by the package's functions.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32,
           "int8": torch.int8, "fp8": torch.float8_e4m3fn}
_BYTES = {"float16": 2, "bfloat16": 2, "float32": 4, "int8": 1, "fp8": 1}
_TOP = {"int8": 127.0, "fp8": 448.0}   # the largest code

# What a drawn case may cost at most (the largest listed ones).
_MOST_BYTES = 2.5e8
_MOST_FLOPS = 2.2e11
_MOST_SCORES = 1.3e9       # of the plain form, hidden ones too


def _attend(name, B, H, G, T, N, D, page, cache, dtype, cap=0.0, slopes=False, window=0, prefix=0, ragged=True, heads=False, lse=False):
    """T new tokens (ragged: up to T) of G query heads for each of H heads of the cache, behind N positions (ragged: up to N)."""
    return _named(name, dict(call="attend", B=B, H=H, G=G, T=T, N=N, D=D, page=page, cache=cache, dtype=dtype, cap=cap, slopes=slopes,
                             window=window, prefix=prefix, ragged=ragged, heads=heads, lse=lse))


def _verify(name, B, T, V, dtype, form):
    """T drafted tokens of V possible ones; form: "drawn" (a chain with the probabilities that it was drawn from), "chain", "tree"."""
    return _named(name, dict(call="verify", B=B, T=T, V=V, dtype=dtype, form=form))


def _accept(name, B, H, T, D, page, cache):
    return _named(name, dict(call="accept", B=B, H=H, T=T, D=D, page=page, cache=cache, N=4 * T + 100))


def _pages(name, B, N, T, page):
    """Sequences of up to N positions that reserve room for up to T more, and give most of it back."""
    return _named(name, dict(call="pages", B=B, N=N, T=T, page=page))


def _named(name, c):
    return dict(c, name=name) if name else c


def listed():
    return [
        # A few tokens behind a short context, biased by distance: all latency.
        _attend("chunk 2x17 fp16 biased", 2, 4, 2, 17, 300, 64, 16, "float16", "float16", slopes=True, lse=True),
        # A decoded token of every sequence of a batch, scores capped.
        _attend("token 48x4096 fp8 capped", 48, 8, 4, 1, 4096, 128, 16, "fp8", "bfloat16", cap=30.0),
        # Chunks of prompts next to contexts of thousands of tokens.
        _attend("chunk 4x512 int8 capped", 4, 8, 4, 512, 8192, 128, 64, "int8", "bfloat16", cap=50.0),
        # Whole prompts that begin with up to 256 tokens that see each other.
        _attend("prompt 2x4096 bf16 biased", 2, 16, 1, 4096, 0, 128, 32, "bfloat16", "bfloat16", slopes=True, prefix=256),
        # A chunk that sees the nearest thousand positions and the first few.
        _attend("window 2x2048 fp16", 2, 8, 2, 2048, 16384, 96, 16, "float16", "float16", window=1024, prefix=64),
        # One user, a short draft.
        _verify("verify 1x4 of 32000", 1, 4, 32000, "float32", "drawn"),
        # A batch of drafts from a large vocabulary.
        _verify("verify 64x7 of 131072", 64, 7, 131072, "float32", "drawn"),
        # Drafted trees, from probabilities as a model in bf16 leaves them.
        _verify("verify 16x63 tree bf16", 16, 63, 100003, "bfloat16", "tree"),
        # The accepted path of one tree, in a layer's cache.
        _accept("accept 1x16 bf16", 1, 8, 16, 128, 16, "bfloat16"),
        _accept("accept 64x63 int8", 64, 32, 63, 128, 16, "int8"),
        # A step of a batch: a page here and there.
        _pages("pages 48 steps", 48, 8192, 8, 16),
        # Prompts of thousands of tokens come and go.
        _pages("pages 256 prompts", 256, 8192, 4096, 16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["attend", "attend", "attend", "verify", "verify", "accept", "pages"])
    page = rng.choice([16, 16, 32, 64, 128])
    cache = rng.choice(["int8", "fp8", "float16", "bfloat16"])
    if call == "verify":
        form = rng.choice(["drawn", "chain", "tree"])
        c = _verify("", _log_int(rng, 1, 128), _log_int(rng, 1, 64 if form == "tree" else 16), _log_int(rng, 1000, 200000),
                    rng.choice(["float32", "float32", "float16", "bfloat16"]), form)
        while c["B"] > 1 and (c["B"] * (c["T"] + 1) * c["V"] > 1.4e8 or work(c)["bytes"] > _MOST_BYTES):
            c["B"] //= 2
        return c
    if call == "accept":
        return _accept("", _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8, 8, 16, 32]), _log_int(rng, 2, 64),
                       rng.choice([64, 80, 96, 128, 128, 192, 256]), page, cache)
    if call == "pages":
        return _pages("", _log_int(rng, 1, 400), _log_int(rng, 64, 8192), _log_int(rng, 1, 4096), page)
    dtype = cache if cache in ("float16", "bfloat16") else rng.choice(["float16", "bfloat16"])
    T = 1 if rng.random() < 0.25 else _log_int(rng, 2, 4096)
    c = _attend("", _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8, 8, 16, 32]), rng.choice([1, 2, 3, 4, 4, 8]), T,
                0 if T > 64 and rng.random() < 0.3 else _log_int(rng, 16, 32768), rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256]), page,
                cache, dtype, cap=rng.choice([0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, window=0 if rng.random() < 0.6 else _log_int(rng, 16, 4096),
                prefix=0 if rng.random() < 0.7 else _log_int(rng, 1, 512), ragged=rng.random() < 0.7, heads=rng.random() < 0.15,
                lse=rng.random() < 0.3)
    while True:
        w, n = work(c), c["N"] + c["T"]
        if w["bytes"] <= _MOST_BYTES and w["flops"] <= _MOST_FLOPS and c["B"] * c["H"] * c["G"] * c["T"] * n <= _MOST_SCORES and \
                c["B"] * c["H"] * n * c["D"] <= 1 << 28:
            return c
        if c["B"] > 1:
            c["B"] //= 2
        elif c["H"] > 8:
            c["H"] = 8
        elif c["N"] > c["T"]:
            c["N"] //= 2
        else:
            c["T"] //= 2


def _codes(rows, cache):
    """Codes and scales of rows: the largest element of a row is the largest code."""
    a = rows.abs().amax(-1)
    c = rows * _TOP[cache] / a.clamp_min(1e-30)[..., None]
    return (c.round().to(torch.int8) if cache == "int8" else c.to(torch.float8_e4m3fn)), a / _TOP[cache]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"attend": _prepare_cache, "accept": _prepare_cache, "verify": _prepare_verify, "pages": _prepare_pages}[c["call"]](c, g)


def _tree(B, T, g):
    """Every drafted token continues an earlier one, or the context (-1); the later ones as a rule."""
    before = torch.arange(T, device="cuda")
    back = (torch.rand((B, T), generator=g, device="cuda") ** 2 * (before + 1)).long().clamp_max(4)
    return (before - 1 - back).clamp_min(-1).int()


def _prepare_cache(c, g):
    B, H, N, D, T, ps = c["B"], c["H"], c["N"], c["D"], c["T"], c["page"]
    per = -(-(N + T) // ps)
    pages = B * per + 3
    # pages in the order in which a pool that has been in use for a while hands them out
    state = {"case": c, "table": torch.randperm(pages, generator=g, device="cuda")[: B * per].view(B, per).int()}
    for name, far in (("k", 8.0), ("v", 1.0)):
        rows = torch.randn((pages, H, ps, D), generator=g, device="cuda", dtype=_DTYPES[c.get("dtype", "bfloat16")])
        rows[..., : D // 32] *= far      # keys have channels far above the others
        if c["cache"] in _TOP:
            state[name], state[name + "_scale"] = _codes(rows.float(), c["cache"])
        else:
            state[name], state[name + "_scale"] = rows.to(_DTYPES[c["cache"]]), None

    def some(least, most, shape):
        return torch.randint(least, most + 1, shape, generator=g, device="cuda", dtype=torch.int32)

    if c["call"] == "accept":
        state["context"] = some(0, N, (B,))
        parents = _tree(B, T, g)
        # the path of the last token, cut where the first token was rejected
        node, on = torch.full((B,), T - 1, device="cuda"), torch.zeros((B, T + 1), device="cuda", dtype=torch.bool)
        for _ in range(T):
            on.scatter_(1, torch.where(node < 0, T, node)[:, None], True)
            node = torch.where(node < 0, -1, parents.long().gather(1, node.clamp_min(0)[:, None])[:, 0])
        on = on[:, :T]
        state["accepted"] = (on.sum(1) * torch.rand(B, generator=g, device="cuda") + 0.5).int()
        first = (~on).to(torch.uint8).argsort(dim=1, stable=True).int()
        state["path"] = torch.where(torch.arange(T, device="cuda") < state["accepted"][:, None], first, -1)
        return state
    shape = (B, H) if c["heads"] else (B,)
    state["context"] = some(N // 2, N, shape) if c["ragged"] else torch.full(shape, N, device="cuda", dtype=torch.int32)
    state["counts"] = some((T + 1) // 2, T, (B,)) if c["ragged"] and T > 1 else None
    state["prefix"] = some(0, c["prefix"], (B,)) if c["prefix"] else None
    heads = H * c["G"]
    state["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if c["slopes"] else None
    # token-major memory seen as heads, as projections leave it
    state["query"] = torch.randn((B, T, heads, D), generator=g, device="cuda", dtype=_DTYPES[c["dtype"]]).transpose(1, 2)
    return state


def _prepare_verify(c, g):
    B, T, V, dtype = c["B"], c["T"], c["V"], _DTYPES[c["dtype"]]
    logits = 3.0 * torch.randn((B, T + 1, V), generator=g, device="cuda")
    state = {"case": c, "draft": None, "parents": None}
    state["target"] = logits.softmax(-1).to(dtype)
    if c["form"] == "tree":
        state["parents"] = _tree(B, T, g)
        rows = (state["parents"].long() + 1)[..., None]
    else:
        rows = torch.arange(T, device="cuda")[None, :, None].expand(B, T, 1)
    # a draft that is right more often than not; trees and chains of likely tokens are drawn at a lower temperature
    near = logits.gather(1, rows.expand(B, T, V))
    near = near + torch.randn((B, T, V), generator=g, device="cuda") if c["form"] == "drawn" else 1.5 * near
    near = near.softmax(-1)
    if c["form"] == "drawn":
        near = near.to(dtype)
        state["draft"] = near
    state["tokens"] = torch.multinomial(near.float().view(B * T, V), 1, generator=g).view(B, T)
    state["uniform"] = torch.rand((B, T), generator=g, device="cuda")
    state["sample"] = torch.rand((B,), generator=g, device="cuda")
    return state


def _prepare_pages(c, g):
    B, N, T, ps = c["B"], c["N"], c["T"], c["page"]
    per = -(-(N + T) // ps)
    pages = B * (-(-N // ps) + -(-T // (2 * ps))) + 1       # now and then too few for all
    lengths = torch.randint(N // 2, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    if T > 64:       # requests that begin hold nothing yet
        lengths = torch.where(torch.rand((B,), generator=g, device="cuda") < 0.5, 0, lengths)
    held = (lengths + ps - 1) // ps
    order = torch.randperm(pages, generator=g, device="cuda").int()
    i = torch.arange(per, device="cuda")
    first = held.cumsum(0) - held
    mine = i < held[:, None]
    table = torch.where(mine, order[(first[:, None] + i).clamp_max(pages - 1)], -1).int()
    used = held.sum()
    free = torch.cat((order, order))[(used + torch.arange(pages, device="cuda")) % pages]
    return {"case": c, "table": table, "held": held.int(), "free": free.contiguous(), "available": (pages - used).int().view(1),
            "wanted": lengths + torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32), "kept": lengths}


def _gather(pages, table):
    """(B, H, positions, ...) of the pages that the table names."""
    x = pages.view(torch.int8)[table.long()].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[table.long()]
    x = x.transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def _values(pages, scale, table):
    x = _gather(pages, table).float()
    return x if scale is None else x * _gather(scale, table)[..., None]


def _seen(position, live, n, window, prefix):
    """Which of n positions tokens see, the positions of the tokens (..., T, 1), those that are there (..., 1, n)."""
    j = torch.arange(n, device=position.device)
    seen = j <= position
    if window:
        seen = seen & (j > position - window)
    if prefix is not None:
        seen = seen | (j < prefix)
    return seen & live


def _plain_attend(s):
    c = s["case"]
    B, H, G, T, D = c["B"], c["H"], c["G"], c["T"], c["D"]
    k, v = _values(s["k"], s["k_scale"], s["table"]), _values(s["v"], s["v_scale"], s["table"])
    n = k.shape[2]
    context = s["context"].view(B, -1, 1, 1)                                    # (B, H or 1, 1, 1)
    t = torch.arange(T, device="cuda")[:, None]
    count = T if s["counts"] is None else s["counts"].view(B, 1, 1, 1)
    j = torch.arange(n, device="cuda")
    seen = _seen(context + t, (j < context + count) & (t < count), n, c["window"], None if s["prefix"] is None else s["prefix"].view(B, 1, 1, 1))
    scores = (s["query"].float().reshape(B, H, G * T, D) @ k.transpose(-1, -2)).view(B, H, G, T, n) * D ** -0.5
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(H, G, 1, 1) * (context + t - j).abs()[:, :, None]
    scores = scores.masked_fill(~seen[:, :, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = (scores - m.clamp_min(-3e38)).exp()
    total = p.sum(-1, keepdim=True)
    out = (p / total.clamp_min(1e-30)).view(B, H, G * T, n) @ v
    out = out.view(B, H * G, T, D).to(_DTYPES[c["dtype"]])
    return (out, ((m + total.log()) * (1 / math.log(2))).view(B, H * G, T)) if c["lse"] else out


def _plain_verify(s):
    target, tokens, draft = s["target"], s["tokens"], s["draft"]
    B, T = tokens.shape
    V = target.shape[2]
    i = torch.arange(T, device="cuda")
    parents = (i - 1).expand(B, T) if s["parents"] is None else s["parents"].long()
    at = target.view(B, -1).gather(1, (parents + 1) * V + tokens).double()      # of every token, in the row that it continues
    u = s["uniform"].double().gather(1, parents + 1)
    if draft is not None:
        taken = u * draft.gather(2, tokens[..., None])[..., 0].double() < at
    else:
        # siblings in front of a token; a token that one of them has already has nothing left
        before = (parents[:, :, None] == parents[:, None, :]) & (i[None, :] < i[:, None])
        again = (before & (tokens[:, :, None] == tokens[:, None, :])).any(2)
        at = torch.where(again, 0.0, at)
        low = (before * at[:, None, :]).sum(2)
        taken = (low <= u) & (u < low + at)
    up = parents
    for _ in range(max(1, T.bit_length())):                                     # a token counts if all before it on its path do
        taken = taken & torch.where(up < 0, True, taken.gather(1, up.clamp_min(0)))
        up = torch.where(up < 0, -1, up.gather(1, up.clamp_min(0)))
    accepted = taken.sum(1, dtype=torch.int32)
    path = torch.where(taken, i, T).sort(1).values
    row = torch.where(taken, i + 1, 0).amax(1)                                  # where the path ends
    p = target.gather(1, row[:, None, None].expand(B, 1, V))[:, 0].double()
    if draft is not None:
        q = draft.gather(1, row.clamp_max(T - 1)[:, None, None].expand(B, 1, V))[:, 0].double()
        rest = torch.where((row < T)[:, None], (p - q).clamp_min(0), p)
    else:
        tried = torch.where(parents + 1 == row[:, None], tokens, V)
        hidden = torch.zeros((B, V + 1), device="cuda", dtype=torch.bool).scatter_(1, tried, True)[:, :V]
        rest = torch.where(hidden, 0.0, p)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    upto = rest.cumsum(1)
    token = (upto > s["sample"].double()[:, None] * upto[:, -1:]).to(torch.uint8).argmax(1)
    return accepted, torch.where(path < T, path, -1).int(), token


def _plain_accept(s):
    c, ps = s["case"], s["case"]["page"]
    T, H = c["T"], c["H"]
    i = torch.arange(T, device="cuda")
    live = i < s["accepted"][:, None]
    to = s["context"].long()[:, None] + i
    at = torch.where(live, s["context"].long()[:, None] + s["path"], to)
    head = torch.arange(H, device="cuda")
    to_page, at_page = (s["table"].long().gather(1, x // ps)[..., None] for x in (to, at))
    to_row, at_row = (to % ps)[..., None], (at % ps)[..., None]
    out = {}
    for name in ("k", "v", "k_scale", "v_scale"):
        if s[name] is not None:
            x = s[name].view(torch.int8) if c["cache"] == "fp8" and name in ("k", "v") else s[name]
            x[to_page, head, to_row] = x[at_page, head, at_row]
            out[name] = s[name]
    return dict(out, context=s["context"] + s["accepted"])


def _plain_reserve(table, held, free, available, lengths, ps):
    """Pages of sequences that need fewer go back on the stack, in their order, then those that need more take theirs from its top, in their order."""
    need = (lengths + ps - 1) // ps
    i = torch.arange(table.shape[1], device="cuda")
    less = (held - need).clamp_min(0)
    back = (i >= need[:, None]) & (i < held[:, None])
    start = less.cumsum(0) - less
    slot = available + start[:, None] + i - need[:, None]
    pages = free.shape[0]
    room = torch.cat((free, free.new_zeros(1)))
    room[torch.where(back, slot, pages)] = table
    free.copy_(room[:pages])
    table.copy_(torch.where(back, -1, table))
    there = available + less.sum()
    more = (need - held).clamp_min(0)
    upto = more.cumsum(0)
    granted = (upto <= there) | (more == 0)
    more = torch.where(granted, more, 0)
    new = (i >= held[:, None]) & (i < (held + more)[:, None])
    slot = there - 1 - ((more.cumsum(0) - more)[:, None] + i - held[:, None])
    table.copy_(torch.where(new, free[slot.clamp(0, pages - 1)], table))
    held.copy_(torch.where(granted, need, held))
    available.copy_(there - more.sum())
    return granted


def _plain_pages(s):
    pool = (s["table"], s["held"], s["free"], s["available"])
    return [_plain_reserve(*pool, s["wanted"], s["case"]["page"]), _plain_reserve(*pool, s["kept"], s["case"]["page"]), *pool]


_PLAIN = {"attend": _plain_attend, "verify": _plain_verify, "accept": _plain_accept, "pages": _plain_pages}


def _own(s):
    """The call that a user of the package makes."""
    import flash_colreduce_amd as fca
    c = s["case"]
    if c["call"] == "verify":
        return list(fca.verify_drafts(s["target"], s["tokens"], s["uniform"], s["sample"], draft=s["draft"], parents=s["parents"]))
    if c["call"] == "pages":
        pool = fca.PagePool(s["free"], s["available"], s["held"])
        return [fca.cache_reserve(pool, s["table"], s["wanted"], c["page"]), fca.cache_reserve(pool, s["table"], s["kept"], c["page"]),
                s["table"], s["held"], s["free"], s["available"]]
    cache = fca.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if c["call"] == "accept":
        context = fca.cache_accept(cache, s["table"], s["context"], s["path"], s["accepted"])
        return dict({x: s[x] for x in ("k", "v", "k_scale", "v_scale") if s[x] is not None}, context=context)
    return fca.chunk_attention(s["query"], cache, s["table"], s["context"], counts=s["counts"], cap=c["cap"] or None, slopes=s["slopes"],
                               window=c["window"] or None, prefix=s["prefix"], return_lse2=c["lse"])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["call"]](state)


def work(case):
    """Every row once, codes and scales, and the products of the scores that are seen; ragged lengths are three quarters of the longest on average."""
    c = case
    if c["call"] == "verify":
        # the row where a draft ends, in which the next token is found
        return {"bytes": int(c["B"] * c["V"] * _BYTES[c["dtype"]] * (2 if c["form"] == "drawn" else 1)), "flops": 0}
    if c["call"] == "pages":
        # pages that come and go, in the table and on the stack
        moved = c["B"] * (c["T"] / 2) / c["page"]
        return {"bytes": int(4 * (4 * moved + 8 * c["B"])), "flops": 0}
    row = c["D"] * _BYTES[c["cache"]] + (4 if c["cache"] in _TOP else 0)
    if c["call"] == "accept":
        # (about an eighth of a tree's tokens)
        return {"bytes": int(4 * c["B"] * c["H"] * row * (c["T"] / 8 + 0.5)), "flops": 0}
    part = 0.75 if c["ragged"] else 1.0
    n, t, e = c["N"] * part, c["T"] * (part if c["T"] > 1 else 1.0), c["D"] * _BYTES[c["dtype"]]
    pairs, rows = t * (n + t / 2), n + t
    if c["window"]:
        pairs, rows = min(pairs, t * (c["window"] + c["prefix"] / 2)), min(rows, t + c["window"] + c["prefix"] / 2)
    heads = c["B"] * c["H"]
    return {"bytes": int(2 * heads * (rows * row + c["G"] * t * e)), "flops": int(4 * heads * c["G"] * pairs * c["D"])}


def _exact_rows(s, name, b, h, n):
    """The first n rows of one head, in 64 bits."""
    ids = s["table"][b, : -(-n // s["case"]["page"])].long()
    x = s[name][:, h].view(torch.uint8)[ids].view(s[name].dtype) if s["case"]["cache"] == "fp8" else s[name][:, h][ids]
    x = x.flatten(0, 1)[:n].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][:, h][ids].flatten()[:n, None].double()
    return x


def exact(case, seed):
    """The definition in 64 bits, one head at a time.  (What the other operators give are whole numbers and copies.)"""
    if case["call"] != "attend" or case["B"] * case["H"] > 512:
        return None
    s = prepare(case, seed)
    c = s["case"]
    B, H, T, G, D = (c[x] for x in ("B", "H", "T", "G", "D"))
    out = torch.zeros((B, H, G, T, D), device="cuda", dtype=torch.float64)
    lse = torch.full((B, H, G, T), -math.inf, device="cuda", dtype=torch.float64)
    for b in range(B):
        count = T if s["counts"] is None else int(s["counts"][b])
        first = 0 if s["prefix"] is None else int(s["prefix"][b])
        for h in range(H):
            context = int(s["context"][b, h] if c["heads"] else s["context"][b])
            n = context + count
            k, v = _exact_rows(s, "k", b, h, n), _exact_rows(s, "v", b, h, n)
            distance = torch.arange(context, n, device="cuda")[:, None] - torch.arange(n, device="cuda")
            hidden = distance < 0
            if c["window"]:
                hidden |= distance >= c["window"]
            hidden[:, :first] = False
            w = torch.matmul(s["query"][b, h * G:(h + 1) * G, :count].double(), k.t().contiguous()) / math.sqrt(D)
            if c["cap"]:
                w = torch.tanh(w / c["cap"]) * c["cap"]
            if s["slopes"] is not None:
                w -= s["slopes"][h * G:(h + 1) * G, None, None].double() * distance.abs()
            w[:, hidden] = -math.inf
            lse[b, h, :, :count] = torch.logsumexp(w, -1) / math.log(2)
            out[b, h, :, :count] = torch.matmul(torch.softmax(w, -1), v)
    out = out.view(B, H * G, T, D)
    return (out, lse.view(B, H * G, T)) if c["lse"] else out
