"""Timed cases of the operators around a paged cache of keys and values: writing it (quantised or not), reading it
back, keeping the rows that a keep-mask names, and attention of drafted tokens over it.

A case is one call as a serving program makes it.  `run` computes it in plain torch operations, or, where `own` is
true, by the package's functions.
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
_MOST_BYTES = 1.2e9
_MOST_FLOPS = 3e11


def _case(name, call, B, H, N, D, page, cache, dtype, G=1, T=1, ragged=False, mask="chain", keep=0.0, heads=False, lse=False):
    """B sequences, H heads of the cache of D elements, N positions per sequence at most, pages of `page` rows; `dtype`: the
    type of the tensors outside the cache.  T tokens are written, or drafted with G query heads for each head of the cache."""
    c = dict(call=call, B=B, H=H, N=N, D=D, page=page, cache=cache, dtype=dtype, G=G, T=T, ragged=ragged, mask=mask, keep=keep,
             heads=heads, lse=lse)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # A decoded token of each of 64 sequences goes into the cache: all latency.
        _case("write 64x1 int8", "write", 64, 8, 4096, 128, 16, "int8", "bfloat16", ragged=True),
        # A prompt of 8192 tokens goes into the cache.
        _case("write 8192 fp8", "write", 1, 32, 8192, 128, 64, "fp8", "float16", T=8192),
        # A batch of prompts of ragged lengths, projections viewed as heads.
        _case("write 8x2929 int8", "write", 8, 24, 2929, 128, 16, "int8", "bfloat16", T=2929, ragged=True),
        # The cache of one prompt is read back for the column reduction.
        _case("read 4096 int8", "read", 1, 8, 4096, 128, 16, "int8", "float16"),
        # A batch of ragged caches is read back.
        _case("read 8x9001 fp8", "read", 8, 32, 9001, 128, 64, "fp8", "bfloat16", ragged=True),
        # Pruning: a quarter of a prompt's keys stays, each head its own.
        _case("keep 8192 int8", "keep", 1, 8, 8192, 128, 16, "int8", "float16", keep=0.25),
        # The same for a batch of long caches of 16-bit rows.
        _case("keep 4x32768 bf16", "keep", 4, 8, 32768, 128, 64, "bfloat16", "bfloat16", keep=0.5, ragged=True),
        # One token of one sequence over a short cache: all latency.
        _case("token 1x1000 int8", "attend", 1, 8, 1000, 128, 16, "int8", "bfloat16", G=4),
        # One token of each sequence of a ragged batch over long caches: reading the cache is the work.
        _case("token 32x16384 fp8", "attend", 32, 8, 16384, 128, 16, "fp8", "bfloat16", G=4, ragged=True),
        # A short chain of drafted tokens over an unquantised cache of plain heads.
        _case("chain 4x8x9001 fp16", "attend", 4, 32, 9001, 64, 64, "float16", "float16", T=8, ragged=True, lse=True),
        # A tree of 64 drafted tokens over pruned caches, whose heads differ in length.
        _case("tree 4x64x8192 int8", "attend", 4, 8, 8192, 128, 16, "int8", "float16", G=4, T=64, ragged=True, mask="tree", heads=True),
        # The largest: trees over a batch of long caches.
        _case("tree 8x64x32768 int8", "attend", 8, 8, 32768, 128, 64, "int8", "bfloat16", G=4, T=64, ragged=True, mask="tree"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["write", "read", "keep", "attend", "attend", "attend"])
    cache = rng.choice(["int8", "int8", "fp8", "fp8", "float16", "bfloat16"])
    dtype = cache if cache in ("float16", "bfloat16") else rng.choice(["float16", "bfloat16"])
    c = _case("", call, _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8, 8, 16, 32]), _log_int(rng, 128, 65536),
              rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256]), rng.choice([16, 16, 32, 64, 128]), cache, dtype,
              ragged=rng.random() < 0.7, heads=rng.random() < 0.2)
    if call == "write":
        c["T"] = 1 if rng.random() < 0.4 else _log_int(rng, 2, c["N"])
    elif call == "keep":
        c["keep"] = rng.choice([0.1, 0.25, 0.5])
    elif call == "attend":
        c["G"] = rng.choice([1, 2, 3, 4, 4, 8])
        c["T"] = 1 if rng.random() < 0.4 else _log_int(rng, 2, 64)
        c["mask"] = rng.choice(["chain", "tree"])
        c["lse"] = rng.random() < 0.3
    while True:
        w = work(c)
        if w["bytes"] <= _MOST_BYTES and w["flops"] <= _MOST_FLOPS and c["B"] * c["H"] * c["N"] * c["D"] <= 1 << 29:
            return c
        if c["B"] > 1:
            c["B"] //= 2
        elif c["H"] > 8:
            c["H"] = 8
        else:
            c["N"] //= 2
            c["T"] = min(c["T"], c["N"])


def _spread(x, cache):
    """Codes and scales of rows: the largest element of a row is the largest code."""
    top = _TOP[cache]
    a = x.abs().amax(-1)
    c = x * top / a.clamp_min(1e-30)[..., None]     # a product without a rounding, for 16-bit x: ties stay ties
    return (c.round().to(torch.int8) if cache == "int8" else c.to(torch.float8_e4m3fn)), a / top


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    B, H, N, D, T, ps = c["B"], c["H"], c["N"], c["D"], c["T"], c["page"]
    dtype = _DTYPES[c["dtype"]]
    drafted = T if c["call"] == "attend" else 0
    per = -(-(N + drafted) // ps)
    pages = B * per + 3

    # pages in the order in which a pool that has been in use for a while hands them out
    state = {"case": c, "table": torch.randperm(pages, generator=g, device="cuda")[: B * per].view(B, per).int()}
    for name, far in (("k", 8.0), ("v", 1.0)):
        rows = torch.randn((pages, H, ps, D), generator=g, device="cuda", dtype=dtype)
        rows[..., : D // 32] *= far      # keys have channels far above the others
        if c["cache"] in _TOP:
            state[name], state[name + "_scale"] = _spread(rows.float(), c["cache"])
        else:
            state[name], state[name + "_scale"] = rows, None
    shape = (B, H) if c["heads"] else (B,)
    most = N - T if c["call"] == "write" else N
    some = torch.randint(most // 2, most + 1, shape, generator=g, device="cuda", dtype=torch.int32)
    lengths = some if c["ragged"] else torch.full_like(some, most)
    state["lengths"] = lengths
    if c["call"] == "write":
        # token-major memory seen as heads, as projections leave it
        for name in ("key", "value"):
            state[name] = torch.randn((B, T, H, D), generator=g, device="cuda", dtype=dtype).transpose(1, 2)
        state["counts"] = None
        if c["ragged"] and T > 1:
            state["counts"] = torch.randint(T // 2, T + 1, shape, generator=g, device="cuda", dtype=torch.int32)
    elif c["call"] == "keep":
        # the columns of largest score stay, as many for each head
        scores = torch.randn((B, H, N), generator=g, device="cuda")
        kept = max(1, int(c["keep"] * N))
        state["keep"] = scores >= scores.topk(kept, dim=-1).values[..., -1:]
        into = -(-kept // ps)
        state["into_table"] = torch.randperm(B * into, generator=g, device="cuda").view(B, into).int()
        for name in ("k", "v"):
            state["into_" + name] = torch.zeros((B * into, H, ps, D), device="cuda", dtype=state[name].dtype)
            scale = state[name + "_scale"]
            state["into_" + name + "_scale"] = None if scale is None else torch.zeros((B * into, H, ps), device="cuda")
    elif c["call"] == "attend":
        state["query"] = torch.randn((B, T, H * c["G"], D), generator=g, device="cuda", dtype=dtype).transpose(1, 2)
        state["mask"] = None
        if c["mask"] == "tree":
            # every drafted token continues an earlier one, or the context
            before = torch.arange(T, device="cuda")
            parent = (torch.rand((B, T), generator=g, device="cuda") * (before + 1)).long() - 1
            seen = torch.eye(T, device="cuda", dtype=torch.bool).repeat(B, 1, 1)
            for t in range(1, T):
                of = parent[:, t].clamp_min(0)
                up = seen[torch.arange(B, device="cuda"), of] & (parent[:, t] >= 0)[:, None]
                seen[:, t] |= up
            state["mask"] = seen
    return state


def _cache(s, name=""):
    """Keys, values and their scales, in the order in which the package's cache holds them."""
    return [s[name + x] for x in ("k", "v", "k_scale", "v_scale")]


def _rows_of(lengths, H):
    return lengths[:, None].expand(-1, H) if lengths.dim() == 1 else lengths


def _gather(pages, table):
    """(B, H, positions, ...) of the pages that the table names."""
    x = pages.view(torch.int8)[table.long()].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[table.long()]
    x = x.transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def _values(pages, scale, table):
    x = _gather(pages, table).float()
    return x if scale is None else x * _gather(scale, table)[..., None]


def _write(s):
    c, ps = s["case"], s["case"]["page"]
    B, H, T = c["B"], c["H"], c["T"]
    t = torch.arange(T, device="cuda")
    at = _rows_of(s["lengths"], H)[..., None].long() + t              # (B, H, T)
    page = s["table"].long().gather(1, (at // ps).reshape(B, -1)).view(B, H, T)
    head = torch.arange(H, device="cuda")[None, :, None]
    row = at % ps
    new = None if s["counts"] is None else t < _rows_of(s["counts"], H)[..., None]
    for to, scale, x in ((s["k"], s["k_scale"], s["key"]), (s["v"], s["v_scale"], s["value"])):
        if scale is None:
            code, factor = x.to(to.dtype), None
        else:
            code, factor = _spread(x.float(), c["cache"])
        if to.dtype == torch.float8_e4m3fn:
            to, code = to.view(torch.int8), code.view(torch.int8)
        if new is not None:
            code = torch.where(new[..., None], code, to[page, head, row])
            factor = None if factor is None else torch.where(new, factor, scale[page, head, row])
        to[page, head, row] = code
        if scale is not None:
            scale[page, head, row] = factor
    return _written(s)


def _written(s, name=""):
    return {x: y for x, y in zip(("k", "v", "k_scale", "v_scale"), _cache(s, name)) if y is not None}


def _read(s):
    c = s["case"]
    N, dtype = c["N"], _DTYPES[c["dtype"]]
    live = torch.arange(N, device="cuda") < _rows_of(s["lengths"], c["H"])[..., None]
    out = []
    for pages, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        x = _values(pages, scale, s["table"])[:, :, :N]
        out.append(torch.where(live[..., None], x, 0.0).to(dtype))
    return out


def _keep(s):
    c, ps = s["case"], s["case"]["page"]
    B, H, N = c["B"], c["H"], c["N"]
    room = s["into_table"].shape[1] * ps
    kept = s["keep"] & (torch.arange(N, device="cuda") < _rows_of(s["lengths"], H)[..., None])
    counts = kept.sum(-1, dtype=torch.int32)
    first = (~kept).to(torch.uint8).argsort(dim=-1, stable=True)[..., :room]      # kept rows first, in their order
    r = torch.arange(first.shape[-1], device="cuda")
    live = r < counts[..., None]
    page = s["into_table"].long()[:, r // ps][:, None, :].expand(B, H, -1)
    head = torch.arange(H, device="cuda")[None, :, None]
    row = (r % ps).expand(B, H, -1)
    source = s["table"].long().gather(1, (first // ps).reshape(B, -1)).view(first.shape)
    for x, to in zip(_cache(s), _cache(s, "into_")):
        if x is None:
            continue
        if x.dtype == torch.float8_e4m3fn:
            x, to = x.view(torch.int8), to.view(torch.int8)
        some = live if x.dim() == 3 else live[..., None]
        to[page, head, row] = torch.where(some, x[source, head, first % ps], to[page, head, row])
    return dict(_written(s, "into_"), counts=counts)


def _attend(s):
    c = s["case"]
    B, H, G, T, D = c["B"], c["H"], c["G"], c["T"], c["D"]
    k, v = _values(s["k"], s["k_scale"], s["table"]), _values(s["v"], s["v_scale"], s["table"])
    scores = s["query"].float().reshape(B, H, G * T, D) @ k.transpose(-1, -2)
    scores = (scores * D ** -0.5).view(B, H, G, T, -1)
    n = scores.shape[-1]
    u = torch.arange(n, device="cuda") - _rows_of(s["lengths"], H)[..., None]      # (B, H, n): which drafted token, < 0: the context
    drafted = (u >= 0) & (u < T)
    if s["mask"] is None:
        seen = u[:, :, None] <= torch.arange(T, device="cuda")[:, None]
    else:
        seen = s["mask"][:, None].expand(B, H, T, T).gather(-1, u.clamp(0, T - 1)[:, :, None].expand(B, H, T, n))
        seen = (u < 0)[:, :, None] | (seen & drafted[:, :, None])
    scores = scores.masked_fill(~seen[:, :, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = (scores - m).exp()
    total = p.sum(-1, keepdim=True)
    out = ((p / total).view(B, H, G * T, n) @ v).view(B, H * G, T, D).to(_DTYPES[c["dtype"]])
    if not c["lse"]:
        return out
    return out, ((m + total.log()) * (1 / math.log(2))).view(B, H * G, T)


_PLAIN = {"write": _write, "read": _read, "keep": _keep, "attend": _attend}


def _own(s):
    """The call that a user of the package makes."""
    import flash_colreduce_amd as fca
    c = s["case"]
    cache = fca.KVCache(*_cache(s))
    if c["call"] == "write":
        fca.cache_write(cache, s["key"], s["value"], s["table"], s["lengths"], s["counts"])
        return _written(s)
    if c["call"] == "read":
        return list(fca.cache_read(cache, s["table"], s["lengths"], c["N"], out_dtype=_DTYPES[c["dtype"]]))
    if c["call"] == "keep":
        counts = fca.cache_keep(cache, s["table"], s["lengths"], s["keep"], fca.KVCache(*_cache(s, "into_")), s["into_table"])
        return dict(_written(s, "into_"), counts=counts)
    return fca.tree_attention(s["query"], cache, s["table"], s["lengths"], s["mask"], return_lse2=c["lse"])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["call"]](state)


def work(case):
    """Every row once, codes and scales; ragged lengths are three quarters of the longest on average."""
    c = case
    row = c["D"] * _BYTES[c["cache"]] + (4 if c["cache"] in _TOP else 0)
    e = c["D"] * _BYTES[c["dtype"]]
    n = c["N"] * (0.75 if c["ragged"] else 1.0)
    heads = c["B"] * c["H"]
    if c["call"] == "write":
        rows = 2 * heads * c["T"] * (0.75 if c["ragged"] and c["T"] > 1 else 1.0)
        return {"bytes": int(rows * (e + row)), "flops": 0}
    if c["call"] == "read":
        return {"bytes": int(2 * heads * (n * row + c["N"] * e)), "flops": 0}
    if c["call"] == "keep":
        return {"bytes": int(heads * (n + 4 * n * c["keep"] * row)), "flops": 0}
    seen = n + c["T"]
    return {"bytes": int(2 * heads * (seen * row + c["G"] * c["T"] * e)),
            "flops": int(4 * heads * c["G"] * c["T"] * seen * c["D"])}


def _exact_rows(s, name, b, h, n):
    """The first n rows of one head, in 64 bits."""
    ps = s["case"]["page"]
    ids = s["table"][b, : -(-n // ps)].long()
    x = s[name][:, h].view(torch.uint8)[ids].view(s[name].dtype) if s["case"]["cache"] == "fp8" else s[name][:, h][ids]
    x = x.flatten(0, 1)[:n].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][:, h][ids].flatten()[:n, None].double()
    return x


def exact(case, seed):
    """The operators' definition in 64 bits, one head at a time."""
    s = prepare(case, seed)
    c = s["case"]
    B, H, N, D, T, G, ps = (c[x] for x in ("B", "H", "N", "D", "T", "G", "page"))
    lengths = [[int(x) for x in (r if isinstance(r, list) else [r] * H)] for r in s["lengths"].tolist()]
    table = s["table"].tolist()
    if c["call"] == "keep":
        return None       # copies
    if c["call"] == "write":
        if B * H > 512 and T == 1 or B * T * H > 1 << 21:
            return None
        got = {x: y.double() if y is not None and y.dtype != torch.int8 else y for x, y in zip(("k", "v", "k_scale", "v_scale"), _cache(s))}
        counts = [[T] * H] * B if s["counts"] is None else [r if isinstance(r, list) else [r] * H for r in s["counts"].tolist()]
        for b in range(B):
            for h in range(H):
                n = counts[b][h]
                at = torch.arange(lengths[b][h], lengths[b][h] + n, device="cuda")
                where = (s["table"][b].long()[at // ps], torch.full_like(at, h), at % ps)
                for name, x in (("k", s["key"]), ("v", s["value"])):
                    x = x[b, h, :n].double()
                    if c["cache"] in _TOP:
                        most = x.abs().max(dim=-1).values
                        got[name + "_scale"][where] = most / _TOP[c["cache"]]
                        x = x * _TOP[c["cache"]] / most[:, None]
                        if c["cache"] == "int8":
                            x = x.round().to(torch.int8)
                        else:      # three bits behind the leading one, steps of 2^-9 at least
                            step = torch.exp2(x.abs().clamp_min(1e-30).log2().floor().clamp_min(-6) - 3)
                            x = (x / step).round() * step
                    elif c["cache"] != c["dtype"]:
                        x = x.to(_DTYPES[c["cache"]]).double()
                    got[name][where] = x
        return {x: y for x, y in got.items() if y is not None and y.dtype != torch.int8}
    if c["call"] == "read":
        if B * H > 1024:
            return None
        out = [torch.zeros((B, H, N, D), device="cuda", dtype=torch.float64) for _ in range(2)]
        for b in range(B):
            for h in range(H):
                n = lengths[b][h]
                for x, name in zip(out, ("k", "v")):
                    x[b, h, :n] = _exact_rows(s, name, b, h, n)
        return out
    if B * H > 1024:
        return None
    out = torch.zeros((B, H, G, T, D), device="cuda", dtype=torch.float64)
    lse = torch.zeros((B, H, G, T), device="cuda", dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            n = lengths[b][h]
            k, v = _exact_rows(s, "k", b, h, n + T), _exact_rows(s, "v", b, h, n + T)
            q = s["query"][b, h * G:(h + 1) * G].double()
            w = torch.matmul(q, k.t().contiguous()) / math.sqrt(D)
            hidden = torch.zeros((T, n + T), device="cuda", dtype=torch.bool)
            hidden[:, n:] = ~s["mask"][b] if s["mask"] is not None else torch.ones((T, T), device="cuda", dtype=torch.bool).triu(1)
            w[:, hidden] = -math.inf
            lse[b, h] = torch.logsumexp(w, -1) / math.log(2)
            out[b, h] = torch.matmul(torch.softmax(w, -1), v)
    out = out.view(B, H * G, T, D)
    return (out, lse.view(B, H * G, T)) if c["lse"] else out
