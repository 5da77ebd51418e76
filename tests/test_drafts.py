"""verify_drafts, cache_accept and cache_reserve against plain forms that take one sequence after the other, and their refusals."""
import ctypes
import math
import random

import numpy as np
import pytest
import torch

import flash_colreduce_amd as fca
from flash_colreduce_amd import KVCache, PagePool, _lib
from flash_colreduce_amd import cache as cache_module
from tests.test_cache import _c_cache

F16, BF16, F32, I8, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn


# Plain forms -------------------------------------------------------------------------------------------------------------

def weights(x):
    x = x.double().numpy()
    return np.where(x > 0, x, 0.0)      # (a NaN too)


def drawn(r, sample):
    """The first token at which the running sum exceeds sample of the whole; -1 without a weight, or with an infinite one."""
    if not (0 < r.sum() < math.inf):
        return -1
    upto = np.cumsum(r)
    at = np.flatnonzero((upto > float(sample) * upto[-1]) & (r > 0))
    return int(at[0]) if len(at) else int(np.flatnonzero(r > 0)[-1])


def verified(target, tokens, uniform, sample, draft=None, parents=None, counts=None):
    B, T = tokens.shape
    V = target.shape[2]
    accepted, path, token = [], [], []
    for b in range(B):
        count = T if counts is None else min(max(int(counts[b]), 0), T)
        up = list(range(-1, T - 1)) if parents is None else (parents if parents.dim() == 1 else parents[b]).tolist()
        x = tokens[b].tolist()
        row, taken = 0, []
        while True:
            p = weights(target[b, row])
            children = [i for i in range(count) if up[i] == row - 1 and -1 <= up[i] < i]
            found, low, seen = None, 0.0, set()
            for i in children:
                if not 0 <= x[i] < V:
                    continue
                mine = 0.0 if x[i] in seen else p[x[i]]
                seen.add(x[i])
                u = float(uniform[b, row])
                if draft is not None:
                    stands = u * weights(draft[b, i])[x[i]] < mine
                else:
                    stands = low <= u < low + mine
                if stands:
                    found = i
                low += mine
            if found is None:
                break
            taken.append(found)
            row = found + 1
        rest = p.copy()
        if draft is not None and row < count:
            rest = np.maximum(p - weights(draft[b, row]), 0)
        elif draft is None:
            for i in children:
                if 0 <= x[i] < V:
                    rest[x[i]] = 0
        token.append(drawn(rest if rest.sum() > 0 else p, sample[b]))
        accepted.append(len(taken))
        path.append(taken + [-1] * (T - len(taken)))
    return (torch.tensor(accepted, dtype=torch.int32), torch.tensor(path, dtype=torch.int32).view(B, T), torch.tensor(token, dtype=tokens.dtype))


def drafts(B, T, V, dtype, form, seed):
    """Probabilities, tokens that are right more often than not, and random numbers."""
    g = torch.Generator().manual_seed(seed)
    logits = 3 * torch.randn((B, T + 1, V), generator=g)
    a = dict(target=logits.softmax(-1).to(dtype), uniform=torch.rand((B, T), generator=g), sample=torch.rand((B,), generator=g))
    if form == "tree":
        a["parents"] = torch.tensor([[random.Random(seed + b).randint(-1, i - 1) if i else -1 for i in range(T)] for b in range(B)], dtype=torch.int32).view(B, T)
    rows = torch.arange(T).expand(B, T) if form != "tree" else a["parents"].long() + 1
    near = logits.gather(1, rows[..., None].expand(B, T, V))
    near = ((near + torch.randn((B, T, V), generator=g)) if form == "drawn" else 1.5 * near).softmax(-1)
    if form == "drawn":
        a["draft"] = near = near.to(dtype)
    a["tokens"] = torch.multinomial(near.float().reshape(B * T, V), 1, generator=g).view(B, T) if T else torch.empty((B, 0), dtype=torch.long)
    return a


def on_gpu(a):
    return {k: x.cuda() if isinstance(x, torch.Tensor) else x for k, x in a.items()}


def call(a):
    a = dict(a)
    return fca.verify_drafts(a.pop("target"), a.pop("tokens"), a.pop("uniform"), a.pop("sample"), **a)


def check(a, moved=None):
    got = call(on_gpu(a) if moved is None else moved)
    want = verified(**a)
    for x, y, name in zip(got, want, ("accepted", "path", "token")):
        assert x.dtype == y.dtype and torch.equal(x.cpu(), y), (name, x.cpu(), y)
    return want


def reserved(table, held, free, available, lengths, page_size):
    """cache_reserve on lists, in place."""
    need = [-(-max(0, *(n if isinstance(n, list) else [n])) // page_size) for n in lengths]
    width = len(table[0])
    for b in range(len(held)):
        while held[b] > need[b]:
            # (entries go back from the lowest on)
            for i in range(need[b], held[b]):
                free[available[0]] = table[b][i]
                available[0] += 1
                table[b][i] = -1
            held[b] = need[b]
    out, refused = [], False
    for b in range(len(held)):
        more = need[b] - held[b]
        if need[b] > width:
            out.append(False)
            continue
        if more <= 0:
            out.append(True)
            continue
        refused = refused or more > available[0]
        out.append(not refused)
        if refused:
            continue
        for i in range(held[b], need[b]):
            available[0] -= 1
            table[b][i] = free[available[0]]
        held[b] = need[b]
    return out


# Without a device --------------------------------------------------------------------------------------------------------

def test_the_plain_form_gives_what_the_target_draws():
    """The rule itself: the token behind the context is distributed as row 0 of the target, whatever was drafted."""
    g = torch.Generator().manual_seed(5)
    n, V = 20000, 6
    p, q = torch.rand(V, generator=g).softmax(0), torch.rand(V, generator=g).pow(3).softmax(0)
    target = p.expand(n, 4, V)
    for form in ("drawn", "chain", "tree"):
        a = dict(target=target, uniform=torch.rand((n, 3), generator=g), sample=torch.rand((n,), generator=g))
        if form == "drawn":
            a["draft"] = q.expand(n, 3, V)
            a["tokens"] = torch.multinomial(q, 3 * n, replacement=True, generator=g).view(n, 3)
        else:
            a["tokens"] = torch.tensor([2, 4, 2]).expand(n, 3)
        if form == "tree":
            a["parents"] = torch.tensor([-1, -1, -1], dtype=torch.int32)
        accepted, path, token = verified(**a)
        first = torch.where(accepted > 0, a["tokens"].gather(1, path[:, :1].long().clamp_min(0))[:, 0], token)
        share = torch.bincount(first, minlength=V) / n
        assert torch.all((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()), form


def _i64x2(*x):
    return cache_module._I64x2(*x)


def _verify_c(**over):
    a = dict(target=16, ts=(400, 100), draft=None, ds=(300, 100), tokens=32, token_bytes=8, parents=None, ps=3, counts=None, uniform=48, sample=64,
             accepted=80, path=96, token=112, ws=128, ws_bytes=1 << 40, dtype=2, B=2, T=3, V=100)
    a.update(over)
    return _lib.load().fcr_verify_drafts(
        a["target"], a["ts"] and _i64x2(*a["ts"]), a["draft"], a["ds"] and _i64x2(*a["ds"]), a["tokens"], a["token_bytes"], a["parents"], a["ps"], a["counts"],
        a["uniform"], a["sample"], a["accepted"], a["path"], a["token"], a["ws"], a["ws_bytes"], a["dtype"], a["B"], a["T"], a["V"], None)


@pytest.mark.parametrize("over, code", [
    (dict(target=None), -1), (dict(ts=None), -1), (dict(draft=16, ds=None), -1), (dict(tokens=None), -1), (dict(uniform=None), -1),
    (dict(sample=None), -1), (dict(accepted=None), -1), (dict(path=None), -1), (dict(token=None), -1), (dict(ws=None), -1),
    (dict(dtype=3), -2), (dict(dtype=-1), -2), (dict(token_bytes=2), -2), (dict(B=0), -3), (dict(T=-1), -3), (dict(T=1025), -3), (dict(V=0), -3),
    (dict(V=(1 << 28) + 1), -3), (dict(B=(1 << 20) + 1), -3), (dict(draft=16, parents=16), -3), (dict(target=18), -4), (dict(tokens=36), -4),
    (dict(uniform=49), -4), (dict(ts=(-1, 100)), -4), (dict(draft=16, ds=(1, -1)), -4), (dict(ps=-1, parents=16), -4), (dict(ws=136), -4), (dict(ws_bytes=15), -7)])
def test_c_abi_verify_refuses(over, code):
    """Every refusal comes before the first launch, so invented pointers are safe."""
    assert _verify_c(**over) == code
    assert _lib.load().fcr_last_error() != b""


def test_c_abi_verify_bytes():
    lib = _lib.load()
    assert lib.fcr_verify_drafts_bytes(0, 1, 1) == 0 and lib.fcr_verify_drafts_bytes(1, 1025, 1) == 0 and lib.fcr_verify_drafts_bytes(1, 0, 1) > 0


@pytest.mark.parametrize("over, code", [
    (dict(table=None), -1), (dict(context=None), -1), (dict(cs=None), -1), (dict(path=None), -1), (dict(accepted=None), -1), (dict(out=None), -1),
    (dict(stride=-1), -4), (dict(pages=0), -3), (dict(B=0), -3), (dict(T=0), -3), (dict(cs=(-1, 0)), -4), (dict(cs=(1, -1)), -4),
    (dict(cache=dict(D=24)), -3), (dict(cache=dict(k_strides=(0, 2048, 64))), -4), (dict(cache=dict(v=16)), -4)])
def test_c_abi_accept_refuses(over, code):
    a = dict(cache={}, table=16, stride=4, pages=4, context=32, cs=(1, 0), path=48, accepted=64, out=80, B=2, T=3)
    a.update(over)
    assert _lib.load().fcr_cache_accept(ctypes.byref(_c_cache(**a["cache"])), a["table"], a["stride"], a["pages"], a["context"],
                                        a["cs"] and _i64x2(*a["cs"]), a["path"], a["accepted"], a["out"], a["B"], a["T"], None) == code


@pytest.mark.parametrize("over, code", [
    (dict(table=None), -1), (dict(held=None), -1), (dict(free=None), -1), (dict(available=None), -1), (dict(lengths=None), -1), (dict(ls=None), -1),
    (dict(granted=None), -1), (dict(B=0), -3), (dict(H=0), -3), (dict(pages=0), -3), (dict(width=0), -3), (dict(page_size=0), -3),
    (dict(width=1 << 16, page_size=1 << 15), -3), (dict(B=1 << 20, width=1 << 11, stride=1 << 11), -3), (dict(stride=3), -4), (dict(ls=(-1, 0)), -4)])
def test_c_abi_reserve_refuses(over, code):
    a = dict(table=16, stride=4, width=4, held=32, free=48, pages=9, available=64, lengths=80, ls=(1, 0), H=1, page_size=16, granted=96, B=2)
    a.update(over)
    assert _lib.load().fcr_cache_reserve(a["table"], a["stride"], a["width"], a["held"], a["free"], a["pages"], a["available"], a["lengths"],
                                         a["ls"] and _i64x2(*a["ls"]), a["H"], a["page_size"], a["granted"], a["B"], None) == code


def test_python_refuses_host_tensors():
    a = drafts(1, 2, 10, F32, "chain", 1)
    with pytest.raises(ValueError, match="CUDA"):
        call(a)
    with pytest.raises(ValueError, match="CUDA"):
        fca.cache_reserve(PagePool.full(4, 2, device="cpu"), torch.full((2, 4), -1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 16)
    cache = KVCache.zeros(2, 2, 16, 16, F16, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        fca.cache_accept(cache, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32),
                         torch.zeros(1, dtype=torch.int32))


# verify_drafts -----------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("form", ["drawn", "chain", "tree"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B, T, V", [(1, 1, 1), (1, 1, 7), (3, 2, 8), (2, 5, 2047), (2, 5, 2048), (5, 4, 2049), (2, 63, 1000), (1, 3, 50001), (33, 6, 4097),
                                     (2, 300, 37), (300, 2, 5000)])
def test_verify(form, dtype, B, T, V):
    check(drafts(B, T, V, dtype, form, 100 * T + V))


@pytest.mark.gpu
def test_verify_of_a_large_vocabulary_and_batch():
    """Pieces of more than one turn of a workgroup."""
    for form in ("drawn", "tree"):
        check(drafts(70, 2, 100003, F32, form, 9))


@pytest.mark.gpu
def test_verify_without_drafts_draws_a_token():
    for dtype in (F32, BF16):
        a = drafts(4, 0, 3001, dtype, "chain", 3)
        check(a)
        a["tokens"] = a["tokens"].int()
        a["draft"] = torch.empty((4, 0, 3001), dtype=dtype)
        assert check(a)[0].sum() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["drawn", "chain", "tree"])
def test_verify_layouts(form):
    """Rows of any alignment, strides, rows that sequences share, tokens of 32 bits, one tree for all."""
    a = drafts(4, 5, 1003, F16, form, 8)
    a["tokens"] = a["tokens"].int()
    if form == "tree":
        a["parents"] = a["parents"][0].contiguous()
    moved = on_gpu(a)
    for name in ("target", "draft"):
        if name in a:
            x = torch.zeros((4, 9, 1100), dtype=F16, device="cuda")
            x[:, 1:1 + a[name].shape[1], 3:1006] = moved[name]
            moved[name] = x[:, 1:1 + a[name].shape[1], 3:1006]
    for name in ("tokens", "uniform"):
        moved[name] = moved[name].t().contiguous().t()
    check(a, moved)
    a["target"] = a["target"][:1].expand(4, -1, -1)
    moved = on_gpu(a)
    moved["target"] = moved["target"][:1].expand(4, -1, -1)
    check(a, moved)
    a["target"] = a["target"].contiguous()
    moved["target"] = a["target"].cuda().transpose(1, 2).contiguous().transpose(1, 2)
    check(a, moved)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["drawn", "chain", "tree"])
def test_verify_counts(form):
    a = drafts(7, 6, 500, F32, form, 2)
    a["uniform"] *= 0.3
    a["counts"] = torch.tensor([0, 1, 3, 6, 7, -2, 5], dtype=torch.int32)
    assert check(a)[0].max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["drawn", "chain", "tree"])
@pytest.mark.parametrize("u", [0.0, 0.5, 1 - 2.0 ** -24])
def test_verify_borders(form, u):
    """Random numbers at both ends, probabilities that are 0, 1 and equal to the draft's, weights next to zeros."""
    a = drafts(6, 4, 700, F32, form, 4)
    a["uniform"].fill_(u)
    a["sample"] = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5, 0.0, 1 - 2.0 ** -24, 0.25])
    a["target"][3:] = 0
    a["target"][3:, :, 650] = 0.25
    a["target"][3:, :, 70] = 0.75
    a["tokens"][3] = 70
    a["tokens"][4] = 650
    a["target"][5] = 0
    a["target"][5, :, 699] = 1
    a["tokens"][5] = 699
    if form == "drawn":
        a["draft"][3:5] = a["target"][3:5, :4]
        a["draft"][5] = 0
        a["draft"][5, :, 699] = 1
    check(a)


@pytest.mark.gpu
def test_verify_siblings_of_one_token_and_wrong_trees():
    """A token that a sibling has already has nothing left; parents that are not earlier tokens and tokens outside the vocabulary never stand."""
    a = drafts(64, 8, 6, F32, "tree", 6)
    a["tokens"] = torch.randint(-1, 8, (64, 8), generator=torch.Generator().manual_seed(1))
    a["parents"] = torch.randint(-3, 9, (64, 8), generator=torch.Generator().manual_seed(2)).int()
    a["parents"][:, 0] = -1
    assert 0 < check(a)[0].max()
    a["parents"][:32] = -1
    a["tokens"][:, 3] = a["tokens"][:, 1]
    check(a)
    a["tokens"][0] = torch.tensor([2 ** 40, -2 ** 40, 6, 5, 2 ** 32 + 1, 1, 1, 1])
    check(a)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["drawn", "chain", "tree"])
def test_verify_what_is_no_probability(form):
    """NaNs and negative numbers count as 0; a row without a weight, or with an infinite one, gives -1 and leaves the other sequences alone."""
    a = drafts(6, 3, 3000, F32, form, 12)
    a["target"][0, :, ::3] = math.nan
    a["target"][1, :, 1::2] = -1
    a["target"][2] = 0
    a["target"][3] = math.nan
    a["target"][4, :, 2500] = math.inf
    a["tokens"][4] = 3
    if form == "drawn":
        a["draft"][1, :, ::5] = math.nan
        a["draft"][5, :, ::5] = -0.5
    want = check(a)
    assert want[2][2] == want[2][3] == want[2][4] == -1


@pytest.mark.gpu
def test_verify_refuses():
    a = on_gpu(drafts(2, 3, 20, F32, "drawn", 1))
    tree = torch.tensor([-1, 0, 0], dtype=torch.int32, device="cuda")
    bad = [dict(target=a["target"][:, :3]), dict(target=a["target"].double()), dict(target=a["target"][0]), dict(tokens=a["tokens"].short()),
           dict(tokens=a["tokens"][:1]), dict(tokens=a["tokens"].cpu()), dict(uniform=a["uniform"].double()), dict(uniform=a["uniform"][:, :2]),
           dict(sample=a["sample"][:1]), dict(sample=a["sample"].half()), dict(draft=a["draft"].half()), dict(draft=a["draft"][:, :, :19]),
           dict(draft=a["draft"][:, :2]), dict(parents=tree), dict(draft=None, parents=tree.long()), dict(draft=None, parents=tree[:2]),
           dict(counts=torch.ones(3, dtype=torch.int32, device="cuda")), dict(counts=torch.ones(2, device="cuda"))]
    for over in bad:
        with pytest.raises(ValueError):
            call({**a, **over})
    long = on_gpu(drafts(1, 1025, 3, F32, "chain", 1))
    with pytest.raises(ValueError, match="1024"):
        call(long)
    out = fca.verify_drafts(torch.empty((0, 3, 5), device="cuda"), torch.empty((0, 2), dtype=torch.long, device="cuda"), torch.empty((0, 2), device="cuda"),
                            torch.empty((0,), device="cuda"))
    assert out.accepted.shape == (0,) and out.path.shape == (0, 2) and out.token.shape == (0,)


# cache_accept ------------------------------------------------------------------------------------------------------------

def some_cache(pages, H, ps, D, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pages, H, ps, D)
    if dtype in (F16, BF16):
        return KVCache(*(torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2)))
    rows = [torch.randint(-100, 100, shape, generator=g, device="cuda", dtype=torch.int8) for _ in range(2)]
    return KVCache(*(x.view(dtype) if dtype == E4M3 else x for x in rows), *(torch.rand(shape[:3], generator=g, device="cuda") for _ in range(2)))


def bits(x):
    return x.view(torch.int8) if x.element_size() == 1 else x.view(torch.int16) if x.element_size() == 2 else x


def accepted_plain(cache, table, context, path, accepted):
    """On the host, one row at a time."""
    pages, H, ps, _ = cache.k.shape
    out = [None if x is None else bits(x).cpu().clone() for x in cache]
    table, path, accepted, context = table.cpu(), path.cpu(), accepted.cpu(), context.cpu()
    for b in range(table.shape[0]):
        for h in range(H):
            c = max(int(context[b] if context.dim() == 1 else context[b, h]), 0)
            for i in range(min(max(int(accepted[b]), 0), path.shape[1])):
                at, to = c + int(path[b, i]), c + i
                if at >= table.shape[1] * ps:
                    continue
                page, to_page = int(table[b, at // ps]), int(table[b, to // ps])
                if 0 <= page < pages and 0 <= to_page < pages:
                    for x in out:
                        if x is not None:
                            x[to_page, h, to % ps] = x[page, h, at % ps].clone()
    return out


def paths(B, T, accepted, seed):
    rng = random.Random(seed)
    out = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        out[b, :accepted[b]] = torch.tensor(sorted(rng.sample(range(T), accepted[b])), dtype=torch.int32)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("B, H, T, D, ps", [(1, 1, 1, 16, 16), (2, 3, 7, 64, 16), (3, 2, 63, 80, 32), (2, 2, 300, 256, 16), (1, 5, 100, 176, 48), (5, 8, 16, 128, 128), (130, 8, 40, 96, 16)])
def test_accept(dtype, B, H, T, D, ps):
    rng = random.Random(T)
    for turn in range(2):
        per = -(-(T + 70) // ps)
        cache = some_cache(B * per + 2, H, ps, D, dtype, 7 + turn)
        table = torch.randperm(B * per + 2, device="cuda")[:B * per].view(B, per).int()
        context = torch.randint(0, 70, (B, H) if turn else (B,), dtype=torch.int32, device="cuda")
        n = [rng.randint(0, T) for _ in range(B)]
        path = paths(B, T, n, 3 + turn).cuda()
        accepted = torch.tensor(n, dtype=torch.int32, device="cuda")
        want = accepted_plain(cache, table, context, path, accepted)
        got = fca.cache_accept(cache, table, context, path, accepted)
        assert torch.equal(got, context + (accepted[:, None] if turn else accepted)) and got.dtype == torch.int32
        for x, y in zip(cache, want):
            assert (x is None) == (y is None) and (x is None or torch.equal(bits(x).cpu(), y))


@pytest.mark.gpu
def test_accept_pages_that_are_not_there_and_odd_arguments():
    cache = some_cache(6, 2, 16, 32, BF16, 1)
    table = torch.tensor([[0, -1, 2, 9], [3, 4, 5, -7]], dtype=torch.int32, device="cuda")
    context = torch.tensor([5, -3], dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 9, 12, 13, 30, 31, 58, 60], [1, 2, 17, 33, 47, 48, 200, -1]], dtype=torch.int32, device="cuda")
    for n in ([8, 7], [0, 0], [-1, 100], [3, 1]):
        accepted = torch.tensor(n, dtype=torch.int32, device="cuda")
        want = accepted_plain(cache, table, context, path, accepted)
        got = fca.cache_accept(cache, table, context, path, accepted)
        assert got.tolist() == [5 + min(max(n[0], 0), 8), min(max(n[1], 0), 8)]
        assert all(x is None or torch.equal(bits(x).cpu(), y) for x, y in zip(cache, want))


@pytest.mark.gpu
def test_accept_views():
    """Keys and values in one allocation, token-major pages, heads' lengths by an expanded view, arguments that are not contiguous."""
    both = torch.randn((9, 2, 16, 3, 64), device="cuda", dtype=F16)
    cache = KVCache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2))
    table = torch.arange(16, device="cuda", dtype=torch.int32).view(2, 8)[:, :4]
    context = torch.tensor([3, 20], dtype=torch.int32, device="cuda")
    path = paths(2, 12, [5, 9], 4).cuda().t().contiguous().t()
    accepted = torch.tensor([5, 0, 9, 0], dtype=torch.int32, device="cuda")[::2]
    want = accepted_plain(cache, table, context, path, accepted)
    got = fca.cache_accept(cache, table, context[:, None].expand(2, 3), path, accepted)
    assert got.tolist() == [[8] * 3, [29] * 3]
    assert all(x is None or torch.equal(bits(x).cpu(), y) for x, y in zip(cache, want))
    empty = fca.cache_accept(cache, table, context, path[:, :0], accepted)
    assert torch.equal(empty, context)


@pytest.mark.gpu
def test_accept_refuses():
    cache = some_cache(4, 2, 16, 32, F16, 1)
    z = dict(dtype=torch.int32, device="cuda")
    good = dict(table=torch.zeros((2, 2), **z), context=torch.zeros(2, **z), path=torch.zeros((2, 3), **z), accepted=torch.zeros(2, **z))
    bad = [dict(table=good["table"].long()), dict(context=good["context"].long()), dict(context=torch.zeros((2, 3), **z)), dict(path=torch.zeros((3, 3), **z)),
           dict(path=good["path"].long()), dict(path=torch.zeros(2, **z)), dict(accepted=torch.zeros(3, **z)), dict(accepted=good["accepted"].cpu())]
    for over in bad:
        with pytest.raises(ValueError):
            fca.cache_accept(cache, *{**good, **over}.values())
    with pytest.raises(_lib.FcrError):
        fca.cache_accept(KVCache(cache.k, cache.k), *good.values())
    with pytest.raises(_lib.FcrError):
        fca.cache_accept(KVCache(cache.k[:1].expand(4, 2, 16, 32), cache.v), *good.values())


# cache_reserve -----------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("B, width, pages, page_size", [(1, 1, 1, 16), (1, 40, 64, 16), (3, 5, 11, 16), (17, 9, 60, 48), (200, 30, 2500, 16), (1024, 4, 2000, 32),
                                                        (1025, 3, 2500, 16), (2600, 6, 6000, 1), (2, 9000, 12000, 16)])
def test_reserve(B, width, pages, page_size):
    """Many steps of one pool: the same table, stack and answers as the plain form, every page once."""
    rng = random.Random(B)
    pool = PagePool.full(pages, B)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    mine = [table.cpu().tolist(), [0] * B, pool.free.cpu().tolist(), [pages]]
    for step in range(8):
        top = width * page_size + (3 if step % 3 == 2 else 0)
        heads = step == 4
        lengths = [0 if rng.random() < 0.2 else rng.randint(-2, top if rng.random() < 0.3 else max(1, min(top, 2 * page_size * pages // B))) for _ in range(B)]
        if heads:
            lengths = [[n, max(n - 5, 0), rng.randint(0, max(n, 0))] for n in lengths]
        granted = fca.cache_reserve(pool, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), page_size)
        want = reserved(mine[0], mine[1], mine[2], mine[3], lengths, page_size)
        assert granted.tolist() == want, step
        assert table.tolist() == mine[0] and pool.held.tolist() == mine[1] and pool.available.tolist() == mine[3]
        assert pool.free.tolist() == mine[2]
        on_stack = pool.free[:int(pool.available)].tolist()
        assert sorted(on_stack + [x for row in mine[0] for x in row if x >= 0]) == list(range(pages))


@pytest.mark.gpu
def test_reserve_views_and_refusals():
    z = dict(dtype=torch.int32, device="cuda")
    pool = PagePool.full(20, 3)
    wide = torch.full((3, 10), -1, **z)
    table = wide[:, 2:8]
    lengths = torch.tensor([[40, 0], [0, 0], [16, 17]], **z)
    assert fca.cache_reserve(pool, table, lengths.t().contiguous().t(), 16).tolist() == [True] * 3
    assert table.tolist() == [[0, 1, 2, -1, -1, -1], [-1] * 6, [3, 4, -1, -1, -1, -1]] and bool((wide[:, :2] == -1).all()) and bool((wide[:, 8:] == -1).all())
    assert fca.cache_reserve(pool, torch.empty((3, 0), **z), lengths, 16).tolist() == [False, True, False]
    assert fca.cache_reserve(PagePool.full(3, 0), torch.empty((0, 4), **z), torch.empty((0,), **z), 16).shape == (0,)
    bad = [dict(table=table.long()), dict(table=wide[:1].expand(3, 10)), dict(table=wide.t()[:3]), dict(lengths=lengths.long()), dict(lengths=lengths[:2]),
           dict(lengths=lengths[:, :0]), dict(page_size=0), dict(page_size=2 ** 30), dict(pool=pool._replace(free=pool.free.long())),
           dict(pool=pool._replace(free=pool.free[::2])), dict(pool=pool._replace(held=pool.held[:2])), dict(pool=pool._replace(available=pool.held)),
           dict(pool=pool._replace(free=pool.free[:0])), dict(lengths=lengths.cpu()), dict(pool=pool._replace(held=pool.held.cpu()))]
    for over in bad:
        a = {**dict(pool=pool, table=table, lengths=lengths, page_size=16), **over}
        with pytest.raises(ValueError):
            fca.cache_reserve(a["pool"], a["table"], a["lengths"], a["page_size"])


# Together ----------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, I8])
def test_a_loop_of_drafted_trees(dtype):
    """Pages, rows, verification and moved rows over several steps: what the cache then reads back is what was written for the tokens that stood."""
    B, H, T, D, ps, V, width = 3, 2, 9, 64, 16, 50, 8
    pool = PagePool.full(B * 5, B)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    cache = some_cache(B * 5, H, ps, D, dtype, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    parents = torch.tensor([-1, -1, 0, 0, 1, 2, 2, 4, 5], dtype=torch.int32, device="cuda")
    mask = torch.eye(T, dtype=torch.bool, device="cuda")
    for i, up in enumerate(parents.tolist()):
        if up >= 0:
            mask[i] |= mask[up]
    context = torch.zeros(B, dtype=torch.int32, device="cuda")
    written = [([], []) for _ in range(B)]
    for step in range(6):
        assert bool(fca.cache_reserve(pool, table, context + T, ps).all())
        key, value = (torch.randn((B, H, T, D), generator=g, device="cuda", dtype=BF16) for _ in range(2))
        fca.cache_write(cache, key, value, table, context)
        whole = [x.float() for x in fca.cache_read(cache, table, context + T, width * ps, out_dtype=F32)]
        query = torch.randn((B, 2 * H, T, D), generator=g, device="cuda", dtype=BF16)
        out = fca.tree_attention(query, cache, table, context, mask)
        a = on_gpu(drafts(B, T, V, F32, "tree", step))
        a["parents"], a["uniform"] = parents, a["uniform"] * 0.2
        accepted, path, token = call(a)
        # the row of a token's result is what its own path gives, whatever else was drafted
        for b in range(B):
            n, c = int(accepted[b]), int(context[b])
            if n:
                at = torch.cat((torch.arange(c), c + path[b, :n].cpu())).cuda()
                k, v = (x[b, :, at].repeat_interleave(2, 0) for x in whole)
                w = (query[b, :, int(path[b, n - 1])].float()[:, None] @ k.transpose(1, 2)) / math.sqrt(D)
                torch.testing.assert_close(out[b, :, int(path[b, n - 1])].float(), (w.softmax(-1) @ v)[:, 0], rtol=2 ** -7, atol=2 ** -7)
            for i in path[b, :n].tolist():
                written[b][0].append(whole[0][b, :, c + i])
                written[b][1].append(whole[1][b, :, c + i])
        context = fca.cache_accept(cache, table, context, path, accepted)
        assert bool(fca.cache_reserve(pool, table, context, ps).all())
        assert context.tolist() == [len(w[0]) for w in written]
        k, v = fca.cache_read(cache, table, context, width * ps, out_dtype=F32)
        for b in range(B):
            for x, rows in ((k, written[b][0]), (v, written[b][1])):
                if rows:
                    assert torch.equal(x[b, :, :len(rows)], torch.stack(rows, 1))
    assert int(context.sum()) > 0


@pytest.mark.gpu
def test_captured_steps():
    """Verification, moved rows and pages in two graphs of one pool, replayed with new inputs between eager calls."""
    B, T, V = 4, 6, 5000
    inputs = [on_gpu(drafts(B, T, V, F32, "tree", s)) for s in range(4)]
    a = {k: x.clone() for k, x in inputs[0].items()}
    table = torch.arange(B * 4, device="cuda", dtype=torch.int32).view(B, 4)
    context = torch.tensor([0, 3, 16, 30], dtype=torch.int32, device="cuda")
    caches = [some_cache(B * 4, 2, 16, 32, F16, 5) for _ in range(2)]
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    pools = [PagePool.full(40, B) for _ in range(2)]
    tables = [torch.full((B, 8), -1, dtype=torch.int32, device="cuda") for _ in range(2)]

    def step(i):
        out = call(a)
        return (*out, fca.cache_accept(caches[i], table, context, out.path, out.accepted), fca.cache_reserve(pools[i], tables[i], lengths, 16))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call(a)
    torch.cuda.current_stream().wait_stream(stream)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(0)
    with torch.cuda.graph(other, pool=graph.pool()):
        got_other = call(a)
    for s in (1, 2, 3, 0, 2):
        for k, x in inputs[s].items():
            a[k].copy_(x)
        lengths.copy_(torch.tensor([s * 16, 100 - s, 0, 17 * s], dtype=torch.int32))
        graph.replay()
        got_now = [x.clone() for x in got]
        other.replay()
        torch.cuda.synchronize()
        want = step(1)
        assert all(torch.equal(x, y) for x, y in zip(got_now, want))
        assert all(torch.equal(x, y) for x, y in zip(got_other, want))
        assert all(torch.equal(x, y) for x, y in zip(caches[0][:2], caches[1][:2]))
        assert all(torch.equal(x, y) for x, y in zip((*pools[0], tables[0]), (*pools[1], tables[1])))


@pytest.mark.gpu
def test_other_streams():
    """Calls on two streams at once, tensors made on a third."""
    sets = [on_gpu(drafts(3, 4, 30000, F32, "drawn", s)) for s in range(2)]
    want = [call(x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for out in got[i] for x, y in zip(out, want[i]))
