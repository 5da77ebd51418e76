"""The paged cache (cache_write, cache_read, cache_keep) and tree_attention against plain forms in 64 bits, at the sizes, layouts
and masks where they can go wrong, and their refusals."""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

import flash_colreduce_amd as fca
from flash_colreduce_amd import KVCache, _lib
from flash_colreduce_amd import cache as cache_module

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16, F32, I8, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn
TOP = {I8: 127.0, E4M3: 448.0}
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


# Without a device --------------------------------------------------------------------------------------------------------

def test_division_by_a_fixed_number(tmp_path):
    """csrc/div.h against C's division: every small divisor, powers of two and their neighbours, dividends at every border."""
    (tmp_path / "d.cpp").write_text(
        '#include "div.h"\n#include <stdint.h>\n'
        'static int64_t bad(uint32_t d, uint32_t n) { fcr_paged::Div v; v.set(d); return v.of(n) == n / d ? 0 : 1; }\n'
        'extern "C" int64_t check(uint32_t d) {\n'
        '  int64_t wrong = 0; const uint32_t top = 0x7fffffffu;\n'
        '  for (uint32_t i = 0; i < 2000; ++i) { wrong += bad(d, i) + bad(d, top - i);\n'
        '    const uint64_t m = (uint64_t)d * i, z = (uint64_t)(top / d - (i < top / d ? i : 0)) * d;\n'
        '    if (m <= top) wrong += bad(d, (uint32_t)m) + (m ? bad(d, (uint32_t)m - 1) : 0);\n'
        '    wrong += bad(d, (uint32_t)z) + (z ? bad(d, (uint32_t)z - 1) : 0); }\n'
        '  return wrong; }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "flash_colreduce_amd", "csrc"),
                    str(tmp_path / "d.cpp"), "-o", str(tmp_path / "d.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "d.so"))
    lib.check.restype = ctypes.c_int64
    rng = random.Random(1)
    for d in [*range(1, 700), *(2 ** e + i for e in range(10, 31) for i in (-1, 0, 1)), 2 ** 31 - 1, *(rng.randint(1, 2 ** 31 - 1) for _ in range(200))]:
        assert lib.check(ctypes.c_uint32(d)) == 0, d


def test_attention_blocks_are_dealt_once_and_joined_in_order():
    """The distribution of csrc/tree_attention.hip restated: every block of every item is taken by one workgroup, and the join finds the
    parts of an item, and no others, in the order of its keys."""
    rng = random.Random(3)
    for _ in range(300):
        items = [max(1, -(-rng.choice([0, 1, 127, 128, 129, rng.randint(0, 9000)]) // 128)) for _ in range(rng.randint(1, 40))]
        wgs = 8 * rng.randint(1, 64)
        total = sum(items)
        per = max(-(-total // wgs), 1)
        parts, first = {}, {}
        for w in range(wgs):
            at, end = w * per, min(w * per + per, total)
            while at < end:
                begun, item = 0, 0
                while at >= begun + items[item]:
                    begun += items[item]
                    item += 1
                blk = at - begun
                stop = min(items[item], blk + end - at)
                if blk == 0:
                    first[item] = at
                if not (blk == 0 and stop == items[item]):
                    slot = 2 * w + (1 if blk == 0 else 0)
                    assert slot not in parts
                    parts[slot] = (item, blk, stop)
                at += stop - blk
        for item, blocks in enumerate(items):
            a, z = first[item] // per, (first[item] + blocks - 1) // per
            if a == z:
                assert not any(p[0] == item for p in parts.values())
                continue
            got = [parts.pop(2 * w + (1 if w == a else 0)) for w in range(a, z + 1)]
            assert [g[0] for g in got] == [item] * len(got)
            assert got[0][1] == 0 and got[-1][2] == blocks and all(x[2] == y[1] for x, y in zip(got, got[1:]))
        assert not parts


def test_pieces_of_one_item_each_cover_it_once():
    """The other distribution: pieces of at most `most` blocks, a workgroup for each; and what the join derives from the first one's length."""
    for blocks in range(1, 400):
        for most in range(1, 60):
            pieces = -(-blocks // most)
            length = -(-blocks // pieces)
            ends = [(i * length, min(i * length + length, blocks)) for i in range(pieces)]
            assert all(a < z <= a + most for a, z in ends) and ends[0][0] == 0 and ends[-1][1] == blocks
            assert -(-(blocks - ends[0][1]) // most) == pieces - 1


def _c_cache(**over):
    a = dict(k=16, v=32, k_scale=48, v_scale=64, k_strides=(16384, 2048, 64), v_strides=(16384, 2048, 64), k_scale_strides=(256, 32, 1),
             v_scale_strides=(256, 32, 1), dtype=3, pages=4, H=8, page_size=32, D=64)
    a.update(over)
    c = cache_module._Cache()
    for name, x in a.items():
        setattr(c, name, tuple(x) if isinstance(x, tuple) else x)
    for name in ("k_strides", "v_strides", "k_scale_strides", "v_scale_strides"):
        setattr(c, name, cache_module._I64x3(*a[name]))
    return c


def _c_call(fn, cache, **over):
    lib = _lib.load()
    a = dict(table=16, stride=4, pages=4, lengths=32, ls=(1, 0), x=48, y=64, dtype=0, B=2, T=3, N=100, G=2, xs=(4096, 512, 64, 1),
             into=None, keep=16, counts=16, mask=None, mask_stride=0, scale=0.1, ws=128, ws_bytes=1 << 40, out=16, more=None, ms=None)
    a.update(over)
    c = None if cache is None else ctypes.byref(cache)
    ls = None if a["ls"] is None else cache_module._I64x2(*a["ls"])
    ms = None if a["ms"] is None else cache_module._I64x2(*a["ms"])
    xs = None if a["xs"] is None else _lib.strides4(a["xs"])
    t = (a["table"], a["stride"], a["pages"])
    if fn == "write":
        return lib.fcr_cache_write(c, *t, a["lengths"], ls, a["more"], ms, a["x"], a["y"], a["dtype"], a["B"], a["T"], xs, xs, None)
    if fn == "read":
        return lib.fcr_cache_read(c, *t, a["lengths"], ls, a["x"], a["y"], a["dtype"], a["B"], a["N"], None)
    if fn == "keep":
        into = a["into"] or _c_cache()
        return lib.fcr_cache_keep(c, *t, a["lengths"], ls, a["keep"], a["N"], ctypes.byref(into), *t, a["counts"], a["B"], None)
    return lib.fcr_tree_attention(a["x"], c, *t, a["lengths"], ls, a["mask"], a["mask_stride"], None, a["out"], None, a["ws"], a["ws_bytes"],
                                  a["dtype"], a["B"], a["G"], a["T"], xs, a["scale"], None)


@pytest.mark.parametrize("fn", ["write", "read", "keep", "attention"])
def test_c_abi_rejects_bad_arguments_without_a_device(fn):
    """Every refusal comes before the first launch, so invented pointers are safe."""
    bad_cache = [(dict(k=None), -1), (dict(v=None), -1), (dict(k_scale=None), -1), (dict(v_scale=None), -1), (dict(dtype=2), -2),
                 (dict(dtype=5), -2), (dict(dtype=-1), -2), (dict(pages=0), -3), (dict(H=0), -3), (dict(page_size=0), -3),
                 (dict(page_size=24), -3), (dict(page_size=-16), -3), (dict(D=8), -3), (dict(D=72), -3), (dict(D=272), -3),
                 (dict(k=20), -4), (dict(v_strides=(16384, 2048, 60)), -4), (dict(k_strides=(16384, -2048, 64)), -4),
                 (dict(k_strides=(16384, 2048, 48)), -4), (dict(v_strides=(16384, 2048, 1 << 25)), -4), (dict(k_strides=(8, 2048, 64)), -4),
                 (dict(k_scale=50), -4), (dict(v_scale_strides=(256, 32, 2)), -4), (dict(k_scale_strides=(256, 30, 1)), -4)]
    for over, code in bad_cache:
        assert _c_call(fn, _c_cache(**over)) == code, over
        assert _lib.load().fcr_last_error() != b""
    if fn == "keep":
        for over, code in bad_cache:
            assert _c_call(fn, _c_cache(), into=_c_cache(**over)) == code, over
    assert _c_call(fn, None) == -1
    bad = [(dict(table=None), -1), (dict(lengths=None), -1), (dict(ls=None), -1), (dict(pages=0), -3), (dict(B=0), -3),
           (dict(pages=1 << 26), -3), (dict(stride=-1), -4), (dict(ls=(-1, 0)), -4), (dict(ls=(1, -1)), -4), (dict(table=18), -4)]
    if fn in ("write", "read"):
        bad += [(dict(x=None), -1), (dict(y=None), -1), (dict(dtype=3), -2), (dict(dtype=-1), -2), (dict(x=24), -4)]
    if fn == "write":
        bad += [(dict(T=0), -3), (dict(T=(1 << 30) + 1), -3), (dict(B=1 << 20, T=1 << 9), -3), (dict(xs=None), -1), (dict(xs=(4096, 512, 64, 2)), -4),
                (dict(xs=(4096, 512, 60, 1)), -4), (dict(xs=(-4096, 512, 64, 1)), -4), (dict(more=16), -1), (dict(more=16, ms=(-1, 0)), -4)]
    if fn == "read":
        bad += [(dict(N=0), -3), (dict(N=(1 << 30) + 1), -3), (dict(B=1 << 20, N=1 << 9), -3)]
    if fn == "keep":
        bad += [(dict(keep=None), -1), (dict(counts=None), -1), (dict(N=0), -3), (dict(N=(1 << 30) + 1), -3), (dict(B=1 << 22), -3),
                (dict(into=_c_cache(dtype=4)), -2), (dict(into=_c_cache(H=4)), -3), (dict(into=_c_cache(D=48)), -3)]
    if fn == "attention":
        bad += [(dict(x=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(xs=None), -1), (dict(dtype=2), -2), (dict(T=0), -3),
                (dict(G=0), -3), (dict(T=1 << 24, G=2), -3), (dict(scale=math.inf), -6), (dict(scale=math.nan), -6), (dict(x=20), -4),
                (dict(xs=(4096, 512, 64, 2)), -4), (dict(xs=(4096, 512, 60, 1)), -4), (dict(mask=16, mask_stride=-1), -4), (dict(ws=24), -4),
                (dict(out=24), -4), (dict(ws_bytes=100), -7)]
        assert _c_call(fn, _c_cache(dtype=1, k_strides=(16384, 2048, 64), v_strides=(16384, 2048, 64)), dtype=0) == -2
    for over, code in bad:
        assert _c_call(fn, _c_cache(), **over) == code, over


def test_workspace_size_of_tree_attention():
    lib = _lib.load()
    for bad in ((0, 8, 4, 1, 128, 1000), (1, 0, 4, 1, 128, 1000), (1, 8, 0, 1, 128, 1000), (1, 8, 4, 0, 128, 1000), (1, 8, 4, 1, 0, 1000),
                (1, 8, 4, 1, 272, 1000), (1, 8, 4, 1, 128, 0), (1 << 20, 1 << 10, 1, 1, 128, 1 << 20)):
        assert lib.fcr_tree_attention_bytes(*bad) == 0, bad
    assert 0 < lib.fcr_tree_attention_bytes(1, 8, 4, 1, 128, 1000) <= lib.fcr_tree_attention_bytes(64, 8, 4, 1, 128, 1000)


def test_native_host_path_leaves_the_rest_to_python():
    """Tensors on the host, other objects, wrong counts of arguments."""
    host, x = cache_module._host(), torch.zeros(1, 1, 1, 16)
    cache, ints = KVCache(x, x), torch.zeros(1, 1, dtype=torch.int32)
    assert host.cache_write(cache, x, x, ints, ints[0], None) is None and host.cache_read(None, ints, ints[0], 1, None) is None
    assert host.cache_keep(cache, ints, ints[0], x, (), ints) is None and host.cache_read((1, 2, 3, 4), ints, ints[0], 1, None) is None
    assert host.tree_attention(x, cache, ints, ints[0], None, None, None, False) is None
    if host is not _lib._PythonOnly:
        for f in (host.cache_write, host.cache_read, host.cache_keep, host.tree_attention):
            with pytest.raises(TypeError):
                f(cache)


def test_masks_past_32_bits_are_refused_without_a_device():
    assert _c_call("attention", _c_cache(), mask=16, T=46341, G=1) == -3


def test_python_refuses_without_a_device():
    c = KVCache.zeros(2, 1, 16, 16, I8, device="cpu")
    i = torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(1, 1, 1, 16)
    for call in (lambda: fca.cache_write(c, x, x, i, i[0]), lambda: fca.cache_read(c, i, i[0], 1),
                 lambda: fca.cache_keep(c, i, i[0], torch.zeros(1, 1, 1, dtype=torch.bool), c, i), lambda: fca.tree_attention(x, c, i, i[0])):
        with pytest.raises(ValueError, match="must be on CUDA device"):
            call()
    with pytest.raises(ValueError, match="A cache holds"):
        KVCache.zeros(2, 1, 16, 16, F32, device="cpu")
    assert KVCache.zeros(2, 1, 16, 16, BF16, device="cpu").k_scale is None


# Plain forms, in 64 bits -------------------------------------------------------------------------------------------------

def randn(*shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def nearest_e4m3(x):
    step = torch.exp2(x.abs().clamp_min(1e-300).log2().floor().clamp_min(-6) - 3)
    return (x / step).round() * step


def ref_codes(x, kind):
    """(values of the codes, scales) of rows x, from the definition."""
    x = x.double()
    a = x.abs().amax(-1)
    fine = x.isfinite().all(-1)
    safe = torch.where(fine & (a > 0), a, 1.0)
    c = torch.where(fine[..., None], x, 0.0) * TOP[kind] / safe[..., None]
    c = c.round() if kind == I8 else nearest_e4m3(c)
    return c, torch.where(fine, a / TOP[kind], math.nan)


def random_table(b, per, pages, seed):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: b * per].view(b, per).int()


def make_cache(pages, h, page, d, kind, dtype, seed, spread=0.0):
    """A cache with random rows everywhere; spread: how far the rows' sizes differ (a power of two, either way)."""
    rows = [randn(pages, h, page, d, seed=seed + i) for i in range(2)]
    if spread:
        rows[1] = rows[1] * torch.exp2(randn(pages, h, page, 1, seed=seed + 2) * spread)
    if kind not in TOP:
        return KVCache(*(r.to(kind) for r in rows))
    codes = [ref_codes(r, kind) for r in rows]
    return KVCache(*(c.to(F32).to(kind) for c, _ in codes), *(s.float() for _, s in codes))


def device(cache):
    return KVCache(*(None if x is None else x.cuda() for x in cache))


def values(cache, table, n):
    """(keys, values) (B, H, n, D) in 64 bits, and which positions are there (B, n)."""
    page_size, pages = cache.k.shape[2], cache.k.shape[0]
    at = torch.arange(n)
    inside = at < table.shape[1] * page_size
    page = table.long()[:, (at // page_size).clamp(max=table.shape[1] - 1)]
    there = inside & (page >= 0) & (page < pages)
    page = torch.where(there, page, 0)
    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        y = x.float().double()[page, :, (at % page_size).expand_as(page)]           # (B, n, H, D)
        if s is not None:
            y = y * s.double()[page, :, (at % page_size).expand_as(page)][..., None]
        out.append(y.transpose(1, 2))
    return out[0], out[1], there


def of_heads(x, h):
    return x[:, None].expand(-1, h) if x.dim() == 1 else x


def ref_attention(query, cache, table, context, mask, scale, tree_lengths):
    """(out, lse2, tolerance of out, of lse2) in 64 bits."""
    b, hq, t, d = query.shape
    h = cache.k.shape[1]
    g = hq // h
    n = min(int(context.clamp_min(0).max()) + t, table.shape[1] * cache.k.shape[2])
    n = max(n, 1)
    k, v, there = values(cache, table, n)
    scale = 1 / math.sqrt(d) if scale is None else scale
    u = torch.arange(n) - of_heads(context.clamp_min(0), h)[..., None].long()                    # (B, H, n)
    lengths = torch.full((b,), t) if tree_lengths is None else tree_lengths.long().clamp(0, t)
    if mask is None:
        mask = torch.ones(t, t, dtype=torch.bool).tril()
    mask = mask.expand(b, t, t)
    tree = mask[:, None].expand(b, h, t, t).gather(-1, u.clamp(0, t - 1)[:, :, None].expand(b, h, t, n))
    seen = (u < 0)[:, :, None] | (tree & (u < lengths[:, None, None])[:, :, None])
    seen = seen & there[:, None, None] & (torch.arange(t) < lengths[:, None])[:, None, :, None]  # (B, H, T, n)
    seen = seen.repeat_interleave(g, 1)
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    q = query.float().double()
    any_seen = seen.any(2, keepdim=True).transpose(2, 3)
    k0, v0 = torch.where(any_seen, k, 0.0), torch.where(any_seen, v, 0.0)
    s = torch.where(seen, q @ k0.transpose(-1, -2) * scale, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(lse.isfinite(), lse, 0.0)[..., None]), 0.0)
    # a value that is not finite reaches the rows that see it, and no others
    out = p @ torch.where(v0.isfinite(), v0, 0.0)
    for bi, hi, j in (~v0.isfinite()).any(-1).nonzero().tolist():
        sees = seen[bi, hi, :, j]
        bad = torch.where(v0[bi, hi, j].isfinite(), 0.0, v0[bi, hi, j])
        out[bi, hi, sees] = out[bi, hi, sees] + p[bi, hi, sees, j][:, None] * bad
    # First order: weights rounded to fp16 (bf16 against a bf16 cache) change a value by half a step of their own; those under 2^-14 of the
    # largest by half a step of fp16's smallest, 2^-25 (references lag the largest weight by a factor of 2 at most); scores are fp32 sums of D products,
    # each off by 2^-24 of the sum of magnitudes at most (in base 2, hence log2 e), their rounding, and exp2's 2^-21.
    rounding = HALF_STEP[BF16 if cache.k.dtype == BF16 else F16]
    v1 = torch.where(v0.isfinite(), v0, 0.0).abs()
    magnitude = torch.where(any_seen.transpose(2, 3) & seen, q.abs() @ torch.where(k0.isfinite(), k0, 0.0).abs().transpose(-1, -2) * abs(scale), 0.0).amax(-1)
    ds = (d + 8) * 2.0 ** -24 * magnitude + 2.0 ** -21
    weighted = p @ v1
    least = 2.0 ** -24 * n * (p.amax(-1, keepdim=True) * v1.amax((-1, -2), keepdim=True) if cache.k_scale is None
                              else (p * v1.amax(-1)[:, :, None]).amax(-1, keepdim=True))
    tol = weighted * (rounding + 2 * ds[..., None]) + 2 * least + out.abs() * HALF_STEP[query.dtype] * 1.01 + 2.0 ** -24
    dead = ~seen.any(-1)
    out[dead], lse[dead] = 0.0, -math.inf
    return out, lse / math.log(2), tol, 2 * (ds + 2.0 ** -22 * (1 + lse.abs()))


def check_attention(query, cache, table, context, mask=None, scale=None, tree_lengths=None, **how):
    got, lse = fca.tree_attention(query.cuda(), device(cache), table.cuda(), context.cuda(), None if mask is None else mask.cuda(), scale,
                                  tree_lengths=None if tree_lengths is None else tree_lengths.cuda(), return_lse2=True)
    assert got.dtype == query.dtype and got.shape == query.shape
    compare_attention(got, lse, ref_attention(query, cache, table, context, mask, scale, tree_lengths))
    return got, lse


def compare_attention(got, lse, ref):
    want, want_lse, tol, tol_lse = ref
    # what rounds to more than the type's largest number is an infinity there (within the tolerance of that border it may be either)
    border = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    got, lse = got.cpu().double(), lse.cpu().double()
    want = torch.where((want.abs() > border) & (got.isinf() | (want.abs() - tol > border)), want.sign() * math.inf, want)
    got = torch.where(got.isinf() & want.isfinite() & (want.abs() + tol >= border), want, got)
    fine = want.isfinite()
    assert torch.equal(got.isfinite(), fine) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~fine].nan_to_num(0), want[~fine].nan_to_num(0))
    over = ((got - want).abs() / tol)[fine]
    assert over.numel() == 0 or over.max() <= 1, over.max()
    live = want_lse.isfinite()
    assert torch.equal(lse.isneginf(), want_lse.isneginf())
    if live.any():
        assert ((lse - want_lse).abs()[live] <= tol_lse[live]).all(), ((lse - want_lse).abs() / tol_lse)[live].max()


# cache_write, cache_read ---------------------------------------------------------------------------------------------------

WRITES = [(1, 1, 1, 16, 16, 1), (3, 2, 5, 32, 16, 4), (2, 3, 17, 48, 32, 3), (1, 8, 129, 64, 16, 12), (2, 5, 33, 80, 48, 2), (1, 2, 70, 96, 16, 7),
          (4, 1, 1, 112, 64, 2), (2, 4, 61, 128, 16, 9), (1, 3, 40, 144, 112, 1), (2, 2, 31, 192, 32, 3), (1, 2, 100, 240, 16, 9), (2, 2, 19, 256, 16, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("kind", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("b,h,t,d,page,per", WRITES)
def test_write_and_read_back(b, h, t, d, page, per, kind, dtype):
    """Codes and scales from the definition (16-bit elements: exactly its codes), everything else left as it was, then the same rows read back."""
    pages = b * per + 2
    cache = device(make_cache(pages, h, page, d, kind, F32, seed=1))
    before = [None if x is None else x.clone() for x in cache]
    table = random_table(b, per, pages, seed=2)
    room = per * page
    start = torch.randint(0, max(1, room - t // 2), (b,), generator=torch.Generator().manual_seed(3)).int()
    key = randn(b, h, t, d, seed=4, dtype=dtype)
    key[..., 0] *= 30
    value = randn(b, t, h, d, seed=5, dtype=dtype).transpose(1, 2)      # token-major memory
    fca.cache_write(cache, key.cuda(), value.cuda(), table.cuda(), start.cuda())
    for side, x in ((0, key), (1, value)):
        want, scales = before[side].cpu().float().double(), None if before[2] is None else before[2 + side].cpu().double()
        codes, factor = ref_codes(x, kind) if kind in TOP else (x.to(kind).double(), None)
        for i in range(b):
            for j in range(t):
                pos = int(start[i]) + j
                if pos < room:
                    want[table[i, pos // page], :, pos % page] = codes[i, :, j]
                    if scales is not None:
                        scales[table[i, pos // page], :, pos % page] = factor[i, :, j]
        got = cache[side].cpu().float().double()
        if kind in TOP and dtype == F32:
            # fp32's 127 x and its quotient are off by half a step each: only a code within 2^-22 of a tie may be the other one
            step = 1.0 if kind == I8 else 2.0 ** -3
            assert ((got - want).abs() <= step * want.abs().clamp_min(1.0)).all() and (got != want).float().mean() < 1e-3
        else:
            assert torch.equal(got, want)
        if scales is not None:
            assert ((cache[2 + side].cpu().double() - scales).abs() <= 2.0 ** -24 * scales.abs()).all()
    # what the cache holds now, read back at once
    host = KVCache(*(None if x is None else x.cpu() for x in cache))
    n = room + 3
    lengths = torch.randint(0, n + 1, (b, h), generator=torch.Generator().manual_seed(6)).int()
    for out in (F16, BF16, F32):
        got = fca.cache_read(cache, table.cuda(), lengths.cuda(), n, out_dtype=out)
        for g, want in zip(got, values(host, table, n)[:2]):
            live = (torch.arange(n) < lengths[..., None]) & (torch.arange(n) < room)
            want = torch.where(live[..., None], want, 0.0)
            # fp32 product, then the result type: two roundings
            assert ((g.cpu().double() - want).abs() <= want.abs() * (HALF_STEP[out] * 1.001 + 2.0 ** -24) + (2.0 ** -25 if out == F16 else 0.0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_codes_at_ties_and_at_the_ends_of_the_range(kind, dtype):
    """Rows whose quotients are ties, zeros, subnormals, the type's largest, infinities and NaNs."""
    d = 64
    rows = []
    for a in (127.0, 254.0, 448.0, 7.0, 1.0, 3.0, 0.4375, 1.984375):
        r = torch.arange(d) * a / 64
        r[0] = a
        rows.append(r)
    rows += [torch.zeros(d), torch.full((d,), 1.0), -torch.arange(d).float(), torch.arange(d) * 2.0 ** -24, torch.arange(d) * 2.0 ** -20]
    big = torch.finfo(dtype).max
    rows += [torch.linspace(-1, 1, d) * big, torch.linspace(-1, 1, d) * (2.0 ** -130 if dtype == BF16 else 2.0 ** -14)]
    for bad in (math.inf, -math.inf, math.nan):
        r = torch.linspace(-1, 1, d)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows).to(dtype).view(1, 1, -1, d)
    x = torch.cat([x, randn(1, 1, 3000, d, seed=8).mul(4).round().div(4).to(dtype)], 2)     # few values: many ties
    t = x.shape[2]
    cache = KVCache.zeros(1, 1, (t + 15) // 16 * 16, d, kind)
    zero = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    fca.cache_write(cache, x.cuda(), -x.cuda(), zero, zero[0])
    codes, scales = ref_codes(x[0, 0], kind)
    for sign, got, scale in ((1, cache.k, cache.k_scale), (-1, cache.v, cache.v_scale)):
        assert torch.equal(got[0, 0, :t].cpu().float().double(), sign * codes)
        got = scale[0, 0, :t].cpu().double()
        assert torch.equal(got.isnan(), scales.isnan())
        # (a scale under fp32's smallest normal number keeps fewer bits)
        assert ((got - scales).abs()[~scales.isnan()] <= (2.0 ** -24 * scales + 2.0 ** -149)[~scales.isnan()]).all()
    k, _ = fca.cache_read(cache, zero, torch.full((1,), t, dtype=torch.int32, device="cuda"), t, out_dtype=F32)
    assert torch.equal(k[0, 0].isnan().all(-1).cpu(), scales.isnan()) and torch.equal(k[0, 0].isnan().any(-1).cpu(), scales.isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, I8])
def test_write_skips_what_has_no_place(kind):
    """Counts, starts in front of and behind the table, pages that are not there; per head where the lengths are."""
    b, h, t, d, page, per = 3, 2, 40, 32, 16, 4
    cache = device(make_cache(b * per, h, page, d, kind, F32, seed=1))
    before = [None if x is None else x.clone() for x in cache]
    table = torch.arange(b * per).view(b, per).int()
    table[0, 1], table[1, 2], table[2, 0] = -1, b * per, 2 ** 31 - 1
    start = torch.tensor([[0, 50], [-7, 1000], [-2 ** 31, 2 ** 31 - 1]]).int()
    counts = torch.tensor([[40, 20], [40, 40], [40, -1]]).int()
    x = randn(b, h, t, d, seed=4, dtype=BF16)
    fca.cache_write(cache, x.cuda(), x.cuda(), table.cuda(), start.cuda(), counts.cuda())
    codes = ref_codes(x, I8)[0] if kind == I8 else x.double()
    want = before[0].cpu().double()
    for i in range(b):
        for head in range(h):
            for j in range(min(t, int(counts[i, head]))):
                pos = int(start[i, head]) + j
                if 0 <= pos < per * page and 0 <= table[i, pos // page] < b * per:
                    want[table[i, pos // page], head, pos % page] = codes[i, head, j]
    assert torch.equal(cache.k.cpu().double(), want)
    lengths = torch.tensor([per * page, -5, 2 ** 31 - 1]).int()
    k, v = fca.cache_read(cache, table.cuda(), lengths.cuda(), 70, out_dtype=F32)
    host = KVCache(*(None if y is None else y.cpu() for y in cache))
    wk, _, there = values(host, table, 70)
    live = there & (torch.arange(70) < lengths[:, None])
    wk = torch.where(live[:, None, :, None], wk, 0.0)
    assert ((k.cpu().double() - wk).abs() <= wk.abs() * 2.0 ** -23).all()
    assert not k[0, :, 16:32].any() and k[1].abs().sum() == 0 and k[2, :, 16:64].abs().sum() > 0


# cache_keep ----------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("b,h,n,d,page,into_page", [(1, 1, 1, 16, 16, 16), (2, 3, 100, 64, 16, 32), (1, 2, 2929, 128, 16, 16), (3, 2, 513, 80, 48, 16),
                                                    (1, 1, 5000, 32, 64, 128), (2, 2, 2048, 256, 32, 32), (1, 1, 40000, 16, 16, 64)])
def test_keep_copies_the_named_rows_in_order(kind, b, h, n, d, page, into_page):
    per = -(-n // page)
    cache = make_cache(b * per + 1, h, page, d, kind, F32, seed=1)
    table = random_table(b, per, b * per + 1, seed=2)
    if per > 3:
        table[0, 2] = -1                    # a page that is not there
    g = torch.Generator().manual_seed(3)
    keep = torch.rand((b, h, n), generator=g) < torch.rand((b, h, 1), generator=g)
    lengths = torch.randint(n // 2, n + 1, (b, h), generator=g).int()
    lengths[0, 0] = n
    room = max(1, (n // 2) // into_page) * into_page
    into = make_cache(b * (room // into_page), h, into_page, d, kind, F32, seed=9)
    into_table = random_table(b, room // into_page, b * (room // into_page), seed=5)
    after = device(into)
    counts = fca.cache_keep(device(cache), table.cuda(), lengths.cuda(), keep.cuda(), after, into_table.cuda()).cpu()
    there = values(cache, table, n)[2]
    want = [None if x is None else x.clone() for x in into]
    for i in range(b):
        for j in range(h):
            rows = (keep[i, j] & there[i] & (torch.arange(n) < lengths[i, j])).nonzero()[:, 0][:room]
            assert counts[i, j] == len(rows)
            r = torch.arange(len(rows))
            for x, y in zip(want, cache):
                if x is not None:
                    # (8-bit floats as the bytes they are)
                    x, y = (x.view(torch.uint8), y.view(torch.uint8)) if x.dtype == E4M3 else (x, y)
                    x[into_table[i].long()[r // into_page], j, r % into_page] = y[table[i].long()[rows // page], j, rows % page]
    for x, y in zip(after, want):
        if y is not None:
            assert torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, I8])
@pytest.mark.parametrize("n", [70001, 140016])
def test_keep_of_more_rows_than_a_workgroup_lists_at_once(kind, n):
    test_keep_copies_the_named_rows_in_order(kind, 1, 2, n, 16, 16, 32)


@pytest.mark.gpu
def test_keep_of_lengths_inside_and_in_front_of_a_range():
    """Lengths of 0, below 0, inside 16 rows, at their end, and behind the mask."""
    b, h, n, d = 2, 3, 700, 16
    cache = device(make_cache(2 * 44, h, 16, d, F16, F32, seed=1))
    table = torch.arange(88).view(2, 44).int().cuda()
    lengths = torch.tensor([[0, -5, 131], [144, 10 ** 6, 1]]).int().cuda()
    into = KVCache.zeros(88, h, 16, d, F16)
    counts = fca.cache_keep(cache, table, lengths, torch.ones((b, h, n), dtype=torch.bool, device="cuda"), into, table)
    assert counts.tolist() == [[0, 0, 131], [144, 700, 1]]
    want = fca.cache_read(cache, table, counts, n)
    assert all(torch.equal(x, y) for x, y in zip(fca.cache_read(into, table, counts, n), want))
    assert not fca.cache_read(into, table, torch.full_like(lengths, n), n)[0][0, :2].any()


# tree_attention ------------------------------------------------------------------------------------------------------------

KINDS = [(F16, F16), (BF16, BF16), (I8, F16), (I8, BF16), (E4M3, F16), (E4M3, BF16)]
SHAPES = [  # B, H, G, T, N, D, page
    (1, 1, 1, 1, 0, 16, 16), (1, 1, 1, 1, 1, 64, 16), (2, 1, 3, 1, 15, 32, 16), (1, 2, 16, 1, 16, 128, 16), (3, 2, 4, 1, 127, 128, 32),
    (2, 2, 5, 1, 129, 80, 16), (1, 2, 8, 2, 300, 96, 48), (2, 1, 1, 7, 1000, 64, 16), (1, 2, 4, 9, 515, 128, 64), (2, 1, 2, 33, 700, 112, 16),
    (1, 1, 4, 64, 900, 128, 16), (1, 1, 1, 100, 130, 48, 16), (5, 3, 2, 3, 400, 144, 16), (1, 1, 3, 17, 260, 160, 32), (1, 2, 2, 1, 600, 176, 16),
    (2, 1, 4, 5, 333, 192, 16), (1, 1, 6, 11, 200, 208, 16), (1, 1, 2, 40, 350, 240, 16), (1, 2, 4, 13, 777, 256, 16), (1, 1, 4, 1, 9001, 128, 16),
    (300, 1, 2, 1, 40, 64, 16), (2, 4, 4, 1, 4097, 128, 4112)]


def random_tree(b, t, seed):
    g = torch.Generator().manual_seed(seed)
    seen = torch.eye(t, dtype=torch.bool).repeat(b, 1, 1)
    for i in range(b):
        for j in range(1, t):
            parent = int(torch.randint(-1, j, (1,), generator=g))
            if parent >= 0:
                seen[i, j] |= seen[i, parent]
    return seen


def problem(b, h, g, t, n, d, page, kind, dtype, seed=1, spread=0.0):
    per = -(-(n + t) // page)
    cache = make_cache(b * per + 1, h, page, d, kind, dtype, seed, spread)
    table = random_table(b, per, b * per + 1, seed + 5)
    context = torch.randint(n // 2, n + 1, (b,), generator=torch.Generator().manual_seed(seed + 6)).int()
    context[0] = n
    return randn(b, h * g, t, d, seed=seed + 7, dtype=dtype), cache, table, context


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_64_bits(shape, kind, dtype):
    query, cache, table, context = problem(*shape, kind, dtype)
    check_attention(query, cache, table, context, random_tree(shape[0], shape[3], 3) if shape[3] > 2 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("shape", [  # more rows than one tile of every kernel has, and rows either side of where another kernel takes over
    (2, 1, 5, 55, 300, 64, 16), (1, 2, 7, 80, 333, 128, 32), (1, 1, 3, 91, 250, 192, 16), (2, 1, 2, 77, 170, 256, 16), (1, 1, 1, 48, 200, 64, 16),
    (1, 2, 7, 7, 200, 128, 16), (1, 1, 1, 129, 150, 96, 16), (1, 2, 4, 4, 300, 176, 16), (3, 1, 17, 1, 210, 256, 16), (1, 1, 128, 1, 100, 32, 16)])
def test_attention_of_many_rows(shape, kind, dtype):
    query, cache, table, context = problem(*shape, kind, dtype)
    check_attention(query, cache, table, context, random_tree(shape[0], shape[3], 3) if shape[3] % 2 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(F16, F16), (I8, BF16)])
@pytest.mark.parametrize("shape", [(1, 64, 1, 1, 16400, 16, 16), (2, 16, 1, 32, 8200, 32, 16), (2, 16, 1, 300, 2000, 32, 16)])
def test_attention_of_many_blocks_per_workgroup(shape, kind, dtype):
    """Enough blocks for pieces of one item each, of equal lengths and, with one short sequence, of lengths that leave none."""
    query, cache, table, context = problem(*shape, kind, dtype)
    context[:] = shape[4]
    check_attention(query, cache, table, context)
    context = of_heads(context, shape[1]).clone()
    context[0, ::3] //= 5
    check_attention(query, cache, table, context)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(BF16, BF16), (I8, F16)])
@pytest.mark.parametrize("b,h,t,g", [(700, 2, 1, 2), (530, 1, 33, 2)])
def test_attention_of_more_sequences_than_threads(kind, dtype, b, h, t, g):
    """Lengths per sequence and per head, among them zeros, for more of them than a workgroup has threads."""
    query, cache, table, context = problem(b, h, g, t, 20, 32, 16, kind, dtype)
    check_attention(query, cache, table, context)
    heads = torch.randint(0, 21, (b, h), generator=torch.Generator().manual_seed(9)).int()
    heads[1], heads[-1] = 0, 20
    check_attention(query, cache, table, heads)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_attention_of_a_chain_a_shared_mask_and_any_mask(kind, dtype):
    """The same drafted tokens with no mask, one mask for all sequences, and masks that hide tokens from themselves; heads of own lengths."""
    b, h, g, t, n, d = 3, 2, 2, 9, 150, 64
    query, cache, table, context = problem(b, h, g, t, n, d, 16, kind, dtype)
    context = torch.tensor([[150, 3], [0, 77], [16, 128]]).int()
    check_attention(query, cache, table, context)
    check_attention(query, cache, table, context, random_tree(1, t, 5)[0], scale=0.7)
    mask = torch.rand((b, t, t), generator=torch.Generator().manual_seed(3)) < 0.4
    check_attention(query, cache, table, context, mask, scale=-0.2)
    check_attention(query, cache, table, context, mask, scale=0.0)
    check_attention(query, cache, table, context, mask, tree_lengths=torch.tensor([9, 0, 4]).int())
    check_attention(query, cache, table, context, None, tree_lengths=torch.tensor([-3, 100, 1]).int())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_rows_that_see_nothing(kind, dtype):
    query, cache, table, _ = problem(2, 2, 3, 5, 60, 64, 16, kind, dtype)
    mask = torch.eye(5, dtype=torch.bool)
    mask[2] = False
    got, lse = check_attention(query, cache, table, torch.tensor([0, 7]).int(), mask)
    assert not got[0, :, 2].any() and lse[0, :, 2].isneginf().all() and lse[1].isfinite().all()
    got, lse = check_attention(query, cache, torch.full_like(table, -1), torch.tensor([50, 7]).int(), mask)
    assert not got.any() and lse.isneginf().all()
    check_attention(query, cache, table, torch.tensor([-2 ** 31, 2 ** 31 - 1]).int(), mask)     # nothing; more than the table names


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("t,d", [(6, 64), (20, 128), (3, 256)])
def test_what_hidden_rows_hold_has_no_influence(kind, dtype, t, d):
    """NaNs, infinities and NaN scales behind the last key, on pages that are not there, and in drafted tokens that some rows do not see."""
    b, h, g, n = 2, 2, 2, 75
    query, cache, table, context = problem(b, h, g, t, n, d, 16, kind, dtype)
    table = torch.cat([table, random_table(b, 2, 40, 77)], 1)
    table[1, 1] = -1
    mask = random_tree(b, t, 3)
    tree = torch.tensor([t, t - 1]).int()
    table = torch.arange(b * table.shape[1]).view(b, -1).int()
    cache = make_cache(b * table.shape[1] + 1, h, 16, d, kind, dtype, seed=4)
    table[1, 1] = -1
    want = ref_attention(query, cache, table, context, mask, None, tree)
    poisoned = [None if x is None else x.clone() for x in cache]
    if kind == I8:
        poisoned[0].fill_(-128), poisoned[1].fill_(-128)
        poisoned[2].fill_(math.nan), poisoned[3].fill_(math.inf)
    elif kind == E4M3:
        poisoned[0].view(torch.uint8).fill_(0x7f), poisoned[1].view(torch.uint8).fill_(0xff)
        poisoned[2].fill_(math.nan), poisoned[3].fill_(math.nan)
    else:
        poisoned[0].fill_(math.nan), poisoned[1].fill_(math.inf)
    for i in range(b):
        for j in range(int(context[i]) + int(tree[i])):
            page = int(table[i, j // 16])
            if page >= 0:
                for x, y in zip(poisoned, cache):
                    if x is not None:
                        x, y = (x.view(torch.uint8), y.view(torch.uint8)) if x.dtype == E4M3 else (x, y)
                        x[page, :, j % 16] = y[page, :, j % 16]
    poisoned = KVCache(*poisoned)
    got, lse = fca.tree_attention(query.cuda(), device(poisoned), table.cuda(), context.cuda(), mask.cuda(), tree_lengths=tree.cuda(),
                                  return_lse2=True)
    compare_attention(got, lse, want)
    # a drafted token that is not finite reaches the rows that see it, and those only
    j = int(context[0]) + t // 2
    page = int(table[0, j // 16])
    if kind in TOP:
        poisoned.k_scale[page, 0, j % 16] = math.nan
        poisoned.v_scale[page, 1, j % 16] = math.nan
    else:
        poisoned.k[page, 0, j % 16, 3] = math.nan
        poisoned.v[page, 1, j % 16, 5] = math.inf
        poisoned.v[page, 1, j % 16, 6] = math.nan
    got, lse = (x.cpu() for x in fca.tree_attention(query.cuda(), device(poisoned), table.cuda(), context.cuda(), mask.cuda(),
                                                    tree_lengths=tree.cuda(), return_lse2=True))
    sees = mask[0, :, t // 2]
    assert sees.any() and not sees.all()
    assert got[0, :g, sees].isnan().all() and lse[0, :g, sees].isnan().all()
    values_bad = got[0, g:, sees]
    if kind in TOP:
        assert values_bad.isnan().all()
    else:
        assert values_bad[..., 5].isinf().all() and values_bad[..., 6].isnan().all() and values_bad[..., :5].isfinite().all()
    got[0, :, sees], lse[0, :, sees] = want[0].to(got.dtype)[0, :, sees], want[1].float()[0, :, sees]
    compare_attention(got, lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t,d", [(5, 64), (14, 96), (30, 128), (5, 256), (60, 192)])
def test_codes_that_are_nans_reach_the_rows_that_see_them_only(dtype, t, d):
    """cache_write makes no such codes; a cache that is filled otherwise may have them."""
    b, h, g, n = 2, 2, 2, 75
    query, cache, table, context = problem(b, h, g, t, n, d, 16, E4M3, dtype)
    mask = random_tree(b, t, 3)
    want = ref_attention(query, cache, table, context, mask, None, None)
    j = int(context[0]) + t // 2
    page = int(table[0, j // 16])
    cache.v.view(torch.uint8)[page, 1, j % 16, d - 1] = 0xff
    cache.k.view(torch.uint8)[page, 0, j % 16, 3] = 0x7f
    got, lse = (x.cpu() for x in fca.tree_attention(query.cuda(), device(cache), table.cuda(), context.cuda(), mask.cuda(), return_lse2=True))
    sees = mask[0, :, t // 2]
    assert sees.any() and not sees.all()
    assert got[0, :g, sees].isnan().all() and got[0, g:, sees, d - 1].isnan().all()
    got[0, :, sees], lse[0, :, sees] = want[0].to(got.dtype)[0, :, sees], want[1].float()[0, :, sees]
    compare_attention(got, lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t", [1, 12])
def test_scales_and_scores_far_apart(kind, dtype, t):
    """Values whose rows differ by 2^20 and more either way, scores from -500 to 500, keys that only a late block's rows prefer."""
    b, h, g, n, d = 2, 1, 3, 700, 64
    query, cache, table, context = problem(b, h, g, t, n, d, 16, kind, dtype, spread=8.0)
    check_attention(query, cache, table, context)
    check_attention((query.float() * 30).to(dtype), cache, table, context)
    # the first blocks have the largest values and the smallest scores, the last ones the other way round
    by = torch.linspace(20, -20, table.shape[1])
    for i in range(b):
        for j in range(table.shape[1]):
            cache.v_scale[int(table[i, j])] = 2.0 ** float(by[j])
            cache.k_scale[int(table[i, j])] = 2.0 ** float(by[j] / -5 - 6)
    check_attention((query.float().abs() * 2).to(dtype), cache, table, context)
    cache.v_scale.zero_()
    check_attention(query, cache, table, context)
    if dtype == BF16:       # queries far outside fp16
        check_attention((query.float() * 2.0 ** 60).to(dtype), cache, table, context, scale=2.0 ** -63)
        check_attention((query.float() * 2.0 ** -100).to(dtype), cache, table, context, scale=2.0 ** 97)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("t,d", [(1, 64), (2, 256), (60, 128), (40, 192)])
def test_scores_whose_last_bit_is_above_one(kind, dtype, t, d):
    """Scores of 2^24 to 2^90, where fp32 has no fractions: one key has all the weight, and nothing overflows."""
    query, cache, table, context = problem(2, 2, 2, t, 400, d, 16, kind, dtype)
    for scale in (2.0 ** 24, -2.0 ** 40, 2.0 ** 90):
        check_attention(query, cache, table, context, scale=scale)
        check_attention(query, cache, table, context, random_tree(2, t, 3), scale=scale, tree_lengths=torch.tensor([t, t - 1]).int())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("t,g", [(1, 4), (3, 5), (40, 4), (90, 3)])
def test_query_rows_far_apart(kind, t, g):
    """bf16 rows whose magnitudes differ by 2^80, rows of zeros and rows that are not finite, side by side: each has its own result."""
    b, h, n, d = 2, 2, 300, 64
    query, cache, table, context = problem(b, h, g, t, n, d, 16, kind, BF16)
    power = torch.randint(-80, 1, (b, h * g, t, 1), generator=torch.Generator().manual_seed(4)).double()
    power[:, 0, 0] = 0
    far = (query.double() * 2.0 ** power).to(BF16)
    check_attention(far, cache, table, context)
    check_attention(far, cache, table, context, scale=2.0 ** 40)
    far[0, 0, 0] = 0
    check_attention(far, cache, table, context)
    bad = far.clone()
    bad[0, 1, 0, 3] = math.nan
    bad[1, h * g - 1, t - 1, 5] = math.inf
    want = list(ref_attention(far, cache, table, context, None, None, None))
    got, lse = (x.cpu() for x in fca.tree_attention(bad.cuda(), device(cache), table.cuda(), context.cuda(), return_lse2=True))
    for at in ((0, 1, 0), (1, h * g - 1, t - 1)):
        assert got[at].isnan().all() and not lse[at].isfinite()
        got[at], lse[at] = want[0].to(BF16)[at], want[1].float()[at]
    compare_attention(got, lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(F16, F16), (BF16, BF16), (I8, BF16), (E4M3, F16)])
def test_layouts(kind, dtype):
    """Keys and values of one allocation, token-major pages, token-major and expanded queries, tables and lengths that are views."""
    b, h, g, t, n, d, page = 2, 3, 2, 5, 200, 64, 16
    query, cache, table, context = problem(b, h, g, t, n, d, page, kind, dtype)
    pages = cache.k.shape[0]
    both = torch.zeros((pages, 2, page, h + 1, d), dtype=torch.uint8 if kind == E4M3 else kind, device="cuda")
    if kind == E4M3:
        both = both.view(E4M3)
    k, v = both[:, 0, :, :h].transpose(1, 2), both[:, 1, :, 1:].transpose(1, 2)
    k.copy_(cache.k.cuda()), v.copy_(cache.v.cuda())
    scales = [None, None]
    if kind in TOP:
        room = torch.zeros((pages, 2, h, page), device="cuda")
        scales = [room[:, 0], room[:, 1]]
        scales[0].copy_(cache.k_scale), scales[1].copy_(cache.v_scale)
    view = KVCache(k, v, *scales)
    wide = torch.full((b, table.shape[1] + 3), -1, dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    some = torch.stack([context, context * 0], 1).cuda()[:, 0]
    major = query.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    ref = ref_attention(query, cache, table, context, None, None, None)
    got, lse = fca.tree_attention(major, view, wide.cuda()[:, : table.shape[1]], some, return_lse2=True)
    compare_attention(got, lse, ref)
    one = query[:, :, :1].expand(b, h * g, t, d)
    got, lse = fca.tree_attention(one.cuda()[:, :, :1].expand(b, h * g, t, d), view, table.cuda(), context.cuda()[:, None].expand(b, h), return_lse2=True)
    compare_attention(got, lse, ref_attention(one, cache, table, context, None, None, None))
    odd = torch.zeros(b * h * g * t * d + 1, dtype=dtype, device="cuda")[1:].view(b, h * g, t, d)     # starts off 16 bytes
    odd.copy_(query)
    got, lse = fca.tree_attention(odd, view, table.cuda(), context.cuda(), return_lse2=True)
    compare_attention(got, lse, ref)
    x = randn(b, h, t, d, seed=9, dtype=dtype)
    fca.cache_write(view, x.cuda(), x.cuda(), table.cuda(), context.cuda())
    fca.cache_write(device(cache), x.cuda(), x.cuda(), table.cuda(), context.cuda())
    plain = device(cache)
    fca.cache_write(plain, x.cuda(), x.cuda(), table.cuda(), context.cuda())
    for a, z in zip(view, plain):
        if a is not None:
            assert torch.equal(a.float(), z.float())
    assert not both[:, 0, :, h].float().any() and not both[:, 1, :, 0].float().any()
    for a, z in zip(fca.cache_read(view, table.cuda(), context.cuda(), n), fca.cache_read(plain, table.cuda(), context.cuda(), n)):
        assert torch.equal(a, z)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, I8])
def test_offsets_past_32_bits(kind):
    """Pages beyond 4 GiB of a pool, bf16, and beyond 2^32 elements, codes."""
    h, page, d = 4, 256, 256
    pages = (5 << 30) // (h * page * d * kind.itemsize)
    pool = [torch.zeros((pages, h, page, d), dtype=kind, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, h, page), device="cuda") for _ in range(2)] if kind in TOP else []
    cache = KVCache(*pool, *scales)
    n, t = 600, 3
    table = torch.tensor([[pages - 1, 0, pages - 7]]).int()
    x = [randn(1, h, n + t, d, seed=i, dtype=BF16) for i in (1, 2)]
    zero = torch.zeros(1, dtype=torch.int32)
    fca.cache_write(cache, x[0].cuda(), x[1].cuda(), table.cuda(), zero.cuda())
    small = KVCache(*(None if p is None else p[[pages - 1, 0, pages - 7]].cpu() for p in cache))
    to = torch.arange(3).view(1, 3).int()
    query = randn(1, 2 * h, t, d, seed=3, dtype=BF16)
    context = torch.full((1,), n, dtype=torch.int32)
    got, lse = fca.tree_attention(query.cuda(), cache, table.cuda(), context.cuda(), return_lse2=True)
    compare_attention(got, lse, ref_attention(query, small, to, context, None, None, None))
    k, v = fca.cache_read(cache, table.cuda(), context.cuda(), n, out_dtype=F32)
    wk, wv, _ = values(small, to, n)
    assert ((k.cpu() - wk).abs() <= wk.abs() * 2.0 ** -23).all() and ((v.cpu() - wv).abs() <= wv.abs() * 2.0 ** -23).all()
    assert wk.abs().amax((-1, -2)).min() > 1
    keep = torch.ones((1, h, n), dtype=torch.bool, device="cuda")
    into = torch.tensor([[pages - 3, 1, pages - 2]]).int()
    fca.cache_keep(cache, table.cuda(), context.cuda(), keep, cache, into.cuda())
    for a, z in zip(fca.cache_read(cache, into.cuda(), context.cuda(), n, out_dtype=F32), (k, v)):
        assert torch.equal(a, z)


@pytest.mark.gpu
def test_streams_graphs_and_repetition():
    """On a side stream and replayed from a graph with eager calls in between, every result is that of the first call, bit for bit."""
    b, h, g, t, n, d = 3, 2, 4, 5, 900, 64
    query, cache, table, context = problem(b, h, g, t, n, d, 16, I8, BF16)
    query, cache, table, context = query.cuda(), device(cache), table.cuda(), context.cuda()
    mask = random_tree(b, t, 3).cuda()
    x = randn(b, h, t, d, seed=9, dtype=BF16).cuda()
    into = KVCache.zeros(cache.k.shape[0], h, 16, d, I8)
    into_table = torch.arange(table.numel(), device="cuda").view(b, -1).int()
    keep = torch.rand((b, h, n), generator=torch.Generator().manual_seed(3)).cuda() < 0.3

    def step():
        fca.cache_write(cache, x, x, table, context)
        out, lse = fca.tree_attention(query, cache, table, context, mask, return_lse2=True)
        counts = fca.cache_keep(cache, table, context, keep, into, into_table)
        again = fca.tree_attention(query, into, into_table, counts, mask)
        return out, lse, counts, again, *fca.cache_read(cache, table, context, n)

    want = [y.clone() for y in step()]
    for _ in range(3):
        assert all(torch.equal(a, z) for a, z in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, z) for a, z in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        for y in held:
            y.zero_()
        graph.replay()
        assert all(torch.equal(a, z) for a, z in zip(held, want)), i
        assert all(torch.equal(a, z) for a, z in zip(step(), want)), i
        torch.cuda.synchronize()
    # the lengths are read by the replay, not by the capture
    context -= 100
    want = [y.clone() for y in step()]
    graph.replay()
    assert all(torch.equal(a, z) for a, z in zip(held, want))


@pytest.mark.gpu
def test_two_graphs_of_one_pool_and_two_streams():
    """Graphs whose workspaces share memory, replayed in turn, and calls on two streams at once."""
    few = problem(2, 2, 4, 3, 3000, 64, 16, I8, BF16)
    many = problem(2, 2, 4, 70, 2000, 128, 16, BF16, BF16, seed=5)
    calls = []
    for query, cache, table, context in (few, many):
        query, cache, table, context = query.cuda(), device(cache), table.cuda(), context.cuda()
        calls.append(lambda q=query, c=cache, t=table, n=context: fca.tree_attention(q, c, t, n, return_lse2=True))
    want = [[y.clone() for y in c()] for c in calls]
    torch.cuda.synchronize()
    graphs, held = [], []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            held.append(c())
        graphs.append(graph)
    for i in range(3):
        for graph, got, w, c in zip(graphs, held, want, calls):
            graph.replay()
            assert all(torch.equal(a, z) for a, z in zip(got, w)), i
            assert all(torch.equal(a, z) for a, z in zip(c(), w)), i
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for k, (stream, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(stream):
                got[k].append(c())
    torch.cuda.synchronize()
    for k, w in enumerate(want):
        assert all(torch.equal(a, z) for g in got[k] for a, z in zip(g, w))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, I8, E4M3])
def test_prune_then_decode(kind):
    """The whole path: a prompt is written, its keys scored by the column reduction and pruned per head, drafted tokens are
    written behind the kept rows and attend to them."""
    b, h, g, n, d, kept, t = 2, 3, 2, 500, 64, 120, 4
    cache = KVCache.zeros(b * 32, h, 16, d, kind)
    table = torch.randperm(b * 32, generator=torch.Generator().manual_seed(1)).view(b, 32).int().cuda()
    key, value = (randn(b, h, n, d, seed=i, dtype=BF16).cuda() for i in (1, 2))
    length = torch.full((b,), n, dtype=torch.int32, device="cuda")
    fca.cache_write(cache, key, value, table, torch.zeros_like(length))
    k, v = fca.cache_read(cache, table, length, n)
    window = randn(b, h, 32, d, seed=3, dtype=BF16).cuda()
    keep = fca.topk_keep_mask(fca.flash_colreduce(window, k, "sum", True), kept)
    pruned = KVCache.zeros(b * 8, h, 16, d, kind)
    pruned_table = torch.arange(b * 8, device="cuda").view(b, 8).int()
    counts = fca.cache_keep(cache, table, length, keep, pruned, pruned_table)
    assert (counts == kept).all()
    new_k, new_v, query = (randn(b, heads, t, d, seed=i, dtype=BF16).cuda() for i, heads in ((4, h), (5, h), (6, h * g)))
    fca.cache_write(pruned, new_k, new_v, pruned_table, counts)
    mask = random_tree(b, t, 7).cuda()
    out, lse = fca.tree_attention(query, pruned, pruned_table, counts, mask, return_lse2=True)
    host = KVCache(*(None if x is None else x.cpu() for x in pruned))
    compare_attention(out, lse, ref_attention(query.cpu(), host, pruned_table.cpu(), counts.cpu(), mask.cpu(), None, None))
    # the rows behind are the ones that the mask named
    pk, pv = fca.cache_read(pruned, pruned_table, counts, kept)
    assert torch.equal(pk, k[keep].view(b, h, kept, d)) and torch.equal(pv, v[keep].view(b, h, kept, d))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F16, BF16, I8, E4M3])
def test_native_host_path_gives_what_the_general_one_gives(kind, monkeypatch):
    """The native path answers the usual calls, leaves the others to Python, and both run the same kernels."""
    b, h, g, t, n, d = 2, 3, 2, 5, 150, 64
    dtype = kind if kind in (F16, BF16) else BF16
    query, cache, table, context = problem(b, h, g, t, n, d, 16, kind, dtype)
    query, cache, table, context = query.cuda(), device(cache), table.cuda(), context.cuda()
    by_head = context[:, None].repeat(1, h)
    x = randn(b, h, t, d, seed=9, dtype=dtype).cuda()
    mask, lengths = random_tree(b, t, 3).cuda(), torch.tensor([t, 2], dtype=torch.int32, device="cuda")
    keep = torch.rand((b, h, n), generator=torch.Generator().manual_seed(3)).cuda() < 0.3
    into_table = torch.arange(table.numel(), device="cuda").view(b, -1).int()

    def run():
        into = KVCache.zeros(cache.k.shape[0], h, 16, d, kind)
        fca.cache_write(cache, x, x, table, context)
        got = [fca.tree_attention(query, cache, table, context), *fca.tree_attention(query, cache, table, by_head, mask, 0.3, return_lse2=True),
               fca.tree_attention(query, cache, table, context, mask[0], tree_lengths=lengths), fca.cache_keep(cache, table, by_head, keep, into, into_table),
               *fca.cache_read(cache, table, context, n), *fca.cache_read(cache, table, by_head, n + 7, out_dtype=F32), *into]
        fca.cache_write(cache, x * 2, x, table, by_head, counts=lengths)
        got += fca.cache_read(cache, table, context + t, n + t)
        # what the native path leaves to Python
        strided = x.transpose(2, 3).contiguous().transpose(2, 3)
        fca.cache_write(cache, strided, x, table, context)
        got += [fca.tree_attention(query, cache, table, context, mask.transpose(1, 2).contiguous().transpose(1, 2), 1),
                fca.cache_keep(cache, table, context, keep.transpose(0, 1).contiguous().transpose(0, 1), into, into_table)]
        return [None if y is None else y.float() if y.dtype == E4M3 else y for y in got]

    native = run()
    host = cache_module._host()
    assert host.cache_write(cache, x, x, table, context, None) is True and host.cache_read(cache, table, context, n, None) is not None
    assert host.tree_attention(query, cache, table, context, None, None, None, False) is not None
    assert host.cache_keep(cache, table, context, keep, KVCache.zeros(cache.k.shape[0], h, 16, d, kind), into_table) is not None
    assert host.tree_attention(query, cache, table, context, None, 1, None, False) is None
    monkeypatch.setattr(cache_module.flash, "_native", _lib._PythonOnly)
    for a, z in zip(run(), native):
        assert (a is None and z is None) or torch.equal(a, z)


@pytest.mark.gpu
def test_rows_whose_elements_are_apart_are_refused():
    cache = KVCache.zeros(4, 2, 16, 32, BF16)
    apart = KVCache(cache.k.transpose(2, 3).contiguous().transpose(2, 3), cache.v)
    table, lengths = torch.arange(4, device="cuda").view(2, 2).int(), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (apart, KVCache(apart[1], apart[0])):
        with pytest.raises(ValueError, match="consecutive"):
            fca.cache_read(bad, table, lengths, 3)


@pytest.mark.gpu
def test_python_refusals_on_the_device():
    b, h, d = 2, 2, 32
    cache = KVCache.zeros(4, h, 16, d, I8)
    table = torch.arange(4, device="cuda").view(b, 2).int()
    lengths = torch.zeros(b, dtype=torch.int32, device="cuda")
    x = torch.zeros(b, h, 3, d, device="cuda", dtype=F16)
    q = torch.zeros(b, 2 * h, 3, d, device="cuda", dtype=F16)
    keep = torch.zeros(b, h, 20, device="cuda", dtype=torch.bool)
    into = KVCache.zeros(4, h, 16, d, I8)
    bad = [lambda: fca.cache_write(cache, x[:, :1], x, table, lengths), lambda: fca.cache_write(cache, x.double(), x.double(), table, lengths),
           lambda: fca.cache_write(cache, x, x.float(), table, lengths), lambda: fca.cache_write(cache, x, x, table.long(), lengths),
           lambda: fca.cache_write(cache, x, x, table[:1], lengths), lambda: fca.cache_write(cache, x, x, table, lengths.long()),
           lambda: fca.cache_write(cache, x, x, table, lengths[:1]), lambda: fca.cache_write(cache, x, x, table, lengths, lengths.cpu()),
           lambda: fca.cache_write(cache._replace(k_scale=None), x, x, table, lengths), lambda: fca.cache_write(cache, x, x, table.t(), lengths),
           lambda: fca.cache_write(KVCache(cache.k.half(), cache.v.half(), cache.k_scale, cache.v_scale), x, x, table, lengths),
           lambda: fca.cache_read(cache, table, lengths, -1), lambda: fca.cache_read(cache, table, lengths, 3, out_dtype=I8),
           lambda: fca.cache_read(cache, table[0], lengths, 3), lambda: fca.cache_read(KVCache(cache.k[..., :24], cache.v[..., :24], *cache[2:]), table, lengths, 3),
           lambda: fca.cache_keep(cache, table, lengths, keep.int(), into, table), lambda: fca.cache_keep(cache, table, lengths, keep[:, :1], into, table),
           lambda: fca.cache_keep(cache, table, lengths, keep, cache, table), lambda: fca.cache_keep(cache, table, lengths, keep, KVCache.zeros(4, h, 16, d, E4M3), table),
           lambda: fca.cache_keep(cache, table, lengths, keep, KVCache.zeros(4, h, 16, 2 * d, I8), table),
           lambda: fca.tree_attention(q[:, :3], cache, table, lengths), lambda: fca.tree_attention(q.float(), cache, table, lengths),
           lambda: fca.tree_attention(q, KVCache.zeros(4, h, 16, d, BF16), table, lengths), lambda: fca.tree_attention(q[..., :16], cache, table, lengths),
           lambda: fca.tree_attention(q, cache, table, lengths, torch.ones(3, 4, device="cuda", dtype=torch.bool)),
           lambda: fca.tree_attention(q, cache, table, lengths, torch.ones(3, 3, device="cuda")),
           lambda: fca.tree_attention(q, cache, table, lengths, tree_lengths=lengths.long()), lambda: fca.tree_attention(q.cpu(), cache, table, lengths)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
    with pytest.raises(_lib.FcrError, match="scale must be finite"):
        fca.tree_attention(q, cache, table, lengths, scale=math.nan)
    with pytest.raises(_lib.FcrError, match="16 bytes"):     # rows of pages that start off 16 bytes
        odd = torch.zeros(4 * h * 16 * d + 8, device="cuda", dtype=I8)[8:].view(4, h, 16, d)
        fca.cache_read(KVCache(odd, odd, *cache[2:]), table, lengths, 3)
    # nothing to do
    fca.cache_write(cache, x[:, :, :0], x[:, :, :0], table, lengths)
    fca.cache_write(cache, x, x, table[:, :0], lengths)
    assert fca.cache_read(cache, table, lengths, 0)[0].shape == (b, h, 0, d)
    assert not fca.cache_read(cache, table[:, :0], lengths, 5)[1].any()
    assert not fca.cache_keep(cache, table, lengths, keep[..., :0], into, table).any()
    out, lse = fca.tree_attention(q, cache, table[:, :0], lengths, return_lse2=True)
    assert not out.any() and lse.isneginf().all()
    assert fca.tree_attention(q[:, :, :0], cache, table, lengths).shape == (b, 2 * h, 0, d)
    assert fca.tree_attention(q[:0], cache, table[:0], lengths[:0]).shape == (0, 2 * h, 3, d)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("t,d", [(1, 16), (3, 48), (2, 80), (33, 96), (60, 112), (1, 176), (40, 240), (2, 64), (70, 128)])
def test_keys_of_infinite_elements_that_are_seen(kind, t, d):
    """A score of minus infinity is no weight, wherever in its row the element lies that makes it one; a row that sees no other score is zeros."""
    query, cache, table, context = problem(2, 2, 2, t, 150, d, 16, kind, kind)
    elements = (0, d // 2, d - 8, d - 1)
    query[..., elements] = query[..., elements].abs() + 0.25
    for i in range(2):
        n = int(context[i])
        for j, e in zip((3, 17, 40, n - 1, n, n + t - 1), (*elements, d - 1, d - 5)):
            cache.k[int(table[i, j // 16]), :, j % 16, e] = -math.inf
    query[..., d - 5] = query[..., d - 5].abs() + 0.25
    check_attention(query, cache, table, context)
    check_attention(query, cache, table, context, random_tree(2, t, 3))
    for page in table[:, 0].tolist():
        cache.k[page, :, :, d - 1] = -math.inf
    check_attention(query, cache, table, torch.tensor([5, 8]).int(), tree_lengths=torch.tensor([min(t, 9), min(t, 4)]).int())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t,d", [(1, 64), (5, 64), (20, 80), (14, 96), (30, 128), (60, 128), (60, 192), (5, 256), (40, 256)])
def test_value_codes_that_are_nans_reach_their_own_element_only(dtype, t, d):
    """Far in front of the drafted tokens, next to them, and among them: the rows that see the code have a NaN where it is, and nowhere else."""
    query, cache, table, context = problem(2, 2, 2, t, 75, d, 16, E4M3, dtype)
    codes = cache.v.view(torch.uint8)
    for i, head, j, e, code in ((0, 0, 74, d - 1, 0x7f), (0, 1, 75 + t // 2, 1, 0xff), (1, 0, 3, d // 2, 0xff), (1, 1, int(context[1]), 0, 0x7f),
                                (1, 1, int(context[1]) - 1, d - 2, 0xff)):
        codes[int(table[i, j // 16]), head, j % 16, e] = code
    check_attention(query, cache, table, context, random_tree(2, t, 3))
    check_attention(query, cache, table, context, tree_lengths=torch.tensor([t, t // 2]).int())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("t,d", [(1, 64), (60, 64)])
@pytest.mark.parametrize("share", [2.0 ** -7, 2.0 ** -10])
def test_many_small_weights_next_to_large_ones(kind, dtype, t, d, share):
    """Four keys have nearly all the weight and one element of value; what the others, 65536 of them, share between them is all of the other elements.

    A row's largest weight is above 2^8 where it is rounded to fp16, so that half of fp16's smallest step, 2^-25, is 2^-33 of it.  Sequences share
    their pages; as many as there are workgroups, so that hardly a sequence is cut and the others are added to the same sums as the four."""
    b, n = 2 * torch.cuda.get_device_properties(0).multi_processor_count, 65540
    pages = -(-(n + t) // 16)
    x = randn(pages * 16, seed=1) * 0.5
    top = math.log(65536 * math.exp(0.125) / (4 * share))
    key, value = torch.zeros(pages * 16, d), torch.rand((pages * 16, d), generator=torch.Generator().manual_seed(2)) / 2 + 0.5
    key[:, 1], value[:, 0], value[:, 1] = x, 0.0, 1.0
    for j in (0, 32, 64, 96):
        key[j, 0], key[j, 1] = top, 0.0
        value[j], value[j, 0] = 0.0, 1.0
    rows = [r.view(pages, 1, 16, d) for r in (key, value)]
    if kind in TOP:
        codes = [ref_codes(r, kind) for r in rows]
        cache = KVCache(*(c.to(F32).to(kind) for c, _ in codes), *(s.float() for _, s in codes))
    else:
        cache = KVCache(*(r.to(kind) for r in rows))
    query = torch.zeros(1, 1, t, d, dtype=dtype)
    query[..., :2] = 1
    table, context = torch.arange(pages).view(1, -1).int(), torch.full((1,), n, dtype=torch.int32)
    want, want_lse, _, tol_lse = ref_attention(query, cache, table, context, None, 1.0, None)
    got, lse = fca.tree_attention(query.cuda().expand(b, 1, t, d), device(cache), table.cuda().expand(b, -1), context.cuda().expand(b), None, 1.0,
                                  return_lse2=True)
    ds = (d + 8) * 2.0 ** -24 * top + 2.0 ** -21                # (of a score, as in ref_attention)
    tol = want * ((HALF_STEP[BF16] if kind == BF16 else HALF_STEP[F16]) + 2 * ds + 1.01 * HALF_STEP[dtype]) + 2.0 ** -25
    if kind != BF16:
        tol = tol + (n + t) * 2.0 ** -33 / 4
    assert (tol[..., 1:] < (2.0 ** -6 if BF16 in (kind, dtype) else 2.0 ** -7) * want[..., 1:]).all()
    assert ((got.cpu().double() - want).abs() <= tol).all(), ((got.cpu().double() - want).abs() / tol).max()
    assert ((lse.cpu().double() - want_lse).abs() <= tol_lse).all()


OVERLAPS = [dict(k_strides=(16384, 0, 64)), dict(v_strides=(0, 2048, 64)), dict(k_strides=(16384, 1024, 64)), dict(v_strides=(8192, 2048, 64)),
            dict(k_strides=(64, 256, 1024)), dict(k_scale_strides=(256, 0, 1)), dict(v_scale_strides=(0, 32, 1)), dict(v_scale_strides=(128, 32, 1)),
            dict(k=1 << 20), dict(k=(1 << 20) + 32), dict(v_scale=1 << 28),
            dict(k_strides=(32768, 64, 1024), v_strides=(32768, 64, 1024), k=(1 << 20) + 64 * 7)]


@pytest.mark.parametrize("fn", ["write", "keep"])
@pytest.mark.parametrize("over", OVERLAPS, ids=str)
def test_caches_whose_rows_share_memory_are_not_written(fn, over):
    """Pages, heads or rows that lie in one another, keys among values."""
    cache = _c_cache(**{**dict(v=1 << 20, k=1 << 24, k_scale=1 << 28, v_scale=1 << 21), **over})
    assert (_c_call("write", cache) if fn == "write" else _c_call("keep", _c_cache(), into=cache)) == -4
    assert b"share memory" in _lib.load().fcr_last_error()


def test_rows_that_lie_apart(tmp_path):
    """csrc/apart.h against the elements themselves: every slice and transpose of a small tensor is apart, whatever overlaps is not."""
    (tmp_path / "a.cpp").write_text(
        '#include "apart.h"\n'
        'extern "C" int one(int64_t row, const int64_t* d, int n) { return fcr_paged::rows_apart(row, (const fcr_paged::Dimension*)d, n); }\n'
        'extern "C" int two(int64_t row, const int64_t* x, int64_t xa, const int64_t* y, int64_t ya, int n, int bytes) {\n'
        '  return fcr_paged::rows_apart(row, (const fcr_paged::Dimension*)x, xa, (const fcr_paged::Dimension*)y, ya, n, bytes); }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "flash_colreduce_amd", "csrc"),
                    str(tmp_path / "a.cpp"), "-o", str(tmp_path / "a.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "a.so"))
    i64 = ctypes.c_int64

    def dims(sizes, strides):
        return (i64 * 6)(*(x for pair in zip(sizes, strides) for x in pair))

    def elements(at, row, sizes, strides):
        return [at + a * strides[0] + b * strides[1] + c * strides[2] + e
                for a in range(sizes[0]) for b in range(sizes[1]) for c in range(sizes[2]) for e in range(row)]

    rng = random.Random(5)
    for _ in range(3000):
        sizes, row = [rng.randint(1, 4) for _ in range(3)], rng.randint(1, 3)
        if rng.random() < 0.5:
            strides = [rng.randint(0, 30) for _ in range(3)]
        else:              # a tensor with room between its rows, its dimensions in any order
            span, strides = row + rng.randint(0, 1), [0] * 3
            for i in rng.sample(range(3), 3):
                strides[i] = span
                span *= sizes[i] + rng.randint(0, 1)
            assert lib.one(i64(row), dims(sizes, strides), 3) == 1
        x, z = elements(0, row, sizes, strides), rng.randint(0, 60)
        if lib.one(i64(row), dims(sizes, strides), 3):
            assert len(set(x)) == len(x)
        y = elements(z, row, sizes, strides)
        if lib.two(i64(row), dims(sizes, strides), i64(1000), dims(sizes, strides), i64(1000 + 2 * z), 3, 2):
            assert len(set(x + y)) == len(x + y)
        span = max(x) + 1      # far enough apart, either way round
        if len(set(x)) == len(x) and lib.one(i64(row), dims(sizes, strides), 3):
            assert lib.two(i64(row), dims(sizes, strides), i64(1000), dims(sizes, strides), i64(1000 + 2 * span), 3, 2) == 1
            assert lib.two(i64(row), dims(sizes, strides), i64(1000 + 2 * span), dims(sizes, strides), i64(1000), 3, 2) == 1
    big = dims((2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1), (2 ** 40 - 1, 16, 2 ** 36))      # spans past 64 bits
    assert lib.one(i64(16), big, 3) == 0
    # keys and values in one allocation: side by side, by pages, by rows
    for sizes, strides, z in (((5, 3, 4), (24, 8, 2), 120), ((5, 3, 4), (48, 8, 2), 24), ((5, 3, 4), (48, 4, 12), 2), ((1, 3, 4), (0, 8, 2), 24)):
        assert lib.two(i64(2), dims(sizes, strides), i64(2 * z), dims(sizes, strides), i64(0), 3, 2) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, I8])
def test_expanded_caches_are_read_and_not_written(kind):
    """Heads that share one's rows: read, attended to and kept elsewhere as their copies are; refused where they would be written."""
    query, cache, table, context = problem(2, 1, 4, 5, 200, 64, 16, kind, BF16)
    cache, table, context, query = device(cache), table.cuda(), context.cuda(), query.cuda()
    wide = KVCache(*(None if x is None else x.expand(-1, 2, *x.shape[2:]) for x in cache))
    copy = KVCache(*(None if x is None else x.contiguous() for x in wide))
    for a, z in zip(fca.cache_read(wide, table, context, 200), fca.cache_read(copy, table, context, 200)):
        assert torch.equal(a, z)
    assert torch.equal(fca.tree_attention(query, wide, table, context), fca.tree_attention(query, copy, table, context))
    keep = torch.rand((2, 2, 200), generator=torch.Generator().manual_seed(3)).cuda() < 0.4
    pages = torch.arange(table.numel(), device="cuda").view(2, -1).int()
    into = [KVCache.zeros(pages.numel(), 2, 16, 64, kind) for _ in range(2)]
    counts = [fca.cache_keep(c, table, context, keep, i, pages) for c, i in zip((wide, copy), into)]
    assert torch.equal(*counts) and all(a is None or torch.equal(a, z) for a, z in zip(*into))
    x = randn(2, 2, 3, 64, seed=9, dtype=BF16).cuda()
    for bad in (wide, cache._replace(v=cache.k)):
        heads = bad.k.shape[1]
        with pytest.raises(_lib.FcrError, match="share memory"):
            fca.cache_write(bad, x[:, :heads], x[:, :heads], table, context)
        with pytest.raises(_lib.FcrError, match="share memory"):
            fca.cache_keep(KVCache.zeros(cache.k.shape[0], heads, 16, 64, kind), table, context, keep[:, :heads], bad, pages)


@pytest.mark.parametrize("d,lanes", [(64, 4), (80, 8), (256, 16)])
def test_rows_of_one_call_without_a_device(d, lanes):
    """B * H * T * L up to 2^31 - 256: a call of as many rows gets as far as the next refusal."""
    strides = (16 * 8 * d, 16 * d, d)
    cache = _c_cache(H=8, D=d, page_size=16, k_strides=strides, v_strides=strides, k=1 << 20, v=1 << 20)
    most, xs = (2 ** 31 - 256) // (64 * lanes), (64 * d, 8 * d, d, 1)
    assert _c_call("write", cache, B=8, T=most, xs=xs) == -4 and b"share memory" in _lib.load().fcr_last_error()
    assert _c_call("write", cache, B=8, T=most + 1, xs=xs) == -3 and b"2^31 - 256" in _lib.load().fcr_last_error()
    assert _c_call("read", cache, B=8, N=most + 1) == -3 and b"2^31 - 256" in _lib.load().fcr_last_error()
    for n in (1 << 30, (1 << 30) - 1):       # (products past 64 bits)
        assert _c_call("write", cache, B=1 << 27, T=n, xs=xs) == -3 and _c_call("read", cache, B=1 << 27, N=n) == -3
    header = open(os.path.join(ROOT, "include", "fcr.h")).read()
    assert "B * H * T * L at most 2^31 - 256" in header and "B * H * N * L at most 2^31 - 256" in header


@pytest.fixture(scope="module")
def deal(tmp_path_factory):
    """csrc/deal.h, as the kernels include it."""
    at = tmp_path_factory.mktemp("deal")
    (at / "d.cpp").write_text(
        '#include "deal.h"\nusing namespace fcr_tree;\nextern "C" {\n'
        'int blocks(int n) { return blocks_of(n); }\n'
        'int tried(int entries, int threads, int per, int tiles, int tall) { return pieces_are_tried(entries, threads, per, tiles, tall); }\n'
        'int allowed(int per, int tiles, int tall) { return most_allowed(per, tiles, tall); }\n'
        'int most(int per, int limit, int wgs, const int* nb, const int* weight, int n, int* last) {\n'
        '  return most_of(per, limit, [&](int p) { int64_t sum = 0; for (int i = 0; i < n; ++i) sum += (int64_t)pieces_of(nb[i], p) * weight[i];\n'
        '    *last = p; return sum <= wgs; }); }\n'
        'int pieces(int nb, int most) { return pieces_of(nb, most); }\nint length(int nb, int pieces) { return piece_length(nb, pieces); }\n'
        'int behind(int others, int unit) { return followers(others, unit); }\n'
        'int form(int64_t rows, int w, int codes) { return form_of(rows, w, codes); }\nint tile(int form, int w) { return rows_of_tile(form, w); }\n}\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "flash_colreduce_amd", "csrc"), str(at / "d.cpp"), "-o",
                    str(at / "d.so")], check=True)
    lib = ctypes.CDLL(str(at / "d.so"))
    lib.form.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    return lib


def test_forms_have_kernels_and_tiles_that_hold_rows(deal):
    """Four waves only for rows of at most 128 elements; a tile of form 4 holds all rows, so that none is left to a second one."""
    for w in range(1, 5):
        for codes in (0, 1):
            forms = [deal.form(rows, w, codes) for rows in range(1, 400)]
            assert sorted(set(forms)) == ([1, 4, 8] if w <= 2 else [1, 8]) and forms == sorted(forms)
            assert all(f != 4 or rows <= deal.tile(4, w) for rows, f in enumerate(forms, 1))
            assert deal.form(1 << 24, w, codes) == 8 and deal.tile(1, w) == 16 and deal.tile(8, w) in (128, 256)


@pytest.mark.parametrize("seed", range(40))
def test_blocks_are_dealt_once_and_the_join_finds_them(deal, seed):
    """By the header that the kernels use: every block of every item is one workgroup's, and from what the workgroup with an item's first part tells the join
    finds the others, one behind the other, in the order of the item's keys.  Pieces of one item each are the longest that are needed, and not longer."""
    rng = random.Random(seed)
    for _ in range(12):
        tall, row_tiles, threads = rng.random() < 0.5, rng.choice([1, 1, 2, 3, 7]), rng.choice([16, 256])
        entries = [deal.blocks(rng.choice([-5, 0, 1, 127, 128, 129, rng.randint(0, 9000), 8192, 8192])) for _ in range(rng.randint(1, 40))]
        assert all(e >= 1 for e in entries) and deal.blocks(128) == 1 and deal.blocks(129) == 2
        heads = rng.choice([1, 1, 2, 8])
        weight = heads * row_tiles
        wgs = 8 * rng.randint(1, 64)
        total = sum(entries) * weight
        per = -(-total // wgs)
        most = 0
        if deal.tried(len(entries), threads, per, row_tiles, tall):
            limit, last, n = deal.allowed(per, row_tiles, tall), ctypes.c_int(), len(entries)
            most = deal.most(per, limit, wgs, (ctypes.c_int * n)(*entries), (ctypes.c_int * n)(*[weight] * n), n, ctypes.byref(last))
            fits = [p for p in range(per, limit + 1) if sum(-(-e // p) for e in entries) * weight <= wgs]
            assert most == (fits[0] if fits else 0) and (not most or last.value == most)
        items = [e for e in entries for _ in range(weight)]
        units = [deal.pieces(e, most) if most else e for e in items]
        unit = 1 if most else per
        parts, told = {}, {}
        for w in range(wgs):
            at, end = w * unit, min(w * unit + unit, sum(units))
            while at < end:
                begun, item = 0, 0
                while at >= begun + units[item]:
                    begun += units[item]
                    item += 1
                nb, blk = items[item], at - begun
                if most:
                    length = deal.length(nb, units[item])
                    blk *= length
                    stop = min(nb, blk + length)
                    at = end
                else:
                    stop = min(nb, blk + end - at)
                    at += stop - blk
                assert 0 <= blk < stop <= nb
                if blk == 0:
                    told[item] = (w, nb - (stop - blk))
                parts.setdefault(item, []).append((w, blk, stop))
        for item, nb in enumerate(items):
            got = parts[item]
            w, others = told[item]
            assert got[0][1] == 0 and got[-1][2] == nb and all(x[2] == y[1] for x, y in zip(got, got[1:]))
            assert [g[0] for g in got] == list(range(w, w + 1 + deal.behind(others, most or per)))
    assert deal.behind(0, 5) == 0 and deal.behind(-3, 5) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(I8, F16), (I8, BF16), (E4M3, F16), (E4M3, BF16)])
@pytest.mark.parametrize("t,d", [(1, 64), (5, 128), (40, 64), (60, 192), (30, 256)])
def test_scales_that_are_infinite(kind, dtype, t, d):
    """A value row of an infinite scale is infinite where its codes are not 0, and a NaN where they are, for the rows that see it; log-sum-exps are of the
    scores alone.  cache_write makes no such scales; a cache that is filled otherwise may have them."""
    query, cache, table, context = problem(2, 2, 2, t, 300, d, 16, kind, dtype)
    cache.v.view(torch.uint8)[:, :, :, 3] = 0
    for i, head, j in ((0, 0, 3), (0, 1, 299), (1, 0, int(context[1])), (1, 1, int(context[1]) + t // 2)):
        cache.v_scale[int(table[i, j // 16]), head, j % 16] = math.inf
    check_attention(query, cache, table, context)
    check_attention(query, cache, table, context, random_tree(2, t, 3))
    # scores of minus infinity: no weight
    for i, head, j in ((0, 0, 9), (1, 1, 40)):
        at = (int(table[i, j // 16]), head, j % 16)
        cache.k[at] = torch.full((d,), 1.0).to(kind)
        cache.k_scale[at] = -math.inf
    check_attention(query.abs() + 0.25, cache, table, context)
