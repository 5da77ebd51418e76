"""chunk_attention against a plain form in 64 bits, at the lengths, windows, prefixes and layouts where it can go wrong, and its refusals."""
import ctypes
import math
import os
import random
import re
import subprocess

import pytest
import torch

import flash_colreduce_amd as fca
from flash_colreduce_amd import KVCache, _lib
from flash_colreduce_amd import cache as cache_module
from tests.test_cache import (BF16, E4M3, F16, F32, HALF_STEP, I8, TOP, _c_cache, compare_attention, device, make_cache, of_heads, problem, randn,
                              random_table, values)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KINDS = [(F16, F16), (BF16, BF16), (I8, F16), (I8, BF16), (E4M3, F16), (E4M3, BF16)]


def ref_chunk(query, cache, table, context, scale=None, counts=None, cap=None, slopes=None, window=None, prefix=None):
    """(out, lse2, tolerance of out, of lse2) in 64 bits."""
    b, hq, t, d = query.shape
    h = cache.k.shape[1]
    g = hq // h
    n = max(min(int(context.clamp_min(0).long().max()) + t, table.shape[1] * cache.k.shape[2]), 1)
    k, v, there = values(cache, table, n)
    scale = 1 / math.sqrt(d) if scale is None else scale
    context = of_heads(context.clamp_min(0), h).long()[..., None, None]                          # (B, H, 1, 1)
    counts = (torch.full((b,), t) if counts is None else counts.long().clamp(0, t))[:, None, None, None]
    j, token = torch.arange(n), torch.arange(t)[:, None]
    distance = context + token - j                                                               # (B, H, T, n)
    seen = distance >= 0
    if window is not None:
        seen = seen & (distance < window)
    if prefix is not None:
        seen = seen | (j < prefix.long()[:, None, None, None])
    seen = seen & (j < context + counts) & (token < counts) & there[:, None, None]
    seen, distance = seen.repeat_interleave(g, 1), distance.repeat_interleave(g, 1).abs()
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    q = query.float().double()
    any_seen = seen.any(2, keepdim=True).transpose(2, 3)
    k0, v0 = torch.where(any_seen, k, 0.0), torch.where(any_seen, v, 0.0)
    s = q @ k0.transpose(-1, -2) * scale
    if cap is not None:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        s = s - slopes.double()[None, :, None, None] * distance
    s = torch.where(seen, s, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(lse.isfinite(), lse, 0.0)[..., None]), 0.0)
    out = p @ torch.where(v0.isfinite(), v0, 0.0)
    for bi, hi, at in (~v0.isfinite()).any(-1).nonzero().tolist():
        sees = seen[bi, hi, :, at]
        bad = torch.where(v0[bi, hi, at].isfinite(), 0.0, v0[bi, hi, at])
        out[bi, hi, sees] = out[bi, hi, sees] + p[bi, hi, sees, at][:, None] * bad
    # As for tree_attention: weights rounded to fp16 (bf16 against a bf16 cache), those under 2^-14 of the largest to half of fp16's smallest step; scores are
    # sums of D products, each off by 2^-24 of the sum of magnitudes, and exp2's 2^-21.  A cap adds, in steps of 2^-24 of it: 1 for its own rounding, 2 for the
    # reciprocal's last bit, 1 for the exponential's and 2 for what is fed to it, twice for safety 12: under 2^-20; it makes no error before it larger.  Above 128 it
    # is formed so that these are steps of the score instead.  A slope times a
    # distance is rounded three times (slope in base 2, product, sum): 2^-22 of it.
    rounding = HALF_STEP[BF16 if cache.k.dtype == BF16 else F16]
    v1 = torch.where(v0.isfinite(), v0, 0.0).abs()
    magnitude = torch.where(any_seen.transpose(2, 3) & seen, q.abs() @ torch.where(k0.isfinite(), k0, 0.0).abs().transpose(-1, -2) * abs(scale), 0.0).amax(-1)
    ds = (d + 8) * 2.0 ** -24 * magnitude + 2.0 ** -21 + (0 if cap is None else cap * 2.0 ** -20 if cap <= 128 else magnitude * 2.0 ** -20)
    if slopes is not None:
        ds = ds + 2.0 ** -22 * (slopes.double()[None, :, None, None] * distance * seen).abs().amax(-1)
    weighted = p @ v1
    least = 2.0 ** -24 * n * (p.amax(-1, keepdim=True) * v1.amax((-1, -2), keepdim=True) if cache.k_scale is None
                              else (p * v1.amax(-1)[:, :, None]).amax(-1, keepdim=True))
    tol = weighted * (rounding + 2 * ds[..., None]) + 2 * least + out.abs() * HALF_STEP[query.dtype] * 1.01 + 2.0 ** -24
    dead = ~seen.any(-1)
    out[dead], lse[dead] = 0.0, -math.inf
    return out, lse / math.log(2), tol, 2 * (ds + 2.0 ** -22 * (1 + lse.abs()))


def call(query, cache, table, context, **how):
    how = {k: x.cuda() if isinstance(x, torch.Tensor) else x for k, x in how.items()}
    return fca.chunk_attention(query.cuda(), device(cache), table.cuda(), context.cuda(), return_lse2=True, **how)


def check(query, cache, table, context, **how):
    got, lse = call(query, cache, table, context, **how)
    assert got.dtype == query.dtype and got.shape == query.shape
    ref = ref_chunk(query, cache, table, context, **how)
    compare_attention(got, lse, ref)
    if query.shape[2] > 1 and query.shape[0] <= 40:
        # where there might be many keys another kernel takes as many rows
        how.setdefault("prefix", torch.zeros(query.shape[0], dtype=torch.int32))
        if how["prefix"] is None:
            how["prefix"] = torch.zeros(query.shape[0], dtype=torch.int32)
        compare_attention(*call(query, cache, wide(table), context, **how), ref)
    return got, lse


def same(table):
    return table


def wide(table):
    """The same pages and many places behind them that have none."""
    return torch.cat([table, torch.full((table.shape[0], 100000), -1, dtype=torch.int32)], 1)


def slopes_of(heads):
    return torch.exp2(-8.0 * torch.arange(1, heads + 1) / heads)


# Without a device --------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def sight(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("sight")
    (tmp / "s.cpp").write_text(
        '#include "deal.h"\nusing namespace fcr_tree;\n'
        'extern "C" void sight(int context, int count, int prefix, int window, int T, int positions, int first, int last, int some, int to, int* out) {\n'
        '  const Sight s(context, count, prefix, window, T, positions, first, last), rows(context, count, prefix, window, T, positions, some, to);\n'
        '  const Steps wave(rows, s, 1);\n'
        '  out[0] = s.blocks(); out[1] = s.n;\n'
        '  if (s.position(128 * out[0]) < s.n || s.position(-32) < s.n || s.key(-32) < s.n) out[0] = -1;\n'
        '  for (int i = 0; i < 4 * out[0]; ++i) { const int p = s.position(32 * i), x = 128 * out[0] - 32 - 32 * i, k = s.key(x); int* const o = out + 2 + 5 * i;\n'
        '    o[0] = p; o[1] = s.whole(p, 32); o[2] = k; o[3] = wave.whole(x); o[4] = wave.some(x); } }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "flash_colreduce_amd", "csrc"), str(tmp / "s.cpp"), "-o",
                    str(tmp / "s.so")], check=True)
    return ctypes.CDLL(str(tmp / "s.so"))


def test_blocks_of_a_tile_hold_every_key_that_it_sees(sight):
    """Every key that a token of the tile sees lies in its blocks, once and in order; steps said to be seen by all of some rows are, those said to be seen by none are
    seen by none."""
    rng = random.Random(2)
    for _ in range(4000):
        T = rng.choice([1, 2, 7, 40, 300])
        context, count = rng.choice([0, 1, rng.randint(0, 1000), -5]), rng.randint(-1, T + 1)
        positions = 16 * rng.randint(1, 90)
        window = rng.choice([2 ** 31 - 1, 1, 2, rng.randint(1, 400)])
        prefix = rng.choice([0, 0, -3, rng.randint(0, 500), 1500])
        first = rng.randint(0, T - 1)
        last = rng.randint(first, T - 1)
        some = rng.randint(first, last)
        to = rng.randint(some, last)
        out = (ctypes.c_int * (2 + 5 * 4 * 80))()
        sight.sight(context, count, prefix, window, T, positions, first, last, some, to, out)
        start, have = max(context, 0), min(max(count, 0), T)
        tokens = range(first, min(last, have - 1) + 1)
        keys = range(min(start + have, positions))
        seen = {t: {j for j in keys if j <= start + t and j > start + t - window or j < prefix} for t in tokens}
        seen_by_any = set().union(*seen.values())
        steps = [out[2 + 5 * i: 7 + 5 * i] for i in range(4 * out[0])]
        at = [p for p, *_ in steps]
        assert out[0] >= 1
        if not seen_by_any:
            assert out[0] == 1
            continue
        # blocks from the last one on, the steps of a block in their order; and all steps from the last one on
        assert all(p % 128 == 32 * (i % 4) and p // 128 == at[i - i % 4] // 128 for i, p in enumerate(at))
        assert all(a > z >= 0 for a, z in zip(at[::4], at[4::4])) and at[-4] >= 0
        assert [k for _, _, k, _, _ in steps] == sorted(at, reverse=True)
        assert seen_by_any <= {j for p in at for j in range(p, p + 32)}
        rows = [seen[t] for t in range(some, to + 1) if t in seen]
        for p, whole, k, wave_whole, wave_some in steps:
            assert not whole or all(set(range(p, p + 32)) <= s for s in seen.values())
            step = set(range(k, k + 32))
            assert not rows or not wave_whole or all(step <= s for s in rows)
            assert wave_some or not any(step & s for s in rows)
        # and no block without a reason
        assert out[0] <= max(1, len({j // 128 for j in seen_by_any}) + 1)


@pytest.fixture(scope="module")
def tile_rule(tmp_path_factory):
    """The kernel that csrc/deal.h gives a call of more than 128 rows of at most 128 elements, on 256 compute units: 1, 4 or 8."""
    tmp = tmp_path_factory.mktemp("tiles")
    (tmp / "t.cpp").write_text(
        '#include "deal.h"\nusing namespace fcr_tree;\n'
        'extern "C" int form(int codes, int B, int H, int G, int T, int D, int positions, int window) {\n'
        '  const int w = (D + 63) / 64, rows = T * G, small = rows_of_tile(1, w), half = rows_of_tile(4, w);\n'
        '  const int64_t heads = (int64_t)B * H;\n'
        '  if (takes_few_rows(heads * quotient_up(rows, small), 256 * (w == 1 ? 3 : 2), most_blocks_of(positions, window, small, G))) return 1;\n'
        '  if (takes_half_tiles(heads * quotient_up(rows, half), 512, most_blocks_of(positions, window, half, G), D, positions, T)) return 4;\n'
        '  return form_of(rows, w, codes); }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "flash_colreduce_amd", "csrc"), str(tmp / "t.cpp"), "-o",
                    str(tmp / "t.so")], check=True)
    return ctypes.CDLL(str(tmp / "t.so")).form


# (B, H, G, T, context, D, page), window: several tiles of 128 rows to a head, more of them than the chip holds; prompts, and a window far behind the first key
HALVES = [((33, 8, 1, 150, 350, 64, 16), 300), ((34, 8, 2, 75, 400, 48, 16), 130), ((33, 8, 1, 300, 20, 64, 16), None), ((33, 8, 1, 270, 0, 128, 16), None),
          ((45, 4, 3, 130, 100, 112, 16), None)]


@pytest.mark.parametrize("shape,window", HALVES)
def test_many_short_tiles_are_of_128_rows(shape, window, tile_rule):
    b, h, g, t, n, d, page = shape
    positions = -(-(n + t) // page) * page
    assert all(tile_rule(codes, b, h, g, t, d, positions, window or 0) == 4 for codes in (0, 1))
    assert tile_rule(0, 1, h, g, 4000, d, 1 << 20, 0) == 8 and tile_rule(0, 1, 1, g, t, d, positions, window or 0) == 1
    assert (positions > 2 * t) == (window is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(F16, F16), (BF16, BF16), (I8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("shape,window", HALVES)
def test_tiles_of_128_rows(shape, window, kind, dtype):
    """Behind a window, and with everything that becomes of scores; ragged counts, contexts of own length for each head."""
    b, h, g, t, n, d, page = shape
    query, cache, table, context = problem(*shape, kind, dtype)
    draw = torch.Generator().manual_seed(t)
    counts, context = torch.randint(0, t + 1, (b,), generator=draw).int(), torch.randint(0, n + 1, (b, h), generator=draw).int()
    counts[0], context[0] = t, n
    for how in (dict(), dict(cap=3.0), dict(slopes=slopes_of(h * g), counts=counts), dict(cap=200.0, slopes=slopes_of(h * g) * 0.1)):
        got = call(query, cache, table, context, window=window, **how)
        compare_attention(*got, ref_chunk(query, cache, table, context, window=window, **how))


def test_shared_arrays_that_are_read_16_bytes_at_a_time_are_aligned_for_it():
    """By their elements' type or by their declaration: where the compiler happens to put them is no promise."""
    csrc, wide_reads = os.path.join(ROOT, "flash_colreduce_amd", "csrc"), 0
    for name in sorted(os.listdir(csrc)):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        for kernel in re.split(r"__global__", text)[1:]:
            arrays = {}
            for aligned, kind, names in re.findall(r"__shared__\s+(?:__attribute__\(\(aligned\((\d+)\)\)\)\s+)?(\w+)\s+([^;]+);", kernel):
                for array in re.findall(r"(\w+)(?:\[[^\]]*\])+", names):
                    arrays[array] = int(aligned or 0) >= 16 or kind in ("u32x4", "f32x4", "int4")
            for array in re.findall(r"reinterpret_cast<\s*(?:const\s+)?(?:u32x4|f32x4|int4|double2)\s*\*>\(\s*(\w+)", kernel):
                if array in arrays:
                    wide_reads += 1
                    assert arrays[array], (name, array)
    assert wide_reads >= 4


def _chunk_c(**over):
    a = dict(q=48, table=16, stride=4, pages=4, context=32, cs=(1, 0), counts=None, prefix=None, slopes=None, out=64, ws=128, ws_bytes=1 << 40, dtype=0, B=2, G=2,
             T=3, qs=(4096, 512, 64, 1), scale=0.1, cap=0.0, window=0)
    a.update(over)
    return _lib.load().fcr_chunk_attention(
        a["q"], ctypes.byref(_c_cache()), a["table"], a["stride"], a["pages"], a["context"], a["cs"] and cache_module._I64x2(*a["cs"]), a["counts"], a["prefix"],
        a["slopes"], a["out"], None, a["ws"], a["ws_bytes"], a["dtype"], a["B"], a["G"], a["T"], a["qs"] and _lib.strides4(a["qs"]), a["scale"], a["cap"],
        a["window"], None)


@pytest.mark.parametrize("over, code", [
    (dict(q=None), -1), (dict(table=None), -1), (dict(context=None), -1), (dict(cs=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(qs=None), -1),
    (dict(dtype=2), -2), (dict(B=0), -3), (dict(G=0), -3), (dict(T=0), -3), (dict(T=(1 << 24) + 1), -3), (dict(pages=0), -3), (dict(window=-1), -3),
    (dict(q=56), -4), (dict(qs=(4096, 512, 60, 1)), -4), (dict(cs=(-1, 0)), -4), (dict(out=72), -4), (dict(ws=136), -4), (dict(ws_bytes=15), -7),
    (dict(scale=math.nan), -6), (dict(cap=-1.0), -6), (dict(cap=math.inf), -6), (dict(cap=math.nan), -6), (dict(cap=1e-38, scale=1e3), -6)])
def test_c_abi_refuses(over, code):
    """Every refusal comes before the first launch, so invented pointers are safe."""
    assert _chunk_c(**over) == code
    assert _lib.load().fcr_last_error() != b""


def test_python_refuses_without_a_device():
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fca.chunk_attention(torch.zeros(1, 2, 1, 16).half(), KVCache.zeros(2, 2, 16, 16, F16, device="cpu"), z[:, None], z)


# On the device -----------------------------------------------------------------------------------------------------------

# (B, H, G, T, context, D, page): rows that every kernel takes, and either side of where another one takes over
SHAPES = [(1, 1, 1, 1, 1, 16, 16), (2, 2, 4, 1, 300, 64, 16), (3, 2, 3, 5, 129, 80, 32), (1, 2, 1, 16, 100, 128, 16), (2, 1, 2, 23, 400, 96, 16),
          (1, 2, 4, 40, 260, 64, 48), (1, 1, 2, 130, 0, 128, 16), (2, 1, 3, 100, 513, 128, 16), (1, 1, 1, 300, 70, 192, 16), (1, 1, 4, 70, 200, 256, 32),
          (2, 2, 1, 257, 129, 64, 16), (1, 1, 8, 3, 1000, 256, 16), (5, 1, 7, 9, 30, 112, 16), (1, 1, 17, 31, 90, 144, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_chunks_match_64_bits(shape, kind, dtype):
    """Plain scores, and everything at once."""
    b, h, g, t, n, d, page = shape
    query, cache, table, context = problem(*shape, kind, dtype)
    check(query, cache, table, context)
    counts = torch.randint(0, t + 1, (b,), generator=torch.Generator().manual_seed(t)).int()
    counts[-1] = t
    check(query, cache, table, context, cap=3.0, slopes=slopes_of(h * g), window=max(1, (n + t) // 3), prefix=torch.full((b,), 20, dtype=torch.int32), counts=counts)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(BF16, BF16), (I8, BF16), (E4M3, F16), (F16, F16)])
@pytest.mark.parametrize("g,t,d", [(1, 200, 64), (4, 60, 128), (2, 5, 128), (3, 90, 256)])
def test_windows_and_prefixes(kind, dtype, g, t, d):
    """Windows of one key to more than there are, prefixes that end inside blocks, behind tokens and behind the last key."""
    query, cache, table, context = problem(2, 1, g, t, 700, d, 16, kind, dtype)
    context[1] = 401
    for window in (1, 2, 31, 128, 333, 5000, None):
        for prefix in ([0, 0], [1, 130], [700 + t // 2, 128], [2000, 401 + t], None):
            check(query, cache, table, context, window=window, prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_lengths(kind, dtype):
    """No context, contexts of own length for each head, counts of none, more than the table names, negative ones."""
    query, cache, table, _ = problem(3, 2, 2, 75, 150, 64, 16, kind, dtype)
    for how in (dict(), dict(window=40, prefix=torch.tensor([5, 0, 300]).int()), dict(cap=2.0, counts=torch.tensor([75, 0, 1]).int())):
        check(query, cache, table, torch.tensor([0, 1, 150]).int(), **how)
        check(query, cache, table, torch.tensor([[150, 3], [0, 77], [16, 128]]).int(), **how)
        check(query, cache, table, torch.tensor([-2 ** 31, 2 ** 31 - 1, 170]).int(), **how)
    check(query, cache, table, torch.tensor([0, 1, 150]).int(), counts=torch.tensor([-3, 100, 74]).int())
    check(query[:, :, :1], cache, table, torch.tensor([[0, 1], [9, 150], [64, 63]]).int(), slopes=slopes_of(4))
    got, lse = call(query, cache, torch.full_like(table, -1), torch.tensor([5, 5, 5]).int(), cap=1.0)
    assert not got.any() and lse.isneginf().all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(BF16, BF16), (I8, F16)])
@pytest.mark.parametrize("b,h,t,g", [(700, 2, 1, 2), (530, 1, 33, 2), (40, 2, 600, 1), (1, 1, 3000, 1)])
def test_more_tiles_than_threads(kind, dtype, b, h, t, g):
    """Lengths per sequence and per head, with zeros among them."""
    query, cache, table, context = problem(b, h, g, t, 20, 32, 16, kind, dtype)
    counts = torch.randint(0, t + 1, (b,), generator=torch.Generator().manual_seed(4)).int()
    check(query, cache, table, context, counts=counts, cap=5.0)
    heads = torch.randint(0, 21, (b, h), generator=torch.Generator().manual_seed(9)).int()
    heads[-1] = 20
    check(query, cache, table, heads, window=15)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(F16, F16), (I8, BF16)])
@pytest.mark.parametrize("shape", [(1, 32, 1, 1, 16400, 16, 16), (2, 8, 1, 40, 8200, 32, 16), (2, 8, 2, 300, 2000, 32, 16)])
def test_many_blocks_per_workgroup(shape, kind, dtype):
    query, cache, table, context = problem(*shape, kind, dtype)
    check(query, cache, table, context, slopes=slopes_of(shape[1] * shape[2]) * 0.05)
    check(query, cache, table, context, window=3000, prefix=torch.full((shape[0],), 300).int())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(F16, F16), (E4M3, BF16)])
@pytest.mark.parametrize("b,h,g,t,n,d", [(70, 8, 2, 1, 2500, 16), (9, 4, 1, 300, 1500, 32), (9, 4, 1, 300, 200, 32), (130, 8, 1, 1, 300, 64), (24, 4, 2, 20, 900, 64),
                                         (45, 4, 1, 400, 100, 64), (40, 2, 4, 200, 60, 128)])
def test_items_whole_and_cut(kind, dtype, b, h, g, t, n, d):
    """Many items, of one length, of drawn lengths, one long among short ones, of nothing but for one, of own lengths for each head."""
    query, cache, table, _ = problem(b, h, g, t, n, d, 16, kind, dtype)
    draw = torch.Generator().manual_seed(n)
    full = torch.full((b,), n, dtype=torch.int32)
    drawn, tokens = torch.randint(0, n + 1, (b,), generator=draw).int(), torch.randint(0, t + 1, (b,), generator=draw).int()
    one, last = torch.full((b,), 3, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    one[b // 2], last[-1] = n, t
    for context, counts in ((full, None), (drawn, tokens), (one, None), (full, last), (torch.randint(0, n + 1, (b, h), generator=draw).int(), tokens)):
        check(query, cache, table, context, counts=counts)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("t,d,places", [(6, 64, same), (130, 128, same), (130, 128, wide), (3, 256, same), (90, 256, wide), (300, 64, wide)])
def test_what_hidden_rows_hold_has_no_influence(kind, dtype, t, d, places):
    """NaNs and infinities, and NaN scales, behind the last key, between prefix and window, on pages that are not there; and in keys that only later tokens see."""
    query, cache, table, _ = problem(2, 1, 2, t, 500, d, 16, kind, dtype)
    context = torch.tensor([400, 300]).int()
    how = dict(window=100, prefix=torch.tensor([3, 40]).int(), cap=4.0, slopes=slopes_of(2))
    want, want_lse = call(query, cache, places(table), context, **how)
    nothing = torch.tensor([math.nan, math.inf, -math.inf])
    dirty = KVCache(*(None if x is None else x.clone() for x in cache))
    for b, (c, p) in enumerate(zip(context.tolist(), (3, 40))):
        for j in [*range(p, c - 100), *range(c + t, table.shape[1] * 16)]:
            page, row = int(table[b, j // 16]), j % 16
            for x, s in ((dirty.k, dirty.k_scale), (dirty.v, dirty.v_scale)):
                if s is None:
                    x[page, 0, row] = nothing[j % 3].to(kind)
                else:
                    s[page, 0, row] = nothing[j % 3]
                    if kind == E4M3:
                        x.view(torch.uint8)[page, 0, row, ::3] = 0x7f
    got, lse = call(query, dirty, places(table), context, **how)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    # values that are not finite, in a key of the chunk itself, reach the tokens from it on
    if kind in (F16, BF16):
        page, row = int(table[0, (400 + t - 2) // 16]), (400 + t - 2) % 16
        dirty.v[page, 0, row, 5] = math.inf
        dirty.v[page, 0, row, 6] = math.nan
        got, lse = check(query, dirty, table, context, **how)
        assert got[0, :, : t - 2].isfinite().all() and not got[0, :, t - 2:, 5].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_scores_at_the_ends(kind, dtype):
    """Scores far above a cap, slopes that leave one key, negative ones, scales of 0 and below, caps next to 0 and above all scores."""
    query, cache, table, context = problem(2, 2, 2, 20, 200, 64, 16, kind, dtype, spread=2.0)
    for how in (dict(scale=50.0, cap=1.0), dict(scale=0.0, cap=3.0), dict(scale=-0.3, cap=20.0), dict(cap=1e-3), dict(cap=128.0), dict(cap=130.0), dict(cap=1e6), dict(scale=30.0, cap=200.0), dict(cap=1e30), dict(slopes=torch.full((4,), 100.0)),
                dict(slopes=torch.full((4,), -0.3)), dict(slopes=torch.zeros(4), window=7), dict(scale=3.0, slopes=torch.tensor([0.0, 1e-4, 2.0, -1.0]), cap=30.0)):
        check(query, cache, table, context, **how)
        check(query[:, :, :3], cache, table, context, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("cap", [1e36, 1e37, 1e38, 2.35e38])
def test_the_largest_caps(kind, dtype, cap):
    """Caps next to which every score is small leave them as they are, whatever powers of two codes and bf16 queries bring with them; scores as large as the caps."""
    query, cache, table, context = problem(2, 2, 2, 20, 200, 64, 16, kind, dtype, spread=2.0)
    for how in (dict(), dict(slopes=slopes_of(4), counts=torch.tensor([20, 7]).int()), dict(scale=3e-4), dict(scale=1e34)):
        check(query, cache, table, context, cap=cap, **how)
        check(query[:, :, :3], cache, table, context, cap=cap, **how)


def test_caps_past_32_bits_are_refused():
    """What a cap is in base 2 has to be a number, too; the text says which of the two it was."""
    assert _chunk_c(cap=2.4e38) == -6 and b"cap in base 2" in _lib.load().fcr_last_error()
    assert _chunk_c(cap=1e-38, scale=1e3) == -6 and b"scale over cap" in _lib.load().fcr_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("t,places", [(3, same), (100, same), (100, wide)])
def test_scores_that_are_not_finite(kind, t, places):
    """Infinite keys: a score of +-infinity is +-cap with one; without, -infinity is no weight."""
    query, cache, table, context = problem(1, 1, 1, t, 100, 64, 16, kind, kind)
    query = query.abs() + 0.01
    query = query.to(kind)
    cache.k[int(table[0, 2]), 0, 3] = -math.inf
    cache.k[int(table[0, 3]), 0, 3] = math.inf
    got, lse = call(query, cache, places(table), context, cap=2.0)
    finite = KVCache(cache.k.clone().clamp(-30000, 30000), cache.v)
    want, want_lse = call(query, finite, places(table), context, cap=2.0)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    cache.k[int(table[0, 3]), 0, 3] = -math.inf
    got, lse = call(query, cache, places(table), context)
    assert got.isfinite().all() and lse.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(F16, F16), (BF16, BF16), (I8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("t,more", [(5, 3), (70, 3), (70, 50000)])
def test_layouts(kind, dtype, t, more):
    """Keys and values of one allocation, token-major pages, token-major and expanded queries, tables and lengths that are views; the native path and the other."""
    b, h, g, n, d, page = 2, 3, 2, 200, 64, 16
    query, cache, table, context = problem(b, h, g, t, n, d, page, kind, dtype)
    pages = cache.k.shape[0]
    both = torch.zeros((pages, 2, page, h + 1, d), dtype=torch.uint8 if kind == E4M3 else kind, device="cuda")
    both = both.view(E4M3) if kind == E4M3 else both
    k, v = both[:, 0, :, :h].transpose(1, 2), both[:, 1, :, 1:].transpose(1, 2)
    k.copy_(cache.k.cuda()), v.copy_(cache.v.cuda())
    scales = [None, None]
    if kind in TOP:
        room = torch.zeros((pages, 2, h, page), device="cuda")
        scales = [room[:, 0], room[:, 1]]
        scales[0].copy_(cache.k_scale), scales[1].copy_(cache.v_scale)
    view = KVCache(k, v, *scales)
    if more > 3:
        table = wide(table)
    padded = torch.full((b, table.shape[1] + more), -1, dtype=torch.int32)
    padded[:, : table.shape[1]] = table
    how = dict(cap=3.0, slopes=slopes_of(h * g), window=90, prefix=torch.tensor([17, 3]).int(), counts=torch.tensor([t, t - 2]).int())
    ref = ref_chunk(query, cache, table, context, **how)
    on = {k: x.cuda() if isinstance(x, torch.Tensor) else x for k, x in how.items()}
    major = query.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    some = torch.stack([context, context * 0], 1).cuda()[:, 0]
    want = fca.chunk_attention(major, view, padded.cuda()[:, : table.shape[1]], some, return_lse2=True, **on)
    compare_attention(*want, ref)
    odd = torch.zeros(b * h * g * t * d + 1, dtype=dtype, device="cuda")[1:].view(b, h * g, t, d)     # starts off 16 bytes
    odd.copy_(query)
    strided = {k: torch.stack([x, x], 1)[:, 0] if isinstance(x, torch.Tensor) else x for k, x in on.items()}
    got = fca.chunk_attention(odd, view, table.cuda(), context.cuda()[:, None].expand(b, h), return_lse2=True, **strided)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = query[:, :, :1].expand(b, h * g, t, d)
    got = fca.chunk_attention(one.cuda()[:, :, :1].expand(b, h * g, t, d), view, table.cuda(), context.cuda(), return_lse2=True, **on)
    compare_attention(*got, ref_chunk(one, cache, table, context, **how))
    got = fca.chunk_attention(major, view, table.cuda(), context.cuda(), cap=3, window=2 ** 40)
    assert torch.equal(got, fca.chunk_attention(major, view, table.cuda(), context.cuda(), cap=3.0))


@pytest.mark.gpu
def test_plain_scores_of_a_chain_are_those_of_tree_attention():
    """Nothing but causality: the same numbers as tree_attention without a mask, within both tolerances."""
    for t, n, places in ((1, 500, same), (30, 300, same), (30, 300, wide), (300, 100, wide)):
        query, cache, table, context = problem(2, 2, 2, t, n, 128, 16, I8, BF16)
        table = places(table)
        got, lse = call(query, cache, table, context)
        want, want_lse = fca.tree_attention(query.cuda(), device(cache), table.cuda(), context.cuda(), return_lse2=True)
        _, _, tol, tol_lse = ref_chunk(query, cache, table, context)
        assert ((got - want).abs().double().cpu() <= 2 * tol).all() and ((lse - want_lse).abs().double().cpu() <= 2 * tol_lse).all()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of a pool."""
    h, page, d = 4, 256, 256
    pages = (5 << 30) // (h * page * d * 2)
    cache = KVCache(*(torch.zeros((pages, h, page, d), dtype=BF16, device="cuda") for _ in range(2)))
    n, t = 600, 70
    table = torch.tensor([[pages - 1, 0, pages - 7]]).int()
    x = [randn(1, h, n + t, d, seed=i, dtype=BF16) for i in (1, 2)]
    fca.cache_write(cache, x[0].cuda(), x[1].cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    small = KVCache(*(None if p is None else p[[pages - 1, 0, pages - 7]].cpu() for p in cache))
    context = torch.full((1,), n, dtype=torch.int32)
    for rows, places in ((t, same), (t, wide), (2, same)):
        query = randn(1, 2 * h, rows, d, seed=3, dtype=BF16)
        got, lse = fca.chunk_attention(query.cuda(), cache, places(table).cuda(), context.cuda(), cap=5.0, return_lse2=True)
        compare_attention(got, lse, ref_chunk(query, small, torch.arange(3).view(1, 3).int(), context, cap=5.0))


@pytest.mark.gpu
def test_streams_graphs_and_repetition():
    """On side streams and replayed from two graphs of one pool with eager calls in between, every result is that of the first call, bit for bit; a replay reads
    the lengths anew."""
    calls = []
    for shape, how in (((3, 2, 4, 1, 3000, 64, 16), dict(cap=30.0)), ((2, 2, 4, 90, 2000, 128, 16), dict(window=700, prefix=torch.tensor([4, 4]).int().cuda()))):
        query, cache, table, context = problem(*shape, I8, BF16)
        query, cache, table, context = query.cuda(), device(cache), (table if shape[3] == 1 else wide(table)).cuda(), context.cuda()
        calls.append((lambda q=query, c=cache, t=table, n=context, how=how: fca.chunk_attention(q, c, t, n, return_lse2=True, **how), context))
    want = [[y.clone() for y in c()] for c, _ in calls]
    torch.cuda.synchronize()
    graphs, held = [], []
    for c, _ in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            held.append(c())
        graphs.append(graph)
    for i in range(4):
        for graph, got, w, (c, context) in zip(graphs, held, want, calls):
            graph.replay()
            assert all(torch.equal(a, z) for a, z in zip(got, w)), i
            assert all(torch.equal(a, z) for a, z in zip(c(), w)), i
            if i == 2:
                context -= 77
        if i == 2:
            torch.cuda.synchronize()
            want = [[y.clone() for y in c()] for c, _ in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for k, (stream, (c, _)) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(stream):
                got[k].append(c())
    torch.cuda.synchronize()
    for k, w in enumerate(want):
        assert all(torch.equal(a, z) for g in got[k] for a, z in zip(g, w))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, I8])
def test_a_prompt_in_chunks(kind):
    """Pages reserved, a prompt written and attended to in chunks of odd lengths, then single tokens: every row as if the prompt had been one chunk."""
    b, h, g, d, ps, total = 2, 2, 2, 64, 16, 150
    pool, table = fca.PagePool.full(24, b), torch.full((b, 12), -1, dtype=torch.int32, device="cuda")
    cache = KVCache.zeros(24, h, ps, d, kind)
    key, value = (randn(b, h, total, d, seed=i, dtype=BF16).cuda() for i in (1, 2))
    query = randn(b, h * g, total, d, seed=3, dtype=BF16).cuda()
    how = dict(cap=4.0, slopes=slopes_of(h * g).cuda(), window=60, prefix=torch.tensor([4, 20]).int().cuda())
    context, parts = torch.zeros(b, dtype=torch.int32, device="cuda"), []
    for t in (37, 1, 80, 30, 1, 1):
        at = int(context[0])
        assert bool(fca.cache_reserve(pool, table, context + t, ps).all())
        fca.cache_write(cache, key[:, :, at:at + t], value[:, :, at:at + t], table, context)
        parts.append(fca.chunk_attention(query[:, :, at:at + t], cache, table, context, return_lse2=True, **how))
        context += t
    whole = KVCache(*(None if x is None else x.cpu() for x in cache))
    ref = ref_chunk(query.cpu(), whole, table.cpu(), torch.zeros(b, dtype=torch.int32), **{k: x.cpu() if isinstance(x, torch.Tensor) else x for k, x in how.items()})
    # (a token in front of the prefix's end sees what of it has been written so far)
    first = 37
    late = [x[:, :, first:] for x in ref]
    compare_attention(torch.cat([p[0] for p in parts], 2)[:, :, first:], torch.cat([p[1] for p in parts], 2)[:, :, first:], late)


@pytest.mark.gpu
def test_refusals_on_the_device():
    query, cache, table, context = problem(2, 2, 2, 3, 40, 64, 16, F16, F16)
    query, cache, table, context = query.cuda(), device(cache), table.cuda(), context.cuda()
    ints = torch.ones(2, dtype=torch.int32, device="cuda")
    bad = [dict(query=query.float()), dict(query=query.bfloat16()), dict(query=query[:, :3]), dict(query=query[..., :32]), dict(query=query[0]), dict(query=query.cpu()),
           dict(table=table.long()), dict(table=table[:1]), dict(context=context.long()), dict(context=context[:1]), dict(counts=ints.long()), dict(counts=ints[:1]),
           dict(prefix=ints.float()), dict(prefix=ints[:, None]), dict(slopes=torch.ones(3, device="cuda")), dict(slopes=torch.ones(4, device="cuda").half()),
           dict(slopes=torch.ones(4)), dict(cap=0.0), dict(cap=-1.0), dict(cap=1e-46), dict(cap=math.inf), dict(cap=math.nan), dict(window=0), dict(window=-5)]
    for over in bad:
        a = {**dict(query=query, table=table, context=context), **over}
        with pytest.raises(ValueError):
            fca.chunk_attention(a.pop("query"), cache, a.pop("table"), a.pop("context"), **a)
    for over in (dict(scale=math.inf), dict(cap=1e-38, scale=1e6)):
        with pytest.raises(_lib.FcrError):
            fca.chunk_attention(query, cache, table, context, **over)
    out, lse = fca.chunk_attention(query[:, :, :0], cache, table, context, return_lse2=True)
    assert out.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    out, lse = fca.chunk_attention(query, cache, table[:, :0], context, return_lse2=True)
    assert not out.any() and lse.isneginf().all()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
def test_random_calls(seed):
    """Calls of any kind, five for each seed."""
    rng = random.Random(seed)
    for _ in range(5):
        kind, dtype = rng.choice(KINDS)
        h, g, t = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 4, 7]), rng.choice([1, 1, 2, 5, rng.randint(1, 40), rng.randint(1, 400)])
        n, d, page = rng.choice([0, 3, rng.randint(0, 300), rng.randint(0, 3000)]), 16 * rng.randint(1, 16), rng.choice([16, 32, 48, 128])
        b = rng.randint(1, max(1, min(200, 40000000 // (h * g * t * (n + t) * d))))
        query, cache, table, context = problem(b, h, g, t, n, d, page, kind, dtype)
        draw = torch.Generator().manual_seed(seed)
        how = {}
        if rng.random() < 0.5:
            how["counts"] = torch.randint(0, t + 1, (b,), generator=draw).int()
        if rng.random() < 0.4:
            how["cap"] = rng.choice([0.5, 5.0, 30.0, 300.0])
        if rng.random() < 0.3:
            how["slopes"] = slopes_of(h * g) * rng.choice([1.0, 0.01, -0.001])
        if rng.random() < 0.4:
            how["window"] = rng.randint(1, n + t + 5)
        if rng.random() < 0.4:
            how["prefix"] = torch.randint(0, n + t + 2, (b,), generator=draw).int()
        if rng.random() < 0.6:
            context = torch.randint(0, n + 1, (b, h) if rng.random() < 0.3 else (b,), generator=draw).int()
        if rng.random() < 0.2:
            table[rng.randrange(b), rng.randrange(table.shape[1])] = -1
        check(query, cache, table, context, **how)
