"""The 8-bit cache on the GPU: stored bytes against the layout restated token by token, attention and weights against 64 bits.

Tolerances.  Stored bytes, rows read back, kept places and moved weights are exact.  Attention: a logit is off by `off` at most
(``kv8_reference.attention``), by 2^-24 |x| for each of two more roundings, and its power of two by 2^-22, so a weight p by d = 2 off + 2^-20 of itself, the sum that
divides it included; a weight times its scale goes to fp16, by 2^-12 of itself
(a second time, by 2^-23, where the output is not bf16) or by 2^-35 of the largest; sums of up to 400 records of a warp, cut 24 bits below them, by
2^-16.  So an output by (2 d + 2^-12 or 2^-15) max |V| and half a step of its type.  The log-sum-exp by off + 2^-20 and four roundings of itself; an account of weights by d and 2^-20 of itself; a
head's weight below 2^-126, where fp32 has no normal numbers, counts as 0: 2^-126 for each head.
"""
import math
import subprocess
import sys

import pytest
import torch

import kv8_reference as ref
from open_ommx_serve_b200 import _lib
from open_ommx_serve_b200 import ommx_kv8_alloc, ommx_kv8_append, ommx_kv8_decode_attention, ommx_kv8_evict, ommx_kv8_gather
from open_ommx_serve_b200.attention.kv8 import kv8_workspace_floats

pytestmark = pytest.mark.gpu
DEV = "cuda"
I8, E4M3, BF16, F16, F32 = torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32
I32 = torch.int32


def tables(lens, page, spare=2, seed=0, dtype=I32):
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=gen)
    table = torch.zeros(len(lens), max(need + [1]) + 1, dtype=dtype)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(dtype)
        at += n
    return table, sum(need) + spare


def cumulated(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


def random_cache(P, H, D, page, code, seed=0, lo=118, hi=126):
    """Codes and scales of every valid kind, and weights: on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    c = ommx_kv8_alloc(P, H, D, page_size=page, dtype=code, weight=True, device="cpu")
    raw = torch.randint(0, 256, c["codes"].shape, generator=gen, dtype=torch.uint8)
    if code == I8:
        raw[raw == 128] = 129
    else:
        raw[(raw & 127) == 127] -= 1
    c["codes"].view(torch.uint8).copy_(raw)
    c["scales"].copy_(torch.randint(lo, hi, c["scales"].shape, generator=gen, dtype=torch.uint8))
    c["weight"].copy_(torch.rand(c["weight"].shape, generator=gen))
    return c


def to_gpu(c):
    return {k: v.to(DEV) for k, v in c.items()}


def rows(T, H, D, dtype, gen, wide=0, spread=1.0):
    x = torch.randn(T, 2 * H, D + wide, generator=gen) * torch.exp(spread * torch.randn(T, 1, 1, generator=gen))
    return x.to(dtype)[..., :D]


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


# ---- append and read back -------------------------------------------------------------------------------------------
APPENDS = [
    # D, page, H, dtype, lens, new, pad
    (128, 16, 2, BF16, [20], [1], 0),
    (128, 16, 3, BF16, [40, 17, 5], [33, 1, 5], 3),
    (128, 32, 2, F16, [70, 31, 64], [37, 2, 64], 1),
    (128, 64, 9, F32, [130, 63], [100, 63], 0),
    (64, 16, 1, BF16, [50, 16, 1, 33], [20, 16, 1, 0], 0),
    (64, 32, 5, F16, [95, 33], [95, 3], 2),
    (64, 128, 4, F32, [300], [211], 0),
    (64, 256, 1, BF16, [600, 255], [345, 7], 0),
]


@pytest.mark.parametrize("D,page,H,dtype,lens,new,pad", APPENDS)
@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("form", ["sliced", "odd strides"])
def test_append_stores_the_layouts_bytes(D, page, H, dtype, lens, new, pad, code, form):
    gen = torch.Generator().manual_seed(7)
    starts = cumulated(new)
    n, T = starts[-1], starts[-1] + pad
    table, P = tables(lens, page, seed=3, dtype=torch.int64 if page == 32 else I32)
    cache = random_cache(P, H, D, page, code, seed=5)
    x = rows(T, H, D, dtype, gen, wide=0 if form == "sliced" else 3)
    gpu = to_gpu(cache)
    xd = torch.empty_strided(x.size(), x.stride(), dtype=dtype, device=DEV)
    xd.copy_(x)
    status, length = i32([0]), i32(lens)
    ref.append(cache["codes"], cache["scales"], cache["weight"], table, lens, starts, x[:, :H], x[:, H:])
    for again in range(2):                                # the same rows again change nothing
        ommx_kv8_append(xd[:, :H], xd[:, H:], gpu["codes"], gpu["scales"], table.to(DEV), length, row_start=i32(starts), weight=gpu["weight"], status=status)
        assert int(status) == 0
        for name in cache:
            assert same(gpu[name], cache[name]), name
    for out in (dtype, F32):
        ko, vo = (torch.full((T, H, D), 9.0, dtype=out, device=DEV) for _ in range(2))
        ommx_kv8_gather(gpu["codes"], gpu["scales"], table.to(DEV), length, ko, vo, row_start=i32(starts), status=status)
        for b in range(len(lens)):
            wk, wv = ref.sequence(cache["codes"], cache["scales"], table[b], lens[b])
            for got, want in ((ko, wk), (vo, wv)):
                assert torch.equal(got[starts[b]:starts[b + 1]].cpu(), want[:, lens[b] - new[b]:].transpose(0, 1).float().to(out))
        assert int(status) == 0 and bool((ko[n:] == 9).all()) and bool((vo[n:] == 9).all())


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_scales_grow_a_token_at_a_time(code, dtype):
    """Steps of one row: sizes that rise, fall, vanish; zeros first and zeros after; no row_start, and weights of nobody's."""
    H, D, page, B = 3, 128, 16, 4
    gen = torch.Generator().manual_seed(1)
    table, P = tables([48] * B, page, seed=2)
    cache = random_cache(P, H, D, page, code, seed=3)
    cache["weight"] = None
    gpu = {k: v.to(DEV) for k, v in cache.items() if v is not None}
    sizes = [0.0, 0.0, 2.0 ** -9, 1.0, 0.5, 300.0, 0.0, 300.0, 2.0 ** -20, 5.0, 0.0, 6.0e4, 1.0, 1.0, 0.1, 3.0, 2.0 ** -14, 0.0, 1.0]
    for t, size in enumerate(sizes):
        x = (rows(B, H, D, F32, gen) * size).clamp(-60000, 60000).to(dtype)
        lens = [t + 1] * B
        ref.append(cache["codes"], cache["scales"], None, table, lens, list(range(B + 1)), x[:, :H], x[:, H:])
        xd = x.to(DEV)
        ommx_kv8_append(xd[:, :H], xd[:, H:], gpu["codes"], gpu["scales"], table.to(DEV), i32(lens))
        assert same(gpu["codes"], cache["codes"]) and same(gpu["scales"], cache["scales"]), t


@pytest.mark.parametrize("code", [I8, E4M3])
def test_numbers_at_every_edge(code):
    """Largest values at and beside each unit's limit, ties between codes, subnormal codes, the smallest and the largest numbers of the types."""
    H, D, page = 1, 128, 16
    top = ref.TOP[code]
    for dtype, span in ((BF16, range(-133, 128, 9)), (F32, range(-149, 128, 11)), (F16, range(-24, 16, 3))):
        table, P = tables([16] * len(span), page)
        cache = random_cache(P, H, D, page, code, seed=4)
        gpu = to_gpu(cache)
        x = torch.zeros(16 * len(span), 2 * H, D)
        for i, e in enumerate(span):
            m = torch.tensor([1.0, -1.0, 127 / 128, 127.5 / 128, 1.75, 1.7578125, -1.7421875, 1.984375, 1.9921875, 0.5, 1.5 / 128, 2.5 / 128, 3.5 / 128, 2.0 ** -10, 2.0 ** -9, 2.0 ** -16])
            values = torch.ldexp(m.double(), torch.tensor(e)).float()
            x[16 * i, 0, :16] = values[:8].repeat(2)
            x[16 * i + 1, 0, :16] = values
            x[16 * i, 1, i % 16] = top * 2.0 ** max(min(e, 100), -100)
            x[16 * i, 1, 20:28] = torch.arange(8) * 2.0 ** max(min(e, 100), -100) / 2
        x = x.to(dtype)
        lens, starts = [16] * len(span), cumulated([16] * len(span))
        ref.append(cache["codes"], cache["scales"], cache["weight"], table, lens, starts, x[:, :H], x[:, H:])
        ommx_kv8_append(x[:, :H].to(DEV), x[:, H:].to(DEV), gpu["codes"], gpu["scales"], table.to(DEV), i32(lens), row_start=i32(starts), weight=gpu["weight"])
        for name in cache:
            assert same(gpu[name], cache[name]), (dtype, name)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_that_are_not_finite(code, dtype):
    H, D, page = 2, 64, 32
    gen = torch.Generator().manual_seed(6)
    lens, new = [40, 21, 5], [9, 3, 2]
    starts = cumulated(new)
    table, P = tables(lens, page)
    x = rows(starts[-1], H, D, dtype, gen)
    x[3, 1, 5], x[9, 2, 0], x[10, 3, 7] = math.nan, math.inf, -math.inf
    if dtype != F16:
        x[13, 0, 0] = 3e38                                # finite, beyond 2^126
    for bad in (True, False):
        if not bad:
            x = torch.nan_to_num(x.float(), nan=0.0, posinf=1.0, neginf=1.0).to(dtype)
        cache = random_cache(P, H, D, page, code, seed=8)
        gpu, status = to_gpu(cache), i32([0])
        ref.append(cache["codes"], cache["scales"], cache["weight"], table, lens, starts, x[:, :H], x[:, H:])
        ommx_kv8_append(x[:, :H].to(DEV), x[:, H:].to(DEV), gpu["codes"], gpu["scales"], table.to(DEV), i32(lens), row_start=i32(starts), weight=gpu["weight"], status=status)
        for name in cache:
            assert same(gpu[name], cache[name]), name
        assert int(status) == (_lib.ST_NONFINITE if bad else 0)


@pytest.mark.parametrize("B", [33, 300, 700])
def test_many_sequences(B):
    """More sequences than a warp, and than a block, has threads; some without rows."""
    H, D, page, code = 1, 64, 16, I8
    gen = torch.Generator().manual_seed(9)
    lens = torch.randint(1, 60, (B,), generator=gen).tolist()
    new = [min(n, m) for n, m in zip(lens, torch.randint(0, 35, (B,), generator=gen).tolist())]
    starts = cumulated(new)
    table, P = tables(lens, page)
    cache = random_cache(P, H, D, page, code)
    gpu, status = to_gpu(cache), i32([0])
    x = rows(starts[-1] + 4, H, D, BF16, gen)
    ref.append(cache["codes"], cache["scales"], cache["weight"], table, lens, starts, x[:, :H], x[:, H:])
    ommx_kv8_append(x[:, :H].to(DEV), x[:, H:].to(DEV), gpu["codes"], gpu["scales"], table.to(DEV), i32(lens), row_start=i32(starts), weight=gpu["weight"], status=status)
    for name in cache:
        assert same(gpu[name], cache[name]), name
    ko, vo = (torch.zeros(starts[-1] + 4, H, D, dtype=F32, device=DEV) for _ in range(2))
    ommx_kv8_gather(gpu["codes"], gpu["scales"], table.to(DEV), i32(lens), ko, vo, row_start=i32(starts), status=status)
    for b in range(0, B, 7):
        wk, wv = ref.sequence(cache["codes"], cache["scales"], table[b], lens[b])
        assert torch.equal(ko[starts[b]:starts[b + 1]].cpu().double(), wk[:, lens[b] - new[b]:].transpose(0, 1))
        assert torch.equal(vo[starts[b]:starts[b + 1]].cpu().double(), wv[:, lens[b] - new[b]:].transpose(0, 1))
    assert int(status) == 0


@pytest.mark.parametrize("B", [4, 40])
def test_bad_ranges_lengths_and_pages_are_reported_and_skipped(B):
    """Sequences 0 and 1 are sound, 2 is not in one way or another, 3 and on are: they are stored, and nothing else changes."""
    H, D, page, code = 2, 64, 16, E4M3
    gen = torch.Generator().manual_seed(10)
    lens = [20, 5] + [18] * (B - 2)
    new = [3] * B
    starts = cumulated(new)
    x = rows(starts[-1], H, D, BF16, gen)
    xd = x.to(DEV)
    table, P = tables(lens, page)
    ways = [("length", dict(length=-1), _lib.ST_BAD_LENGTH), ("length", dict(length=2), _lib.ST_BAD_LENGTH), ("length", dict(length=10 ** 6), _lib.ST_BAD_LENGTH),
            ("page", dict(page=P), _lib.ST_BAD_PAGE), ("page", dict(page=-1), _lib.ST_BAD_PAGE), ("page", dict(page=2 ** 31 - 1), _lib.ST_BAD_PAGE)]
    for _, way, want in ways:
        cache = random_cache(P, H, D, page, code)
        gpu, status, t, given = to_gpu(cache), i32([0]), table.clone(), list(lens)
        if "length" in way:
            given[2] = way["length"]
        else:
            t[2, 1] = way["page"]
        sound = list(lens)
        lacks = list(starts)
        # the reference stores sequence 2's rows on a copy that is thrown away: its first block's rows are stored where only the second page is bad
        for b in range(B):
            if b == 2:
                if "page" in way:                         # tokens 15 lie on the first page, 16 and 17 on the bad one
                    ref.append(cache["codes"], cache["scales"], cache["weight"], t[2:3], [16], [0, 1], x[lacks[2]:lacks[2] + 1, :H], x[lacks[2]:lacks[2] + 1, H:])
                continue
            ref.append(cache["codes"], cache["scales"], cache["weight"], t[b:b + 1], [sound[b]], [0, 3], x[lacks[b]:lacks[b] + 3, :H], x[lacks[b]:lacks[b] + 3, H:])
        ommx_kv8_append(xd[:, :H], xd[:, H:], gpu["codes"], gpu["scales"], t.to(DEV), i32(given), row_start=i32(starts), weight=gpu["weight"], status=status)
        assert int(status) == want, way
        for name in cache:
            assert same(gpu[name], cache[name]), (way, name)
        status.zero_()
        ko, vo = (torch.full((starts[-1], H, D), 9.0, dtype=F32, device=DEV) for _ in range(2))
        ommx_kv8_gather(gpu["codes"], gpu["scales"], t.to(DEV), i32(given), ko, vo, row_start=i32(starts), status=status)
        assert int(status) == want
        wk, _ = ref.sequence(cache["codes"], cache["scales"], t[3], 18)
        assert torch.equal(ko[9:12].cpu().double(), wk[:, 15:].transpose(0, 1))
        assert bool((ko[7 if "page" in way else 6:9] == 9).all())
    # ranges that are none of the rows: two sequences share a bound, so the neighbour goes with it
    for bad in (-1, starts[-1] + 1, 2 ** 31 - 1, -2 ** 31):
        cache = random_cache(P, H, D, page, code)
        gpu, status, given = to_gpu(cache), i32([0]), list(starts)
        given[2] = bad
        for b in range(B):
            if b not in (1, 2):
                ref.append(cache["codes"], cache["scales"], cache["weight"], table[b:b + 1], [lens[b]], [0, 3], x[3 * b:3 * b + 3, :H], x[3 * b:3 * b + 3, H:])
        ommx_kv8_append(xd[:, :H], xd[:, H:], gpu["codes"], gpu["scales"], table.to(DEV), i32(lens), row_start=i32(given), weight=gpu["weight"], status=status)
        assert int(status) == _lib.ST_BAD_LENGTH
        for name in cache:
            assert same(gpu[name], cache[name]), (bad, name)


def test_one_row_each_of_bad_sequences():
    """Without row_start: lengths of 0 and below, past the table, pages out of range."""
    H, D, page, code = 2, 128, 16, I8
    x = rows(5, H, D, BF16, torch.Generator().manual_seed(2))
    table, P = tables([20] * 5, page)
    cache = random_cache(P, H, D, page, code)
    gpu, status, t = to_gpu(cache), i32([0]), table.clone()
    t[3, 1] = P
    ref.append(cache["codes"], cache["scales"], cache["weight"], table[4:], [20], [0, 1], x[4:, :H], x[4:, H:])
    ommx_kv8_append(x[:, :H].to(DEV), x[:, H:].to(DEV), gpu["codes"], gpu["scales"], t.to(DEV), i32([0, -3, 49, 20, 20]), weight=gpu["weight"], status=status)
    assert int(status) == _lib.ST_BAD_LENGTH | _lib.ST_BAD_PAGE
    for name in cache:
        assert same(gpu[name], cache[name]), name


# ---- attention ------------------------------------------------------------------------------------------------------
def check(q, cache, table, lens, o, lse, *, sm_scale=None, cap=0.0, window=None, sinks=0, weight=None, before=None, keep=1.0):
    D, page = q.shape[-1], 16 * cache["codes"].shape[2]
    sm = D ** -0.5 if sm_scale is None else sm_scale
    half = torch.finfo(o.dtype).eps / 2
    H, group = cache["codes"].shape[1], q.shape[1] // cache["codes"].shape[1]
    want_weight = None if weight is None else before.double().clone()
    off_weight = None if weight is None else torch.zeros_like(want_weight)
    for b, n in enumerate(lens):
        k, v = ref.sequence(cache["codes"], cache["scales"], table[b], n)
        seen = ref.visible(n, window, sinks)
        wo, wl, p, off = ref.attention(q[b], k[:, seen], v[:, seen], sm, cap)
        if len(seen) == 0:
            assert bool((o[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        d = (2 * off + 2.0 ** -20)[:, None]
        vmax = v[:, seen].abs().amax((1, 2)).repeat_interleave(group)[:, None]
        err = (o[b].double() - wo).abs()
        tol = (2 * d + 2.0 ** (-12 if o.dtype == BF16 else -15)) * vmax + half * wo.abs() + torch.finfo(o.dtype).tiny
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()))
        err, tol = (lse[b].double() - wl).abs(), off + 2.0 ** -20 + 2.0 ** -22 * wl.abs()
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()))
        if weight is not None:
            t = torch.arange(n)
            ids, at = table[b, t // page].long(), t % page
            add, tol = torch.zeros(H, n, dtype=torch.float64, device=q.device), torch.zeros(H, n, dtype=torch.float64, device=q.device)
            add[:, seen] = p.view(H, group, -1).sum(1)
            tol[:, seen] = (p * d).view(H, group, -1).sum(1)
            now = want_weight[ids, :, at].T.clone() * keep + add
            want_weight[ids, :, at], off_weight[ids, :, at] = now.T, (tol + 2.0 ** -20 * now.abs() + group * 2.0 ** -126).T
    if weight is not None:
        err = (weight.double() - want_weight).abs()
        assert bool((err <= off_weight).all()), float((err - off_weight).max())


def attend(lens, H, Hq, D, page, code, dtype=BF16, out=None, seed=0, weigh=False, keep=1.0, cache=None, q_scale=1.0, spare=2, max_len="longest", table_type=I32, **more):
    gen = torch.Generator().manual_seed(seed)
    table, P = tables(lens, page, seed=seed, spare=spare, dtype=table_type)
    cache = to_gpu(cache or random_cache(P, H, D, page, code, seed=seed))
    q = (torch.randn(len(lens), Hq, D, generator=gen) * q_scale).to(dtype).to(DEV)
    o, lse = torch.full((len(lens), Hq, D), 7.0, dtype=out or dtype, device=DEV), torch.full((len(lens), Hq), 7.0, device=DEV)
    status = i32([0])
    before = cache["weight"].clone()
    if weigh:
        more = dict(more, weight=cache["weight"], keep=keep)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, status=status,
                              max_seq_len=max(lens) if max_len == "longest" else max_len, **more)
    assert int(status) == 0
    kw = dict(sm_scale=more.get("sm_scale"), cap=more.get("logit_cap", 0.0), window=more.get("window"), sinks=more.get("sink_tokens", 0))
    check(q, cache, table.to(DEV), lens, o, lse, **kw, weight=cache["weight"] if weigh else None, before=before, keep=keep)
    return q, cache, table, o, lse


@pytest.mark.parametrize("D,page,H,Hq,dtype,code", [
    (128, 16, 2, 8, BF16, I8), (128, 32, 1, 1, F16, E4M3), (64, 16, 3, 6, BF16, E4M3), (64, 64, 2, 10, F16, I8), (128, 16, 1, 7, BF16, E4M3),
    (128, 128, 2, 16, F16, I8), (64, 256, 1, 9, BF16, I8), (128, 16, 1, 40, F16, E4M3)])
@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [0, 100, 33, 0, 257, 512]])
def test_attention(lens, D, page, H, Hq, dtype, code):
    attend(lens, H, Hq, D, page, code, dtype)
    attend(lens, H, Hq, D, page, code, dtype, out=F32, seed=1, weigh=True, keep=0.5, table_type=torch.int64)


@pytest.mark.parametrize("lens,H,Hq", [
    ([700], 2, 8), ([4000], 1, 4),                        # a cluster to a row
    ([6000, 1, 5000], 2, 8), ([33000], 1, 8),             # rows in pieces
    ([4000] + [10] * 40, 4, 8),                           # even shares of all rows
    ([900] * 9 + [0, 1, 2000], 8, 64),                    # four-warp blocks
    ([300, 0, 511, 64] * 20, 4, 36)])                     # a block to a row, two blocks of heads
@pytest.mark.parametrize("code", [I8, E4M3])
def test_every_way_of_dealing(lens, H, Hq, code):
    attend(lens, H, Hq, 128, 16, code, BF16)
    attend(lens, H, Hq, 64, 32, code, F16, seed=2, weigh=True, max_len=None)
    attend(lens, H, Hq, 128, 64, code, BF16, out=F32, seed=3, window=333, sink_tokens=5)


@pytest.mark.parametrize("lens,H,Hq,D", [([4700], 8, 32, 128), ([5009, 31, 0], 1, 8, 128), ([9000], 8, 32, 64), ([6000, 4999, 1, 16, 17], 3, 9, 64), ([4800] * 2, 7, 7, 128), ([4800] * 2, 8, 8, 128), ([600] * 36, 1, 4, 64)])
@pytest.mark.parametrize("code", [I8, E4M3])
def test_clusters_of_every_size(lens, H, Hq, D, code):
    """Rows in clusters of eight blocks of sixteen warps, just fewer and just more of them than run at once; and as many as would be one more than run at
    once in clusters of eight of eight warps."""
    attend(lens, H, Hq, D, 32, code, BF16, weigh=True, keep=0.5)
    attend(lens, H, Hq, D, 32, code, F16, out=F32)


def test_a_first_call_may_be_captured():
    """In a process of its own: what a call asks of the device for the first time it may ask while a graph is captured."""
    code = """
import torch
from open_ommx_serve_b200 import ommx_kv8_alloc, ommx_kv8_append, ommx_kv8_decode_attention, ommx_kv8_evict
c = ommx_kv8_alloc(400, 8, 128, weight=True, device="cuda")
k = torch.randn(5000, 8, 128, device="cuda")
table, length = torch.arange(400, dtype=torch.int32, device="cuda").view(1, -1), torch.tensor([5000], dtype=torch.int32, device="cuda")
starts, q, o, lse = torch.tensor([0, 5000], dtype=torch.int32, device="cuda"), torch.randn(1, 8, 128, device="cuda").bfloat16(), torch.empty(1, 8, 128, device="cuda"), torch.empty(1, 8, device="cuda")
kept, work = torch.empty(1, 8, 100, dtype=torch.int32, device="cuda"), torch.empty(1 << 21, device="cuda")
def step():
    ommx_kv8_append(k, k, c["codes"], c["scales"], table, length, row_start=starts, weight=c["weight"])
    ommx_kv8_decode_attention(q, c["codes"], c["scales"], table, length, o, lse, weight=c["weight"], keep=0.0, workspace=work, max_seq_len=5000)
    ommx_kv8_evict(c["codes"], c["scales"], c["weight"], table, length, kept)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
first = [x.clone() for x in (o, lse, kept)]
step()
assert all(torch.equal(a, b) for a, b in zip(first, (o, lse, kept)))
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (15, 3), (16, 16), (17, 17), (40, 0), (100, 33), (99, 1000), (1000, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("code", [I8, E4M3])
def test_window_and_first_tokens(window, sinks, code):
    lens = [1, 14, 16, 17, 33, 40, 41, 99, 130, 131, 0, 611]
    for weigh in (False, True):
        attend(lens, 2, 4, 64, 16, code, BF16, window=window, sink_tokens=sinks, weigh=weigh, keep=0.9)
    attend([5000, 4999], 1, 8, 128, 32, code, F16, window=window, sink_tokens=sinks, weigh=True, keep=0.0, max_len=None)


@pytest.mark.parametrize("code,D", [(I8, 128), (E4M3, 64)])
def test_first_tokens_and_lengths_near_the_end_of_32_bits(code, D):
    """More first tokens than any sequence has beside a window; and a sequence of up to 2^31 - 2^10 tokens, as many as are
    counted, whose table names four pages over and over, through a window."""
    attend([1, 16, 40, 611, 0, 3000], 2, 4, D, 16, code, window=30, sink_tokens=2 ** 31 - 1, weigh=True, keep=0.5)
    page, H, Hq, sinks, window = 256, 2, 8, 20, 1000
    cache = to_gpu(random_cache(4, H, D, page, code))
    table = (torch.arange(2 ** 31 // page, dtype=I32, device=DEV) % 4).view(1, -1)
    k, v = ref.sequence(cache["codes"], cache["scales"], torch.arange(4), 4 * page)
    q = torch.randn(1, Hq, D, device=DEV).bfloat16()
    for length in (2 ** 31 - 2 ** 10 - x for x in (0, 1, 15, 16, 17)):
        o, lse, status = torch.empty(1, Hq, D, device=DEV), torch.empty(1, Hq, device=DEV), i32([0])
        ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table, i32([length]), o, lse, window=window, sink_tokens=sinks, status=status)
        assert int(status) == 0
        at = torch.tensor(list(range(sinks)) + [t % (4 * page) for t in range(length - window, length)])
        wo, wl, _, off = ref.attention(q[0], k[:, at], v[:, at], D ** -0.5)
        assert float((o[0].double() - wo).abs().max()) <= (4 * float(off.max()) + 2.0 ** -14) * float(v.abs().max())
        assert bool(((lse[0].double() - wl).abs() <= off + 2.0 ** -20 + 2.0 ** -22 * wl.abs()).all())
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table, i32([2 ** 31 - 1]), o, lse, window=window, sink_tokens=sinks, status=status)
    assert int(status) == _lib.ST_BAD_LENGTH


@pytest.mark.parametrize("code,D", [(I8, 128), (E4M3, 64)])
def test_windows_of_many_rows(code, D):
    """A window's rows in a block each, where there are blocks for all and not for two each; and more rows than that."""
    lens = [[1200, 0, 650, 17, 900, 1, 601, 600][b % 8] + b // 8 for b in range(50)]
    attend(lens, 8, 8, D, 16, code, BF16, window=600, sink_tokens=5, weigh=True, keep=0.5)
    attend([700] * 76, 8, 8, D, 16, code, F16, window=600)


def test_what_is_not_visible_is_not_read():
    """Pages wholly outside the window may be anybody's, or none: their table entries are out of range here."""
    lens, page = [400, 390], 16
    table, P = tables(lens, page)
    cache = to_gpu(random_cache(P, 2, 64, page, I8))
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    got = []
    for hide in (False, True):
        t = table.clone()
        if hide:
            t[:, 1:16] = 10 ** 6
        o, lse, status = torch.empty(2, 4, 64, device=DEV), torch.empty(2, 4, device=DEV), i32([0])
        ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], t.to(DEV), i32(lens), o, lse, window=130, sink_tokens=7, status=status)
        assert int(status) == 0
        got.append((o, lse))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("code,fill", [(I8, 0x80), (I8, 0x7F), (E4M3, 0x7F), (E4M3, 0xFF)])
def test_places_behind_the_last_token_may_hold_anything(code, fill):
    """The lowest int8 and e4m3's NaN in a record's unused tokens; scales of 255 on pages that nothing is on."""
    lens, page, H, D = [1, 9, 30, 50], 32, 2, 128
    table, P = tables(lens, page)
    cache = random_cache(P, H, D, page, code)
    raw = cache["codes"].view(torch.uint8)
    used = torch.zeros(P, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[table[b, t // page], t % page] = True
    raw.copy_(torch.where(used.view(P, 1, page // 16, 1, 16, 1), raw, torch.full_like(raw, fill)))
    cache["scales"].copy_(torch.where(used.view(P, 1, page // 16, 16).any(-1, keepdim=True), cache["scales"], torch.full_like(cache["scales"], 255)))
    attend(lens, H, 8, D, page, code, cache=cache, weigh=True)
    attend(lens, H, 8, D, page, code, cache=cache, weigh=True, window=5, sink_tokens=2)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("more", [dict(logit_cap=30.0), dict(logit_cap=1e-3), dict(sm_scale=0.0), dict(sm_scale=-0.3), dict(sm_scale=1.7, logit_cap=50.0), dict(sm_scale=1e-30)])
def test_caps_and_scales_of_logits(code, more):
    attend([40, 700, 3], 2, 8, 128, 16, code, out=F32, weigh=True, **more)
    attend([40, 700, 3], 2, 8, 64, 16, code, window=20, sink_tokens=3, **more)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("E", [1, 20, 60, 127, 200, 240])
def test_values_of_every_size(code, E):
    """Scales of values from 2^-126 up, alike or 2^12 apart from record to record; outputs in 32 bits hold to their own size."""
    lens, page, H, D = [5, 300, 2500], 16, 2, 64
    for spread in (0, 6):
        table, P = tables(lens, page)
        cache = random_cache(P, H, D, page, code, seed=E)
        gen = torch.Generator().manual_seed(E)
        cache["scales"][..., 1] = (E + torch.randint(-spread, spread + 1, cache["scales"][..., 1].shape, generator=gen)).clamp(1, 245).to(torch.uint8)
        attend(lens, H, 8, D, page, code, out=F32, cache=cache, seed=E)


@pytest.mark.parametrize("code", [I8, E4M3])
def test_a_light_token_with_large_values_counts(code):
    """One record's values are 2^40 times the others' and its weights e^-25 of theirs: it is most of the output."""
    page, H, D, L = 16, 1, 128, 320
    table, P = tables([L], page)
    cache = random_cache(P, H, D, page, code, lo=120, hi=121)
    p = int(table[0, 11])
    cache["scales"][p, :, 0, 1] = 160
    q = torch.zeros(1, 4, D)
    q[..., 0] = 1.0
    sign = torch.ones(P, 16)
    sign[p] = -1.0
    top = 100.0 if code == I8 else 96.0
    cache["codes"][:, 0, 0, 0, :, 0] = (sign * top).to(torch.float32).to(code)
    cache = to_gpu(cache)
    o, lse = torch.empty(1, 4, D, device=DEV), torch.empty(1, 4, device=DEV)
    sm = 12.5 / (top * 2.0 ** -7)
    ommx_kv8_decode_attention(q.bfloat16().to(DEV), cache["codes"], cache["scales"], table.to(DEV), i32([L]), o, lse, sm_scale=sm)
    k, v = ref.sequence(cache["codes"], cache["scales"], table[0].to(DEV), L)
    want, wl, _, off = ref.attention(q[0].bfloat16().to(DEV), k, v, sm)
    # 16 tokens make the output up: (2 d + 2^-15) of what they add, by their largest value
    share = torch.softmax(k[0] @ q[0, 0].double().to(DEV) * sm, 0)[176:192].sum()
    tol = (4 * off.max() + 2.0 ** -14) * share * v[0, 176:192].abs().max() + 2.0 ** -15 * v[0, :176].abs().max()
    assert bool(((o[0].double() - want).abs() <= tol).all()), float((o[0].double() - want).abs().max() / tol)


@pytest.mark.parametrize("size", [2.0 ** -90, 2.0 ** -30, 2.0 ** 20, 2.0 ** 100])
def test_queries_and_keys_of_every_size(size):
    lens, page, H, D = [40, 900], 16, 2, 128
    table, P = tables(lens, page)
    for code in (I8, E4M3):
        cache = random_cache(P, H, D, page, code)
        cache["scales"][..., 0] = max(1, min(245, 120 - round(math.log2(size))))
        attend(lens, H, 8, D, page, code, BF16, out=F32, cache=cache, q_scale=size)


def test_channels_of_a_query_far_below_its_largest():
    """Where all that a logit gets is from bf16 channels 2^-20 of the largest, it is off by the rounding of those, a few steps wide, and no more."""
    page, H, D, L = 16, 1, 64, 64
    table, P = tables([L], page)
    cache = random_cache(P, H, D, page, I8)
    cache["codes"][:, 0, 0, 0, :, 0] = 0                  # no key has anything in the large channel
    q = torch.randn(1, 2, D, generator=torch.Generator().manual_seed(0)) * 2.0 ** -20
    q[..., 0] = 1.0
    q = q.bfloat16().to(DEV)
    cache = to_gpu(cache)
    o, lse = torch.empty(1, 2, D, device=DEV), torch.empty(1, 2, device=DEV)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32([L]), o, lse, sm_scale=2.0 ** 20)
    check(q, cache, table.to(DEV), [L], o, lse, sm_scale=2.0 ** 20)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_queries_that_are_not_finite(code, bad, cap):
    """The head whose row it is gives NaN; the others of its product hold to their bounds (their references move when its do)."""
    for lens in ([40, 0, 700], [6000, 20, 3000]):
        table, P = tables(lens, 16)
        cache = to_gpu(random_cache(P, 2, 128, 16, code))
        q = torch.randn(3, 12, 128, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
        o, lse = torch.empty(2, 3, 12, 128, device=DEV), torch.empty(2, 3, 12, device=DEV)
        for i in range(2):
            given = q.clone()
            if i:
                given[0, 7, 3], given[2, 0, 127] = bad, bad
            ommx_kv8_decode_attention(given, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o[i], lse[i], logit_cap=cap)
        hit = torch.zeros(3, 12, dtype=torch.bool, device=DEV)
        hit[0, 7] = hit[2, 0] = True
        assert bool(o[1][hit].isnan().all()) and bool(lse[1][hit].isnan().all())
        check(q, cache, table.to(DEV), lens, torch.where(hit[..., None], o[0], o[1]), torch.where(hit, lse[0], lse[1]), cap=cap)


@pytest.mark.parametrize("code,D,H,page", [(I8, 128, 8, 16), (E4M3, 64, 4, 64)])
def test_offsets_past_32_bits(code, D, H, page):
    """The same sequences at the front of a small cache and at the back of one of more than 2^32 bytes: append, read back, attend, evict."""
    need = 12
    big = 2 ** 32 // (H * page * 2 * D) + 2 * need
    gen = torch.Generator().manual_seed(3)
    lens = [5 * page - 3, 4 * page]
    x, q = rows(sum(lens), H, D, BF16, gen).to(DEV), torch.randn(2, 4 * H, D, generator=gen).bfloat16().to(DEV)
    got = []
    for pages in (need, big):
        c = ommx_kv8_alloc(pages, H, D, page_size=page, dtype=code, weight=True, device=DEV)
        where = (c["codes"], c["scales"])
        table = (torch.arange(need, device=DEV, dtype=I32).flip(0).view(2, 6) + (pages - need)).contiguous()
        length, starts = i32(lens), i32(cumulated(lens))
        ommx_kv8_append(x[:, :H], x[:, H:], *where, table, length, row_start=starts, weight=c["weight"])
        o, lse, kept = torch.empty(2, 4 * H, D, device=DEV), torch.empty(2, 4 * H, device=DEV), torch.empty(2, H, 40, dtype=I32, device=DEV)
        status = i32([0])
        ommx_kv8_decode_attention(q, *where, table, length, o, lse, weight=c["weight"], keep=0.5, status=status)
        weights = c["weight"][pages - need:].clone()
        ommx_kv8_evict(*where, c["weight"], table, length, kept, sink_tokens=1, recent_tokens=3, len_out=length, status=status)
        k, v = (torch.empty(80, H, D, device=DEV) for _ in range(2))
        ommx_kv8_gather(*where, table, length, k, v, row_start=i32([0, 40, 80]), status=status)
        assert int(status) == 0
        got.append((o, lse, weights, kept, k, v, c["weight"][pages - need:].clone(), c["codes"].view(torch.uint8)[pages - need:].clone(), c["scales"][pages - need:].clone()))
        assert pages == need or not bool(c["scales"][:need].any())         # what 32 bits would have reached
        del c, where
    for a, b in zip(*got):
        assert same(a, b)


def test_strides_alignment_and_padding():
    """q in slices of one projection and off 16-byte boundaries, outputs with gaps, lse rows apart; what lies between stays."""
    lens, page, H, Hq, D = [50, 0, 700], 16, 2, 6, 128
    table, P = tables(lens, page)
    cache = to_gpu(random_cache(P, H, D, page, I8))
    base = torch.randn(3, Hq + 2, D + 5, device=DEV).bfloat16()
    for q in (base[:, 1:Hq + 1, :D], base[:, 1:Hq + 1, 3:D + 3]):
        o_all, l_all = torch.full((3, Hq + 3, D + 7), 5.0, device=DEV, dtype=F16), torch.full((3, Hq + 9), 5.0, device=DEV)
        o, lse = o_all[:, 2:Hq + 2, 1:D + 1], l_all[:, :Hq]
        ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse)
        check(q, cache, table.to(DEV), lens, o, lse)
        o.fill_(5.0), lse.fill_(5.0)
        assert bool((o_all == 5).all()) and bool((l_all == 5).all())


def test_pages_out_of_range_and_lengths_past_the_table():
    """Tokens on pages that are not there are left out and reported; so is what lies past the table."""
    page, H, D = 16, 2, 64
    lens = [100, 60, 33]
    table, P = tables(lens, page)
    cache = to_gpu(random_cache(P, H, D, page, E4M3))
    before = cache["weight"].clone()
    q = torch.randn(3, 4, D, device=DEV).bfloat16()
    t = table.clone()
    t[0, 2], t[1, 0] = -1, P
    o, lse, status = torch.empty(3, 4, D, device=DEV), torch.empty(3, 4, device=DEV), i32([0])
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], t.to(DEV), i32(lens), o, lse, status=status, weight=cache["weight"])
    assert int(status) == _lib.ST_BAD_PAGE
    for b, gone in ((0, 2), (1, 0)):
        k, v = ref.sequence(cache["codes"], cache["scales"], table[b].to(DEV), lens[b])
        there = torch.tensor([i for i in range(lens[b]) if i // page != gone])
        wo, wl, _, off = ref.attention(q[b], k[:, there], v[:, there], D ** -0.5)
        assert float((o[b].double() - wo).abs().max()) <= (4 * float(off.max()) + 2.0 ** -14) * float(v.abs().max())
        assert same(cache["weight"][table[b, gone]], before[table[b, gone]])         # the page it should have been
    for n in (-5, 10 ** 6):
        status.zero_()
        ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32([lens[0], n, lens[2]]), o, lse, status=status)
        assert int(status) & _lib.ST_BAD_LENGTH
        check(q[2:], cache, table[2:].to(DEV), lens[2:], o[2:], lse[2:])
        assert n > 0 or bool((lse[1] == -math.inf).all())


def test_lengths_past_max_seq_len():
    """An output does not depend on max_seq_len; an account past it is not kept, and reported."""
    lens, page, H, D = [800, 90, 3000], 16, 2, 128
    table, P = tables(lens, page)
    cache = to_gpu(random_cache(P, H, D, page, I8))
    before, q = cache["weight"].clone(), torch.randn(3, 8, D, device=DEV).bfloat16()
    for most in (1, 100, 513, 2999):
        o, lse, status = torch.empty(3, 8, D, device=DEV), torch.empty(3, 8, device=DEV), i32([0])
        ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, max_seq_len=most, status=status)
        assert int(status) == 0
        check(q, cache, table.to(DEV), lens, o, lse)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, max_seq_len=100, status=status, weight=cache["weight"])
    assert int(status) == _lib.ST_BAD_LENGTH
    check(q, cache, table.to(DEV), lens, o, lse)
    check(q[1:2], cache, table[1:2].to(DEV), lens[1:2], o[1:2], lse[1:2])
    t = torch.arange(90)
    got = cache["weight"][table[1, t // page].long(), :, t % page]
    assert bool((got > before[table[1, t // page].long(), :, t % page]).any())
    for b in (0, 2):                                      # past the 112 tokens that have a place nothing changes
        t = torch.arange(112, lens[b])
        ids = table[b, t // page].long()
        assert torch.equal(cache["weight"][ids, :, t % page], before[ids, :, t % page])


@pytest.mark.parametrize("most,H", [(200, 32), (500, 18), (3000, 32), (40000, 32)])
def test_an_account_leaves_sequences_of_too_many_records_alone(most, H):
    """A sequence of so many records that they are not counted, beside a short one: its weights stay as they were, and where records are dealt out (the
    last two) both sequences'. Records in a block to a row, a cluster to a row, and in shares with the account beside the join and behind it."""
    page, D, P = 256, 64, 6
    cache = to_gpu(random_cache(P, H, D, page, I8))
    before = cache["weight"].clone()
    table = (torch.arange(2 ** 31 // page, dtype=I32, device=DEV) % 4).repeat(2, 1)
    table[1, 0] = 5
    lens = [2 ** 31 - 2 ** 10, 180]
    q, o, lse, status = torch.randn(2, H, D, device=DEV).bfloat16(), torch.empty(2, H, D, device=DEV), torch.empty(2, H, device=DEV), i32([0])
    work = torch.full((kv8_workspace_floats(2, H, D, most, weight=True),), 7.0, device=DEV)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table, i32(lens), o, lse, weight=cache["weight"], keep=0.5, workspace=work, max_seq_len=most, status=status)
    assert int(status) == _lib.ST_BAD_LENGTH
    assert torch.equal(cache["weight"][:5], before[:5])
    if most <= 500:
        short = table[1:, :1].contiguous()
        check(q[1:], cache, short, lens[1:], o[1:], lse[1:], weight=cache["weight"], before=before, keep=0.5)
    else:
        assert torch.equal(cache["weight"], before)


# ---- the account of weights ------------------------------------------------------------------------------------------
def test_weights_accumulate_over_steps():
    lens, page, H, Hq, D = [35, 610, 0], 32, 2, 12, 64
    table, P = tables(lens, page)
    for code in (I8, E4M3):
        cache = to_gpu(random_cache(P, H, D, page, code))
        for step, keep in enumerate((1.0, 0.75, 0.0, -0.5)):
            q = torch.randn(3, Hq, D, device=DEV).half()
            before = cache["weight"].clone()
            if keep == 0.0:
                cache["weight"].fill_(math.nan)           # not read
                before = torch.nan_to_num(before * 0)
            o, lse = torch.empty(3, Hq, D, device=DEV), torch.empty(3, Hq, device=DEV)
            ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, weight=cache["weight"], keep=keep)
            cache["weight"] = torch.nan_to_num(cache["weight"])
            check(q, cache, table.to(DEV), lens, o, lse, weight=cache["weight"], before=before, keep=keep)


def test_weights_beside_those_before():
    """weight_before is another tensor, and stays; tokens behind the last keep what weight held."""
    lens, page, H, Hq, D = [35, 610], 16, 2, 4, 128
    table, P = tables(lens, page)
    cache = to_gpu(random_cache(P, H, D, page, I8))
    before, q = torch.rand(P, H, page, device=DEV), torch.randn(2, Hq, D, device=DEV).bfloat16()
    held, kept = cache["weight"].clone(), before.clone()
    o, lse = torch.empty(2, Hq, D, device=DEV), torch.empty(2, Hq, device=DEV)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, weight=cache["weight"], weight_before=before, keep=0.5, window=50, sink_tokens=2)
    assert torch.equal(before, kept)
    used = torch.zeros(P, page, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        t = torch.arange(n)
        used[table[b, t // page].long(), t % page] = True
    assert torch.equal(cache["weight"].transpose(1, 2)[~used], held.transpose(1, 2)[~used])
    check(q, cache, table.to(DEV), lens, o, lse, window=50, sinks=2, weight=torch.where(used[:, None], cache["weight"], before), before=before, keep=0.5)
    # each head's weights add up to 1 (no keep)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, weight=cache["weight"], keep=0.0)
    for b, n in enumerate(lens):
        t = torch.arange(n)
        total = cache["weight"][table[b, t // page].long(), :, t % page].double().sum(0)
        assert bool(((total - Hq // H).abs() <= 2.0 ** -18 * Hq).all())


# ---- eviction --------------------------------------------------------------------------------------------------------
def evict(lens, H, D, page, code, budget, sinks=0, recent=0, seed=0, apart=False, weights=None, alias=False, max_len=None, table_type=I32):
    table, P = tables(lens, page, seed=seed, dtype=table_type)
    keep = [min(n, budget) for n in lens]
    to = None
    if apart:
        to, more = tables(keep, page, seed=seed + 1, dtype=table_type)
        to += P
        P += more
    cache = random_cache(P, H, D, page, code, seed=seed, lo=112, hi=126)
    cache["scales"][::5] = 0                              # blocks of zeros
    cache["codes"].view(torch.uint8)[::5] = 0
    if weights is not None:
        weights(cache["weight"])
    gpu = to_gpu(cache)
    kept, status, length = torch.full((len(lens), H, budget), 77, dtype=I32, device=DEV), i32([0]), i32(lens)
    len_out = length if alias else i32([5] * len(lens))
    want = []
    for b, n in enumerate(lens):
        t = torch.arange(n)
        w = cache["weight"][table[b, t // page].long(), :, t % page] if n else torch.zeros(0, H)
        want.append([ref.evict(w[:, h].tolist(), n, budget, sinks, recent) for h in range(H)])
    moved = [[k if apart or n > budget else [] for k in row] for row, n in zip(want, lens)]
    ref.move(cache["codes"], cache["scales"], cache["weight"], table, to if apart else table, moved)
    ommx_kv8_evict(gpu["codes"], gpu["scales"], gpu["weight"], table.to(DEV), length, kept, sink_tokens=sinks, recent_tokens=recent, to_table=to.to(DEV) if apart else None,
                   len_out=len_out, max_seq_len=max_len, status=status)
    assert int(status) == 0
    assert len_out.tolist() == keep and (alias or length.tolist() == lens)
    got = kept.tolist()
    for b in range(len(lens)):
        for h in range(H):
            assert got[b][h] == want[b][h] + [-1] * (budget - len(want[b][h])), (b, h)
    for name in cache:
        assert same(gpu[name], cache[name]), name


@pytest.mark.parametrize("lens,budget,sinks,recent", [
    ([1], 1, 0, 0), ([2], 1, 0, 1), ([40], 17, 1, 3), ([33, 0, 16, 100], 16, 4, 5), ([300, 20, 299], 100, 4, 32), ([65], 64, 0, 0), ([70, 71], 48, 48, 0), ([70], 20, 7, 13),
    ([130, 600], 333, 0, 100)])
@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("apart", [False, True])
def test_eviction(lens, budget, sinks, recent, code, apart):
    evict(lens, 2, 64, 16, code, budget, sinks, recent, apart=apart)
    evict(lens, 3, 128, 64, code, budget, sinks, recent, apart=apart, seed=4, alias=True, table_type=torch.int64)


@pytest.mark.parametrize("kind", ["ties", "alike", "zeros", "signs", "infinite", "nan", "narrow", "wide"])
def test_eviction_by_weights_of_every_kind(kind):
    def fill(w):
        gen = torch.Generator().manual_seed(3)
        u = torch.rand(w.shape, generator=gen)
        w.copy_({"ties": (u * 4).floor(), "alike": torch.full_like(u, 0.3), "zeros": torch.where(u < 0.5, -0.0, 0.0), "signs": u - 0.5,
                 "infinite": torch.where(u < 0.2, math.inf, torch.where(u < 0.4, -math.inf, u)), "nan": torch.where(u < 0.6, math.nan, u),
                 "narrow": 1.0 + u * 2.0 ** -20, "wide": torch.exp(80 * (u - 0.5)) * torch.where(u < 0.3, 1e-38, 1.0)}[kind])
    evict([500, 77, 1000], 2, 64, 16, I8, 200, 3, 20, weights=fill)
    evict([500, 77, 1000], 1, 64, 32, E4M3, 64, 0, 0, weights=fill, apart=True)


@pytest.mark.parametrize("L,budget", [(4200, 1500), (9000, 40), (20000, 3001), (5000, 4999)])
def test_eviction_of_long_rows(L, budget):
    """Rows that a cluster shares (with and without a bound on lengths), and more passes than one."""
    for max_len in (L, None, 100):
        evict([L, 60], 1, 64, 16, I8, budget, 4, min(30, budget - 4), max_len=max_len, apart=max_len == 100)


@pytest.mark.parametrize("kind", ["ties", "alike", "zeros", "signs"])
def test_eviction_of_long_rows_of_like_weights(kind):
    """More tokens of one weight than a block finishes for itself."""
    def fill(w):
        u = torch.rand(w.shape, generator=torch.Generator().manual_seed(3))
        w.copy_({"ties": (u * 2).floor(), "alike": torch.full_like(u, 0.3), "zeros": torch.where(u < 0.97, 0.0, u), "signs": torch.where(u < 0.5, -1.0, -2.0)}[kind])
    for max_len in (20000, 100):
        evict([20000, 60, 9000], 1, 64, 16, E4M3, 2500, 4, 30, weights=fill, max_len=max_len)


@pytest.mark.parametrize("H", [1, 2])
def test_eviction_where_keys_do_not_fit(H):
    """Many rows, so that one block, of either size, has a row of more keys than it holds."""
    lens = [50000] + [30] * 80
    evict(lens, H, 64, 256, I8, 64, 2, 8)


@pytest.mark.parametrize("B,H", [(5, 3), (8, 2), (17, 2), (36, 1)])
def test_eviction_in_clusters_of_every_size(B, H):
    """As many rows as clusters of eight blocks run at once and one more, and the same of four."""
    evict([4200 + 7 * b for b in range(B)], H, 64, 16, I8, 300, 2, 30, seed=B)


@pytest.mark.parametrize("code,D", [(I8, 128), (E4M3, 64)])
def test_eviction_of_many_rows(code, D):
    """More rows than SMs: blocks of half the size."""
    lens = [700, 3, 0, 5000, 333] + [90 + 7 * i for i in range(50)]
    for apart in (False, True):
        evict(lens, 3, D, 32, code, 300, 4, 60, apart=apart)
    evict(lens, 3, D, 32, code, 64, 0, 0, weights=lambda w: w.copy_((torch.rand(w.shape, generator=torch.Generator().manual_seed(1)) * 2).floor()), alias=True)


def test_sequences_with_pages_out_of_range_are_not_evicted_from():
    lens, page, H, D, budget = [100, 90, 80, 70, 60], 16, 2, 64, 40
    table, P = tables(lens, page)
    cache = random_cache(P, H, D, page, E4M3)
    gpu, status, t = to_gpu(cache), i32([0]), table.clone()
    t[0, 6], t[1, 0] = P, -1
    given = list(lens)
    given[2], given[3] = -4, 10 ** 5
    kept, len_out = torch.full((5, H, budget), 7, dtype=I32, device=DEV), i32([1] * 5)
    ommx_kv8_evict(gpu["codes"], gpu["scales"], gpu["weight"], t.to(DEV), i32(given), kept, len_out=len_out, status=status)
    assert int(status) == _lib.ST_BAD_PAGE | _lib.ST_BAD_LENGTH
    assert bool((kept[:4] == -1).all()) and len_out.tolist() == given[:4] + [budget]
    i = torch.arange(60)
    w = cache["weight"][table[4, i // page].long(), :, i % page]
    want = [ref.evict(w[:, h].tolist(), 60, budget, 0, 0) for h in range(H)]
    assert kept[4].tolist() == want
    ref.move(cache["codes"], cache["scales"], cache["weight"], table[4:], table[4:], [want])
    for name in cache:
        assert same(gpu[name], cache[name]), name
    # a table that does not hold what is kept, and one with pages that are not there
    cache2 = to_gpu(cache)
    for to, want in ((torch.zeros(5, 1, dtype=I32), _lib.ST_BAD_LENGTH), (torch.full((5, 3), P, dtype=I32), _lib.ST_BAD_PAGE)):
        status.zero_()
        ommx_kv8_evict(cache2["codes"], cache2["scales"], cache2["weight"], table.to(DEV), i32(lens), kept, to_table=to.to(DEV), status=status)
        assert int(status) == want
        for name in cache:
            assert same(cache2[name], cache[name]), name


def test_sequences_of_more_tokens_than_are_counted_are_not_evicted_from():
    """Beside one that is. The table of the long one names four pages over and over."""
    page, H, D, budget = 256, 2, 64, 40
    cache = random_cache(5, H, D, page, I8)
    gpu, status = to_gpu(cache), i32([0])
    table = (torch.arange(2 ** 30 // page, dtype=I32, device=DEV) % 4).repeat(2, 1)
    table[1, 0] = 4
    given = [2 ** 30 - 2 ** 16 + 1, 100]
    kept, len_out = torch.full((2, H, budget), 7, dtype=I32, device=DEV), i32([1, 1])
    ommx_kv8_evict(gpu["codes"], gpu["scales"], gpu["weight"], table, i32(given), kept, len_out=len_out, status=status)
    assert int(status) == _lib.ST_BAD_LENGTH
    assert bool((kept[0] == -1).all()) and len_out.tolist() == [given[0], budget]
    want = [ref.evict(cache["weight"][4, h, :100].tolist(), 100, budget, 0, 0) for h in range(H)]
    assert kept[1].tolist() == want
    short = torch.tensor([[4]])
    ref.move(cache["codes"], cache["scales"], cache["weight"], short, short, [want])
    for name in cache:
        assert same(gpu[name], cache[name]), name


# ---- together --------------------------------------------------------------------------------------------------------
class Layer:
    """A layer's cache and buffers, and a step as a user makes it."""

    def __init__(self, code, B, H, Hq, D, page, pages, seed=0):
        self.cache = to_gpu(ommx_kv8_alloc(B * pages, H, D, page_size=page, dtype=code, weight=True, device="cpu"))
        self.table = torch.randperm(B * pages, generator=torch.Generator().manual_seed(seed)).view(B, pages).to(I32).to(DEV)
        self.length = torch.zeros(B, dtype=I32, device=DEV)
        self.x = torch.zeros(B, Hq + 2 * H, D, dtype=BF16, device=DEV)
        self.o, self.lse = torch.zeros(B, Hq, D, dtype=BF16, device=DEV), torch.zeros(B, Hq, device=DEV)
        self.kept = torch.zeros(B, H, 40, dtype=I32, device=DEV)
        self.status = i32([0])
        self.H, self.Hq, self.most = H, Hq, pages * page
        self.work = torch.empty(max(1, kv8_workspace_floats(B, Hq, D, self.most, weight=True)), device=DEV)

    def step(self, **more):
        c, q, k, v = self.cache, *self.x.split([self.Hq, self.H, self.H], 1)
        self.length += 1
        ommx_kv8_append(k, v, c["codes"], c["scales"], self.table, self.length, weight=c["weight"], status=self.status)
        ommx_kv8_decode_attention(q, c["codes"], c["scales"], self.table, self.length, self.o, self.lse, weight=c["weight"], keep=0.98, workspace=self.work, status=self.status, **more)

    def evict(self):
        c = self.cache
        ommx_kv8_evict(c["codes"], c["scales"], c["weight"], self.table, self.length, self.kept, sink_tokens=2, recent_tokens=8, len_out=self.length, status=self.status)

    def state(self):
        return {**self.cache, "length": self.length, "o": self.o, "lse": self.lse, "kept": self.kept, "status": self.status}


@pytest.mark.parametrize("code,D", [(I8, 128), (E4M3, 64)])
def test_decode_steps_with_evictions(code, D):
    """Prompts, steps, an eviction, more steps: each step's output against 64 bits over what the cache holds, and the cache against the reference."""
    B, H, Hq, page = 3, 2, 6, 16
    layer = Layer(code, B, H, Hq, D, page, 8)
    cpu = {k: v.cpu() for k, v in layer.cache.items()}
    gen = torch.Generator().manual_seed(5)
    lens = [50, 1, 73]
    starts = cumulated(lens)
    x = rows(starts[-1], H, D, BF16, gen, spread=0.3)
    layer.length.copy_(i32(lens))
    table = layer.table.cpu()
    ommx_kv8_append(x[:, :H].to(DEV), x[:, H:].to(DEV), layer.cache["codes"], layer.cache["scales"], layer.table, layer.length, row_start=i32(starts), weight=layer.cache["weight"],
                    status=layer.status)
    ref.append(cpu["codes"], cpu["scales"], cpu["weight"], table, lens, starts, x[:, :H], x[:, H:])
    for step in range(24):
        new = torch.randn(B, Hq + 2 * H, D, generator=gen).bfloat16()
        layer.x.copy_(new)
        before = layer.cache["weight"].clone()
        lens = [n + 1 for n in lens]
        layer.step()
        ref.append(cpu["codes"], cpu["scales"], cpu["weight"], table, lens, list(range(B + 1)), new[:, Hq:Hq + H], new[:, Hq + H:])
        assert same(layer.cache["codes"], cpu["codes"]) and same(layer.cache["scales"], cpu["scales"])
        for b, n in enumerate(lens):
            before[table[b, (n - 1) // page].long(), :, (n - 1) % page] = 0
        check(new[:, :Hq].to(DEV), layer.cache, layer.table, lens, layer.o, layer.lse, weight=layer.cache["weight"], before=before, keep=0.98)
        cpu["weight"].copy_(layer.cache["weight"].cpu())  # sums in 32 bits: held to their bound above
        if step % 9 == 8:
            want = []
            for b, n in enumerate(lens):
                t = torch.arange(n)
                w = cpu["weight"][table[b, t // page].long(), :, t % page]
                want.append([ref.evict(w[:, h].tolist(), n, 40, 2, 8) for h in range(H)])
            layer.evict()
            ref.move(cpu["codes"], cpu["scales"], cpu["weight"], table, table, [k if n > 40 else [[]] * H for k, n in zip(want, lens)])
            lens = [min(n, 40) for n in lens]
            assert layer.length.tolist() == lens
            assert [[[t for t in h if t >= 0] for h in b] for b in layer.kept.tolist()] == want
            for name in cpu:
                assert same(layer.cache[name], cpu[name]), name
    assert int(layer.status) == 0


def test_a_captured_step_follows_its_lengths():
    """One graph of a step (and one of the eviction) replayed is bit for bit what eager calls give, on a stream of its own."""
    eager, graph = (Layer(I8, 4, 2, 8, 128, 16, 8) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step, clear = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        saved = {k: v.clone() for k, v in graph.state().items()}
        graph.step()
        graph.evict()
        for k, v in graph.state().items():
            v.copy_(saved[k])
        with torch.cuda.graph(step, stream=side):
            graph.step()
        with torch.cuda.graph(clear, stream=side):
            graph.evict()
    gen = torch.Generator().manual_seed(1)
    for t in range(130):
        x = torch.randn(eager.x.shape, generator=gen).bfloat16()
        eager.x.copy_(x)
        eager.step()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.x.copy_(x)
            step.replay()
        if t % 37 == 36:
            eager.evict()
            with torch.cuda.stream(side):
                clear.replay()
        side.synchronize()
        torch.cuda.synchronize()
        for k, v in eager.state().items():
            assert same(v, graph.state()[k]), (t, k)
    assert int(eager.status) == 0


def test_calls_side_by_side():
    """Calls on two streams with caches and workspaces of their own, begun while others run, give what they give alone."""
    a, b = Layer(I8, 2, 4, 16, 128, 16, 300, seed=1), Layer(E4M3, 3, 2, 16, 128, 32, 100, seed=2)
    for layer, n in ((a, 4700), (b, 3100)):
        cache = random_cache(layer.table.numel(), layer.H, 128, layer.cache["weight"].shape[2], layer.cache["codes"].dtype, seed=n)
        for k in cache:
            layer.cache[k].copy_(cache[k])
        layer.length.fill_(n)
        layer.x.copy_(torch.randn(layer.x.shape, generator=torch.Generator().manual_seed(n)).bfloat16())
    saved = [{k: v.clone() for k, v in layer.state().items()} for layer in (a, b)]
    alone = []
    for layer in (a, b):
        for _ in range(3):
            layer.step()
        layer.evict()
        layer.step()
        torch.cuda.synchronize()
        alone.append({k: v.clone() for k, v in layer.state().items()})
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(5):
        for layer, s in zip((a, b), saved):
            for k, v in layer.state().items():
                v.copy_(s[k])
        torch.cuda.synchronize()
        for i in range(5):
            for layer, stream in zip((a, b), streams):
                with torch.cuda.stream(stream):
                    layer.evict() if i == 3 else layer.step()
        torch.cuda.synchronize()
        for layer, want in zip((a, b), alone):
            for k, v in layer.state().items():
                assert same(v, want[k]), (turn, k)


def test_nothing_to_do():
    cache = to_gpu(random_cache(3, 2, 64, 16, I8))
    none, table = torch.zeros(0, dtype=I32, device=DEV), torch.zeros(0, 4, dtype=I32, device=DEV)
    empty = torch.zeros(0, 2, 64, device=DEV, dtype=BF16)
    ommx_kv8_append(empty, empty, cache["codes"], cache["scales"], table, none)
    ommx_kv8_gather(cache["codes"], cache["scales"], table, none, empty, empty)
    ommx_kv8_decode_attention(empty, cache["codes"], cache["scales"], table, none, torch.zeros(0, 2, 64, device=DEV), torch.zeros(0, 2, device=DEV), weight=cache["weight"])
    ommx_kv8_evict(cache["codes"], cache["scales"], cache["weight"], table, none, torch.zeros(0, 2, 5, dtype=I32, device=DEV))
    # sequences of no tokens, in a table of no pages
    two, table = torch.zeros(2, dtype=I32, device=DEV), torch.zeros(2, 0, dtype=I32, device=DEV)
    q, o, lse, kept = torch.ones(2, 4, 64, device=DEV, dtype=BF16), torch.ones(2, 4, 64, device=DEV), torch.ones(2, 4, device=DEV), torch.ones(2, 2, 5, dtype=I32, device=DEV)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table, two, o, lse, weight=cache["weight"])
    ommx_kv8_evict(cache["codes"], cache["scales"], cache["weight"], table, two, kept)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all()) and bool((kept == -1).all())
    ommx_kv8_append(empty, empty, cache["codes"], cache["scales"], table, two, row_start=torch.zeros(3, dtype=I32, device=DEV))


def test_launches():
    """Append and read back are one launch each, attention one or two (two with an account), eviction one (two where
    it shortens the lengths it reads)."""
    lib = _lib.load()

    def launches(f):
        before = lib.ommx_b200_launch_count()
        f()
        return lib.ommx_b200_launch_count() - before

    layer = Layer(I8, 2, 2, 8, 128, 16, 600)
    layer.length.fill_(9000)
    c, q, k, v = layer.cache, *layer.x.split([8, 2, 2], 1)
    where = (c["codes"], c["scales"], layer.table, layer.length)
    assert launches(lambda: ommx_kv8_append(k, v, *where)) == 1
    assert launches(lambda: ommx_kv8_gather(*where, k, v)) == 1
    for n, more, want in ((None, {}, 2), (None, dict(weight=c["weight"]), 2), (None, dict(window=300, sink_tokens=4), 1), (200, {}, 1), (200, dict(weight=c["weight"]), 2)):
        assert launches(lambda: ommx_kv8_decode_attention(q, *where, layer.o, layer.lse, max_seq_len=n, **more)) == want
    assert launches(layer.evict) == 2
    assert launches(lambda: ommx_kv8_evict(c["codes"], c["scales"], c["weight"], layer.table, layer.length, layer.kept)) == 1
