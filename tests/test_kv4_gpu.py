"""The 4-bit cache on the GPU: stored bytes and summaries against the layout restated word by word, attention against 64 bits.

Tolerances.  Stored bytes, rotated queries, rows read back, summaries and selected pages are exact.  Attention: a weight p s is
rounded to fp16, an error of 2^-12 of it at most, so a channel's is 2^-12 sum p s code / sum p <= 2^-12 max (V - zero) <= 2^-12 R,
R the largest range (15 scales) of a group; weights below 2^-36 of the largest are lost, which is below that for any length
here.  Logits are fp32 sums of a few hundred terms: an absolute error of 2^-24 * 2^7 * |q|.|K| sm_scale moves weights by that
share, and an output by twice that times R at most.  The output's own rounding is half a step.
"""
import math

import pytest
import torch

import kv4_reference as ref
from open_ommx_serve_b200 import (ommx_kv4_alloc, ommx_kv4_append, ommx_kv4_decode_attention, ommx_kv4_gather,
                                  ommx_kv4_select_pages)
from open_ommx_serve_b200 import _lib
from open_ommx_serve_b200.attention.kv4 import kv4_select_workspace_bytes, kv4_workspace_floats

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tables(lens, page, spare=2, seed=0, dtype=torch.int32):
    """A shuffled page table for sequences of these lengths: (table [B, pages], number of pages)."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=gen)
    table = torch.zeros(len(lens), max(need + [1]) + 1, dtype=dtype)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(dtype)
        at += n
    return table, sum(need) + spare


def rows_of(lens, new):
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return torch.tensor(start, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)


def angles(positions, rot, base=10000.0):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return a.cos().float(), a.sin().float()


def filled(lens, H, D, page, seed=0, dtype=torch.bfloat16, summary=True, scale=1.0):
    """A cache that holds random sequences, appended by the library: (cache, table, lens) on the GPU."""
    gen = torch.Generator().manual_seed(seed)
    table, P = tables(lens, page, seed=seed)
    cache = ommx_kv4_alloc(P, H, D, page_size=page, summary=summary, device=DEV)
    start, length = rows_of(lens, lens)
    T = int(start[-1])
    if T:
        offset = 2 * torch.randn(1, H, D, generator=gen)
        k = ((torch.randn(T, H, D, generator=gen) + offset) * scale).to(dtype)
        v = (torch.randn(T, H, D, generator=gen) * scale).to(dtype)
        ommx_kv4_append(k.to(DEV), v.to(DEV), cache["records"], table.to(DEV), length.to(DEV), row_start=start.to(DEV), summary=cache["summary"])
    return cache, table.to(DEV), length.to(DEV)


# ---- append ------------------------------------------------------------------------------------------------------
APPENDS = [
    # D, page, H, Hq, dtype, rot, interleaved, lens, new, pad
    (128, 16, 2, 4, torch.bfloat16, 128, False, [20], [1], 0),
    (128, 16, 3, 3, torch.bfloat16, 128, False, [40, 17, 5], [33, 1, 5], 3),
    (128, 32, 2, 14, torch.float16, 64, True, [70, 31, 64], [37, 2, 64], 1),
    (128, 64, 5, 10, torch.float32, 128, True, [130, 63], [100, 63], 0),
    (64, 16, 1, 8, torch.bfloat16, 32, False, [50, 16, 1], [20, 16, 1], 0),
    (64, 32, 2, 2, torch.float16, 64, False, [95, 33], [95, 3], 2),
    (64, 128, 4, 4, torch.float32, 32, True, [300], [211], 0),
    (64, 256, 1, 1, torch.bfloat16, 64, True, [600, 255], [345, 7], 0),
    (128, 256, 2, 2, torch.bfloat16, 0, False, [270], [40], 5),
]


@pytest.mark.parametrize("D,page,H,Hq,dtype,rot,interleaved,lens,new,pad", APPENDS)
@pytest.mark.parametrize("form", ["sliced", "odd strides"])
def test_append_stores_the_layouts_bytes(D, page, H, Hq, dtype, rot, interleaved, lens, new, pad, form):
    gen = torch.Generator().manual_seed(7)
    start, length = rows_of(lens, new)
    n, T = int(start[-1]), int(start[-1]) + pad
    table, P = tables(lens, page, seed=3, dtype=torch.int64 if page == 32 else torch.int32)
    records = torch.randint(0, 256, (P, H, page // 16, 20 * D), generator=gen, dtype=torch.uint8)
    summary = torch.randn(P, H, 2, D, generator=gen).to(torch.bfloat16)
    wide = torch.randn(T, Hq + 2 * H, D + (0 if form == "sliced" else 3), generator=gen).to(dtype)[..., :D]
    q, k, v = wide[:, :Hq], wide[:, Hq:Hq + H], wide[:, Hq + H:]
    cos, sin = angles(max(lens) + 4, rot) if rot else (None, None)
    want_records, want_summary = records.clone(), summary.clone()
    want_q = torch.full_like(q, 5.0)
    for b in range(len(lens)):
        for i in range(new[b]):
            row, pos = int(start[b]) + i, lens[b] - new[b] + i
            kk = k[row:row + 1]
            if rot:
                kk = ref.rotate(kk, cos[pos:pos + 1], sin[pos:pos + 1], interleaved)
                want_q[row] = ref.rotate(q[row:row + 1], cos[pos:pos + 1], sin[pos:pos + 1], interleaved)[0]
            p = int(table[b, pos // page])
            kq, vq = ref.quantize(kk[0]), ref.quantize(v[row])
            for h in range(H):
                ref.put(want_records, p, h, pos % page // 16, pos % 16, [x[h] for x in kq], [x[h] for x in vq])
            top, bottom = ref.to_bf16(kk[0].float(), True), ref.to_bf16(kk[0].float(), False)
            if pos % page:
                top, bottom = torch.maximum(top, want_summary[p, :, 0].float()), torch.minimum(bottom, want_summary[p, :, 1].float())
            want_summary[p, :, 0], want_summary[p, :, 1] = top.bfloat16(), bottom.bfloat16()
    wide_d = torch.empty_strided(wide.size(), wide.stride(), dtype=dtype, device=DEV)
    wide_d.copy_(wide)
    qd, kd, vd = wide_d[:, :Hq], wide_d[:, Hq:Hq + H], wide_d[:, Hq + H:]
    rec_d, sum_d, status = records.to(DEV), summary.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 5.0, device=DEV)
    more = dict(q=qd, q_out=out, cos=cos.to(DEV), sin=sin.to(DEV), interleaved=interleaved) if rot else {}
    got = ommx_kv4_append(kd, vd, rec_d, table.to(DEV), length.to(DEV), row_start=start.to(DEV), summary=sum_d, status=status, **more)
    assert int(status) == 0
    assert torch.equal(rec_d.cpu(), want_records)
    assert torch.equal(sum_d.cpu(), want_summary)
    if rot:
        assert got is out and torch.equal(out.cpu(), want_q)
        assert torch.equal(out[n:].cpu(), torch.full_like(q[n:], 5.0))
    # the same rows read back
    ko, vo = (torch.full((T, H, D), 9.0, dtype=dtype, device=DEV) for _ in range(2))
    ommx_kv4_gather(rec_d, table.to(DEV), length.to(DEV), ko, vo, row_start=start.to(DEV), status=status)
    for b in range(len(lens)):
        wk, wv = ref.sequence(want_records, table[b], lens[b])
        for got, want in ((ko, wk), (vo, wv)):
            assert torch.equal(got[int(start[b]):int(start[b + 1])].cpu(), want[:, lens[b] - new[b]:].transpose(0, 1).float().to(dtype))
    assert int(status) == 0 and bool((ko[n:] == 9).all()) and bool((vo[n:] == 9).all())


def test_one_row_each_in_place_and_at_given_positions():
    """A decode step: no row_start, the queries rotated where they lie, positions that are not the places in the sequence."""
    lens, page, H, Hq, D = [33, 1, 16, 100, 64], 16, 2, 6, 128
    cache, table, length = filled(lens, H, D, page, seed=1)
    gen = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(5, n, D, generator=gen).bfloat16() for n in (Hq, H, H))
    cos, sin = angles(50, 128)
    for dtype in (torch.int32, torch.int64):
        positions = torch.tensor([3, 49, 0, 7, 20], dtype=dtype)
        qd = q.to(DEV)
        before = cache["records"].clone()
        same = ommx_kv4_append(k.to(DEV), v.to(DEV), cache["records"], table, length, q=qd, q_out=qd, cos=cos.to(DEV), sin=sin.to(DEV),
                               positions=positions.to(DEV))
        assert same is qd
        assert torch.equal(qd.cpu(), ref.rotate(q, cos[positions.long()], sin[positions.long()], False))
        want = before.cpu()
        kr = ref.rotate(k, cos[positions.long()], sin[positions.long()], False)
        for b, n in enumerate(lens):
            for h in range(H):
                ref.put(want, int(table[b, (n - 1) // page]), h, (n - 1) % page // 16, (n - 1) % 16,
                        [x[h] for x in ref.quantize(kr[b])], [x[h] for x in ref.quantize(v[b])])
        assert torch.equal(cache["records"].cpu(), want)
    fresh = ommx_kv4_append(k.to(DEV), v.to(DEV), cache["records"], table, length, q=q.to(DEV), cos=cos.to(DEV), sin=sin.to(DEV), positions=positions.to(DEV))
    assert torch.equal(fresh, qd)


def test_rotation_on_the_way_equals_rotation_before():
    lens, H, D = [77], 2, 128
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randn(77, H, D, generator=gen).half() for _ in range(2))
    cos, sin = angles(77, 64)
    table, P = tables(lens, 32)
    start, length = rows_of(lens, lens)
    both = []
    for before in (True, False):
        c = ommx_kv4_alloc(P, H, D, page_size=32, summary=True, device=DEV)
        kk, more = (ref.rotate(k, cos, sin, False), {}) if before else (k, dict(cos=cos.to(DEV), sin=sin.to(DEV)))
        ommx_kv4_append(kk.to(DEV), v.to(DEV), c["records"], table.to(DEV), length.to(DEV), row_start=start.to(DEV), summary=c["summary"], **more)
        both.append(c)
    assert torch.equal(both[0]["records"], both[1]["records"]) and torch.equal(both[0]["summary"], both[1]["summary"])


def test_token_by_token_equals_at_once():
    """However a sequence is cut into calls, the bytes and the summary are the same (pages written before hold what they did)."""
    H, D, page, n = 3, 64, 32, 75
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(n, H, D, generator=gen).bfloat16().to(DEV) for _ in range(2))
    table, P = tables([n], page)
    caches = [ommx_kv4_alloc(P, H, D, page_size=page, summary=True, device=DEV) for _ in range(3)]
    start, length = rows_of([n], [n])
    ommx_kv4_append(k, v, caches[0]["records"], table.to(DEV), length.to(DEV), row_start=start.to(DEV), summary=caches[0]["summary"])
    for i in range(n):
        ommx_kv4_append(k[i:i + 1], v[i:i + 1], caches[1]["records"], table.to(DEV), torch.tensor([i + 1], dtype=torch.int32, device=DEV), summary=caches[1]["summary"])
    for lo, hi in ((0, 7), (7, 8), (8, 33), (33, 64), (64, 75)):
        s, m = rows_of([hi], [hi - lo])
        ommx_kv4_append(k[lo:hi], v[lo:hi], caches[2]["records"], table.to(DEV), m.to(DEV), row_start=s.to(DEV), summary=caches[2]["summary"])
    used = table[0, :3].long()
    for c in caches[1:]:
        assert torch.equal(c["records"], caches[0]["records"])
        assert torch.equal(c["summary"][used], caches[0]["summary"][used])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_values_that_quantize_badly(dtype):
    """Constants, zeros of both signs, NaN, infinities, the largest and smallest numbers, ties between codes."""
    big = torch.finfo(dtype).max
    rows = [torch.zeros(128), -torch.zeros(128), torch.full((128,), 3.25), torch.full((128,), -1e-3),
            torch.arange(128).float() / 2, torch.linspace(-big, big, 128, dtype=torch.float64).clamp(-big, big).to(dtype).float(),
            torch.cat((torch.tensor([math.nan, math.inf, -math.inf]), torch.ones(125))), torch.cat((torch.ones(127), torch.tensor([math.nan]))),
            torch.full((128,), torch.finfo(dtype).tiny), torch.randn(128, generator=torch.Generator().manual_seed(0)) * 1e-6,
            torch.cat((torch.zeros(31), torch.ones(1), torch.tensor([15.0]), torch.arange(95) % 16 * 1.0)),
            torch.full((128,), 100.0) + torch.arange(128) % 3 * 0.5]
    k = torch.stack(rows).to(dtype)[:, None]
    v = k.flip(0).contiguous()
    T = len(rows)
    table, P = tables([T], 16)
    c = ommx_kv4_alloc(P, 1, 128, page_size=16, summary=True, device=DEV)
    want = c["records"].cpu()
    for i in range(T):
        ref.put(want, int(table[0, 0]), 0, 0, i, [x[0] for x in ref.quantize(k[i])], [x[0] for x in ref.quantize(v[i])])
    start, length = rows_of([T], [T])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ommx_kv4_append(k.to(DEV), v.to(DEV), c["records"], table.to(DEV), length.to(DEV), row_start=start.to(DEV), summary=c["summary"], status=status)
    assert int(status) == _lib.ST_NONFINITE
    assert torch.equal(c["records"].cpu(), want)
    held = ref.finite(k[:, 0])
    s = c["summary"][int(table[0, 0]), 0].float().cpu()
    assert torch.equal(s[0], ref.to_bf16(held.max(0).values, True)) and torch.equal(s[1], ref.to_bf16(held.min(0).values, False))
    o, lse = torch.empty(1, 1, 128, device=DEV), torch.empty(1, 1, device=DEV)
    ommx_kv4_decode_attention(torch.zeros(1, 1, 128, dtype=torch.bfloat16, device=DEV), c["records"], table.to(DEV), length.to(DEV), o, lse)
    assert torch.isfinite(o).all() and abs(float(lse) - math.log(T)) < 1e-5


# ---- attention ---------------------------------------------------------------------------------------------------
def bounds(q, k, v, sm_scale, o_dtype):
    """The largest error of o and lse that the module's comment derives; k, v [H, tokens, D] in 64 bits."""
    if k.shape[1] == 0:
        return 0.0, 0.0
    group = q.shape[0] // k.shape[0]
    reach = max(float((q[h].double().abs()[None] * k[h // group].abs()).sum(-1).max()) for h in range(q.shape[0])) * sm_scale
    R = float((v.unflatten(-1, (-1, 32)).amax(-1) - v.unflatten(-1, (-1, 32)).amin(-1)).max())
    drift = 2.0 ** -17 * reach + 2.0 ** -20
    return 2.0 ** -12 * R + 2 * drift * (R + float(v.abs().max())) + torch.finfo(o_dtype).eps / 2 * float(v.abs().max()), drift


def check_attention(cache, table, lens, q, o, lse, cap=0.0, selected=None, sm_scale=None):
    D = q.shape[-1]
    sm_scale = sm_scale or D ** -0.5
    page = cache["records"].shape[2] * 16
    for b, n in enumerate(lens):
        k, v = ref.sequence(cache["records"], table[b], n)
        if selected is not None:
            keep = []
            for h in range(k.shape[0]):
                listed = selected[b, h, :-(-n // page)].tolist()
                keep.append([t for p in listed if p >= 0 for t in range(p * page, min(n, (p + 1) * page))])
            ks, vs = [k[h, i] for h, i in enumerate(keep)], [v[h, i] for h, i in enumerate(keep)]
        else:
            ks, vs = list(k), list(v)
        wo, wl = ref.attention(q[b], ks, vs, sm_scale, cap)
        off, drift = bounds(q[b], k, v, sm_scale, o.dtype)
        assert torch.equal(torch.isinf(lse[b]), torch.isinf(wl)), (b, n)
        assert float((o[b].double() - wo).abs().max()) <= off, (b, n, off)
        some = ~torch.isinf(wl)
        if some.any():
            assert float((lse[b].double() - wl)[some].abs().max()) <= drift + 2.0 ** -22 * float(wl[some].abs().max()), (b, n, drift)


ATTENTION = [
    # D, page, H, Hq, q dtype, o dtype, lens, cap
    (128, 16, 8, 32, torch.bfloat16, torch.bfloat16, [1], 0.0),
    (128, 16, 8, 32, torch.bfloat16, torch.float32, [333], 0.0),
    (128, 16, 2, 2, torch.bfloat16, torch.float32, [0, 1, 15, 16, 17, 31, 32, 33, 0], 0.0),
    (128, 32, 1, 7, torch.float16, torch.float16, [5, 1000, 64, 63], 0.0),
    (128, 64, 3, 24, torch.bfloat16, torch.float32, [4097, 2, 700], 30.0),
    (128, 16, 1, 16, torch.bfloat16, torch.float32, [900, 1], 0.0),
    (128, 128, 2, 38, torch.float16, torch.float32, [130, 500], 0.0),
    (64, 16, 4, 4, torch.bfloat16, torch.bfloat16, [2049, 77], 0.0),
    (64, 32, 2, 10, torch.float16, torch.float32, [1, 0, 5000], 5.0),
    (64, 256, 8, 64, torch.bfloat16, torch.float32, [257, 300, 1, 511], 0.0),
    (128, 16, 1, 1, torch.bfloat16, torch.float32, [30011], 0.0),
    (128, 16, 2, 8, torch.bfloat16, torch.float32, [17] * 70, 0.0),
]


@pytest.mark.parametrize("D,page,H,Hq,qd,od,lens,cap", ATTENTION)
def test_attention_against_64_bits(D, page, H, Hq, qd, od, lens, cap):
    cache, table, length = filled(lens, H, D, page, seed=11)
    gen = torch.Generator().manual_seed(12)
    q = torch.randn(len(lens), Hq, D, generator=gen).to(qd).to(DEV)
    o, lse = torch.full((len(lens), Hq, D), 7.0, dtype=od, device=DEV), torch.full((len(lens), Hq), 7.0, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, logit_cap=cap, max_seq_len=max(lens), status=status)
    assert int(status) == 0
    check_attention(cache, table, lens, q, o, lse, cap)
    again, lse2 = torch.empty_like(o), torch.empty_like(lse)
    ommx_kv4_decode_attention(q, cache["records"], table, length, again, lse2, logit_cap=cap, max_seq_len=max(lens))
    assert torch.equal(o, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 30.0, 1e4])
def test_attention_of_small_and_large_values(scale):
    """Weights meet the values' scales before the product: their size must not cost bits."""
    lens = [200, 40]
    cache, table, length = filled(lens, 2, 128, 16, seed=21, scale=scale)
    q = (torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(3)) / scale).bfloat16().to(DEV)
    o, lse = torch.empty(2, 8, 128, device=DEV), torch.empty(2, 8, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse)
    check_attention(cache, table, lens, q, o, lse)


def test_attention_when_late_tokens_take_over():
    """Logits that grow along the sequence move the reference again and again; so do scales that grow."""
    n, D = 2000, 128
    gen = torch.Generator().manual_seed(8)
    k = 0.1 * torch.randn(n, 1, D, generator=gen) + torch.linspace(-4, 4, n)[:, None, None]
    v = torch.randn(n, 1, D, generator=gen) * torch.logspace(-6, 3, n)[:, None, None]
    table, P = tables([n], 16)
    c = ommx_kv4_alloc(P, 1, D, device=DEV)
    start, length = rows_of([n], [n])
    ommx_kv4_append(k.bfloat16().to(DEV), v.bfloat16().to(DEV), c["records"], table.to(DEV), length.to(DEV), row_start=start.to(DEV))
    for sign in (1.0, -1.0):
        q = (sign * (1 + 0.1 * torch.randn(1, 4, D, generator=gen))).bfloat16().to(DEV)
        o, lse = torch.empty(1, 4, D, device=DEV), torch.empty(1, 4, device=DEV)
        ommx_kv4_decode_attention(q, c["records"], table.to(DEV), length.to(DEV), o, lse)
        check_attention(c, table, [n], q, o, lse)


def test_what_lies_behind_the_last_token_is_not_read_as_one():
    """Records of a page's unwritten tokens hold anything, NaN and infinite parameters among it."""
    lens = [5, 24, 49]
    cache, table, length = filled(lens, 2, 128, 32, seed=31)
    q = torch.randn(3, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    out = []
    for fill in (0x00, 0xFF, 0x7F):
        rec = cache["records"].clone()
        k, v = ref.values(rec)
        for b, n in enumerate(lens):
            for pos in range(n, -(-n // 32) * 32):
                page, part, tau = int(table[b, pos // 32]), pos % 32 // 16, pos % 16
                G = 4
                rec[page, :, part, 16 * tau * G:16 * (tau + 1) * G] = fill
                for at in (16 * 128 + 4 * G * tau, 18 * 128 + 4 * G * tau):
                    rec[page, :, part, at:at + 4 * G] = fill
        o, lse = torch.empty(3, 4, 128, device=DEV), torch.empty(3, 4, device=DEV)
        ommx_kv4_decode_attention(q, rec, table, length, o, lse)
        out.append((o, lse))
    assert torch.isfinite(out[0][0]).all()
    for o, lse in out[1:]:
        assert torch.equal(o, out[0][0]) and torch.equal(lse, out[0][1])


def test_strided_queries_and_outputs():
    lens = [100, 300]
    cache, table, length = filled(lens, 2, 64, 16, seed=41)
    wide = torch.randn(2, 12, 67, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    q = wide[:, 2:10, :64]
    o_wide, lse_wide = torch.zeros(2, 9, 70, device=DEV), torch.zeros(2, 11, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o_wide[:, 1:, 3:67], lse_wide[:, 2:10], sm_scale=0.3)
    check_attention(cache, table, lens, q, o_wide[:, 1:, 3:67], lse_wide[:, 2:10], sm_scale=0.3)
    assert bool((o_wide[:, 0] == 0).all()) and bool((o_wide[..., :3] == 0).all()) and bool((lse_wide[:, 10:] == 0).all())


# ---- selected pages ----------------------------------------------------------------------------------------------
SELECT = [
    # D, page, H, Hq, dtype, lens, n, first, last
    (128, 16, 2, 8, torch.bfloat16, [400, 16, 1, 0, 130], 7, 1, 2),
    (128, 32, 1, 5, torch.float16, [3000, 64], 20, 0, 0),
    (64, 16, 3, 3, torch.bfloat16, [1000, 999, 17], 5, 2, 3),
    (64, 64, 2, 16, torch.bfloat16, [5000], 1, 0, 1),
    (128, 16, 1, 12, torch.float16, [20000], 300, 1, 1),
]


@pytest.mark.parametrize("D,page,H,Hq,dtype,lens,n,first,last", SELECT)
def test_selected_pages_and_attention_over_them(D, page, H, Hq, dtype, lens, n, first, last):
    cache, table, length = filled(lens, H, D, page, seed=51, dtype=dtype)
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(52)).to(dtype).to(DEV)
    sel = torch.full((len(lens), H, n), 99, dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ommx_kv4_select_pages(q, cache["summary"], table, length, sel, page_size=page, first_pages=first, last_pages=last, status=status)
    s = cache["summary"].cpu()
    for b, length_b in enumerate(lens):
        want = ref.select(q[b].cpu(), s, table[b].cpu(), length_b, page, n, first, last)
        for h in range(H):
            assert sel[b, h].tolist() == want[h] + [-1] * (n - len(want[h])), (b, h)
    o, lse = torch.empty(len(lens), Hq, D, device=DEV), torch.empty(len(lens), Hq, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, selected=sel, status=status)
    assert int(status) == 0
    check_attention(cache, table, lens, q, o, lse, selected=sel)


def test_equal_scores_go_to_the_lowest_pages():
    n, page = 640, 16
    table, P = tables([n], page)
    c = ommx_kv4_alloc(P, 1, 64, page_size=page, summary=True, device=DEV)
    k = torch.ones(n, 1, 64, dtype=torch.bfloat16, device=DEV)
    k[16 * 30:16 * 31] = 2.0
    start, length = rows_of([n], [n])
    ommx_kv4_append(k, k, c["records"], table.to(DEV), length.to(DEV), row_start=start.to(DEV), summary=c["summary"])
    for value, want in ((1.0, [0, 1, 2, 30, 39]), (-1.0, [0, 1, 2, 3, 39]), (0.0, [0, 1, 2, 3, 39])):
        q = torch.full((1, 2, 64), value, dtype=torch.bfloat16, device=DEV)
        sel = torch.zeros(1, 1, 5, dtype=torch.int32, device=DEV)
        ommx_kv4_select_pages(q, c["summary"], table.to(DEV), length.to(DEV), sel, page_size=page, first_pages=1, last_pages=1)
        assert sel[0, 0].tolist() == want, value


def test_lists_of_the_callers_own():
    """Entries below 0 and behind the sequence are passed over, a page listed twice counts twice, a list of none is no tokens."""
    lens = [200, 50]
    cache, table, length = filled(lens, 2, 128, 16, seed=61)
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    sel = torch.tensor([[[12, 3, -1, 5000], [3, 3, 0, -7]], [[-1, -1, -1, -1], [1, -1, 2, 0]]], dtype=torch.int32, device=DEV)
    o, lse = torch.empty(2, 4, 128, device=DEV), torch.empty(2, 4, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, selected=sel, status=status)
    check_attention(cache, table, lens, q, o, lse, selected=sel)
    assert int(status) == 0 and bool((o[1, :2] == 0).all()) and bool(torch.isinf(lse[1, :2]).all())


# ---- together ----------------------------------------------------------------------------------------------------
def test_a_served_run_eager_and_captured():
    """A prompt, then steps of append + select + attend over two layers: a captured and replayed step does what the eager one does,
    and attention over what was appended agrees with 64 bits."""
    B, H, Hq, D, page, steps, layers, n = 3, 2, 8, 128, 16, 20, 2, 6
    prompt = [100, 37, 1]
    lens = [m + steps for m in prompt]
    gen = torch.Generator().manual_seed(71)
    table, P = tables(lens, page)
    table = table.to(DEV)
    cos, sin = (x.to(DEV) for x in angles(max(lens), D))
    rows = [[torch.randn(B, Hq + 2 * H, D, generator=gen).bfloat16().to(DEV) for _ in range(steps)] for _ in range(layers)]
    start, length = rows_of(prompt, prompt)
    pk = torch.randn(layers, int(start[-1]), 2 * H, D, generator=gen).bfloat16().to(DEV)

    def serve(captured):
        caches = [ommx_kv4_alloc(P, H, D, page_size=page, summary=True, device=DEV) for _ in range(layers)]
        seq = length.to(DEV)
        for i, c in enumerate(caches):
            ommx_kv4_append(pk[i, :, :H], pk[i, :, H:], c["records"], table, seq, row_start=start.to(DEV), cos=cos, sin=sin, summary=c["summary"])
        now = [torch.empty(B, Hq + 2 * H, D, dtype=torch.bfloat16, device=DEV) for _ in range(layers)]
        q, o = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV), torch.empty(layers, B, Hq, D, device=DEV)
        lse, sel = torch.empty(layers, B, Hq, device=DEV), torch.empty(B, H, n, dtype=torch.int32, device=DEV)
        work, keys = torch.empty(kv4_workspace_floats(D), device=DEV), torch.empty(kv4_select_workspace_bytes(B, H, table.shape[1]), dtype=torch.uint8, device=DEV)

        def step():
            seq.add_(1)
            for i, c in enumerate(caches):
                ommx_kv4_append(now[i][:, Hq:Hq + H], now[i][:, Hq + H:], c["records"], table, seq, q=now[i][:, :Hq], q_out=q, cos=cos, sin=sin,
                                summary=c["summary"])
                ommx_kv4_select_pages(q, c["summary"], table, seq, sel, page_size=page, workspace=keys)
                ommx_kv4_decode_attention(q, c["records"], table, seq, o[i], lse[i], selected=sel, workspace=work)

        graph = None
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
        outs = []
        for s in range(steps):
            for i in range(layers):
                now[i].copy_(rows[i][s])
            graph.replay() if captured else step()
            outs.append((o.clone(), lse.clone(), sel.clone(), q.clone()))
        return caches, seq, outs

    eager, seq, outs = serve(False)
    other, seq2, outs2 = serve(True)
    assert seq.tolist() == lens == seq2.tolist()
    for a, b in zip(eager, other):
        assert torch.equal(a["records"], b["records"]) and torch.equal(a["summary"], b["summary"])
    for a, b in zip(outs, outs2):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    o, lse, sel, q = outs[-1]
    check_attention(eager[-1], table, lens, q, o[-1], lse[-1], selected=sel)


def test_another_stream_and_two_calls_at_once():
    """Calls on two streams with workspaces of their own; each matches the call made alone."""
    caches = [filled([5000 + 700 * i], 4, 128, 16, seed=80 + i) for i in range(2)]
    qs = [torch.randn(1, 16, 128, generator=torch.Generator().manual_seed(i)).bfloat16().to(DEV) for i in range(2)]
    alone = []
    for (c, t, n), q in zip(caches, qs):
        o, lse = torch.empty(1, 16, 128, device=DEV), torch.empty(1, 16, device=DEV)
        ommx_kv4_decode_attention(q, c["records"], t, n, o, lse)
        alone.append((o, lse))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [(torch.empty(1, 16, 128, device=DEV), torch.empty(1, 16, device=DEV)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (c, t, n), q, (o, lse) in zip(streams, caches, qs, got):
            with torch.cuda.stream(s):
                ommx_kv4_decode_attention(q, c["records"], t, n, o, lse)
    torch.cuda.synchronize()
    for (o, lse), (wo, wl) in zip(got, alone):
        assert torch.equal(o, wo) and torch.equal(lse, wl)


# ---- what only the device sees -----------------------------------------------------------------------------------
def test_bad_pages_and_lengths_are_reported_and_skipped():
    lens, H, D, page = [40, 40, 40], 2, 64, 16
    cache, table, length = filled(lens, H, D, page, seed=91)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(9)
    k, v = (torch.randn(3, H, D, generator=gen).bfloat16().to(DEV) for _ in range(2))
    bad = table.clone()
    bad[0, 2], bad[1, 2] = cache["records"].shape[0], -1
    before, s_before = cache["records"].clone(), cache["summary"].clone()
    ommx_kv4_append(k, v, cache["records"], bad, length, summary=cache["summary"], status=status)
    assert int(status) == _lib.ST_BAD_PAGE
    same = torch.arange(before.shape[0], device=DEV) != table[2, 2]
    assert torch.equal(cache["records"][same], before[same]) and torch.equal(cache["summary"][same], s_before[same])
    assert not torch.equal(cache["records"], before)
    # lengths: more rows than tokens, and past the table
    for n in ([0, 40, 40], [-5, 40, 40], [16 * table.shape[1] + 1, 40, 40]):
        status.zero_()
        rec = before.clone()
        ommx_kv4_append(k, v, rec, table, torch.tensor(n, dtype=torch.int32, device=DEV), status=status)
        assert int(status) == _lib.ST_BAD_LENGTH
        keep = torch.arange(before.shape[0], device=DEV)
        keep = (keep != table[1, 2]) & (keep != table[2, 2])
        assert torch.equal(rec[keep], before[keep])
    # positions outside the rotation's tables: neither the key nor the query is written
    status.zero_()
    rec, cos, sin = before.clone(), *(x.to(DEV) for x in angles(10, 64))
    q, out = torch.randn(3, 4, D, generator=gen).bfloat16().to(DEV), torch.full((3, 4, D), 3.0, dtype=torch.bfloat16, device=DEV)
    ommx_kv4_append(k, v, rec, table, length, q=q, q_out=out, cos=cos, sin=sin, positions=torch.tensor([10, -1, 1 << 40], device=DEV), status=status)
    assert int(status) == _lib.ST_BAD_LENGTH and torch.equal(rec, before) and bool((out == 3).all())
    # attention, reading back and selection skip bad pages and say so
    o, lse = torch.empty(3, 4, D, device=DEV), torch.empty(3, 4, device=DEV)
    status.zero_()
    ommx_kv4_decode_attention(q, before, bad, length, o, lse, status=status)
    assert int(status) == _lib.ST_BAD_PAGE and torch.isfinite(o).all()
    want, wl = torch.empty_like(o), torch.empty_like(lse)
    short = torch.tensor([32, 32, 40], dtype=torch.int32, device=DEV)
    ommx_kv4_decode_attention(q, before, table, short, want, wl)
    assert float((o - want).abs().max()) < 1e-2 and float((lse - wl).abs().max()) < 1e-4
    status.zero_()
    ko, vo = torch.zeros(3, H, D, device=DEV), torch.zeros(3, H, D, device=DEV)
    ommx_kv4_gather(before, bad, length, ko, vo, status=status)
    assert int(status) == _lib.ST_BAD_PAGE and bool((ko[:2] == 0).all()) and bool((ko[2] != 0).any())
    status.zero_()
    sel = torch.empty(3, H, 2, dtype=torch.int32, device=DEV)
    ommx_kv4_select_pages(q, cache["summary"], bad, length, sel, page_size=page, first_pages=0, last_pages=0, status=status)
    assert int(status) == _lib.ST_BAD_PAGE and int(sel.min()) >= 0 and int(sel.max()) <= 2


def test_row_starts_out_of_order_stay_inside():
    """Malformed row ranges are clamped: nothing outside the rows is read, nothing outside the sequences' pages written."""
    lens, H, D, page = [40, 40], 1, 64, 16
    cache, table, length = filled(lens, H, D, page, seed=95)
    k = torch.randn(4, H, D, generator=torch.Generator().manual_seed(9)).bfloat16().to(DEV)
    spare = torch.ones(cache["records"].shape[0], dtype=torch.bool, device=DEV)
    spare[table[:, :3].long().flatten()] = False
    before = cache["records"].clone()
    for start in ([0, 9, 4], [-3, 2, 100], [4, 2, 0], [5, 5, 5]):
        ommx_kv4_append(k, k, cache["records"], table, length, row_start=torch.tensor(start, dtype=torch.int32, device=DEV))
        assert torch.equal(cache["records"][spare], before[spare])
        ko = torch.full((4, H, D), 2.0, device=DEV)
        ommx_kv4_gather(cache["records"], table, length, ko, ko.clone(), row_start=torch.tensor(start, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("dtype,allowed", [(torch.bfloat16, 2.0 ** -9), (torch.float32, 0.0)])
def test_long_even_sums_keep_their_bits(dtype, allowed):
    """130 thousand tokens that weigh alike: the output is what is left of codes and zeros that nearly cancel, so what a sum of hundreds
    of products loses would show.  Of a value's error a weight's rounding gives 2^-12 of its group's range R at most, of either sign:
    averaged over N tokens 2^-12 R / sqrt(N).  A sum that is cut by up to half a step in 2^23 at each of 64 additions (bf16 output;
    32 else, where weights have 22 bits) is off by 2^-18 (2^-19) of itself, 15 scales <= R.  Both are doubled for the tail; outputs of bf16
    are rounded by 2^-9 of themselves."""
    n, D = 131072, 128
    cache, table, length = filled([n], 1, D, 64, seed=101)
    q = torch.zeros(1, 4, D, dtype=torch.bfloat16, device=DEV)
    o, lse = torch.empty(1, 4, D, dtype=dtype, device=DEV), torch.empty(1, 4, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse)
    k, v = ref.sequence(cache["records"], table[0], n)
    want = v.mean(1)                                                        # [1, D]
    R = float((v.unflatten(-1, (-1, 32)).amax(-1) - v.unflatten(-1, (-1, 32)).amin(-1)).max())
    off = 2 * (2.0 ** -12 * R / math.sqrt(n) + 2.0 ** -18 * R) if dtype == torch.bfloat16 else 2 * 2.0 ** -19 * R
    assert float((o[0].double() - want).abs().max()) <= off + allowed * float(want.abs().max())
    assert abs(float(lse[0, 0]) - math.log(n)) < 1e-4


@pytest.mark.parametrize("D,page,B,n,od", [(128, 16, 64, 8101, torch.bfloat16), (64, 64, 100, 6007, torch.float32), (128, 32, 9, 65003, torch.float32)])
def test_more_records_to_a_warp_than_it_looks_up_at_once(D, page, B, n, od):
    """Sequences that share their pages (one prompt, many continuations): hundreds of records to a warp, several lookups, partial sums."""
    H, Hq = 8, 16
    cache, table, _ = filled([n], H, D, page, seed=111)
    table = table.expand(B, -1).contiguous()
    lens = [n - 37 * b for b in range(B)]
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    o, lse = torch.empty(B, Hq, D, dtype=od, device=DEV), torch.empty(B, Hq, device=DEV)
    length = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse)
    k, v = ref.sequence(cache["records"], table[0], n)
    for b in range(0, B, 4):
        wo, wl = ref.attention(q[b], list(k[:, :lens[b]]), list(v[:, :lens[b]]), D ** -0.5)
        off, drift = bounds(q[b], k, v, D ** -0.5, od)
        assert float((o[b].double() - wo).abs().max()) <= off, b
        assert float((lse[b].double() - wl).abs().max()) <= drift + 2.0 ** -22 * float(wl.abs().max()), b
    again, lse2 = torch.empty_like(o), torch.empty_like(lse)
    for _ in range(3):
        ommx_kv4_decode_attention(q, cache["records"], table, length, again, lse2)
        assert torch.equal(o, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("H,width", [(8, 30), (8, 250), (2, 250), (16, 2000)])
def test_a_captured_call_follows_its_lengths(H, width):
    """One graph, replayed with other lengths, past `max_seq_len` too: whole rows, clusters, and rows shared by two kernels."""
    D, page, B, Hq = 128, 16, 3, 16
    cache, table, _ = filled([width * page], H, D, page, seed=121)
    table = table[:, :width].expand(B, -1).contiguous()
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    o, lse = torch.empty(B, Hq, D, device=DEV), torch.empty(B, Hq, device=DEV)
    length = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    work = torch.empty(kv4_workspace_floats(D), device=DEV)
    for most in (None, 40):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, workspace=work, max_seq_len=most)
        for lens in ([0, 0, 0], [width * page, 1, 0], [17, width * page // 2 + 3, 100], [width * page] * 3):
            length.copy_(torch.tensor(lens, dtype=torch.int32))
            o.fill_(7), lse.fill_(7)
            graph.replay()
            check_attention(cache, table, lens, q, o, lse)


def test_calls_behind_one_another_on_their_own_stream():
    """Selection, attention and an append of other rows back to back, each begun while the one before still runs: nothing is read early."""
    lens, H, D, page = [3000, 1234], 4, 128, 32
    cache, table, length = filled(lens, H, D, page, seed=131)
    gen = torch.Generator().manual_seed(7)
    table = torch.cat((table, table[:, -1:]), 1)
    steps = [torch.randn(2, 8 + 2 * H, D, generator=gen).bfloat16().to(DEV) for _ in range(12)]
    cos, sin = (x.to(DEV) for x in angles(4000, D))

    def run(wait):
        c = {k: v.clone() for k, v in cache.items()}
        n, out = length.clone(), []
        for x in steps:
            q, sel = torch.empty(2, 8, D, dtype=torch.bfloat16, device=DEV), torch.empty(2, H, 9, dtype=torch.int32, device=DEV)
            o, lse = torch.empty(2, 8, D, device=DEV), torch.empty(2, 8, device=DEV)
            for call in (lambda: n.add_(1),
                         lambda: ommx_kv4_append(x[:, 8:8 + H], x[:, 8 + H:], c["records"], table, n, q=x[:, :8], q_out=q, cos=cos, sin=sin, summary=c["summary"]),
                         lambda: ommx_kv4_select_pages(q, c["summary"], table, n, sel, page_size=page),
                         lambda: ommx_kv4_decode_attention(q, c["records"], table, n, o, lse, selected=sel),
                         lambda: ommx_kv4_decode_attention(q, c["records"], table, n, o[:, :], lse, selected=sel, max_seq_len=1)):
                call()
                if wait:
                    torch.cuda.synchronize()
            out += [q, sel, o, lse]
        return [c["records"], c["summary"]] + out

    slow = run(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        fast = run(False)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(slow, fast))


@pytest.mark.parametrize("B", [2, 70])
def test_bad_row_ranges_are_reported_and_their_sequences_skipped(B):
    """A range below 0, past the rows, or that ends before it begins: nothing of its sequence is stored, rotated or read, the others' is."""
    H, D, page, T = 2, 64, 16, 2 * B
    lens = [40 + b for b in range(B)]
    cache, table, length = filled(lens, H, D, page, seed=141)
    gen = torch.Generator().manual_seed(142)
    k, v, q = (torch.randn(T, n, D, generator=gen).bfloat16().to(DEV) for n in (H, H, 4))
    cos, sin = (x.to(DEV) for x in angles(200, D))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    good = [2 * b for b in range(B + 1)]
    for start, wrong in (([-2] + good[1:], [0]), (good[:-1] + [T + 1], [B - 1]), (good[:-1] + [T - 4], [B - 1]), ([T + 7] * (B + 1), list(range(B))),
                         (good[:-1] + [2 ** 31 - 1], [B - 1]), ([-2 ** 31] + good[1:], [0])):
        start = torch.tensor(start, dtype=torch.int32, device=DEV)
        rec, summ, q_out = cache["records"].clone(), cache["summary"].clone(), torch.full_like(q, 5.0)
        want, w_summ, w_out = rec.clone(), summ.clone(), q_out.clone()
        status.zero_()
        ommx_kv4_append(k, v, rec, table, length, row_start=start, q=q, q_out=q_out, cos=cos, sin=sin, summary=summ, status=status)
        assert int(status) == _lib.ST_BAD_LENGTH
        ko, vo = torch.full((T, H, D), 2.0, device=DEV), torch.full((T, H, D), 2.0, device=DEV)
        status.zero_()
        ommx_kv4_gather(rec, table, length, ko, vo, row_start=start, status=status)
        assert int(status) == _lib.ST_BAD_LENGTH
        for b in range(B):                        # each good sequence by a call of its own
            if b in wrong:
                continue
            mine = slice(2 * b, 2 * b + 2)
            two = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
            ommx_kv4_append(k[mine], v[mine], want, table[b:b + 1], length[b:b + 1], row_start=two, q=q[mine], q_out=w_out[mine], cos=cos, sin=sin, summary=w_summ)
            wk, wv = ref.sequence(want, table[b], lens[b])
            assert torch.equal(ko[mine], wk[:, -2:].transpose(0, 1).float()) and torch.equal(vo[mine], wv[:, -2:].transpose(0, 1).float())
        assert torch.equal(rec, want) and torch.equal(summ, w_summ) and torch.equal(q_out, w_out)
        rows = torch.zeros(T, dtype=torch.bool, device=DEV)
        for b in wrong:
            rows[2 * b:2 * b + 2] = True
        assert bool((ko[rows] == 2).all()) and bool((vo[rows] == 2).all())


@pytest.mark.parametrize("B,H,group,longest", [(8, 8, 4, 6000), (1, 2, 4, 30000), (3, 4, 2, 700)])
def test_lengths_that_change_between_calls_that_overlap(B, H, group, longest):
    """Steps of a length update, an append, a selection and attention in three forms, each begun while the one before still runs and each with
    outputs of its own: what the later kernels read before they wait is what the step wrote.  Lengths jump, so the deal of records to blocks
    does too; the first two cases take the second kernel (64 rows of parts, and two)."""
    D, page, steps = 128, 32, 10
    cache, table, _ = filled([longest] * B, H, D, page, seed=151)
    gen = torch.Generator().manual_seed(152)
    lens = [torch.randint(1, longest + 1, (B,), generator=gen, dtype=torch.int32) for _ in range(steps)]
    lens[1][:], lens[2][:] = 1, longest
    lens = [n.to(DEV) for n in lens]
    rows = [torch.randn(B, (group + 2) * H, D, generator=gen).bfloat16().to(DEV) for _ in range(steps)]
    cos, sin = (x.to(DEV) for x in angles(longest, D))
    Hq = group * H

    def run(wait):
        c = {k: v.clone() for k, v in cache.items()}
        n = torch.zeros(B, dtype=torch.int32, device=DEV)
        out = []
        for x, now in zip(rows, lens):
            q, sel = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV), torch.empty(B, H, 5, dtype=torch.int32, device=DEV)
            o, lse = [torch.full((B, Hq, D), 7.0, device=DEV) for _ in range(3)], [torch.full((B, Hq), 7.0, device=DEV) for _ in range(3)]
            for call in (lambda: n.copy_(now),
                         lambda: ommx_kv4_append(x[:, Hq:Hq + H], x[:, Hq + H:], c["records"], table, n, q=x[:, :Hq], q_out=q, cos=cos, sin=sin, summary=c["summary"]),
                         lambda: ommx_kv4_decode_attention(q, c["records"], table, n, o[0], lse[0]),
                         lambda: ommx_kv4_select_pages(q, c["summary"], table, n, sel, page_size=page),
                         lambda: ommx_kv4_decode_attention(q, c["records"], table, n, o[1], lse[1], selected=sel),
                         lambda: ommx_kv4_decode_attention(q, c["records"], table, n, o[2], lse[2], max_seq_len=1)):
                call()
                if wait:
                    torch.cuda.synchronize()
            out += [q, sel, *o, *lse]
        return [c["records"], c["summary"]] + out, c

    slow, c = run(True)
    check_attention(c, table, lens[-1].tolist(), slow[-8], slow[-6], slow[-3])
    check_attention(c, table, lens[-1].tolist(), slow[-8], slow[-5], slow[-2], selected=slow[-7])
    check_attention(c, table, lens[-1].tolist(), slow[-8], slow[-4], slow[-1])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):
            fast, _ = run(False)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(slow, fast))


def test_rows_read_back_with_ranges_in_order_and_out():
    """The clamped form's neighbours: of ranges in and out of order in one call, the good ones' rows come back, the others' stay as they were."""
    lens, H, D, page = [40, 50, 60], 1, 64, 16
    cache, table, length = filled(lens, H, D, page, seed=161)
    wants = [ref.sequence(cache["records"], table[b], lens[b]) for b in range(3)]
    for start, good in (([-1, 2, 1, 4], [2]), ([2, 0, 3, 3], [1]), ([0, 1, 4, 9], [0, 1])):
        ko, vo = torch.full((4, H, D), 2.0, device=DEV), torch.full((4, H, D), 3.0, device=DEV)
        wk, wv = ko.clone(), vo.clone()
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        ommx_kv4_gather(cache["records"], table, length, ko, vo, row_start=torch.tensor(start, dtype=torch.int32, device=DEV), status=status)
        for b in good:
            n = start[b + 1] - start[b]
            for to, want in ((wk, wants[b][0]), (wv, wants[b][1])):
                to[start[b]:start[b + 1]] = want[:, lens[b] - n:].transpose(0, 1).float()
        assert torch.equal(ko, wk) and torch.equal(vo, wv) and int(status) == _lib.ST_BAD_LENGTH


@pytest.mark.parametrize("shift", [-132, -125, -110, -60, 0, 60, 120])
def test_selection_does_not_depend_on_the_size_of_the_queries(shift):
    """The same queries, and keys, times a power of two: the same pages, down to the smallest numbers of bf16."""
    lens, H, D, page, n = [1500], 2, 64, 16, 9
    cache, table, length = filled(lens, H, D, page, seed=171)
    q = torch.randint(-1, 3, (1, 6, D), generator=torch.Generator().manual_seed(172)).double()
    want = ref.select(q[0], cache["summary"].cpu(), table[0].cpu(), lens[0], page, n, 1, 2)
    sel = torch.empty(1, H, n, dtype=torch.int32, device=DEV)
    scaled = (q * 2.0 ** shift).bfloat16().to(DEV)
    assert torch.equal(scaled.cpu().double(), q * 2.0 ** shift)
    ommx_kv4_select_pages(scaled, cache["summary"], table, length, sel, page_size=page)
    assert sel[0].tolist() == want
    if -90 < shift < 100:
        summary = (cache["summary"].double() * 2.0 ** shift).bfloat16()
        ommx_kv4_select_pages(q.bfloat16().to(DEV), summary, table, length, sel, page_size=page)
        assert sel[0].tolist() == want
