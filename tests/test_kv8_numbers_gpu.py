"""Attention over the 8-bit cache where numbers are unusual.  Every output is held to a bound of its own, for its head and channel.

Bounds, with p the softmax in 64 bits, V the cached values, s their scales, n tokens, `off` what a logit is off by (``kv8_reference.attention``):
* a weight is off by the share d = 2 off + 2^-20, the sum that divides it included, an output by 2 d sum p |V|;
* a weight times a scale goes to fp16: by 2^-11 of itself at most, by 2^-21 where the output is finer than bf16 (what the first rounding left is
  rounded once more).  The largest product of a warp lies above 2^10 in the units that fp16 has, whose last steps are 2^-24: half of one is 2^-35 of the
  largest, and codes are 448 at most: n 448 2^-35 max p s;
* a weight below 2^-126 of its reference counts as 0, and the sum that divides it is 1/2 at least: n 2^-125 max |V|;
* sums of up to 400 records of a warp are cut 24 bits below them: 2^-15 sum p |V|;
* the output is rounded by half a step.
The log-sum-exp is off by off + 2^-20 and four roundings of itself.
"""
import math

import pytest
import torch

import kv8_reference as ref
from test_kv8_gpu import BF16, DEV, E4M3, F32, I8, i32, random_cache, tables, to_gpu
from open_ommx_serve_b200 import ommx_kv8_decode_attention

pytestmark = pytest.mark.gpu


def hold(q, cache, table, lens, o, lse, sm, cap=0.0):
    """All outputs against 64 bits, within the bounds above."""
    group, page = q.shape[1] // cache["codes"].shape[1], 16 * cache["codes"].shape[2]
    half, fp16 = torch.finfo(o.dtype).eps / 2, 2.0 ** (-11 if o.dtype == BF16 else -21)
    for b, n in enumerate(lens):
        k, v = ref.sequence(cache["codes"], cache["scales"], table[b], n)
        wo, wl, p, off = ref.attention(q[b], k, v, sm, cap)
        t = torch.arange(n, device=q.device)
        E = cache["scales"][table[b, t // page].long(), :, t % page // 16, 1].T.double()                # [H, n]
        s = torch.where(E > 0, torch.exp2(E - 127), 0.0).repeat_interleave(group, 0)
        v = v.abs().repeat_interleave(group, 0)
        size, d = torch.einsum("ht,htd->hd", p, v), (2 * off + 2.0 ** -20)[:, None]
        tol = (2 * d + fp16 + 2.0 ** -15) * size + n * (448 * 2.0 ** -35 * (p * s).amax(1)[:, None] + 2.0 ** -125 * v.amax((1, 2))[:, None])
        tol = tol + half * wo.abs() + torch.finfo(o.dtype).tiny
        err = (o[b].double() - wo).abs()
        assert bool((err <= tol).all()), (b, n, int(o[b].isnan().sum()), float((err / tol).max()))
        err, tol = (lse[b].double() - wl).abs(), off + 2.0 ** -20 + 2.0 ** -22 * wl.abs()
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()))


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("D,large,light", [(128, 130, -1), (64, 130, -1), (128, 200, -71)])
@pytest.mark.parametrize("run,lens,H", [(4, [190], 64), (8, [384, 777], 2), (8, [3000], 3), (16, [5000], 4), (8, [2500, 20, 9000], 9)])
def test_blocks_of_zeros_before_large_values(run, lens, H, D, large, light, code, out):
    """Runs of blocks of three kinds: values of zero, which the even heads look at 200 powers of two above all others; small values; large ones, which
    count for nothing in the even heads and as much as the small ones in the odd heads.  The even heads' outputs are next to 0."""
    page = 16
    table, P = tables(lens, page)
    cache = random_cache(P, H, D, page, code, lo=127, hi=128)
    kinds = torch.zeros(P, dtype=torch.long)
    for b, n in enumerate(lens):
        need = -(-n // page)
        kinds[table[b, :need].long()] = torch.arange(need) // run % 3
    # keys of unit 1: channel 0 is 1 in the zeros' blocks, channel 1 in those of large values
    codes = cache["codes"]
    codes.view(torch.uint8)[:, :, :, 0] = 0
    codes[:, :, :, 0, :, 0] = (kinds == 0).float()[:, None, None, None].expand(-1, H, 1, 16).to(code)
    codes[:, :, :, 0, :, 1] = (kinds == 2).float()[:, None, None, None].expand(-1, H, 1, 16).to(code)
    codes.view(torch.uint8)[kinds == 0, :, :, 1] = 0
    cache["scales"][..., 1] = torch.tensor([0, 125, large], dtype=torch.uint8)[kinds][:, None, None]
    q = torch.zeros(len(lens), 6 * H, D)
    q[:, 0::2, 0] = 200.0
    q[:, 1::2, 1] = light
    cache, q = to_gpu(cache), q.bfloat16().to(DEV)
    o, lse, status = torch.empty(q.shape, dtype=out, device=DEV), torch.empty(q.shape[:2], device=DEV), i32([0])
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, sm_scale=math.log(2.0), status=status)
    assert int(status) == 0
    hold(q, cache, table.to(DEV), lens, o, lse, math.log(2.0))


def attend(lens, H, Hq, D, cache, table, q_scale, sm, dtype=BF16, cap=0.0, out=F32, seed=0):
    cache = to_gpu(cache)
    q = (torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(seed)).double() * q_scale).to(dtype).to(DEV)
    o, lse, status = torch.empty(q.shape, dtype=out, device=DEV), torch.empty(q.shape[:2], device=DEV), i32([0])
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, sm_scale=sm, logit_cap=cap, status=status)
    assert int(status) == 0
    hold(q, cache, table.to(DEV), lens, o, lse, sm, cap)


@pytest.mark.parametrize("code,D", [(I8, 128), (E4M3, 128), (I8, 64), (E4M3, 64)])
@pytest.mark.parametrize("size,sm,E", [(-104, 0, 224), (-118, 0, 238), (-128, 0, 245), (-128, 10, 235), (118, -4, 8), (100, -124, 146), (110, -145, 157), (-100, 120, 105),
                                       (-40, -60, 220), (-60, -50, 230), (60, 60, 3), (0, -130, 245)])
def test_queries_and_scales_of_every_size(size, sm, E, code, D):
    """Queries of 2^size, sm_scale 2^sm and keys of unit 2^(E - 127), whose logits are some powers of two."""
    lens = [40, 900]
    table, P = tables(lens, 16)
    cache = random_cache(P, 2, D, 16, code)
    cache["scales"][..., 0] = E
    attend(lens, 2, 8, D, cache, table, 2.0 ** size, 2.0 ** sm)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_a_large_channel_that_no_key_has(code, cap):
    """Queries of one channel, 2^110, which is 0 in every key: all logits are 0, whatever the keys' scales."""
    lens, D = [40, 900], 128
    table, P = tables(lens, 16)
    cache = random_cache(P, 2, D, 16, code, lo=1, hi=246)
    cache["scales"][..., 1] = 120
    cache["codes"].view(torch.uint8)[:, :, :, 0, :, 5] = 0
    q = torch.zeros(2, 4, D)
    q[..., 5] = 2.0 ** 110
    q, cache = q.bfloat16().to(DEV), to_gpu(cache)
    o, lse = torch.empty(q.shape, device=DEV), torch.empty(q.shape[:2], device=DEV)
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, sm_scale=1.0, logit_cap=cap)
    for b, n in enumerate(lens):
        _, v = ref.sequence(cache["codes"], cache["scales"], table[b].to(DEV), n)
        want = v.mean(1).repeat_interleave(2, 0)
        size = v.abs().mean(1).repeat_interleave(2, 0)
        # weights are 1, sums of them exact; values as above
        assert bool(((o[b].double() - want).abs() <= (2.0 ** -15 + 2.0 ** -21) * size + 2.0 ** -24 * want.abs()).all())
        assert float((lse[b].double() - math.log(n)).abs().max()) <= 2.0 ** -22 * math.log(n)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("cap", [3.4028234663852886e38, 1e38, 2.0 ** 60, 2.0 ** 41, 2.0 ** 39, 1e6, 1e-30, 1e-38, 1e-45])
@pytest.mark.parametrize("sm", [0.1, -3.0])
def test_caps_of_every_size(code, cap, sm):
    """Some keys are zeros, which no scale of logits makes anything else."""
    lens = [40, 0, 900]
    table, P = tables(lens, 16)
    cache = random_cache(P, 2, 128, 16, code)
    cache["scales"][::3, ..., 0] = 0
    cache["codes"].view(torch.uint8)[::3, :, :, 0] = 0
    lens[1] = 7                                           # on the first page of the pool, which is somebody's
    attend(lens, 2, 8, 128, cache, table, 1.0, sm, cap=cap)
