"""Attention over the 4-bit cache where numbers are unusual: scales of logits of every sign, values of every size the cache holds, weights
far below the largest.  Every output is held to a bound of its own, for its head and its group of 32 channels.

Bounds, with p the softmax in 64 bits, s, z and V the cached scales, zeros and values of a group, n tokens:
* a weight times a scale is rounded to fp16, by 2^-11 of it at most, and its codes are 15 at most: 2^-11 * 15 sum p s; where the output is
  finer than bf16 the rest is rounded once more: 2^-21 * 15 sum p s;
* the largest product p s of a warp (over its tokens and all groups) lies above 2^9 in the units that fp16 has, whose steps are 2^-24: what is
  lost of a small one is half a step, 2^-34 of the largest, so n * 15 * 2^-34 max p s in all;
* the tensor cores line the addends of a product of 16 up with the largest and cut them 25 bits below its leading one.  A masked nibble is an
  fp16 subnormal, code * 2^-24, that counts as 2^-14 there: an addend (16 and the sum so far) loses up to 2^-15 of one code of the record's
  heaviest token, 17 * 2^-15 max p s a record, 18 with the product of what the rounding left; and the sum, where it is the largest, up to
  2^-23 of itself at each of 64 additions: 2^-17 * 15 sum p s;
* the same in the two products of a group's logits, 33 * 2^-15 max |q| s_K of the group (its channels); beside it they are fp32 sums of a
  few hundred terms, off by 2^-17 of |q|.|K|.  Times sm_scale, and with 2^-20 for the exponential, that is the share d by which a weight
  is off, an output by 2 d (sum p |V| + |o|) <= 4 d sum p |V|;
* sums of zeros and of weights are 32-bit chains.  A warp has n / 64 records at most (four warps or more share a row in turns); a lane adds two
  tokens' zeros of each, n / 32 additions and up to 64 more to merge, each rounded by 2^-24 of the sum, all the same way where all addends
  are alike: (n / 32 + 64) 2^-24 sum p |z|, and of weights, one addition a record, (n / 64 + 64) 2^-24 of the output;
* the output is rounded by half a step.
The log-sum-exp is off by d, by the share that the sum of weights is, and by 2^-22 of itself.
"""
import math

import pytest
import torch

import kv4_reference as ref
from test_kv4_gpu import DEV, filled, rows_of, tables
from open_ommx_serve_b200 import ommx_kv4_alloc, ommx_kv4_append, ommx_kv4_decode_attention

pytestmark = pytest.mark.gpu


def parameters(records, table, length, at):
    """Scales and zeros of a sequence's keys (at 16) or values (18): [H, length, D / 32] each, in 64 bits."""
    S, D = records.shape[2], records.shape[3] // 20
    rec = records[table[:-(-length // (16 * S))].long()]
    words = rec[..., at * D:(at + 2) * D].contiguous().view(torch.int32).unflatten(-1, (16, D // 32)).transpose(0, 1).flatten(1, 3)[:, :length]
    return (words & -65536).view(torch.float32).double(), (words << 16).view(torch.float32).double()


def expected(q, records, table, n, sm_scale, cap, o_dtype):
    """o, lse of one sequence in 64 bits, and how far from them a kernel may be: q [Hq, D]."""
    k, v = ref.sequence(records, table, n)
    (s, z), (sk, _) = parameters(records, table, n, 18), parameters(records, table, n, 16)
    group = q.shape[0] // k.shape[0]
    eps = torch.finfo(o_dtype).eps / 2
    outs = []
    for h in range(q.shape[0]):
        kk, vv, ss, zz, sq = (x[h // group] for x in (k, v, s, z, sk))
        x = kk @ q[h].double() * sm_scale
        top = q[h].double().abs().unflatten(0, (-1, 32)).amax(-1)            # of each group
        d = float((2.0 ** -17 * (kk.abs() @ q[h].double().abs()) + 33 * 2.0 ** -15 * (sq @ top)).max()) * abs(sm_scale) + 2.0 ** -20
        if cap:
            x = cap * torch.tanh(x / cap)
        p = torch.softmax(x, 0)
        o, lse = p @ vv, torch.logsumexp(x, 0)
        codes = 15 * (p @ ss)                                                # of each group
        ps = p[:, None] * ss
        heaviest = torch.cat((ps, ps.new_zeros(-n % 16, ps.shape[1]))).unflatten(0, (-1, 16)).amax(1).sum(0)
        lost = 15 * n * 2.0 ** -34 * float(ps.max()) + 18 * 2.0 ** -15 * heaviest
        off = (codes * (2.0 ** -11 if o_dtype == torch.bfloat16 else 2.0 ** -21) + lost + 2.0 ** -17 * codes + (n / 32 + 64) * 2.0 ** -24 * (p @ zz.abs())).repeat_interleave(32)
        share = (n / 64 + 64) * 2.0 ** -24
        outs.append((o, lse, off + 4 * d * (p @ vv.abs()) + (eps + share) * o.abs(), d + share + 2.0 ** -22 * abs(float(lse))))
    return outs


def check(cache, table, lens, q, o, lse, sm_scale=None, cap=0.0, which=None):
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    for b in which or range(len(lens)):
        n = lens[b]
        for h, (wo, wl, off, drift) in enumerate(expected(q[b], cache["records"], table[b], n, sm_scale, cap, o.dtype)):
            worst = ((o[b, h].double() - wo).abs() / off.clamp(min=1e-300)).max()
            assert float(worst) <= 1, (b, h, n, float(worst))
            assert abs(float(lse[b, h]) - float(wl)) <= drift, (b, h, n, float(lse[b, h]), float(wl), drift)


# ---- the scale of the logits ---------------------------------------------------------------------------------------
FORMS = [
    # D, H, Hq, lens: a block to a row, a cluster to one, pieces of rows, even shares of all rows
    (128, 2, 6, [17, 250, 1, 5]),
    (128, 2, 8, [4001]),
    (64, 2, 2, [9001, 33]),
    (128, 8, 8, [611] + [300 + 3 * i for i in range(79)]),
]


@pytest.mark.parametrize("D,H,Hq,lens", FORMS)
@pytest.mark.parametrize("sm_scale,cap", [(0.0, 0.0), (-0.3, 0.0), (-0.05, 4.0), (0.0, 2.0), (1e-44, 0.0)])
def test_logit_scales_of_zero_and_below(D, H, Hq, lens, sm_scale, cap):
    """Tokens behind a sequence's end stay out whatever the scale's sign; a scale of 0 gives the mean."""
    cache, table, length = filled(lens, H, D, 16, seed=141)
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(142)).bfloat16().to(DEV)
    o, lse = torch.full((len(lens), Hq, D), 7.0, device=DEV), torch.full((len(lens), Hq), 7.0, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, sm_scale=sm_scale, logit_cap=cap, max_seq_len=max(lens))
    check(cache, table, lens, q, o, lse, sm_scale, cap, which=range(min(len(lens), 6)))
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()


# ---- the size of the values ----------------------------------------------------------------------------------------
def cache_of(k, v, page=16):
    """One sequence per entry of the lists k, v ([tokens, H, D]): (cache, table, lens tensor, lens)."""
    lens = [len(x) for x in k]
    table, P = tables(lens, page)
    cache = ommx_kv4_alloc(P, k[0].shape[1], k[0].shape[2], page_size=page, device=DEV)
    start, length = rows_of(lens, lens)
    ommx_kv4_append(torch.cat(k).to(DEV), torch.cat(v).to(DEV), cache["records"], table.to(DEV), length.to(DEV), row_start=start.to(DEV))
    return cache, table.to(DEV), length.to(DEV), lens


SIZES = [1e-30, 1e-24, 1e-20, 1e-16, 1e-12, 1e-3, 1e5, 1e12, 1e20, 1e30, 6e36]


@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("o_dtype", [torch.bfloat16, torch.float32])
def test_values_of_every_size(form, o_dtype):
    """Random values and constant ones from 2^-100 to near the 2^126 that the cache holds, with equal weights and others."""
    D, H, Hq, lens = FORMS[form]
    if lens[0] > 5000:
        lens = [4500, 33]                         # still in pieces, two launches
    gen = torch.Generator().manual_seed(151)
    k = torch.randn(sum(lens), H, D, generator=gen)
    v = torch.randn(sum(lens), H, D, generator=gen)
    q = torch.randn(len(lens), Hq, D, generator=gen)
    q[:, ::2] = 0
    q = q.bfloat16().to(DEV)
    o, lse = torch.empty(len(lens), Hq, D, dtype=o_dtype, device=DEV), torch.empty(len(lens), Hq, device=DEV)
    for size in SIZES:
        for values in (v * size, torch.full_like(v, size), torch.full_like(v, -size)):
            cache, table, length, _ = cache_of(k.split(lens), values.split(lens))
            ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, max_seq_len=max(lens))
            check(cache, table, lens, q, o, lse, which=range(min(len(lens), 4)))


@pytest.mark.parametrize("o_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("small,large", [(1.0, 1e36), (1e-20, 1e20), (1e-28, 1e8), (1e-25, 1e-5), (1.0, 0.0)])
def test_values_of_several_sizes_together(small, large, o_dtype):
    """Tokens that differ in size by up to 2^120, the large ones first, last, in between, heavy and light: sums of weights keep every token,
    whatever their values."""
    n, D = 700, 128
    gen = torch.Generator().manual_seed(152)
    at = [torch.arange(n) < 3, torch.arange(n) >= n - 3, torch.arange(n) % 50 == 7, torch.arange(n) % 2 == 0]
    k = [0.05 * torch.randn(n, 1, D, generator=gen) + a[:, None, None].float() for a in at]          # large ones are heavy, or light
    v = [torch.randn(n, 1, D, generator=gen) * torch.where(a, large, small)[:, None, None] for a in at]
    cache, table, length, lens = cache_of(k, v)
    for most in (None, n, 256 * 16):
        for weight in (0.0, 0.08, -0.08, 0.4, -0.4):
            q = torch.full((4, 2, D), weight).bfloat16().to(DEV)
            o, lse = torch.empty(4, 2, D, dtype=o_dtype, device=DEV), torch.empty(4, 2, device=DEV)
            ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, max_seq_len=most)
            check(cache, table, lens, q, o, lse)


# ---- a few tokens that outweigh all others ------------------------------------------------------------------------
@pytest.mark.parametrize("o_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,H,B,n", [(128, 8, 80, 15001), (64, 1, 1, 6001), (128, 4, 1, 130), (128, 2, 1, 4001)])
def test_tokens_far_below_the_heaviest_keep_their_bits(D, H, B, n, o_dtype):
    """Four tokens weigh 2^12 to 2^24 times as much as each of the thousands behind them, which all have the same weight and value, so that what
    is lost of one is lost of all; one group's values are 2^-10 of the others'.  The largest case has hundreds of records to a warp."""
    gen = torch.Generator().manual_seed(161)
    k, v = torch.zeros(n, H, D), torch.randn(1, H, D, generator=gen).repeat(n, 1, 1)
    heavy = [0, 16, 32, 48]
    k[heavy] = 1.0
    v[heavy] = torch.randn(4, H, D, generator=gen)
    v[..., 32:64] *= 2.0 ** -10
    cache, table, _, _ = cache_of([k], [v])
    table = table.expand(B, -1).contiguous()
    length = torch.full((B,), n, dtype=torch.int32, device=DEV)
    powers = torch.tensor([12, 15, 16.3, 18.7, 20, 20.6, 22.2, 24])
    q = (powers * math.log(2) / D ** 0.5).repeat(H)[None, :, None].expand(B, 8 * H, D).bfloat16().to(DEV)
    o, lse = torch.empty(*q.shape, dtype=o_dtype, device=DEV), torch.empty(*q.shape[:2], device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse)
    check(cache, table, [n] * B, q, o, lse, which=sorted({0, B // 2, B - 1}))


# ---- the size of the queries ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,lens", [(128, [40, 17]), (64, [3001])])
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_queries_of_every_size(D, lens, cap):
    """Queries from 2^-110 to 2^119 against keys as small or large, constant in their groups, so that the logits are ordinary numbers."""
    gen = torch.Generator().manual_seed(171)
    n = sum(lens)
    k = torch.randn(n, 2, D // 32, 1, generator=gen).expand(-1, -1, -1, 32).flatten(-2)
    v, q0 = torch.randn(n, 2, D, generator=gen), torch.randn(len(lens), 4, D, generator=gen).clamp(-3, 3)
    for e in (-110, -60, -14, 0, 60, 100, 110, 115, 117):
        cache, table, length, _ = cache_of((k * 2.0 ** -e).split(lens), v.split(lens))
        q = (q0 * 2.0 ** e).bfloat16().to(DEV)
        o, lse = torch.empty(len(lens), 4, D, device=DEV), torch.empty(len(lens), 4, device=DEV)
        ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, logit_cap=cap)
        check(cache, table, lens, q, o, lse, cap=cap)


# ---- weights and values that grow along a sequence -----------------------------------------------------------------
@pytest.mark.parametrize("o_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,n", [(1, 2000), (4, 250), (2, 9000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_small_values_that_hold_all_the_weight(H, n, o_dtype, sign):
    """Values grow by 2^30 along the sequence and the weights with them, or against them: then the output is of the size of the first values,
    some 1e-6, beside last ones of 1e3, and is held to its own size."""
    D = 128
    gen = torch.Generator().manual_seed(181)
    k = 0.1 * torch.randn(n, H, D, generator=gen) + torch.linspace(-4, 4, n)[:, None, None]
    v = torch.randn(n, H, D, generator=gen) * torch.logspace(-6, 3, n)[:, None, None]
    cache, table, length, lens = cache_of([k.bfloat16()], [v.bfloat16()])
    q = (sign * (1 + 0.1 * torch.randn(1, 4 * H, D, generator=gen))).bfloat16().to(DEV)
    o, lse = torch.empty(1, 4 * H, D, dtype=o_dtype, device=DEV), torch.empty(1, 4 * H, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse)
    check(cache, table, lens, q, o, lse)
    for h, (wo, _, off, _) in enumerate(expected(q[0], cache["records"], table[0], n, D ** -0.5, 0.0, o_dtype)):
        assert float(off.max()) < 0.5 * float(wo.abs().max()), h             # of the bound itself: an output of zeros would not pass


# ---- the size of the logits ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,H,lens", [(128, 2, [1, 17, 250]), (64, 2, [4001]), (128, 1, [9000])])
@pytest.mark.parametrize("power", [10, 20, 24, 27])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logits_of_every_size(D, H, lens, power, sign):
    """Logits of sign * 2^power * 1..4, exact in 32 bits, and values of 3e4: the output is the mean over the tokens of the largest logit.  In
    bf16 that is 2^-9 of itself off; the weights alike, products of codes off by 2^-11 and 2^-15 of a group's range R (2^-10 in all)."""
    gen = torch.Generator().manual_seed(191)
    n = sum(lens)
    steps = torch.randint(1, 5, (n, H, 1), generator=gen).float()
    k, v = steps.expand(n, H, D), 3e4 * torch.randn(n, H, D, generator=gen)
    cache, table, length, _ = cache_of(k.split(lens), v.split(lens))
    q = torch.ones(len(lens), 3 * H, D, dtype=torch.bfloat16, device=DEV)
    o, lse = torch.empty(len(lens), 3 * H, D, dtype=torch.bfloat16, device=DEV), torch.empty(len(lens), 3 * H, device=DEV)
    ommx_kv4_decode_attention(q, cache["records"], table, length, o, lse, sm_scale=sign * 2.0 ** power / D, max_seq_len=max(lens))
    for b, rows in enumerate(steps.split(lens)):
        _, cached = ref.sequence(cache["records"], table[b], lens[b])
        for h in range(3 * H):
            score = sign * rows[:, h // 3, 0].double().to(DEV)
            best = cached[h // 3][score == score.max()]
            want, size = best.mean(0), float(best.abs().max())
            R = float((best.unflatten(-1, (-1, 32)).amax(-1) - best.unflatten(-1, (-1, 32)).amin(-1)).max())
            assert float((o[b, h].double() - want).abs().max()) <= 2.0 ** -9 * size + 2.0 ** -10 * R
            top = float(score.max()) * 2.0 ** power
            assert abs(float(lse[b, h]) - top) <= math.log(len(best)) + 1e-3 + 2.0 ** -22 * abs(top)
