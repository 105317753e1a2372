"""The account of attention weights that the 8-bit cache's attention keeps, against 64 bits, where tests of its other forms do not go."""
import math

import pytest
import torch

import kv8_reference as ref
from test_kv8_gpu import DEV, E4M3, I8, i32, random_cache, tables, to_gpu
from open_ommx_serve_b200 import _lib, ommx_kv8_decode_attention

pytestmark = pytest.mark.gpu


def account(lens, H, Hq, D, code, bad=(), keep=0.5, window=None, sinks=0, page=16, max_len=None, value=math.nan):
    """Weights of one call against 64 bits; `bad`: heads (sequence, head) whose query row is not finite, which are left out.  A weight is off by its
    share d and 2^-20 of itself; a head's below 2^-126 of its reference counts as 0, and the sum that divides it is 1/2 at least."""
    table, P = tables(lens, page)
    cache = to_gpu(random_cache(P, H, D, page, code))
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    given, group = q.clone(), Hq // H
    for b, h in bad:
        given[b, h, (7 * h + b) % D] = value
    o, lse, status = torch.empty(q.shape, device=DEV), torch.empty(q.shape[:2], device=DEV), i32([0])
    before = cache["weight"].clone()
    ommx_kv8_decode_attention(given, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, weight=cache["weight"], keep=keep, window=window,
                              sink_tokens=sinks, max_seq_len=max_len or max(lens), status=status)
    want, off_all = before.double().clone(), torch.zeros(before.shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        k, v = ref.sequence(cache["codes"], cache["scales"], table[b].to(DEV), n)
        seen = ref.visible(n, window, sinks)
        _, _, p, off = ref.attention(q[b], k[:, seen], v[:, seen], D ** -0.5)
        for h in range(Hq):
            wild = (b, h) in bad
            assert n == 0 or bool(o[b, h].isnan().all()) == wild and bool(lse[b, h].isnan()) == wild
            p[h] *= not wild
        t = torch.arange(n)
        ids, at = table[b, t // page].long().to(DEV), (t % page).to(DEV)
        add, tol = torch.zeros(2, H, n, dtype=torch.float64, device=DEV)
        add[:, seen] = p.view(H, group, -1).sum(1)
        tol[:, seen] = (p * (2 * off + 2.0 ** -20)[:, None]).view(H, group, -1).sum(1)
        now = want[ids, :, at].T * keep + add
        want[ids, :, at], off_all[ids, :, at] = now.T, (tol + 2.0 ** -20 * now.abs() + group * 2.0 ** -125).T
    err = (cache["weight"].double() - want).abs()
    assert bool((err <= off_all).all()), (int(cache["weight"].isnan().sum()), float((err - off_all).max()))
    return int(status)


# a block to a row, a cluster to a row, dealt rows with the account beside the join and behind it
FORMS = [[40, 0, 200], [1500], [900, 20, 12000], [20000, 4500, 3, 16000, 30000, 100]]


@pytest.mark.parametrize("lens", FORMS)
@pytest.mark.parametrize("H,Hq,bad", [(2, 8, [1, 6]), (2, 6, [0, 3, 4, 5]), (1, 33, [32]), (1, 72, [0, 70])])
@pytest.mark.parametrize("code,value", [(I8, math.nan), (E4M3, math.inf), (I8, -math.inf)])
def test_an_account_leaves_query_rows_out_that_are_not_finite(lens, H, Hq, bad, code, value):
    assert account(lens, H, Hq, 128, code, [(0, h) for h in bad], value=value) == _lib.ST_NONFINITE
    assert account(lens, H, Hq, 64, code, [(0, h) for h in bad], keep=0.0, window=300, sinks=5, value=value) == _lib.ST_NONFINITE


@pytest.mark.parametrize("lens", FORMS)
@pytest.mark.parametrize("H,group", [(1, 65), (2, 70), (1, 128), (2, 100)])
@pytest.mark.parametrize("code", [I8, E4M3])
def test_an_account_of_more_heads_than_a_block_holds(lens, H, group, code):
    """Their references and sums are made 64 at a time for each stretch of tokens: counts that four divides and others, blocks of several stretches."""
    assert account(lens, H, H * group, 64, code) == 0
    assert account(lens, H, H * group, 64, code, keep=-1.5, window=1000, sinks=20) == 0


def test_an_account_behind_the_join_and_its_launches():
    """Attention, the join and the account are three launches where the tokens are more than blocks beside the join take at once."""
    lib, H, D = _lib.load(), 8, 64
    for lens, want in (([20000] * 4, 3), ([20000], 2), ([200] * 4, 2)):
        table, P = tables(lens, 64)
        cache = to_gpu(random_cache(P, H, D, 64, I8))
        q, table, n = torch.randn(len(lens), H, D, device=DEV).bfloat16(), table.to(DEV), i32(lens)
        o, lse = torch.empty(q.shape, device=DEV), torch.empty(q.shape[:2], device=DEV)
        before = lib.ommx_b200_launch_count()
        ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table, n, o, lse, weight=cache["weight"], max_seq_len=max(lens))
        assert lib.ommx_b200_launch_count() - before == want


@pytest.mark.parametrize("H", [2, 40])
def test_the_account_of_a_sequence_beside_ones_past_max_seq_len(H):
    """Tokens within max_seq_len, in a sequence that is and in those that are not, get their weights; what is past it keeps its own."""
    lens, page, D, most = [800, 90, 3000], 16, 64, 100
    table, P = tables(lens, page)
    cache = to_gpu(random_cache(P, H, D, page, I8))
    before, q = cache["weight"].clone(), torch.randn(3, 4 * H, D, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    o, lse, status = torch.empty(q.shape, device=DEV), torch.empty(q.shape[:2], device=DEV), i32([0])
    ommx_kv8_decode_attention(q, cache["codes"], cache["scales"], table.to(DEV), i32(lens), o, lse, weight=cache["weight"], keep=0.25, max_seq_len=most, status=status)
    assert int(status) == _lib.ST_BAD_LENGTH
    for b, n in enumerate(lens):
        k, v = ref.sequence(cache["codes"], cache["scales"], table[b].to(DEV), n)
        _, _, p, off = ref.attention(q[b], k, v, D ** -0.5)
        add, tol = (x.view(H, 4, n).sum(1) for x in (p, p * (2 * off + 2.0 ** -20)[:, None]))
        t = torch.arange(n)
        ids, at = table[b, t // page].long().to(DEV), (t % page).to(DEV)
        was, now = before[ids, :, at].T.double(), cache["weight"][ids, :, at].T
        kept = -(-min(n, most) // 16) * 16                # records are counted, not tokens
        want = 0.25 * was + add
        assert bool(((now.double() - want).abs() <= tol + 2.0 ** -20 * want.abs() + 4 * 2.0 ** -125)[:, :kept].all())
        assert torch.equal(now[:, kept:], was[:, kept:].float())
