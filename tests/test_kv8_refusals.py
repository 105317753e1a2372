"""What the 8-bit cache's entry points refuse, on the host and before anything is launched: no GPU is needed to be told."""
import ctypes as C

import pytest
import torch

from open_ommx_serve_b200 import ommx_kv8_alloc, ommx_kv8_append, ommx_kv8_decode_attention, ommx_kv8_evict, ommx_kv8_gather
from open_ommx_serve_b200 import _lib
from open_ommx_serve_b200.attention.kv8 import kv8_workspace_floats

B, H, HQ, D, PAGE = 3, 2, 4, 64, 32
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def base(dtype=torch.int8):
    c = ommx_kv8_alloc(5, H, D, page_size=PAGE, weight=True, dtype=dtype, device="cpu")
    return dict(codes=c["codes"], scales=c["scales"], weight=c["weight"], page_table=torch.zeros(B, 4, dtype=torch.int32), b_seq_len=torch.ones(B, dtype=torch.int32),
                k=torch.zeros(B, H, D, dtype=BF16), v=torch.zeros(B, H, D, dtype=BF16), q=torch.zeros(B, HQ, D, dtype=BF16), o=torch.zeros(B, HQ, D),
                lse=torch.zeros(B, HQ), kept=torch.zeros(B, H, 5, dtype=torch.int32))


def append(a, **more):
    return ommx_kv8_append(a["k"], a["v"], a["codes"], a["scales"], a["page_table"], a["b_seq_len"], **{"weight": a["weight"], **more})


def gather(a, **more):
    return ommx_kv8_gather(a["codes"], a["scales"], a["page_table"], a["b_seq_len"], a["k"], a["v"], **more)


def decode(a, **more):
    return ommx_kv8_decode_attention(a["q"], a["codes"], a["scales"], a["page_table"], a["b_seq_len"], a["o"], a["lse"], **{"weight": a["weight"], **more})


def evict(a, **more):
    return ommx_kv8_evict(a["codes"], a["scales"], a["weight"], a["page_table"], a["b_seq_len"], a["kept"], **more)


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("call", [append, gather, decode, evict])
def test_host_tensors_are_refused_last(call, dtype):
    with pytest.raises(RuntimeError, match="CUDA"):
        call(base(dtype))


I8 = torch.int8
ANY = [(dict(page_table=torch.zeros(B, 4)), ValueError, "page_table"), (dict(page_table=torch.zeros(2, 4, dtype=torch.int32)), ValueError, "rows for"),
       (dict(b_seq_len=torch.ones(B, dtype=torch.int64)), ValueError, "b_seq_len"), (dict(b_seq_len=torch.ones(2 * B, dtype=torch.int32)[::2]), ValueError, "b_seq_len"),
       (dict(page_table=torch.zeros(4, B, dtype=torch.int32).t()), ValueError, "contiguous rows"), (dict(page_table=[[0]]), TypeError, "tensor"),
       (dict(codes=torch.zeros(5, H, 2, 2, 16, D)), ValueError, "int8 or"), (dict(codes=torch.zeros(5, H, 2, 2, 16, D, dtype=torch.uint8)), ValueError, "int8 or"),
       (dict(codes=torch.zeros(5, H, 2, 2, 16, D, dtype=torch.float8_e5m2)), ValueError, "int8 or"), (dict(codes=torch.zeros(5, H, 2, 16, D, dtype=I8)), ValueError, "codes must"),
       (dict(codes=torch.zeros(5, H, 2, 2, 8, D, dtype=I8)), ValueError, "codes is"), (dict(codes=torch.zeros(5, H, 2, 1, 16, D, dtype=I8)), ValueError, "codes is"),
       (dict(codes=torch.zeros(5, H, 3, 2, 16, D, dtype=I8)), NotImplementedError, "page_size"), (dict(codes=torch.zeros(5, H, 2, 2, 16, 96, dtype=I8)), NotImplementedError, "head_dim"),
       (dict(codes=torch.zeros(5, 2 * H, 2, 2, 16, D, dtype=I8)[:, ::2]), ValueError, "contiguous"), (dict(codes=None), ValueError, "needed"),
       (dict(scales=torch.zeros(5, H, 2, 2)), ValueError, "scales"), (dict(scales=torch.zeros(4, H, 2, 2, dtype=torch.uint8)), ValueError, "scales"), (dict(scales=None), ValueError, "needed")]
WEIGHT = [(dict(weight=torch.zeros(5, H, PAGE, dtype=BF16)), ValueError, "weight"), (dict(weight=torch.zeros(5, H, 16)), ValueError, "weight"), (dict(weight=torch.zeros(5, PAGE, H).transpose(1, 2)), ValueError, "weight")]


@pytest.mark.parametrize("change,error,text", ANY + WEIGHT + [
    (dict(k=torch.zeros(B, H, D, dtype=torch.float64)), ValueError, "k_new"), (dict(v=torch.zeros(B, H, D)), ValueError, "v_new"),
    (dict(k=torch.zeros(B, H + 1, D, dtype=BF16)), ValueError, "k_new"), (dict(k=torch.zeros(B, D, H, dtype=BF16).transpose(1, 2)), ValueError, "contiguous"),
    (dict(k=torch.zeros(B + 1, H, D, dtype=BF16), v=torch.zeros(B + 1, H, D, dtype=BF16)), ValueError, "row_start")])
def test_append_refuses(change, error, text):
    with pytest.raises(error, match=text):
        append({**base(), **change})


@pytest.mark.parametrize("call", [append, gather])
@pytest.mark.parametrize("more,text", [(dict(row_start=torch.zeros(B, dtype=torch.int32)), "row_start"), (dict(row_start=torch.zeros(B + 1, dtype=torch.int64)), "row_start"),
                                       (dict(status=torch.zeros(1)), "status")])
def test_append_and_gather_refuse_options(call, more, text):
    with pytest.raises(ValueError, match=text):
        call(base(), **more)


@pytest.mark.parametrize("change,error,text", ANY + [
    (dict(k=torch.zeros(B, H, 2 * D, dtype=BF16)), ValueError, "k_out"), (dict(v=torch.zeros(B, H, D)), ValueError, "v_out"),
    (dict(k=torch.zeros(1, H, D, dtype=BF16).expand(B, H, D)), ValueError, "expanded")])
def test_gather_refuses(change, error, text):
    with pytest.raises(error, match=text):
        gather({**base(), **change})


@pytest.mark.parametrize("change,error,text", ANY + WEIGHT + [
    (dict(q=torch.zeros(B, HQ, D)), ValueError, "q must be"), (dict(q=torch.zeros(B, 5, D, dtype=BF16), o=torch.zeros(B, 5, D)), NotImplementedError, "multiple"),
    (dict(q=torch.zeros(B, 1, D, dtype=BF16)), NotImplementedError, "multiple"), (dict(o=torch.zeros(B, HQ + 1, D)), ValueError, "o is"),
    (dict(o=torch.zeros(B, HQ, D, dtype=torch.float64)), ValueError, "o must be"), (dict(o=torch.zeros(1, HQ, D).expand(B, HQ, D)), ValueError, "expanded"),
    (dict(lse=torch.zeros(B, HQ, dtype=BF16)), ValueError, "lse"), (dict(lse=torch.zeros(HQ, B).t()), ValueError, "lse"), (dict(lse=torch.zeros(1, HQ).expand(B, HQ)), ValueError, "lse")])
def test_decode_refuses(change, error, text):
    with pytest.raises(error, match=text):
        decode({**base(), **change})


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("more,text", [
    (dict(logit_cap=-1.0), "logit_cap"), (dict(logit_cap=NAN), "logit_cap"), (dict(logit_cap=INF), "logit_cap"), (dict(sm_scale=INF), "sm_scale"), (dict(sm_scale=1e39), "sm_scale"),
    (dict(max_seq_len=-1), "max_seq_len"), (dict(max_seq_len=1 << 40), "max_seq_len"), (dict(window=0), "window"), (dict(window=-5), "window"), (dict(window=1 << 31), "window"),
    (dict(sink_tokens=-1), "sink_tokens"), (dict(keep=NAN), "keep"), (dict(keep=INF), "keep"), (dict(weight_before=torch.zeros(5, H, 16)), "weight_before"),
    (dict(weight=None, weight_before=torch.zeros(5, H, PAGE)), "without weight"), (dict(status=torch.zeros(1)), "status")])
def test_decode_refuses_options(more, text):
    with pytest.raises(ValueError, match=text):
        decode(base(), **more)


@pytest.mark.parametrize("change,error,text", ANY + WEIGHT + [
    (dict(weight=None), ValueError, "needed"), (dict(kept=torch.zeros(B, H, 0, dtype=torch.int32)), ValueError, "kept"), (dict(kept=torch.zeros(B, H, 5, dtype=torch.int64)), ValueError, "kept"),
    (dict(kept=torch.zeros(B, HQ, 5, dtype=torch.int32)), ValueError, "kept")])
def test_evict_refuses(change, error, text):
    with pytest.raises(error, match=text):
        evict({**base(), **change})


@pytest.mark.parametrize("more,text", [
    (dict(sink_tokens=3, recent_tokens=3), "fit into"), (dict(sink_tokens=-1), "sink_tokens"), (dict(recent_tokens=-1), "recent_tokens"), (dict(recent_tokens=6), "fit into"),
    (dict(to_table=torch.zeros(B, 4)), "to_table"), (dict(to_table=torch.zeros(B + 1, 4, dtype=torch.int32)), "to_table"), (dict(to_table=torch.zeros(B, 0, dtype=torch.int32)), "to_table"),
    (dict(len_out=torch.zeros(B, dtype=torch.int64)), "len_out"), (dict(len_out=torch.zeros(B + 1, dtype=torch.int32)), "len_out"), (dict(max_seq_len=-1), "max_seq_len")])
def test_evict_refuses_options(more, text):
    with pytest.raises(ValueError, match=text):
        evict(base(), **more)


@pytest.mark.parametrize("more,error", [(dict(head_dim=80), NotImplementedError), (dict(page_size=48), NotImplementedError), (dict(dtype=torch.uint8), NotImplementedError),
                                        (dict(num_pages=0), ValueError), (dict(n_kv_heads=0), ValueError)])
def test_alloc_refuses(more, error):
    keys = {**dict(num_pages=4, n_kv_heads=2, head_dim=64, device="cpu"), **more}
    with pytest.raises(error):
        ommx_kv8_alloc(keys.pop("num_pages"), keys.pop("n_kv_heads"), keys.pop("head_dim"), **keys)


def c_args(cls):
    a = cls()
    a.cache.codes, a.cache.scales, a.cache.weight = 256, 256, 256
    a.cache.num_pages, a.cache.n_kv_heads, a.cache.head_dim, a.cache.page_size = 5, H, D, PAGE
    a.seqs.b_seq_len = a.seqs.page_table = 256
    a.seqs.page_table_stride, a.seqs.pages_per_seq, a.seqs.batch = 4, 4, B
    return a


@pytest.mark.parametrize("cls,entry", [(_lib.KV8AppendArgs, "append"), (_lib.KV8GatherArgs, "gather"), (_lib.KV8DecodeArgs, "decode"), (_lib.KV8EvictArgs, "evict")])
def test_the_c_entries_refuse_caches(cls, entry):
    f = getattr(_lib.load(), "ommx_b200_kv8_" + entry)
    assert f(None, None) == -1 and "null" in _lib.last_error()
    for change, rc, text in ((dict(head_dim=96), -2, "head_dim"), (dict(page_size=24), -2, "page_size"), (dict(code=2), -1, "code"), (dict(n_kv_heads=0), -1, "kv heads"),
                             (dict(codes=264), -1, "aligned"), (dict(scales=257), -1, "aligned"), (dict(weight=260), -1, "aligned"), (dict(codes=0), -1, "given")):
        a = c_args(cls)
        for k, v in change.items():
            setattr(a.cache, k, v)
        assert f(C.byref(a), None) == rc and text in _lib.last_error(), change
    a = c_args(cls)
    a.seqs.batch = -1
    assert f(C.byref(a), None) == -1 and "batch" in _lib.last_error()
    a = c_args(cls)
    a.seqs.b_seq_len = 0
    assert f(C.byref(a), None) == -1 and "b_seq_len" in _lib.last_error()


def test_the_c_entries_refuse_calls():
    lib = _lib.load()
    a = c_args(_lib.KV8AppendArgs)
    a.k_new = a.v_new = 256
    for change, text in ((dict(num_rows=-1), "num_rows"), (dict(num_rows=B, dtype=9), "dtype"), (dict(num_rows=B + 1), "row_start"), (dict(num_rows=B, k_new=0), "null")):
        b = c_args(_lib.KV8AppendArgs)
        b.k_new = b.v_new = 256
        b.dtype = _lib.OMMX_DT_BF16
        for k, v in change.items():
            setattr(b, k, v)
        assert lib.ommx_b200_kv8_append(C.byref(b), None) == -1 and text in _lib.last_error(), change

    def decode_with(**change):
        d = c_args(_lib.KV8DecodeArgs)
        d.q = d.o = d.lse = d.workspace = d.weight_before = 256
        d.q_dtype = d.o_dtype = _lib.OMMX_DT_BF16
        d.n_q_heads, d.sm_scale, d.keep, d.workspace_floats = HQ, 1.0, 1.0, 1 << 30
        for k, v in change.items():
            setattr(d, k, v)
        return lib.ommx_b200_kv8_decode(C.byref(d), None)

    for change, rc, text in ((dict(q_dtype=_lib.OMMX_DT_F32), -2, "q must"), (dict(o_dtype=7), -1, "o dtype"), (dict(n_q_heads=3), -2, "multiple"), (dict(logit_cap=-1.0), -1, "logit_cap"),
                             (dict(sm_scale=INF), -1, "sm_scale"), (dict(window=-1), -1, "window"), (dict(sink_tokens=-1), -1, "sink_tokens"), (dict(keep=NAN), -1, "keep"),
                             (dict(weight_before=None), -1, "kept must be given"), (dict(weight_before=260), -1, "aligned"), (dict(lse=None), -1, "null"), (dict(workspace_floats=4), -1, "workspace"), (dict(workspace=260), -1, "workspace")):
        assert decode_with(**change) == rc and text in _lib.last_error(), change

    def evict_with(**change):
        e = c_args(_lib.KV8EvictArgs)
        e.kept, e.budget = 256, 5
        for k, v in change.items():
            setattr(e, k, v)
        return lib.ommx_b200_kv8_evict(C.byref(e), None)

    for change, text in ((dict(budget=0), "budget"), (dict(sink_tokens=6), "fit into"), (dict(recent_tokens=-1), "fit into"), (dict(kept=None), "kept"), (dict(max_seq_len=-1), "max_seq_len")):
        assert evict_with(**change) == -1 and text in _lib.last_error(), change
    e = c_args(_lib.KV8EvictArgs)
    e.kept, e.budget, e.cache.weight = 256, 5, None
    assert lib.ommx_b200_kv8_evict(C.byref(e), None) == -1 and "weights" in _lib.last_error()


def test_lengths_that_overlap_are_refused():
    e = c_args(_lib.KV8EvictArgs)
    e.kept, e.budget = 256, 5
    for at in (256 + 4, 256 - 4 * (B - 1)):
        e.len_out = at
        assert _lib.load().ommx_b200_kv8_evict(C.byref(e), None) == -1 and "len_out" in _lib.last_error()


def test_weights_before_that_overlap_are_refused():
    """A step reads one token's weight before and writes another's: weights a few tokens apart would be read after they are written."""
    n = 5 * H * PAGE
    d = c_args(_lib.KV8DecodeArgs)
    d.q = d.o = d.lse = d.workspace = 256
    d.q_dtype = d.o_dtype = _lib.OMMX_DT_BF16
    d.n_q_heads, d.sm_scale, d.keep, d.workspace_floats = HQ, 1.0, 1.0, 1 << 30
    d.cache.weight = 1 << 20
    for off in (16, -16, 4 * n - 16, 16 - 4 * n):
        d.weight_before = (1 << 20) + off
        assert _lib.load().ommx_b200_kv8_decode(C.byref(d), None) == -1 and "apart" in _lib.last_error()


def test_workspace_sizes():
    assert kv8_workspace_floats(4, 32, 128, 512) == 0
    whole = kv8_workspace_floats(1, 32, 128, 513)
    assert whole > 0 and whole == kv8_workspace_floats(64, 32, 128, 100000)
    assert kv8_workspace_floats(2, 32, 128, 512, weight=True) == 2 * 2 * 32 + 512 * 2 * 32
    assert kv8_workspace_floats(1, 32, 128, 100000, window=300, sink_tokens=4) == 0         # 21 records
    assert kv8_workspace_floats(1, 8, 64, 100000, window=300, sink_tokens=4, weight=True) == 2 * 8 + 21 * 16 * 8
