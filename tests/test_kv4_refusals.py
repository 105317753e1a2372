"""What the 4-bit cache's entry points refuse, on the host and before anything is launched: no GPU is needed to be told."""
import ctypes as C

import pytest
import torch

from open_ommx_serve_b200 import (ommx_kv4_alloc, ommx_kv4_append, ommx_kv4_decode_attention, ommx_kv4_gather,
                                  ommx_kv4_select_pages)
from open_ommx_serve_b200 import _lib
from open_ommx_serve_b200.attention.kv4 import kv4_select_workspace_bytes, kv4_workspace_floats

B, H, HQ, D, PAGE = 3, 2, 4, 64, 32
BF16 = torch.bfloat16


def base():
    c = ommx_kv4_alloc(5, H, D, page_size=PAGE, summary=True, device="cpu")
    return dict(records=c["records"], summary=c["summary"], page_table=torch.zeros(B, 4, dtype=torch.int32), b_seq_len=torch.ones(B, dtype=torch.int32),
                k_new=torch.zeros(B, H, D, dtype=BF16), v_new=torch.zeros(B, H, D, dtype=BF16), q=torch.zeros(B, HQ, D, dtype=BF16),
                o=torch.zeros(B, HQ, D), lse=torch.zeros(B, HQ), selected=torch.zeros(B, H, 3, dtype=torch.int32),
                cos=torch.zeros(9, 32), sin=torch.zeros(9, 32))


def append(a, **more):
    keys = {k: a[k] for k in ("q", "cos", "sin", "summary")}
    keys.update(more)
    return ommx_kv4_append(a["k_new"], a["v_new"], a["records"], a["page_table"], a["b_seq_len"], **keys)


def decode(a, **more):
    return ommx_kv4_decode_attention(a["q"], a["records"], a["page_table"], a["b_seq_len"], a["o"], a["lse"], **more)


def gather(a, **more):
    return ommx_kv4_gather(a["records"], a["page_table"], a["b_seq_len"], a["k_new"], a["v_new"], **more)


def select(a, **more):
    keys = dict(page_size=PAGE)
    keys.update(more)
    return ommx_kv4_select_pages(a["q"], a["summary"], a["page_table"], a["b_seq_len"], a["selected"], **keys)


@pytest.mark.parametrize("call", [append, decode, gather, select])
def test_host_tensors_are_refused_last(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call(base())


ANY = [(dict(page_table=torch.zeros(B, 4)), ValueError, "page_table"), (dict(page_table=torch.zeros(2, 4, dtype=torch.int32)), ValueError, "rows for"),
       (dict(b_seq_len=torch.ones(B, dtype=torch.int64)), ValueError, "b_seq_len"), (dict(b_seq_len=torch.ones(2 * B, dtype=torch.int32)[::2]), ValueError, "b_seq_len"),
       (dict(page_table=torch.zeros(4, B, dtype=torch.int32).t()), ValueError, "contiguous rows"), (dict(page_table=[[0]]), TypeError, "tensor")]
RECORDS = [(dict(records=torch.zeros(5, H, 2, 20 * D)), ValueError, "uint8"), (dict(records=torch.zeros(5, H, 2, 20 * D + 1, dtype=torch.uint8)), ValueError, "20"),
           (dict(records=torch.zeros(5, H, 3, 20 * D, dtype=torch.uint8)), NotImplementedError, "page_size"),
           (dict(records=torch.zeros(5, H, 2, 20 * 96, dtype=torch.uint8)), NotImplementedError, "head_dim"),
           (dict(records=torch.zeros(5, 2 * H, 2, 20 * D, dtype=torch.uint8)[:, ::2]), ValueError, "contiguous")]


@pytest.mark.parametrize("change,error,text", ANY + RECORDS + [
    (dict(k_new=torch.zeros(B, H, D, dtype=torch.float64)), ValueError, "k_new"), (dict(v_new=torch.zeros(B, H, D)), ValueError, "v_new"),
    (dict(k_new=torch.zeros(B, H + 1, D, dtype=BF16)), ValueError, "k_new"), (dict(k_new=torch.zeros(B, D, H, dtype=BF16).transpose(1, 2)), ValueError, "contiguous"),
    (dict(k_new=torch.zeros(B + 1, H, D, dtype=BF16), v_new=torch.zeros(B + 1, H, D, dtype=BF16), q=torch.zeros(B + 1, HQ, D, dtype=BF16)), ValueError, "row_start"),
    (dict(q=torch.zeros(B, HQ, D)), ValueError, "dtype"), (dict(q=torch.zeros(B, HQ, 2 * D, dtype=BF16)), ValueError, "q is"),
    (dict(cos=None), ValueError, "together"), (dict(cos=None, sin=None), ValueError, "nothing to do"), (dict(cos=torch.zeros(9, 32, dtype=BF16)), ValueError, "float32"),
    (dict(sin=torch.zeros(8, 32)), ValueError, "same size"), (dict(cos=torch.zeros(9, 64), sin=torch.zeros(9, 64)), ValueError, "channels of heads"),
    (dict(cos=torch.zeros(9, 24), sin=torch.zeros(9, 24)), NotImplementedError, "48"), (dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)), ValueError, "row"),
    (dict(cos=torch.zeros(9, 33)[:, :32], sin=torch.zeros(9, 33)[:, :32]), ValueError, "16-byte"),
    (dict(summary=torch.zeros(5, H, 2, D)), ValueError, "summary"), (dict(summary=torch.zeros(4, H, 2, D, dtype=BF16)), ValueError, "summary")])
def test_append_refuses(change, error, text):
    with pytest.raises(error, match=text):
        append({**base(), **change})


@pytest.mark.parametrize("more,text", [
    (dict(row_start=torch.zeros(B, dtype=torch.int32)), "row_start"), (dict(row_start=torch.zeros(B + 1, dtype=torch.int64)), "row_start"),
    (dict(positions=torch.zeros(B - 1, dtype=torch.int32)), "positions"), (dict(positions=torch.zeros(B)), "positions"),
    (dict(q=None, q_out=torch.zeros(B, HQ, D, dtype=BF16)), "q_out without q"), (dict(q=None, cos=None, sin=None, positions=torch.zeros(B, dtype=torch.int32)), "positions without"),
    (dict(q_out=torch.zeros(1, HQ, D, dtype=BF16).expand(B, HQ, D)), "expanded"), (dict(q_out=torch.zeros(B, HQ, D)), "q_out"), (dict(status=torch.zeros(1)), "status")])
def test_append_refuses_options(more, text):
    with pytest.raises(ValueError, match=text):
        append(base(), **more)


@pytest.mark.parametrize("change,error,text", ANY + RECORDS + [
    (dict(q=torch.zeros(B, HQ, D)), ValueError, "q must be"), (dict(q=torch.zeros(B, 5, D, dtype=BF16), o=torch.zeros(B, 5, D)), NotImplementedError, "multiple"),
    (dict(q=torch.zeros(B, 1, D, dtype=BF16)), NotImplementedError, "multiple"), (dict(o=torch.zeros(B, HQ + 1, D)), ValueError, "o is"),
    (dict(o=torch.zeros(B, HQ, D, dtype=torch.float64)), ValueError, "o must be"), (dict(o=torch.zeros(1, HQ, D).expand(B, HQ, D)), ValueError, "expanded"),
    (dict(lse=torch.zeros(B, HQ, dtype=BF16)), ValueError, "lse"), (dict(lse=torch.zeros(HQ, B).t()), ValueError, "lse"), (dict(lse=torch.zeros(1, HQ).expand(B, HQ)), ValueError, "lse")])
def test_decode_refuses(change, error, text):
    with pytest.raises(error, match=text):
        decode({**base(), **change})


@pytest.mark.parametrize("more,text", [
    (dict(logit_cap=-1.0), "logit_cap"), (dict(logit_cap=float("nan")), "logit_cap"), (dict(logit_cap=float("inf")), "logit_cap"), (dict(selected=torch.zeros(B, H, 3)), "selected"),
    (dict(selected=torch.zeros(B, H + 1, 3, dtype=torch.int32)), "selected"), (dict(selected=torch.zeros(B, H, 0, dtype=torch.int32)), "selected"),
    (dict(max_seq_len=-1), "max_seq_len"), (dict(max_seq_len=1 << 40), "max_seq_len")])
def test_decode_refuses_options(more, text):
    with pytest.raises(ValueError, match=text):
        decode(base(), **more)


@pytest.mark.parametrize("change,error,text", ANY + RECORDS + [
    (dict(k_new=torch.zeros(B, H, 2 * D, dtype=BF16)), ValueError, "k_out"), (dict(v_new=torch.zeros(B, H, D)), ValueError, "v_out"),
    (dict(k_new=torch.zeros(1, H, D, dtype=BF16).expand(B, H, D)), ValueError, "expanded")])
def test_gather_refuses(change, error, text):
    with pytest.raises(error, match=text):
        gather({**base(), **change})


@pytest.mark.parametrize("change,error,text", ANY + [
    (dict(q=torch.zeros(B, HQ, D)), ValueError, "q must be"), (dict(q=torch.zeros(B, 3, D, dtype=BF16)), NotImplementedError, "multiple"),
    (dict(summary=torch.zeros(5, H, 2, D)), ValueError, "summary"), (dict(summary=None), ValueError, "needed"), (dict(selected=torch.zeros(B, H, 3)), ValueError, "selected"),
    (dict(selected=torch.zeros(B, H, 2, dtype=torch.int32)), ValueError, "fit into")])
def test_select_refuses(change, error, text):
    with pytest.raises(error, match=text):
        select({**base(), **change})


@pytest.mark.parametrize("more,error", [(dict(page_size=48), NotImplementedError), (dict(page_size=0), ValueError), (dict(first_pages=-1), ValueError), (dict(last_pages=3), ValueError)])
def test_select_refuses_options(more, error):
    with pytest.raises(error):
        select(base(), **more)


def test_alloc_refuses():
    for bad, error in ((dict(head_dim=96), NotImplementedError), (dict(page_size=8), NotImplementedError), (dict(page_size=48), NotImplementedError)):
        with pytest.raises(error):
            ommx_kv4_alloc(4, 2, **bad, device="cpu")
    with pytest.raises(ValueError):
        ommx_kv4_alloc(0, 2, device="cpu")


def test_the_c_abi_refuses_before_it_launches():
    lib = _lib.load()
    a = _lib.KV4AppendArgs()

    def says(fn, args, rc, text):
        assert fn(C.byref(args), None) == rc and text in _lib.last_error(), _lib.last_error()

    assert lib.ommx_b200_kv4_append(None, None) == -1 and lib.ommx_b200_kv4_gather(None, None) == -1
    assert lib.ommx_b200_kv4_decode(None, None) == -1 and lib.ommx_b200_kv4_select(None, None) == -1
    for args, fn in ((_lib.KV4AppendArgs(), lib.ommx_b200_kv4_append), (_lib.KV4GatherArgs(), lib.ommx_b200_kv4_gather),
                     (_lib.KV4DecodeArgs(), lib.ommx_b200_kv4_decode), (_lib.KV4SelectArgs(), lib.ommx_b200_kv4_select)):
        says(fn, args, -2, "head_dim")
        args.cache.head_dim, args.cache.page_size = 128, 24
        says(fn, args, -2, "page_size")
        args.cache.page_size = 16
        says(fn, args, -1, "kv heads")
        args.cache.n_kv_heads, args.cache.num_pages = 2, 4
        says(fn, args, -1, "records")
        args.cache.records = 4096 + 8
        says(fn, args, -1, "records")
        args.cache.records, args.cache.summary = 4096, 4096 + 2
        says(fn, args, -1, "summary")
        args.cache.summary, args.seqs.batch, args.seqs.pages_per_seq = 4096, 2, 3
        says(fn, args, -1, "b_seq_len")
        args.seqs.b_seq_len = args.seqs.page_table = 4096
        if isinstance(args, (_lib.KV4AppendArgs, _lib.KV4GatherArgs)):
            args.num_rows, args.dtype = 2, 7
            says(fn, args, -1, "dtype")
            args.dtype = _lib.OMMX_DT_F16
            says(fn, args, -1, "null")
    a.cache = _lib.KV4Cache(4096, None, 4, 2, 64, 16)
    a.seqs = _lib.KV4Seqs(4096, 4096, 3, 0, 3, 2)
    a.k_new = a.v_new = 4096
    a.dtype, a.num_rows = _lib.OMMX_DT_BF16, 3
    says(lib.ommx_b200_kv4_append, a, -1, "row_start")
    a.num_rows, a.rot_dim = 2, 48
    says(lib.ommx_b200_kv4_append, a, -2, "rot_dim")
    a.rot_dim = 128
    says(lib.ommx_b200_kv4_append, a, -1, "heads of 64")
    a.rot_dim = 64
    says(lib.ommx_b200_kv4_append, a, -1, "cos")
    a.cos = a.sin = 4096
    a.num_positions, a.cs_stride = 4, 31
    says(lib.ommx_b200_kv4_append, a, -1, "16-byte")
    a.cs_stride, a.q = 32, 4096
    says(lib.ommx_b200_kv4_append, a, -1, "q_out")
    d = _lib.KV4DecodeArgs(cache=a.cache, seqs=a.seqs)
    says(lib.ommx_b200_kv4_decode, d, -2, "q must be")
    d.q_dtype, d.n_q_heads = _lib.OMMX_DT_BF16, 3
    says(lib.ommx_b200_kv4_decode, d, -2, "multiple")
    d.n_q_heads, d.logit_cap = 4, -1.0
    says(lib.ommx_b200_kv4_decode, d, -1, "logit_cap")
    d.logit_cap = 0.0
    says(lib.ommx_b200_kv4_decode, d, -1, "null")
    d.q = d.o = d.lse = 4096
    assert lib.ommx_b200_kv4_decode_workspace_floats(C.byref(d)) == 0                       # 48 tokens: one launch without any
    d.seqs.pages_per_seq = 100
    assert lib.ommx_b200_kv4_decode_workspace_floats(C.byref(d)) == kv4_workspace_floats(64) > 0
    says(lib.ommx_b200_kv4_decode, d, -1, "workspace")
    d.workspace, d.workspace_floats = 4096, kv4_workspace_floats(64) - 1
    says(lib.ommx_b200_kv4_decode, d, -1, "workspace")
    d.workspace_floats, d.seqs.pages_per_seq, d.seqs.batch = 1 << 40, 1 << 24, 100
    says(lib.ommx_b200_kv4_decode, d, -2, "max_seq_len")
    d.cache.num_pages, d.cache.records = 0, None
    says(lib.ommx_b200_kv4_decode, d, -1, "no pages")
    s = _lib.KV4SelectArgs(cache=a.cache, seqs=a.seqs, q_dtype=_lib.OMMX_DT_F16, n_q_heads=4, num_selected=2, first_pages=1, last_pages=2)
    says(lib.ommx_b200_kv4_select, s, -1, "fit into")
    s.last_pages, s.n_q_heads = 1, 2 * 161
    says(lib.ommx_b200_kv4_select, s, -2, "query heads to a kv head")
    s.n_q_heads = 4
    says(lib.ommx_b200_kv4_select, s, -1, "null")
    s.q = s.selected = 4096
    says(lib.ommx_b200_kv4_select, s, -1, "summary")
    s.cache.summary = 4096
    says(lib.ommx_b200_kv4_select, s, -1, "workspace")
    assert kv4_select_workspace_bytes(2, 2, 3) >= 48 and kv4_select_workspace_bytes(-1, 2, 3) == 0 and kv4_workspace_floats(96) == 0


def test_struct_layouts_match_the_header():
    import os
    import re
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ommx_b200.h")).read()
    for struct, cls in (("ommx_kv4_cache", _lib.KV4Cache), ("ommx_kv4_seqs", _lib.KV4Seqs), ("ommx_kv4_append_args", _lib.KV4AppendArgs),
                        ("ommx_kv4_gather_args", _lib.KV4GatherArgs), ("ommx_kv4_decode_args", _lib.KV4DecodeArgs), ("ommx_kv4_select_args", _lib.KV4SelectArgs)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), header, re.S).group(1), flags=re.S)
        names = [n.strip().lstrip("*") for decl in body.split(";") if decl.strip() for n in re.sub(r"^(const\s+)?\w+\s+", "", decl.strip()).split(",")]
        assert names == [f[0] for f in cls._fields_], struct


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e300])
def test_a_logit_scale_that_is_no_32_bit_number_is_refused(bad):
    with pytest.raises(ValueError, match="sm_scale"):
        decode(base(), sm_scale=bad)
    d = _lib.KV4DecodeArgs(cache=_lib.KV4Cache(4096, None, 4, 2, 64, 16), seqs=_lib.KV4Seqs(4096, 4096, 3, 0, 3, 2), q_dtype=_lib.OMMX_DT_BF16, n_q_heads=4)
    d.sm_scale = bad if abs(bad) != 1e300 else float("inf")
    assert _lib.load().ommx_b200_kv4_decode(C.byref(d), None) == -1 and "sm_scale" in _lib.last_error()
