"""A paged KV cache held in 8 bits: append, read back, attend (to all tokens or a window), keep account of what is attended to, evict.

It stands beside the 4-bit cache (``attention.kv4``) and the 2-bit OMMX planes (``attention.kv_pool``) for models and layers that fewer
bits hurt, and has no counterpart in the reference.  A token's keys and values are int8 or e4m3 codes under a power of two for each
16 tokens and kv head: 256 bytes and 1/8 a token and kv head at ``head_dim`` 128, half of what bf16 takes.  int8 keeps more bits
where a block's values are alike, e4m3 where they differ in size.  ``include/ommx_b200.h`` gives the layout and the quantizer to the bit.

A decode step of a layer, all of it on the current stream, without host synchronisation, capturable in a CUDA graph::

    cache = ommx_kv8_alloc(num_pages, n_kv_heads, 128, page_size=32, weight=True)
    codes, scales, weight = cache["codes"], cache["scales"], cache["weight"]
    seq_len += 1                                                        # device lengths count the rows being appended
    ommx_kv8_append(k, v, codes, scales, table, seq_len, weight=weight)              # k, v as the model has them, rotated
    ommx_kv8_decode_attention(q, codes, scales, table, seq_len, o, lse, weight=weight)
    ...                                                                 # every few hundred tokens
    ommx_kv8_evict(codes, scales, weight, table, seq_len, kept, sink_tokens=4, recent_tokens=512, len_out=seq_len)

Layers that share ``seq_len`` give a ``len_out`` of their own.  Positions are the caller's: after an eviction a token's place in the cache is
not its position in the text.  Codes whose block's scale grows are rounded to it, so evict many tokens at a time rather than one a step.
Conditions that only the device sees (a length past its table, a page id out of range, rows that are not finite) are OR-ed into
``status`` (int32 ``[1]``, ``_lib.ST_*``), and the access is skipped.
"""
from __future__ import annotations

from typing import Dict, Optional

import torch

from .. import _lib

_HOST = None


def _host():
    global _HOST
    if _HOST is None:
        _HOST = _lib.host()
    return _HOST


def ommx_kv8_alloc(num_pages: int, n_kv_heads: int, head_dim: int = 128, *, page_size: int = 16, dtype: torch.dtype = torch.int8,
                   weight: bool = False, device="cuda") -> Dict[str, Optional[torch.Tensor]]:
    """An empty cache: ``codes`` (``dtype``: int8 or float8_e4m3fn) ``[num_pages, n_kv_heads, page_size / 16, 2, 16, head_dim]`` with a
    block's keys and then its values, ``scales`` uint8 ``[num_pages, n_kv_heads, page_size / 16, 2]`` (a value is
    ``code * 2 ** (scale - 127)``) and, to keep account of attention weights, ``weight`` fp32 ``[num_pages, n_kv_heads, page_size]``
    (``None`` without)."""
    if head_dim not in (64, 128):
        raise NotImplementedError(f"head_dim {head_dim}: this build serves 64 and 128")
    if page_size not in (16, 32, 64, 128, 256):
        raise NotImplementedError(f"page_size {page_size}: this build serves 16, 32, 64, 128 and 256")
    if dtype not in (torch.int8, torch.float8_e4m3fn):
        raise NotImplementedError(f"dtype {dtype}: this build holds int8 and float8_e4m3fn")
    if num_pages < 1 or n_kv_heads < 1:
        raise ValueError(f"a cache of {num_pages} pages of {n_kv_heads} kv heads")
    blocks = (num_pages, n_kv_heads, page_size // 16)
    return {"codes": torch.zeros(*blocks, 2, 16, head_dim, dtype=dtype, device=device),
            "scales": torch.zeros(*blocks, 2, dtype=torch.uint8, device=device),
            "weight": torch.zeros(num_pages, n_kv_heads, page_size, dtype=torch.float32, device=device) if weight else None}


def _check(rc, name):
    if rc != 0:
        _lib.check(rc, name)


def ommx_kv8_append(k_new: torch.Tensor, v_new: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor,
                    b_seq_len: torch.Tensor, *, row_start: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                    status: Optional[torch.Tensor] = None) -> None:
    """Store new rows.

    ``k_new`` / ``v_new`` ``[rows, n_kv_heads, D]`` in bf16, fp16 or fp32, any strides with a contiguous last dimension (slices of one
    projection's output).  ``b_seq_len`` (int32) counts the new rows: rows ``row_start[b] .. row_start[b + 1]`` (int32 ``[batch + 1]``)
    are the last tokens of sequence ``b``, without it row ``b`` is.  Rows behind ``row_start[-1]`` (a padded batch) are left alone.  A
    range that is none of the rows (below 0, past them, ending before it begins) is reported and its sequence skipped.  ``page_table``
    (int32 or int64 ``[batch, pages]``) gives the page of every ``page_size`` tokens; a page that takes rows belongs to one sequence.

    A block of 16 tokens has one scale for its keys and one for its values, which grow with what it takes; tokens it holds already are
    rounded to the larger one.  Rows that are stored again (a draft that was rejected) leave it as large as it was unless the
    block's first token is among them.  ``weight``: that of the new tokens is set to 0."""
    _check((_HOST or _host()).kv8_append(k_new, v_new, codes, scales, page_table, b_seq_len, row_start, weight, status), "ommx_b200_kv8_append")


def ommx_kv8_gather(codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, b_seq_len: torch.Tensor, k_out: torch.Tensor,
                    v_out: torch.Tensor, *, row_start: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """Read rows back into ``k_out`` / ``v_out`` ``[rows, n_kv_heads, D]`` (bf16, fp16 or fp32): the last ``row_start[b + 1] - row_start[b]``
    tokens of sequence ``b``, without ``row_start`` its last one.  With ``row_start = [0, cumsum(b_seq_len)]`` whole sequences."""
    _check((_HOST or _host()).kv8_gather(codes, scales, page_table, b_seq_len, k_out, v_out, row_start, status), "ommx_b200_kv8_gather")


def ommx_kv8_decode_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, b_seq_len: torch.Tensor,
                              o: torch.Tensor, lse: torch.Tensor, *, sm_scale: Optional[float] = None, logit_cap: float = 0.0,
                              window: Optional[int] = None, sink_tokens: int = 0, weight: Optional[torch.Tensor] = None,
                              weight_before: Optional[torch.Tensor] = None, keep: float = 1.0, workspace: Optional[torch.Tensor] = None,
                              max_seq_len: Optional[int] = None, status: Optional[torch.Tensor] = None) -> None:
    """Attention of one query row per sequence, written to ``o`` ``[batch, n_q_heads, D]`` and ``lse`` (fp32).

    ``q`` bf16 or fp16, ``o`` bf16, fp16 or fp32; any number of query heads to a kv head, whose cache is read once for each eight of
    them.  ``sm_scale`` defaults to ``D ** -0.5`` and may be any finite number; ``logit_cap`` c makes a logit ``c tanh(x / c)``.  A
    sequence of no tokens gives ``o = 0``, ``lse = -inf``; a query row that is not finite NaN, for its head alone.
    ``window``: only the last ``window`` tokens and the first ``sink_tokens`` are visible (all without one); what is not visible is not read.
    A token whose weight is below 2^-126 of the heaviest counts for nothing.
    ``weight``: every token of a sequence gets ``keep * weight_before`` (``weight`` itself, the default, or apart from it) plus the attention weights, each head's
    adding up to 1, of the query heads that share its kv head; with ``keep = 0`` those of this step alone.  A head whose query row is not finite is
    left out and reported (``ST_NONFINITE``).  Their pages belong to one sequence each.
    ``max_seq_len`` sizes the grid (the table's width without it); ``workspace`` (fp32, ``kv8_workspace_floats`` values) is
    allocated per call when one is needed and none is given; calls that run side by side need their own."""
    _check((_HOST or _host()).kv8_decode(q, codes, scales, page_table, b_seq_len, o, lse, sm_scale, logit_cap, window, sink_tokens, weight,
                                         weight_before, keep, workspace, max_seq_len, status), "ommx_b200_kv8_decode")


def ommx_kv8_evict(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, page_table: torch.Tensor, b_seq_len: torch.Tensor,
                   kept: torch.Tensor, *, sink_tokens: int = 0, recent_tokens: int = 0, to_table: Optional[torch.Tensor] = None,
                   len_out: Optional[torch.Tensor] = None, max_seq_len: Optional[int] = None,
                   status: Optional[torch.Tensor] = None) -> None:
    """Keep ``kept.shape[2]`` tokens of each sequence and kv head, and move them with their weights to the front, in their order.

    Kept are the first ``sink_tokens``, the last ``recent_tokens`` and of the others those of the largest ``weight`` (equal ones: the lower
    place; NaN last); all of a sequence that has no more.  Appended tokens weigh 0 until a step attends to them, so right after a prompt the lowest
    places stay: attend a few steps with an account first.  ``kept`` (int32 ``[batch, n_kv_heads, n]``) gets their places, ascending, then
    -1; ``len_out`` (int32 ``[batch]``, may be ``b_seq_len``) the new lengths.  They take the first pages of the sequence itself or,
    with ``to_table`` (int32 or int64 ``[batch, pages]``), pages that no sequence holds, and then the old ones are left as they were (a
    prefix that sequences share).  ``max_seq_len`` sizes the launch."""
    _check((_HOST or _host()).kv8_evict(codes, scales, weight, page_table, b_seq_len, kept, sink_tokens, recent_tokens, to_table, len_out,
                                        max_seq_len, status), "ommx_b200_kv8_evict")


def kv8_workspace_floats(batch: int, n_q_heads: int, head_dim: int, max_seq_len: int, *, window: Optional[int] = None, sink_tokens: int = 0,
                         weight: bool = False) -> int:
    """fp32 values of workspace that such calls of ``ommx_kv8_decode_attention`` need on the current device: where they keep account, mostly
    the logits of the visible tokens."""
    a = _lib.KV8DecodeArgs()
    a.cache.head_dim, a.cache.page_size, a.cache.weight = head_dim, 16, 16 if weight else None
    a.seqs.batch, a.seqs.pages_per_seq = batch, (max_seq_len + 15) // 16
    a.n_q_heads, a.max_seq_len, a.window, a.sink_tokens = n_q_heads, max_seq_len, window or 0, sink_tokens
    return int(_lib.load().ommx_b200_kv8_decode_workspace_floats(_lib.C.byref(a)))


__all__ = ["ommx_kv8_alloc", "ommx_kv8_append", "ommx_kv8_gather", "ommx_kv8_decode_attention", "ommx_kv8_evict",
           "kv8_workspace_floats"]
