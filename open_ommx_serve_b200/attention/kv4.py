"""A paged KV cache held in 4 bits: append with the position rotation on the way, read back, attend, attend to selected pages.

It stands beside the 2-bit OMMX planes (``attention.kv_pool``, ``attention.paged_decode``) for models and layers that 2 bits
hurt, and has no counterpart in the reference.  Keys and values of a token are 4-bit codes with a bf16 scale and zero for each
32 channels - 160 bytes a token and kv head at ``head_dim`` 128, where bf16 takes 512 and the OMMX planes 132 - and no token
waits in a residual ring: a row is in the cache when the call that appends it is.  ``include/ommx_b200.h`` gives the record's
layout and the quantizer to the bit.

A decode step of a layer, all of it on the current stream, without host synchronisation, capturable in a CUDA graph::

    cache = ommx_kv4_alloc(num_pages, n_kv_heads, 128, page_size=32, summary=True)
    seq_len += 1                                                        # device lengths count the rows being appended
    ommx_kv4_append(k, v, cache["records"], table, seq_len, q=q, q_out=q, cos=cos, sin=sin, summary=cache["summary"])
    ommx_kv4_select_pages(q, cache["summary"], table, seq_len, selected, page_size=32)         # long contexts only
    ommx_kv4_decode_attention(q, cache["records"], table, seq_len, o, lse, selected=selected)

A prompt, or a chunk of one, is appended the same way with ``row_start``; the history that the chunk's own attention needs comes
back through ``ommx_kv4_gather``.  Conditions that only the device sees (a length past its table, a page id out of range, keys
that are not finite) are OR-ed into ``status`` (int32 ``[1]``, ``_lib.ST_*``), and the access is skipped.
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


def ommx_kv4_alloc(num_pages: int, n_kv_heads: int, head_dim: int = 128, *, page_size: int = 16, summary: bool = False,
                   device="cuda") -> Dict[str, Optional[torch.Tensor]]:
    """An empty cache: ``records`` uint8 ``[num_pages, n_kv_heads, page_size / 16, 20 * head_dim]`` and, for
    ``ommx_kv4_select_pages``, ``summary`` bf16 ``[num_pages, n_kv_heads, 2, head_dim]`` (``None`` without)."""
    if head_dim not in (64, 128):
        raise NotImplementedError(f"head_dim {head_dim}: this build serves 64 and 128")
    if page_size not in (16, 32, 64, 128, 256):
        raise NotImplementedError(f"page_size {page_size}: this build serves 16, 32, 64, 128 and 256")
    if num_pages < 1 or n_kv_heads < 1:
        raise ValueError(f"a cache of {num_pages} pages of {n_kv_heads} kv heads")
    return {"records": torch.zeros(num_pages, n_kv_heads, page_size // 16, 20 * head_dim, dtype=torch.uint8, device=device),
            "summary": torch.zeros(num_pages, n_kv_heads, 2, head_dim, dtype=torch.bfloat16, device=device) if summary else None}


def _check(rc, name):
    if isinstance(rc, int) and rc != 0:
        _lib.check(rc, name)


def ommx_kv4_append(k_new: torch.Tensor, v_new: torch.Tensor, records: torch.Tensor, page_table: torch.Tensor, b_seq_len: torch.Tensor, *,
                    row_start: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                    cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                    interleaved: bool = False, summary: Optional[torch.Tensor] = None,
                    status: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Store new rows; rotate their keys and, into ``q_out`` (returned; a fresh tensor when not given, may be ``q``), their queries.

    ``k_new`` / ``v_new`` ``[rows, n_kv_heads, D]`` and ``q`` ``[rows, n_q_heads, D]`` in bf16, fp16 or fp32, any strides with a
    contiguous last dimension (slices of one projection's output).  ``b_seq_len`` (int32) counts the new rows: rows
    ``row_start[b] .. row_start[b + 1]`` (int32 ``[batch + 1]``) are the last tokens of sequence ``b``, without it row ``b`` is.
    Rows behind ``row_start[-1]`` (a padded batch) are left alone, those of ``q_out`` too.  A range that is none of the
    rows (below 0, past them, ending before it begins) is reported and its sequence skipped.  ``page_table`` (int32 or int64
    ``[batch, pages]``) gives the page of every ``page_size`` tokens; a page that takes rows belongs to one sequence.

    ``cos`` / ``sin`` fp32 ``[positions, rot_dim / 2]`` turn the first ``rot_dim`` (32, 64, 128) channels, pairs
    ``(c, c + rot_dim / 2)`` or, ``interleaved``, ``(2 i, 2 i + 1)``, by the token's place in its sequence or by ``positions``
    (``[rows]``, int32 or int64).  A rotated key is rounded to its type before it is quantized: the cache holds what it would
    with a rotation of its own before the call.  ``summary`` keeps each touched page's channel maxima and minima; a page whose
    rows are stored again (a draft that was rejected) keeps what they held in its bounds until its first token is stored again.
    """
    out = (_HOST or _host()).kv4_append(k_new, v_new, records, page_table, b_seq_len, row_start, q, q_out, cos, sin, positions, interleaved,
                                        summary, status)
    _check(out, "ommx_b200_kv4_append")
    return out


def ommx_kv4_gather(records: torch.Tensor, page_table: torch.Tensor, b_seq_len: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, *,
                    row_start: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """Read rows back into ``k_out`` / ``v_out`` ``[rows, n_kv_heads, D]`` (bf16, fp16 or fp32; keys as stored, rotated): the last
    ``row_start[b + 1] - row_start[b]`` tokens of sequence ``b``, without ``row_start`` its last one.  With
    ``row_start = [0, cumsum(b_seq_len)]`` whole sequences."""
    _check((_HOST or _host()).kv4_gather(records, page_table, b_seq_len, k_out, v_out, row_start, status), "ommx_b200_kv4_gather")


def ommx_kv4_decode_attention(q: torch.Tensor, records: torch.Tensor, page_table: torch.Tensor, b_seq_len: torch.Tensor, o: torch.Tensor,
                              lse: torch.Tensor, *, sm_scale: Optional[float] = None, logit_cap: float = 0.0,
                              selected: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                              max_seq_len: Optional[int] = None, status: Optional[torch.Tensor] = None) -> None:
    """Attention of one (rotated) query row per sequence, written to ``o`` ``[batch, n_q_heads, D]`` and ``lse`` (fp32).

    ``q`` bf16 or fp16, ``o`` bf16, fp16 or fp32; any number of query heads to a kv head, whose cache is read once for each eight of
    them.  ``sm_scale`` defaults to ``D ** -0.5`` and may be any finite number; ``logit_cap`` c makes a logit ``c tanh(x / c)``.  A
    sequence of no tokens gives ``o = 0``, ``lse = -inf``.
    ``selected`` (int32 ``[batch, n_kv_heads, n]``, as ``ommx_kv4_select_pages`` writes it) limits a kv head to these places of
    the page table; the first ``min(n, pages)`` entries count, one below 0 is passed over, one listed twice counts twice.
    ``max_seq_len`` sizes the grid (the table's width without it; up to 512 tokens, and up to 4096 where sequences and heads are few, it
    is one launch); ``workspace`` (fp32, ``kv4_workspace_floats(D)`` values) is allocated per call when that may be more than 512 and
    none is given; calls that run side by side need their own."""
    _check((_HOST or _host()).kv4_decode(q, records, page_table, b_seq_len, o, lse, sm_scale, logit_cap, selected, workspace, max_seq_len, status),
           "ommx_b200_kv4_decode")


def ommx_kv4_select_pages(q: torch.Tensor, summary: torch.Tensor, page_table: torch.Tensor, b_seq_len: torch.Tensor, selected: torch.Tensor, *,
                          page_size: int, first_pages: int = 1, last_pages: int = 2, workspace: Optional[torch.Tensor] = None,
                          status: Optional[torch.Tensor] = None) -> None:
    """Write the pages that sequence ``b`` and kv head ``h`` attend to into ``selected[b, h]`` (int32 ``[batch, n_kv_heads, n]``):
    places in the page table, ascending, then -1.

    All pages where there are at most ``n``; else the first ``first_pages``, the last ``last_pages`` and those of the largest
    score: an estimate of the largest ``q . k`` of the page's keys from its channel maxima and minima in 7 bits and ``q`` in 8, the
    largest over the kv head's query heads.  Scores are whole numbers (``include/ommx_b200.h``), equal ones go to the lower page: the choice is the same
    however it is computed.  ``workspace``: uint8, ``kv4_select_workspace_bytes(batch, n_kv_heads, pages)``."""
    _check((_HOST or _host()).kv4_select(q, summary, page_table, b_seq_len, selected, page_size, first_pages, last_pages, workspace, status),
           "ommx_b200_kv4_select")


def kv4_workspace_floats(head_dim: int) -> int:
    """fp32 values of workspace that ``ommx_kv4_decode_attention`` needs on the current device."""
    return int(_lib.load().ommx_b200_kv4_workspace_floats(head_dim))


def kv4_select_workspace_bytes(batch: int, n_kv_heads: int, pages_per_seq: int) -> int:
    """Bytes of workspace that ``ommx_kv4_select_pages`` needs."""
    return int(_lib.load().ommx_b200_kv4_select_workspace_bytes(batch, n_kv_heads, pages_per_seq))


__all__ = ["ommx_kv4_alloc", "ommx_kv4_append", "ommx_kv4_gather", "ommx_kv4_decode_attention", "ommx_kv4_select_pages",
           "kv4_workspace_floats", "kv4_select_workspace_bytes"]
