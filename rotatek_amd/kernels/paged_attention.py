"""Attention over the pages of a KV cache, and over the last tokens of a text.

The queries of a request's new tokens stand at its last positions; the one at
position p sees the tokens j <= p, with ``window`` only the last ``window`` of
them (p among them) and the first ``sinks`` of the request.  Scores are
q . k / sqrt(D); a query that sees nothing, or whose scores are all -inf, gives
zeros.  No counterpart in the reference, whose prefill attention is a library's and
whose caches are one tensor a layer.

fp16 and bf16, D a multiple of 8 up to 128.  Rows of Keys and Values lie in
whole 16-byte pieces (unit last stride, other strides multiples of 8 elements,
16-byte aligned); queries and outputs may have any strides.  Sums and softmax
statistics are fp32; the weights of many new tokens enter the products (and the sum
that divides them) rounded to the inputs' type, those of a single one in two terms
of it.

Values that are not finite count as the formula says for the queries that see them,
and not at all for the others (an infinity whose weight is below 2^-126 of the row's
largest may give a NaN).  They cost time: rows that do not see one in their tile are
summed again one by one (20 ms for 8192 tokens with one infinity, 0.4 without).

How the work is cut is planned from the table's width, since only the device knows
the lengths: a table much wider than its requests costs up to 1.8 times as much (16
requests of 500 tokens, 32/8 heads: 11.8 us, 14.9 with room for 32768; a prompt of
300, 28/4 heads: 14.9 and 27.1).  A KV head of more than 16 query heads is read once
for every 16 of them in ``paged_decode``.
"""
from __future__ import annotations

from typing import Optional

import torch

from rotatek_amd import _lib
from rotatek_amd.paged import check_requests
from rotatek_amd.quantized import check_lens, refused
from rotatek_amd.rotary import no_grad_only


def _seen(window: Optional[int]) -> int:
    if window is None:
        return 0
    if window < 1:
        raise ValueError(f"window must be at least 1 (or None), got {window}")
    return int(window)


def _paged(what, q, starts, k_pages, v_pages, table, lens, num_kv_groups, window, sinks, out):
    dev = q.get_device()
    r = _lib.bind().paged_attention(q, starts, k_pages, v_pages, table, lens, int(num_kv_groups),
                                    _seen(window), int(sinks), out, _lib.raw_stream(dev))
    if r.__class__ is int:
        no_grad_only(what, r)
        check_requests(table, lens, starts)
        refused(what, r, dev, q, starts, k_pages, v_pages, table, lens, out)
    return r


def paged_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 lens: torch.Tensor, num_kv_groups: int, window: Optional[int] = None, sinks: int = 0,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token of every request: ``q`` [B, H_q, D] at position
    ``lens[b] - 1`` over the pages of ``paged.append_pages``.  Returns
    [B, 1, H_q, D] (``out``: [B, H_q, D] to write to)."""
    if q.dim() != 3:
        raise ValueError(f"q needs 3 dims [B, H_q, D], got shape {tuple(q.shape)}")
    r = _paged("paged_decode", q, None, k_pages, v_pages, table, lens, num_kv_groups, window, sinks, out)
    return r if out is None else r.unsqueeze(1)


def paged_prefill(q: torch.Tensor, starts: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                  table: torch.Tensor, lens: torch.Tensor, num_kv_groups: int, window: Optional[int] = None,
                  sinks: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Many new tokens: ``q`` [N, H_q, D], request b's the rows ``starts[b] ..
    starts[b + 1] - 1`` (device int32 [B + 1], ascending), their Keys and Values
    already in the pages.  Returns [N, H_q, D]; rows that belong to no request
    are not written."""
    if q.dim() != 3:
        raise ValueError(f"q needs 3 dims [N, H_q, D], got shape {tuple(q.shape)}")
    if starts is None:
        raise ValueError("starts is needed (paged_decode takes one token of every request)")
    return _paged("paged_prefill", q, starts, k_pages, v_pages, table, lens, num_kv_groups, window, sinks, out)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_kv_groups: int = 1,
                     window: Optional[int] = None, sinks: int = 0, lens: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The same over plain rows: ``q`` [B, H_q, T, D] are the last T of the
    tokens of ``k`` / ``v`` [B, H_kv, S, D], of which the first ``lens[b]`` (device
    int32 [B]; None: all) are there.  Returns [B, H_q, T, D]."""
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.dim() != 4:
            raise ValueError(f"{name} needs 4 dims [B, H, tokens, D], got shape {tuple(x.shape)}")
    dev = q.get_device()
    r = _lib.bind().window_attention(q, k, v, lens, int(num_kv_groups), _seen(window), int(sinks), out,
                                     _lib.raw_stream(dev))
    if r.__class__ is int:
        no_grad_only("window_attention", r)
        if lens is not None:
            check_lens(lens, q.shape[0], "lens")
        refused("window_attention", r, dev, q, k, v, lens, out)
    return r


__all__ = ["paged_decode", "paged_prefill", "window_attention"]
