"""Pages of a KV cache that requests of different lengths share.

No counterpart in the reference, whose caches are one tensor a layer, as long
as the longest request.  Here Keys and Values lie in pages of a few tokens
[pages, H_kv, page, D], and a table gives each request its pages, in any order:
token t of request b is row ``t % page`` of page ``table[b, t // page]``.
``lens[b]`` counts the request's tokens; every call takes the count with the
new tokens in it, so a step of a layer is

    q = append_pages(k, v, k_pages, v_pages, table, lens, q=q, positions=pos, inv_freq=f)
    out = kernels.paged_decode(q, k_pages, v_pages, table, lens, groups)

``paged_cache.PagedCache`` keeps table, lengths and pages of all layers.  The
kernels run on the current stream of the tensors' device, synchronise nothing
and may be captured in a HIP graph: lengths, starts and table are read on the
device.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from rotatek_amd import _lib
from rotatek_amd.quantized import check_lens, refused
from rotatek_amd.rotary import no_grad_only


def check_requests(table: torch.Tensor, lens: torch.Tensor, starts: Optional[torch.Tensor]) -> None:
    """Word what is wrong with a table, its lengths or starts."""
    if not isinstance(table, torch.Tensor) or table.dtype != torch.int32 or table.dim() != 2:
        raise ValueError("table must be an int32 tensor [B, pages of a request]")
    check_lens(lens, table.shape[0], "lens")
    if starts is not None and (not isinstance(starts, torch.Tensor) or starts.dtype != torch.int32
                               or tuple(starts.shape) != (table.shape[0] + 1,) or not starts.is_contiguous()):
        raise ValueError("starts must be a contiguous int32 tensor [B + 1]")


def append_pages(k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 table: torch.Tensor, lens: torch.Tensor, starts: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                 q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write new tokens to their pages, the Keys (and ``q``) rotated on the way.

    ``k_new`` / ``v_new`` [N, H_kv, D] with ``starts`` (device int32 [B + 1],
    ascending: request b's tokens are ``starts[b] .. starts[b + 1] - 1``; None:
    one token each), or [B, H_kv, T, D], T tokens each.  ``k_pages`` /
    ``v_pages`` [pages, H_kv, page, D] of the same type (fp16, bf16 or fp32; any
    strides; page a power of two from 8 on; ``kernels``' attention takes fp16 and
    bf16 pages alone), ``table`` device int32 [B, per],
    ``lens`` device int32 [B], new tokens counted.

    With ``positions`` ([axes, N] or [axes, B, T]) the Keys turn as in
    ``rotary.apply_rotary``; so does ``q`` ([N, H_q, D] or [B, H_q, T, D]), into
    ``q_out`` or a new tensor, which is returned.  Positions of the rotation need
    not be places in the cache.

    Tokens past a request's table, or whose page number is none of the pool's,
    are dropped; no other row changes.  Two tokens must not share a row."""
    if positions is None and (inv_freq is not None or sections is not None or q is not None):
        raise ValueError("inv_freq, sections and q go with positions")
    if positions is not None and inv_freq is None:
        raise ValueError("positions go with inv_freq")
    if q is None and q_out is not None:
        raise ValueError("q_out goes with q")
    if positions is not None and positions.dim() == k_new.dim() - 2:
        positions = positions.unsqueeze(0)
    dev = k_new.get_device()
    r = _lib.bind().paged_append(k_new, v_new, k_pages, v_pages, table, lens, starts, q, q_out, positions, inv_freq,
                                 sections, interleaved, _lib.raw_stream(dev))
    if r.__class__ is int:
        no_grad_only("append_pages", r)
        check_requests(table, lens, starts)
        refused("append_pages", r, dev, k_new, v_new, k_pages, v_pages, table, lens, starts, q, q_out, positions,
                inv_freq)
    return r


__all__ = ["append_pages"]
