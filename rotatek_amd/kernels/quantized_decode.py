"""Decode over quantised rows (``rotatek_amd.quantized.MXRows``).

The attention of ``rotatek_decode`` and ``full_channel_decode`` straight from
8- or 4-bit rows: nothing is widened in memory.  No counterpart in the
reference.  Queries enter the products exactly (as two bf16 terms, three for
fp32; a rotated query is q R rounded to as many), code times scale is exact in
bf16 (8-bit blocks below 2^-116 excepted), weights are two or three bf16
terms, and sums are fp32, so the result differs from the same attention over
the dequantised rows by those roundings, at most 2^-16 of a weight, and the
output's.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from rotatek_amd.kernels._span import check_query, launch
from rotatek_amd.quantized import MXRows


def _check_rows(**rows) -> None:
    for name, x in rows.items():
        if not isinstance(x, MXRows):
            raise ValueError(f"{name} must be MXRows (quantize_rows makes them)")


def rotatek_decode_quantized(q_full: torch.Tensor, R_partial: torch.Tensor, delta_mu: Optional[torch.Tensor],
                             k_full: MXRows, v_full: MXRows, mask_full: Optional[torch.Tensor], k_sparse: MXRows,
                             v_sparse: MXRows, num_kv_groups: int, len_full: Optional[torch.Tensor] = None,
                             out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, None, None]:
    """``rotatek_decode`` with the four spans quantised.

    ``q_full`` [B, H_q, D] fp16, bf16 or fp32; ``k_full`` / ``v_full`` rows
    [B, H_kv, S_f, D], ``k_sparse`` [B, H_kv, S_v, Dk], ``v_sparse``
    [B, H_kv, S_v, D], all of one format; ``R_partial`` [B, H_kv, D, Dk],
    ``delta_mu`` [B, H_kv, D] or None.  ``mask_full`` [B, S_f] uint8 / bool or
    None, ``len_full`` device int32 [B] or None: the prompt / text rows that
    count (what the others hold does not matter).  Returns
    ``(out [B, 1, H_q, D], None, None)`` in q's dtype; a request with nothing
    to attend gets zeros."""
    check_query(q_full)
    _check_rows(k_full=k_full, v_full=v_full, k_sparse=k_sparse, v_sparse=v_sparse)
    o = launch("rotatek_decode_quantized", q_full, (R_partial, delta_mu),
               (k_full, v_full, k_sparse, v_sparse, None, None), mask_full, len_full, num_kv_groups, out, False)
    return o, None, None


def full_channel_decode_quantized(q: torch.Tensor, k: MXRows, v: MXRows, num_kv_groups: int = 1,
                                  mask: Optional[torch.Tensor] = None, lens: Optional[torch.Tensor] = None,
                                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``full_channel_decode`` with the Keys and Values quantised: ``q``
    [B, H_q, D], ``k`` / ``v`` rows [B, H_kv, S, D]; ``mask`` [B, S] uint8 /
    bool and ``lens`` device int32 [B] as above.  Returns [B, 1, H_q, D]."""
    check_query(q)
    _check_rows(k=k, v=v)
    return launch("full_channel_decode_quantized", q, (None, None), (k, v, None, None, None, None), mask, lens,
                  num_kv_groups, out, False)


__all__ = ["full_channel_decode_quantized", "rotatek_decode_quantized"]
