"""Decode of a batch whose requests share a prompt and an image.

Many questions about one image (or behind one system prompt) attend over the
same Keys and Values.  ``rotatek_decode`` on an expanded batch reads them once
per request; here all the batch's queries on a KV head work on the same rows at
the same time, so the shared rows come from memory once, and a request's own
text is joined to the result in the same step.  No counterpart in the
reference.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from rotatek_amd.kernels._span import check_query, launch
from rotatek_amd.quantized import MXRows

Rows = Union[torch.Tensor, MXRows]


def shared_prefix_decode(q: torch.Tensor, k_prefix: Rows, v_prefix: Rows, k_suffix: Optional[Rows],
                         v_suffix: Optional[Rows], num_kv_groups: int, len_suffix: Optional[torch.Tensor] = None,
                         R_partial: Optional[torch.Tensor] = None, delta_mu: Optional[torch.Tensor] = None,
                         k_sparse: Optional[Rows] = None, v_sparse: Optional[Rows] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One decode step of B requests behind one prefix.

    ``q`` [B, H_q, D]; shared by all requests: ``k_prefix`` / ``v_prefix``
    [1, H_kv, S_p, D] and, for a pruned image, ``k_sparse`` [1, H_kv, S_v, Dk],
    ``v_sparse`` [1, H_kv, S_v, D] with ``R_partial`` [1, H_kv, D, Dk] and
    ``delta_mu`` [1, H_kv, D] (or None); each request's own: ``k_suffix`` /
    ``v_suffix`` [B, H_kv, S_s, D], of which the first ``len_suffix[b]``
    (device int32 [B]; None: all) rows count.  Rows are either all plain
    tensors in q's dtype (fp16, bf16; any strides) or all ``MXRows`` of one
    format (q fp16, bf16 or fp32).  Plain fp32 rows are refused: expand the
    prefix and call ``rotatek_decode``.

    The same as ``rotatek_decode`` of every request over its prefix, image and
    text.  Returns [B, 1, H_q, D] in q's dtype."""
    check_query(q)
    if (k_sparse is None) != (v_sparse is None) or (k_sparse is None) != (R_partial is None):
        raise ValueError("k_sparse, v_sparse and R_partial go together")
    if delta_mu is not None and R_partial is None:
        raise ValueError("delta_mu goes with R_partial")
    if (k_suffix is None) != (v_suffix is None) or (k_suffix is None and len_suffix is not None):
        raise ValueError("k_suffix and v_suffix go together, len_suffix with them")
    return launch("shared_prefix_decode", q, (R_partial, delta_mu),
                  (k_prefix, v_prefix, k_sparse, v_sparse, k_suffix, v_suffix), None, len_suffix, num_kv_groups, out,
                  True)


__all__ = ["shared_prefix_decode"]
