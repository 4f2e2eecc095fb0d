"""Launcher of the attention over quantised and shared spans."""
from __future__ import annotations

import torch

from rotatek_amd import _lib
from rotatek_amd.quantized import MXRows, check_lens, refused


def rows_of(x):
    """rk_rows descriptor of MXRows or of a plain [B, H, S, D] tensor, for callers of
    the C entries (``launch`` forms its own in C++)."""
    if x is None:
        return None
    if isinstance(x, MXRows):
        return x.desc()
    return _lib.rows_desc(x, None, x.shape[-1] if x.dim() else 0, _lib.RK_ROWS_PLAIN)


def check_query(q: torch.Tensor) -> None:
    if q.dim() != 3:
        raise ValueError(f"q needs 3 dims [B, H_q, D], got shape {tuple(q.shape)}")


def launch(what, q, rotation, rows, mask, lens, num_kv_groups, out, shared):
    """Validate, allocate ``out`` (if None) and the workspace, and launch;
    returns ``out`` as [B, 1, H_q, D].

    ``rotation``: (R_partial, delta_mu); ``rows``: (K, V) of the full-width,
    rotated and suffix spans.  The workspace is this call's own, from torch's
    allocator: calls on two streams, and graphs captured one after the other,
    share none."""
    dev = q.get_device()
    r = _lib.bind().decode(shared, q, *rotation, *rows, mask, lens, int(num_kv_groups), out, _lib.raw_stream(dev))
    if r.__class__ is int:
        if lens is not None:
            check_lens(lens, q.shape[0], "lens")
        refused(what, r, dev, q, *rotation, *rows, mask, lens, out)
    return r
