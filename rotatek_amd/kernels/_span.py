"""Launcher of the attention over quantised and shared spans."""
from __future__ import annotations

import ctypes

import torch

from rotatek_amd import _lib
from rotatek_amd.quantized import MXRows, _same_device, check_lens, on_device


def rows_of(x):
    """rk_rows descriptor of MXRows or of a plain [B, H, S, D] tensor."""
    if x is None:
        return None
    if isinstance(x, MXRows):
        return x.desc()
    return _lib.rows_desc(x, None, x.shape[-1] if x.dim() else 0, _lib.RK_ROWS_PLAIN)


def check_query(q: torch.Tensor) -> None:
    if q.dim() != 3:
        raise ValueError(f"q needs 3 dims [B, H_q, D], got shape {tuple(q.shape)}")


def launch(what, q, rotation, rows, mask, lens, num_kv_groups, out, shared):
    """Validate, allocate ``out`` [B, H_q, D] and the workspace, and launch.

    ``rotation``: (R_partial, delta_mu); ``rows``: (K, V) of the full-width,
    rotated and, if ``shared``, suffix spans.  The workspace is this call's
    own, from torch's allocator: calls on two streams, and graphs captured one
    after the other, share none."""
    _same_device(what, q.device, *rotation, *rows, mask, lens, out)
    if lens is not None:
        check_lens(lens, q.shape[0], "lens")
    lib = _lib.load()
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dq, dR, dm, do, dk = (_lib.desc(t) for t in (q, *rotation, out, mask))
    dr = [rows_of(x) for x in rows]
    ref = _lib.ref
    head = (ref(dq), ref(dR), ref(dm))
    groups, need = int(num_kv_groups), ctypes.c_size_t(0)
    lens_ptr = None if lens is None else lens.data_ptr()
    r = [ref(x) for x in dr]
    with on_device(q.device):
        if shared:
            args = (*head, *r)
            st = lib.rk_shared_prefix_decode_check(*args, groups, ref(do), 0, ctypes.byref(need))
        else:
            st = lib.rk_quantized_decode_check(*head, r[0], r[1], ref(dk), r[2], r[3], groups, ref(do), 0,
                                               ctypes.byref(need))
        _lib.check(st, what)
        ws = torch.empty(max(need.value, 256), dtype=torch.uint8, device=q.device)
        s = _lib.stream_handle(q.device)
        if shared:
            st = lib.rk_shared_prefix_decode(*args, lens_ptr, groups, ref(do), ws.data_ptr(), ws.numel(), s)
        else:
            st = lib.rk_quantized_decode(*head, r[0], r[1], ref(dk), lens_ptr, r[2], r[3], groups, ref(do),
                                         ws.data_ptr(), ws.numel(), s)
        _lib.check(st, what)
    return out.unsqueeze(1)
