"""Launcher of the attention over quantised and shared spans."""
from __future__ import annotations

import ctypes

import torch

from rotatek_amd import _lib
from rotatek_amd.quantized import MXRows, check_lens, on_device, same_device

# Workspace bytes that calls on queries of a shape have needed so far: a call
# asks for as many, and sizes itself only where they do not suffice (the entry
# point checks).
_need: dict = {}


def rows_of(x):
    """rk_rows descriptor of MXRows or of a plain [B, H, S, D] tensor."""
    if x is None:
        return None
    if isinstance(x, MXRows):
        return x.desc()
    return _lib.rows_desc(x, None, x.shape[-1] if x.dim() else 0, _lib.RK_ROWS_PLAIN)


def _pack(x):
    """rows_of as bytes."""
    if x is None:
        return None
    if isinstance(x, MXRows):
        return x.pack()
    return _lib.pack_rows(x, None, x.shape[-1] if x.dim() else 0, _lib.RK_ROWS_PLAIN)


def check_query(q: torch.Tensor) -> None:
    if q.dim() != 3:
        raise ValueError(f"q needs 3 dims [B, H_q, D], got shape {tuple(q.shape)}")


def launch(what, q, rotation, rows, mask, lens, num_kv_groups, out, shared):
    """Validate, allocate ``out`` and the workspace, and launch; returns ``out``
    as [B, 1, H_q, D].

    ``rotation``: (R_partial, delta_mu); ``rows``: (K, V) of the full-width,
    rotated and, if ``shared``, suffix spans.  The workspace is this call's
    own, from torch's allocator: calls on two streams, and graphs captured one
    after the other, share none."""
    dev = q.get_device()
    same_device(what, dev, *rotation, *rows, mask, lens, out)
    if lens is not None:
        check_lens(lens, q.shape[0], "lens")
    lib = _lib.load()
    pack = _lib.pack
    dq = pack(q)
    shape = q.shape
    if out is None:
        out = torch.empty((shape[0], 1, *shape[1:]), dtype=q.dtype, device=q.device)
        do = _lib.pack_contiguous(out.data_ptr(), q.dtype, shape)
    else:
        do = pack(out)
        out = out.unsqueeze(1)
    dR, dm, dk = pack(rotation[0]), pack(rotation[1]), pack(mask)
    r = [_pack(x) for x in rows]
    groups = int(num_kv_groups)
    lens_ptr = None if lens is None else lens.data_ptr()
    key = (dev, shared, shape)
    with on_device(dev):
        s = _lib.raw_stream(dev)

        def call(nbytes):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            if shared:
                return lib.rk_shared_prefix_decode(dq, dR, dm, *r, lens_ptr, groups, do, ws.data_ptr(), nbytes, s)
            return lib.rk_quantized_decode(dq, dR, dm, r[0], r[1], dk, lens_ptr, r[2], r[3], groups, do, ws.data_ptr(),
                                           nbytes, s)

        st = call(_need.get(key, 256))
        if st == _lib.RK_ERR_WORKSPACE:
            need = ctypes.c_size_t(0)
            if shared:
                st = lib.rk_shared_prefix_decode_check(dq, dR, dm, *r, groups, do, 0, need)
            else:
                st = lib.rk_quantized_decode_check(dq, dR, dm, r[0], r[1], dk, r[2], r[3], groups, do, 0, need)
            _lib.check(st, what)
            if len(_need) > 4096:
                _need.clear()
            _need[key] = need.value
            st = call(need.value)
    _lib.check(st, what)
    return out
