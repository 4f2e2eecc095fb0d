"""Quantised rows of a KV cache: 8- or 4-bit codes with a power-of-two scale
for every 32 channels.

No counterpart in the reference, whose caches hold the model's dtype.  A row
takes 33/32 (``"mx8"``: e4m3 codes) or 17/32 (``"mx4"``: e2m1 codes) bytes a
channel instead of two.  A block of 32 channels is stored as the smallest
power of two that brings its largest magnitude to at most the element type's
largest value, and its values divided by that, rounded to nearest (ties to
even); a block with an infinity or a NaN reads back as NaN.

    rows = quantize_rows(x)                 # a span, at prefill
    append_rows(k_new, v_new, k, v, lens)   # new tokens, at decode
    x = dequantize_rows(rows)               # values again

``kernels.rotatek_decode_quantized``, ``kernels.full_channel_decode_quantized``
and ``kernels.shared_prefix_decode`` attend over such rows as they are.  The
kernels run on the current stream of the tensors' device and synchronise
nothing.
"""
from __future__ import annotations

from typing import Optional

import torch

from rotatek_amd import _lib

BLOCK = 32
FORMATS = {"mx8": _lib.RK_ROWS_MX8, "mx4": _lib.RK_ROWS_MX4}


def _format(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f"{fmt!r} is not a row format (use 'mx8' or 'mx4')")
    return FORMATS[fmt]


def _width(head_dim: int) -> int:
    return -(-head_dim // BLOCK) * BLOCK


class MXRows:
    """Quantised rows [B, H, S, head_dim] (a span of Keys or Values).

    ``codes`` uint8 [B, H, S, W], W = 32 ceil(head_dim / 32) (``"mx4"``:
    [B, H, S, W / 2], the even channel in the low four bits); ``scales`` uint8
    [B, H, W / 32, S'] with S' >= 32 ceil(S / 32): the exponents + 127, tokens
    adjacent, padded to whole groups of 32.
    """

    __slots__ = ("codes", "scales", "head_dim", "fmt")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, head_dim: int, fmt: str = "mx8") -> None:
        _format(fmt)
        self.codes, self.scales, self.head_dim, self.fmt = codes, scales, int(head_dim), fmt

    @classmethod
    def empty(cls, batch: int, heads: int, tokens: int, head_dim: int, fmt: str = "mx8", device="cuda") -> "MXRows":
        """Room for ``tokens`` rows, their content undefined until written."""
        _format(fmt)
        if not 0 <= head_dim <= 128:
            raise ValueError("head_dim must be 0..128")
        w = _width(head_dim)
        codes = torch.empty(batch, heads, tokens, w if fmt == "mx8" else w // 2, dtype=torch.uint8, device=device)
        scales = torch.empty(batch, heads, w // BLOCK, _width(tokens), dtype=torch.uint8, device=device)
        return cls(codes, scales, head_dim, fmt)

    @property
    def shape(self):
        """[B, H, S, head_dim]."""
        return (*self.codes.shape[:3], self.head_dim)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def narrow(self, start: int, tokens: int) -> "MXRows":
        """The rows ``start .. start + tokens - 1`` as a view; ``start`` a
        multiple of 32 (the scales' groups)."""
        if start < 0 or tokens < 0 or start % BLOCK or start + tokens > self.codes.shape[2]:
            raise ValueError(f"narrow needs start a multiple of {BLOCK} and start + tokens within the rows")
        return MXRows(self.codes.narrow(2, start, tokens), self.scales.narrow(3, start, _width(tokens)), self.head_dim,
                      self.fmt)

    def batch(self, start: int, count: int) -> "MXRows":
        """The rows of ``count`` requests as a view."""
        return MXRows(self.codes.narrow(0, start, count), self.scales.narrow(0, start, count), self.head_dim, self.fmt)

    def desc(self):
        """rk_rows of these rows, for callers of the C entries."""
        return _lib.rows_desc(self.codes, self.scales, self.head_dim, FORMATS[self.fmt])

    def __repr__(self) -> str:
        return f"MXRows({tuple(self.shape)}, {self.fmt!r}, device={str(self.device)!r})"


def same_device(what: str, index: int, *tensors) -> None:
    """All on GPU ``index`` (a tensor, MXRows or None each)."""
    if index < 0:
        raise RuntimeError(f"{what}: the kernels run only on the HIP device")
    for t in tensors:
        if t is None:
            continue
        if isinstance(t, MXRows):
            ok = t.codes.get_device() == index and t.scales.get_device() == index
        else:
            ok = t.get_device() == index
        if not ok:
            raise ValueError(f"{what}: every tensor must be on cuda:{index}")


def refused(what: str, status: int, index: int, *tensors) -> None:
    """Raise for a call that the host path answered with ``status``."""
    if status == _lib.bind().OTHER_DEVICE:
        same_device(what, index, *tensors)
    _lib.check(status, what)


def check_lens(lens: torch.Tensor, batch: int, name: str) -> None:
    if (not isinstance(lens, torch.Tensor) or lens.dtype != torch.int32 or lens.dim() != 1 or lens.shape[0] != batch
            or not lens.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor [B]")


def quantize_rows(x: torch.Tensor, fmt: str = "mx8", out: Optional[MXRows] = None) -> MXRows:
    """Quantise a span ``x`` [B, H, S, D] (fp16, bf16 or fp32, any strides, D
    up to 128), into ``out`` if given (rows of the same shape and format)."""
    _format(fmt)
    if x.dim() != 4:
        raise ValueError(f"x needs 4 dims [B, H, S, D], got shape {tuple(x.shape)}")
    if out is not None and out.fmt != fmt:
        raise ValueError(f"out holds {out.fmt} rows, not {fmt}")
    dev = x.get_device()
    r = _lib.bind().write(x, out, fmt, _lib.raw_stream(dev))
    if r.__class__ is tuple:
        return MXRows(*r, x.shape[3], fmt)
    if r:
        refused("quantize_rows", r, dev, x, out)
    return out


def dequantize_rows(rows: MXRows, dtype: torch.dtype = torch.bfloat16,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values [B, H, S, head_dim] that ``rows`` stand for, rounded once to
    ``dtype`` (into ``out``, of any strides and its own dtype, if given)."""
    dev = rows.codes.get_device()
    r = _lib.bind().read(rows, out, dtype, _lib.raw_stream(dev))
    if r.__class__ is not int:
        return r
    if r:
        refused("dequantize_rows", r, dev, rows, out)
    return out


def append_rows(k_new: torch.Tensor, v_new: Optional[torch.Tensor], k_rows: MXRows, v_rows: Optional[MXRows],
                lens: torch.Tensor, advance: bool = True) -> None:
    """Quantise new tokens ``k_new`` / ``v_new`` [B, H, T, D] into rows
    ``lens[b] ..`` of a cache, ``lens`` device int32 [B].

    Tokens past the capacity are dropped; no other row changes.  ``lens[b]``
    becomes ``min(lens[b] + T, capacity)``, or stays with ``advance=False``
    (drafted tokens, counted once they are accepted).  Device-only: may be
    captured in a HIP graph and replayed."""
    if (v_new is None) != (v_rows is None):
        raise ValueError("v_new and v_rows go together")
    dev = k_new.get_device()
    st = _lib.bind().append(k_new, v_new, k_rows, v_rows, lens, advance, _lib.raw_stream(dev))
    if st:
        check_lens(lens, k_new.shape[0], "lens")
        refused("append_rows", st, dev, k_new, v_new, k_rows, v_rows, lens)


__all__ = ["MXRows", "append_rows", "dequantize_rows", "quantize_rows"]
