"""Rotation of queries and Keys by their positions, of one axis or several.

A text's tokens have one position each; an image's or a video's have one for
each axis (time, height, width), and each pair of channels turns by one of
them.  The reference leaves this to the models it patches, whose attention
rotates before it stores the Keys (integrations/lmms_eval/models/model_utils/
qwen/qwen2_5vl_visionzip.py:911-1077).

    q, k = apply_rotary(q, k, positions, inv_freq, sections=(16, 24, 24))

``paged.append_pages`` does the same on the way into a paged cache.  The
kernel runs on the current stream of the tensors' device and synchronises
nothing.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from rotatek_amd import _lib
from rotatek_amd.quantized import refused


def inverse_frequencies(channels: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """base^(-2i / channels), i = 0 .. channels / 2 - 1, fp32: the frequencies of
    a head that turns ``channels`` channels."""
    if channels < 2 or channels % 2:
        raise ValueError(f"channels must be even and at least 2, got {channels}")
    i = torch.arange(channels // 2, dtype=torch.float64)
    return (float(base) ** (-2.0 * i / channels)).to(torch.float32).to(device)


def no_grad_only(what: str, status: int) -> None:
    """Raise for a call whose inputs autograd would follow, backward or forward."""
    if status == _lib.bind().NEEDS_GRAD:
        raise RuntimeError(f"{what} has no gradient: call it on detached tensors or, where none has a tangent, under "
                           "torch.no_grad()")


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False, inverse: bool = False,
                 out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None,
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(q, k)`` rotated.

    ``q`` [B, H_q, T, D], ``k`` [B, H_kv, T, D] or None, ``positions``
    [axes, B, T]; or ``q`` [N, H_q, D], ``k`` [N, H_kv, D], ``positions``
    [axes, N] (int32 or int64; one axis may be left out).  fp16, bf16 or fp32,
    any strides, D up to 128.  ``inv_freq`` fp32 [P], 2 P <= D: pair i, channels
    i and i + P, turns by a = position inv_freq[i]:

        x_i cos a - x_(i+P) sin a,   x_(i+P) cos a + x_i sin a

    with the position of its axis: ``sections`` counts the pairs of each axis (up
    to four, P in all; None: one axis), one axis after the other, or with
    ``interleaved`` dealt in turn to the axes that have pairs left.  Channels
    from 2 P on are copied.  Angles are formed in 64 bits, so far positions keep
    their fractions of a turn.  ``inverse`` turns back (which moves a rotated Key
    to another position, and is the gradient's way).

    ``out``: tensors to write to, which may be ``q`` and ``k`` themselves."""
    if q.dim() not in (3, 4):
        raise ValueError(f"q needs 3 dims [N, H, D] or 4 [B, H, T, D], got shape {tuple(q.shape)}")
    if positions.dim() == q.dim() - 2:
        positions = positions.unsqueeze(0)
    q_out, k_out = (None, None) if out is None else out
    dev = q.get_device()
    r = _lib.bind().rotary(q, k, positions, inv_freq, sections, interleaved, inverse, q_out, k_out,
                           _lib.raw_stream(dev))
    if r.__class__ is int:
        no_grad_only("apply_rotary", r)
        refused("apply_rotary", r, dev, q, k, positions, inv_freq, q_out, k_out)
    return r


__all__ = ["apply_rotary", "inverse_frequencies"]
