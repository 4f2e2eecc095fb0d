"""Inputs, 64-bit results and tolerances shared by the tests of the attention
over quantised and shared spans.

Tolerance of an output o = sum w v / sum w, from the arithmetic (A = sum w |v|
/ sum w, eps of the type):
  * o is rounded once to its type: eps / 2 |o| (and half the smallest step);
  * a weight enters the product as 16-bit terms: bf16 in two, 2^-16 of it,
    fp16 in two, 2^-22, bf16 in three, 2^-24;
  * an exponent is a sum of products in fp32, each of the at most 129 + 8
    additions off by 2^-24 of the sum of magnitudes `size`, and the
    hardware's 2^x by 2^-22: relative error of a weight, and twice that for
    the quotient; queries of a rotated span are 16-bit terms of q R, 2^-16
    (fp32 2^-24; fp16 rows 2^-22 and, below fp16's smallest normal, 2^-25);
  * sums over tokens in fp32: one addition per 32 tokens and 64 for the
    joins, 2^-23 each, of A.
"""
import numpy as np
import torch

from oracle import quantized as oq

EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7, torch.float32: 2.0 ** -23}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def np64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def rows(x, fmt):
    """Plain [B, H, S, D] as the oracle's codes, as MXRows on the GPU, and as
    64-bit values of those codes."""
    from rotatek_amd.quantized import MXRows
    D = x.shape[-1]
    codes, scales = oq.quantize(np64(x), fmt)
    return MXRows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), D, fmt), \
        oq.values(codes, scales, fmt, D)


def tolerance(want, amean, size, tokens, dtype, fmt, rotated):
    term = 2.0 ** -22 if fmt == "plain" and dtype == torch.float16 else 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -16
    expo = size * 137 * 2.0 ** -24 + 2.0 ** -22
    if rotated:
        expo += size * (term + (2.0 ** -25 if fmt == "plain" and dtype == torch.float16 else 0.0))
    rel = term + 2 * expo + (tokens / 32 + 64) * 2.0 ** -23
    return EPS[dtype] / 2 * np.abs(want) + rel * (amean + np.abs(want)) + TINY[dtype]


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def check(out, q, groups, spans, fmt, dtype):
    """``out`` [B, 1, H_q, D] against the oracle over ``spans``."""
    want, amean, size = oq.attend(np64(q), groups, spans)
    tokens = sum(s["k"].shape[2] for s in spans)
    rotated = any(s.get("R") is not None for s in spans)
    assert out.shape == (q.shape[0], 1, *q.shape[1:]) and out.dtype == dtype
    got = np64(out)[:, 0]
    assert np.isfinite(got).all()
    over = np.abs(got - want) - tolerance(want, amean, size, tokens, dtype, fmt, rotated)
    assert (over <= 0).all(), f"past the tolerance by {over.max():.3e} (max error {np.abs(got - want).max():.3e})"
