"""Quantised cache rows and attention over spans of rows, in 64 bits.

No counterpart in the reference: these are written from the operators'
definitions, and pinned by closed forms in ``tests/test_oracle_quantized.py``
(half-step bounds, ties, exponent limits, NaN blocks, ``torch.float8_e4m3fn``,
attention against a loop over tokens).
"""
import math

import numpy as np

BLOCK = 32
TOP = {"mx8": 448.0, "mx4": 6.0}
_E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _e4m3():
    """The 128 non-negative e4m3 codes' values; 0x7f is NaN."""
    c = np.arange(128)
    e, m = c >> 3, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    v[127] = np.nan
    return v


GRID = {"mx8": _e4m3(), "mx4": _E2M1}


def _encode(y, grid):
    """Nearest code of each magnitude (ties to the even code) with its sign."""
    g = grid[np.isfinite(grid)]
    a = np.abs(y)
    hi = np.clip(np.searchsorted(g, a), 1, len(g) - 1)
    lo = hi - 1
    below, above = a - g[lo], g[hi] - a
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    code = np.where(up, hi, lo)
    return code + np.where(np.signbit(y), 128 if len(grid) == 128 else 8, 0)


def quantize(x, fmt):
    """x [B, H, S, D] -> codes uint8 [B, H, S, W] (mx4: W / 2), scales uint8
    [B, H, W / 32, 32 ceil(S / 32)] (padding 0)."""
    x = np.asarray(x, dtype=np.float64)
    B, H, S, D = x.shape
    nb = -(-D // BLOCK)
    pad = np.zeros((B, H, S, nb * BLOCK))
    pad[..., :D] = x
    blk = pad.reshape(B, H, S, nb, BLOCK)
    with np.errstate(invalid="ignore"):
        amax = np.abs(blk).max(-1) if S and nb else np.zeros((B, H, S, nb))
    bad = ~np.isfinite(amax)
    amax = np.where(bad, 0.0, amax)
    # smallest e with amax <= top 2^e, by comparison from the logarithm
    with np.errstate(divide="ignore"):
        e = np.where(amax > 0, np.floor(np.log2(np.where(amax > 0, amax, 1.0) / TOP[fmt])), -200)
    e = np.where(amax > TOP[fmt] * np.exp2(e), e + 1, e)
    e = np.where(amax > TOP[fmt] * np.exp2(e), e + 1, e)
    e = np.clip(e, -127, 127)
    y = np.where(bad[..., None], 0.0, blk) / np.exp2(e)[..., None]
    code = _encode(y, GRID[fmt]).reshape(B, H, S, nb * BLOCK)
    code = np.where(np.repeat(bad, BLOCK, -1), 0, code).astype(np.uint8)
    if fmt == "mx4":
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    sc = np.where(bad, 255, e + 127).astype(np.uint8)
    scales = np.zeros((B, H, nb, -(-S // BLOCK) * BLOCK), dtype=np.uint8)
    scales[..., :S] = sc.transpose(0, 1, 3, 2)
    return code, scales


def values(codes, scales, fmt, D):
    """What codes and scales stand for [B, H, S, D]."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    S = codes.shape[2]
    if fmt == "mx4":
        codes = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:3], 2 * codes.shape[3])
    half = 128 if fmt == "mx8" else 8
    v = GRID[fmt][codes & (half - 1)] * np.where(codes & half, -1.0, 1.0)
    sc = scales[..., :S].astype(np.float64).transpose(0, 1, 3, 2)
    two = np.where(sc == 255, np.nan, np.exp2(sc - 127))
    return (v * np.repeat(two, BLOCK, -1))[..., :D]


def attend(q, groups, spans):
    """softmax attention of one token per request over several spans.

    q [B, H_q, D]; spans: dicts of k [N, H, S, *], v [N, H, S, D] (N = B, or 1:
    shared by the batch), valid [B, S] or None, and for a rotated span R
    [N, H, D, Dk] and dm [N, H, D] or None.  Returns (out [B, H_q, D],
    mean of |v| under the same weights, bound on the exponents' size: the
    largest sum of |products| behind a score, in nats)."""
    B, Hq, D = q.shape
    out, amean = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    size = 0.0
    for b in range(B):
        for h in range(Hq):
            kv = h // groups
            sc, vv = [], []
            for s in spans:
                n = b if s["k"].shape[0] == B else 0
                k, v = s["k"][n, kv], s["v"][n, kv]
                on = np.ones(len(k), bool) if s.get("valid") is None else s["valid"][b].astype(bool)
                k, v = k[on], v[on]
                x, bias, bsize = q[b, h], 0.0, 0.0
                xa = np.abs(x)
                if s.get("R") is not None:
                    R = s["R"][n, kv]
                    if s.get("dm") is not None:
                        bias, bsize = x @ s["dm"][n, kv], xa @ np.abs(s["dm"][n, kv])
                    xa, x = xa @ np.abs(R), x @ R
                sc.append((k @ x + bias) / math.sqrt(D))
                vv.append(v)
                if len(k):
                    size = max(size, float((np.abs(k) @ xa + bsize).max()) / math.sqrt(D))
            sc, vv = np.concatenate(sc), np.concatenate(vv)
            if len(sc) == 0:
                continue
            w = np.exp(sc - sc.max())
            out[b, h] = w @ vv / (w.sum() + 1e-6)
            amean[b, h] = w @ np.abs(vv) / (w.sum() + 1e-6)
    return out, amean, size
