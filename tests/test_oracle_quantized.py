"""The 64-bit restatement of quantised rows, pinned by closed forms (CPU)."""
import math

import numpy as np
import pytest
import torch

from oracle import quantized as oq

STEP = {"mx8": 2.0 ** -4, "mx4": 2.0 ** -2}       # half a step relative to the value (e4m3, e2m1)
SMALL = {"mx8": 2.0 ** -10, "mx4": 0.25}          # half the smallest step, in units of 2^e


def _x(seed, *shape, spread=4.0):
    g = np.random.default_rng(seed)
    return (g.standard_normal(shape) * np.exp2(g.uniform(-spread, spread, shape))).astype(np.float32)


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
@pytest.mark.parametrize("D", [1, 31, 32, 40, 128])
def test_every_value_is_within_half_a_step(fmt, D):
    x = _x(D, 2, 3, 37, D)
    codes, scales = oq.quantize(x, fmt)
    w = 32 * (-(-D // 32))
    assert codes.shape == (2, 3, 37, w if fmt == "mx8" else w // 2)
    assert scales.shape == (2, 3, w // 32, 64)
    y = oq.values(codes, scales, fmt, D)
    e = scales[..., :37].astype(float).transpose(0, 1, 3, 2) - 127
    two = np.repeat(np.exp2(e), 32, -1)[..., :D]
    assert (np.abs(y - x) <= np.maximum(STEP[fmt] * np.abs(x), SMALL[fmt] * two)).all()
    # the exponent is the smallest that holds the block
    for i in range(0, D, 32):
        a = np.abs(x[..., i:i + 32]).max(-1)
        assert (a <= oq.TOP[fmt] * np.exp2(e[..., i // 32])).all()
        assert (a > oq.TOP[fmt] * np.exp2(e[..., i // 32] - 1)).all()
    # what is on the grid stays
    again = oq.values(*oq.quantize(y, fmt), fmt, D)
    assert np.array_equal(again, y)


def test_e4m3_codes_are_torchs():
    x = torch.from_numpy(_x(5, 1, 1, 64, 32))
    x = x / x.abs().amax(-1, keepdim=True) * 400.0      # exponent 0 throughout
    codes, scales = oq.quantize(x.numpy(), "mx8")
    assert (scales == 127).all()
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes, want)
    every = torch.arange(256, dtype=torch.uint8).view(1, 1, 8, 32)
    got = oq.values(every.numpy(), np.full((1, 1, 1, 32), 127, np.uint8), "mx8", 32)
    assert np.array_equal(got, every.view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)


def test_ties_go_to_even_codes():
    row = np.zeros((1, 1, 1, 32))
    row[0, 0, 0, :8] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    y = oq.values(*oq.quantize(row, "mx4"), "mx4", 32)[0, 0, 0, :8]
    assert list(y) == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    row[0, 0, 0, :5] = [448.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0]
    row[0, 0, 0, 5:8] = 0
    y = oq.values(*oq.quantize(row, "mx8"), "mx8", 32)[0, 0, 0, :5]
    assert list(y) == [448.0, 0.0, 2 * 2.0 ** -9, 16.0, 20.0]


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_zeros_limits_and_nan_blocks(fmt):
    x = np.zeros((1, 1, 4, 64), np.float32)
    x[0, 0, 1, 3] = np.inf
    x[0, 0, 2, 40] = np.nan
    x[0, 0, 3, 0] = np.finfo(np.float32).max
    x[0, 0, 3, 33] = np.finfo(np.float32).smallest_subnormal
    codes, scales = oq.quantize(x, fmt)
    y = oq.values(codes, scales, fmt, 64)
    assert (scales[0, 0, :, 0] == 0).all() and (y[0, 0, 0] == 0).all()
    assert np.isnan(y[0, 0, 1, :32]).all() and (y[0, 0, 1, 32:] == 0).all()
    assert (y[0, 0, 2, :32] == 0).all() and np.isnan(y[0, 0, 2, 32:]).all()
    assert scales[0, 0, 0, 1] == 255 and scales[0, 0, 1, 2] == 255
    assert abs(y[0, 0, 3, 0] / np.finfo(np.float32).max - 1) <= STEP[fmt]
    assert scales[0, 0, 1, 3] == 0 and y[0, 0, 3, 33] == 0


def test_attention_is_a_loop_over_tokens():
    g = np.random.default_rng(1)
    B, H, G, D, Dk = 2, 2, 3, 8, 3
    q = g.standard_normal((B, H * G, D))
    spans = [dict(k=g.standard_normal((1, H, 5, D)), v=g.standard_normal((1, H, 5, D))),
             dict(k=g.standard_normal((1, H, 4, Dk)), v=g.standard_normal((1, H, 4, D)),
                  R=g.standard_normal((1, H, D, Dk)), dm=g.standard_normal((1, H, D))),
             dict(k=g.standard_normal((B, H, 3, D)), v=g.standard_normal((B, H, 3, D)),
                  valid=np.array([[1, 0, 1], [0, 0, 0]]))]
    out, amean, size = oq.attend(q, G, spans)
    for b in range(B):
        for h in range(H * G):
            kv, num, den, top = h // G, np.zeros(D), 0.0, -np.inf
            toks = []
            for t in range(5):
                toks.append((q[b, h] @ spans[0]["k"][0, kv, t], spans[0]["v"][0, kv, t]))
            for t in range(4):
                s = spans[1]["k"][0, kv, t] @ (q[b, h] @ spans[1]["R"][0, kv]) + q[b, h] @ spans[1]["dm"][0, kv]
                toks.append((s, spans[1]["v"][0, kv, t]))
            for t in range(3):
                if spans[2]["valid"][b, t]:
                    toks.append((q[b, h] @ spans[2]["k"][b, kv, t], spans[2]["v"][b, kv, t]))
            top = max(s for s, _ in toks) / math.sqrt(D)
            for s, v in toks:
                w = math.exp(s / math.sqrt(D) - top)
                num, den = num + w * v, den + w
            assert np.allclose(out[b, h], num / (den + 1e-6), rtol=1e-12, atol=1e-13)
    assert (amean >= np.abs(out) - 1e-12).all() and size > 0


def test_nothing_to_attend_is_zero():
    q = np.ones((1, 1, 4))
    out, _, _ = oq.attend(q, 1, [dict(k=np.ones((1, 1, 2, 4)), v=np.ones((1, 1, 2, 4)), valid=np.zeros((1, 2)))])
    assert (out == 0).all()
