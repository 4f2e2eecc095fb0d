"""How exactly a rotation turns and rounds."""
import numpy as np
import pytest
import torch

from rotatek_amd.rotary import apply_rotary, inverse_frequencies
from tests.paged import DTYPES, f64, half

pytestmark = pytest.mark.gpu


def unit(N, P, dt):
    """Pairs (1, 0): they turn into the cosine and the sine."""
    x = torch.zeros(N, 1, 2 * P, dtype=dt, device="cuda")
    x[..., :P] = 1.0
    return x


@pytest.mark.parametrize("inverse", [False, True])
def test_sine_and_cosine_are_rounded_once(inverse):
    """fp32: each within half a step of the exact one, 2^-24 of it, and what 64-bit
    angles of 4 10^4 radians leave, 2^-36."""
    N, P = 4000, 64
    pos = torch.randint(0, 40000, (N,), generator=torch.Generator().manual_seed(0))
    freq = inverse_frequencies(2 * P)
    y, _ = apply_rotary(unit(N, P, torch.float32), None, pos.cuda(), freq, inverse=inverse)
    angle = pos.double().numpy()[:, None] * f64(freq)[None]
    for got, want in ((y[:, 0, :P], np.cos(angle)), (y[:, 0, P:], np.sin(angle) * (-1 if inverse else 1))):
        err, bound = np.abs(f64(got) - want), np.abs(want) * 2.0 ** -24 + 2.0 ** -36
        assert (err <= bound).all(), (int((err > bound).sum()), float((err / bound).max()))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_results_are_rounded_to_nearest(dtype):
    """A pair (1, 0) turned by angles of all kinds: half a step of the type, where
    cutting off would leave up to a whole one, and as often up as down."""
    dt, N, P = DTYPES[dtype], 2000, 32
    pos = torch.randint(0, 40000, (N,), generator=torch.Generator().manual_seed(1))
    freq = inverse_frequencies(2 * P)
    y, _ = apply_rotary(unit(N, P, dt), None, pos.cuda(), freq)
    angle = pos.double().numpy()[:, None] * f64(freq)[None]
    want, got = np.concatenate([np.cos(angle), np.sin(angle)], -1), f64(y[:, 0])
    # the sine and cosine behind it are rounded to fp32 first; fp16 steps end at 2^-24
    slack = 0.0 if dt == torch.float32 else 2.0 ** -23
    floor = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -36
    assert (np.abs(got - want) <= np.abs(want) * (half(dt) + slack) + floor).all()
    off = got - want
    up = np.abs(got) > np.abs(want)
    assert 0.45 < up[off != 0].mean() < 0.55        # of 10^5: cut off it would be none
