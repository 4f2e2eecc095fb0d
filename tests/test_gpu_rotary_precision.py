"""How exactly a rotation turns and rounds."""
import numpy as np
import pytest
import torch

from rotatek_amd.rotary import apply_rotary, inverse_frequencies
from tests.paged import f64

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
