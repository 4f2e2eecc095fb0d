"""How exactly the weights of a softmax enter the products with Values."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd.kernels import window_attention
from tests.paged import DTYPES, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("below", [12, 15, 17, 18, 20, 24])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_small_weights_in_fp16(below, T):
    """One token of every 32 is 2^below above the others, and its Value is 0: the
    small weights answer for all of the output.

    The largest weight is at least 1 and weights are raised by 2^7, so one that is
    2^-b of the largest is at least 2^(7-b) where it is rounded to fp16: by half a
    step of 2^-11, in two terms (T = 1) 2^-22, or by 2^-25, whichever is more.  The
    largest is rounded too.  Scores: products are exact; the scale, the maximum and
    their difference are taken off by 2^-23 of `below` log2 each at most, and exp2 is
    good to 2^-22.  Sums of S positive numbers in fp32: S 2^-24.  The output is
    rounded once (2^-11, 2^-25 at least)."""
    dt, S, g = torch.float16, 700, torch.Generator().manual_seed(below)
    q, k = torch.zeros(1, 2, T, 64), torch.zeros(1, 1, S, 64)
    q[..., 0] = 8.0
    k[0, 0, ::32, 0] = below * float(np.log(2.0))      # q k / sqrt(64) = below ln 2
    v = (0.5 + torch.rand(1, 1, S, 64, generator=g)) * 2.0 ** (below - 9)
    v[0, 0, ::32] = 0.0
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), 2)
    want, _, _ = op.attend(f64(q[0]).swapaxes(0, 1), f64(k[0]), f64(v[0]), np.ones(S, bool), S - T, 2)
    term = 2.0 ** -22 if T == 1 else 2.0 ** -11
    rel = max(term, 2.0 ** (below - 32)) + term + 3 * below * 2.0 ** -23 + 2.0 ** -21 + S * 2.0 ** -24
    err = np.abs(f64(got[0].transpose(0, 1)) - want)
    bound = np.abs(want) * (rel + 2.0 ** -11 * (1 + rel)) + 2.0 ** -25
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("raised", [0.3, 1.2, 5.0, 7.1])
def test_equal_values_come_back(dtype, raised):
    """All Values alike: whatever the weights, the output is that Value, as what the
    Values are multiplied by is what is summed.  64 tokens first, against which
    the others' weights are 2^raised: no 16-bit number.  A sum of S tokens is off by
    S 2^-24 before it is rounded, far below half a step."""
    dt, S, T, H = DTYPES[dtype], 400, 256, 40       # (one part: the first tokens are everybody's)
    q, k = torch.zeros(1, H, T, 64), torch.zeros(1, H, S, 64)
    q[..., 0] = 8.0
    k[0, :, 64:, 0] = raised * float(np.log(2.0))
    v = (2.0 - torch.finfo(dt).eps * torch.arange(1, 65)).expand(1, H, S, 64).contiguous()
    got = window_attention(q.to(dt).cuda(), k.to(dt).cuda(), v.to(dt).cuda(), 1)
    assert torch.equal(got.cpu(), v[:, :, :1].to(dt).expand(1, H, T, 64))
