"""Seeded random calls with infinities and NaN among Keys and Values, seen and unseen."""
import random

import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd.kernels import paged_decode, paged_prefill, window_attention
from tests.paged import Pool, attention_bound, f64

pytestmark = pytest.mark.gpu


def pick(seed):
    r = random.Random(seed)
    c = dict(B=r.choice([1, 2, 3, 5]), H=r.choice([1, 2, 3]), G=r.choice([1, 2, 3, 7, 16, 33]), D=8 * r.randint(1, 16),
             page=r.choice([8, 16, 64]), dt=r.choice([torch.bfloat16, torch.float16]),
             window=r.choice([None, None, r.randint(1, 300)]))
    c["sinks"] = r.choice([0, 1, 4, r.randint(0, 100)]) if c["window"] else 0
    c["lens"] = [r.choice([1, r.randint(1, 40), r.randint(1, 700)]) for _ in range(c["B"])]
    return r, c


def odd(r):
    return r.choice([float("inf"), -float("inf"), float("nan")])


def check(q, k, v, there, first, c, got, single):
    """k, v [H, S, D] of one request, q and got [T, Hq, D].  A Key that is not finite
    makes weights 0 or NaN; how large scores are goes by the others.  Where all scores
    are -inf there are no weights, and the answer is that of seeing nothing, 0, or NaN
    in channels with a Value that is not finite."""
    want, amp, _ = op.attend(q, k, v, there, first, c["G"], c["window"], c["sinks"])
    j = np.arange(k.shape[1])
    for t in range(q.shape[0]):
        on = there & (j <= first + t)
        if c["window"] is not None:
            on &= (j > first + t - c["window"]) | (j < c["sinks"])
        for h in range(q.shape[1]):
            with np.errstate(invalid="ignore"):
                s = k[h // c["G"]][on] @ q[t, h]
            if on.any() and (s == -np.inf).all():
                want[t, h] = np.where(np.isfinite(v[h // c["G"]][on]).all(0), 0.0, np.nan)
                amp[t, h] = 0.0
    _, _, big = op.attend(q, np.where(np.isfinite(k), k, 0.0), np.zeros_like(v), there, first, c["G"], c["window"], c["sinks"])
    bad = ~np.isfinite(want)
    np.testing.assert_array_equal(got[bad], want[bad])
    bound = attention_bound(np.where(bad, 0.0, want), np.where(bad, 0.0, amp), big, k.shape[1], c["dt"], single)
    off = np.abs(np.where(bad, 0.0, got) - np.where(bad, 0.0, want))
    assert (off <= bound)[~bad].all()


@pytest.mark.parametrize("seed", range(300, 340))
def test_pages(seed):
    r, c = pick(seed)
    torch.manual_seed(seed)
    pool = Pool(c["lens"], c["H"], c["D"], c["page"], c["dt"], seed)
    for x, n in ((pool.v, r.randint(1, 5)), (pool.k, r.choice([0, 0, 1, 2]))):
        for _ in range(n):
            b = r.randrange(c["B"])
            t = r.choice([0, c["lens"][b] - 1, r.randrange(c["lens"][b])])
            x[int(pool.table[b, t // c["page"]]), r.randrange(c["H"]), t % c["page"], r.randrange(c["D"])] = odd(r)
    pool.cuda()

    def one(b, x, got, single):
        n = c["lens"][b]
        k, there = op.rows(f64(pool.k), pool.table.numpy(), b, n)
        v, _ = op.rows(f64(pool.v), pool.table.numpy(), b, n)
        check(f64(x), k, v, there, n - x.shape[0], c, f64(got), single)

    q = torch.randn(c["B"], c["H"] * c["G"], c["D"], device="cuda").to(c["dt"])
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, c["G"], c["window"], c["sinks"])
    for b in range(c["B"]):
        one(b, q[b:b + 1], got[b], True)
    new = [r.choice([1, min(n, 3), r.randint(1, min(n, 150))]) for n in c["lens"]]
    starts = [0] + list(np.cumsum(new))
    q = torch.randn(sum(new), c["H"] * c["G"], c["D"], device="cuda").to(c["dt"])
    got = paged_prefill(q, torch.tensor(starts, dtype=torch.int32, device="cuda"), pool.dk, pool.dv, pool.dtable, pool.dlens,
                        c["G"], c["window"], c["sinks"])
    for b in range(c["B"]):
        one(b, q[starts[b]:starts[b + 1]], got[starts[b]:starts[b + 1]], False)


@pytest.mark.parametrize("seed", range(400, 420))
def test_plain_rows(seed):
    r, c = pick(seed)
    torch.manual_seed(seed)
    S, T, B = r.randint(1, 500), r.choice([1, 2, 33, r.randint(1, 140)]), c["B"]
    q = torch.randn(B, c["H"] * c["G"], T, c["D"]).to(c["dt"])
    k, v = (torch.randn(B, c["H"], S, c["D"]).to(c["dt"]) for _ in range(2))
    for x, n in ((v, r.randint(1, 5)), (k, r.choice([0, 0, 1, 2]))):
        for _ in range(n):
            x[r.randrange(B), r.randrange(c["H"]), r.choice([0, S - 1, r.randrange(S)]), r.randrange(c["D"])] = odd(r)
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), c["G"], c["window"], c["sinks"])
    for b in range(B):
        check(f64(q[b]).swapaxes(0, 1), f64(k[b]), f64(v[b]), np.ones(S, bool), S - T, c, f64(got[b].transpose(0, 1)), T == 1)
