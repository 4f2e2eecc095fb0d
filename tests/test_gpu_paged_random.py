"""Seeded random calls of the paged cache's operators against the oracle."""
import random

import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd.kernels import paged_decode, paged_prefill, window_attention
from rotatek_amd.paged import append_pages
from rotatek_amd.rotary import inverse_frequencies
from tests.paged import Pool, attention_bound, check, f64, rotation_bound

pytestmark = pytest.mark.gpu


def pick(seed):
    r = random.Random(seed)
    c = dict(B=r.choice([1, 2, 3, 5, 9]), H=r.choice([1, 2, 3]), G=r.choice([1, 2, 3, 4, 7, 8, 16, 17, 33]),
             D=8 * r.randint(1, 16), page=r.choice([8, 16, 32, 64, 128]), dt=r.choice([torch.bfloat16, torch.float16]),
             window=r.choice([None, None, r.randint(1, 400)]), strided=r.random() < 0.3)
    c["sinks"] = r.choice([0, 1, 4, r.randint(0, 200)]) if c["window"] else 0
    c["lens"] = [r.choice([0, 1, r.randint(0, 40), r.randint(0, 700)]) for _ in range(c["B"])]
    return r, c


@pytest.mark.parametrize("seed", range(24))
def test_decode_and_prefill(seed):
    r, c = pick(seed)
    pool = Pool(c["lens"], c["H"], c["D"], c["page"], c["dt"], seed, strided=c["strided"]).cuda()
    q = torch.randn(c["B"], c["H"] * c["G"], c["D"], device="cuda").to(c["dt"])
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, c["G"], c["window"], c["sinks"])
    for b in range(c["B"]):
        want, amp, big = pool.want(b, q[b:b + 1].cpu(), c["G"], c["window"], c["sinks"])
        check(got[b], want, attention_bound(want, amp, big, 1024, c["dt"], True))
    # new tokens up to all that a request holds, and sometimes more
    new = [r.choice([0, 1, min(n, 3), r.randint(0, min(n, 150) + 2)]) for n in c["lens"]]
    starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    q = torch.randn(sum(new), c["H"] * c["G"], c["D"], device="cuda").to(c["dt"])
    got = paged_prefill(q, starts, pool.dk, pool.dv, pool.dtable, pool.dlens, c["G"], c["window"], c["sinks"])
    at = 0
    for b, n in enumerate(new):
        if n:
            want, amp, big = pool.want(b, q[at:at + n].cpu(), c["G"], c["window"], c["sinks"])
            check(got[at:at + n], want, attention_bound(want, amp, big, 1024, c["dt"], False))
        at += n


@pytest.mark.parametrize("seed", range(100, 116))
def test_plain_rows(seed):
    r, c = pick(seed)
    S, T, B = r.randint(1, 500), r.choice([1, 2, r.randint(1, 140)]), c["B"]
    q = torch.randn(B, c["H"] * c["G"], T, c["D"]).to(c["dt"])
    k, v = (torch.randn(B, S, c["H"], c["D"]).to(c["dt"]).transpose(1, 2) for _ in range(2))
    lens = [r.randint(0, S) for _ in range(B)]
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), c["G"], c["window"], c["sinks"],
                           torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for b, n in enumerate(lens):
        want, amp, big = op.attend(f64(q[b]).swapaxes(0, 1), f64(k[b, :, :n]), f64(v[b, :, :n]), np.ones(n, bool), n - T, c["G"],
                                   c["window"], c["sinks"])
        check(got[b].transpose(0, 1), want, attention_bound(want, amp, big, S, c["dt"], T == 1))


@pytest.mark.parametrize("seed", range(200, 216))
def test_append(seed):
    r, c = pick(seed)
    dt = r.choice([torch.bfloat16, torch.float16, torch.float32])
    pool = Pool(c["lens"], c["H"], c["D"], c["page"], dt, seed, strided=c["strided"], fill=0.5).cuda()
    new = [r.choice([0, min(n, 1), r.randint(0, n)]) for n in c["lens"]]
    N, P = sum(new), r.randint(1, c["D"] // 2)
    starts = [0] + list(np.cumsum(new))
    sections = [r.randint(0, P) for _ in range(r.randint(0, 3))]
    while sum(sections) > P:
        sections.pop()
    sections.append(P - sum(sections))
    interleaved = r.random() < 0.5
    q, k, v = (torch.randn(N, h, c["D"], device="cuda").to(dt) for h in (c["H"] * c["G"], c["H"], c["H"]))
    pos = torch.randint(-50, 100000, (len(sections), N), device="cuda")
    freq = inverse_frequencies(2 * P)
    k0, v0 = f64(pool.dk), f64(pool.dv)
    out = append_pages(k, v, pool.dk, pool.dv, pool.dtable, pool.dlens, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                       pos, freq, sections, interleaved, q)
    p, f = pos.cpu().numpy(), freq.cpu().numpy()
    want = op.rotate(f64(q), p, f, sections, interleaved)
    check(out, want, rotation_bound(f64(q), want, P, dt))
    turned = op.rotate(f64(k), p, f, sections, interleaved)
    bound = rotation_bound(f64(k), turned, P, dt)
    table, zero = pool.table.numpy(), np.zeros_like(k0)
    want_k, want_v = op.append(turned, f64(v), k0, v0, table, c["lens"], starts)
    check(pool.dk, want_k, op.append(bound, bound, zero, zero, table, c["lens"], starts)[0])
    np.testing.assert_array_equal(f64(pool.dv), want_v)


def test_many_requests():
    """More requests than a wave has lanes, and than a workgroup has threads."""
    dt = torch.bfloat16
    for B in (70, 300):
        r = random.Random(B)
        lens = [r.choice([0, 3, 20, 90]) for _ in range(B)]
        new = [min(n, r.choice([0, 1, 5])) for n in lens]
        pool = Pool(lens, 1, 64, 16, dt, B).cuda()
        starts = [0] + list(np.cumsum(new))
        q = torch.randn(sum(new), 2, 64, device="cuda").to(dt)
        ds = torch.tensor(starts, dtype=torch.int32, device="cuda")
        got = paged_prefill(q, ds, pool.dk, pool.dv, pool.dtable, pool.dlens, 2, 30, 2)
        for b in range(B):
            x = q[starts[b]:starts[b + 1]]
            if len(x):
                want, amp, big = pool.want(b, x.cpu(), 2, 30, 2)
                check(got[starts[b]:starts[b + 1]], want, attention_bound(want, amp, big, 90, dt, False))
        k = torch.randn(sum(new), 1, 64, device="cuda").to(dt)
        k0 = f64(pool.dk)
        append_pages(k, k, pool.dk, pool.dv, pool.dtable, pool.dlens, ds)
        want, _ = op.append(f64(k), f64(k), k0, k0, pool.table.numpy(), lens, starts)
        np.testing.assert_array_equal(f64(pool.dk), want)
