"""Decodes whose work is shared out evenly among the workgroups: shares of several
pieces, that begin and end inside units and reach over units and requests, units
of few and of many shares, more requests than a wave has lanes."""
import random

import pytest
import torch

from rotatek_amd.kernels import paged_decode
from tests.paged import DTYPES, Pool, attention_bound, check

pytestmark = pytest.mark.gpu


def pieces(lens, H, G):
    return sum(-(-n // 128) for n in lens) * H * -(-G // 16)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens, H, G, D, page, window, sinks", [
    ([3000, 2999, 1, 0, 1500, 2900], 8, 2, 128, 64, None, 0),       # a share: one piece or two
    ([9000, 3, 8999, 6000, 129, 9001], 4, 3, 128, 128, None, 0),    # four or so, of units of 14 shares
    ([2500] * 20, 7, 1, 64, 16, None, 0),                           # 17 units of one length to 100 shares
    ([2100, 5000, 1, 3000, 40, 128, 2048, 4999] * 2, 8, 2, 128, 32, None, 0),   # short shares' records, joined by single waves
    ([5000, 90, 4000, 3500, 2900] * 3, 6, 18, 64, 8, 3000, 70),     # pages of eight rows, two blocks of heads, a window
])
def test_shares(dtype, lens, H, G, D, page, window, sinks):
    dt, cus = DTYPES[dtype], torch.cuda.get_device_properties(0).multi_processor_count
    workers = (3 if D <= 64 else 2) * cus
    seen = [min(n, (window or n) + sinks) for n in lens]
    assert pieces(seen, H, G) > workers and max(-(-n // 128) for n in lens) > 16
    pool = Pool(lens, H, D, page, dt, seed=D + G).cuda()
    q = torch.randn(len(lens), H * G, D, device="cuda").to(dt)
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, G, window, sinks)
    for b in range(len(lens)):
        want, amp, big = pool.want(b, q[b:b + 1].cpu(), G, window, sinks)
        check(got[b], want, attention_bound(want, amp, big, 4096, dt, True))
    assert torch.equal(got, paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, G, window, sinks))


@pytest.mark.parametrize("B, H, G, D, page", [(70, 5, 2, 128, 16), (300, 2, 4, 64, 8), (65, 5, 1, 128, 64)])
def test_shares_of_many_requests(B, H, G, D, page):
    """Pieces found by the whole workgroup; many requests are empty."""
    dt, r = torch.bfloat16, random.Random(B)
    lens = [r.choice([0, 1, 127, 128, 129, r.randint(200, 1200)]) for _ in range(B)]
    lens[r.randrange(B)] = 2100
    lens[0], lens[-1] = 0, 900
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert pieces(lens, H, G) > (3 if D <= 64 else 2) * cus
    pool = Pool(lens, H, D, page, dt, seed=B).cuda()
    q = torch.randn(B, H * G, D, device="cuda").to(dt)
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, G)
    for b in range(B):
        want, amp, big = pool.want(b, q[b:b + 1].cpu(), G, None, 0)
        check(got[b], want, attention_bound(want, amp, big, 4096, dt, True))


def test_captured_shares_follow_the_lengths():
    """The plan is the table's; a replay's shares are the lengths'."""
    dt, B, H, G, D, page, per = torch.float16, 6, 4, 4, 128, 64, 80
    torch.manual_seed(3)
    k, v = (torch.randn(B * per, H, page, D, device="cuda").to(dt) for _ in range(2))
    table = torch.randperm(B * per, device="cuda").to(torch.int32).view(B, per)
    lens = torch.full((B,), 100, dtype=torch.int32, device="cuda")
    q = torch.randn(B, H * G, D, device="cuda").to(dt)
    call = lambda: paged_decode(q, k, v, table, lens, G)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i, n in enumerate((0, 1, 100, 3000, per * page, 1500)):
        lens.copy_(torch.tensor([max(0, n - 37 * b * (b % 3)) for b in range(B)]))
        q.copy_(torch.randn(q.shape, device="cuda").to(dt))
        want = call().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.isfinite(out).all()
