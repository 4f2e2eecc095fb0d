"""Values that are not finite, at tokens that are seen: the formula's answer in
every kernel (oracle.paged.attend: an infinity times its weight)."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd.kernels import paged_decode, paged_prefill, window_attention
from tests.paged import DTYPES, Pool, attention_bound, f64

pytestmark = pytest.mark.gpu
HALF = ["bf16", "fp16"]
INF, NAN = float("inf"), float("nan")


def check_odd(got, want, amp, big, S, dt, single):
    """Where the formula is not finite, the same infinity or a NaN; elsewhere within its bound."""
    got, odd = f64(got), ~np.isfinite(want)
    np.testing.assert_array_equal(got[odd], want[odd])
    bound = attention_bound(np.where(odd, 0.0, want), np.where(odd, 0.0, amp), big, S, dt, single)
    off = np.abs(np.where(odd, 0.0, got) - np.where(odd, 0.0, want))
    assert (off <= bound)[~odd].all(), np.argwhere(~(off <= bound) & ~odd)[:4].tolist()


def starts_of(new):
    return torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("T, S, G, D", [(33, 100, 1, 64), (33, 33, 1, 80), (2, 1000, 1, 128), (9, 77, 32, 40), (65, 128, 1, 16)])
def test_window_with_an_odd_last_token(dtype, bad, T, S, G, D):
    """Rows of a wave that all stand at the last token, and others."""
    dt, g = DTYPES[dtype], torch.Generator().manual_seed(T + S)
    q, k, v = (torch.randn(1, h, n, D, generator=g).to(dt) for h, n in ((2 * G, T), (2, S), (2, S)))
    v[0, 1, S - 1, 5] = bad
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), G)
    want, amp, big = op.attend(f64(q[0]).swapaxes(0, 1), f64(k[0]), f64(v[0]), np.ones(S, bool), S - T, G)
    check_odd(got[0].transpose(0, 1), want, amp, big, S, dt, False)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("window, sinks", [(None, 0), (20, 2)])
def test_prefill_with_an_odd_last_token(dtype, bad, window, sinks):
    """A request of one new token among others: all its rows see the last one."""
    dt, lens, new, G = DTYPES[dtype], [50, 1, 90, 700], [1, 1, 40, 1], 3
    pool = Pool(lens, 2, 64, 16, dt, seed=3)
    for b, n in enumerate(lens):
        pool.v[int(pool.table[b, (n - 1) // 16]), 0, (n - 1) % 16, 9] = bad
    pool.cuda()
    q = torch.randn(sum(new), 2 * G, 64, device="cuda").to(dt)
    got = paged_prefill(q, starts_of(new), pool.dk, pool.dv, pool.dtable, pool.dlens, G, window, sinks)
    at = 0
    for b, n in enumerate(new):
        want, amp, big = pool.want(b, q[at:at + n].cpu(), G, window, sinks)
        check_odd(got[at:at + n], want, amp, big, 700, dt, False)
        at += n


@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("T, S, at", [(40, 300, 100), (40, 300, 259), (4, 900, 3)])
def test_window_with_an_odd_token_of_little_weight(bad, T, S, at):
    """A weight of 2^-50 is none in fp16; times an infinity it is one all the same."""
    dt, g = torch.float16, torch.Generator().manual_seed(S)
    q, k, v = (torch.randn(1, h, n, 64, generator=g).to(dt) for h, n in ((2, T), (1, S), (1, S)))
    q[..., 0], k[..., 0] = 16.0, 0.0
    k[0, 0, at, 0] = -20.0      # 16 * 20 / 8 log2(e) = 57.7 below the others
    v[0, 0, at, 5] = bad
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), 2)
    want, amp, big = op.attend(f64(q[0]).swapaxes(0, 1), f64(k[0]), f64(v[0]), np.ones(S, bool), S - T, 2)
    check_odd(got[0].transpose(0, 1), want, amp, big, S, dt, False)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("lens, H, G, D, page, per_more, window, sinks", [
    ([1, 2, 33, 700], 2, 7, 128, 16, 1, None, 0),       # a workgroup to a unit
    ([1, 40, 129], 1, 20, 80, 8, 1, None, 0),
    ([1, 300, 2500], 2, 3, 64, 64, 1, None, 0),         # shares and a join
    ([64, 2200], 1, 1, 128, 8, 1, 2100, 5),
    ([90, 500], 2, 4, 40, 16, 1, 30, 3),
])
def test_decode_with_odd_tokens(dtype, lens, H, G, D, page, per_more, window, sinks):
    """+inf, -inf, NaN and both infinities at tokens that are seen, each in a channel
    of its own, at the ends and in the middle; one that is not seen."""
    dt = DTYPES[dtype]
    pool = Pool(lens, H, D, page, dt, seed=D + G, per_more=per_more)

    def put(b, t, c, x):
        pool.v[int(pool.table[b, t // page]), H - 1, t % page, c] = x
    for b, n in enumerate(lens):
        put(b, n - 1, 0, INF)
        put(b, 0, 1, -INF)
        put(b, n // 2, 2, NAN)
        put(b, n - 1, 3, INF)
        put(b, max(n - 2, 0), 3, -INF)
        put(b, max(n - 20, 0), 4, -INF)
    pool.cuda()
    q = torch.randn(len(lens), H * G, D, device="cuda").to(dt)
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, G, window, sinks)
    for b in range(len(lens)):
        want, amp, big = pool.want(b, q[b:b + 1].cpu(), G, window, sinks)
        check_odd(got[b], want, amp, big, 4096, dt, True)


@pytest.mark.parametrize("dtype", HALF)
def test_single_row_with_odd_tokens(dtype):
    """window_attention of one new token, weights of 2^-50 among them."""
    dt, S, g = DTYPES[dtype], 200, torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, h, n, 64, generator=g).to(dt) for h, n in ((4, 1), (2, S), (2, S)))
    q[..., 0], k[..., 0] = 16.0, 0.0
    k[0, :, 50, 0] = -20.0
    v[0, 0, 50, 5], v[0, 1, S - 1, 6], v[0, 1, 50, 7] = INF, -INF, NAN
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), 2)
    want, amp, big = op.attend(f64(q[0]).swapaxes(0, 1), f64(k[0]), f64(v[0]), np.ones(S, bool), S - 1, 2)
    check_odd(got[0].transpose(0, 1), want, amp, big, S, dt, True)
