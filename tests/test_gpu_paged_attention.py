"""paged_decode, paged_prefill and window_attention against the oracle in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd.kernels import paged_decode, paged_prefill, window_attention
from tests.paged import DTYPES, Pool, attention_bound, check, f64

pytestmark = pytest.mark.gpu
HALF = ["bf16", "fp16"]


def starts_of(new):
    return torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ decode
def decode_check(pool, q, groups, window, sinks, got, dt, lens=None):
    for b in range(q.shape[0]):
        want, amp, big = pool.want(b, q[b:b + 1].cpu(), groups, window, sinks, None if lens is None else lens[b])
        check(got[b], want, attention_bound(want, amp, big, 4096, dt, True))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("lens, H, G, D, page, window, sinks, strided", [
    ([1, 0, 33, 700], 2, 7, 128, 16, None, 0, False),
    ([31, 32, 33, 127, 128, 129], 1, 1, 64, 8, None, 0, True),
    ([2000, 5], 2, 4, 128, 64, 100, 4, False),
    ([300, 299, 1, 64], 1, 16, 96, 32, 1, 0, False),     # the new token alone
    ([300, 90, 40], 2, 3, 80, 8, 50, 37, True),          # sinks end inside a block, or past the text
    ([513, 20], 1, 20, 40, 16, 64, 1, False),            # more heads than a unit has rows
    ([9, 600], 1, 2, 8, 128, 33, 500, False),            # sinks reach the window
    ([64] * 70, 1, 1, 128, 64, None, 0, False),          # more requests than a wave has lanes
])
def test_decode(dtype, lens, H, G, D, page, window, sinks, strided):
    dt = DTYPES[dtype]
    pool = Pool(lens, H, D, page, dt, seed=D + G, strided=strided).cuda()
    q = torch.randn(len(lens), H * G, D, device="cuda").to(dt)
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, G, window, sinks)
    assert got.shape == (len(lens), 1, H * G, D) and got.dtype == dt
    decode_check(pool, q, G, window, sinks, got, dt)


def test_decode_of_many_requests():
    """More requests than a workgroup has threads; most of them empty."""
    dt, g = torch.bfloat16, np.random.default_rng(0)
    lens = [int(n) for n in g.choice([0, 0, 0, 1, 40, 300], 600)]
    pool = Pool(lens, 1, 64, 16, dt).cuda()
    q = torch.randn(600, 2, 64, device="cuda").to(dt)
    decode_check(pool, q, 2, None, 0, paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, 2), dt)


@pytest.mark.parametrize("dtype", HALF)
def test_decode_layouts(dtype):
    """Queries and outputs of any strides, a table with more room than is used."""
    dt = DTYPES[dtype]
    pool = Pool([50, 260], 2, 80, 16, dt, per_more=9).cuda()
    q = torch.randn(80, 2, 8, device="cuda").to(dt).permute(1, 2, 0)
    out = torch.full((2, 8, 161), 3.0, dtype=dt, device="cuda")
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, 4, out=out[..., 1::2])
    assert got.data_ptr() == out.data_ptr() + out.element_size()
    decode_check(pool, q, 4, None, 0, out[..., 1::2].unsqueeze(1), dt)
    assert (out[..., ::2] == 3).all()
    # a table that is a view of a wider one
    wide = torch.full((2, pool.table.shape[1] + 5), 77777, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + pool.table.shape[1]] = pool.dtable
    again = paged_decode(q, pool.dk, pool.dv, wide[:, 2:2 + pool.table.shape[1]], pool.dlens, 4)
    assert torch.equal(again, got)


@pytest.mark.parametrize("window, sinks", [(None, 0), (40, 12)])
def test_pages_that_are_none_count_for_nothing(window, sinks):
    dt = torch.bfloat16
    pool = Pool([200, 64, 128], 2, 64, 16, dt, per_more=0).cuda()
    pool.table[0, 0], pool.table[0, 5], pool.table[0, 11], pool.table[1, :] = -1, 2 ** 31 - 1, -2 ** 31, 10 ** 6
    pool.dtable.copy_(pool.table)
    lens = [200, 64, 1000]      # the last one past its table
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 6, 64, device="cuda").to(dt)
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, dl, 3, window, sinks)
    decode_check(pool, q, 3, window, sinks, got, dt, lens)
    assert (got[1] == 0).all()
    dl.copy_(torch.tensor([-3, -2 ** 31, 0]))
    assert (paged_decode(q, pool.dk, pool.dv, pool.dtable, dl, 3, window, sinks) == 0).all()
    new = [3, 1, 5]
    dl.copy_(torch.tensor(lens))
    q = torch.randn(9, 6, 64, device="cuda").to(dt)
    got = paged_prefill(q, starts_of(new), pool.dk, pool.dv, pool.dtable, dl, 3, window, sinks)
    prefill_check(pool, q, new, 3, window, sinks, got, dt, lens)


def test_scores_of_any_size():
    """All scores near the lowest a type holds, and far above each other."""
    dt = torch.bfloat16
    pool = Pool([100, 100], 1, 64, 16, dt).cuda()
    pool.dk[..., 0] = -3e38
    q = torch.zeros(2, 1, 64, device="cuda").to(dt)
    q[0, 0, 0] = 1.0
    q[1, 0, 1] = 300.0
    pool.k = pool.dk.cpu()
    got = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, 1)
    want, amp, _ = pool.want(0, q[:1].cpu(), 1, None, 0)     # equal scores: no rounding tells them apart
    check(got[0], want, attention_bound(want, amp, 0.0, 100, dt, True))
    assert torch.isfinite(got).all()
    q3 = q[:1].expand(40, 1, 64).contiguous()
    got = paged_prefill(q3, starts_of([40, 0]), pool.dk, pool.dv, pool.dtable, pool.dlens, 1)
    want, amp, _ = pool.want(0, q3.cpu(), 1, None, 0)
    check(got, want, attention_bound(want, amp, 0.0, 100, dt, False))


# ------------------------------------------------------------------ window
def prefill_check(pool, q, new, groups, window, sinks, got, dt, lens=None):
    at = 0
    for b, n in enumerate(new):
        if n:
            x = q[at:at + n]
            want, amp, big = pool.want(b, x.cpu(), groups, window, sinks, None if lens is None else lens[b])
            check(got[at:at + n], want, attention_bound(want, amp, big, 4096, dt, False))
        at += n


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("lens, new, H, G, D, page, window, sinks", [
    ([40, 7, 100], [40, 7, 1], 2, 4, 128, 16, None, 0),
    ([200, 0, 65, 300], [3, 0, 65, 129], 1, 7, 64, 8, None, 0),
    ([700, 128], [130, 128], 1, 1, 128, 64, 70, 5),
    ([400, 300, 20], [257, 1, 20], 2, 3, 80, 32, 1, 0),
    ([90, 333], [64, 33], 1, 16, 96, 16, 65, 40),
    ([256, 90], [17, 90], 1, 40, 40, 8, 33, 100),
    ([600], [5], 1, 2, 8, 16, None, 0),         # few rows: the tokens are cut
    ([3, 2], [5, 2], 1, 2, 32, 8, None, 0),     # more queries than tokens: the first see nothing
])
def test_prefill(dtype, lens, new, H, G, D, page, window, sinks):
    dt = DTYPES[dtype]
    pool = Pool(lens, H, D, page, dt, seed=D + G).cuda()
    q = torch.randn(sum(new), H * G, D, device="cuda").to(dt)
    got = paged_prefill(q, starts_of(new), pool.dk, pool.dv, pool.dtable, pool.dlens, G, window, sinks)
    assert got.shape == q.shape and got.dtype == dt
    prefill_check(pool, q, new, G, window, sinks, got, dt)


@pytest.mark.parametrize("new, H, D", [
    ([300, 0, 130, 5, 260], 40, 16),                    # 360 workgroups: two a CU, tiles of all requests in turn
    ([300, 0, 130, 5, 260, 0], 64, 16),                 # 576: three
    ([int(n) for n in (np.arange(70) * 37) % 140], 4, 8),  # more requests than a wave has lanes
    ([0, 0, 1, 0] * 16, 20, 80),                        # one token each, the others none
])
def test_prefill_of_one_round(new, H, D):
    dt, lens = torch.bfloat16, [n + 9 * (i % 3) for i, n in enumerate(new)]
    pool = Pool(lens, H, D, 16, dt, seed=H).cuda()
    q = torch.randn(sum(new), H, D, device="cuda").to(dt)
    got = paged_prefill(q, starts_of(new), pool.dk, pool.dv, pool.dtable, pool.dlens, 1, 200, 3)
    prefill_check(pool, q, new, 1, 200, 3, got, dt)


@pytest.mark.parametrize("B, H, T, D", [(3, 40, 300, 16), (2, 24, 700, 72)])
def test_window_of_one_round(B, H, T, D):
    dt, g = torch.float16, torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(B, H, T, D, generator=g).to(dt) for _ in range(3))
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), 1)
    for b in range(B):
        want, amp, big = op.attend(f64(q[b]).swapaxes(0, 1), f64(k[b]), f64(v[b]), np.ones(T, bool), 0, 1, None, 0)
        check(got[b].transpose(0, 1), want, attention_bound(want, amp, big, T, dt, False))


@pytest.mark.parametrize("splits", [False, True])
def test_rows_of_no_request_stay(splits):
    dt, lens = torch.float16, [600, 90]
    pool = Pool(lens, 1, 64, 16, dt).cuda()
    reps = 1 if splits else 40
    q = torch.randn(10 * reps, 2 * reps, 64, device="cuda").to(dt)
    pool.dk, pool.dv = pool.dk.expand(-1, reps, -1, -1).contiguous(), pool.dv.expand(-1, reps, -1, -1).contiguous()
    starts = torch.tensor([2, 5, 9], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    paged_prefill(q, starts, pool.dk, pool.dv, pool.dtable, pool.dlens, 2, out=out)
    assert (out[:2] == 7).all() and (out[9:] == 7).all()
    for b, (s, e) in enumerate(((2, 5), (5, 9))):
        for h in range(0, 2 * reps, 16):
            want, amp, big = pool.want(b, q[s:e, h:h + 2].cpu(), 2, None, 0)
            check(out[s:e, h:h + 2], want, attention_bound(want, amp, big, 1024, dt, False))


def test_starts_past_the_queries():
    """Ranges that do not ascend or pass the queries: nothing outside is touched."""
    dt = torch.bfloat16
    pool = Pool([64, 64], 1, 64, 16, dt).cuda()
    q = torch.randn(4, 2, 64, device="cuda").to(dt)
    for bad in ([0, 4, 900], [-3, 2, 4], [3, 1, 4], [2 ** 31 - 1, 0, -2 ** 31]):
        out = torch.full((6, 2, 64), 7.0, dtype=dt, device="cuda")
        paged_prefill(q, torch.tensor(bad, dtype=torch.int32, device="cuda"), pool.dk, pool.dv, pool.dtable, pool.dlens, 2,
                      out=out[1:5])
        assert (out[0] == 7).all() and (out[5] == 7).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("B, H, G, T, S, D, window, sinks, lens", [
    (2, 2, 4, 5, 77, 128, None, 0, None),
    (1, 1, 2, 300, 300, 64, 65, 3, None),
    (3, 1, 7, 1, 500, 128, 100, 4, [500, 0, 33]),        # a single token
    (2, 1, 3, 9, 4, 80, None, 0, None),                  # more queries than tokens
    (2, 1, 1, 200, 200, 40, 33, 0, [200, 120]),          # a padded batch
    (2, 2, 1, 64, 700, 96, 1, 1, None),
    (1, 8, 4, 2, 3000, 128, None, 0, None),              # few rows, many tokens
])
def test_window(dtype, B, H, G, T, S, D, window, sinks, lens):
    dt, g = DTYPES[dtype], torch.Generator().manual_seed(T + S)
    q, k, v = (torch.randn(B, h, n, D, generator=g).to(dt) for h, n in ((H * G, T), (H, S), (H, S)))
    dl = None
    if lens:
        dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):
            k[b, :, n:], v[b, :, n:] = float("nan"), float("inf")
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), G, window, sinks, dl)
    for b in range(B):
        n = lens[b] if lens else S
        want, amp, big = op.attend(f64(q[b]).swapaxes(0, 1), f64(k[b, :, :n]), f64(v[b, :, :n]), np.ones(n, bool), n - T, G,
                                   window, sinks)
        check(got[b].transpose(0, 1), want, attention_bound(want, amp, big, S, dt, T == 1))


def test_window_layouts():
    """Slices of one projection [B, T, heads, D], an output of other strides."""
    dt, B, T, H, G, D = torch.bfloat16, 2, 90, 2, 3, 64
    x = torch.randn(B, T, H * (G + 2), D, device="cuda").to(dt)
    q, k, v = (y.transpose(1, 2) for y in x.split([H * G, H, H], 2))
    want = window_attention(q.contiguous(), k.contiguous(), v.contiguous(), G, 20, 2)
    assert torch.equal(window_attention(q, k, v, G, 20, 2), want)
    out = torch.zeros(B, T, H * G, D, device="cuda", dtype=dt).transpose(1, 2)
    assert torch.equal(window_attention(q, k, v, G, 20, 2, out=out), want) and torch.equal(out, want)
    odd = torch.zeros(B, H * G, D, T, device="cuda", dtype=dt).transpose(2, 3)
    assert torch.equal(window_attention(q, k, v, G, 20, 2, out=odd), want)
    away = q.transpose(2, 3).contiguous().transpose(2, 3)     # channels far apart
    assert torch.equal(window_attention(away, k, v, G, 20, 2), want)
    with pytest.raises(ValueError):
        window_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, G)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("T, S, window, sinks, at", [(200, 200, None, 0, 150), (200, 200, 40, 3, 20), (4, 900, None, 0, 898)])
@pytest.mark.parametrize("D", [64, 80, 40])
def test_what_is_not_seen_does_not_matter(bad, where, T, S, window, sinks, at, D):
    """One odd value at a token: queries that do not see it are as without it, the
    others as the formula says (a NaN there is a NaN here)."""
    dt, g = torch.bfloat16, torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(1, h, n, D, generator=g).to(dt) for h, n in ((4, T), (2, S), (2, S)))
    if where == "k":
        q[..., 7] = q[..., 7].abs() + 0.5       # inf times it keeps its sign
    clean = window_attention(q.cuda(), k.cuda(), v.cuda(), 2, window, sinks).cpu()
    (k if where == "k" else v)[0, 1, at, 7] = bad
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), 2, window, sinks).cpu()
    p = torch.arange(S - T, S)
    sees = (p >= at) & ((p - at < window) | (at < sinks) if window else True)
    assert sees.any() and not sees.all()
    assert torch.equal(got[:, :2], clean[:, :2])
    same = [7] if where == "v" else []
    rest = [c for c in range(D) if c not in same]
    blind = got[0, 2:, ~sees]
    # summed in another order where a neighbour is not finite
    torch.testing.assert_close(blind.float(), clean[0, 2:, ~sees].float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    assert torch.isfinite(blind).all()
    if where == "v":
        torch.testing.assert_close(got[0, 2:, sees][..., rest].float(), clean[0, 2:, sees][..., rest].float(), rtol=2.0 ** -6,
                                   atol=2.0 ** -6)
        seen = got[0, 2:, sees][..., 7].float()
        assert torch.isnan(seen).all() if bad != bad else (seen == bad).all()
    elif bad == -float("inf"):
        assert torch.isfinite(got).all()        # its weight is zero
    else:
        assert torch.isnan(got[0, 2:, sees]).all()


@pytest.mark.parametrize("dtype", HALF)
def test_values_that_are_not_finite(dtype):
    """Rows ahead of the text see nothing, whatever token 0 holds; all NaN gives NaN;
    an infinity that all rows see stays in its channel."""
    dt, g = DTYPES[dtype], torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(1, h, n, 64, generator=g).to(dt) for h, n in ((2, 300), (1, 270), (1, 270)))
    clean = window_attention(q.cuda(), k.cuda(), v.cuda(), 2).cpu()
    v[0, 0, 0, 3] = float("inf")
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), 2).cpu()
    assert (got[:, :, :30] == 0).all() and (got[:, :, 30:, 3] == float("inf")).all()
    got[..., 3] = clean[..., 3]
    # (in a wave whose rows do not all see it, sums are formed in another order)
    torch.testing.assert_close(got.float(), clean.float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    assert torch.equal(got[:, :, 96:], clean[:, :, 96:])
    v[:] = float("nan")
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), 2).cpu()
    assert (got[:, :, :30] == 0).all() and torch.isnan(got[:, :, 30:]).all()


@pytest.mark.parametrize("per, window", [(2, None), (40, None), (40, 70)])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 1, 30]])
def test_captured_calls(per, window, new):
    """Every form in a graph (a launch or two, tokens cut or not), replayed with other
    lengths, queries and pages, against the eager call, with eager work between."""
    dt, page, H, G, D = torch.float16, 16, 2, 3, 64
    torch.manual_seed(7)
    k, v = (torch.randn(3 * per + 2, H, page, D, device="cuda").to(dt) for _ in range(2))
    table = torch.randperm(3 * per + 2, device="cuda")[:3 * per].to(torch.int32).view(3, per)
    lens = torch.full((3,), 30, dtype=torch.int32, device="cuda")
    q, starts = torch.randn(sum(new), H * G, D, device="cuda").to(dt), starts_of(new)

    def call():
        if max(new) == 1:
            return paged_decode(q, k, v, table, lens, G, window, 3)[:, 0]
        return paged_prefill(q, starts, k, v, table, lens, G, window, 3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(12):
        lens.copy_(torch.randint(0, per * page + 3, (3,)))
        q.copy_(torch.randn(q.shape, device="cuda").to(dt))
        table.copy_(torch.randperm(3 * per + 2, device="cuda")[:3 * per].to(torch.int32).view(3, per))
        want = call().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_decode_is_its_prefill():
    """The same tokens through both: within both's bounds of each other."""
    dt, lens = torch.bfloat16, [1, 77, 640]
    pool = Pool(lens, 2, 128, 16, dt).cuda()
    q = torch.randn(3, 8, 128, device="cuda").to(dt)
    a = paged_decode(q, pool.dk, pool.dv, pool.dtable, pool.dlens, 4, 200, 4)[:, 0]
    b = paged_prefill(q, starts_of([1, 1, 1]), pool.dk, pool.dv, pool.dtable, pool.dlens, 4, 200, 4)
    for i in range(3):
        want, amp, big = pool.want(i, q[i:i + 1].cpu(), 4, 200, 4)
        bound = attention_bound(want, amp, big, 640, dt, False)
        check(a[i:i + 1], want, bound)
        check(b[i:i + 1], want, bound)


def test_empty_calls():
    k = torch.zeros(3, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    t, n = torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    assert paged_decode(k.new_zeros(0, 4, 64), k, k, t, n, 2).shape == (0, 1, 4, 64)
    t, n = torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.full((2,), 9, dtype=torch.int32, device="cuda")
    assert (paged_decode(k.new_ones(2, 4, 64), k, k, t, n, 2) == 0).all()
    assert (paged_decode(k.new_ones(2, 4, 64), k[:0], k[:0], torch.zeros(2, 3, dtype=torch.int32, device="cuda"), n, 2) == 0).all()
    assert paged_prefill(k.new_zeros(0, 4, 64), starts_of([0, 0]), k, k, t, n, 2).shape == (0, 4, 64)
    assert (paged_prefill(k.new_ones(2, 4, 64), starts_of([1, 1]), k, k, t, n, 2) == 0).all()
    e = k.new_zeros(2, 2, 0, 64)
    assert (window_attention(k.new_ones(2, 4, 3, 64), e, e, 2) == 0).all()
    assert window_attention(k.new_ones(2, 4, 0, 64), k[:2], k[:2], 2).shape == (2, 4, 0, 64)


def test_gradients_are_refused():
    x = torch.randn(1, 2, 8, 64, device="cuda").bfloat16().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        window_attention(x, x.detach(), x.detach())
    with torch.no_grad():
        window_attention(x, x, x)
