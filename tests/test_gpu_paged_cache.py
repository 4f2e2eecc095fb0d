"""PagedCache through a service's life: prompts of many lengths, tokens, requests
that leave and come, captured steps, streams."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd.kernels import paged_decode
from rotatek_amd.paged_cache import PagedCache
from rotatek_amd.rotary import inverse_frequencies
from tests.paged import attention_bound, check, f64

pytestmark = pytest.mark.gpu
H, G, D, SECTIONS = 2, 3, 64, (8, 12, 12)


class Model:
    """Projections of every token that a request has had, as the oracle keeps them."""

    def __init__(self, layers, requests, dtype):
        self.dtype, self.g = dtype, torch.Generator().manual_seed(0)
        self.k = [[np.zeros((0, H, D)) for _ in range(requests)] for _ in range(layers)]
        self.v = [[np.zeros((0, H, D)) for _ in range(requests)] for _ in range(layers)]
        self.freq = inverse_frequencies(D)

    def step(self, cache, layer, counts, window=None, sinks=0):
        N = sum(counts)
        q, k, v = (torch.randn(N, h, D, generator=self.g).to(self.dtype).cuda() for h in (H * G, H, H))
        pos = torch.randint(0, 20000, (3, N), generator=self.g).cuda()
        rq = cache.append(layer, k, v, pos, self.freq, SECTIONS, True, q)
        out = cache.attend(layer, rq, G, window, sinks)
        turned = op.rotate(f64(k), pos.cpu().numpy(), self.freq.cpu().numpy(), SECTIONS, True)
        at = 0
        for b, n in enumerate(counts):
            # as stored: rounded to the cache's type
            new = torch.from_numpy(turned[at:at + n]).to(self.dtype).double().numpy()
            self.k[layer][b] = np.concatenate([self.k[layer][b], new])
            self.v[layer][b] = np.concatenate([self.v[layer][b], f64(v[at:at + n])])
            if n:
                kk, vv = (x[layer][b].swapaxes(0, 1) for x in (self.k, self.v))
                m = kk.shape[1]
                want, amp, big = op.attend(f64(rq[at:at + n]), kk, vv, np.ones(m, bool), m - n, G, window, sinks)
                # a Key's rotation may round the other way: half a step more of each score
                bound = attention_bound(want, amp, big, m, self.dtype, False)
                bound = bound + amp * np.expm1(2 * big * torch.finfo(self.dtype).eps)
                check(out[at:at + n], want, bound)
            at += n

    def gone(self, b):
        for x in (self.k, self.v):
            for layer in x:
                layer[b] = np.zeros((0, H, D))


@pytest.mark.parametrize("window, sinks", [(None, 0), (20, 3)])
def test_a_service(window, sinks):
    cache = PagedCache(2, H, D, pages=40, page=8, requests=4, max_tokens=120, dtype=torch.bfloat16)
    m = Model(2, 4, torch.bfloat16)
    for counts in ([30, 7, 0, 1], [1, 1, 0, 1], [2, 0, 65, 1], [1, 1, 1, 1], [1, 1, 1, 1]):
        cache.begin(counts)
        for layer in range(2):
            m.step(cache, layer, counts, window, sinks)
    cache.free(2)
    m.gone(2)
    for counts in ([1, 1, 50, 1], [1, 1, 1, 1]):      # another request in the same pages
        cache.begin(counts)
        for layer in range(2):
            m.step(cache, layer, counts, window, sinks)


def test_captured_steps():
    """A step of every layer in a graph, replayed while lengths and pages grow;
    each replay against an eager run over a copy, with eager work between."""
    dt = torch.bfloat16
    cache = PagedCache(2, H, D, pages=64, page=8, requests=3, max_tokens=160, dtype=dt)
    freq = inverse_frequencies(D)
    q, k, v = (torch.randn(3, h, D, device="cuda").to(dt) for h in (H * G, H, H))
    pos = torch.zeros(3, 3, dtype=torch.int64, device="cuda")
    cache.begin([40, 1, 77])
    for layer in range(2):
        x = torch.randn(118, H, D, device="cuda").to(dt)
        cache.append(layer, x, x)

    def step(c):
        return [c.attend(i, c.append(i, k, v, pos, freq, SECTIONS, False, q), G, 50, 2) for i in range(2)]

    cache.begin([1, 1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cache)
    for i in range(20):
        cache.begin([1, 1, 1])
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda").to(dt))
        pos.fill_(i)
        held = [x.clone() for x in cache.k + cache.v]
        want = [o.clone() for o in step(cache)]
        grown = [x.clone() for x in cache.k + cache.v]
        for x, y in zip(cache.k + cache.v, held):
            x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(cache.k + cache.v, grown))


def test_two_streams_share_nothing():
    """Calls on two streams at once, each with a workspace of its own."""
    dt = torch.bfloat16
    caches = []
    for seed in range(2):
        c = PagedCache(1, H, D, pages=300, page=16, requests=2, max_tokens=2048, dtype=dt)
        torch.manual_seed(seed)
        c.begin([2000, 1500 + seed])
        x = torch.randn(3500 + seed, H, D, device="cuda").to(dt)
        c.append(0, x, x)
        caches.append(c)
    qs = [torch.randn(2, H * G, D, device="cuda").to(dt) for _ in range(2)]
    call = lambda i: paged_decode(qs[i], caches[i].k[0], caches[i].v[0], caches[i].table, caches[i].lens, G)  # noqa: E731
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(30):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(call(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements: its last pages are read and written."""
    dt, pages, page = torch.bfloat16, 16500, 64
    big = torch.empty(pages, 16, page, 128, dtype=dt, device="cuda")
    assert big.numel() > 2 ** 31
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(100, 16, 128, generator=g).to(dt).cuda()
    table = torch.tensor([[pages - 1, 3]], dtype=torch.int32, device="cuda")
    from rotatek_amd.paged import append_pages
    lens, starts = torch.tensor([100], dtype=torch.int32, device="cuda"), torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    append_pages(rows, rows, big, big, table, lens, starts)
    assert torch.equal(big[pages - 1].transpose(0, 1), rows[:64]) and torch.equal(big[3, :, :36].transpose(0, 1), rows[64:])
    q = torch.randn(1, 16, 128, generator=g).to(dt).cuda()
    k = f64(rows).swapaxes(0, 1)
    want, amp, bigs = op.attend(f64(q), k, k, np.ones(100, bool), 99, 1)
    check(paged_decode(q, big, big, table, lens, 1)[0], want, attention_bound(want, amp, bigs, 100, dt, True))
    from rotatek_amd.kernels import paged_prefill
    got = paged_prefill(q, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), big, big, table, lens, 1)
    check(got, want, attention_bound(want, amp, bigs, 100, dt, False))
