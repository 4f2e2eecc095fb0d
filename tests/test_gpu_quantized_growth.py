"""Rows of the quantised cache that move as it grows, with tokens that only the
device has counted."""
import numpy as np
import pytest
import torch

import spans as sp
from test_gpu_quantized_serving import _cache, _prefill, _q

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.mark.parametrize("fmt,dtype", [("mx8", torch.bfloat16), ("mx4", torch.float16)])
@pytest.mark.parametrize("how", ["reserve", "update", "replays"])
def test_growth_after_appends_of_the_device(fmt, dtype, how):
    """Tokens of ``append_`` (eager, or replayed) that the host has not counted are
    neither lost when the rows move nor in the way of those that follow."""
    _say(f"{how} {fmt} {dtype}")
    g = torch.Generator().manual_seed(41)
    B, H, G, D, s_p, s_v, s_t = 2, 2, 4, 128, 21, 70, 5
    x = _prefill(g, B, H, D, 32, s_p, s_v, s_t, dtype)
    cache = _cache(x, fmt, 7)
    k = np.concatenate([_q(x["prompt"], fmt), _q(x["text"], fmt)], 2)
    v = np.concatenate([_q(x["V"][:, :, :s_p], fmt), _q(x["V"][:, :, s_p + s_v:], fmt)], 2)
    vis = dict(k=_q(x["kp"], fmt), v=_q(x["V"][:, :, s_p:s_p + s_v], fmt), R=sp.np64(x["R"]), dm=sp.np64(x["dm"]))
    new = lambda T: [sp.randn(g, B, H, T, D, dtype=dtype).cuda() for _ in range(2)]  # noqa: E731

    def add(call, T=1):
        nonlocal k, v
        kn, vn = new(T)
        call(kn, vn)
        k, v = np.concatenate([k, _q(kn, fmt)], 2), np.concatenate([v, _q(vn, fmt)], 2)

    def check():
        q = sp.randn(g, B, H * G, D, dtype=dtype)
        sp.check(cache.decode_rotatek(q.cuda(), 0, G)[0], q, G, [vis, dict(k=k, v=v)], fmt, dtype)
        assert cache.lengths(0).tolist() == [k.shape[2]] * B

    if how == "replays":
        ks, vs = new(1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.append_(0, ks, vs)

        def step(kn, vn):
            ks.copy_(kn)
            vs.copy_(vn)
            graph.replay()
    else:
        step = lambda kn, vn: cache.append_(0, kn, vn)  # noqa: E731
    for _ in range(6):      # 6 of the 7 free rows
        add(step)
    check()
    if how == "replays":    # counted from the device, without growth
        cache.reserve(1)
        assert cache.get_seq_length() == s_v + k.shape[2]
        add(lambda kn, vn: cache.update(kn, vn, 0))
    elif how == "reserve":
        cache.reserve(30)
        check()
        for _ in range(30):
            add(step)
    else:
        add(lambda kn, vn: cache.update(kn, vn, 0), 9)
        add(lambda kn, vn: cache.update(kn, vn, 0))
        assert cache.get_seq_length() == s_v + k.shape[2]
    check()


@pytest.mark.parametrize("what", ["append", "decode"])
def test_rows_that_a_graph_holds_stay_where_they_are(what):
    """Growth under a captured graph is refused, nothing changed; with the graph
    released the rows move and a new capture works on them."""
    _say(f"held {what}")
    g = torch.Generator().manual_seed(42)
    B, H, G, D, dtype = 2, 2, 2, 128, torch.bfloat16
    x = _prefill(g, B, H, D, 32, 9, 40, 3, dtype)
    a, b = _cache(x, "mx8", 4), _cache(x, "mx8", 64)
    q, kn, vn = (sp.randn(g, *s, dtype=dtype).cuda() for s in ((B, H * G, D), (B, H, 1, D), (B, H, 1, D)))

    def capture():
        a.decode_rotatek(q, 0, G)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            if what == "append":
                a.append_(0, kn, vn)
            out = a.decode_rotatek(q, 0, G)[0]
        return graph, out

    def step(graph, out):
        kn.copy_(sp.randn(g, *kn.shape, dtype=dtype))
        vn.copy_(sp.randn(g, *vn.shape, dtype=dtype))
        if what == "decode":
            a.append_(0, kn, vn)
        graph.replay()
        b.update(kn, vn, 0)
        assert torch.equal(out, b.decode_rotatek(q, 0, G)[0])
        assert torch.equal(a.lengths(0), b.lengths(0))

    graph, out = capture()
    for _ in range(3):
        step(graph, out)
    codes = a.spans(0)[0].codes
    with pytest.raises(RuntimeError, match="graph"):
        a.reserve(2)
    with pytest.raises(RuntimeError, match="graph"):
        a.update(kn.expand(B, H, 2, D), vn.expand(B, H, 2, D), 0)
    assert a.spans(0)[0].codes.data_ptr() == codes.data_ptr()
    assert torch.equal(a.lengths(0), b.lengths(0))
    a.reserve(1)            # one row is free
    step(graph, out)
    del graph
    a.release_graphs()
    a.reserve(20)
    graph, out = capture()
    for _ in range(20):
        step(graph, out)


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_prefix_of_a_cache_with_room(fmt):
    """The shared spans of a cache that has free rows, NaN codes in them: prompt
    and text alone, as they grow."""
    from rotatek_amd.kernels import shared_prefix_decode
    _say(f"prefix {fmt}")
    g = torch.Generator().manual_seed(43)
    B, H, G, D, s_p, s_v, dtype = 6, 2, 4, 128, 30, 70, torch.bfloat16
    x = _prefill(g, 1, H, D, 32, s_p, s_v, 3, dtype)
    cache = _cache(x, fmt, 256)
    for rows in cache.spans(0)[:2]:
        rows.codes[:, :, s_p + 3:] = 0x7f
        rows.scales[..., s_p + 3:] = 255
    k = np.concatenate([_q(x["prompt"], fmt), _q(x["text"], fmt)], 2)
    v = np.concatenate([_q(x["V"][:, :, :s_p], fmt), _q(x["V"][:, :, s_p + s_v:], fmt)], 2)
    vis = dict(k=_q(x["kp"], fmt), v=_q(x["V"][:, :, s_p:s_p + s_v], fmt), R=sp.np64(x["R"]), dm=sp.np64(x["dm"]))
    q = sp.randn(g, B, H * G, D, dtype=dtype)
    for call in (None, lambda kn, vn: cache.update(kn, vn, 0), lambda kn, vn: cache.append_(0, kn, vn)):
        if call is not None:
            kn, vn = (sp.randn(g, 1, H, 5, D, dtype=dtype).cuda() for _ in range(2))
            call(kn, vn)
            k, v = np.concatenate([k, _q(kn, fmt)], 2), np.concatenate([v, _q(vn, fmt)], 2)
        kp, vp, ks, vs = cache.prefix(0)
        assert kp.shape == vp.shape == (1, H, k.shape[2], D)
        out = shared_prefix_decode(q.cuda(), kp, vp, None, None, G, R_partial=x["R"], delta_mu=x["dm"], k_sparse=ks,
                                   v_sparse=vs)
        sp.check(out, q, G, [vis, dict(k=k, v=v)], fmt, dtype)
    with pytest.raises(ValueError):
        _cache(_prefill(g, 2, H, D, 32, s_p, s_v, 3, dtype), fmt, 0).prefix(0)
    with pytest.raises(IndexError):
        cache.prefix(1)
