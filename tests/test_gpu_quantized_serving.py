"""The quantised cache and the shared prefix as a server uses them: prefill,
growing text, captured steps, several streams."""
import numpy as np
import pytest
import torch

import spans as sp
from oracle import quantized as oq

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _prefill(g, B, H, D, Dk, s_p, s_v, s_t, dtype):
    r = lambda *s: sp.randn(g, *s, dtype=dtype).cuda()  # noqa: E731
    R = torch.linalg.qr(torch.randn(B, H, D, D, generator=g))[0][..., :Dk].contiguous().to(dtype).cuda()
    return {"kp": r(B, H, s_v, Dk), "prompt": r(B, H, s_p, D), "text": r(B, H, s_t, D),
            "V": r(B, H, s_p + s_v + s_t, D), "R": R, "dm": r(B, H, D)}


def _cache(x, fmt, reserve):
    from rotatek_amd.quantized_cache import QuantizedCache
    c = QuantizedCache(fmt, reserve_tokens=reserve)
    c.store_pruned(x["kp"], x["prompt"], x["text"], None, x["V"], 0)
    c.rotatek_rotations.append(x["R"])
    c.rotatek_means.append(x["dm"])
    return c


def _q(t, fmt):
    """The values a tensor's quantised form stands for."""
    return oq.values(*oq.quantize(sp.np64(t), fmt), fmt, t.shape[-1])


@pytest.mark.parametrize("fmt,dtype", [("mx8", torch.bfloat16), ("mx4", torch.float16)])
def test_prefill_then_growing_text(fmt, dtype):
    _say(f"growing text {fmt} {dtype}")
    g = torch.Generator().manual_seed(1)
    B, H, G, D, Dk, s_p, s_v, s_t = 2, 2, 4, 128, 32, 37, 150, 11
    x = _prefill(g, B, H, D, Dk, s_p, s_v, s_t, dtype)
    cache = _cache(x, fmt, 3)       # grows after three tokens
    s_all = s_p + s_v
    k = np.concatenate([_q(x["prompt"], fmt), _q(x["text"], fmt)], 2)
    v = np.concatenate([_q(x["V"][:, :, :s_p], fmt), _q(x["V"][:, :, s_all:], fmt)], 2)
    vis = dict(k=_q(x["kp"], fmt), v=_q(x["V"][:, :, s_p:s_all], fmt), R=sp.np64(x["R"]), dm=sp.np64(x["dm"]))
    for step in range(6):
        T = 1 if step != 3 else 5
        kn, vn = sp.randn(g, B, H, T, D, dtype=dtype).cuda(), sp.randn(g, B, H, T, D, dtype=dtype).cuda()
        cache.update(kn, vn, 0)
        k, v = np.concatenate([k, _q(kn, fmt)], 2), np.concatenate([v, _q(vn, fmt)], 2)
        q = sp.randn(g, B, H * G, D, dtype=dtype)
        out, a, b = cache.decode_rotatek(q.cuda(), 0, G)
        assert a is None and b is None
        sp.check(out, q, G, [vis, dict(k=k, v=v)], fmt, dtype)
        assert cache.get_seq_length() == s_v + k.shape[2]
        assert cache.lengths(0).tolist() == [k.shape[2]] * B


def test_captured_steps_equal_eager_ones():
    """append_ + decode in a graph, replayed as the text grows, with eager work
    and synchronisations between the replays."""
    _say("captured steps")
    g = torch.Generator().manual_seed(2)
    B, H, G, D = 3, 2, 7, 128
    x = _prefill(g, B, H, D, 32, 20, 500, 5, torch.bfloat16)
    a, b = _cache(x, "mx8", 40), _cache(x, "mx8", 40)
    q, kn, vn = (torch.zeros(*s, dtype=torch.bfloat16, device="cuda") for s in
                 ((B, H * G, D), (B, H, 1, D), (B, H, 1, D)))
    a.decode_rotatek(q, 0, G)       # workspace size known before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.append_(0, kn, vn)
        out, _, _ = a.decode_rotatek(q, 0, G)
    for step in range(5):
        for t in (q, kn, vn):
            t.copy_(sp.randn(g, *t.shape, dtype=torch.bfloat16))
        graph.replay()
        b.append_(0, kn, vn)
        want, _, _ = b.decode_rotatek(q, 0, G)
        if step % 2:
            torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(a.lengths(0), b.lengths(0))
        torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
    a.sync_lengths()
    assert a.get_seq_length() == 20 + 500 + 5 + 5


def test_two_graphs_and_two_streams_share_no_workspace():
    from rotatek_amd.kernels import full_channel_decode_quantized
    _say("two graphs, two streams")
    g = torch.Generator().manual_seed(3)
    B, H, G, D, S = 4, 4, 2, 128, 3000
    sets = []
    for i in range(2):
        k, _ = sp.rows(sp.randn(g, B, H, S, D), "mx8")
        v, _ = sp.rows(sp.randn(g, B, H, S, D), "mx8")
        q = sp.randn(g, B, H * G, D, dtype=torch.float16).cuda()
        want = full_channel_decode_quantized(q, k, v, G).clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = full_channel_decode_quantized(q, k, v, G)
        sets.append((q, k, v, want, graph, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for q, k, v, want, graph, out, stream in sets:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for q, k, v, want, graph, out, stream in sets:
        assert torch.equal(out, want)
    got = []
    for _ in range(10):
        for q, k, v, want, graph, out, stream in sets:
            with torch.cuda.stream(stream):
                got.append((full_channel_decode_quantized(q, k, v, G), want))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in got)


@pytest.mark.parametrize("fmt", ["mx8", "mx4", "plain"])
def test_many_questions_about_one_image(fmt):
    """A prefix stored once, text of each request appended as it comes, decode
    of all requests together, against the oracle; some have no text yet."""
    from rotatek_amd.kernels import shared_prefix_decode
    from rotatek_amd.quantized import MXRows, append_rows
    _say(f"one image {fmt}")
    g = torch.Generator().manual_seed(4)
    B, H, G, D, dtype, s_p, s_v, cap = 12, 2, 4, 128, torch.bfloat16, 40, 333, 64
    x = _prefill(g, 1, H, D, 32, s_p, s_v, 0, dtype)
    if fmt == "plain":
        kf, vf, ks, vs = x["prompt"], x["V"][:, :, :s_p], x["kp"], x["V"][:, :, s_p:]
        k2, v2 = (torch.full((B, H, cap, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    else:
        cache = _cache(x, fmt, 0)
        kf, vf, ks, vs = cache.spans(0)
        k2, v2 = MXRows.empty(B, H, cap, D, fmt), MXRows.empty(B, H, cap, D, fmt)
    as64 = sp.np64 if fmt == "plain" else (lambda t: _q(t, fmt))
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    tk, tv = np.zeros((B, H, cap, D)), np.zeros((B, H, cap, D))
    host = np.zeros(B, int)
    for step in range(4):
        # some requests get tokens, others wait
        T, some = 1 + 7 * step, torch.arange(B) % (step + 1) == 0
        kn, vn = sp.randn(g, B, H, T, D, dtype=dtype).cuda(), sp.randn(g, B, H, T, D, dtype=dtype).cuda()
        k64, v64 = as64(kn), as64(vn)
        for b in range(B):
            if some[b]:
                tk[b, :, host[b]:host[b] + T], tv[b, :, host[b]:host[b] + T] = k64[b], v64[b]
                if fmt == "plain":
                    k2[b, :, host[b]:host[b] + T], v2[b, :, host[b]:host[b] + T] = kn[b], vn[b]
                host[b] += T
        if fmt != "plain":
            append_rows(kn, vn, k2, v2, lens, advance=False)
        lens += T * some.to(torch.int32).cuda()
        q = sp.randn(g, B, H * G, D, dtype=dtype)
        out = shared_prefix_decode(q.cuda(), kf, vf, k2, v2, G, len_suffix=lens, R_partial=x["R"], delta_mu=x["dm"],
                                   k_sparse=ks, v_sparse=vs)
        spans = [dict(k=as64(x["prompt"]), v=as64(x["V"][:, :, :s_p])),
                 dict(k=as64(x["kp"]), v=as64(x["V"][:, :, s_p:]), R=sp.np64(x["R"]), dm=sp.np64(x["dm"])),
                 dict(k=tk, v=tv, valid=np.arange(cap)[None] < host[:, None])]
        sp.check(out, q, G, spans, fmt, dtype)


def test_store_and_growth_refusals():
    from rotatek_amd.quantized_cache import QuantizedCache
    with pytest.raises(ValueError):
        QuantizedCache("int8")
    with pytest.raises(ValueError):
        QuantizedCache(reserve_tokens=-1)
    g = torch.Generator().manual_seed(5)
    x = _prefill(g, 1, 1, 64, 16, 3, 40, 2, torch.float16)
    c = QuantizedCache("mx8")
    with pytest.raises(ValueError):
        c.store_pruned(x["kp"], x["prompt"], x["text"], None, x["V"], 1)
    with pytest.raises(ValueError):
        c.store_pruned(x["kp"], x["prompt"], x["text"], None, x["V"][:, :, 1:], 0)
    assert c.get_seq_length() == 0
    c.store_pruned(x["kp"], x["prompt"], x["text"], None, x["V"], 0)
    before = c.spans(0)[0].codes.clone()
    c.reserve(1000)
    assert c.spans(0)[0].shape[2] >= 1005
    assert torch.equal(c.spans(0)[0].codes[:, :, :5], before[:, :, :5])
    assert c.nbytes > 0 and len(c) == 1


def test_threads_issue_at_once():
    """Calls of several threads, a stream each, on shared rows."""
    from concurrent.futures import ThreadPoolExecutor
    from rotatek_amd.kernels import full_channel_decode_quantized, shared_prefix_decode
    from rotatek_amd.quantized import dequantize_rows, quantize_rows
    _say("threads")
    g = torch.Generator().manual_seed(6)
    x = sp.randn(g, 2, 4, 700, 128, dtype=torch.bfloat16).cuda()
    rows = quantize_rows(x, "mx8")
    back = dequantize_rows(rows)
    qs = [sp.randn(g, 2, 8, 128, dtype=torch.bfloat16).cuda() for _ in range(6)]
    want = [full_channel_decode_quantized(q, rows, rows, 2) for q in qs]
    both = [shared_prefix_decode(q, x[:1], x[:1], x, x, 2) for q in qs]
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                a = full_channel_decode_quantized(qs[i], rows, rows, 2)
                b = shared_prefix_decode(qs[i], x[:1], x[:1], x, x, 2)
                c = dequantize_rows(quantize_rows(x, "mx8"))
        stream.synchronize()
        return torch.equal(a, want[i]) and torch.equal(b, both[i]) and torch.equal(c, back)

    with ThreadPoolExecutor(6) as pool:
        assert all(pool.map(work, range(6)))


def test_tensors_elsewhere_and_other_objects_are_refused():
    from rotatek_amd.kernels import full_channel_decode_quantized, rotatek_decode_quantized, shared_prefix_decode
    from rotatek_amd.quantized import MXRows, append_rows, dequantize_rows, quantize_rows
    _say("elsewhere")
    x = torch.randn(1, 2, 40, 128, device="cuda")
    r, q = quantize_rows(x), torch.randn(1, 4, 128, device="cuda")
    away = MXRows(r.codes.cpu(), r.scales, 128)
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    for call in (lambda: full_channel_decode_quantized(q, r, away, 2),
                 lambda: full_channel_decode_quantized(q, r, r, 2, lens=lens.cpu()),
                 lambda: full_channel_decode_quantized(q, r, r, 2, lens=lens.long()),
                 lambda: full_channel_decode_quantized(q, r, r, 2, lens=torch.zeros(2, dtype=torch.int32, device="cuda")),
                 lambda: full_channel_decode_quantized(q, r, r, 2, mask=torch.ones(1, 40, dtype=torch.bool)),
                 lambda: full_channel_decode_quantized(q, r, r, 2, out=torch.empty(1, 4, 128)),
                 lambda: full_channel_decode_quantized(q, r, r, 2, out=torch.empty(1, 4, 128, device="cuda").half()),
                 lambda: full_channel_decode_quantized(q, r, r, 3),
                 lambda: full_channel_decode_quantized(q, r, r, 0),
                 lambda: full_channel_decode_quantized(q, r, quantize_rows(x, "mx4"), 2),
                 lambda: full_channel_decode_quantized(q, MXRows(None, r.scales, 128), r, 2),
                 lambda: rotatek_decode_quantized(q, x[..., :32], None, r, r, None, None, None, 2),
                 lambda: shared_prefix_decode(q, x, x, None, None, 2),      # plain fp32 rows
                 lambda: quantize_rows(x, out=away),
                 lambda: quantize_rows(x.double()),
                 lambda: quantize_rows(torch.zeros(1, 1, 4, 129, device="cuda")),
                 lambda: dequantize_rows(r, torch.int32),
                 lambda: dequantize_rows(r, out=torch.empty(1, 2, 40, 128)),
                 lambda: append_rows(x[:, :, :1], None, r, None, lens.cpu()),
                 lambda: append_rows(x[:, :, :1], None, r, None, lens.long()),
                 lambda: append_rows(x[:, :, :1], None, away, None, lens)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(AttributeError):
        shared_prefix_decode(q, [x], [x], None, None, 2)
    with pytest.raises(ValueError):     # int("two")
        full_channel_decode_quantized(q, r, r, "two")
    with pytest.raises(RuntimeError):
        full_channel_decode_quantized(q.cpu(), r, r, 2)
    # after all that a call as it should be
    assert torch.isfinite(full_channel_decode_quantized(q, r, r, 2)).all()
