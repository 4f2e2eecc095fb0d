"""Decode of a batch that shares a prefix against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import spans as sp

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _hold(x, fmt):
    return (x.cuda(), sp.np64(x)) if fmt == "plain" else sp.rows(x, fmt)


def _case(B, Hq, H, D, S_p, Dk, S_v, S_s, dtype, fmt, seed=0, lens=None, bias=True):
    g = torch.Generator().manual_seed(seed)
    c = {"q": sp.randn(g, B, Hq, D, dtype=dtype), "groups": Hq // H, "fmt": fmt, "dtype": dtype, "kw": {}}
    c["k"], k = _hold(sp.randn(g, 1, H, S_p, D, dtype=dtype), fmt)
    c["v"], v = _hold(sp.randn(g, 1, H, S_p, D, dtype=dtype), fmt)
    c["spans"] = [dict(k=k, v=v, valid=np.ones((B, S_p), bool))]
    c["k2"] = c["v2"] = None
    if S_v:
        R = torch.linalg.qr(torch.randn(1, H, D, D, generator=g))[0][..., :Dk].contiguous().to(dtype)
        dm = sp.randn(g, 1, H, D, dtype=dtype, scale=0.5) if bias else None
        ks, ks64 = _hold(sp.randn(g, 1, H, S_v, Dk, dtype=dtype, scale=2.0), fmt)
        vs, vs64 = _hold(sp.randn(g, 1, H, S_v, D, dtype=dtype), fmt)
        c["kw"] = dict(R_partial=R.cuda(), delta_mu=None if dm is None else dm.cuda(), k_sparse=ks, v_sparse=vs)
        c["spans"].append(dict(k=ks64, v=vs64, R=sp.np64(R), dm=sp.np64(dm)))
    if S_s is not None:
        c["k2"], k2 = _hold(sp.randn(g, B, H, S_s, D, dtype=dtype), fmt)
        c["v2"], v2 = _hold(sp.randn(g, B, H, S_s, D, dtype=dtype), fmt)
        valid = np.ones((B, S_s), bool)
        if lens is not None:
            n = torch.tensor([lens[b % len(lens)] for b in range(B)], dtype=torch.int32)
            c["kw"]["len_suffix"] = n.cuda()
            valid &= np.arange(S_s)[None] < n.numpy()[:, None]
        c["spans"].append(dict(k=k2, v=v2, valid=valid))
    return c


def _run(c):
    from rotatek_amd.kernels import shared_prefix_decode
    out = shared_prefix_decode(c["q"].cuda(), c["k"], c["v"], c["k2"], c["v2"], c["groups"], **c["kw"])
    torch.cuda.synchronize()
    return out


def _check(c):
    sp.check(_run(c), c["q"], c["groups"], c["spans"], c["fmt"], c["dtype"])


CASES = [
    # B, Hq, H, D, S_p, Dk, S_v, S_s, lens
    (1, 2, 2, 128, 1, 0, 0, 1, None),
    (2, 4, 2, 128, 100, 0, 0, 33, [0, 7]),
    (3, 28, 4, 128, 60, 32, 517, 20, [1, 20, 0]),      # G = 7, 21 rows: one unit of 64
    (9, 14, 2, 128, 300, 0, 0, 40, [3, 40, 0, 31]),    # 63 rows
    (20, 8, 2, 128, 129, 40, 200, 5, [5, 0, 2]),       # 80 rows: two units
    (5, 3, 3, 128, 1, 64, 333, 65, None),
    (4, 4, 1, 128, 0, 32, 400, 10, [10]),              # no prompt
    (4, 4, 1, 128, 200, 0, 0, None, None),             # no text
    (2, 8, 8, 64, 333, 16, 70, 31, [31, 1]),
    (17, 4, 1, 64, 150, 0, 0, 64, [64, 0, 63]),        # 68 rows, D = 64
    (3, 6, 2, 96, 90, 48, 130, 7, None),
    (2, 4, 2, 80, 257, 0, 0, 12, [12, 3]),
    (2, 2, 1, 128, 5000, 0, 0, 600, [600, 599]),       # several workgroups
    (2, 20, 1, 128, 64, 128, 100, 9, None),
    (1, 80, 1, 128, 100, 0, 0, 50, None),              # 80 heads on one KV head
]


@pytest.mark.parametrize("fmt,dtype", [("plain", torch.bfloat16), ("plain", torch.float16), ("mx8", torch.bfloat16),
                                       ("mx8", torch.float16), ("mx4", torch.bfloat16), ("mx4", torch.float32)])
@pytest.mark.parametrize("case", CASES)
def test_shared_prefix_matches_the_oracle(case, fmt, dtype):
    _say(f"{case} {fmt} {dtype}")
    _check(_case(*case[:8], dtype, fmt, seed=sum(case[:7]), lens=case[8]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [
    (3, 4, 2, 33, 70, 0, 0, 20, [20, 3, 0]), (2, 4, 2, 1, 40, 1, 30, 5, None), (2, 6, 2, 127, 100, 33, 64, 9, [9, 0]),
    (1, 4, 1, 60, 64, 20, 33, None, None),
])
def test_odd_head_dims(case, dtype):
    _say(f"{case} {dtype}")
    _check(_case(*case[:8], dtype, "plain", seed=3, lens=case[8]))


def test_strided_rows():
    from rotatek_amd.kernels import shared_prefix_decode
    _say("strides")
    c = _case(6, 8, 2, 128, 150, 32, 70, 40, torch.bfloat16, "plain", seed=11, lens=[40, 0, 13])
    want = _run(c)
    kw = dict(c["kw"])

    def spread(t):      # every second channel of a wider tensor
        w = torch.full((*t.shape[:-1], 2 * t.shape[-1]), float("nan"), dtype=t.dtype, device="cuda")
        w[..., ::2] = t
        return w[..., ::2]

    def heads_last(t):  # [N, S, H, D] storage, 16-byte rows
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    for f in (spread, heads_last):
        kw["k_sparse"], kw["v_sparse"] = f(c["kw"]["k_sparse"]), f(c["kw"]["v_sparse"])
        got = shared_prefix_decode(c["q"].cuda(), f(c["k"]), f(c["v"]), f(c["k2"]), f(c["v2"]), c["groups"], **kw)
        sp.check(got, c["q"], c["groups"], c["spans"], "plain", torch.bfloat16)
        if f is heads_last:
            assert torch.equal(got, want)


def test_rows_past_the_length_may_hold_anything():
    _say("garbage")
    for fmt in ("plain", "mx8"):
        c = _case(3, 8, 2, 128, 40, 32, 70, 50, torch.bfloat16, fmt, seed=12, lens=[0, 13, 33])
        want = _run(c).clone()
        for b, n in enumerate([0, 13, 33]):
            for r in (c["k2"], c["v2"]):
                if fmt == "plain":
                    r[b, :, n:] = float("nan")
                else:
                    r.codes[b, :, n:] = 0x7f
                    r.scales[b, :, :, n:] = 255
        assert torch.equal(_run(c), want)


def test_infinite_keys_past_the_head():
    """Channels of a wider buffer behind the head's are not read into it."""
    from rotatek_amd.kernels import shared_prefix_decode
    _say("neighbouring channels")
    c = _case(3, 4, 2, 96, 64, 40, 64, 32, torch.float16, "plain", seed=13)
    want = _run(c)

    def wide(t):
        w = torch.full((*t.shape[:-1], 128), float("inf"), dtype=t.dtype, device="cuda")
        w[..., :t.shape[-1]] = t
        return w[..., :t.shape[-1]]

    kw = dict(c["kw"])
    kw["k_sparse"], kw["v_sparse"] = wide(kw["k_sparse"]), wide(kw["v_sparse"])
    got = shared_prefix_decode(c["q"].cuda(), wide(c["k"]), wide(c["v"]), wide(c["k2"]), wide(c["v2"]), 2, **kw)
    assert torch.equal(got, want)


def test_same_as_the_expanded_batch():
    """rotatek_decode of every request over its own copy gives the same."""
    from rotatek_amd.kernels.gqa_decode import rotatek_decode_gqa
    _say("expanded batch")
    B = 5
    c = _case(B, 8, 2, 128, 60, 32, 300, 30, torch.float16, "plain", seed=14)
    got = _run(c)
    x = lambda t: t.expand(B, *t.shape[1:])  # noqa: E731
    kw = c["kw"]
    want, _, _ = rotatek_decode_gqa(c["q"].cuda(), x(kw["R_partial"]), x(kw["delta_mu"]),
                                    torch.cat([x(c["k"]), c["k2"]], 2), torch.cat([x(c["v"]), c["v2"]], 2),
                                    torch.ones(B, 90, dtype=torch.uint8, device="cuda"), x(kw["k_sparse"]),
                                    x(kw["v_sparse"]), c["groups"])
    # two roundings to fp16 of values within 4 of zero
    assert (got.float() - want.float()).abs().max() <= 2 * 2.0 ** -11 * want.float().abs().max() + 1e-4


# As many queries on the same rows as make the waves take queries (from 2048
# bytes of a token times blocks of 16 queries), in every format.
MANY = [
    (61, 8, 2, 128, 100, 0, 0, 20, [20, 0, 3]),        # 244 rows: 4 blocks of 64, the last of 52
    (101, 4, 1, 128, 33, 32, 517, 9, [9, 0, 1, 4]),
    (101, 4, 1, 128, 1, 64, 70, 5, None),
    (65, 4, 1, 128, 0, 128, 130, None, None),          # no prompt, no text, all channels kept
    (150, 4, 1, 64, 150, 16, 70, 31, [31, 0]),
    (130, 4, 1, 96, 257, 40, 64, 0, None),             # a suffix of no rows
    (160, 2, 1, 80, 1, 8, 1, 1, None),                 # single tokens
]


@pytest.mark.parametrize("fmt,dtype", [("plain", torch.bfloat16), ("plain", torch.float16), ("mx8", torch.bfloat16),
                                       ("mx8", torch.float16), ("mx4", torch.bfloat16), ("mx4", torch.float32)])
@pytest.mark.parametrize("case", MANY)
def test_many_requests(case, fmt, dtype):
    _say(f"{case} {fmt} {dtype}")
    _check(_case(*case[:8], dtype, fmt, seed=sum(case[:7]), lens=case[8]))


@pytest.mark.parametrize("rows", [63, 64, 65, 79, 81, 127, 128, 129])
def test_either_side_of_a_block_of_queries(rows):
    _say(f"{rows} rows")
    _check(_case(rows, 1, 1, 128, 130, 0, 0, 3, torch.bfloat16, "plain", seed=rows, lens=[3, 0]))
    _check(_case(rows, 1, 1, 128, 66, 32, 130, 3, torch.float16, "plain", seed=rows, lens=[2, 1]))


@pytest.mark.parametrize("B,S_s,lens", [(40, 4200, [4200, 0, 4097, 31]), (40, 4096, [4096, 1]), (3, 4200, [4200, 129])])
def test_long_texts(B, S_s, lens):
    _say(f"long texts {B} {S_s}")
    _check(_case(B, 2, 1, 128, 200, 0, 0, S_s, torch.bfloat16, "plain", seed=S_s, lens=lens))


@pytest.mark.parametrize("B", [3, 70])
@pytest.mark.parametrize("fmt,dtype", [("plain", torch.bfloat16), ("mx8", torch.float16)])
def test_other_layouts_of_the_queries_and_the_rotation(B, fmt, dtype):
    """Queries and rotations that are not in whole aligned pieces of one type."""
    from rotatek_amd.kernels import shared_prefix_decode
    _say(f"layouts {B} {fmt}")
    c = _case(B, 4, 1, 128, 40, 32, 150, 7, dtype, fmt, seed=21, lens=[7, 0])
    kw = dict(c["kw"])
    wide = torch.zeros(B, 4, 260, dtype=dtype, device="cuda")
    wide[..., 1::2] = torch.cat([c["q"].cuda(), torch.zeros(B, 4, 2, dtype=dtype, device="cuda")], -1)
    q = wide[..., 1:257:2]
    assert torch.equal(q, c["q"].cuda())
    call = lambda q, **k: shared_prefix_decode(q, c["k"], c["v"], c["k2"], c["v2"], 4, **{**kw, **k})  # noqa: E731
    sp.check(call(q), c["q"], 4, c["spans"], fmt, dtype)
    sp.check(call(c["q"].cuda(), R_partial=kw["R_partial"].float()), c["q"], 4, c["spans"], fmt, dtype)
    sp.check(call(c["q"].cuda(), R_partial=kw["R_partial"].transpose(2, 3).contiguous().transpose(2, 3)), c["q"], 4,
             c["spans"], fmt, dtype)
    sp.check(call(c["q"].cuda(), delta_mu=kw["delta_mu"].float()), c["q"], 4, c["spans"], fmt, dtype)
    out = torch.full((B, 8, 128), 7.0, dtype=dtype, device="cuda")
    sp.check(call(q, out=out[:, ::2]), c["q"], 4, c["spans"], fmt, dtype)
    assert (out[:, 1::2] == 7).all()


@pytest.mark.parametrize("B", [3, 70])
@pytest.mark.parametrize("fmt", ["plain", "mx8"])
def test_rotation_that_keeps_no_channel(B, fmt):
    """Scores of the image are q . delta_mu alone."""
    _say(f"no channel kept {B} {fmt}")
    dtype = torch.bfloat16
    c = _case(B, 4, 1, 128, 40, 0, 150, 7, dtype, fmt, seed=22, lens=[7, 0])
    _check(c)


@pytest.mark.parametrize("B", [4, 70])
def test_scores_of_minus_infinity(B):
    """Products past the range of fp32: weight zero, also where a row's first
    tokens are all such and its neighbours' are not."""
    from rotatek_amd.kernels import shared_prefix_decode
    _say(f"scores past the range {B}")
    c = _case(B, 2, 1, 128, 300, 0, 0, 33, torch.bfloat16, "plain", seed=23)
    q, k = c["q"].clone(), c["k"].clone()
    # channel 0 is the odd heads' alone: 2^126 there, Keys of -2^10 in 0 .. 259,
    # of 0 behind and in the text
    q[:, 0, 0], q[:, 1, 0] = 0, 2.0 ** 126
    k[..., 0] = 0
    k[:, :, :260, 0] = -2.0 ** 10
    c["k2"][..., 0] = 0
    got = shared_prefix_decode(q.cuda(), k, c["v"], c["k2"], c["v2"], 2)
    even, odd = [dict(s) for s in c["spans"]], [dict(s) for s in c["spans"]]
    even[0]["k"] = odd[0]["k"] = sp.np64(k)
    even[1]["k"] = odd[1]["k"] = sp.np64(c["k2"])
    odd[0]["valid"] = np.broadcast_to(np.arange(300) >= 260, (B, 300))
    for h, spans in ((0, even), (1, odd)):
        qh = q[:, h:h + 1].clone()
        qh[..., 0] = 0
        sp.check(got[:, :, h:h + 1], qh, 1, spans, "plain", torch.bfloat16)
    # nothing else to attend: zeros
    alone = shared_prefix_decode(q.cuda(), k[:, :, :260], c["v"][:, :, :260], None, None, 2)
    assert (alone[:, 0, 1] == 0).all() and torch.isfinite(alone).all()


def test_heads_far_apart():
    """Offsets between heads and requests past 32 bits."""
    from rotatek_amd.kernels import shared_prefix_decode
    _say("far apart")
    c = _case(3, 4, 2, 128, 70, 0, 0, 20, torch.bfloat16, "plain", seed=24, lens=[20, 0, 5])
    want = _run(c)
    far = 1100 * 2 ** 20        # elements: 2.2 GB
    buf = torch.zeros(2 * far + 2 ** 16, dtype=torch.bfloat16, device="cuda")
    at = 0

    def apart(t, sb, sh):
        nonlocal at
        w = buf.as_strided(t.shape, (sb, sh, 128, 1), at)
        w.copy_(t)
        at += t.shape[2] * 128
        return w

    k, v = apart(c["k"], 0, far), apart(c["v"], 0, far)
    k2, v2 = (apart(t, far, 40 * 128) for t in (c["k2"], c["v2"]))
    got = shared_prefix_decode(c["q"].cuda(), k, v, k2, v2, 2, **c["kw"])
    assert torch.equal(got, want)


def test_captured_with_tiles():
    """Replays as the text grows, with eager work between."""
    from rotatek_amd.kernels import shared_prefix_decode
    _say("captured")
    c = _case(70, 4, 1, 128, 90, 32, 300, 40, torch.bfloat16, "plain", seed=25, lens=[1])
    q, kw = c["q"].cuda(), c["kw"]
    call = lambda: shared_prefix_decode(q, c["k"], c["v"], c["k2"], c["v2"], 4, **kw)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(5):
        kw["len_suffix"].fill_(1 + 9 * step)
        q.mul_(-0.9)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        torch.randn(500, 500, device="cuda").sum()
