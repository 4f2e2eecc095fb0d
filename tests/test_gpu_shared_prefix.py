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
