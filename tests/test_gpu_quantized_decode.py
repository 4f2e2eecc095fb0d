"""Decode over quantised rows against the 64-bit oracle over the same codes."""
import numpy as np
import pytest
import torch

import spans as sp

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _case(B, Hq, H, D, Dk, S_v, S_f, dtype, fmt, seed=0, mask=False, lens=None, bias=True):
    g = torch.Generator().manual_seed(seed)
    c = {"q": sp.randn(g, B, Hq, D, dtype=dtype), "groups": Hq // H, "fmt": fmt, "dtype": dtype, "spans": []}
    c["k_full"], kf = sp.rows(sp.randn(g, B, H, S_f, D), fmt)
    c["v_full"], vf = sp.rows(sp.randn(g, B, H, S_f, D), fmt)
    valid = np.ones((B, S_f), bool)
    c["mask"] = c["lens"] = None
    if mask:
        m = torch.rand(B, S_f, generator=g) < 0.7
        m[0] = False
        c["mask"] = m.to(torch.uint8).cuda()
        valid &= m.numpy()
    if lens is not None:
        n = torch.tensor([lens[b % len(lens)] for b in range(B)], dtype=torch.int32)
        c["lens"] = n.cuda()
        valid &= np.arange(S_f)[None] < n.numpy()[:, None]
    c["spans"].append(dict(k=kf, v=vf, valid=valid))
    if S_v:
        R = torch.linalg.qr(torch.randn(B, H, D, D, generator=g))[0][..., :Dk].contiguous().to(dtype)
        dm = sp.randn(g, B, H, D, dtype=dtype, scale=0.5) if bias else None
        c["R"], c["dm"] = R.cuda(), None if dm is None else dm.cuda()
        c["k_sparse"], ks = sp.rows(sp.randn(g, B, H, S_v, Dk, scale=2.0), fmt)
        c["v_sparse"], vs = sp.rows(sp.randn(g, B, H, S_v, D), fmt)
        c["spans"].append(dict(k=ks, v=vs, R=sp.np64(R), dm=sp.np64(dm)))
    return c


def _run(c):
    from rotatek_amd.kernels import full_channel_decode_quantized, rotatek_decode_quantized
    q = c["q"].cuda()
    if "R" in c:
        out, a, b = rotatek_decode_quantized(q, c["R"], c["dm"], c["k_full"], c["v_full"], c["mask"], c["k_sparse"],
                                             c["v_sparse"], c["groups"], len_full=c["lens"])
        assert a is None and b is None
    else:
        out = full_channel_decode_quantized(q, c["k_full"], c["v_full"], c["groups"], mask=c["mask"], lens=c["lens"])
    torch.cuda.synchronize()
    return out


def _check(c):
    sp.check(_run(c), c["q"], c["groups"], c["spans"], c["fmt"], c["dtype"])


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", [
    # B, Hq, H, D, Dk, S_v, S_f
    (1, 2, 2, 128, 32, 1, 1),
    (2, 4, 4, 128, 32, 300, 50),
    (1, 28, 4, 128, 32, 517, 129),      # G = 7
    (2, 8, 1, 128, 64, 333, 31),
    (1, 40, 2, 128, 40, 200, 20),       # G = 20: more than one block of 16 rows
    (1, 70, 1, 128, 32, 129, 33),       # G = 70: two units
    (2, 2, 2, 128, 128, 260, 7),
    (1, 4, 2, 128, 96, 150, 40),
    (2, 4, 2, 128, 1, 100, 64),
    (1, 4, 4, 128, 32, 700, 0),         # no prompt or text
    (2, 8, 2, 128, 0, 0, 600),          # dense
    (1, 3, 3, 64, 16, 400, 65),
    (2, 8, 2, 64, 64, 130, 31),
    (3, 4, 2, 64, 0, 0, 333),
    (1, 4, 2, 80, 24, 140, 90),
    (2, 6, 3, 96, 33, 70, 100),
    (1, 2, 1, 1, 1, 40, 40),
    (1, 4, 1, 33, 17, 64, 95),
    (1, 2, 2, 127, 100, 50, 200),
    (1, 1, 1, 128, 32, 4500, 1000),     # several workgroups
])
def test_decode_matches_the_oracle(case, dtype, fmt):
    _say(f"{case} {dtype} {fmt}")
    _check(_case(*case, dtype, fmt, seed=sum(case)))


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
@pytest.mark.parametrize("case", [
    (4, 4, 2, 128, 32, 200, 150), (3, 8, 2, 128, 0, 0, 300), (4, 2, 2, 64, 16, 40, 129), (5, 20, 1, 128, 0, 0, 1100),
])
def test_masks_and_lengths(case, fmt):
    for mask, lens in ((True, None), (False, [0, 1, 31, 32, 33]), (True, [0, 5, 64, 100000, -3])):
        _say(f"{case} {fmt} mask={mask} lens={lens}")
        _check(_case(*case, torch.bfloat16, fmt, seed=7, mask=mask, lens=lens))


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_rows_that_do_not_count_may_hold_anything(fmt):
    _say(f"garbage {fmt}")
    c = _case(3, 4, 2, 128, 32, 70, 100, torch.float16, fmt, seed=3, mask=True, lens=[40, 100, 64])
    want = _run(c).clone()
    dead = torch.from_numpy(~c["spans"][0]["valid"]).cuda()
    for r in (c["k_full"], c["v_full"]):
        r.codes[dead.unsqueeze(1).expand(3, 2, 100)] = 0x7f         # e4m3: NaN
        r.scales[..., :100][dead.view(3, 1, 1, 100).expand(3, 2, 4, 100)] = 255
        r.scales[..., 100:] = 255                                    # the padding as well
    assert torch.equal(_run(c), want)


def test_nan_reaches_only_the_requests_that_attend_it():
    _say("nan")
    c = _case(2, 4, 2, 128, 32, 70, 100, torch.bfloat16, "mx8", seed=4)
    c["k_full"].scales[1, 1, 2, 50] = 255
    out = _run(c)
    assert torch.isnan(out[1, 0, 2:]).all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, 0, :2]).all()


def test_no_bias_and_no_kept_channels():
    _say("no bias, Dk = 0")
    _check(_case(2, 4, 2, 128, 32, 200, 50, torch.bfloat16, "mx8", seed=5, bias=False))
    # every channel pruned: the visual logits are the bias alone
    for fmt in ("mx8", "mx4"):
        for D in (64, 128):
            _check(_case(2, 4, 2, D, 0, 70, 50, torch.bfloat16, fmt, seed=6))
            _check(_case(2, 4, 2, D, 0, 70, 0, torch.bfloat16, fmt, seed=6, bias=False))


def test_large_scores_and_equal_scores():
    _say("large scores")
    c = _case(1, 4, 4, 128, 0, 0, 500, torch.float32, "mx8", seed=8)
    c["q"] = c["q"] * 30
    _check(c)
    c["q"] = c["q"] * 0
    _check(c)


def test_nothing_at_all():
    from rotatek_amd.kernels import full_channel_decode_quantized
    from rotatek_amd.quantized import MXRows
    _say("empty")
    q = torch.randn(2, 4, 128, device="cuda", dtype=torch.bfloat16)
    k, v = MXRows.empty(2, 2, 0, 128), MXRows.empty(2, 2, 0, 128)
    assert (full_channel_decode_quantized(q, k, v, 2) == 0).all()
    e = full_channel_decode_quantized(q[:0], MXRows.empty(0, 2, 5, 128), MXRows.empty(0, 2, 5, 128), 2)
    assert e.shape == (0, 1, 4, 128)


def test_strided_queries_rows_masks_and_outputs():
    from rotatek_amd.kernels import full_channel_decode_quantized, rotatek_decode_quantized
    _say("strides")
    c = _case(3, 8, 2, 128, 32, 130, 96, torch.bfloat16, "mx8", seed=9, mask=True)
    want = _run(c)
    q = torch.zeros(3, 128, 8, device="cuda", dtype=torch.bfloat16).transpose(1, 2).copy_(c["q"])
    R = torch.zeros(3, 2, 32, 128, device="cuda", dtype=torch.bfloat16).transpose(2, 3).copy_(c["R"])
    mask = torch.zeros(96, 6, device="cuda", dtype=torch.bool)[:, ::2].t().copy_(c["mask"])
    out = torch.full((3, 8, 256), 9.0, device="cuda", dtype=torch.bfloat16)
    got, _, _ = rotatek_decode_quantized(q, R.float(), c["dm"].half().float(), c["k_full"], c["v_full"], mask,
                                         c["k_sparse"], c["v_sparse"], 4, out=out[..., ::2])
    # queries of other layouts and types are rotated in another order of
    # summation: the oracle's tolerance, not the same bits
    sp.check(got, c["q"], 4, c["spans"], "mx8", torch.bfloat16)
    assert got.data_ptr() == out.data_ptr() and (out[..., 1::2] == 9.0).all()
    # the same layouts but q's and R's: the same bits
    got, _, _ = rotatek_decode_quantized(c["q"].cuda(), c["R"], c["dm"], c["k_full"], c["v_full"], mask, c["k_sparse"],
                                         c["v_sparse"], 4, out=out[..., ::2])
    assert torch.equal(got, want)
    # rows that are views: the second half of a buffer, and every other request
    from rotatek_amd.quantized import MXRows
    c = _case(2, 4, 2, 128, 0, 0, 64, torch.float16, "mx4", seed=10)
    want = _run(c)
    big_k, big_v = MXRows.empty(4, 2, 128, 128, "mx4"), MXRows.empty(4, 2, 128, 128, "mx4")
    views = []
    for big, r in ((big_k, c["k_full"]), (big_v, c["v_full"])):
        big.codes.fill_(0x77)
        big.scales.fill_(255)
        view = MXRows(big.codes[::2], big.scales[::2], 128, "mx4").narrow(64, 64)
        view.codes.copy_(r.codes)
        view.scales.copy_(r.scales)
        views.append(view)
    assert torch.equal(full_channel_decode_quantized(c["q"].cuda(), *views, 2), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("S_f", [1, 2, 31, 32, 33, 100, 700])
def test_masks_in_every_layout(S_f, dtype):
    """Neighbouring bytes at any address, every third byte, one row for all."""
    from rotatek_amd.kernels import full_channel_decode_quantized, rotatek_decode_quantized
    _say(f"mask layouts {S_f} {dtype}")
    for Dk, S_v in ((0, 0), (32, 70)):
        c = _case(3, 8, 2, 128, Dk, S_v, S_f, dtype, "mx8", seed=31 + S_f, mask=True)
        m = c["mask"]
        flat = torch.full((3 * S_f + 1,), 255, dtype=torch.uint8, device="cuda")
        flat[1:] = m.reshape(-1)
        wide = torch.full((3, S_f, 3), 255, dtype=torch.uint8, device="cuda")
        wide[..., 1] = m
        for mask in (m, m.bool(), flat[1:].view(3, S_f), wide[..., 1], m * 128):
            if S_v:
                out = rotatek_decode_quantized(c["q"].cuda(), c["R"], c["dm"], c["k_full"], c["v_full"], mask, c["k_sparse"],
                                               c["v_sparse"], c["groups"])[0]
            else:
                out = full_channel_decode_quantized(c["q"].cuda(), c["k_full"], c["v_full"], c["groups"], mask=mask)
            sp.check(out, c["q"], c["groups"], c["spans"], "mx8", dtype)
        one = m[1:2].expand(3, S_f)
        same = full_channel_decode_quantized(c["q"].cuda(), c["k_full"], c["v_full"], c["groups"], mask=one)
        want = full_channel_decode_quantized(c["q"].cuda(), c["k_full"], c["v_full"], c["groups"], mask=one.contiguous())
        assert torch.equal(same, want)
