"""fp16 queries whose rotation leaves fp16's range (65504): the shared-prefix
decode over plain fp16 rows forms q R in 16-bit terms and has to scale them.

Most inputs are whole numbers times powers of two, chosen so that q R, every
product and every sum of a score is exact in fp32: the scores are then of
ordinary size and the oracle's tolerance (``spans.tolerance``) is tight.
"""
import numpy as np
import pytest
import torch

import spans as sp

pytestmark = pytest.mark.gpu

D, F16 = 128, torch.float16


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _ints(g, top, *shape):
    return torch.randint(-top, top + 1, shape, generator=g).float()


def _exact(g, B, H, G, Dk, S_p, S_v, S_s, bias):
    """q up to 7 2^13, column c of R adds 128 / Dk of its channels (twice one
    where all are kept), Keys and means up to 2 2^-14: products are whole
    multiples of 2^-1, q R reaches 14 2^13 at least."""
    c = {"q": (_ints(g, 7, B, H * G, D) * 2.0 ** 13).half()}
    R = torch.zeros(1, H, D, Dk)
    per = D // Dk
    for i in range(Dk):
        R[:, :, per * i:per * (i + 1), i] = 2.0 if per == 1 else 1.0
    c["R"] = R.half()
    c["dm"] = (_ints(g, 2, 1, H, D) * 2.0 ** -14).half() if bias else None
    k = lambda *s: (_ints(g, 2, *s) * 2.0 ** -14).half()  # noqa: E731
    v = lambda *s: sp.randn(g, *s, dtype=F16)  # noqa: E731
    c["k"], c["v"] = k(1, H, S_p, D), v(1, H, S_p, D)
    c["ks"], c["vs"] = k(1, H, S_v, Dk), v(1, H, S_v, D)
    c["k2"], c["v2"] = (k(B, H, S_s, D), v(B, H, S_s, D)) if S_s else (None, None)
    qr = torch.matmul(c["q"].double().view(B, H, G, D), R.double())
    assert qr.abs().max() > 65504
    return c


def _call(c, G, **kw):
    from rotatek_amd.kernels import shared_prefix_decode
    d = {n: None if t is None else t.cuda() for n, t in {**c, **kw}.items()}
    return shared_prefix_decode(d["q"], d["k"], d["v"], d["k2"], d["v2"], G, R_partial=d["R"], delta_mu=d["dm"],
                                k_sparse=d["ks"], v_sparse=d["vs"])


def _spans(c):
    s = [dict(k=sp.np64(c["k"]), v=sp.np64(c["v"]), valid=np.ones((len(c["q"]), c["k"].shape[2]), bool)),
         dict(k=sp.np64(c["ks"]), v=sp.np64(c["vs"]), R=sp.np64(c["R"]), dm=sp.np64(c["dm"]))]
    if c["k2"] is not None:
        s.append(dict(k=sp.np64(c["k2"]), v=sp.np64(c["v2"]), valid=np.ones((len(c["q"]), c["k2"].shape[2]), bool)))
    return s


@pytest.mark.parametrize("B", [1, 3, 70])     # one request; waves take tokens; waves take queries
@pytest.mark.parametrize("Dk", [16, 32, 64, 128])
def test_rotations_past_the_range(B, Dk):
    _say(f"past the range {B} {Dk}")
    g = torch.Generator().manual_seed(100 * B + Dk)
    c = _exact(g, B, 1, 4, Dk, 40, 200, 9 if B > 1 else 0, Dk != 64)
    s = _spans(c)
    sp.check(_call(c, 4), c["q"], 4, s, "plain", F16)
    # rotations formed ahead: another type, another order in memory
    sp.check(_call(c, 4, R=c["R"].float()), c["q"], 4, s, "plain", F16)
    sp.check(_call(c, 4, R=c["R"].transpose(2, 3).contiguous().transpose(2, 3)), c["q"], 4, s, "plain", F16)


@pytest.mark.parametrize("B", [3, 70])
def test_a_large_query_leaves_its_neighbours_alone(B):
    """Each query has a scale of its own: the others' terms do not change.  (Their
    results may, in fp32's roundings: a wave raises the running maxima of its 16
    rows together, where one asks for it, and p 2^-up is rounded to 16-bit terms
    after that: 2^-22 of a weight, as the oracle's tolerance counts it.)"""
    _say(f"neighbours {B}")
    g = torch.Generator().manual_seed(B)
    c = _exact(g, B, 1, 4, 32, 40, 200, 9, True)
    for n in ("ks", "k", "k2"):
        c[n] = sp.randn(g, *c[n].shape, dtype=F16)
    small, large = sp.randn(g, B, 4, D, dtype=F16), c["q"]
    mixed = small.clone()
    mixed[1, 2] = large[1, 2]
    rest = [b for b in range(B) if b != 1]
    for R in (c["R"], c["R"].float()):
        got = _call(c, 4, q=mixed, R=R)
        assert torch.isfinite(got).all()
        for h in range(4):
            on = rest if h == 2 else list(range(B))
            part = {**c, "q": small[on][:, h:h + 1], "k2": c["k2"][on], "v2": c["v2"][on]}
            sp.check(got[on][:, :, h:h + 1], part["q"], 1, _spans(part), "plain", F16)


@pytest.mark.parametrize("B", [2, 70])
@pytest.mark.parametrize("G", [2, 4])
def test_random_queries_past_the_range(B, G):
    """Queries of order 3e4 under an orthonormal R: scores of order 1e4, of which
    the largest takes all the weight.  An fp32 score is off by at most 137 2^-24 of
    its sum of magnitudes; where the two best lie further apart than twice that and
    20 nats, the others weigh 2e-9 and 340 of them 1e-6 in all: the output is the
    best token's value / (1 + 1e-6), off by half a step and 2e-6 of the largest."""
    _say(f"random past the range {B} {G}")
    H, Dk, S_v, S_p = 4, 32, 300, 40
    g = torch.Generator().manual_seed(30000 + B)
    q = (torch.randn(B, H * G, D, generator=g) * 3e4).clamp(-6e4, 6e4).half()
    c = {"q": q, "k2": None, "v2": None, "dm": sp.randn(g, 1, H, D, dtype=F16, scale=0.5),
         "R": torch.linalg.qr(torch.randn(1, H, D, D, generator=g))[0][..., :Dk].contiguous().half(),
         "k": sp.randn(g, 1, H, S_p, D, dtype=F16), "v": sp.randn(g, 1, H, S_p, D, dtype=F16),
         "ks": sp.randn(g, 1, H, S_v, Dk, dtype=F16, scale=2.0), "vs": sp.randn(g, 1, H, S_v, D, dtype=F16)}
    n = {k: sp.np64(t) for k, t in c.items()}
    clear, want = np.zeros((B, H * G), bool), np.zeros((B, H * G, D))
    past = 0.0
    for b in range(B):
        for h in range(H * G):
            x, kv = n["q"][b, h], h // G
            qr, xa = x @ n["R"][0, kv], np.abs(x)
            past = max(past, np.abs(qr).max())
            s = np.concatenate([n["k"][0, kv] @ x, n["ks"][0, kv] @ qr + x @ n["dm"][0, kv]]) / D ** 0.5
            size = max((np.abs(n["k"][0, kv]) @ xa).max(),
                       (np.abs(n["ks"][0, kv]) @ (xa @ np.abs(n["R"][0, kv])) + xa @ np.abs(n["dm"][0, kv])).max())
            top = np.argsort(s)
            clear[b, h] = s[top[-1]] - s[top[-2]] > 2 * 137 * 2.0 ** -24 * size / D ** 0.5 + 20
            want[b, h] = np.concatenate([n["v"][0, kv], n["vs"][0, kv]])[top[-1]]
    assert past > 65504 and clear.mean() > 0.9
    for R in (c["R"], c["R"].float()):
        got = _call(c, G, R=R)
        assert torch.isfinite(got).all()
        over = np.abs(sp.np64(got)[:, 0] - want) - (2.0 ** -11 * np.abs(want) + 2e-6 * 6 + sp.TINY[F16])
        assert over[clear].max() <= 0
