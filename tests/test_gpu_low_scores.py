"""Rows whose scores are finite and far below zero: the first maximum that a row
sees is then a long way under the zero that its sums start from.

Channel 0 carries the offset: 16 in the queries, -x in the Keys (or in delta_mu),
so that a token scores 16 x / sqrt(D) nats below its other channels' product.
The tolerance is the oracle's (``spans.tolerance``), whose `size` counts the
offset.
"""
import numpy as np
import pytest
import torch

import spans as sp

pytestmark = pytest.mark.gpu

D, DOWN = 128, [90.0, 100.0, 1000.0]


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _x(nats):
    return nats * D ** 0.5 / 16


def _q(g, B, Hq, dtype):
    q = sp.randn(g, B, Hq, D)
    q[..., 0] = 16
    return q.to(dtype)


def _keys(g, nats, low, *shape):
    """Keys whose tokens ``low`` score ``nats`` lower."""
    k = sp.randn(g, *shape)
    k[..., 0] = 0
    k[:, :, low, 0] = -_x(nats)
    return k


def _hold(x, fmt, dtype):
    if fmt != "plain":
        return sp.rows(x, fmt)
    x = x.to(dtype)
    return x.cuda(), sp.np64(x)


@pytest.mark.parametrize("nats", DOWN)
@pytest.mark.parametrize("fmt,dtype", [("mx8", torch.bfloat16), ("mx8", torch.float32), ("mx4", torch.float16),
                                       ("mx4", torch.float32)])
def test_dense_rows(fmt, dtype, nats):
    """All tokens low; only the waves' first blocks low; a length or a mask that
    leaves one token, or those of the first block."""
    from rotatek_amd.kernels import full_channel_decode_quantized
    _say(f"dense {fmt} {dtype} {nats}")
    g = torch.Generator().manual_seed(int(nats))
    B, H, G, S = 3, 2, 4, 300
    for low in (slice(None), slice(0, 128), slice(0, 32)):
        k, k64 = _hold(_keys(g, nats, low, B, H, S, D), fmt, dtype)
        v, v64 = _hold(sp.randn(g, B, H, S, D), fmt, dtype)
        q = _q(g, B, H * G, dtype)
        one = torch.zeros(B, S, dtype=torch.uint8)
        one[torch.arange(B), torch.tensor([0, 17, 31])] = 1
        for lens, mask in ((None, None), ([1, 20, 300], None), (None, one)):
            valid = np.ones((B, S), bool) if mask is None else mask.numpy().astype(bool)
            if lens is not None:
                valid = valid & (np.arange(S)[None] < np.array(lens)[:, None])
            out = full_channel_decode_quantized(
                q.cuda(), k, v, G, mask=None if mask is None else mask.cuda(),
                lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda"))
            sp.check(out, q, G, [dict(k=k64, v=v64, valid=valid)], fmt, dtype)


@pytest.mark.parametrize("nats", DOWN)
@pytest.mark.parametrize("S_f", [0, 1, 50])
@pytest.mark.parametrize("fmt,dtype", [("mx8", torch.bfloat16), ("mx8", torch.float16), ("mx4", torch.float32)])
def test_rotated_rows_by_their_means(fmt, dtype, S_f, nats):
    """q . delta_mu alone brings every token of the rotated span down."""
    from rotatek_amd.kernels import rotatek_decode_quantized
    _say(f"means {fmt} {dtype} {S_f} {nats}")
    g = torch.Generator().manual_seed(S_f + 7)
    B, H, G, Dk, S_v = 2, 2, 4, 32, 200
    R = torch.linalg.qr(torch.randn(B, H, D, D, generator=g))[0][..., :Dk].contiguous()
    R[:, :, 0] = 0
    dm = sp.randn(g, B, H, D, scale=0.5)
    dm[..., 0] = -_x(nats)
    R, dm, q = R.to(dtype), dm.to(dtype), _q(g, B, H * G, dtype)
    ks, ks64 = _hold(sp.randn(g, B, H, S_v, Dk), fmt, dtype)
    vs, vs64 = _hold(sp.randn(g, B, H, S_v, D), fmt, dtype)
    kf, kf64 = _hold(_keys(g, nats, slice(None), B, H, S_f, D), fmt, dtype)
    vf, vf64 = _hold(sp.randn(g, B, H, S_f, D), fmt, dtype)
    out, _, _ = rotatek_decode_quantized(q.cuda(), R.cuda(), dm.cuda(), kf, vf, None, ks, vs, G)
    sp.check(out, q, G, [dict(k=kf64, v=vf64), dict(k=ks64, v=vs64, R=sp.np64(R), dm=sp.np64(dm))], fmt, dtype)


@pytest.mark.parametrize("nats", DOWN)
@pytest.mark.parametrize("B", [3, 70])     # waves take tokens; waves take queries
@pytest.mark.parametrize("fmt,dtype", [("plain", torch.bfloat16), ("plain", torch.float16), ("mx8", torch.bfloat16),
                                       ("mx4", torch.float16), ("mx8", torch.float32)])
def test_shared_prefixes(fmt, dtype, B, nats):
    """The prefix low, the text low, both, a prefix of one token."""
    from rotatek_amd.kernels import shared_prefix_decode
    _say(f"shared {fmt} {dtype} {B} {nats}")
    g = torch.Generator().manual_seed(B)
    H, G = 1, 4
    q = _q(g, B, H * G, dtype)
    for S_p, low_p, low_s in ((200, slice(None), slice(0, 0)), (200, slice(0, 0), slice(None)),
                              (200, slice(None), slice(None)), (200, slice(0, 128), slice(0, 32)),
                              (1, slice(None), slice(None))):
        k, k64 = _hold(_keys(g, nats, low_p, 1, H, S_p, D), fmt, dtype)
        v, v64 = _hold(sp.randn(g, 1, H, S_p, D), fmt, dtype)
        k2, k264 = _hold(_keys(g, nats, low_s, B, H, 40, D), fmt, dtype)
        v2, v264 = _hold(sp.randn(g, B, H, 40, D), fmt, dtype)
        n = torch.tensor([[40, 0, 1, 33][b % 4] for b in range(B)], dtype=torch.int32)
        valid = np.arange(40)[None] < n.numpy()[:, None]
        out = shared_prefix_decode(q.cuda(), k, v, k2, v2, G, len_suffix=n.cuda())
        prefix = dict(k=k64, v=v64, valid=np.ones((B, S_p), bool))
        sp.check(out, q, G, [prefix, dict(k=k264, v=v264, valid=valid)], fmt, dtype)
        sp.check(shared_prefix_decode(q.cuda(), k, v, None, None, G), q, G, [prefix], fmt, dtype)


@pytest.mark.parametrize("B", [3, 70])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shared_rotated_rows_by_their_means(B, dtype):
    from rotatek_amd.kernels import shared_prefix_decode
    _say(f"shared means {B} {dtype}")
    g = torch.Generator().manual_seed(B)
    H, G, Dk, S_v, S_p = 1, 4, 32, 150, 30
    R = torch.linalg.qr(torch.randn(1, H, D, D, generator=g))[0][..., :Dk].contiguous()
    R[:, :, 0] = 0
    dm = sp.randn(g, 1, H, D, scale=0.5)
    dm[..., 0] = -_x(500.0)
    R, dm, q = R.to(dtype), dm.to(dtype), _q(g, B, H * G, dtype)
    ks, ks64 = _hold(sp.randn(g, 1, H, S_v, Dk), "plain", dtype)
    vs, vs64 = _hold(sp.randn(g, 1, H, S_v, D), "plain", dtype)
    for S in (0, S_p):
        k, k64 = _hold(_keys(g, 500.0, slice(None), 1, H, S, D), "plain", dtype)
        v, v64 = _hold(sp.randn(g, 1, H, S, D), "plain", dtype)
        out = shared_prefix_decode(q.cuda(), k, v, None, None, G, R_partial=R.cuda(), delta_mu=dm.cuda(), k_sparse=ks,
                                   v_sparse=vs)
        sp.check(out, q, G, [dict(k=k64, v=v64), dict(k=ks64, v=vs64, R=sp.np64(R), dm=sp.np64(dm))], "plain", dtype)
