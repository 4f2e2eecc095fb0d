"""apply_rotary and append_pages against the oracle in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd.paged import append_pages
from rotatek_amd.rotary import apply_rotary, inverse_frequencies
from tests.paged import DTYPES, Pool, check, f64, half, rotation_bound

pytestmark = pytest.mark.gpu


def rand(g, *shape):
    return torch.randn(*shape, generator=g)


def batch_want(x, pos, freq, sections, interleaved, inverse=False):
    """x [B, H, T, D], pos [A, B, T]."""
    return np.stack([op.rotate(f64(x[b]).swapaxes(0, 1), pos[:, b].cpu().numpy(), freq.cpu().numpy(), sections, interleaved,
                               inverse).swapaxes(0, 1) for b in range(x.shape[0])])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("B, Hq, H, T, D, sections, interleaved", [
    (2, 7, 1, 5, 128, (16, 24, 24), False),
    (3, 4, 2, 1, 128, (24, 20, 20), True),
    (1, 1, 1, 1, 2, None, False),
    (2, 3, 3, 9, 80, (20, 20), True),
    (2, 5, 1, 4, 80, (8, 12), False),       # 40 channels are copied
    (1, 2, 1, 6, 127, (3, 0, 7, 1), True),  # odd head, four axes, one of none
    (1, 2, 2, 700, 96, (48,), False),
    (5, 2, 1, 601, 64, (5, 13, 14), False),  # four tokens a workgroup, the last one short
])
def test_rotary(dtype, B, Hq, H, T, D, sections, interleaved):
    g, dt = torch.Generator().manual_seed(B * T + D), DTYPES[dtype]
    P = sum(sections) if sections else D // 2
    q, k = rand(g, B, Hq, T, D).to(dt).cuda(), (5 * rand(g, B, H, T, D)).to(dt).cuda()
    A = len(sections) if sections else 1
    pos = torch.randint(0, 40000, (A, B, T), generator=g).cuda()
    freq = inverse_frequencies(2 * P)
    for positions in (pos, pos.int()):
        for inverse in (False, True):
            yq, yk = apply_rotary(q, k, positions, freq, sections, interleaved, inverse)
            for x, y in ((q, yq), (k, yk)):
                assert y.dtype == dt and y.shape == x.shape
                want = batch_want(x, pos, freq, sections or [P], interleaved, inverse)
                check(y, want, rotation_bound(f64(x), want, P, dt))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layouts_and_outputs(dtype):
    """Slices of one projection, tokens ahead of heads, in place, broadcast
    positions, outputs with strides of their own, no Keys."""
    g, dt = torch.Generator().manual_seed(1), DTYPES[dtype]
    B, T, Hq, H, D, P = 2, 11, 4, 2, 40, 20
    qkv = rand(g, B, T, Hq + 2 * H, D).to(dt).cuda()
    q, k = qkv[:, :, :Hq].transpose(1, 2), qkv[:, :, Hq:Hq + H].transpose(1, 2)
    pos = torch.arange(T).expand(1, B, T).cuda()
    freq = inverse_frequencies(D)
    want = [batch_want(x, pos, freq, [P], False) for x in (q, k)]
    bound = [rotation_bound(f64(x), w, P, dt) for x, w in zip((q, k), want)]
    for y, w, b in zip(apply_rotary(q, k, pos[0], freq), want, bound):
        check(y, w, b)
    odd = torch.full((B, Hq, D, T + 1), 7.0, dtype=dt, device="cuda")
    yq, yk = apply_rotary(q, k, pos, freq, out=(odd.transpose(2, 3)[:, :, 1:], torch.empty_like(k)))
    check(odd.transpose(2, 3)[:, :, 1:], want[0], bound[0])
    assert (odd[..., 0] == 7).all() and yq.data_ptr() == odd.data_ptr() + odd.element_size()
    only, none = apply_rotary(q, None, pos, freq)
    assert none is None and torch.equal(only, yq)
    # tokens one after the other
    n3, k3 = apply_rotary(qkv[0, :, :Hq], qkv[0, :, Hq:Hq + H], pos[0, 0], freq)
    assert torch.equal(n3, yq[0].transpose(0, 1)) and torch.equal(k3, yk[0].transpose(0, 1))
    v = qkv[:, :, Hq + H:].clone()
    apply_rotary(q, k, pos, freq, out=(q, k))
    check(q, want[0], bound[0])
    check(k, want[1], bound[1])
    assert torch.equal(qkv[:, :, Hq + H:], v)


def test_far_positions_keep_their_angles():
    """At 2^30 an angle in 32 bits is off by 64; in 64 bits by less than 2^-20 of a radian."""
    pos = torch.tensor([[2 ** 30 + 1, 2 ** 30, 10 ** 6 + 3, -5]], device="cuda")
    x = torch.zeros(4, 1, 8, device="cuda")
    x[..., :4] = 1.0
    freq = inverse_frequencies(8)
    y, _ = apply_rotary(x, None, pos, freq)
    want = op.rotate(f64(x), pos.cpu().numpy(), freq.cpu().numpy())
    check(y, want, rotation_bound(f64(x), want, 4, torch.float32) + 2.0 ** -20)


def test_gradient_is_the_inverse():
    """<g, d rotate(x)> by differences in 64 bits against inverse(g): the rotation
    is linear, so a central difference is its product but for rounding."""
    g = torch.Generator().manual_seed(3)
    x, up = rand(g, 6, 2, 16).cuda(), rand(g, 6, 2, 16).cuda()
    pos, freq = torch.arange(6, device="cuda") * 97, inverse_frequencies(16)
    grad, _ = apply_rotary(up, None, pos, freq, inverse=True)
    d = np.random.default_rng(0).standard_normal(x.shape)
    p = pos.cpu().numpy()[None]
    f = freq.cpu().numpy()
    diff = (op.rotate(f64(x) + 1e-3 * d, p, f) - op.rotate(f64(x) - 1e-3 * d, p, f)) / 2e-3
    lhs, rhs = float((f64(up) * diff).sum()), float((f64(grad) * d).sum())
    bound = float((rotation_bound(f64(up), f64(grad), 8, torch.float32) * np.abs(d)).sum()) + 1e-9
    assert abs(lhs - rhs) <= bound


def test_empty_calls():
    f = inverse_frequencies(16)
    for shape in ((0, 2, 3, 16), (2, 2, 0, 16)):
        q, k = apply_rotary(torch.empty(shape, device="cuda"), None, torch.zeros(1, shape[0], shape[2], device="cuda",
                                                                                dtype=torch.int64), f)
        assert tuple(q.shape) == shape and k is None


# ------------------------------------------------------------------ append
def append_case(lens, new, H, Hq, D, page, dt, strided=False, seed=0, pages_more=0):
    pool = Pool(lens, H, D, page, dt, seed, strided=strided, fill=0.25, spare=3 + pages_more).cuda()
    g = torch.Generator().manual_seed(seed + 1)
    N = sum(new)
    starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    q, k, v = (rand(g, N, h, D).to(dt).cuda() for h in (Hq, H, H))
    return pool, starts, q, k, v


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lens, new, H, Hq, D, page, strided", [
    ([1, 8, 9, 40], [1, 1, 1, 1], 2, 6, 128, 8, False),
    ([5, 0, 17, 64, 33], [5, 0, 1, 20, 9], 1, 3, 64, 16, True),
    ([70, 130], [70, 2], 3, 3, 80, 64, False),
    ([700, 1900], [600, 1900], 2, 2, 40, 128, False),
    ([12, 3], [4, 3], 2, 2, 7, 8, False),           # odd heads: element by element
])
def test_append(dtype, lens, new, H, Hq, D, page, strided):
    dt = DTYPES[dtype]
    pool, starts, q, k, v = append_case(lens, new, H, Hq, D, page, dt, strided)
    N, P = sum(new), max(D // 4, 1)
    sections = (P - P // 3, P // 3)
    pos = torch.randint(0, 30000, (2, N), device="cuda")
    freq = inverse_frequencies(2 * P)
    k0, v0 = f64(pool.dk), f64(pool.dv)
    turned = op.rotate(f64(k), pos.cpu().numpy(), freq.cpu().numpy(), sections, True)
    bound = rotation_bound(f64(k), turned, P, dt)
    want_k, want_v = op.append(turned, f64(v), k0, v0, pool.table.numpy(), lens, starts.cpu().numpy())
    bound_k, _ = op.append(bound, bound, np.zeros_like(k0), np.zeros_like(k0), pool.table.numpy(), lens, starts.cpu().numpy())
    yq = append_pages(k, v, pool.dk, pool.dv, pool.dtable, pool.dlens, starts, pos, freq, sections, True, q)
    want_q = op.rotate(f64(q), pos.cpu().numpy(), freq.cpu().numpy(), sections, True)
    check(yq, want_q, rotation_bound(f64(q), want_q, P, dt))
    check(pool.dk, want_k, bound_k)      # nothing where no token went
    np.testing.assert_array_equal(f64(pool.dv), want_v)


def test_append_without_rotation_and_as_a_batch():
    dt, lens, T = torch.bfloat16, [9, 24, 3], 3
    pool, _, _, k, v = append_case(lens, [T] * 3, 2, 2, 64, 8, dt)
    k0, v0 = f64(pool.dk), f64(pool.dv)
    assert append_pages(k.view(3, T, 2, 64).transpose(1, 2), v.view(3, T, 2, 64).transpose(1, 2), pool.dk, pool.dv,
                        pool.dtable, pool.dlens) is None
    want = op.append(f64(k), f64(v), k0, v0, pool.table.numpy(), lens, None, T)
    np.testing.assert_array_equal(f64(pool.dk), want[0])
    np.testing.assert_array_equal(f64(pool.dv), want[1])
    # one token each, without starts, in place of q
    q = torch.randn(3, 4, 64, device="cuda").to(dt)
    pos, freq = torch.tensor([3, 4, 5], device="cuda"), inverse_frequencies(64)
    q0 = f64(q)
    r = append_pages(k[:3], v[:3], pool.dk, pool.dv, pool.dtable, pool.dlens, positions=pos, inv_freq=freq, q=q, q_out=q)
    assert r is q
    want_q = op.rotate(q0, pos.cpu().numpy()[None], freq.cpu().numpy())
    check(q, want_q, rotation_bound(q0, want_q, 32, dt))


def test_append_drops_what_has_no_place():
    """Lengths past the table and below the new tokens, page numbers of no page,
    tokens of no request: the pool keeps every other row."""
    dt = torch.float16
    pool = Pool([16, 16, 16], 1, 16, 8, dt, fill=0.5, per_more=0).cuda()
    pool.table[1, 1], pool.table[2, 0] = 99, -7
    pool.dtable.copy_(pool.table)
    lens = [20, 16, 2]      # past the table; a page of none; one of three tokens before the first position
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(14, 1, 16, device="cuda").to(dt) for _ in range(2))
    starts = torch.tensor([1, 7, 10, 13], dtype=torch.int32, device="cuda")
    k0, v0 = f64(pool.dk), f64(pool.dv)
    append_pages(k, v, pool.dk, pool.dv, pool.dtable, dl, starts)
    want = op.append(f64(k), f64(v), k0, v0, pool.table.numpy(), lens, starts.cpu().numpy())
    np.testing.assert_array_equal(f64(pool.dk), want[0])
    np.testing.assert_array_equal(f64(pool.dv), want[1])


def test_append_is_refused_gradients():
    pool, starts, q, k, v = append_case([3], [3], 1, 1, 16, 8, torch.float32)
    with pytest.raises(RuntimeError, match="no gradient"):
        append_pages(k.requires_grad_(), v, pool.dk, pool.dv, pool.dtable, pool.dlens, starts)
    with pytest.raises(RuntimeError, match="no gradient"):
        apply_rotary(k, None, torch.zeros(3, dtype=torch.int64, device="cuda"), torch.ones(8, device="cuda"))
    with torch.no_grad():
        apply_rotary(k, None, torch.zeros(3, dtype=torch.int64, device="cuda"), torch.ones(8, device="cuda"))
    with pytest.raises(ValueError, match="table"):
        append_pages(k.detach(), v, pool.dk, pool.dv, pool.dtable.long(), pool.dlens, starts)
    with pytest.raises(ValueError, match="starts"):
        append_pages(k.detach(), v, pool.dk, pool.dv, pool.dtable, pool.dlens, starts[:1])
    with pytest.raises(ValueError, match="lens"):
        append_pages(k.detach(), v, pool.dk, pool.dv, pool.dtable, pool.dlens.long(), starts)


def test_rounding_is_to_nearest():
    """Angle zero: every value comes back as it is."""
    for dt in DTYPES.values():
        x = torch.randn(3, 2, 64, device="cuda").to(dt)
        y, _ = apply_rotary(x, None, torch.zeros(3, dtype=torch.int64, device="cuda"), inverse_frequencies(64))
        assert torch.equal(x, y) and half(dt) > 0


def test_tensors_that_others_allocated():
    """Inference mode, and tensors whose memory is not from torch's allocator."""
    dt = torch.bfloat16
    q, k = torch.randn(5, 4, 64, device="cuda").to(dt), torch.randn(5, 2, 64, device="cuda").to(dt)
    pos, freq = torch.arange(5, device="cuda"), inverse_frequencies(64)
    want = apply_rotary(q, k, pos, freq)
    for x, y in ((torch.from_dlpack(q), torch.from_dlpack(k)), (q.view(torch.int16).view(dt), k[:, :, :])):
        assert all(torch.equal(a, b) for a, b in zip(apply_rotary(x, y, pos, freq), want))
    with torch.inference_mode():
        got = apply_rotary(q.clone(), k.clone(), pos, freq)
        assert all(a.is_inference() for a in got)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
