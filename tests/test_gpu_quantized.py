"""Quantised rows on the GPU: written codes and scales equal the 64-bit
restatement's bit for bit, reading back is exact, appends touch their rows
alone."""
import numpy as np
import pytest
import torch

from oracle import quantized as oq

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _np(t):
    return t.detach().cpu().double().numpy()


def _x(seed, *shape, dtype):
    """Blocks of unequal size, zeros and tiny values among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-12, 8, (*shape[:-1], 1), generator=g).float())
    x = x * torch.exp2(torch.randint(-6, 1, shape, generator=g).float())
    x[torch.rand(shape, generator=g) < 0.05] = 0.0
    if shape[2]:
        x[:, :, shape[2] // 2] = 0.0
    return x.to(dtype)


def _codes_equal(rows, want, S=None):
    codes, scales = want
    S = codes.shape[2] if S is None else S
    assert np.array_equal(rows.codes.cpu().numpy()[:, :, :S], codes[:, :, :S])
    assert np.array_equal(rows.scales.cpu().numpy()[..., :S], scales[..., :S])


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 3, 70, 128), (1, 1, 1, 128), (1, 2, 65, 64), (3, 2, 33, 96), (2, 1, 129, 40),
                                   (1, 2, 31, 1), (1, 1, 64, 31), (2, 2, 100, 80), (1, 4, 63, 127)])
def test_write_and_read(shape, dtype, fmt):
    from rotatek_amd.quantized import dequantize_rows, quantize_rows
    _say(f"write {shape} {dtype} {fmt}")
    x = _x(sum(shape), *shape, dtype=dtype)
    rows = quantize_rows(x.cuda(), fmt)
    torch.cuda.synchronize()
    want = oq.quantize(_np(x), fmt)
    _codes_equal(rows, want)
    vals = oq.values(*want, fmt, shape[-1])
    for dt in DTYPES:
        y = dequantize_rows(rows, dt)
        assert y.dtype == dt and torch.equal(y.cpu().double(), torch.from_numpy(vals).to(torch.float32).to(dt).double())


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_every_16_bit_value(fmt):
    """All fp16 and bf16 values, blocks of neighbours (an infinity or a NaN
    spoils its own block alone)."""
    from rotatek_amd.quantized import dequantize_rows, quantize_rows
    for dt in (torch.float16, torch.bfloat16):
        _say(f"every {dt} {fmt}")
        x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt).view(1, 1, 512, 128)
        rows = quantize_rows(x.cuda(), fmt)
        want = oq.quantize(_np(x), fmt)
        _codes_equal(rows, want)
        got = _np(dequantize_rows(rows, torch.float32))
        # bf16's largest values round up to 2^128 (17/16 steps from 1.9375 2^127
        # to the grid's 2^128), past fp32's largest: an infinity in fp32
        with np.errstate(over="ignore"):
            vals = oq.values(*want, fmt, 128).astype(np.float32)
        assert np.array_equal(got, vals, equal_nan=True)


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_strides(fmt):
    from rotatek_amd.quantized import MXRows, dequantize_rows, quantize_rows
    _say(f"strides {fmt}")
    base = _x(3, 2, 5, 70, 160, dtype=torch.bfloat16).cuda()
    for x in (base[:, 1:4, 3:60, 16:144], base[:, :, :, 1:128], base.transpose(1, 2)[..., :96], base[..., ::2],
              base[:1].expand(3, 5, 70, 160)[..., 32:64], base.transpose(2, 3)[..., :64]):
        rows = quantize_rows(x, fmt)
        _codes_equal(rows, oq.quantize(_np(x), fmt))
        # into a part of a larger buffer, and back into a strided one
        big = MXRows.empty(x.shape[0], x.shape[1], x.shape[2] + 100, x.shape[3], fmt)
        big.codes.fill_(0xA5)
        big.scales.fill_(0x5A)
        part = big.narrow(32, x.shape[2])
        quantize_rows(x, fmt, out=part)
        _codes_equal(part, oq.quantize(_np(x), fmt))
        S = x.shape[2]
        assert (big.codes[:, :, :32] == 0xA5).all() and (big.codes[:, :, 32 + S:] == 0xA5).all()
        assert (big.scales[..., :32] == 0x5A).all() and (big.scales[..., 32 + S:] == 0x5A).all()
        out = torch.full((*x.shape[:3], 2 * x.shape[3] + 1), 7.0, device="cuda")
        dequantize_rows(part, out=out[..., 1::2])
        assert torch.equal(out[..., 1::2], dequantize_rows(rows, torch.float32))
        assert (out[..., ::2] == 7.0).all()


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,advance", [(1, 128, True), (1, 64, False), (5, 80, True), (70, 128, True), (129, 40, False)])
def test_append(T, D, advance, dtype, fmt):
    from rotatek_amd.quantized import MXRows, append_rows
    _say(f"append T={T} D={D} {dtype} {fmt}")
    B, H, C = 5, 3, 150
    k, v = (MXRows.empty(B, H, C, D, fmt) for _ in range(2))
    for r in (k, v):
        r.codes.fill_(0x33)
        r.scales.fill_(0x44)
    start = [0, 7, C - 1, C, C - T if T < C else 3]
    lens = torch.tensor(start, dtype=torch.int32, device="cuda")
    kn, vn = _x(T, B, H, T, D, dtype=dtype), _x(T + 1, B, H, T, D, dtype=dtype)
    append_rows(kn.cuda(), vn.cuda(), k, v, lens, advance=advance)
    torch.cuda.synchronize()
    assert lens.tolist() == ([min(n + T, C) for n in start] if advance else start)
    for r, x in ((k, kn), (v, vn)):
        codes, scales = oq.quantize(_np(x), fmt)
        want_c = np.full(r.codes.shape, 0x33, np.uint8)
        want_s = np.full(r.scales.shape, 0x44, np.uint8)
        for b, n in enumerate(start):
            m = min(T, C - n)
            want_c[b, :, n:n + m] = codes[b, :, :m]
            want_s[b, :, :, n:n + m] = scales[b, :, :, :m]
        assert np.array_equal(r.codes.cpu().numpy(), want_c)
        assert np.array_equal(r.scales.cpu().numpy(), want_s)


def test_append_keys_alone_and_unequal_widths():
    from rotatek_amd.quantized import MXRows, append_rows, dequantize_rows
    _say("append keys alone")
    lens = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    k, v = MXRows.empty(2, 2, 40, 32), MXRows.empty(2, 2, 40, 128)
    kn, vn = _x(1, 2, 2, 2, 32, dtype=torch.bfloat16).cuda(), _x(2, 2, 2, 2, 128, dtype=torch.bfloat16).cuda()
    append_rows(kn, vn, k, v, lens, advance=False)
    append_rows(kn, None, k, None, lens)
    assert lens.tolist() == [5, 2]
    for r, x in ((k, kn), (v, vn)):
        want = torch.from_numpy(oq.values(*oq.quantize(_np(x), "mx8"), "mx8", x.shape[-1])).float()
        got = dequantize_rows(r, torch.float32).cpu()
        assert torch.equal(got[0, :, 3:5], want[0]) and torch.equal(got[1, :, :2], want[1])


def test_lengths_below_zero_and_past_the_capacity():
    from rotatek_amd.quantized import MXRows, append_rows
    _say("append odd lengths")
    k = MXRows.empty(3, 1, 10, 32)
    k.codes.zero_()
    k.scales.zero_()
    lens = torch.tensor([-5, 12, 9], dtype=torch.int32, device="cuda")
    append_rows(torch.ones(3, 1, 2, 32, device="cuda"), None, k, None, lens)
    torch.cuda.synchronize()
    assert lens.tolist() == [2, 10, 10]
    assert (k.codes[0, 0, :2] != 0).all() and (k.codes[0, 0, 2:] == 0).all()
    assert (k.codes[1] == 0).all()
    assert (k.codes[2, 0, 9] != 0).all() and (k.codes[2, 0, :9] == 0).all()


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_requests_far_apart(fmt):
    """Offsets between requests past 32 bits: write, append, read, attend."""
    from rotatek_amd.kernels import full_channel_decode_quantized
    from rotatek_amd.quantized import MXRows, append_rows, dequantize_rows, quantize_rows
    _say(f"far apart {fmt}")
    B, S, D, far = 3, 40, 128, 2200 * 2 ** 20
    near = MXRows.empty(B, 1, S, D, fmt)
    buf = torch.zeros(2 * far + 2 ** 14, dtype=torch.uint8, device="cuda")
    codes = buf.as_strided(near.codes.shape, (far, 0, near.codes.shape[3], 1))
    scales = buf.as_strided(near.scales.shape, (far, 0, 64, 1), 2 ** 13)
    rows = MXRows(codes, scales, D, fmt)
    x = _x(41, B, 1, S, D, dtype=torch.bfloat16).cuda()
    quantize_rows(x, fmt, out=near)
    assert quantize_rows(x, fmt, out=rows) is rows
    new = _x(42, B, 1, 3, D, dtype=torch.bfloat16).cuda()
    lens = torch.tensor([5, 0, 39], dtype=torch.int32, device="cuda")
    for r in (near, rows):
        append_rows(new, new, r, MXRows.empty(B, 1, S, D, fmt), lens, advance=False)
    assert torch.equal(rows.codes, near.codes) and torch.equal(rows.scales[..., :S], near.scales[..., :S])
    assert torch.equal(dequantize_rows(rows), dequantize_rows(near))
    q = torch.randn(B, 4, D, device="cuda").half()
    assert torch.equal(full_channel_decode_quantized(q, rows, rows, 4), full_channel_decode_quantized(q, near, near, 4))


def test_one_address_for_two_rows_is_refused():
    from rotatek_amd.kernels import full_channel_decode_quantized
    from rotatek_amd.quantized import MXRows, append_rows, dequantize_rows, quantize_rows
    _say("overlap")
    x = torch.randn(2, 1, 8, 32, device="cuda")
    one = MXRows.empty(1, 1, 8, 32)
    both = MXRows(one.codes.expand(2, 1, 8, 32), one.scales.expand(2, 1, 1, 32), 32)
    with pytest.raises(ValueError):
        quantize_rows(x, out=both)
    with pytest.raises(ValueError):
        append_rows(x, x, both, both, torch.zeros(2, dtype=torch.int32, device="cuda"))
    quantize_rows(x[:1], out=one)
    with pytest.raises(ValueError):
        dequantize_rows(both, out=torch.empty(1, 1, 8, 32, device="cuda").expand(2, 1, 8, 32))
    assert torch.equal(dequantize_rows(both)[0], dequantize_rows(one)[0])      # read, they may repeat
    q = torch.randn(2, 1, 32, device="cuda")
    with pytest.raises(ValueError):
        full_channel_decode_quantized(q, both, both, 1, out=torch.empty(1, 1, 32, device="cuda").expand(2, 1, 32))
    a, b = full_channel_decode_quantized(q, both, both, 1), full_channel_decode_quantized(q[1:], one, one, 1)
    assert torch.equal(a[1:], b)
