"""CPU checks of the quantised and shared-prefix entry points: refusals come
from the host, before any HIP call, and the plan's workspace is sane."""
import ctypes

import pytest
import torch

from rotatek_amd import _lib
from rotatek_amd.kernels._span import rows_of
from rotatek_amd.quantized import MXRows, append_rows, dequantize_rows, quantize_rows

MX8, MX4 = _lib.RK_ROWS_MX8, _lib.RK_ROWS_MX4
ref = _lib.ref


def _rows(B=2, H=2, S=64, D=128, fmt="mx8"):
    r = MXRows.empty(B, H, S, D, fmt, device="cpu")
    # aligned like device memory
    r.codes = _aligned(r.codes.shape)
    r.scales = _aligned(r.scales.shape)
    return r


def _aligned(shape, dtype=torch.uint8):
    n = 1
    for s in shape:
        n *= s
    el = torch.tensor([], dtype=dtype).element_size()
    buf = torch.zeros(n * el + 256, dtype=torch.uint8)
    at = -buf.data_ptr() % 256
    return buf[at:at + n * el].view(dtype).view(shape)


def _decode(q=None, R=None, dm=None, kf=None, vf=None, mask=None, ks=None, vs=None, G=2, out=None, cus=256):
    n = ctypes.c_size_t(0)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16) if q is None else q
    kf, vf = _rows() if kf is None else kf, _rows() if vf is None else vf
    d = [_lib.desc(t) for t in (q, R, dm)]
    do, dk = _lib.desc(out), _lib.desc(mask)
    dr = [rows_of(x) for x in (kf, vf, ks, vs)]
    st = _lib.load().rk_quantized_decode_check(*[ref(x) for x in d], ref(dr[0]), ref(dr[1]), ref(dk), ref(dr[2]),
                                               ref(dr[3]), G, ref(do), cus, ctypes.byref(n))
    return st, n.value


def _shared(q, kp, vp, ks=None, vs=None, k2=None, v2=None, R=None, dm=None, G=2, out=None, cus=256):
    n = ctypes.c_size_t(0)
    d = [_lib.desc(t) for t in (q, R, dm)]
    do = _lib.desc(out)
    dr = [rows_of(x) for x in (kp, vp, ks, vs, k2, v2)]
    st = _lib.load().rk_shared_prefix_decode_check(*[ref(x) for x in d], *[ref(x) for x in dr], G, ref(do), cus,
                                                   ctypes.byref(n))
    return st, n.value


def test_decode_accepts_and_sizes_its_workspace():
    st, n = _decode()
    assert st == 0 and 0 < n < 1 << 20
    R, dm = torch.zeros(2, 2, 128, 40), torch.zeros(2, 2, 128)
    st, m = _decode(R=R, dm=dm, ks=_rows(D=40, S=500), vs=_rows(S=500))
    assert st == 0 and m > n
    # more tokens never need less; the split follows sizes alone
    last = 0
    for S in (1, 100, 1000, 10000):
        st, m = _decode(kf=_rows(S=S), vf=_rows(S=S))
        assert st == 0 and m >= last
        last = m


def test_decode_refusals():
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    assert _decode(q=q[0])[0] == _lib.RK_ERR_RANK
    assert _decode(q=q.int())[0] == _lib.RK_ERR_DTYPE
    assert _decode(q=q.double())[0] == _lib.RK_ERR_DTYPE
    assert _decode(q=q[:1])[0] == _lib.RK_ERR_SHAPE
    assert _decode(q=q[..., :64])[0] == _lib.RK_ERR_SHAPE
    assert _decode(q=torch.zeros(2, 4, 129))[0] == _lib.RK_ERR_HEAD_DIM
    assert _decode(G=3)[0] == _lib.RK_ERR_HEADS
    assert _decode(G=0)[0] == _lib.RK_ERR_ARG
    assert _decode(q=torch.zeros(2, 5, 128))[0] == _lib.RK_ERR_HEADS
    assert _decode(vf=_rows(S=63))[0] == _lib.RK_ERR_SHAPE
    assert _decode(vf=_rows(fmt="mx4"))[0] == _lib.RK_ERR_DTYPE
    assert _decode(kf=torch.zeros(2, 2, 64, 128, dtype=torch.bfloat16))[0] == _lib.RK_ERR_DTYPE
    assert _decode(mask=torch.zeros(2, 63, dtype=torch.uint8))[0] == _lib.RK_ERR_SHAPE
    assert _decode(mask=torch.zeros(2, 64, dtype=torch.int32))[0] == _lib.RK_ERR_DTYPE
    assert _decode(out=torch.zeros(2, 4, 128))[0] == _lib.RK_ERR_DTYPE
    assert _decode(out=q[:, :3])[0] == _lib.RK_ERR_SHAPE
    assert _decode(cus=-1)[0] == _lib.RK_ERR_ARG
    ks, vs, R = _rows(D=32, S=96), _rows(S=96), torch.zeros(2, 2, 128, 32)
    assert _decode(ks=ks, vs=vs)[0] == _lib.RK_ERR_NULL                 # no rotation
    assert _decode(R=R, ks=ks)[0] == _lib.RK_ERR_NULL                   # Keys without Values
    assert _decode(R=R[..., :31], ks=ks, vs=vs)[0] == _lib.RK_ERR_SHAPE
    assert _decode(R=R[:1], ks=ks, vs=vs)[0] == _lib.RK_ERR_SHAPE
    assert _decode(R=R, dm=torch.zeros(2, 2, 127), ks=ks, vs=vs)[0] == _lib.RK_ERR_SHAPE
    assert _decode(R=R, ks=ks, vs=_rows(S=95))[0] == _lib.RK_ERR_SHAPE
    assert _decode(R=R, ks=_rows(D=32, S=96, fmt="mx4"), vs=vs)[0] == _lib.RK_ERR_DTYPE


def test_row_layout_refusals():
    r = _rows()
    r.codes = r.codes.transpose(2, 3)[:, :, :, :64].transpose(2, 3)[..., ::2]
    assert _decode(kf=r)[0] == _lib.RK_ERR_SHAPE
    r = _rows()
    r.codes = _aligned((2, 2, 64, 136))[..., :128]          # rows off 16 bytes
    assert _decode(kf=r)[0] == _lib.RK_ERR_STRIDE
    r = _rows()
    r.codes = _aligned((2 * 2 * 64 * 128 + 16,))[8:-8].view(2, 2, 64, 128)
    assert _decode(kf=r)[0] == _lib.RK_ERR_STRIDE
    r = _rows(S=65)
    r.scales = r.scales[..., :65]                           # not padded to whole groups
    assert _decode(kf=r, vf=_rows(S=65))[0] == _lib.RK_ERR_SHAPE
    r = _rows()
    r.scales = _aligned((2, 2, 4, 68))[..., :64]
    assert _decode(kf=r)[0] == _lib.RK_ERR_STRIDE
    r = _rows()
    r.scales = r.scales.float()
    assert _decode(kf=r)[0] == _lib.RK_ERR_DTYPE
    # a head that 32-bit offsets do not span
    d = rows_of(_rows(B=1, H=1, S=64))
    d.data.shape[2] = d.scales.shape[3] = (1 << 24) + 64
    dq, n = _lib.desc(torch.zeros(1, 2, 128)), ctypes.c_size_t(0)
    assert _lib.load().rk_quantized_decode_check(ref(dq), None, None, ref(d), ref(d), None, None, None, 2, None, 256,
                                                 ctypes.byref(n)) == _lib.RK_ERR_STRIDE
    d.format = 7
    assert _lib.load().rk_quantized_decode_check(ref(dq), None, None, ref(d), ref(d), None, None, None, 2, None, 256,
                                                 ctypes.byref(n)) == _lib.RK_ERR_ARG


def test_shared_prefix_refusals():
    bf = torch.bfloat16
    q = torch.zeros(3, 4, 128, dtype=bf)
    p, t = torch.zeros(1, 2, 100, 128, dtype=bf), torch.zeros(3, 2, 20, 128, dtype=bf)
    assert _shared(q, p, p, k2=t, v2=t)[0] == 0
    assert _shared(q, p, p)[0] == 0
    assert _shared(q, t, t)[0] == _lib.RK_ERR_SHAPE                       # a prefix of its own per request
    assert _shared(q, p, p, k2=t)[0] == _lib.RK_ERR_NULL
    assert _shared(q, p, p, k2=t[:2], v2=t[:2])[0] == _lib.RK_ERR_SHAPE
    assert _shared(q, p, p, k2=t, v2=t[:, :, :19])[0] == _lib.RK_ERR_SHAPE
    assert _shared(q.half(), p, p)[0] == _lib.RK_ERR_DTYPE
    assert _shared(q.float(), p.float(), p.float())[0] == _lib.RK_ERR_DTYPE
    m = _rows(B=1, S=100)
    assert _shared(q, m, m)[0] == 0 and _shared(q.float(), m, m)[0] == 0
    assert _shared(q, m, m, k2=t, v2=t)[0] == _lib.RK_ERR_DTYPE           # one format for all spans
    R, ks, vs = torch.zeros(1, 2, 128, 32), torch.zeros(1, 2, 50, 32, dtype=bf), torch.zeros(1, 2, 50, 128, dtype=bf)
    assert _shared(q, p, p, ks=ks, vs=vs, R=R, dm=torch.zeros(1, 2, 128))[0] == 0
    assert _shared(q, p, p, ks=ks, vs=vs, R=R.expand(3, 2, 128, 32))[0] == _lib.RK_ERR_SHAPE
    assert _shared(q, p, p, ks=ks, vs=vs, R=R, dm=torch.zeros(3, 2, 128))[0] == _lib.RK_ERR_SHAPE
    big = torch.zeros(1, 1, 1, 128, dtype=bf).expand(1, 2, 1 << 24, 128)
    d = [rows_of(big) for _ in range(2)]
    for x in d:
        x.data.stride[2] = 128
    dq, n = _lib.desc(q), ctypes.c_size_t(0)
    assert _lib.load().rk_shared_prefix_decode_check(ref(dq), None, None, ref(d[0]), ref(d[1]), None, None, None, None,
                                                     2, None, 256, ctypes.byref(n)) == _lib.RK_ERR_STRIDE


def test_launch_entries_refuse_before_the_device():
    """Workspace and pointer errors of the launching entries, without a GPU."""
    lib = _lib.load()
    q = torch.zeros(1, 2, 128)
    dq, do, dr = _lib.desc(q), _lib.desc(q), rows_of(_rows(B=1, H=1))
    null = rows_of(_rows(B=1, H=1))
    null.data.data = None
    args = (None, None, ref(null), ref(dr), None, None, None, None, 2, ref(do), None, 0, None)
    assert lib.rk_quantized_decode(ref(dq), *args) == _lib.RK_ERR_NULL
    if not torch.cuda.is_available():
        args = (None, None, ref(dr), ref(dr), None, None, None, None, 2, ref(do), None, 0, None)
        assert lib.rk_quantized_decode(ref(dq), *args) == _lib.RK_ERR_NO_DEVICE


def test_write_read_and_append_refusals():
    lib = _lib.load()
    x = _aligned((2, 2, 64, 128), torch.bfloat16)
    r = _rows()

    def write(t, rows):
        dt, dr = _lib.desc(t), rows.desc()
        return lib.rk_mx_write(ref(dt), ref(dr), None)

    assert write(x[0], r) == _lib.RK_ERR_RANK
    assert write(x.to(torch.int32), r) == _lib.RK_ERR_DTYPE
    assert write(x.double(), r) == _lib.RK_ERR_DTYPE
    assert write(x[:, :, :63], r) == _lib.RK_ERR_SHAPE
    assert write(x[..., :96], r) == _lib.RK_ERR_SHAPE
    assert write(torch.zeros(2, 2, 64, 129), r) == _lib.RK_ERR_HEAD_DIM
    dx, plain = _lib.desc(x), rows_of(x)
    assert lib.rk_mx_write(ref(dx), ref(plain), None) == _lib.RK_ERR_ARG
    assert lib.rk_mx_read(ref(plain), ref(dx), None) == _lib.RK_ERR_ARG
    assert lib.rk_mx_write(None, ref(plain), None) == _lib.RK_ERR_NULL

    lens = torch.zeros(2, dtype=torch.int32)

    def append(k, v, kr, vr, n=lens):
        d = [_lib.desc(k), _lib.desc(v), kr.desc(), None if vr is None else vr.desc()]
        return lib.rk_mx_append(*[ref(t) for t in d], None if n is None else n.data_ptr(), 1, None)

    t = x[:, :, :1]
    assert append(t, t, r, None) == _lib.RK_ERR_NULL
    assert append(t, t, r, r, None) == _lib.RK_ERR_NULL
    assert append(t, x[:, :, :2], r, r) == _lib.RK_ERR_SHAPE
    assert append(t, t.half(), r, r) == _lib.RK_ERR_DTYPE
    assert append(t, t, r, _rows(fmt="mx4")) == _lib.RK_ERR_DTYPE
    assert append(t, t, r, _rows(S=32)) == _lib.RK_ERR_SHAPE
    assert append(t[:1], t[:1], r, r) == _lib.RK_ERR_SHAPE


def test_python_refusals():
    x = torch.zeros(1, 2, 5, 128)
    with pytest.raises(ValueError):
        quantize_rows(x, "mx6")
    with pytest.raises(ValueError):
        quantize_rows(x[0], "mx8")
    with pytest.raises(RuntimeError):
        quantize_rows(x, "mx8")                      # not on a GPU
    with pytest.raises(RuntimeError):
        dequantize_rows(_rows())
    with pytest.raises(ValueError):
        append_rows(x, None, _rows(), _rows(), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        MXRows.empty(1, 1, 1, 129, device="cpu")
    r = _rows(S=70)
    for start, n in ((16, 10), (0, 71), (64, 7), (-32, 5)):
        with pytest.raises(ValueError):
            r.narrow(start, n)
    assert r.narrow(32, 38).shape == (2, 2, 38, 128)
    from rotatek_amd.kernels import full_channel_decode_quantized, shared_prefix_decode
    q = torch.zeros(1, 2, 128)
    with pytest.raises(ValueError):
        full_channel_decode_quantized(q, x, x)
    with pytest.raises(ValueError):
        full_channel_decode_quantized(q[0], _rows(), _rows())
    with pytest.raises(ValueError):
        shared_prefix_decode(q, x, x, x, None, 1)
    with pytest.raises(ValueError):
        shared_prefix_decode(q, x, x, None, None, 1, k_sparse=x)
    with pytest.raises(RuntimeError):
        shared_prefix_decode(q, x, x, None, None, 1)
    with pytest.raises(ValueError):
        shared_prefix_decode(q, x, x, None, None, 1, delta_mu=torch.zeros(1, 2, 128))
    with pytest.raises(ValueError):
        shared_prefix_decode(q, x, x, None, None, 1, len_suffix=torch.zeros(1, dtype=torch.int32))


def test_outputs_that_repeat_are_refused():
    x = _aligned((2, 2, 64, 128), torch.bfloat16)
    q, r = torch.zeros(2, 4, 128, dtype=torch.bfloat16), _rows()
    assert _decode(q, out=q)[0] == 0
    assert _decode(q, out=q[:1].expand(2, 4, 128))[0] == _lib.RK_ERR_STRIDE
    assert _decode(q, out=q[:, :1].expand(2, 4, 128))[0] == _lib.RK_ERR_STRIDE
    once = MXRows(r.codes[:1].expand(2, 2, 64, 128), r.scales[:1].expand(2, 2, 4, 64), 128)
    assert _decode(q, kf=once, vf=once)[0] == 0         # read, rows may repeat
    dx, dr = _lib.desc(x), once.desc()
    lens = torch.zeros(2, dtype=torch.int32)
    lib = _lib.load()
    assert lib.rk_mx_write(ref(dx), ref(dr), None) == _lib.RK_ERR_STRIDE
    assert lib.rk_mx_append(ref(dx), None, ref(dr), None, lens.data_ptr(), 1, None) == _lib.RK_ERR_STRIDE
    dx, dr = _lib.desc(x[:1].expand(2, 2, 64, 128)), r.desc()
    assert lib.rk_mx_read(ref(dr), ref(dx), None) == _lib.RK_ERR_STRIDE


def test_sizes_past_a_launch_are_refused():
    bf = torch.bfloat16
    lib, n = _lib.load(), ctypes.c_size_t(0)
    # rows that repeat by stride 0 can be any number
    p = torch.zeros(1, 1, 1, 128, dtype=bf).expand(1, 2, 1 << 31, 128)
    q = torch.zeros(3, 4, 128, dtype=bf)
    assert _shared(q, p, p)[0] == _lib.RK_ERR_SHAPE
    assert _shared(q, p[:, :, :1 << 20], p[:, :, :1 << 20])[0] == 0
    p = torch.zeros(1, 2, 8, 128, dtype=bf)
    many = torch.zeros(1, 4, 128, dtype=bf).expand(1 << 24, 4, 128)
    assert _shared(many, p, p)[0] == _lib.RK_ERR_SHAPE
    st, size = _shared(many[:1 << 20], p, p)
    assert st == 0 and size < 1 << 34
    r = _rows(B=1)
    wide = MXRows(r.codes.expand(1 << 24, 2, 64, 128), r.scales.expand(1 << 24, 2, 4, 64), 128)
    assert _decode(many, kf=wide, vf=wide)[0] == _lib.RK_ERR_SHAPE
    x = torch.zeros(1, 1, 1, 128).expand(1 << 23, 2, 64, 128)
    part = MXRows(wide.codes[:1 << 23], wide.scales[:1 << 23], 128)
    dx, dr = _lib.desc(x), part.desc()
    assert lib.rk_mx_write(ref(dx), ref(dr), None) == _lib.RK_ERR_SHAPE
    assert lib.rk_mx_read(ref(dr), ref(dx), None) == _lib.RK_ERR_SHAPE


@pytest.mark.parametrize("cus", [1, 64, 256, 304])
def test_every_plan_is_bounded(cus):
    """Workspace over sizes, batch and formats: never more than a record for 512
    KB of rows, 32 per CU and one a unit and span."""
    for dtype, fmt in ((torch.bfloat16, "plain"), (torch.float16, "mx8"), (torch.float32, "mx4")):
        for B in (1, 3, 64, 1000):
            for S in (0, 1, 31, 33, 4096, 100000):
                for S_s in (None, 1, 300, 9000):
                    q = torch.zeros(1, 8, 128, dtype=dtype).expand(B, 8, 128)
                    if fmt == "plain":
                        p = torch.zeros(1, 1, 1, 128, dtype=dtype).expand(1, 2, S, 128)
                        t = None if S_s is None else p.new_zeros(1, 1, 1, 128).expand(B, 2, S_s, 128)
                    else:
                        p = _rows(B=1, S=S, fmt=fmt)
                        t = None
                        if S_s is not None:
                            t = _rows(B=1, S=S_s, fmt=fmt)
                            t = MXRows(t.codes.expand(B, *t.codes.shape[1:]), t.scales.expand(B, *t.scales.shape[1:]), 128,
                                       fmt)
                    st, size = _shared(q, p, p, k2=t, v2=t, G=4, cus=cus)
                    assert st == 0
                    units = 2 * (B + -(-4 * B // 16))
                    rows_bytes = 512 * (S * 2 * -(-4 * B // 16) + (S_s or 0) * 2 * B)
                    records = 64 * (2 * units + 32 * cus + rows_bytes // (1 << 18))
                    assert size <= records * (128 * 4 + 8) + 4096 + B * 8 * 128 * 8, (B, S, S_s, size)
