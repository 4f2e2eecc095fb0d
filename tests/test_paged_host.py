"""Paged cache on the host: the oracle's own pins, the index code that the
kernels compile, what the entry points refuse, and PagedCache's counts."""
import ctypes
import os
import random
import shutil
import subprocess

import numpy as np
import pytest
import torch

from oracle import paged as op
from rotatek_amd import _lib
from rotatek_amd.paged_cache import PagedCache
from rotatek_amd.rotary import inverse_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------- oracle
def test_oracle_rotation_is_a_rotation():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 2, 12))
    f = np.array([1.0, 0.3, 0.1, 0.01])
    pos = rng.integers(0, 1000, (2, 5))
    y = op.rotate(x, pos, f, [1, 3], True)
    np.testing.assert_allclose(np.hypot(y[..., :4], y[..., 4:8]), np.hypot(x[..., :4], x[..., 4:8]), rtol=1e-12)
    np.testing.assert_array_equal(y[..., 8:], x[..., 8:])
    np.testing.assert_allclose(op.rotate(y, pos, f, [1, 3], True, inverse=True), x, atol=1e-12)
    # scores go by the distance alone, for one axis
    a, b = x[:, :1], x[:, 1:]
    s = [(op.rotate(a, p, f) * op.rotate(b, p + 7, f)).sum(-1) for p in (pos[:1], pos[:1] + 123)]
    np.testing.assert_allclose(s[0], s[1], atol=1e-10)


@pytest.mark.parametrize("sections, want", [([2, 3, 1], [0, 1, 2, 0, 1, 1]), ([0, 2], [1, 1]), ([3], [0, 0, 0])])
def test_oracle_pairs_dealt_in_turn(sections, want):
    assert op.axis_of(sections, True) == want
    assert op.axis_of(sections, False) == [a for a, n in enumerate(sections) for _ in range(n)]


def test_oracle_attention_by_hand():
    k = np.zeros((1, 6, 2))
    v = np.arange(12.0).reshape(1, 6, 2)
    q = np.ones((3, 1, 2))
    there = np.array([True] * 5 + [False])
    out, _, _ = op.attend(q, k, v, there, 3, 1, window=2, sinks=1)
    np.testing.assert_allclose(out[0, 0], v[0, [0, 2, 3]].mean(0))
    np.testing.assert_allclose(out[1, 0], v[0, [0, 3, 4]].mean(0))
    np.testing.assert_allclose(out[2, 0], v[0, [0, 4]].mean(0))     # the last token is not there
    out, _, _ = op.attend(q, k, v, there, -1, 1)
    np.testing.assert_array_equal(out[0, 0], 0.0)


# -------------------------------------------------------------- index code
SHIM = r"""
#include "rk_page_map.h"
using namespace rk;
extern "C" void place(const int32_t* table, long t_sb, const int32_t* lens, const int32_t* starts, int B, int per,
                      int pages, int shift, int each, long n, long* page, int* row) {
  PageMap m{table, lens, starts, t_sb, B, per, pages, each, shift, per << shift};
  *page = place_of(m, n, starts ? request_of(starts, B, n) : 0, row);
}
extern "C" int length(const int32_t* lens, int b, int cap) {
  PageMap m{nullptr, lens, nullptr, 0, 0, 0, 0, 0, 31, cap};
  return len_of(m, b);
}
// marks every token that the blocks cover (2 if covered twice); returns the blocks
extern "C" int cover(int lo, int hi, int window, int sinks, int* mark, int most) {
  const Seen<32> s(lo, hi, window, sinks);
  for (int i = 0; i < s.blocks; ++i)
    for (int j = s.token(i); j < s.token(i) + 32 && j < most; ++j) ++mark[j];
  return s.blocks;
}
extern "C" int visible(int p, int j, int window, int sinks) { return sees(p, j, window, sinks); }
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("shim")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT}/rotatek_amd/csrc", str(d / "shim.cpp"), "-o",
                    str(d / "shim.so")], check=True)
    return ctypes.CDLL(str(d / "shim.so"))


def ptr(a):
    return None if a is None else a.ctypes.data_as(ctypes.c_void_p)


def place(shim, n, table, lens, starts, page, pages, each=1):
    pg, row = ctypes.c_long(-7), ctypes.c_int(-7)
    shim.place(ptr(table), ctypes.c_long(table.strides[0] // 4), ptr(lens), ptr(starts), table.shape[0], table.shape[1],
               pages, page.bit_length() - 1, each, ctypes.c_long(n), ctypes.byref(pg), ctypes.byref(row))
    return None if pg.value < 0 else (pg.value, row.value)


@pytest.mark.parametrize("seed", range(6))
def test_places_of_new_tokens(shim, seed):
    """Lengths below zero and past the table, page numbers that are none, empty
    requests, tokens of no request: nowhere, or where the oracle says."""
    rng = random.Random(seed)
    B, page, per, pages = rng.randint(1, 7), rng.choice([8, 16, 64]), rng.randint(1, 5), 9
    table = np.array([[rng.choice([-1, -2 ** 31, 9, 2 ** 31 - 1, *range(9)]) for _ in range(per)] for _ in range(B)],
                     dtype=np.int32)
    lens = np.array([rng.choice([0, -5, 2 ** 31 - 1, -2 ** 31, rng.randint(0, per * page + 9)]) for _ in range(B)],
                    dtype=np.int32)
    starts = np.cumsum([rng.randint(0, 3)] + [rng.choice([0, 1, rng.randint(0, 30)]) for _ in range(B)]).astype(np.int32)
    for n in range(int(starts[-1]) + 5):
        assert place(shim, n, table, lens, starts, page, pages) == op.place(n, table, lens, starts, page, pages)
    for each in (1, 3):
        for n in range(B * each):
            assert place(shim, n, table, lens, None, page, pages, each) == \
                op.place(n, table, lens, None, page, pages, each)


@pytest.mark.parametrize("starts", [[5, 3, 9, 2], [0, 0, 0, 0], [9, 9, 9, 9], [-4, 2, 2, 40], [2 ** 31 - 1, -2 ** 31, 0, 1]])
def test_starts_that_do_not_ascend_stay_inside(shim, starts):
    """Whatever they say, a token goes to a row of a page of the table, or nowhere."""
    table = np.arange(6, dtype=np.int32).reshape(3, 2)
    lens = np.array([16, 3, 9], dtype=np.int32)
    for n in range(12):
        at = place(shim, n, table, lens, np.array(starts, dtype=np.int32), 8, 6)
        assert at is None or (0 <= at[0] < 6 and 0 <= at[1] < 8)


def test_lengths_are_cut(shim):
    lens = np.array([-2 ** 31, -1, 0, 5, 64, 65, 2 ** 31 - 1], dtype=np.int32)
    assert [shim.length(ptr(lens), b, 64) for b in range(7)] == [0, 0, 0, 5, 64, 64, 64]


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 1, 4, 32, 33, 90, 2 ** 31 - 1])
def test_blocks_cover_what_is_seen_once(shim, window, sinks):
    for lo, hi in ((0, 0), (0, 31), (0, 32), (5, 5), (64, 64), (63, 90), (100, 130), (150, 150), (0, -1), (7, -1)):
        most = 192
        mark = np.zeros(most, dtype=np.int32)
        blocks = shim.cover(lo, hi, window, sinks, ptr(mark), most)
        assert mark.max() <= 1
        if hi < 0:
            assert blocks == 0
            continue
        seen = [j for j in range(most) for p in (lo, hi) if shim.visible(p, j, window, sinks)]
        want = [j for j in range(most) for p in (lo, hi) if j <= p and (p - j < window or j < sinks)]
        assert seen == want and all(mark[j] for j in seen)
        # no more than the window's and the sinks' blocks
        assert blocks <= (min(window, hi + 1) + hi - lo + 62) // 32 + 1 + -(-min(sinks, hi + 1) // 32)


# ---------------------------------------------------------------- refusals
NEVER = ctypes.c_void_p(0x1000)    # a pointer that no refused call follows


def desc(shape, dtype=_lib.RK_BF16, stride=None, data=0x1000):
    d = _lib.RkTensor()
    d.data, d.dtype, d.ndim = data, dtype, len(shape)
    if stride is None:
        stride, n = [], 1
        for s in reversed(shape):
            stride.insert(0, n)
            n *= s
    for i, (a, b) in enumerate(zip(shape, stride)):
        d.shape[i], d.stride[i] = a, b
    return d


def pool(pages=4, heads=2, page=16, dim=64, requests=3, per=2, dtype=_lib.RK_BF16, **more):
    p = _lib.RkPages()
    p.k = desc((pages, heads, page, dim), dtype, more.get("stride"))
    p.v = desc((more.get("v_pages", pages), heads, page, dim), more.get("v_dtype", dtype))
    p.table = desc((requests, per), more.get("table_dtype", _lib.RK_I32), more.get("table_stride"))
    p.lens = 0x1000
    return p


def attention(q=None, p=None, groups=2, window=0, sinks=0, out=None, starts=None):
    p = p or pool()
    q = q or desc((3, 4, 64))
    need = ctypes.c_size_t(0)
    return _lib.load().rk_paged_attention_check(ctypes.byref(q), starts, ctypes.byref(p), groups, window, sinks,
                                                None if out is None else ctypes.byref(out), 256, ctypes.byref(need))


def test_attention_takes():
    assert attention() == 0
    assert attention(q=desc((7, 4, 64)), starts=NEVER) == 0
    assert attention(window=2 ** 40, sinks=2 ** 40) == 0
    assert attention(q=desc((3, 4, 64), stride=(1, 192, 3))) == 0
    assert attention(q=desc((0, 4, 64)), p=pool(requests=0)) == 0


@pytest.mark.parametrize("call, status", [
    (dict(q=desc((2, 4, 64))), _lib.RK_ERR_SHAPE),                       # one token of every request
    (dict(q=desc((3, 4, 64, 1))), _lib.RK_ERR_RANK),
    (dict(q=desc((3, 5, 64))), _lib.RK_ERR_HEADS),
    (dict(groups=0), _lib.RK_ERR_HEADS),
    (dict(groups=-2), _lib.RK_ERR_HEADS),
    (dict(q=desc((3, 4, 60)), p=pool(dim=60)), _lib.RK_ERR_HEAD_DIM),
    (dict(q=desc((3, 4, 136)), p=pool(dim=136)), _lib.RK_ERR_HEAD_DIM),
    (dict(q=desc((3, 4, 32))), _lib.RK_ERR_HEAD_DIM),
    (dict(q=desc((3, 4, 64), _lib.RK_F16)), _lib.RK_ERR_DTYPE),
    (dict(q=desc((3, 4, 64), _lib.RK_F32), p=pool(dtype=_lib.RK_F32)), _lib.RK_ERR_DTYPE),
    (dict(p=pool(v_dtype=_lib.RK_F16)), _lib.RK_ERR_DTYPE),
    (dict(p=pool(table_dtype=_lib.RK_I64)), _lib.RK_ERR_DTYPE),
    (dict(p=pool(v_pages=5)), _lib.RK_ERR_SHAPE),
    (dict(p=pool(page=12)), _lib.RK_ERR_SHAPE),
    (dict(p=pool(page=4)), _lib.RK_ERR_SHAPE),
    (dict(p=pool(per=1 << 27)), _lib.RK_ERR_SHAPE),
    (dict(p=pool(table_stride=(1, 3))), _lib.RK_ERR_STRIDE),
    (dict(p=pool(stride=(2048, 1024, 64, 2))), _lib.RK_ERR_STRIDE),
    (dict(p=pool(stride=(2112, 1056, 66, 1))), _lib.RK_ERR_STRIDE),
    (dict(p=pool(stride=(1 << 32, 1 << 31, 1 << 27, 1))), _lib.RK_ERR_STRIDE),  # eight rows past 32 bits of bytes
    (dict(window=-1), _lib.RK_ERR_ARG),
    (dict(sinks=-1), _lib.RK_ERR_ARG),
    (dict(out=desc((3, 4, 72))), _lib.RK_ERR_SHAPE),
    (dict(out=desc((3, 4, 64), stride=(0, 64, 1))), _lib.RK_ERR_STRIDE),
    (dict(out=desc((3, 4, 64), _lib.RK_F16)), _lib.RK_ERR_DTYPE),
])
def test_attention_refuses(call, status):
    assert attention(**call) == status


def test_attention_refuses_more_than_a_launch():
    """A launch's threads are counted in 32 bits: 2^24 workgroups of 256 are too many."""
    most = 1 << 24

    def single(B, H, groups, tokens=16):
        return window(q=(B, H * groups, 1, 64), k=(B, H, tokens, 64), groups=groups)

    assert single(most - 1, 1, 1) == 0
    assert single(most, 1, 1) == _lib.RK_ERR_SHAPE
    assert single(most // 8, 8, 4) == _lib.RK_ERR_SHAPE
    assert single(most // 8 - 1, 8, 4) == 0
    assert single(most // 2, 1, 8, 16) == _lib.RK_ERR_SHAPE          # rows to join, four a workgroup
    assert window(q=(most - 1, 1, 2, 64), k=(most - 1, 1, 16, 64), groups=1) == 0
    assert window(q=(most, 1, 2, 64), k=(most, 1, 16, 64), groups=1) == _lib.RK_ERR_SHAPE


def test_attention_without_a_pool_or_output():
    lib, q, p = _lib.load(), desc((3, 4, 64)), pool()
    assert lib.rk_paged_attention(ctypes.byref(q), None, None, 2, 0, 0, ctypes.byref(q), None, 0, None) == _lib.RK_ERR_NULL
    assert lib.rk_paged_attention(ctypes.byref(q), None, ctypes.byref(p), 2, 0, 0, None, None, 0, None) == _lib.RK_ERR_NULL
    p.lens = None
    assert lib.rk_paged_attention(ctypes.byref(q), None, ctypes.byref(p), 2, 0, 0, ctypes.byref(q), None, 0,
                                  None) == _lib.RK_ERR_NULL


def window(q=(2, 4, 5, 64), k=(2, 2, 9, 64), v=None, groups=2, stride=None, **more):
    d = [desc(q), desc(k, stride=stride), desc(v or k)]
    return _lib.load().rk_window_attention_check(*(ctypes.byref(x) for x in d), None, groups, more.get("window", 0),
                                                 more.get("sinks", 0), None, 256, None)


def test_window_attention_refuses():
    assert window() == 0
    assert window(q=(2, 4, 50, 64)) == 0        # more queries than tokens: the first see nothing
    assert window(q=(3, 4, 5, 64)) == _lib.RK_ERR_SHAPE
    assert window(v=(2, 2, 8, 64)) == _lib.RK_ERR_SHAPE
    assert window(k=(2, 2, 1 << 30, 64)) == _lib.RK_ERR_SHAPE
    assert window(groups=1) == _lib.RK_ERR_HEADS
    assert window(stride=(1152, 576, 1, 9)) == _lib.RK_ERR_STRIDE
    assert window(window=-3) == _lib.RK_ERR_ARG


def rotary(q=None, k=None, pos=None, freq=None, sections=(32,), axes=1, interleaved=0, inverse=0, qo=None, ko=None):
    q = q or desc((2, 4, 5, 64))
    pos, freq = pos or desc((axes, 2, 5), _lib.RK_I64), freq or desc((32,), _lib.RK_F32)
    s = (ctypes.c_int32 * max(len(sections), 1))(*sections)
    ref = _lib.ref
    return _lib.load().rk_rotary(ref(q), ref(k), ref(pos), ref(freq), s, axes, interleaved, inverse, ref(qo or q),
                                 ref(ko or k), None)


@pytest.mark.parametrize("call, status", [
    (dict(q=desc((2, 4, 5, 136))), _lib.RK_ERR_HEAD_DIM),
    (dict(q=desc((4, 64))), _lib.RK_ERR_RANK),
    (dict(q=desc((2, 4, 5, 62))), _lib.RK_ERR_SHAPE),                  # 2 P > D
    (dict(q=desc((2, 4, 5, 64), _lib.RK_F64)), _lib.RK_ERR_DTYPE),
    (dict(k=desc((2, 2, 6, 64))), _lib.RK_ERR_SHAPE),
    (dict(k=desc((2, 2, 5, 64), _lib.RK_F16)), _lib.RK_ERR_DTYPE),
    (dict(pos=desc((1, 2, 6), _lib.RK_I64)), _lib.RK_ERR_SHAPE),
    (dict(pos=desc((2, 2, 5), _lib.RK_I64)), _lib.RK_ERR_SHAPE),
    (dict(pos=desc((1, 2, 5), _lib.RK_F32)), _lib.RK_ERR_DTYPE),
    (dict(freq=desc((32,), _lib.RK_F64)), _lib.RK_ERR_DTYPE),
    (dict(freq=desc((65,), _lib.RK_F32), sections=(65,)), _lib.RK_ERR_SHAPE),
    (dict(freq=desc((0,), _lib.RK_F32), sections=(0,)), _lib.RK_ERR_SHAPE),
    (dict(sections=(31,)), _lib.RK_ERR_ARG),
    (dict(sections=(33, -1), axes=2), _lib.RK_ERR_ARG),
    (dict(sections=(8, 8, 8, 4, 4), axes=5), _lib.RK_ERR_ARG),
    (dict(sections=(32,), axes=0, pos=desc((1, 2, 5), _lib.RK_I64)), _lib.RK_ERR_ARG),
    (dict(interleaved=2), _lib.RK_ERR_ARG),
    (dict(qo=desc((2, 4, 5, 64), stride=(0, 320, 64, 1))), _lib.RK_ERR_STRIDE),
    (dict(qo=desc((2, 4, 6, 64))), _lib.RK_ERR_SHAPE),
])
def test_rotary_refuses(call, status):
    assert rotary(**call) == status


def test_rotary_refuses_more_than_a_launch():
    most = 1 << 25
    assert rotary(q=desc((1, 1, most, 64)), pos=desc((1, 1, most), _lib.RK_I32)) == _lib.RK_ERR_SHAPE
    assert append(k=desc((3, 2, most, 64))) == _lib.RK_ERR_SHAPE


def append(k=None, v=None, p=None, starts=None, q=None, qo=None, pos=None, freq=None):
    k = k or desc((3, 2, 64))
    s = (ctypes.c_int32 * 1)(32)
    ref = _lib.ref
    return _lib.load().rk_paged_append(ref(k), ref(v or k), ref(p or pool()), starts, ref(q), ref(qo), ref(pos), ref(freq),
                                       s, 1, 0, None)


@pytest.mark.parametrize("call, status", [
    (dict(k=desc((4, 2, 64))), _lib.RK_ERR_SHAPE),                     # one token of every request
    (dict(k=desc((2, 2, 5, 64))), _lib.RK_ERR_SHAPE),
    (dict(k=desc((3, 2, 5, 64)), starts=NEVER), _lib.RK_ERR_SHAPE),    # starts and a batch
    (dict(k=desc((3, 3, 64))), _lib.RK_ERR_HEADS),
    (dict(k=desc((3, 2, 32))), _lib.RK_ERR_HEAD_DIM),
    (dict(k=desc((3, 2, 64), _lib.RK_F16)), _lib.RK_ERR_DTYPE),
    (dict(v=desc((3, 2, 32))), _lib.RK_ERR_SHAPE),
    (dict(q=desc((3, 4, 64))), _lib.RK_ERR_NULL),
    (dict(q=desc((3, 4, 64)), qo=desc((3, 4, 64))), _lib.RK_ERR_NULL),  # q without positions
    (dict(pos=desc((1, 3), _lib.RK_I64)), _lib.RK_ERR_NULL),
    (dict(pos=desc((1, 4), _lib.RK_I64), freq=desc((32,), _lib.RK_F32)), _lib.RK_ERR_SHAPE),
    (dict(p=pool(stride=(0, 1024, 64, 1))), _lib.RK_ERR_STRIDE),
    (dict(p=pool(page=24)), _lib.RK_ERR_SHAPE),
])
def test_append_refuses(call, status):
    assert append(**call) == status


def test_python_refuses_on_the_host():
    from rotatek_amd.kernels import paged_decode, paged_prefill, window_attention
    from rotatek_amd.paged import append_pages
    from rotatek_amd.rotary import apply_rotary
    q, k = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        paged_decode(q, k, k, table, lens, 2)
    with pytest.raises(ValueError, match="dims"):
        paged_decode(q.unsqueeze(0), k, k, table, lens, 2)
    with pytest.raises(ValueError, match="window"):
        paged_decode(q, k, k, table, lens, 2, window=0)
    with pytest.raises(ValueError, match="starts"):
        paged_prefill(q, None, k, k, table, lens, 2)
    with pytest.raises(ValueError, match="dims"):
        window_attention(q, k, k, 2)
    with pytest.raises(ValueError, match="positions"):
        append_pages(q[:, :2], q[:, :2], k, k, table, lens, q=q)
    with pytest.raises(RuntimeError):
        apply_rotary(q, None, torch.zeros(3, dtype=torch.int64), torch.ones(32))
    with pytest.raises(ValueError):
        inverse_frequencies(7, device="cpu")
    f = inverse_frequencies(8, 100.0, "cpu")
    np.testing.assert_allclose(f.numpy(), [1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], rtol=1e-6)


# -------------------------------------------------------------- PagedCache
def test_cache_counts_and_pages():
    c = PagedCache(2, 2, 16, pages=6, page=8, requests=3, max_tokens=30, device="cpu")
    assert (len(c), c.max_tokens, c.free_pages) == (2, 32, 6)
    assert c.begin([9, 1, 0]) == 10 and c.free_pages == 3
    assert c.lens.tolist() == [9, 1, 0] and c.starts.tolist() == [0, 9, 10, 10]
    used = [p for row in c.table.tolist() for p in row if p >= 0]
    assert sorted(used) == sorted(set(used)) and len(used) == 3
    assert c.begin([7, 7, 1]) == 15 and c.free_pages == 2       # pages fill up to their ends first
    assert c.begin([1, 1, 1]) == 3 and c.free_pages == 0
    before = c.table.clone(), c.lens.clone(), c.free_pages
    with pytest.raises(RuntimeError, match="pages"):
        c.begin([8, 0, 0])
    with pytest.raises(ValueError, match="max_tokens"):
        c.begin([0, 24, 0])
    for bad in ([1, 1], [1, 1, -1]):
        with pytest.raises(ValueError):
            c.begin(bad)
    assert torch.equal(before[0], c.table) and torch.equal(before[1], c.lens) and c.free_pages == before[2]
    c.free(0)
    assert c.free_pages == 3 and c.lens.tolist() == [0, 9, 2] and c.length(0) == 0 and c.get_seq_length() == 9
    assert c.begin([8, 8, 0]) == 16 and c.free_pages == 1
    used = [p for row in c.table.tolist() for p in row if p >= 0]
    assert sorted(used) == sorted(set(used)) and len(used) == 5
    with pytest.raises(ValueError, match="new tokens"):
        c.attend(0, torch.zeros(3, 4, 16), 2)


@pytest.mark.parametrize("args", [dict(page=12), dict(page=4), dict(pages=0), dict(requests=0), dict(max_tokens=0),
                                  dict(dtype=torch.float32), dict(head_dim=20), dict(head_dim=136)])
def test_cache_refuses(args):
    with pytest.raises(ValueError):
        PagedCache(**{**dict(layers=1, heads_kv=1, head_dim=16, pages=2, device="cpu"), **args})
