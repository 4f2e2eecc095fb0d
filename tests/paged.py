"""Inputs and bounds that the tests of the paged cache share."""
import numpy as np
import torch

from oracle import paged as op

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def half(dtype):
    """A rounding to nearest is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def rotation_bound(x, want, pairs, dtype):
    """Rounding of the result, and of a rotation in fp32 of channels i and i + P.

    The fraction of a turn (at most 1/2) is rounded to fp32: 2^-26 turns, an
    angle of 2 pi 2^-26 < 2^-23.3.  Sine and cosine are good to two units in the
    last place, 2^-23 each; two products and a sum round by 2^-24 each: in all
    less than 2^-21 of |x_i| + |x_(i+P)|.  The outermost 2 of 64-bit positions
    times frequency are below 2^-40."""
    b = np.abs(want) * half(dtype) + (2.0 ** -24 if dtype == torch.float16 else 0.0)
    both = np.abs(x[..., :pairs]) + np.abs(x[..., pairs:2 * pairs])
    b[..., :pairs] += both * 2.0 ** -21
    b[..., pairs:2 * pairs] += both * 2.0 ** -21
    b[..., 2 * pairs:] = 0.0
    return b


def attention_bound(want, amp, big, S, dtype, single):
    """amp: sum of w |v| / sum of w; big: the largest sum of |q k| / sqrt(D).

    Scores.  Products of 16-bit numbers are exact in fp32; 128 of them summed in
    fp32 are off by at most 128 2^-24 of their magnitudes, the scale and the
    maximum taken off by 2^-23 of them: d = big 2^-16.9 (+ 2^-21 for exp2), and
    a weight by e^(2 d) - 1 (its own score and the largest one).
    Weights.  One 16-bit term rounds by half a step of its type; two leave 2^-16
    (bf16) or less.  fp16 ends at 2^-24: a weight (of at most 1, the largest
    being 1) loses at most 2^-25 there, S of them S 2^-25 of the largest |v|.
    Sums of S products of fp32: S 2^-24, in blocks, so at most 2^-14 at the sizes
    here.  The output is rounded once."""
    d = 2.0 * big * 2.0 ** -16.9 + 2.0 ** -20
    w = 2.0 ** -16 if single else half(dtype)
    b = amp * (np.expm1(d) + w + min(S, 1024) * 2.0 ** -24)
    if dtype == torch.float16:
        b = b + S * 2.0 ** -25 * float(np.max(amp, initial=0.0)) * 4 + 2.0 ** -24
    return (np.abs(want) + b) * half(dtype) + b


class Pool:
    """Pages of requests of the given lengths, in a shuffled order, with pages of
    NaN between them, unused rows NaN, and table entries past a request's last
    page that are none."""

    def __init__(self, lens, heads_kv, dim, page, dtype, seed=0, spare=3, per_more=1, strided=False, fill=float("nan")):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.lens, self.page, self.heads, self.dim = list(lens), page, heads_kv, dim
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        table = torch.full((len(lens), max(need + [0]) + per_more), -1, dtype=torch.int32)
        k = torch.full((self.pages, heads_kv, page, dim), fill)
        v = torch.full((self.pages, heads_kv, page, dim), fill)
        at = 0
        for b, n in enumerate(lens):
            for i in range(need[b]):
                table[b, i] = order[at]
                rows = min(page, n - i * page)
                k[order[at], :, :rows] = torch.randn(heads_kv, rows, dim, generator=g)
                v[order[at], :, :rows] = torch.randn(heads_kv, rows, dim, generator=g)
                at += 1
        self.k, self.v, self.table = k.to(dtype), v.to(dtype), table
        if strided:  # [pages, page, H, D] underneath, with room between the rows
            for name in ("k", "v"):
                x = torch.full((self.pages, page, heads_kv, dim + 8), fill, dtype=dtype)[..., :dim].transpose(1, 2)
                x.copy_(getattr(self, name))
                setattr(self, name, x)

    def cuda(self):
        def up(x):
            y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
            return y.copy_(x)
        self.dk, self.dv, self.dtable = up(self.k), up(self.v), self.table.cuda()
        self.dlens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        return self

    def want(self, b, q, groups, window, sinks, length=None):
        """Oracle of request b's last tokens, q [T, Hq, D]."""
        n = self.lens[b] if length is None else length
        n = max(0, min(n, self.table.shape[1] * self.page))
        k, there = op.rows(f64(self.k), self.table.numpy(), b, n)
        v, _ = op.rows(f64(self.v), self.table.numpy(), b, n)
        return op.attend(f64(q), k, v, there, n - q.shape[0], groups, window, sinks)


def check(got, want, bound):
    got = f64(got)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4].tolist(), float(np.nanmax(np.abs(got - want) / bound)))
