"""Numpy oracle of a paged KV cache (64 bits): rotation by position, append,
and attention over pages or plain rows with a window and sinks.  Token by token
and row by row, from the definitions; used by the tests alone."""
from __future__ import annotations

import numpy as np


def axis_of(sections, interleaved):
    """The axis of each pair: axis after axis, or dealt in turn to those that have pairs left."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def rotate(x, positions, inv_freq, sections=None, interleaved=False, inverse=False):
    """x [..., D] of one token each, positions [axes, ...] without the head dim:
    x [T, H, D] with positions [axes, T]."""
    P = len(inv_freq)
    axes = axis_of(sections or [P], interleaved)
    y = np.array(x, np.float64)
    for i, a in enumerate(axes):
        angle = positions[a].astype(np.float64) * float(inv_freq[i])
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None] * (-1 if inverse else 1)
        u, v = x[..., i].astype(np.float64), x[..., i + P].astype(np.float64)
        y[..., i], y[..., i + P] = u * c - v * s, v * c + u * s
    return y


def place(n, table, lens, starts, page, pages, each=1):
    """(page, row) of new token n, or None where it goes nowhere."""
    B, per = table.shape
    if starts is not None:
        found = [b for b in range(B) if starts[b] <= n < starts[b + 1]]
        if not found:
            return None
        b = found[-1]
        i, each = n - starts[b], starts[b + 1] - starts[b]
    else:
        b, i = divmod(n, each)
    p = int(lens[b]) - int(each) + int(i)
    if p < 0 or p >= per * page:
        return None
    at = int(table[b, p // page])
    return (at, p % page) if 0 <= at < pages else None


def append(k_new, v_new, k_pages, v_pages, table, lens, starts=None, each=1):
    """New tokens [N, H, D] into copies of the pages."""
    k, v = k_pages.copy(), v_pages.copy()
    for n in range(len(k_new)):
        at = place(n, table, lens, starts, k.shape[2], k.shape[0], each)
        if at is not None:
            k[at[0], :, at[1]], v[at[0], :, at[1]] = k_new[n], v_new[n]
    return k, v


def rows(pages, table, b, length):
    """(rows [H, length, D] of request b, which of them are there)."""
    P, H, page, D = pages.shape
    out, there = np.zeros((H, length, D)), np.zeros(length, bool)
    for j in range(length):
        at = int(table[b, j // page])
        if 0 <= at < P:
            out[:, j], there[j] = pages[at, :, j % page], True
    return out, there


def attend(q, k, v, there, first, groups, window=None, sinks=0):
    """q [T, Hq, D] at positions first, first + 1, ..; k, v [H, S, D] ->
    (out, sum of w |v| / sum of w, largest sum of |q k| / sqrt(D)) [T, Hq, D]."""
    T, Hq, D = q.shape
    out, amp, big = np.zeros((T, Hq, D)), np.zeros((T, Hq, D)), 0.0
    j = np.arange(k.shape[1])
    for t in range(T):
        p = first + t
        on = there & (j <= p)
        if window is not None:
            on &= (j > p - window) | (j < sinks)
        if not on.any():
            continue
        for h in range(Hq):
            kk, vv = k[h // groups][on], v[h // groups][on]
            with np.errstate(invalid="ignore", over="ignore"):
                s = kk @ q[t, h] / np.sqrt(D)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h], amp[t, h] = w @ vv, w @ np.abs(vv)
                big = max(big, float(np.max(np.abs(kk) @ np.abs(q[t, h])) / np.sqrt(D)))
    return out, amp, big
