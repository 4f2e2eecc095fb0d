"""KV cache of requests of different lengths, in pages.

``cache.DynamicCache`` holds a batch as one tensor a layer, as long as its
longest request; here each request holds the pages that its own tokens take,
and gives them back when it is done (see ``paged``).  No counterpart in the
reference.

    cache = PagedCache(layers=28, heads_kv=4, head_dim=128, pages=4096, requests=16, max_tokens=32768)
    cache.begin([812, 40, 1, 0, ...])                      # a step: new tokens of each request
    for layer in range(28):
        q = cache.append(layer, k, v, q=q, positions=pos, inv_freq=f, sections=(16, 24, 24))
        out = cache.attend(layer, q, groups)
    cache.free(2)                                          # a request is done

``begin`` counts on the host and copies table, lengths and starts to the device
without waiting; ``append`` and ``attend`` work on the device alone, with
buffers that never move, so a step's layers may be captured in a HIP graph and
replayed behind a ``begin`` of the same counts (``begin`` and ``free`` themselves
may not be captured).

``attend`` is planned for requests of ``max_tokens`` (see ``kernels.paged_attention``),
and a ``begin`` that adds pages writes the table's rows anew: 0.8 ms where 32 requests
of up to 32768 tokens come to a page's end at once, 13 of up to 10^6, 0.03 where none
does.  So ``max_tokens`` should be no more than is needed.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from rotatek_amd.cache import Cache
from rotatek_amd.kernels.paged_attention import paged_decode, paged_prefill
from rotatek_amd.paged import append_pages


class PagedCache(Cache):
    """``pages`` pages of ``page`` tokens a layer, ``requests`` requests of at
    most ``max_tokens`` (None: all the pages') tokens."""

    def __init__(self, layers: int, heads_kv: int, head_dim: int, pages: int, page: int = 64, requests: int = 1,
                 max_tokens: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device="cuda") -> None:
        if page < 8 or page & (page - 1):
            raise ValueError(f"page must be a power of two from 8 on, got {page}")
        if min(layers, heads_kv, head_dim, pages, requests) < 1:
            raise ValueError("layers, heads_kv, head_dim, pages and requests must be at least 1")
        if dtype not in (torch.float16, torch.bfloat16) or head_dim % 8 or head_dim > 128:
            raise ValueError(f"pages hold fp16 or bf16, head_dim a multiple of 8 up to 128; got {dtype}, {head_dim}")
        most = pages * page if max_tokens is None else max_tokens
        if most < 1:
            raise ValueError("max_tokens must be at least 1")
        self.page, self.pages, self.requests = int(page), int(pages), int(requests)
        per = -(-most // page)
        self.max_tokens = per * page
        shape = (pages, heads_kv, page, head_dim)
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.table = torch.full((requests, per), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.starts = torch.zeros(requests + 1, dtype=torch.int32, device=device)
        self._free: List[int] = list(range(pages - 1, -1, -1))
        self._own: List[List[int]] = [[] for _ in range(requests)]
        self._held = [0] * requests
        self._new = [0] * requests

    def __len__(self) -> int:
        return len(self.k)

    @property
    def nbytes(self) -> int:
        """Bytes of all layers' pages."""
        return sum(x.numel() * x.element_size() for x in (*self.k, *self.v))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """Tokens of the longest request."""
        return max(self._held)

    def length(self, request: int) -> int:
        """Tokens that a request holds, the present step's among them."""
        return self._held[request]

    def _outside_capture(self) -> None:
        """A copy that is captured would be replayed from pinned memory that others
        have by then."""
        if self.table.is_cuda:
            with torch.cuda.device(self.table.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("begin and free count on the host: call them outside a capture, ahead of a replay")

    def _put(self, to: torch.Tensor, values) -> None:
        """Copy to the device in the current stream's order, without waiting (the
        pinned copy is kept by torch's allocator until it has been read)."""
        x = torch.tensor(values, dtype=torch.int32)
        if to.is_cuda:
            x = x.pin_memory()
        to.copy_(x, non_blocking=True)

    def _put_table(self, requests: Sequence[int]) -> None:
        per = self.table.shape[1]
        for b in requests:
            self._put(self.table[b], self._own[b] + [-1] * (per - len(self._own[b])))

    def begin(self, counts: Sequence[int]) -> int:
        """The next step: ``counts[b]`` new tokens of each request, with pages
        found for them.  Returns their sum N.  Where a request would pass
        ``max_tokens`` (ValueError) or pages run out (RuntimeError), nothing
        changes."""
        self._outside_capture()
        counts = [int(n) for n in counts]
        if len(counts) != self.requests or min(counts) < 0:
            raise ValueError(f"counts must hold {self.requests} numbers from 0 on")
        need = []
        for held, own, n in zip(self._held, self._own, counts):
            if held + n > self.max_tokens:
                raise ValueError(f"a request of {held} tokens takes no {n} more: max_tokens is {self.max_tokens}")
            need.append(-(-(held + n) // self.page) - len(own))
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages are needed, {len(self._free)} are free")
        for own, n in zip(self._own, need):
            own.extend(self._free.pop() for _ in range(n))
        for b, n in enumerate(counts):
            self._held[b] += n
        self._put_table([b for b, n in enumerate(need) if n])
        self._put(self.lens, self._held)
        if counts != self._new:
            at = [0]
            for n in counts:
                at.append(at[-1] + n)
            self._put(self.starts, at)
            self._new = counts
        return sum(counts)

    def free(self, request: int) -> None:
        """A request is done: its pages go to the next ones that ask."""
        self._outside_capture()
        self._free.extend(reversed(self._own[request]))
        self._own[request] = []
        self._held[request] = 0
        self._put_table([request])
        self._put(self.lens, self._held)

    def _starts(self) -> Optional[torch.Tensor]:
        """None where every request has one new token: the form of single ones."""
        return None if all(n == 1 for n in self._new) else self.starts

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, positions: Optional[torch.Tensor] = None,
               inv_freq: Optional[torch.Tensor] = None, sections: Optional[Sequence[int]] = None,
               interleaved: bool = False, q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """The step's Keys and Values [N, H_kv, D] of a layer, request by request;
        rotation as ``paged.append_pages``.  Returns the rotated ``q``."""
        self._check_step(k_new)
        return append_pages(k_new, v_new, self.k[layer], self.v[layer], self.table, self.lens, self._starts(),
                            positions, inv_freq, sections, interleaved, q)

    def attend(self, layer: int, q: torch.Tensor, num_kv_groups: int, window: Optional[int] = None, sinks: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The step's queries [N, H_q, D] over a layer; returns [N, H_q, D]."""
        self._check_step(q)
        starts = self._starts()
        if starts is None:
            return paged_decode(q, self.k[layer], self.v[layer], self.table, self.lens, num_kv_groups, window, sinks,
                                out).squeeze(1)
        return paged_prefill(q, starts, self.k[layer], self.v[layer], self.table, self.lens, num_kv_groups, window,
                             sinks, out)

    def _check_step(self, x: torch.Tensor) -> None:
        if x.dim() != 3 or x.shape[0] != sum(self._new):
            raise ValueError(f"the step has {sum(self._new)} new tokens [N, H, D], got shape {tuple(x.shape)}")


__all__ = ["PagedCache"]
