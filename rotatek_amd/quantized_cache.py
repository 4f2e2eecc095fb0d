"""Span cache with quantised rows.

``cache.DynamicCache`` holds prompt, visual and text spans in the model's
dtype; here the same spans are quantised as they are stored (8 or 4 bits, see
``quantized``), so a layer of 128-channel heads takes 0.52 or 0.27 of the bytes
and a decode step reads as much less.  No counterpart in the reference.

    cache = QuantizedCache("mx8")
    cache.store_pruned(k_pruned, k_prompt, k_text, None, values, layer)   # prefill
    cache.rotatek_rotations.append(R); cache.rotatek_means.append(dmu)
    cache.update(k, v, layer)                                             # a token
    out, _, _ = cache.decode_rotatek(q, layer, groups)

``append_`` and ``decode_rotatek`` work on the device alone (lengths are device
tensors, shapes are fixed by the capacity), so a step may be captured in a HIP
graph and replayed while the text grows; call ``reserve`` first (rows that a graph
holds do not move, ``release_graphs``).
"""
from __future__ import annotations

from typing import List, Optional

import torch

from rotatek_amd.cache import Cache
from rotatek_amd.kernels.quantized_decode import rotatek_decode_quantized
from rotatek_amd.quantized import BLOCK, MXRows, _format, append_rows, quantize_rows


class _Layer:
    """One layer's rows: ``k`` / ``v`` prompt | text | free, ``ks`` / ``vs``
    visual.  ``lens[b]`` (device int32) counts prompt and text tokens, ``n`` is
    the host's count of ``update``'s, ``ahead`` whether ``append_`` has moved the
    lengths past it, ``captured`` whether a graph holds the rows."""

    __slots__ = ("k", "v", "ks", "vs", "lens", "s_prompt", "s_vision", "n", "ahead", "captured")


class QuantizedCache(Cache):
    """``fmt``: "mx8" or "mx4"; ``reserve_tokens``: decode headroom at prefill."""

    def __init__(self, fmt: str = "mx8", reserve_tokens: int = 256) -> None:
        _format(fmt)
        if reserve_tokens < 0:
            raise ValueError("reserve_tokens must be >= 0")
        self.fmt, self.reserve_tokens = fmt, int(reserve_tokens)
        self.rotatek_rotations: List[Optional[torch.Tensor]] = []
        self.rotatek_means: List[Optional[torch.Tensor]] = []
        self._layers: List[_Layer] = []

    def __len__(self) -> int:
        return len(self._layers)

    @property
    def nbytes(self) -> int:
        """Bytes of all layers' rows, capacity included."""
        return sum(r.nbytes for x in self._layers for r in (x.k, x.v, x.ks, x.vs))

    def store_pruned(self, key_states_pruned, key_states_prompt, key_states_text, mask, value_states,
                     layer_idx: int) -> None:
        """Prefill-time write of the next layer; arguments as
        ``DynamicCache.store_pruned`` (``value_states``: prompt | visual | text;
        ``mask``, the kept channels, is not needed at decode)."""
        if layer_idx != len(self._layers):
            raise ValueError(f"layers are stored in order: the next one is {len(self._layers)}, not {layer_idx}")
        s_p, s_v, s_t = (t.shape[-2] for t in (key_states_prompt, key_states_pruned, key_states_text))
        if value_states.shape[-2] != s_p + s_v + s_t:
            raise ValueError("value_states must hold the prompt, visual and text tokens")
        B, H, _, D = key_states_prompt.shape
        x = _Layer()
        x.s_prompt, x.s_vision, x.n, x.ahead, x.captured = s_p, s_v, s_t, False, False
        dev, cap = key_states_prompt.device, s_p + s_t + self.reserve_tokens
        x.k, x.v = (MXRows.empty(B, H, cap, D, self.fmt, dev) for _ in range(2))
        x.lens = torch.zeros(B, dtype=torch.int32, device=dev)
        for k, v in ((key_states_prompt, value_states[:, :, :s_p]), (key_states_text, value_states[:, :, s_p + s_v:])):
            append_rows(k, v, x.k, x.v, x.lens)
        x.ks = quantize_rows(key_states_pruned, self.fmt)
        x.vs = quantize_rows(value_states[:, :, s_p:s_p + s_v], self.fmt)
        self._layers.append(x)

    def _grow(self, x: _Layer, need: int) -> None:
        """Reallocate one layer at >= twice its text capacity.  Every row moves:
        the device's lengths may be ahead of the host's count.  Refused while a
        captured graph holds the rows: its replays would write to memory that is
        free and count tokens that the new rows lack."""
        if x.captured:
            raise RuntimeError(f"{need} text rows are needed, but a captured graph holds the layer's rows; reserve() "
                               "enough tokens before the capture, or release_graphs() when the graphs are gone")
        rows = x.k.shape[2]
        cap = x.s_prompt + max(2 * (rows - x.s_prompt), need)
        for name in ("k", "v"):
            old = getattr(x, name)
            new = MXRows.empty(*old.shape[:2], cap, old.head_dim, self.fmt, old.device)
            new.codes[:, :, :rows].copy_(old.codes)
            new.scales[..., :old.scales.shape[3]].copy_(old.scales)
            setattr(x, name, new)

    def reserve(self, tokens: int) -> None:
        """Room for ``tokens`` more in every layer, behind what ``append_`` and
        replays have added (synchronises; before graph capture: the rows may
        move)."""
        self.sync_lengths()
        for x in self._layers:
            if x.s_prompt + x.n + tokens > x.k.shape[2]:
                self._grow(x, x.n + tokens)

    def release_graphs(self) -> None:
        """The graphs that were captured over this cache are gone, or will not be
        replayed again: the rows may move."""
        for x in self._layers:
            x.captured = False

    @staticmethod
    def _held(x: _Layer) -> bool:
        """Whether this call is being captured; the graph then holds the rows."""
        capturing = torch.cuda.is_current_stream_capturing()
        x.captured |= capturing
        return capturing

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int) -> None:
        """Append decode tokens [B, H_kv, T, D] to a layer, with room made for
        them.  The host counts along; the first after an ``append_``, and every one
        while a captured graph holds the rows, asks the device."""
        x = self._layers[layer_idx]
        steps = key_states.shape[-2]
        if not self._held(x) and (x.ahead or x.captured):
            self._sync(x)
        if x.s_prompt + x.n + steps > x.k.shape[2]:
            self._grow(x, x.n + steps)
        append_rows(key_states, value_states, x.k, x.v, x.lens)
        x.n += steps

    def append_(self, layer_idx: int, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        """Append on the device alone, at each request's own length; a full
        request drops the tokens."""
        x = self._layers[layer_idx]
        append_rows(key_states, value_states, x.k, x.v, x.lens)
        x.ahead = True
        self._held(x)

    def _sync(self, x: _Layer) -> None:
        x.n = int(x.lens.max()) - x.s_prompt if x.lens.numel() else x.n
        x.ahead = False

    def sync_lengths(self) -> None:
        """The host's counts from the device's (synchronises); the largest where
        requests differ."""
        for x in self._layers:
            self._sync(x)

    def lengths(self, layer_idx: int) -> torch.Tensor:
        """Device int32 [B]: prompt + text tokens per request."""
        return self._layers[layer_idx].lens

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """Tokens cached for a layer (prompt + visual + text), 0 for one not
        stored yet."""
        if layer_idx >= len(self._layers):
            return 0
        x = self._layers[layer_idx]
        return x.s_prompt + x.s_vision + x.n

    def spans(self, layer_idx: int):
        """A layer's rows ``(k_full, v_full, k_sparse, v_sparse)`` as they lie in
        memory: the full ones to their capacity, undefined past ``lengths``."""
        x = self._layers[layer_idx]
        return x.k, x.v, x.ks, x.vs

    def prefix(self, layer_idx: int):
        """What ``shared_prefix_decode`` takes as its shared spans ``(k_prefix,
        v_prefix, k_sparse, v_sparse)``: a batch of one's rows, the full ones cut
        to the prompt and text they hold now (asks the device where the host has
        not counted along).  Views: good until the rows move."""
        x = self._layers[layer_idx]
        if x.k.shape[0] != 1:
            raise ValueError(f"a shared prefix is one request's, this layer holds {x.k.shape[0]}")
        if not self._held(x) and (x.ahead or x.captured):
            self._sync(x)
        filled = x.s_prompt + x.n
        return x.k.narrow(0, filled), x.v.narrow(0, filled), x.ks, x.vs

    def decode_rotatek(self, q_full: torch.Tensor, layer_idx: int, num_kv_groups: int,
                       out: Optional[torch.Tensor] = None):
        """RotateK decode over a layer's rows, ``(out [B, 1, H_q, D], None,
        None)`` like ``rotatek_decode``."""
        x = self._layers[layer_idx]
        self._held(x)
        return rotatek_decode_quantized(q_full, self.rotatek_rotations[layer_idx], self.rotatek_means[layer_idx], x.k,
                                        x.v, None, x.ks, x.vs, num_kv_groups, len_full=x.lens, out=out)


__all__ = ["QuantizedCache"]
