"""Decode kernels, selected by ``ROTATEK_KERNEL`` (rotatek/kernels/__init__.py:15-24):

    paper (default)  one work unit per query head (fused_decode.py /
                     full_channel_flash_decoding.py launch structure)
    gqa              the query heads of a KV group share each K/V tile

Both families run the same hand-written HIP kernels (librotatek_hip.so);
the variable only selects the work decomposition.  The value is read once
at import and anything else raises ``ValueError``, as in the reference.

The decodes over quantised rows (``rotatek_decode_quantized``,
``full_channel_decode_quantized``) and over a prefix that the batch shares
(``shared_prefix_decode``) have one decomposition whatever the variable says.
"""
import os

# read once at import; any value but the two families is an error
ROTATEK_KERNEL = os.environ.get("ROTATEK_KERNEL", "paper").strip().lower()
_FAMILIES = {
    "paper": ("rotatek_amd.kernels.fused_decode", "rotatek_decode_fused",
              "rotatek_amd.kernels.full_channel_flash_decoding", "full_channel_decode"),
    "gqa": ("rotatek_amd.kernels.gqa_decode", "rotatek_decode_gqa",
            "rotatek_amd.kernels.gqa_decode", "full_channel_decode_gqa"),
}
if ROTATEK_KERNEL not in _FAMILIES:
    raise ValueError(f"ROTATEK_KERNEL={ROTATEK_KERNEL!r} is not a kernel family (use 'paper' or 'gqa')")


def _pick():
    import importlib
    mod_r, name_r, mod_d, name_d = _FAMILIES[ROTATEK_KERNEL]
    return getattr(importlib.import_module(mod_r), name_r), getattr(importlib.import_module(mod_d), name_d)


rotatek_decode, full_channel_decode = _pick()

from rotatek_amd.kernels.quantized_decode import full_channel_decode_quantized, rotatek_decode_quantized  # noqa: E402
from rotatek_amd.kernels.shared_prefix import shared_prefix_decode  # noqa: E402

__all__ = ["ROTATEK_KERNEL", "rotatek_decode", "full_channel_decode", "rotatek_decode_quantized",
           "full_channel_decode_quantized", "shared_prefix_decode"]
