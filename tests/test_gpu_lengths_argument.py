"""Lengths that are no int32 tensor [B] are refused as such."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [None, 3, [0, 0], (3, torch.int32), (2, torch.float32), (2, torch.int64)])
def test_append_refuses(lens):
    from rotatek_amd.quantized import MXRows, append_rows
    if isinstance(lens, tuple):
        lens = torch.zeros(lens[0], dtype=lens[1], device="cuda")
    x = torch.zeros(2, 2, 1, 128, device="cuda")
    with pytest.raises(ValueError, match="lens"):
        append_rows(x, x, MXRows.empty(2, 2, 4, 128), MXRows.empty(2, 2, 4, 128), lens)


@pytest.mark.parametrize("lens", [3, [0, 0]])
def test_decode_refuses(lens):
    from rotatek_amd.kernels import full_channel_decode_quantized, shared_prefix_decode
    from rotatek_amd.quantized import quantize_rows
    x, q = torch.zeros(2, 2, 8, 128, device="cuda"), torch.zeros(2, 4, 128, device="cuda")
    r = quantize_rows(x)
    with pytest.raises(ValueError, match="lens"):
        full_channel_decode_quantized(q, r, r, 2, lens=lens)
    with pytest.raises(ValueError, match="lens"):
        shared_prefix_decode(q, r.batch(0, 1), r.batch(0, 1), r, r, 2, len_suffix=lens)
