"""Tensors that share their memory until one is written (copy-on-write): a call
that writes one leaves the others as they were."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(x, fmt="mx8"):
    from rotatek_amd.quantized import MXRows, quantize_rows
    r = quantize_rows(x, fmt)
    return r, MXRows(torch._lazy_clone(r.codes), torch._lazy_clone(r.scales), r.head_dim, fmt)


def test_outputs():
    from rotatek_amd.kernels import full_channel_decode_quantized, shared_prefix_decode
    from rotatek_amd.quantized import dequantize_rows, quantize_rows
    print("[case] outputs", flush=True)
    x = torch.randn(2, 2, 40, 128, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(2, 4, 128, device="cuda", dtype=torch.bfloat16)
    rows = quantize_rows(x)
    for call in (lambda out: full_channel_decode_quantized(q, rows, rows, 2, out=out),
                 lambda out: shared_prefix_decode(q, x[:1], x[:1], x, x, 2, out=out)):
        kept = torch.full_like(q, 7.0)
        out = torch._lazy_clone(kept)
        want = call(None)
        call(out)
        assert torch.equal(out.unsqueeze(1), want) and (kept == 7).all()
    kept = torch.full_like(x, 7.0)
    out = torch._lazy_clone(kept)
    dequantize_rows(rows, out=out)
    assert torch.equal(out, dequantize_rows(rows)) and (kept == 7).all()


@pytest.mark.parametrize("fmt", ["mx8", "mx4"])
def test_rows_and_lengths(fmt):
    from rotatek_amd.quantized import append_rows, quantize_rows
    print(f"[case] rows {fmt}", flush=True)
    x, y = (torch.randn(2, 2, 40, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kept, mine = _rows(x, fmt)
    before = kept.codes.clone(), kept.scales.clone()
    quantize_rows(y, fmt, out=mine)
    want = quantize_rows(y, fmt)
    assert torch.equal(mine.codes, want.codes) and torch.equal(kept.codes, before[0])
    assert torch.equal(kept.scales, before[1])
    kept, mine = _rows(x, fmt)
    kept_v, mine_v = _rows(x, fmt)
    lens = torch.tensor([3, 39], dtype=torch.int32, device="cuda")
    own = torch._lazy_clone(lens)
    append_rows(y[:, :, :2], y[:, :, :2], mine, mine_v, own)
    assert own.tolist() == [5, 40] and lens.tolist() == [3, 39]
    for a, b in ((kept, mine), (kept_v, mine_v)):
        assert torch.equal(a.codes, before[0]) and torch.equal(a.scales[..., :40], before[1][..., :40])
        assert not torch.equal(b.codes, a.codes)
