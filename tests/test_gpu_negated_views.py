"""Views whose memory holds the negatives of their values (the imaginary part of a
conjugate): refused, not read as they lie."""
import pytest
import torch

from rotatek_amd.paged import append_pages
from rotatek_amd.quantized import quantize_rows
from rotatek_amd.rotary import apply_rotary, inverse_frequencies

pytestmark = pytest.mark.gpu


def negated(*shape):
    x = torch.randn(*shape, dtype=torch.complex64, device="cuda").conj().imag
    assert x.is_neg()
    return x


def test_negated_views():
    pos, freq = torch.arange(3, device="cuda"), inverse_frequencies(16)
    x = negated(3, 2, 16)
    with pytest.raises(ValueError, match="resolve_neg"):
        apply_rotary(x, None, pos, freq)
    with pytest.raises(ValueError, match="resolve_neg"):
        apply_rotary(x.resolve_neg(), None, pos, freq, out=(negated(3, 2, 16), None))
    got, _ = apply_rotary(x.resolve_neg(), None, pos, freq)
    assert torch.equal(got[0], x[0])        # position 0
    k, v = torch.randn(3, 2, 16, device="cuda"), torch.randn(3, 2, 16, device="cuda")
    pages = [torch.zeros(3, 2, 8, 16, device="cuda") for _ in range(2)]
    table = torch.arange(3, dtype=torch.int32, device="cuda").view(3, 1)
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    for call in (lambda: append_pages(x, v, *pages, table, lens), lambda: append_pages(k, x, *pages, table, lens),
                 lambda: append_pages(k, v, negated(3, 2, 8, 16), pages[1], table, lens)):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    assert all((p == 0).all() for p in pages)
    with pytest.raises(ValueError, match="resolve_neg"):
        quantize_rows(negated(1, 1, 4, 32))
