"""Groups whose product with the KV heads passes 64 bits are refused, also where
it comes out as the query heads."""
import pytest
import torch

from rotatek_amd import _lib
from test_quantized_host import _decode, _rows, _shared


@pytest.mark.parametrize("groups", [2 ** 62 + 2, 2 ** 63 - 1, 3, 1, 8, 9])
def test_groups(groups):
    q, p = torch.zeros(2, 8, 128, dtype=torch.bfloat16), torch.zeros(1, 4, 64, 128, dtype=torch.bfloat16)
    r = _rows(H=4)
    assert _decode(q, kf=r, vf=r, G=2)[0] == 0 and _shared(q, p, p, G=2)[0] == 0
    assert _decode(q, kf=r, vf=r, G=groups)[0] == _lib.RK_ERR_HEADS
    assert _shared(q, p, p, G=groups)[0] == _lib.RK_ERR_HEADS


def test_no_query_heads():
    q, p = torch.zeros(2, 0, 128, dtype=torch.bfloat16), torch.zeros(1, 4, 64, 128, dtype=torch.bfloat16)
    assert _shared(q, p, p, G=1)[0] == _lib.RK_ERR_HEADS
