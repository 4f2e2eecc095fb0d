"""A batch of no requests: sized on the host, answered without a launch."""
import pytest
import torch

from test_quantized_host import _decode, _rows, _shared


@pytest.mark.parametrize("cus", [1, 256])
@pytest.mark.parametrize("S", [0, 1, 5000])
def test_plan_of_no_requests(S, cus):
    bf = torch.bfloat16
    q, p, t = torch.zeros(0, 4, 128, dtype=bf), torch.zeros(1, 2, S, 128, dtype=bf), torch.zeros(0, 2, 9, 128, dtype=bf)
    R, ks = torch.zeros(1, 2, 128, 32), torch.zeros(1, 2, 50, 32, dtype=bf)
    vs = torch.zeros(1, 2, 50, 128, dtype=bf)
    assert _shared(q, p, p, cus=cus)[0] == 0
    assert _shared(q, p, p, k2=t, v2=t, cus=cus)[0] == 0
    assert _shared(q, p, p, ks=ks, vs=vs, R=R, k2=t, v2=t, cus=cus)[0] == 0
    m = _rows(B=1, S=S)
    assert _shared(q, m, m, cus=cus)[0] == 0 and _shared(q.float(), m, m, cus=cus)[0] == 0
    r = _rows(B=0, S=S)
    assert _decode(q, kf=r, vf=r, cus=cus)[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["plain", "mx8"])
def test_no_requests_behind_a_prefix(fmt):
    from rotatek_amd.kernels import shared_prefix_decode
    from rotatek_amd.quantized import quantize_rows
    q, p, t = (torch.randn(*s, device="cuda", dtype=torch.bfloat16) for s in
               ((0, 4, 128), (1, 2, 100, 128), (0, 2, 9, 128)))
    lens = torch.zeros(0, dtype=torch.int32, device="cuda")
    if fmt != "plain":
        p, t = quantize_rows(p, fmt), quantize_rows(t, fmt)
    for out in (shared_prefix_decode(q, p, p, None, None, 2), shared_prefix_decode(q, p, p, t, t, 2, len_suffix=lens)):
        assert out.shape == (0, 1, 4, 128) and out.dtype == torch.bfloat16
