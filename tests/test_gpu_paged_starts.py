"""Starts that do not ascend, of more requests than a wave has lanes: whatever they
say, nothing outside the output's rows is written, and the call ends."""
import pytest
import torch

from rotatek_amd.kernels import paged_prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [65, 300])
@pytest.mark.parametrize("N, G", [(40, 3), (700, 64)])
def test_every_request_claims_every_token(B, N, G):
    dt, page = torch.bfloat16, 16
    torch.manual_seed(B)
    k, v = (torch.randn(B, 1, page, 64, device="cuda").to(dt) for _ in range(2))
    table = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1)
    lens = torch.full((B,), page, dtype=torch.int32, device="cuda")
    q = torch.randn(N, G, 64, device="cuda").to(dt)
    for low, high in ((0, N), (0, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1)):
        starts = torch.tensor([high if i % 2 else low for i in range(B + 1)], dtype=torch.int32, device="cuda")
        out = torch.full((N + 2, G, 64), 7.0, dtype=dt, device="cuda")
        paged_prefill(q, starts, k, v, table, lens, G, out=out[1:-1])
        torch.cuda.synchronize()
        assert (out[0] == 7).all() and (out[-1] == 7).all()
        assert torch.isfinite(out).all()
