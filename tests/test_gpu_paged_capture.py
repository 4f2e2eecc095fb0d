"""What of PagedCache may not be captured."""
import pytest
import torch

from rotatek_amd.paged_cache import PagedCache

pytestmark = pytest.mark.gpu


def test_counts_are_not_captured():
    cache = PagedCache(1, 2, 64, pages=8, page=8, requests=2, max_tokens=32)
    cache.begin([9, 3])
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="capture"):
            cache.begin([8, 8])
        with pytest.raises(RuntimeError, match="capture"):
            cache.free(0)
    assert (cache.length(0), cache.length(1), cache.free_pages) == (9, 3, 5)
    graph.replay()
    assert cache.lens.tolist() == [9, 3] and x.tolist() == [1.0] * 4
    assert cache.begin([1, 1]) == 2 and cache.lens.tolist() == [10, 4]
