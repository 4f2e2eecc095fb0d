"""Shared-prefix calls between the other tests' sizes: heads of odd width, more
heads to a KV head than a block of queries, long texts in every format, all with
waves that take queries."""
import pytest
import torch

import test_gpu_shared_prefix as shared

pytestmark = pytest.mark.gpu

FORMATS = [("plain", torch.float16), ("mx8", torch.bfloat16), ("mx8", torch.float16), ("mx4", torch.bfloat16)]


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("case", [
    (150, 4, 1, 33, 70, 20, 40, 9, [9, 0]), (150, 4, 1, 127, 65, 127, 64, 3, [3, 0, 1]),
    (200, 4, 1, 1, 64, 1, 65, 2, None),
    (160, 4, 1, 57, 1, 0, 0, 33, [33, 32]),
])
def test_odd_heads_of_many_requests(case, fmt, dtype):
    print(f"[case] {case} {fmt} {dtype}", flush=True)
    shared._check(shared._case(*case[:8], dtype, fmt, seed=sum(case[:7]), lens=case[8]))


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("case", [
    (4, 160, 2, 128, 100, 32, 70, 20, [20, 0, 1]),     # 80 heads to a KV head
    (9, 65, 1, 128, 64, 0, 0, 5, [5, 0]), (70, 17, 1, 64, 64, 64, 1, 40, [40, 39, 0]),
])
def test_many_heads_to_a_kv_head(case, fmt, dtype):
    print(f"[case] {case} {fmt} {dtype}", flush=True)
    shared._check(shared._case(*case[:8], dtype, fmt, seed=sum(case[:7]), lens=case[8]))


@pytest.mark.parametrize("fmt,dtype", FORMATS)
def test_texts_past_the_joining_launch(fmt, dtype):
    case = (33, 4, 1, 128, 90, 32, 40, 4099, [4099, 0, 4096, 1, 31])
    print(f"[case] {case} {fmt} {dtype}", flush=True)
    shared._check(shared._case(*case[:8], dtype, fmt, seed=9, lens=case[8]))
