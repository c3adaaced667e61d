"""Launches of one kernel from several host threads with problems of different size: what one thread's call sets up for a
kernel must not take anything from another thread's."""

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from tileops_b200 import functional as F
from tileops_b200 import workloads as W

pytestmark = pytest.mark.gpu
DEV = "cuda"


def alternate(large, small):
    """One thread makes the large call, another the small one, then the first the large one again."""
    with ThreadPoolExecutor(1) as a, ThreadPoolExecutor(1) as b:
        first = a.submit(large).result()
        b.submit(small).result()
        again = a.submit(large).result()
        assert torch.equal(first, again)


@pytest.mark.parametrize("H,D", [(8, 128), (8, 64), (16, 128), (24, 64)])
def test_int4_decode_of_a_large_and_of_a_small_batch(H, D):
    pages = torch.zeros(4, 2, F.int4_page_bytes(16, D), dtype=torch.uint8, device=DEV)

    def call(batch):
        q = torch.ones(batch, H, D, dtype=torch.bfloat16, device=DEV)
        lens = torch.full((batch,), 20, dtype=torch.int32, device=DEV)
        table = torch.tensor([[1, 2]], dtype=torch.int32, device=DEV).repeat(batch, 1)
        return lambda: F.gqa_decode_int4(q, pages, lens, table, page_size=16)

    alternate(call(900), call(3))
