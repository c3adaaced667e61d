"""Launches of one kernel from several host threads with problems of different size: what one thread's call sets up for a
kernel must not take anything from another thread's."""

import threading
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


def test_plan_and_release_of_batches_above_48_kilobytes():
    """The large and the small batch both ask for more shared memory than a function has by itself; two threads launch them
    at the same time."""
    page, rounds, start = 16, 1000, threading.Barrier(2, timeout=60)

    def prepare(batch):
        seq = torch.arange(batch, dtype=torch.int32, device=DEV) % 40
        new, table = torch.ones_like(seq), torch.arange(batch * 3, dtype=torch.int32, device=DEV).view(batch, 3)
        done, free, count = (torch.zeros(n, dtype=t, device=DEV) for n, t in ((batch, torch.bool), (4, torch.int32), (1, torch.int32)))

        def run():
            start.wait()
            for _ in range(rounds):
                got = F.paged_kv_plan(seq, new, table, None, None, batch, page_size=page)
                F.paged_kv_release(done, seq, table, free, count, page_size=page)
            want = F.paged_kv_plan(seq, new, table, None, None, batch, page_size=page)
            return all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)

        return run

    calls = [prepare(batch) for batch in (4096, 3200)]
    with ThreadPoolExecutor(2) as pool:
        results = [pool.submit(call) for call in calls]
        assert all(r.result(timeout=120) for r in results)


def decode_call(batch, fp8, config):
    inp = W.make_paged_decode(5, 2, 8, 2, 128, 64, lens=[20, 64], device=DEV, dtype=torch.bfloat16)
    q = inp.q[:1].repeat(batch, 1, 1)
    lens = torch.full((batch,), 20, dtype=torch.int32, device=DEV)
    table = inp.block_table[:1].repeat(batch, 1)
    k, v, scales = inp.k, inp.v, {}
    if fp8:
        k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
        ones = torch.ones(k.shape[0] // 64, 2, device=DEV)
        scales = dict(k_scale=ones, v_scale=ones)
    return lambda: F.gqa_decode(q, k, v, real_seqlen_kv=lens, block_table=table, page_size=64, config=config, **scales)


@pytest.mark.parametrize("fp8", [False, True])
def test_tma_decode_of_a_large_and_of_a_small_batch(fp8):
    alternate(decode_call(300, fp8, None), decode_call(3, fp8, None))
    decode_call(3, fp8, None)()
    assert F.decode_last_kernel() == "tma"


@pytest.mark.parametrize("fp8", [False, True])
def test_cp_async_decode_of_a_large_and_of_a_small_batch(fp8):
    alternate(decode_call(300, fp8, {"tma": False}), decode_call(3, fp8, {"tma": False}))
    decode_call(3, fp8, {"tma": False})()
    assert F.decode_last_kernel() == "cp_async"


def test_two_prefills_over_an_fp8_cache_whose_launches_interleave(monkeypatch):
    """Another call of the same shape on the same stream between this call's read-back and its attention must leave this call's
    keys and values alone."""
    H, Hkv, D, page, T = 8, 2, 128, 64, 9

    def problem(seed):
        g = torch.Generator().manual_seed(seed)
        q, k, v = (torch.randn(T, h, D, generator=g).bfloat16().to(DEV) for h in (H, Hkv, Hkv))
        pages = [torch.randn(4 * page, Hkv, D, generator=g).to(torch.float8_e4m3fn).to(DEV) for _ in range(2)]
        one = torch.ones(1, device=DEV)
        cu, old, table = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 4, 9], [20, 9], [[1, 3], [0, 2]]))
        return lambda: F.gqa_prefill_paged_fp8_cache(q, k, v, *(p.clone() for p in pages), one, one, cu, old, table, 5, page_size=page)

    call, other = problem(0), problem(1)
    want, attend, inside = call(), F.gqa_prefill_paged, []

    def interleaved(*args, **kwargs):
        if not inside:
            inside.append(True)
            other()
        return attend(*args, **kwargs)

    monkeypatch.setattr(F, "gqa_prefill_paged", interleaved)
    got = call()
    assert inside and torch.equal(got, want)
