"""The plan of a serving step, the per-head norm with the rotation and the append, and the 4-bit cache's append and
read-back, against the CPU oracle (Python integers, 64 bits, and the quantiser in the 32-bit arithmetic it is defined in).

Integers, codes, scales, offsets and read-back values are compared bit for bit.  The norm and rotation round once, to the
output's 16 bits (eps / 2 of the value, and half of the smallest subnormal); before that, in fp32, a row's sum of squares has a
relative error below (D / lanes + log2 lanes + 2) 2^-24 < 2^-19, its rsqrt and the three products add 2^-22, the angle
(fraction of a turn rounded to 2^-25, sincospif to 2 ulp) 2^-21 of the larger of the two rotated values: together below
2^-18 of the row's largest value, times 1 + 2^-6 for the final rounding of a value that lies beyond a border.
"""

import random

import pytest
import torch

from oracle import paged_kv_oracle as O
from tileops_b200 import functional as F
from tileops_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- plan -------------------------------------------------------------------------------------------------------------
def check_plan(seq, new, width, page, free_count=None, total=None, seed=0, host_pages=False, inplace=False):
    rng = random.Random(seed)
    B = len(seq)
    held = [max(0, min(width, -(-max(s, 0) // page))) for s in seq]
    wanted = sum(max(0, -(-(s + n) // page) - -(-s // page)) for s, n in zip(seq, new) if s >= 0 and n >= 0)
    pool = sum(held) + wanted + 5
    ids = list(range(pool))
    rng.shuffle(ids)
    table = [[-7] * width for _ in range(B)]
    at = 0
    for b in range(B):
        cells = width if host_pages else held[b]
        for j in range(cells):
            table[b][j] = ids[at % pool]
            at += 1
    free = ids[at:] if not host_pages else None
    count = (len(free) if free_count is None else free_count) if not host_pages else None
    total = sum(max(n, 0) for n in new) if total is None else total
    want = O.plan_ref(seq, new, table, free, count, total, page)
    t_seq, t_table = i32(seq), i32(table)
    t_free = None if host_pages else i32(free if free else [0])[:len(free)]
    t_count = None if host_pages else i32([count])
    op = ops.PagedKVCachePlanFwdOp(B, width, page)
    got = op(t_seq, i32(new), t_table, t_free, t_count, total, inplace=inplace)
    assert t_table.tolist() == want[0]
    assert got.cu_seqlens_q.tolist() == want[1]
    assert got.slot_mapping.tolist() == want[2]
    assert got.positions.tolist() == want[3]
    assert got.seq_lens.tolist() == want[4]
    assert got.granted.tolist() == want[6]
    if not host_pages:
        assert got.free_count.tolist() == [want[5]]
        assert t_free.tolist() == free
    if inplace:
        assert t_seq.tolist() == want[4] and t_count.tolist() == [want[5]]
    else:
        assert t_seq.tolist() == seq
    return got


@pytest.mark.parametrize("page", [1, 16, 48, 128])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan_small_batches(page, inplace):
    check_plan([0], [1], 3, page, inplace=inplace)
    check_plan([page], [1], 3, page, inplace=inplace)
    check_plan([page - 1, 0, 2 * page, page + 1], [1, 2 * page + 1, 0, 1], 4, page, inplace=inplace, seed=1)


def test_plan_requests_without_new_tokens_and_rows_behind_the_last():
    check_plan([5, 0, 0, 33], [0, 0, 0, 0], 4, 16, total=6)
    check_plan([5, 0, 0, 33], [0, 3, 0, 0], 4, 16, total=9)
    check_plan([5, 0, 0, 33], [0, 3, 0, 4], 4, 16, total=4)       # fewer rows than tokens: the first rows only


def test_plan_refuses_lengths_that_make_no_sense_one_by_one():
    check_plan([-1, 3, 60, 10, 2 ** 31 - 100], [2, -4, 5, 6, 9], 4, 16)


@pytest.mark.parametrize("free", [0, 1, 2, 3, 4, 100, -3])
def test_plan_grants_in_order_while_the_stack_lasts(free):
    check_plan([16, 16, 7, 32, 16], [1, 17, 4, 16, 1], 6, 16, free_count=free, seed=3)


@pytest.mark.parametrize("B,most,page", [(513, 9, 16), (1025, 40, 32), (4096, 8, 16), (3, 9000, 64)])
def test_plan_large_batches(B, most, page):
    rng = random.Random(B)
    seq = [rng.randint(0, 300) for _ in range(B)]
    new = [rng.choice([0, 1, 1, rng.randint(1, most)]) for _ in range(B)]
    check_plan(seq, new, -(-(300 + most) // page), page, seed=B)
    check_plan(seq, new, -(-(300 + most) // page), page, seed=B, total=sum(new) + 3, inplace=True)


def test_plan_with_pages_that_the_host_manages():
    check_plan([0, 17, 40], [5, 1, 30], 5, 16, host_pages=True)
    check_plan([0, 17, 79], [5, 1, 30], 5, 16, host_pages=True)


def test_plan_reads_a_table_with_a_row_stride():
    wide = i32([[3, 9, 1, 4, 8], [2, 7, 6, 5, 0]])
    got = ops.PagedKVCachePlanFwdOp(2, 3, 16)(i32([17, 30]), i32([2, 5]), wide[:, 1:4], None, None, 7)
    assert got.slot_mapping.tolist() == [1 * 16 + 1, 1 * 16 + 2, 6 * 16 + 14, 6 * 16 + 15, 5 * 16, 5 * 16 + 1, 5 * 16 + 2]


def test_release_returns_pages_and_the_next_plan_takes_them():
    B, W, page = 5, 4, 16
    seq, table = i32([33, 0, 16, 64, 5]), i32([[10, 11, 12, -1], [-1] * 4, [13, -1, -1, -1], [14, 15, 16, 17], [18, -1, -1, -1]])
    free, count = i32([20, 21] + [0] * 9), i32([2])
    release = ops.PagedKVCacheReleaseFwdOp(B, W, page)
    release(torch.tensor([True, True, False, True, False], device=DEV), seq, table, free, count)
    assert seq.tolist() == [0, 0, 16, 0, 5]
    assert count.tolist() == [9]
    assert free.tolist()[:9] == [20, 21, 12, 11, 10, 17, 16, 15, 14]
    # the same request twice gives nothing more
    release(torch.tensor([True, True, False, True, False], device=DEV), seq, table, free, count)
    assert count.tolist() == [9]
    plan = ops.PagedKVCachePlanFwdOp(B, W, page)(seq, i32([20, 0, 1, 0, 0]), table, free, count, 21, inplace=True)
    assert table.tolist()[0][:2] == [14, 15] and table.tolist()[2][1] == 16
    assert count.tolist() == [6] and plan.seq_lens.tolist() == [20, 0, 17, 0, 5]


def test_release_never_writes_behind_the_stack():
    seq, table = i32([64]), i32([[1, 2, 3, 4]])
    whole = i32([9, 9, 9, 9, 9])
    count = i32([1])
    ops.PagedKVCacheReleaseFwdOp(1, 4, 16)(torch.tensor([True], device=DEV), seq, table, whole[:3], count)
    assert whole.tolist() == [9, 4, 3, 9, 9] and count.tolist() == [3]


def test_plan_in_a_graph_replays_a_decode_loop():
    page, W = 16, 6
    seq, new, table = i32([15, 31, 0]), i32([1, 1, 1]), i32([[0] + [-1] * 5, [1, 2] + [-1] * 4, [-1] * 6])
    free, count = i32(list(range(20, 3, -1))), i32([17])
    op = ops.PagedKVCachePlanFwdOp(3, W, page)
    op(seq.clone(), new, table.clone(), free, count.clone(), 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = op(seq, new, table, free, count, 3, inplace=True)
    state = ([15, 31, 0], [[0] + [-1] * 5, [1, 2] + [-1] * 4, [-1] * 6], 17)
    for _ in range(40):
        graph.replay()
        want = O.plan_ref(state[0], [1, 1, 1], state[1], free.tolist(), state[2], 3, page)
        assert plan.slot_mapping.tolist() == want[2] and plan.positions.tolist() == want[3]
        assert table.tolist() == want[0] and seq.tolist() == want[4] and count.tolist() == [want[5]]
        state = (want[4], want[0], want[5])


# ---- norm and rotation --------------------------------------------------------------------------------------------------
def norm_tolerance(ref, dtype):
    top = ref.abs().amax(-1, keepdim=True)
    return (1 + 2 ** -6) * ref.abs() * torch.finfo(dtype).eps / 2 + top * 2 ** -18 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_within(got, ref, tol, what):
    off = (got.double().cpu() - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float((off / tol.clamp(min=1e-300)).max())} tolerances"


def qkv(T, H, Hkv, D, dtype, seed, fused=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H + 2 * Hkv, D, generator=g) * torch.exp(torch.randn(T, H + 2 * Hkv, 1, generator=g))
    x = x.to(dtype).to(DEV)
    parts = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(DEV) for _ in range(2)]
    return (*(p if fused else p.contiguous() for p in parts), *w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,Hkv,D,rotary", [(1, 1, 1, 64, 64), (3, 32, 8, 128, 128), (5, 7, 1, 80, 32), (2, 3, 3, 256, 64),
                                              (17, 5, 2, 96, 96), (4, 4, 2, 8, 0), (3, 2, 1, 40, 16), (2, 2, 2, 192, 192),
                                              (130, 20, 5, 64, 64)])
def test_norm_rope_matches_64_bits(T, H, Hkv, D, rotary, dtype):
    q, k, _, qw, kw = qkv(T, H, Hkv, D, dtype, T + D)
    if D != 96:
        qw, kw = qw.to(dtype), kw.to(dtype)      # D = 96: fp32 weights
    pos = torch.randint(0, 200_000, (T,), dtype=torch.int32)
    q2, k2 = ops.QKNormRopeFwdOp(H, Hkv, D, rotary)(q, k, qw, kw, pos.to(DEV))
    for got, x, w in ((q2, q, qw), (k2, k, kw)):
        ref = O.norm_rope_ref(x.cpu(), w.cpu(), pos, rotary, 1e-6)
        assert got.dtype == dtype and got.is_contiguous()
        assert_within(got, ref, norm_tolerance(ref, dtype), f"{T} {H} {Hkv} {D} {rotary}")


@pytest.mark.parametrize("T", [600, 1021, 2500])
@pytest.mark.parametrize("H,Hkv,D,rotary", [(1, 1, 64, 64), (7, 1, 128, 128), (20, 5, 80, 32), (3, 3, 96, 96), (2, 1, 256, 64),
                                            (32, 8, 128, 128), (5, 2, 8, 0)])
def test_many_tokens_share_blocks(T, H, Hkv, D, rotary):
    """Batches large enough for blocks of several tokens: the whole call equals calls on pieces of it (one token a block),
    which the tests above hold to 64 bits; nothing but the rows is written."""
    dtype = torch.bfloat16
    q, k, v, qw, kw = qkv(T, H, Hkv, D, dtype, T, fused=True)
    pos = torch.randint(0, 9999, (T,), dtype=torch.int32, device=DEV)
    pool = T + 5
    slots = torch.randperm(pool, device=DEV)[:T].to(torch.int32)
    slots[T // 3] = -1
    op = ops.QKNormRopeKVCacheAppendFwdOp(H, Hkv, D, rotary)
    pages = [torch.zeros(pool, Hkv, D, dtype=dtype, device=DEV) for _ in range(4)]
    q1, k1 = op(q, k, v, qw, kw, pos, slots, pages[0], pages[1], return_k=True)
    for i in range(0, T, 200):
        j = slice(i, i + 200)
        q2, k2 = op(q[j], k[j], v[j], qw, kw, pos[j], slots[j], pages[2], pages[3], return_k=True)
        assert torch.equal(q1[j], q2) and torch.equal(k1[j], k2)
    assert torch.equal(pages[0], pages[2]) and torch.equal(pages[1], pages[3])
    if D in (64, 128):
        page = 16
        four = [torch.zeros(-(-pool // page), Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV) for _ in range(3)]
        op4, append = ops.QKNormRopeInt4KVCacheAppendFwdOp(H, Hkv, D, page, rotary), ops.Int4KVCacheAppendFwdOp(Hkv, D, page)
        assert torch.equal(op4(q, k, v, qw, kw, pos, slots, four[0]), q1)
        append(k1, v, slots, four[1])
        for i in range(0, T, 200):
            j = slice(i, i + 200)
            append(k1[j], v[j], slots[j], four[2])
        assert torch.equal(four[0], four[1]) and torch.equal(four[1], four[2])


def test_norm_rope_reads_parts_of_one_projection_and_odd_strides():
    T, H, Hkv, D = 9, 6, 2, 128
    q, k, v, qw, kw = qkv(T, H, Hkv, D, torch.bfloat16, 5, fused=True)
    pos = torch.arange(T, dtype=torch.int32, device=DEV) * 31
    op = ops.QKNormRopeFwdOp(H, Hkv, D)
    want = op(q.contiguous(), k.contiguous(), qw, kw, pos)
    got = op(q, k, qw, kw, pos)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a head-major tensor, and rows that start off the 16-byte boundary
    hm = q.transpose(0, 1).contiguous().transpose(0, 1)
    off = torch.empty(T * H * D + 1, dtype=q.dtype, device=DEV)[1:].view(T, H, D).copy_(q)
    every_other = torch.zeros(T, H, 2 * D, dtype=q.dtype, device=DEV)[..., ::2].copy_(q)
    shared = k[:, :1].expand(T, Hkv, D)
    for x in (hm, off, every_other):
        assert torch.equal(op(x, k, qw, kw, pos)[0], want[0])
    assert torch.equal(op(q, shared, qw, kw, pos)[1], op(q, shared.contiguous(), qw, kw, pos)[1])


def test_norm_rope_without_weights_with_frequencies_of_its_own_and_at_far_positions():
    T, H, Hkv, D = 6, 4, 1, 64
    q, k, _, _, _ = qkv(T, H, Hkv, D, torch.float16, 8)
    freq = torch.rand(16, dtype=torch.float64)
    pos = torch.tensor([0, 1, 2 ** 20 - 1, 2 ** 24 + 1, 2 ** 31 - 1, -5], dtype=torch.int32)
    q2, k2 = ops.QKNormRopeFwdOp(H, Hkv, D, 32, inv_freq=freq, eps=0.5)(q, k, None, None, pos.to(DEV))
    for got, x in ((q2, q), (k2, k)):
        ref = O.norm_rope_ref(x.cpu(), None, pos, 32, 0.5, inv_freq=freq)
        assert_within(got, ref, norm_tolerance(ref, torch.float16), "far positions")


def test_norm_rope_of_zero_huge_and_nan_rows():
    x = torch.randn(5, 2, 64).to(torch.bfloat16).to(DEV)
    x[0] = 0
    x[1] *= 1e18                       # squares stay below the largest fp32
    x[2, 0, 5] = float("nan")
    x[3, 1, 7] = float("inf")
    pos = torch.arange(5, dtype=torch.int32, device=DEV)
    q2, k2 = ops.QKNormRopeFwdOp(2, 2, 64)(x, x, None, None, pos)
    assert torch.equal(torch.nan_to_num(q2), torch.nan_to_num(k2))
    assert (q2[0] == 0).all()
    ref = O.norm_rope_ref(x.cpu(), None, pos.cpu(), 64, 1e-6)
    for t, h in ((1, 0), (1, 1), (2, 1), (3, 0), (4, 0), (4, 1)):
        assert_within(q2[t, h], ref[t, h], norm_tolerance(ref[t, h], torch.bfloat16), f"row {t} {h}")
    assert q2[2, 0].isnan().all() and q2[3, 1].isnan().any()


def test_empty_batches():
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    none = i32([])
    q2, k2 = ops.QKNormRopeFwdOp(2, 2, 64)(e, e, None, None, none)
    assert q2.shape == k2.shape == e.shape
    pages = torch.zeros(1, 2, 16 * 72, dtype=torch.uint8, device=DEV)
    ops.Int4KVCacheAppendFwdOp(2, 64, 16)(e, e, none, pages)
    k, v = ops.Int4KVCacheGatherFwdOp(2, 64, 16)(pages, i32([[0]]), i32([0, 0]), 0)
    assert k.shape == v.shape == (0, 2, 64) and not pages.any()


# ---- append to a 16-bit and to a 4-bit cache ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,Hkv,D,rotary", [(1, 8, 1, 128, 128), (37, 6, 3, 64, 32), (6, 10, 5, 80, 80), (5, 2, 1, 256, 256)])
def test_append_to_a_16_bit_cache(T, H, Hkv, D, rotary, dtype):
    q, k, v, qw, kw = qkv(T, H, Hkv, D, dtype, D, fused=True)
    pos = torch.arange(T, dtype=torch.int32, device=DEV) + 100
    pool = 64
    slots = torch.randperm(pool)[:T].to(torch.int32)
    if T > 3:
        slots[1], slots[3] = -1, pool       # neither is a row of the pool
    kp = torch.randn(pool, Hkv, D).to(dtype).to(DEV)
    vp = torch.randn(pool, Hkv, D).to(dtype).to(DEV)
    k_want, v_want = kp.clone(), vp.clone()
    q_want, k_new = ops.QKNormRopeFwdOp(H, Hkv, D, rotary)(q, k, qw, kw, pos)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pool:
            k_want[s], v_want[s] = k_new[t], v[t]
    op = ops.QKNormRopeKVCacheAppendFwdOp(H, Hkv, D, rotary)
    q2 = op(q, k, v, qw, kw, pos, slots.to(DEV), kp, vp)
    assert torch.equal(q2, q_want) and torch.equal(kp, k_want) and torch.equal(vp, v_want)
    q3, k3 = op(q, k, v, qw, kw, pos, slots.to(DEV), kp, vp, return_k=True)
    assert torch.equal(q3, q_want) and torch.equal(k3, k_new)


def special_rows(T, Hkv, D, dtype, seed):
    """Ordinary rows, and rows where a quantiser can go wrong."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, Hkv, D, generator=g) * torch.exp(2 * torch.randn(T, Hkv, 1, generator=g))).to(dtype)
    big = torch.finfo(dtype).max
    rows = x.view(T * Hkv, D)
    makers = [lambda r: r.zero_(), lambda r: r.fill_(1.25), lambda r: r.fill_(-3.0), lambda r: r[1:].zero_(),
              lambda r: r.copy_(torch.arange(D) % 16), lambda r: r.copy_((torch.arange(D) % 31) * 0.5),
              lambda r: r.mul_(1e-6), lambda r: r.copy_(torch.randn(D, generator=g) * 3e-8), lambda r: r[3:5].fill_(big),
              lambda r: r[0:1].fill_(float("inf")), lambda r: r[D - 1:].fill_(float("-inf")),
              lambda r: r[2:3].fill_(float("nan")), lambda r: r.fill_(big), lambda r: r[::2].fill_(-big)]
    for i, make in enumerate(makers):
        if 2 * i + 1 < T * Hkv:
            make(rows[2 * i])
            rows[2 * i + 1] = rows[2 * i]
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page,Hkv,T", [(64, 16, 1, 31), (128, 48, 3, 40), (64, 64, 2, 1), (128, 128, 1, 257)])
def test_int4_append_and_read_back_bit_for_bit(D, page, Hkv, T, dtype):
    pool = -(-T // page) + 2
    k, v = special_rows(T, Hkv, D, dtype, 3), special_rows(T, Hkv, D, dtype, 4)
    g = torch.Generator().manual_seed(5)
    slots = torch.randperm(pool * page, generator=g)[:T].to(torch.int32)
    if T > 9:
        slots[4], slots[9] = -1, pool * page
    want = torch.randint(0, 256, (pool, Hkv, F.int4_page_bytes(page, D)), dtype=torch.uint8, generator=g)
    got = want.to(DEV)
    O.store_ref(want, k, v, slots, page)
    ops.Int4KVCacheAppendFwdOp(Hkv, D, page)(k.to(DEV), v.to(DEV), slots.to(DEV), got)
    # NaN has many bit patterns: parameters that are NaN on both sides compare equal
    a, b = (F.int4_cache_views(x.cpu(), page, D) for x in (got, want))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(a[2].isnan(), b[2].isnan())
    assert torch.equal(torch.nan_to_num(a[2], nan=1.0), torch.nan_to_num(b[2], nan=1.0))
    # read back: one request whose pages are the pool in an order of its own
    table = torch.randperm(pool, generator=g)
    total = pool * page
    gk, gv = ops.Int4KVCacheGatherFwdOp(Hkv, D, page, dtype)(got, i32([table.tolist()]), i32([0, total]), total)
    rk, rv, _ = O.rows_ref(got.cpu(), table, total, page, D)
    for x, r in ((gk, rk), (gv, rv)):
        r = r.float().to(dtype)
        x = x.cpu()
        assert torch.equal(x.isnan(), r.isnan())
        assert torch.equal(torch.nan_to_num(x, nan=0.0), torch.nan_to_num(r, nan=0.0))


def test_int4_values_are_within_half_a_step_of_the_row():
    # half a step, and 15 steps times the scale's rounding (2^-11 of it, or half of the smallest float16 subnormal), the
    # read-back's rounding (bf16: 2^-8 of the value) and, where the offset is no float16, its rounding
    T, Hkv, D, page = 64, 2, 128, 16
    x = (torch.randn(T, Hkv, D) * torch.exp(torch.randn(T, Hkv, 1))).to(torch.bfloat16)
    pages = torch.zeros(T // page, Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    ops.Int4KVCacheAppendFwdOp(Hkv, D, page)(x.to(DEV), -x.to(DEV), i32(list(range(T))), pages)
    k, v = ops.Int4KVCacheGatherFwdOp(Hkv, D, page)(pages, i32([list(range(T // page))]), i32([0, T]), T)
    x = x.double()
    step = (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)) / 15
    tol = step / 2 + 15 * (step * 2 ** -11 + 2 ** -25) + x.abs() * 2 ** -11 + (x.abs() + step) * 2 ** -8
    assert_within(k, x, tol, "k")
    assert_within(v, -x, tol, "v")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_fused_append_equals_norm_then_append(D, dtype):
    T, H, Hkv, page, pool = 29, 10, 5, 32, 3
    q, k, v, qw, kw = qkv(T, H, Hkv, D, dtype, D, fused=True)
    pos = torch.randint(0, 9000, (T,), dtype=torch.int32, device=DEV)
    slots = torch.randperm(pool * page)[:T].to(torch.int32).to(DEV)
    slots[6] = -1
    a = torch.zeros(pool, Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    b = a.clone()
    q1, k1 = ops.QKNormRopeFwdOp(H, Hkv, D)(q, k, qw, kw, pos)
    ops.Int4KVCacheAppendFwdOp(Hkv, D, page)(k1, v, slots, a)
    q2 = ops.QKNormRopeInt4KVCacheAppendFwdOp(H, Hkv, D, page)(q, k, v, qw, kw, pos, slots, b)
    assert torch.equal(q1, q2) and torch.equal(a, b)


def test_gather_of_ragged_requests_leaves_the_rest_alone():
    D, page, Hkv = 128, 16, 2
    lens = [0, 5, 16, 1, 40, 0]
    pool = 12
    pages = torch.randint(0, 256, (pool, Hkv, F.int4_page_bytes(page, D)), dtype=torch.uint8, device=DEV)
    F.int4_cache_views(pages, page, D)[2].copy_(torch.randn(pool, Hkv, 1, 16, 4))
    table = torch.full((len(lens), 4), 99, dtype=torch.int32)     # entries behind a request's pages are not read
    ids = torch.randperm(pool)
    at = 0
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            table[b, j] = int(ids[at])
            at += 1
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    total = cu[-1] + 7
    out = tuple(torch.full((total, Hkv, D), 77.0, dtype=torch.float16, device=DEV) for _ in range(2))
    F.int4_cache_gather(pages, table.to(DEV), i32(cu), total, dim=D, page_size=page, dtype=torch.float16, out=out)
    for part, x in enumerate(out):
        want = torch.cat([O.rows_ref(pages.cpu(), table[b], n, page, D)[part] for b, n in enumerate(lens) if n])
        assert torch.equal(x[:cu[-1]].cpu(), want.float().half())
        assert (x[cu[-1]:] == 77).all()
    # a page id outside the pool reads as NaN, and only its own tokens do
    table[4, 1] = pool
    F.int4_cache_gather(pages, table.to(DEV), i32(cu), total, dim=D, page_size=page, dtype=torch.float16, out=out)
    nan = out[0].isnan().all(-1).all(-1).cpu()
    assert nan[cu[4] + 16:cu[4] + 32].all() and int(nan.sum()) == 16


def test_gather_reads_no_row_that_the_chunk_does_not_have():
    D, page, Hkv = 64, 16, 2
    pages = torch.zeros(4, Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    table = i32([[0, 1], [2, 3]])
    new = torch.randn(8, Hkv, D, device=DEV).bfloat16()
    # request 0: 3 cached and 4 new rows; request 1: its lengths ask for rows behind the chunk's 8
    k, _ = F.int4_cache_gather(pages, table, i32([0, 7, 20]), 20, dim=D, page_size=page, dtype=torch.bfloat16,
                               cache_seqlens=i32([3, 5]), cu_seqlens_new=i32([0, 4, 8]), k_new=new, v_new=new)
    assert (k[:3] == 0).all() and torch.equal(k[3:7], new[:4]) and (k[7:12] == 0).all() and torch.equal(k[12:16], new[4:])
    assert k[16:].isnan().all()
    # a negative length asks for rows in front of them
    k, _ = F.int4_cache_gather(pages, table, i32([0, 7, 20]), 20, dim=D, page_size=page, dtype=torch.bfloat16,
                               cache_seqlens=i32([0, 5]), cu_seqlens_new=i32([-3, 4, 8]), k_new=new, v_new=new)
    assert k[:3].isnan().all() and torch.equal(k[3:7], new[:4])


def test_calls_on_another_stream_and_in_a_graph():
    T, H, Hkv, D, page = 33, 8, 2, 64, 16
    q, k, v, qw, kw = qkv(T, H, Hkv, D, torch.bfloat16, 1, fused=True)
    pos, slots = torch.arange(T, dtype=torch.int32, device=DEV), torch.randperm(48, device=DEV)[:T].to(torch.int32)
    pages = torch.zeros(3, Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    append, gather = ops.QKNormRopeInt4KVCacheAppendFwdOp(H, Hkv, D, page), ops.Int4KVCacheGatherFwdOp(Hkv, D, page)
    table, cu = i32([[0, 1, 2]]), i32([0, 48])

    def step():
        return append(q, k, v, qw, kw, pos, slots, pages), *gather(pages, table, cu, 48)

    want = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pages.zero_()
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    pages.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- page ids that the pool does not have ------------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("bad", [2 ** 30, -2 ** 31, 2 ** 31 - 1, 2 ** 28, 2 ** 27, -1, -7])
def test_a_slot_of_a_page_that_32_bits_do_not_hold_is_none(bad, page):
    """id * page_size is formed in 64 bits: a page that no pool has must not become a row of another one."""
    old, new = page + 5, 3
    table = i32([[3, bad], [5, 6]])
    plan = ops.PagedKVCachePlanFwdOp(2, 2, page)(i32([old, old]), i32([new, new]), table, None, None, 2 * new)
    slots = plan.slot_mapping.tolist()
    assert slots[new:] == [6 * page + 5 + i for i in range(new)]
    fits = bad >= 0 and bad * page + page <= 2 ** 31
    assert slots[:new] == ([bad * page + 5 + i for i in range(new)] if fits else [-1] * new)
    # an append to these slots changes no page but its own
    D, Hkv, pool = 64, 2, 8
    pages = torch.full((pool, Hkv, F.int4_page_bytes(page, D)), 7, dtype=torch.uint8, device=DEV)
    k = torch.randn(2 * new, Hkv, D, device=DEV).bfloat16()
    ops.Int4KVCacheAppendFwdOp(Hkv, D, page)(k, k, plan.slot_mapping, pages)
    changed = (pages != 7).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [6]
    # the same from the stack
    plan = ops.PagedKVCachePlanFwdOp(1, 2, page)(i32([page]), i32([2]), i32([[1, 0]]), i32([4, bad]), i32([2]), 2)
    assert plan.slot_mapping.tolist() == ([bad * page, bad * page + 1] if fits else [-1, -1])


# ---- values at the ends of the quantiser's range ------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
def test_float16_read_back_saturates(D):
    """15 steps of f16((65504 + 65504) / 15) = 8736 end 32 beyond the largest float16: the read-back must not overflow."""
    page, Hkv = 16, 1
    big = torch.finfo(torch.float16).max
    k = torch.zeros(4, Hkv, D, dtype=torch.float16)
    k[:, :, ::2], k[:, :, 1::2] = big, -big
    k[2:, 0, 3] = float("inf")
    v = -k
    v[3, 0, 5] = float("nan")
    pages = torch.zeros(1, Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    ops.Int4KVCacheAppendFwdOp(Hkv, D, page)(k.to(DEV), v.to(DEV), i32([0, 1, 2, 3]), pages)
    got_k, got_v = ops.Int4KVCacheGatherFwdOp(Hkv, D, page, torch.float16)(pages, i32([[0]]), i32([0, 4]), 4)
    assert torch.equal(got_k.cpu(), torch.nan_to_num(k, posinf=big))
    assert torch.equal(got_v[:3].cpu(), torch.nan_to_num(v[:3], neginf=-big)) and got_v[3].isnan().all()


def test_rows_whose_step_is_a_subnormal_keep_the_stated_bound():
    """Half a step, 15 times the rounding of the scale and the rounding of the offset and of the read-back, each 2^-11 of the
    value or 2^-25, half of float16's smallest subnormal; a step of 2^-25 or less has scale 0 and is all rounding."""
    T, D, page = 32, 64, 16
    g = torch.Generator().manual_seed(6)
    span = torch.logspace(-8, -3, T, dtype=torch.float64)[:, None, None]
    x = (torch.rand(T, 1, D, generator=g, dtype=torch.float64) * span).to(torch.float16)
    pages = torch.zeros(T // page, 1, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    ops.Int4KVCacheAppendFwdOp(1, D, page)(x.to(DEV), -x.to(DEV), i32(list(range(T))), pages)
    k, v = ops.Int4KVCacheGatherFwdOp(1, D, page, torch.float16)(pages, i32([[0, 1]]), i32([0, T]), T)
    x = x.double()
    step = (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)) / 15
    rounding = lambda y: torch.clamp(y.abs() * 2 ** -11, min=2 ** -25)  # noqa: E731
    tol = step / 2 + 15 * rounding(step) + rounding(x.amax(-1, keepdim=True)) + rounding(x.abs() + step)
    assert_within(k, x, tol, "k")
    assert_within(v, -x, tol, "v")


def test_plan_refuses_to_enter_pages_in_a_row_that_requests_share():
    shared = i32([[1, 2, 3]]).expand(2, 3)
    with pytest.raises(ValueError, match="must not overlap"):
        ops.PagedKVCachePlanFwdOp(2, 3, 16)(i32([0, 0]), i32([1, 1]), shared, i32([4, 5]), i32([2]), 2)
    # a table that is only read may be shared
    plan = ops.PagedKVCachePlanFwdOp(2, 3, 16)(i32([17, 3]), i32([1, 1]), shared, None, None, 2)
    assert plan.slot_mapping.tolist() == [2 * 16 + 1, 16 + 3]


def test_a_rotation_is_captured_after_its_first_call():
    T, H, Hkv, D = 3, 4, 2, 64
    q, k, _, qw, kw = qkv(T, H, Hkv, D, torch.bfloat16, 2)
    pos = i32([5, 6, 7])
    op = ops.QKNormRopeFwdOp(H, Hkv, D)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="call it once before the capture"):
        with torch.cuda.graph(graph):
            op(q, k, qw, kw, pos)
    want = op(q, k, qw, kw, pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op(q, k, qw, kw, pos)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
