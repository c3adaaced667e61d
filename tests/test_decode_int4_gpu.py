"""Single-token decode and chunked prefill over a paged cache held in 4 bits, against dequantise-then-attend in 64 bits.

Tolerance of the decode with an fp32 output, per (sequence, KV head), from the arithmetic the kernel may use:
  * P times the V scale is rounded to float16 before it meets the codes (0..15): 2^-11 * 15 max|vs|;
  * a score is a sum of D products accumulated in fp32 and scaled: off by at most 2^-19 A, A = scale * sum|q| *
    max(15 |ks| + |km|); a q below 2^-6 of its head's largest may be rounded to an integer of a scale where that is
    2^13 or more, which adds scale * 15 max|ks| * 2^-14 max|q| for each such value; with a softcap the capped score is off by
    2^-20 cap more; probabilities move by as much (relative) and the output by at most twice that times max|v|;
  * the row sums and the exponentials: 2^-16 max|v| at the lengths used here.
A 16-bit output adds half a step of its type.  The LSE is off by the score's error, 2^-16 and the rounding of its value.
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


def make(lens, H, Hkv, D, page, dtype=torch.bfloat16, seed=0, kscale=1.0, vscale=1.0, width=None, ragged_scale=False):
    """(q, pool, lens, table): every request has pages of its own in random order, slots without a token hold NaN
    parameters and codes of all ones, and table entries behind a request's pages are no page ids."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    pool = sum(need) + 2
    pages = torch.full((pool, Hkv, F.int4_page_bytes(page, D)), 255, dtype=torch.uint8, device=DEV)
    ids = torch.randperm(pool, generator=g)
    table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32)
    at = 0
    slots = []
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
        t = torch.arange(lens[b])
        slots.append(table[b].long()[t // page] * page + t % page)
    slots = torch.cat(slots).to(torch.int32)
    T = slots.numel()
    k = torch.randn(T, Hkv, D, generator=g) * kscale + 0.3
    v = torch.randn(T, Hkv, D, generator=g) * vscale - 0.7 * vscale
    if ragged_scale:      # tokens of very different size
        v = v * torch.exp(4 * torch.randn(T, Hkv, 1, generator=g))
    if T:
        F.int4_cache_append(k.to(dtype).to(DEV), v.to(dtype).to(DEV), slots.to(DEV), pages, page_size=page)
    q = torch.randn(len(lens), H, D, generator=g).to(dtype)
    return q.to(DEV), pages, i32(lens), table.to(DEV)


def tolerances(q, pages, lens, table, page, scale, softcap):
    """(absolute tolerance of o [B,H,1], of the LSE [B,H])."""
    B, H, D = q.shape
    Hkv = pages.shape[1]
    to, tl = torch.zeros(B, H, 1, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        _, v, params = O.rows_ref(pages, table[b], n, page, D)
        a = params.abs()
        for h in range(H):
            hk = h // (H // Hkv)
            A = scale * float(q[b, h].double().abs().sum()) * float((15 * a[:, hk, 0] + a[:, hk, 1]).max())
            x = q[b, h].double().abs()
            small = float((x < 2.0 ** -6 * x.max()).sum()) * 2.0 ** -14 * float(x.max())
            score = 2.0 ** -19 * A + scale * 15 * float(a[:, hk, 0].max()) * small + 2.0 ** -20 * softcap
            vmax = float(v[:, hk].abs().max())
            to[b, h] = 2.0 ** -11 * 15 * float(a[:, hk, 2].max()) + 2 * score * vmax + 2.0 ** -16 * vmax
            tl[b, h] = 1.4427 * score + 2.0 ** -16
    return to, tl


def check(lens, H, Hkv, D, page, dtype=torch.bfloat16, softcap=0.0, sm_scale=None, config=None, out_dtype=torch.float32, **kw):
    q, pages, t_lens, table = make(lens, H, Hkv, D, page, dtype, **kw)
    got, lse = F.gqa_decode_int4(q, pages, t_lens, table, page_size=page, softcap=softcap, sm_scale=sm_scale,
                                 return_lse=True, out_dtype=out_dtype, config=config)
    q, pages, table = q.cpu(), pages.cpu(), table.cpu()
    ref, ref_lse = O.decode_ref(q, pages, lens, table, page, sm_scale, softcap)
    scale = D ** -0.5 if sm_scale is None else abs(sm_scale)
    to, tl = tolerances(q, pages, lens, table, page, scale, softcap)
    if out_dtype != torch.float32:
        to = to + ref.abs() * torch.finfo(out_dtype).eps / 2 * (1 + 2 ** -6)
    empty = torch.tensor(lens) == 0
    got, lse = got.double().cpu(), lse.double().cpu()
    assert (got[empty] == 0).all() and (lse[empty] == -float("inf")).all()
    off = (got - ref).abs()
    assert (off <= to).all(), f"o off by {float((off / to.clamp(min=1e-30))[~empty].max()):.3g} tolerances"
    off = (lse - ref_lse).abs()[~empty]
    lim = (tl + ref_lse.abs().nan_to_num(posinf=0) * 2.0 ** -22)[~empty]
    assert (off <= lim).all(), f"LSE off by {float((off / lim).max()):.3g} tolerances"
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 700])
def test_one_request_of_every_awkward_length(n, D, dtype):
    check([n], 8, 2, D, 16, dtype, seed=n)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 256])
def test_ragged_requests_and_page_sizes(page):
    check([0, 1, page, page - 1, page + 1, 0, 3 * page + 7, 500], 16, 4, 128, page, seed=page)
    check([5, 2 * page, 0], 4, 4, 64, page, torch.float16, seed=page)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 1), (5, 5), (7, 1), (8, 1), (9, 1), (16, 1), (32, 2), (40, 8), (17, 1), (24, 1),
                                   (64, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_layouts(H, Hkv, D):
    check([33, 200, 0, 1], H, Hkv, D, 32, seed=H)


def test_all_requests_empty():
    got, lse = F.gqa_decode_int4(torch.randn(3, 8, 128, device=DEV).bfloat16(), torch.zeros(1, 2, 16 * 136, dtype=torch.uint8, device=DEV),
                                 i32([0, 0, -4]), i32([[0], [0], [0]]), page_size=16, return_lse=True)
    assert (got == 0).all() and (lse == -float("inf")).all()


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16])
def test_output_types(out_dtype):
    check([77, 300], 8, 2, 128, 16, torch.bfloat16, out_dtype=out_dtype)


@pytest.mark.parametrize("D", [64, 128])
def test_softcap_and_scale(D):
    check([100, 1, 37], 8, 2, D, 16, softcap=30.0, seed=1)
    check([100, 1, 37], 8, 2, D, 16, softcap=0.5, sm_scale=2.0, seed=2)
    check([100, 1, 37], 8, 2, D, 16, sm_scale=-0.3, seed=3)
    check([100, 1, 37], 8, 2, D, 16, sm_scale=0.0, seed=4)


@pytest.mark.parametrize("kscale,vscale", [(1e-4, 1e-4), (30.0, 1.0), (1.0, 1e-3), (1.0, 2000.0), (300.0, 1.0)])
@pytest.mark.parametrize("D", [64, 128])
def test_small_and_large_values(kscale, vscale, D):
    check([450, 20], 8, 2, D, 16, kscale=kscale, vscale=vscale, seed=7)


def test_tokens_of_very_different_size():
    check([900, 300], 8, 2, 128, 16, ragged_scale=True, seed=9)


def test_a_large_q_of_one_head_does_not_blur_the_others():
    q, pages, lens, table = make([300], 4, 1, 128, 16, torch.bfloat16, seed=3)
    alone = F.gqa_decode_int4(q, pages, lens, table, page_size=16, out_dtype=torch.float32)
    q[0, 1] *= 2.0 ** 20
    q[0, 2] *= 2.0 ** -20
    got = F.gqa_decode_int4(q, pages, lens, table, page_size=16, out_dtype=torch.float32)
    ref, _ = O.decode_ref(q.cpu(), pages.cpu(), [300], table.cpu(), 16)
    to, _ = tolerances(q.cpu(), pages.cpu(), [300], table.cpu(), 16, 128 ** -0.5, 0.0)
    for h in (0, 2, 3):
        assert ((got[0, h].double().cpu() - ref[0, h]).abs() <= to[0, h]).all()
    torch.testing.assert_close(got[0, 0], alone[0, 0], atol=float(to[0, 0]), rtol=0)


@pytest.mark.parametrize("lens,H,Hkv,D,page", [([5000], 8, 1, 128, 64), ([4097, 3, 2048], 32, 8, 128, 16), ([3000] * 5, 8, 2, 64, 128),
                                               ([1024] * 12, 16, 2, 128, 64), ([2500, 0, 2500], 16, 1, 64, 32)])
def test_long_contexts_split_over_blocks(lens, H, Hkv, D, page):
    check(lens, H, Hkv, D, page, seed=len(lens))


@pytest.mark.parametrize("seed", range(24))
def test_random_problems(seed):
    rng = random.Random(900 + seed)
    D, page = rng.choice([64, 128]), rng.choice([16, 32, 48, 64, 128, 256])
    Hkv, group = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 4, 5, 8, 11, 16])
    top = rng.choice([40, 400, 2500])
    lens = [rng.choice([0, 1, page, rng.randint(1, top)]) for _ in range(rng.choice([1, 2, 5, 19]))]
    check(lens, Hkv * group, Hkv, D, page, rng.choice([torch.bfloat16, torch.float16]), softcap=rng.choice([0.0, 20.0]), seed=seed)


def test_calls_are_bit_reproducible_and_independent_of_the_rest_of_the_batch():
    q, pages, lens, table = make([1500, 4000, 0, 700, 2222] * 6, 32, 8, 128, 16, seed=4)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    for _ in range(20):
        assert torch.equal(F.gqa_decode_int4(q, pages, lens, table, page_size=16), want)


def test_bad_pages_and_lengths_give_nan_and_stay_in_bounds():
    q, pages, lens, table = make([100, 40, 64, 500], 8, 2, 128, 16, seed=5, width=32)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    assert not want.isnan().any()
    for b, j, page_id in ((0, 6, pages.shape[0]), (3, 0, -1), (1, 1, -2 ** 31), (2, 3, 2 ** 31 - 1)):
        bad = table.clone()
        bad[b, j] = page_id
        got, lse = F.gqa_decode_int4(q, pages, lens, bad, page_size=16, return_lse=True)
        assert got[b].isnan().all() and lse[b].isnan().all()
        others = [x for x in range(4) if x != b]
        assert torch.equal(got[others], want[others])
    long = lens.clone()
    long[1] = 32 * 16 + 1
    got = F.gqa_decode_int4(q, pages, long, torch.where(table < pages.shape[0], table, 0), page_size=16)
    assert got[1].isnan().all() and not got[0].isnan().any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [32, 48, 64, 128, 256])
def test_a_bad_page_of_any_size_reaches_its_request_only(page, D):
    lens = [3 * page + 5, 700, 2 * page, 1]
    for H in (8, 12):
        q, pages, t_lens, table = make(lens, H, 2, D, page, seed=page, width=32)
        want = F.gqa_decode_int4(q, pages, t_lens, table, page_size=page)
        assert not want.isnan().any()
        for b, j in ((0, 3), (0, 1), (1, 0), (2, 1), (3, 0)):
            bad = table.clone()
            bad[b, j] = pages.shape[0]
            got = F.gqa_decode_int4(q, pages, t_lens, bad, page_size=page)
            assert got[b].isnan().all()
            others = [x for x in range(4) if x != b]
            assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("D", [64, 128])
def test_nan_in_a_cached_token_reaches_its_heads_only(D):
    q, pages, lens, table = make([50, 300], 8, 2, D, 16, seed=6)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    for token, column in ((7, 0), (7, 2), (299, 1), (0, 3)):
        b = 0 if token < 50 and token else 1
        bad = pages.clone()
        F.int4_cache_views(bad, 16, D)[2][int(table[b, token // 16]), 1, 0, token % 16, column] = float("nan")
        got = F.gqa_decode_int4(q, bad, lens, table, page_size=16)
        assert got[b, 4:].isnan().all(), (token, column)
        keep = torch.ones(2, 8, dtype=torch.bool, device=DEV)
        keep[b, 4:] = False
        assert torch.equal(got[keep], want[keep])


def test_tables_and_q_with_strides_of_their_own():
    q, pages, lens, table = make([100, 40], 8, 2, 128, 16, seed=8)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 3:3 + table.shape[1]] = table
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    for x in (q, qt, off):
        assert torch.equal(F.gqa_decode_int4(x, pages, lens, wide[:, 3:3 + table.shape[1]], page_size=16), want)


def test_graphs_have_scratch_of_their_own():
    q, pages, lens, table = make([3000, 2500, 777], 8, 2, 128, 16, seed=10)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(30):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    torch.cuda.synchronize()
    assert torch.equal(eager, want) and all(torch.equal(out, want) for _, out in graphs)
    # lengths change between replays
    lens.copy_(i32([1, 0, 776]))
    for graph, _ in graphs:
        graph.replay()
    assert all(torch.equal(out, F.gqa_decode_int4(q, pages, lens, table, page_size=16)) for _, out in graphs)


def test_a_stream_other_than_the_tensors_own():
    q, pages, lens, table = make([3000, 11], 8, 2, 128, 16, seed=11)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    side.synchronize()
    assert torch.equal(got, want)


# ---- the whole step, and the chunked prefill -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page,H,Hkv", [(128, 16, 8, 2), (64, 64, 6, 6)])
def test_a_serving_loop_of_plan_norm_append_attend_and_release(D, page, H, Hkv, dtype):
    """Requests of different length arrive, are prefilled in chunks, decode, finish and give their pages back; every
    output is compared with attention in 64 bits over the values the cache stands for."""
    rng = random.Random(17)
    B, W, pool = 3, 12, 30
    g = torch.Generator().manual_seed(2)
    pages = torch.full((pool, Hkv, F.int4_page_bytes(page, D)), 255, dtype=torch.uint8, device=DEV)
    seq, table = torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B, W, dtype=torch.int32, device=DEV)
    free, count = torch.randperm(pool, generator=g).to(torch.int32).to(DEV), i32([pool])
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype).to(DEV) for _ in range(2))
    plan_op, release = ops.PagedKVCachePlanFwdOp(B, W, page), ops.PagedKVCacheReleaseFwdOp(B, W, page)
    norm, append = ops.QKNormRopeFwdOp(H, Hkv, D), ops.QKNormRopeInt4KVCacheAppendFwdOp(H, Hkv, D, page)
    prefill = ops.GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp(B, H, Hkv, W, page, D)
    attend = ops.GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp(B, H, Hkv, pool * page, D, page)

    def qkv(T):
        x = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(DEV)
        return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]

    lens = [0, 0, 0]
    for step in range(9):
        if step in (0, 4):            # a chunk for some requests
            if step == 4:
                release(torch.tensor([False, True, False], device=DEV), seq, table, free, count)
                lens[1] = 0
            new = [rng.randint(1, 2 * page), rng.randint(1, 40), 0 if step else 5]
            T = sum(new)
            plan = plan_op(seq, i32(new), table, free, count, T, inplace=False)
            assert plan.granted.all()
            q, k, v = qkv(T)
            q, k = norm(q, k, qw, kw, plan.positions)
            o = prefill(q, k, v.contiguous(), pages, plan.cu_seqlens_q, seq, table, max(new))
            # rows see the cached tokens as the cache holds them, and the chunk as it is
            old, at = list(lens), 0
            for b, n in enumerate(new):
                kc, vc, _ = O.rows_ref(pages.cpu(), table[b].cpu(), old[b], page, D) if old[b] else (torch.zeros(0, Hkv, D).double(),) * 2 + (None,)
                kc, vc = (x.float().to(dtype).double() for x in (kc, vc))
                keys = torch.cat([kc, k[at:at + n].double().cpu()]).repeat_interleave(H // Hkv, 1)
                vals = torch.cat([vc, v[at:at + n].double().cpu()]).repeat_interleave(H // Hkv, 1)
                s = torch.einsum("ihd,jhd->hij", q[at:at + n].double().cpu(), keys) * D ** -0.5
                s.masked_fill_(torch.arange(old[b] + n)[None, :] > torch.arange(n)[:, None] + old[b], -float("inf"))
                ref = torch.einsum("hij,jhd->ihd", s.softmax(-1), vals)
                torch.testing.assert_close(o[at:at + n].double().cpu(), ref, atol=2e-2, rtol=1e-2)   # the prefill tests' own
                at += n
                lens[b] += n
            seq, count = plan.seq_lens.clone(), plan.free_count.clone()
            assert seq.tolist() == lens
        else:
            plan = plan_op(seq, i32([1] * B), table, free, count, B, inplace=True)
            assert plan.granted.all()
            q, k, v = qkv(B)
            q = append(q, k, v, qw, kw, plan.positions, plan.slot_mapping, pages)
            o = attend(q, pages, plan.seq_lens, table)
            lens = [n + 1 for n in lens]
            assert seq.tolist() == lens
            ref, _ = O.decode_ref(q.cpu(), pages.cpu(), lens, table.cpu(), page)
            to, _ = tolerances(q.cpu(), pages.cpu(), lens, table.cpu(), page, D ** -0.5, 0.0)
            to = to + ref.abs() * torch.finfo(dtype).eps / 2 * (1 + 2 ** -6)
            assert ((o.double().cpu() - ref).abs() <= to).all()


def test_prefill_reads_the_cache_as_gather_does_and_appends_as_append_does():
    B, H, Hkv, D, page, W = 3, 8, 2, 128, 16, 8
    old, new = [30, 0, 64], [20, 40, 1]
    q0, pages, _, table = make([a + b for a, b in zip(old, new)], H, Hkv, D, page, seed=12, width=W)
    table = torch.where(table < pages.shape[0], table, 0)
    T = sum(new)
    q = torch.randn(T, H, D).bfloat16().to(DEV)
    k, v = (torch.randn(T, Hkv, D).bfloat16().to(DEV) for _ in range(2))
    cu = i32([0, 20, 60, 61])
    op = ops.GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp(B, H, Hkv, W, page, D)
    before = pages.clone()
    o = op(q, k, v, pages, cu, i32(old), table, 40)
    want = before.clone()
    plan = ops.PagedKVCachePlanFwdOp(B, W, page)(i32(old), i32(new), table, None, None, T)
    ops.Int4KVCacheAppendFwdOp(Hkv, D, page)(k, v, plan.slot_mapping, want)
    assert torch.equal(pages, want)
    total = [a + b for a, b in zip(old, new)]
    kc, vc = ops.Int4KVCacheGatherFwdOp(Hkv, D, page)(before, table, i32([0, 30, 30, 94]), 94)
    k_all = torch.cat([kc[:30], k[:20], k[20:60], kc[30:], k[60:]])
    v_all = torch.cat([vc[:30], v[:20], v[20:60], vc[30:], v[60:]])
    cu_kv = i32([0, total[0], total[0] + total[1], sum(total)])
    ref = F.gqa_prefill_paged(q, k_all, v_all, None, None, cu, None, None, 40, cu_seqlens_kv=cu_kv)
    assert torch.equal(o, ref)


@pytest.mark.parametrize("chunk", [1, 2, 3, 7])
@pytest.mark.parametrize("H,D,page", [(8, 128, 16), (8, 64, 128), (32, 128, 128), (24, 64, 48)])
def test_fixed_runs_agree_with_the_partition_the_kernel_picks(H, D, page, chunk):
    lens = [700, 3000, 0, 1, 2049, 128]
    check(lens, H, 2, D, page, config={"chunk_tiles": chunk}, seed=chunk)


@pytest.mark.parametrize("lens,H,Hkv,D", [
    ([1300] * 60, 8, 8, 64),              # equal lanes, more than blocks, that no whole number per block fits
    ([700] * 37, 16, 4, 128),             # equal lanes, fewer than blocks
    ([640] * 8, 8, 4, 128),               # equal lanes that are cut into equal parts
    ([i % 151 for i in range(200)], 8, 4, 128),       # short lanes, some without a token, several per block
    ([i * 37 % 400 for i in range(90)], 24, 2, 64),   # the same with two head tiles
    ([1] * 64 + [3000], 8, 2, 128),       # one long request among very short ones
    ([60000], 4, 1, 128),                 # one lane cut over all blocks: more runs than a merge has in flight
    ([60000, 5], 32, 2, 64)])
def test_every_kind_of_partition(lens, H, Hkv, D):
    for dtype in (torch.bfloat16, torch.float16):
        check(lens, H, Hkv, D, 64, dtype, seed=len(lens))


def test_many_short_segments_per_block_are_bit_reproducible():
    q, pages, lens, table = make([2000, 1333, 128, 999] * 16, 16, 4, 128, 64, seed=14)
    for chunk in (1, 2, 5):
        want = F.gqa_decode_int4(q, pages, lens, table, page_size=64, config={"chunk_tiles": chunk})
        for _ in range(60):
            assert torch.equal(F.gqa_decode_int4(q, pages, lens, table, page_size=64, config={"chunk_tiles": chunk}), want)
    assert F.decode_status() == 0


@pytest.mark.parametrize("top", [4.1e37, 4.3e37, 1e38, 3.3e38])
@pytest.mark.parametrize("H,D", [(4, 128), (8, 64), (16, 128)])
def test_q_up_to_the_largest_bfloat16(H, D, top):
    """Heads whose largest |q| is near the type's end, with a scale that keeps their scores ordinary."""
    q, pages, lens, table = make([300, 45], H, 1, D, 16, torch.bfloat16, seed=13)
    q = (q.double() / q.double().abs().amax(-1, keepdim=True) * top).to(torch.bfloat16)
    sm_scale = 2.0 ** -124
    got, lse = F.gqa_decode_int4(q, pages, lens, table, page_size=16, sm_scale=sm_scale, out_dtype=torch.float32, return_lse=True)
    q, pages, table = q.cpu(), pages.cpu(), table.cpu()
    ref, ref_lse = O.decode_ref(q, pages, [300, 45], table, 16, sm_scale)
    to, tl = tolerances(q, pages, [300, 45], table, 16, sm_scale, 0.0)
    assert ((got.double().cpu() - ref).abs() <= to).all()
    assert ((lse.double().cpu() - ref_lse).abs() <= tl + ref_lse.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("H,D", [(4, 128), (8, 64), (16, 128)])
def test_scores_beyond_32_bits_do_not_pass_for_an_empty_sequence(H, D):
    """Scores of -infinity throughout are no softmax: NaN, as in the plain form, and not the zeros of an empty sequence."""
    page = 16
    pages = torch.zeros(400, 1, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    rows = torch.ones(400 * page, 1, D, dtype=torch.bfloat16, device=DEV)
    F.int4_cache_append(rows, rows, torch.arange(400 * page, dtype=torch.int32, device=DEV), pages, page_size=page)
    q = torch.full((4, H, D), -3e38, dtype=torch.bfloat16, device=DEV)
    q[1] = 1.0
    table = torch.arange(400, dtype=torch.int32, device=DEV).repeat(4, 1)
    o, lse = F.gqa_decode_int4(q, pages, i32([1, 40, 0, 6400]), table, page_size=page, return_lse=True)
    for b in (0, 3):
        assert o[b].isnan().all() and lse[b].isnan().all()
    assert (o[1] == 1).all() and (o[2] == 0).all() and (lse[2] == -float("inf")).all()


def chunk_problem(B, T, H=8, Hkv=2, D=128, page=16, W=2, pool=16, seed=0):
    """A pool whose every token holds values, tables of distinct pages, and the rows of a chunk."""
    g = torch.Generator().manual_seed(seed)
    pages = torch.zeros(pool, Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    rows = [torch.randn(pool * page, Hkv, D, generator=g).bfloat16().to(DEV) for _ in range(2)]
    F.int4_cache_append(*rows, torch.arange(pool * page, dtype=torch.int32, device=DEV), pages, page_size=page)
    table = torch.randperm(pool, generator=g)[:B * W].view(B, W).to(torch.int32).to(DEV)
    q, k, v = (torch.randn(T, h, D, generator=g).bfloat16().to(DEV) for h in (H, Hkv, Hkv))
    op = ops.GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp(B, H, Hkv, W, page, D)
    op.validate_inputs = False
    return op, q, k, v, pages, table


def test_two_prefills_whose_launches_interleave(monkeypatch):
    """Another call of the same shape on the same stream between this call's read-back and its attention, as a second host
    thread can make it, must leave this call's keys and values alone."""
    op, q, k, v, pages, table = chunk_problem(2, 9)
    cu, old = i32([0, 4, 9]), i32([20, 9])
    want = op(q, k, v, pages.clone(), cu, old, table, 5)
    other = chunk_problem(2, 9, seed=1)
    attend, inside = F.gqa_prefill_paged, []

    def interleaved(*args, **kwargs):
        if not inside:
            inside.append(True)
            other[0](*other[1:5], cu, old, other[5], 5)
        return attend(*args, **kwargs)

    monkeypatch.setattr(F, "gqa_prefill_paged", interleaved)
    got = op(q, k, v, pages, cu, old, table, 5)
    assert inside and torch.equal(got, want)


@pytest.mark.parametrize("cached", [33, 90, 2 ** 31 - 1, -1, -7, -2 ** 31])
def test_prefill_of_a_request_longer_than_its_table_stays_with_that_request(cached):
    """Lengths are range checked on the host; without that check a request that claims more tokens than its table has
    becomes NaN, is not stored, and changes nothing for the others."""
    op, q, k, v, pages, table = chunk_problem(3, 15)
    cu = i32([0, 5, 9, 15])
    before = pages.clone()
    want = op(q, k, v, pages.clone(), cu, i32([10, 20, 20]), table, 6)
    got = op(q, k, v, pages, cu, i32([10, cached, 20]), table, 6)
    assert torch.equal(got[:5], want[:5]) and torch.equal(got[9:], want[9:])
    assert got[5:9].isnan().all()
    mine = table[1].long()
    assert torch.equal(pages[mine], before[mine])


def test_prefill_of_a_chunk_that_the_table_has_no_room_for():
    """The attention of such a request is as well defined as any other; its chunk is not stored."""
    op, q, k, v, pages, table = chunk_problem(3, 15, W=3)
    narrow = ops.GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp(3, 8, 2, 2, 16, 128)
    narrow.validate_inputs = False
    cu, old = i32([0, 5, 9, 15]), i32([10, 30, 20])
    before = pages.clone()
    want = op(q, k, v, pages.clone(), cu, old, table, 6)
    assert torch.equal(narrow(q, k, v, pages, cu, old, table[:, :2].contiguous(), 6), want)
    mine = table[1].long()
    assert torch.equal(pages[mine], before[mine])


def test_a_wait_that_runs_out_ends_the_launch_and_is_reported():
    """A limit far below a copy's latency: the launch gives up, says so, and the next call is as good as ever."""
    q, pages, lens, table = make([60000, 3000, 500], 32, 8, 128, 16, seed=21)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    assert F.decode_status() == 0
    for _ in range(3):
        F.gqa_decode_int4(q, pages, lens, table, page_size=16, config={"wait_log2": 1})
        torch.cuda.synchronize()
        assert F.decode_status() in (601, 602, 603)
        assert F.decode_status() == 0
        assert torch.equal(F.gqa_decode_int4(q, pages, lens, table, page_size=16), want)
    assert F.decode_status() == 0


def test_a_wait_that_runs_out_in_a_graph_is_reported():
    """The counters of a captured call are the graph's own and are cleared on every replay; what went wrong is kept."""
    q, pages, lens, table = make([60000, 3000, 500], 32, 8, 128, 16, seed=22)
    want = F.gqa_decode_int4(q, pages, lens, table, page_size=16)
    graphs = []
    for config in ({"wait_log2": 1}, None):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = F.gqa_decode_int4(q, pages, lens, table, page_size=16, config=config)
        graphs.append((graph, out))
    assert F.decode_status() == 0
    (short, _), (good, out) = graphs
    for _ in range(2):
        short.replay()
        good.replay()                    # a good launch behind it does not hide it
        torch.cuda.synchronize()
        assert F.decode_status() in (601, 602, 603)
        assert F.decode_status() == 0
        assert torch.equal(out, want)
    good.replay()
    assert F.decode_status() == 0


def test_a_request_alone_agrees_with_itself_in_a_batch():
    """The partition depends on the whole batch, so the sums' order may differ: each side is within its tolerance of 64 bits,
    and the two within twice that of one another."""
    lens, H, Hkv, D, page = [1500, 4000, 0, 700, 2222] * 6, 32, 8, 128, 16
    q, pages, t_lens, table = make(lens, H, Hkv, D, page, seed=4)
    whole = F.gqa_decode_int4(q, pages, t_lens, table, page_size=page, out_dtype=torch.float32)
    for b in (0, 1, 2, 8):
        one = F.gqa_decode_int4(q[b:b + 1], pages, t_lens[b:b + 1], table[b:b + 1], page_size=page, out_dtype=torch.float32)
        to, _ = tolerances(q[b:b + 1].cpu(), pages.cpu(), lens[b:b + 1], table[b:b + 1].cpu(), page, D ** -0.5, 0.0)
        assert ((one - whole[b:b + 1]).abs().double().cpu() <= 2 * to).all()


@pytest.mark.parametrize("cache", ["16bit", "int4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_captured_step_of_plan_append_and_attend_replays_a_decode_loop(cache, dtype):
    """The chain over either cache: one graph of the plan (in place), the norm with the append and the attention, replayed with
    new rows, equals the eager calls bit for bit, and attention in 64 bits over what the cache then holds."""
    B, H, Hkv, D, page, W, pool = 4, 8, 2, 128, 64, 5, 24
    g = torch.Generator().manual_seed(3)
    start = [130, 0, 63, 64]
    plan = ops.PagedKVCachePlanFwdOp(B, W, page)
    if cache == "int4":
        append = ops.QKNormRopeInt4KVCacheAppendFwdOp(H, Hkv, D, page)
        attend = ops.GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp(B, H, Hkv, pool * page, D, page)
        empty = (torch.full((pool, Hkv, F.int4_page_bytes(page, D)), 255, dtype=torch.uint8, device=DEV),)
    else:
        append = ops.QKNormRopeKVCacheAppendFwdOp(H, Hkv, D)
        attend = ops.GroupedQueryAttentionDecodePagedWithKVCacheFwdOp(B, H, Hkv, pool * page, D, page)
        empty = tuple(torch.full((pool * page, Hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    w = (1 + 0.2 * torch.randn(2, D, generator=g)).to(dtype).to(DEV)

    def rows(T):
        return torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(DEV)

    def step(x, s, new):
        p = plan(s["seq"], new, s["table"], s["free"], s["count"], x.shape[0], inplace=True)
        q = append(x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], w[0], w[1], p.positions, p.slot_mapping, *s["cache"])
        return q, p

    def decode(x, s):
        q, p = step(x, s, ones)
        return q, attend(q, *s["cache"], p.seq_lens, s["table"])

    ones = i32([1] * B)
    order, first = torch.randperm(pool, generator=g).to(torch.int32).to(DEV), rows(sum(start))
    states = []
    for _ in range(2):
        s = dict(seq=i32([0] * B), table=i32([[-1] * W] * B), free=order.clone(), count=i32([pool]),
                 cache=tuple(x.clone() for x in empty))
        step(first, s, i32(start))
        states.append(s)
    eager, captured = states
    x = rows(B)
    warm = dict(captured, **{k: captured[k].clone() for k in ("seq", "table", "free", "count")}, cache=tuple(c.clone() for c in captured["cache"]))
    decode(x, warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got_q, got_o = decode(x, captured)
    for n in range(70):
        x.copy_(rows(B))
        graph.replay()
        q, o = decode(x, eager)
        assert torch.equal(got_q, q) and torch.equal(got_o, o), n
    assert all(torch.equal(a, b) for a, b in zip((eager["seq"], eager["table"], eager["count"]), (captured["seq"], captured["table"], captured["count"])))
    lens = [n + 70 for n in start]
    assert eager["seq"].tolist() == lens
    table = eager["table"].cpu().long()
    if cache == "int4":
        ref, _ = O.decode_ref(q.cpu(), eager["cache"][0].cpu(), lens, table, page)
    else:
        k, v = (c.double().cpu() for c in eager["cache"])
        ref = torch.zeros(B, H, D, dtype=torch.float64)
        for b, n in enumerate(lens):
            t = torch.arange(n)
            at = table[b][t // page] * page + t % page
            for h in range(H):
                p = torch.softmax(k[at, h // (H // Hkv)] @ q[b, h].double().cpu() * D ** -0.5, 0)
                ref[b, h] = p @ v[at, h // (H // Hkv)]
    torch.testing.assert_close(o.double().cpu(), ref, atol=2e-2, rtol=1e-2)      # the decode tests' own


def test_pools_whose_offsets_pass_32_bits():
    page, Hkv, D, H = 64, 8, 128, 16
    g = torch.Generator().manual_seed(8)
    pool = (1 << 32) // (Hkv * F.int4_page_bytes(page, D)) + 40          # bytes of the 4-bit pool
    pages = torch.empty(pool, Hkv, F.int4_page_bytes(page, D), dtype=torch.uint8, device=DEV)
    lens = [130, 64]
    table = i32([[pool - 1, 0, pool - 7], [pool - 2, 3, 5]])
    T = sum(lens)
    plan = ops.PagedKVCachePlanFwdOp(2, 3, page)(i32([0, 0]), i32(lens), table, None, None, T)
    k, v = (torch.randn(T, Hkv, D, generator=g).bfloat16().to(DEV) for _ in range(2))
    F.int4_cache_append(k, v, plan.slot_mapping, pages, page_size=page)
    few = torch.zeros(8, *pages.shape[1:], dtype=torch.uint8, device=DEV)     # the same in a small pool
    small = i32([[7, 0, 1], [6, 3, 5]])
    slots = ops.PagedKVCachePlanFwdOp(2, 3, page)(i32([0, 0]), i32(lens), small, None, None, T).slot_mapping
    F.int4_cache_append(k, v, slots, few, page_size=page)
    q = torch.randn(2, H, D, generator=g).bfloat16().to(DEV)
    assert torch.equal(F.gqa_decode_int4(q, pages, i32(lens), table, page_size=page), F.gqa_decode_int4(q, few, i32(lens), small, page_size=page))
    both = [F.int4_cache_gather(p, t, i32([0, 130, 194]), T, dim=D, page_size=page, dtype=torch.bfloat16) for p, t in ((pages, table), (few, small))]
    assert all(torch.equal(a, b) for a, b in zip(*both))
    del pages
    rows = (1 << 31) // (Hkv * D) + 4 * page                              # elements of a 16-bit pool
    kp, vp = (torch.empty(rows, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    slots = torch.randperm(page, generator=g).to(torch.int32).to(DEV) + (rows - page)
    x = torch.randn(page, H + 2 * Hkv, D, generator=g).bfloat16().to(DEV)
    op = ops.QKNormRopeKVCacheAppendFwdOp(H, Hkv, D)
    pos = torch.arange(page, dtype=torch.int32, device=DEV)
    _, k1 = op(x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], None, None, pos, slots, kp, vp, return_k=True)
    assert torch.equal(kp[slots.long()], k1) and torch.equal(vp[slots.long()], x[:, H + Hkv:])


def test_prefill_refuses_a_table_of_more_tokens_than_a_request_may_hold():
    op, q, k, v, pages, _ = chunk_problem(1, 4)
    wide = torch.empty(1, 1 << 27, dtype=torch.int32, device=DEV)
    for width in (1 << 27, (1 << 26) + 1):
        big = ops.GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp(1, 8, 2, width, 16, 128)
        big.validate_inputs = False
        with pytest.raises(ValueError, match="2\\^30 tokens"):
            big(q, k, v, pages, i32([0, 4]), i32([3]), wide[:, :width], 4)
