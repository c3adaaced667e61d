"""CPU-only tests of the operators around the paged KV cache: what their constructors and the C ABI refuse (nothing is
launched), the oracle's own properties, and the kernel_map seam."""

import ctypes

import pytest
import torch

from oracle import paged_kv_oracle as O
from tileops_b200 import _native
from tileops_b200 import functional as F
from tileops_b200 import ops
from tileops_b200.kernels import Kernel
from tileops_b200.manifest import load_manifest
from tileops_b200.perf import formulas

I4Decode = ops.GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp
I4Prefill = ops.GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp


@pytest.mark.parametrize("make,message", [
    (lambda: ops.PagedKVCachePlanFwdOp(0, 4, 16), "batch must be positive"),
    (lambda: ops.PagedKVCachePlanFwdOp(4097, 4, 16), "at most 4096 requests"),
    (lambda: ops.PagedKVCachePlanFwdOp(1, 1 << 20, 2048), "at most 2\\^30 tokens"),
    (lambda: ops.PagedKVCacheReleaseFwdOp(1, 0, 16), "max_pages_per_req must be positive"),
    (lambda: ops.QKNormRopeFwdOp(8, 2, 100), "dim must be a multiple of 8 up to 256"),
    (lambda: ops.QKNormRopeFwdOp(8, 2, 264), "dim must be a multiple of 8 up to 256"),
    (lambda: ops.QKNormRopeFwdOp(8, 2, 72), "rotary_dim must be a multiple of 16"),
    (lambda: ops.QKNormRopeFwdOp(8, 2, 128, 24), "rotary_dim must be a multiple of 16"),
    (lambda: ops.QKNormRopeFwdOp(8, 2, 64, 80), "rotary_dim must be a multiple of 16"),
    (lambda: ops.QKNormRopeFwdOp(8, 2, 64, eps=-1.0), "eps must be non-negative"),
    (lambda: ops.QKNormRopeFwdOp(8, 2, 64, inv_freq=torch.ones(31)), "inv_freq must have shape"),
    (lambda: ops.QKNormRopeInt4KVCacheAppendFwdOp(8, 2, 96, 16), "head dim 64 and 128"),
    (lambda: ops.QKNormRopeInt4KVCacheAppendFwdOp(8, 2, 64, 8), "multiple of 16"),
    (lambda: ops.Int4KVCacheAppendFwdOp(2, 256, 16), "head dim 64 and 128"),
    (lambda: ops.Int4KVCacheGatherFwdOp(2, 64, 24), "multiple of 16"),
    (lambda: ops.Int4KVCacheGatherFwdOp(2, 64, 16, torch.float32), "Expected dtype"),
    (lambda: I4Decode(1, 30, 8, 128, 64, 16), "heads must be divisible by heads_kv"),
    (lambda: I4Decode(1, 8, 2, 128, 64, 0), "page_size must be positive"),
    (lambda: I4Prefill(1, 8, 2, 4, 16, 64, softcap=-1.0), "softcap must be non-negative"),
])
def test_constructors_refuse(make, message):
    with pytest.raises(ValueError, match=message):
        make()


def test_calls_refuse_tensors_that_are_not_on_a_gpu_or_have_another_shape():
    q, pool = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16 * 72, dtype=torch.uint8)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    for call in (lambda: F.gqa_decode_int4(q, pool, lens, table, page_size=16),
                 lambda: F.paged_kv_plan(lens, lens, table, None, None, 2, page_size=16),
                 lambda: F.paged_kv_release(lens.bool(), lens, table, lens, lens[:1], page_size=16),
                 lambda: F.qk_norm_rope(q, q, lens, None),
                 lambda: F.int4_cache_append(q, q, lens, pool, page_size=16),
                 lambda: F.int4_cache_gather(pool, table, lens, 3, dim=64, page_size=16, dtype=torch.float16),
                 lambda: F.gqa_prefill_paged_int4_cache(q, q, q, pool, lens, lens, table, 1, page_size=16)):
        with pytest.raises(ValueError, match="must be on a cuda device"):
            call()
    op = I4Decode(2, 8, 2, 64, 64, 16)
    with pytest.raises(ValueError, match="q must have shape"):
        op(q[:1], pool, lens, table)
    with pytest.raises(ValueError, match="kv_pages must have shape"):
        op(q, pool[:3], lens, table)
    with pytest.raises(ValueError, match="seq_lens must have shape"):
        ops.PagedKVCachePlanFwdOp(3, 2, 16)(lens, lens, table, None, None, 2)
    with pytest.raises(ValueError, match="block_table shape must be"):
        ops.PagedKVCachePlanFwdOp(2, 3, 16)(lens, lens, table, None, None, 2)
    with pytest.raises(ValueError, match="k must have shape"):
        ops.QKNormRopeFwdOp(8, 2, 64)(q, q, None, None, lens)
    with pytest.raises(ValueError, match="k must have shape"):
        ops.Int4KVCacheAppendFwdOp(2, 64, 16)(q, q, lens, pool)


def test_checks_of_vectors_tables_and_pools():
    cpu = torch.device("cpu")
    ok = torch.zeros(4, dtype=torch.int32)
    F._check_vector("x", ok, 4, cpu)
    for bad in (ok.long(), ok[:3], ok.view(2, 2), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="x must"):
            F._check_vector("x", bad, 4, cpu)
    table = torch.zeros(4, 6, dtype=torch.int32)
    F._check_table(table[:, 1:3], 4, cpu)
    for bad in (table.long(), table[:3], table.view(-1), table[:, :0], torch.zeros(6, 4, dtype=torch.int32).T):
        with pytest.raises(ValueError, match="block_table"):
            F._check_table(bad, 4, cpu)
    pool = torch.zeros(3, 2, 32 * 72, dtype=torch.uint8)
    F._check_int4_pool(pool, 2, 64, 32, cpu)
    for args in ((pool.to(torch.int8), 2, 64, 32), (pool, 3, 64, 32), (pool, 2, 128, 32), (pool, 2, 64, 16),
                 (pool[:, :, :16 * 72], 2, 64, 16), (pool, 2, 80, 32), (pool, 2, 64, 24), (pool, 2, 64, 0)):
        with pytest.raises(ValueError):
            F._check_int4_pool(*args, cpu)
    whole = torch.zeros(32 * 72 + 16, dtype=torch.uint8)
    start = (-whole.data_ptr()) % 16
    F._check_int4_pool(whole[start:start + 32 * 72].view(1, 1, -1), 1, 64, 32, cpu)
    with pytest.raises(ValueError, match="16-byte boundary"):
        F._check_int4_pool(whole[start + 8:start + 8 + 32 * 72].view(1, 1, -1), 1, 64, 32, cpu)


def test_rows_are_copied_only_when_they_have_to_be():
    x = torch.zeros(4, 10, 64, dtype=torch.float16)
    assert F._rows(x[:, 2:5])[0].data_ptr() == x[:, 2:5].data_ptr() and F._rows(x[:, 2:5])[1:] == (640, 64)
    assert F._rows(x[:1, :1].as_strided((1, 1, 64), (3, 5, 1)))[1:] == (64, 64)      # strides of lone rows mean nothing
    assert F._rows(x.transpose(0, 1))[1:] == (64, 640)
    y, tok, head = F._rows(x[..., ::2])
    assert y.is_contiguous() and (tok, head) == (320, 32)
    z = torch.zeros(4 * 64 + 8, dtype=torch.float16)
    z = z[(-z.data_ptr() % 16) // 2 + 1:][:4 * 64].view(2, 2, 64)
    copy = F._rows(z)[0]
    assert copy.data_ptr() != z.data_ptr() and copy.data_ptr() % 16 == 0


def test_abi_refuses_without_touching_a_gpu():
    lib = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    err = lambda: lib.tb200_last_error()  # noqa: E731

    plan = lambda batch=2, width=4, page=16, cap=4, total=2, slots=p, free=p: lib.tb200_paged_kv_plan(  # noqa: E731
        p, p, p, 4, p, cap, free, p, slots, p, p, p, p, batch, width, page, total, None)
    assert plan(batch=0) == 1 and plan(page=0) == 1 and plan(total=-1) == 1
    assert plan(slots=None) == 1 and b"non-null" in err()
    assert plan(batch=4097) == 2 and plan(width=1 << 27) == 2 and plan(cap=-1) == 2
    assert lib.tb200_paged_kv_release(None, p, p, 4, p, 4, p, 2, 4, 16, None) == 1
    assert lib.tb200_paged_kv_release(p, p, p, 4, p, 4, p, 5000, 4, 16, None) == 2

    def norm(dtype=1, cache=0, tokens=1, heads=2, dim=64, rotary=64, q=p, stride=128, wd=1, page=16, pool=16, v=p):
        return lib.tb200_qk_norm_rope(q, p, v, p, p, p, p, wd, p, p, p, p, p, dtype, cache, tokens, heads, 2, dim, rotary,
                                      stride, 64, 128, 64, 128, 64, page, pool, 1e-6, None)
    assert norm(heads=0) == 1 and norm(tokens=-1) == 1 and norm(cache=3) == 1 and norm(q=None) == 1
    assert norm(cache=1, v=None) == 1 and b"cache" in err()
    assert norm(dtype=3) == 2 and norm(dim=68) == 2 and norm(dim=512) == 2 and norm(rotary=72) == 2 and norm(rotary=8) == 2
    assert norm(wd=0) == 2 and norm(cache=2, dim=96, rotary=96) == 2 and norm(cache=2, page=8) == 2 and norm(pool=1 << 31) == 2
    assert norm(q=p + 2) == 2 and norm(stride=129) == 2 and b"16-byte" in err()
    assert norm(tokens=0) == 0

    append = lambda dtype=1, tokens=1, hkv=1, dim=64, page=16, k=p, stride=64: lib.tb200_int4_cache_append(  # noqa: E731
        k, p, p, p, dtype, tokens, hkv, dim, page, 16, stride, 64, 64, 64, None)
    assert append(tokens=-1) == 1 and append(k=None) == 1 and append(hkv=0) == 1
    assert append(dtype=2) == 2 and append(dim=96) == 2 and append(page=24) == 2 and append(stride=4) == 2 and append(k=p + 8) == 2
    assert append(tokens=0) == 0

    gather = lambda dtype=1, total=1, dim=64, page=16, pages=p, cached=None, width=1: lib.tb200_int4_cache_gather(  # noqa: E731
        pages, p, 1, width, p, cached, None, None, None, p, p, dtype, total, 1, 1, dim, page, 1, None)
    assert gather(total=-1) == 1 and gather(pages=None) == 1 and gather(cached=p) == 1 and gather(width=0) == 1
    assert gather(dtype=3) == 2 and gather(dim=256) == 2 and gather(page=8) == 2 and gather(pages=p + 4) == 2
    assert gather(total=0) == 0

    def decode(q=p, heads=8, hkv=2, dim=64, page=16, qd=1, od=1, pool=1, ws=p, nbytes=1 << 30, width=1, batch=1):
        return lib.tb200_gqa_decode_int4(q, p, p, None, p, p, 1, width, qd, od, batch, heads, hkv, dim, page, pool, 1.0, 0.0, 0,
                                         ws, nbytes, None)
    assert decode(q=None) == 1 and decode(heads=7) == 1 and decode(width=0) == 1 and decode(batch=0) == 1 and decode(ws=None) == 1
    assert decode(dim=96) == 2 and decode(page=8) == 2 and decode(qd=3) == 2 and decode(od=2) == 2 and decode(pool=0) == 2
    size = lib.tb200_gqa_decode_int4_workspace_bytes
    assert size(0, 8, 2, 64) == 0 and size(1, 7, 2, 64) == 0 and size(1, 8, 2, 96) == 0 and size(4, 32, 8, 128) > 0


def test_row_counts_that_32_bits_do_not_hold_are_refused():
    lib = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    many = (1 << 30) + 1
    assert lib.tb200_paged_kv_plan(p, p, p, 4, p, 4, p, p, p, p, p, p, p, 2, 4, 16, many, None) == 2
    assert b"2^30" in lib.tb200_last_error()
    assert lib.tb200_qk_norm_rope(p, p, p, p, p, p, p, 1, p, p, p, p, p, 1, 0, many, 2, 2, 64, 64, 128, 64, 128, 64, 128, 64, 16,
                                  16, 1e-6, None) == 2
    assert lib.tb200_int4_cache_append(p, p, p, p, 1, many, 1, 64, 16, 16, 64, 64, 64, 64, None) == 2
    assert lib.tb200_int4_cache_gather(p, p, 1, 1, p, None, None, None, None, p, p, 1, many, 1, 1, 64, 16, 1, None) == 2


class _Recorder(Kernel):
    supported_archs = None
    general = True

    def __init__(self, *args, **kwargs):
        self.args, self.kwargs, self.config = args, kwargs, {}

    def forward(self, q, *rest, **kw):
        return q


def test_kernel_map_replaces_the_kernels():
    q, pool = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16 * 72, dtype=torch.uint8)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    op = I4Decode(2, 8, 2, 64, 64, 16, softcap=3.0, kernel_map={"gqa_decode_paged_int4_kernel": _Recorder})
    assert op(q, pool, lens, table) is q and op(q, pool, lens, table) is q
    (kern,) = op.built_kernels("gqa_decode_paged_int4_kernel").values()
    assert kern.args == (2, 8, 2, 64, 64, 16, torch.bfloat16) and kern.kwargs["softcap"] == 3.0
    assert op.eval_roofline() == formulas.gqa_decode_paged_int4_roofline(
        batch=2, heads=8, heads_kv=2, seqlen_kv=64, dim=64, page_size=16, dtype=torch.bfloat16)
    plan = ops.PagedKVCachePlanFwdOp(2, 2, 16, kernel_map={"paged_kv_plan_kernel": _Recorder})
    assert plan(lens, lens, table, None, None, 2) is lens
    norm = ops.QKNormRopeFwdOp(8, 8, 64, kernel_map={"qk_norm_rope_kernel": _Recorder})
    assert norm(q, q, None, None, lens) is q


def test_decode_can_range_check_its_block_table():
    q, pool = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16 * 72, dtype=torch.uint8)
    op = I4Decode(2, 8, 2, 64, 64, 16, kernel_map={"gqa_decode_paged_int4_kernel": _Recorder})
    op.validate_inputs = True
    lens = torch.tensor([17, 1], dtype=torch.int32)
    assert op(q, pool, lens, torch.tensor([[3, 0], [2, 9]], dtype=torch.int32)) is q
    with pytest.raises(ValueError, match="outside the pool of 4 pages"):
        op(q, pool, lens, torch.tensor([[3, 4], [2, 9]], dtype=torch.int32))
    with pytest.raises(ValueError, match="needs 3 pages"):
        op(q, pool, lens + 16, torch.tensor([[3, 1], [2, 0]], dtype=torch.int32))


# ---- the oracle ----------------------------------------------------------------------------------------------------------
def test_oracle_quantiser_keeps_ends_and_errors_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 128, generator=g).bfloat16()
    for odd in (False, True):
        code, scale, offset = O.quantise_ref(x, torch.full((64,), odd))
        value = scale.double()[:, None] * code.double() + offset.double()[:, None]
        step = ((x.double().amax(-1) - x.double().amin(-1)) / 15)[:, None]
        assert ((value - x.double()).abs() <= step / 2 + 15 * step * 2 ** -11).all()
        assert (code.min(-1).values == 0).all() and (code.max(-1).values == 15).all()
        assert ((scale < 0) == odd).all()


def test_oracle_cache_round_trip_and_views():
    g = torch.Generator().manual_seed(1)
    pages = torch.zeros(3, 2, F.int4_page_bytes(32, 64), dtype=torch.uint8)
    k, v = (torch.randn(5, 2, 64, generator=g).half() for _ in range(2))
    slots = torch.tensor([70, 3, -1, 95, 16], dtype=torch.int32)
    O.store_ref(pages, k, v, slots, 32)
    kc, vc, params = F.int4_cache_views(pages, 32, 64)
    for t, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        for x, codes, at in ((k, kc, 0), (v, vc, 2)):
            code, scale, offset = O.quantise_ref(x[t], torch.full((2,), s % 2 == 1))
            got = codes[s // 32, :, s % 32 // 16, s % 16]
            assert torch.equal(torch.stack([got & 15, got >> 4], -1).flatten(-2), code)
            par = params[s // 32, :, s % 32 // 16, s % 16]
            assert torch.equal(par[:, at], scale) and torch.equal(par[:, at + 1], offset)
    rows, _, _ = O.rows_ref(pages, torch.tensor([2, 0, 1]), 40, 32, 64)
    code, scale, offset = O.quantise_ref(k[0], torch.zeros(2, dtype=torch.bool))
    assert torch.equal(rows[6], scale.double()[:, None] * code.double() + offset.double()[:, None])


def test_oracle_plan_by_hand():
    got = O.plan_ref([15, 32], [2, 1], [[4, 0], [5, 6]], [7, 8, 9], 3, 4, 16)
    assert got == ([[4, 9], [5, 6]], [0, 2, 3], [4 * 16 + 15, 9 * 16, -1, -1], [15, 16, 32, 0], [17, 32], 2, [1, 0])


def test_decode_flags_of_the_wait_limit():
    assert _native.decode_flags({"wait_log2": 5, "chunk_tiles": 3}) == (5 << 24) | (3 << 8)
    for bad in (-1, 32):
        with pytest.raises(ValueError, match="wait_log2"):
            _native.decode_flags({"wait_log2": bad})


def test_status_of_the_4_bit_decode_wants_a_place_for_the_code():
    assert _native.lib().tb200_gqa_decode_int4_status(None, 0, None) == 1
    assert F.decode_status("cpu") == 0


# ---- manifest ------------------------------------------------------------------------------------------------------------
FAMILY = ["PagedKVCachePlanFwdOp", "PagedKVCacheReleaseFwdOp", "QKNormRopeFwdOp", "QKNormRopeKVCacheAppendFwdOp",
          "QKNormRopeInt4KVCacheAppendFwdOp", "Int4KVCacheAppendFwdOp", "Int4KVCacheGatherFwdOp",
          "GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp", "GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp"]


def make_op(name, kernel=None):
    args = {"PagedKVCachePlanFwdOp": (2, 2, 16), "PagedKVCacheReleaseFwdOp": (2, 2, 16), "QKNormRopeFwdOp": (8, 2, 64, 32),
            "QKNormRopeKVCacheAppendFwdOp": (8, 2, 64), "QKNormRopeInt4KVCacheAppendFwdOp": (8, 2, 64, 16),
            "Int4KVCacheAppendFwdOp": (2, 64, 16), "Int4KVCacheGatherFwdOp": (2, 64, 16, torch.float16),
            "GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp": (2, 8, 2, 64, 64, 16),
            "GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp": (2, 8, 2, 2, 16, 64)}[name]
    cls = getattr(ops, name)
    slot = load_manifest()[name]["source"]["kernel_map"]
    return cls(*args, kernel_map={key: kernel for key in slot} if kernel else None)


@pytest.mark.parametrize("name", FAMILY)
def test_every_operator_of_the_step_has_a_manifest_entry(name):
    entry = load_manifest()[name]
    assert name in ops.__all__ and entry["roofline"]["func"].split(".")[-1] in formulas.__all__
    assert entry["source"]["kernel_map"] == {k: c.__name__ for k, c in make_op(name).kernel_map.items()}
    for label in entry["workloads"]:
        work = {k: v for k, v in label.items() if k not in ("label", "dtypes")}
        flops, nbytes = getattr(formulas, entry["roofline"]["func"].split(".")[-1])(
            **(dict(batch=128, heads=64, heads_kv=8, seqlen_kv=524288, dim=128) if "q_shape" in work else {}), **work)
        assert flops >= 0 and nbytes > 0
    params = make_op(name)._manifest_params()
    assert list(params) == list(entry["signature"]["params"])


def test_manifest_params_reach_a_builder():
    assert make_op("GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp")._manifest_params() == {
        "max_pages_per_req": 2, "page_size": 16, "is_causal": True, "sm_scale": 64 ** -0.5, "softcap": 0.0}
    assert make_op("QKNormRopeInt4KVCacheAppendFwdOp")._manifest_params() == {
        "page_size": 16, "rotary_dim": 64, "rope_base": 10000.0, "eps": 1e-6, "inv_freq": None}
    assert make_op("Int4KVCacheGatherFwdOp")._manifest_params() == {"dim": 64, "page_size": 16, "dtype": torch.float16}


def test_rooflines_of_the_step():
    q, k = torch.zeros(5, 8, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    slots, pool = torch.zeros(5, dtype=torch.int32), torch.zeros(4, 2, 16 * 72, dtype=torch.uint8)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    op = make_op("QKNormRopeFwdOp", _Recorder)
    with pytest.raises(RuntimeError, match="after a forward"):
        op.eval_roofline()
    op(q, k, None, None, slots)
    assert op.eval_roofline() == (50 * (4 * 64 + 3 * 32), 2 * 50 * 64 * 2 + 5 * 4 + 2 * 64 * 2)
    op = make_op("QKNormRopeKVCacheAppendFwdOp", _Recorder)
    op(q, k, k, None, None, slots, slots, k, k)
    want = (50 * 7 * 64, 2 * 50 * 64 * 2 + 5 * 4 + 256 + 2 * 10 * 64 * 2 + 5 * 4)
    assert op.eval_roofline() == want
    op = make_op("QKNormRopeInt4KVCacheAppendFwdOp", _Recorder)
    op(q, k, k, None, None, slots, slots, pool)
    assert op.eval_roofline() == (want[0], want[1] - 2 * 10 * 64 * 2 + 10 * 72)
    op = make_op("Int4KVCacheAppendFwdOp", _Recorder)
    op(k, k, slots, pool)
    assert op.eval_roofline() == (8 * 10 * 64, 10 * (256 + 72) + 20)
    op = make_op("Int4KVCacheGatherFwdOp", _Recorder)
    op(pool, table, torch.zeros(3, dtype=torch.int32), 20)
    assert op.eval_roofline() == (4 * 40 * 64, 40 * (256 + 72) + 8)
    op = make_op("PagedKVCachePlanFwdOp", _Recorder)
    op(lens, lens, table, None, None, 20)
    assert op.eval_roofline() == (0, 4 * (10 + 1 + 4 + 40))
    assert make_op("PagedKVCacheReleaseFwdOp").eval_roofline() == (0, 2 * (9 + 16))
    work = dict(total_q=24, batch=2, q_lens=[20, 4], cache_lens=[7, 30], heads=8, heads_kv=2, dim=64, page_size=16,
                max_pages_per_req=3, max_seqlen_q=20, is_causal=True, dtype=torch.bfloat16)
    flops, nbytes = formulas.gqa_prefill_paged_with_kv_cache_fwd_roofline(**work)
    # of the 16-bit form's K and V, those read from the cache (37 tokens) and those appended (24) have 72 bytes a head
    assert formulas.gqa_prefill_paged_int4_roofline(**work) == (flops, nbytes - (37 + 24) * 2 * (256 - 72))


def test_tables_that_pages_are_entered_in_have_rows_of_their_own():
    F._check_rows_apart(torch.zeros(3, 4, dtype=torch.int32))
    F._check_rows_apart(torch.zeros(3, 9, dtype=torch.int32)[:, 2:6])
    F._check_rows_apart(torch.zeros(1, 4, dtype=torch.int32).expand(1, 4))
    for bad in (torch.zeros(1, 4, dtype=torch.int32).expand(3, 4), torch.zeros(12, dtype=torch.int32).as_strided((3, 4), (2, 1))):
        with pytest.raises(ValueError, match="must not overlap"):
            F._check_rows_apart(bad)


def test_the_first_call_of_a_rotation_is_refused_under_capture(monkeypatch):
    monkeypatch.setattr(F, "_capturing", lambda device: True)
    op = ops.QKNormRopeFwdOp(8, 2, 64)
    with pytest.raises(RuntimeError, match="call it once before the capture"):
        op._turns(torch.device("cuda", 0))
    assert ops.QKNormRopeFwdOp(8, 2, 64, 0)._turns(torch.device("cuda", 0)) is None
