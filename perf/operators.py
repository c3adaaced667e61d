"""Cases of the operators around a paged KV cache held in 4 bits, and the operators' plain forms.

A decode step of a serving program calls them in this order: the plan (block tables and slot maps built on the GPU from
the requests' lengths), the norm and rotation of q and k with the append to the cache, and the attention over the cache.

Layout of the 4-bit cache: ``kv_pages`` uint8 ``[pages, heads_kv, page_size * (dim + 8)]``.  The bytes of one (page, head)
are records of 16 tokens: K codes ``[16, dim / 2]``, V codes ``[16, dim / 2]``, float16 parameters ``[16, 4]`` = K scale,
K offset, V scale, V offset.  Dim 2j is the low half of byte j, dim 2j + 1 the high half; value = scale * code + offset.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6
_ROPE_BASE = 10000.0


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the plan of a decode step: 64 running requests, one new token each
        dict(name="plan_decode_64", op="plan", requests=64, cached=8192, new=1, page=64, room=1.0),
        # the plan of a step that mixes chunked prefills into a large batch (about 49 thousand new tokens), with a pool
        # that is short of pages for the last requests
        dict(name="plan_mixed_512", op="plan", requests=512, cached=4096, new=128, page=16, room=0.9),
        # norm + rotation + append of a decode step with a handful of requests: latency
        dict(name="qk_append_7", op="qk16", tokens=7, heads=32, heads_kv=8, dim=128, rotary=128, dtype="bf16", page=64),
        # a prefill step of 8192 packed tokens, 32 / 8 heads
        dict(name="qk_append_8192", op="qk16", tokens=8192, heads=32, heads_kv=8, dim=128, rotary=128, dtype="bf16", page=64),
        # head dim 80 of which 32 dims rotate, fp16, an odd token count
        dict(name="qk_append_odd", op="qk16", tokens=1021, heads=20, heads_kv=5, dim=80, rotary=32, dtype="fp16", page=16),
        # the same pass with a 4-bit cache behind it, read back for a chunked prefill
        dict(name="qk_int4_2047", op="qk4", tokens=2047, heads=16, heads_kv=4, dim=64, rotary=64, dtype="bf16", page=16),
        # append and read back: short prompts
        dict(name="int4_cache_small", op="cache4", requests=5, cached=90, new=33, heads_kv=8, dim=128, dtype="bf16", page=16),
        # append and read back: 16 chunks of 1024 tokens behind 4096 cached ones
        dict(name="int4_cache_chunks", op="cache4", requests=16, cached=4096, new=1024, heads_kv=8, dim=128, dtype="bf16", page=64),
        # one request with a thousand tokens: latency
        dict(name="decode_1x1000", op="decode4", requests=1, shortest=1000, longest=1000, heads=32, heads_kv=8, dim=128, page=16, softcap=0.0, dtype="bf16"),
        # a ragged batch of 64 requests, 512 to 8192 tokens: the ordinary decode step
        dict(name="decode_ragged_64", op="decode4", requests=64, shortest=512, longest=8192, heads=32, heads_kv=8, dim=128, page=64, softcap=0.0, dtype="bf16"),
        # head dim 64, 16 q heads to a KV head, a softcap, pages of 32, requests that have no token yet
        dict(name="decode_d64_group16", op="decode4", requests=33, shortest=0, longest=5000, heads=64, heads_kv=4, dim=64, page=32, softcap=30.0, dtype="fp16"),
        # long contexts: 8 requests of 131072 tokens
        dict(name="decode_8x131072", op="decode4", requests=8, shortest=131072, longest=131072, heads=32, heads_kv=8, dim=128, page=128, softcap=0.0, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "qk16", "qk16", "qk4", "cache4", "decode4", "decode4", "decode4"])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "plan":
        return dict(op=op, requests=_log_int(rng, 1, 2048), cached=_log_int(rng, 16, 16384), new=_log_int(rng, 1, 64), page=page,
                    room=rng.choice([1.0, 1.0, 0.5]))
    heads_kv = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
    if op in ("qk16", "qk4"):
        dim = rng.choice([64, 80, 96, 128, 256]) if op == "qk16" else rng.choice([64, 128])
        rotary = rng.choice([dim, dim, 32])
        return dict(op=op, tokens=_log_int(rng, 1, 4096), heads=heads_kv * min(group, 8), heads_kv=heads_kv, dim=dim,
                    rotary=rotary, dtype=dtype, page=page)
    dim = rng.choice([64, 128])
    if op == "cache4":
        return dict(op=op, requests=_log_int(rng, 1, 16), cached=_log_int(rng, 1, 4096), new=_log_int(rng, 1, 1024),
                    heads_kv=heads_kv, dim=dim, dtype=dtype, page=page)
    longest = _log_int(rng, 1, 131072)
    most = max(1, min(256, 8 * 131072 // longest))
    return dict(op=op, requests=_log_int(rng, 1, most), shortest=rng.choice([0, longest // 8, longest]), longest=longest,
                heads=heads_kv * group, heads_kv=heads_kv, dim=dim, page=page, softcap=rng.choice([0.0, 0.0, 30.0]), dtype=dtype)


def _lengths(case):
    """The lengths of a case's requests: part of its size, the same for every seed.  (cached, new) for a plan or an
    append, the context lengths for a decode step."""
    rng = random.Random("%s %s" % (case["op"], case["requests"]))
    n = case["requests"]
    if case["op"] == "decode4":
        lens = [rng.randint(case["shortest"], case["longest"]) for _ in range(n)]
        if case["shortest"] == 0 and n > 2:
            lens[1] = 0
        lens[-1] = case["longest"]
        return lens
    cached = [rng.randint(case["cached"] // 4, case["cached"]) for _ in range(n)]
    new = [rng.randint(max(1, case["new"] // 2), case["new"]) for _ in range(n)]
    return cached, new


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(pages_of, width, g, spare=1.25):
    """A table of distinct pages for every request, in an order that the seed makes, and the pages nobody holds."""
    total = sum(pages_of)
    pool = total + 1 + int(total * (spare - 1.0))
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    held = _int32(pages_of).long()
    start = torch.cumsum(held, 0) - held
    column = torch.arange(width, device="cuda")
    table = torch.where(column < held[:, None], order[(start[:, None] + column).clamp(max=pool - 1)], 0)
    return table.to(torch.int32).contiguous(), order[total:].contiguous(), pool


def _slots(table, first, count, page):
    """Pool slots of `count[b]` tokens from position `first[b]` on, request after request, and their positions."""
    first, count = _int32(first).long(), _int32(count).long()
    request = torch.repeat_interleave(torch.arange(first.numel(), device="cuda"), count)
    position = torch.arange(request.numel(), device="cuda") - (torch.cumsum(count, 0) - count)[request] + first[request]
    slot = table.long()[request, position // page] * page + position % page
    return slot.to(torch.int32), position.to(torch.int32)


def _outliers(x, g):
    """Keys of trained models have a few head dims that are much larger than the others."""
    boost = torch.ones(x.shape[-1], device="cuda")
    boost[torch.randperm(x.shape[-1], generator=g, device="cuda")[:2]] = 4.0
    return x * boost


def prepare(case, seed):
    g = _gen(seed)
    op, page = case["op"], case["page"]
    s = dict(case)
    if op == "plan":
        cached, new = _lengths(case)
        width = -(-(case["cached"] + case["new"]) // page)
        held = sum(-(-n // page) for n in cached)
        need = sum(-(-(a + b) // page) for a, b in zip(cached, new)) - held
        s["table"], s["free"], _ = _tables([-(-n // page) for n in cached], width, g, 1.0 + (need + 8) / held)
        s["free_count"] = _int32([min(s["free"].numel(), int(need * case["room"]) + seed % 5)])
        s["seq"], s["new"], s["total"] = _int32(cached), _int32(new), sum(new)
        if own:
            from tileops_b200.ops import PagedKVCachePlanFwdOp
            s["plan"] = PagedKVCachePlanFwdOp(case["requests"], width, page)
        return s
    dtype, heads_kv, dim = _DTYPES[case["dtype"]], case["heads_kv"], case["dim"]
    if op == "decode4":
        lens = _lengths(case)
        width = max(1, -(-case["longest"] // page))
        s["table"], _, pool = _tables([-(-n // page) for n in lens], width, g)
        # a cache as an append leaves it, page by page; slots that no token was written to hold NaN parameters
        s["pages"] = torch.empty(pool, heads_kv, page * (dim + 8), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (heads_kv * page * dim))
        slot = torch.arange(step * page, device="cuda")
        for i in range(0, pool, step):
            n = min(step, pool - i)
            k = _outliers(torch.randn(n * page, heads_kv, dim, generator=g, device="cuda"), g).to(dtype)
            v = torch.randn(n * page, heads_kv, dim, generator=g, device="cuda").to(dtype)
            s["pages"][i:i + n] = 255
            _store4(s["pages"][i:i + n], k, v, slot[:n * page], page)
        live = _int32(lens)
        position = torch.arange(width * page, device="cuda")
        last = (live - 1).clamp(min=0) // page
        dead = (position >= live[:, None]) & (position // page == last[:, None]) & (live[:, None] > 0)
        request, at = dead.nonzero(as_tuple=True)
        _records(s["pages"], page, dim)[2][s["table"].long()[request, at // page], :, (at % page) // 16, at % 16] = float("nan")
        s["lens"] = live
        s["q"] = torch.randn(case["requests"], case["heads"], dim, generator=g, device="cuda").to(dtype)
        if own:
            from tileops_b200.ops import GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp
            s["attend"] = GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp(
                case["requests"], case["heads"], heads_kv, pool * page, dim, page, softcap=case["softcap"] or None)
        return s
    if op == "cache4":
        cached, new = _lengths(case)
    else:
        # packed prompts of up to 512 tokens (a prefill step), or one token each (a decode step)
        each = 512 if case["tokens"] > 256 else 1
        new = [each] * (case["tokens"] // each) + ([case["tokens"] % each] if case["tokens"] % each else [])
        cached = [0] * len(new) if op == "qk4" or each > 1 else [37 * i % 4096 for i in range(len(new))]
    total = [a + b for a, b in zip(cached, new)]
    s["table"], _, pool = _tables([-(-n // page) for n in total], -(-max(total) // page), g)
    s["slots"], s["positions"] = _slots(s["table"], cached, new, page)
    tokens = sum(new)
    s["k"] = _outliers(torch.randn(tokens, heads_kv, dim, generator=g, device="cuda"), g).to(dtype)
    s["v"] = torch.randn(tokens, heads_kv, dim, generator=g, device="cuda").to(dtype)
    if op == "qk16":
        s["k_pages"] = torch.zeros(pool * page, heads_kv, dim, dtype=dtype, device="cuda")
        s["v_pages"] = torch.zeros(pool * page, heads_kv, dim, dtype=dtype, device="cuda")
    else:
        s["pages"] = torch.zeros(pool, heads_kv, page * (dim + 8), dtype=torch.uint8, device="cuda")
        if sum(cached):
            old, _ = _slots(s["table"], [0] * len(cached), cached, page)
            k = _outliers(torch.randn(sum(cached), heads_kv, dim, generator=g, device="cuda"), g).to(dtype)
            v = torch.randn(sum(cached), heads_kv, dim, generator=g, device="cuda").to(dtype)
            _store4(s["pages"], k, v, old, page)
        s["cu"] = _int32([0] + total).cumsum(0).to(torch.int32)
        s["total"] = sum(total)
        s["total_lens"] = _int32(total)
    if op != "cache4":
        heads, rotary = case["heads"], case["rotary"]
        # q, k and v are parts of one projection's output, as a layer hands them over
        qkv = torch.empty(tokens, heads + 2 * heads_kv, dim, dtype=dtype, device="cuda")
        qkv[:, :heads] = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(dtype) * 3
        qkv[:, heads:heads + heads_kv], qkv[:, heads + heads_kv:] = s["k"], s["v"]
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + heads_kv], qkv[:, heads + heads_kv:]
        s["q_weight"] = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype)
        s["k_weight"] = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype)
    if own:
        from tileops_b200 import ops
        if op == "qk16":
            s["append"] = ops.QKNormRopeKVCacheAppendFwdOp(heads, heads_kv, dim, rotary_dim=rotary, rope_base=_ROPE_BASE, eps=_EPS)
        elif op == "qk4":
            s["append"] = ops.QKNormRopeInt4KVCacheAppendFwdOp(heads, heads_kv, dim, page, rotary_dim=rotary, rope_base=_ROPE_BASE, eps=_EPS)
        else:
            s["append"] = ops.Int4KVCacheAppendFwdOp(heads_kv, dim, page)
        if op != "qk16":
            s["gather"] = ops.Int4KVCacheGatherFwdOp(heads_kv, dim, page, dtype)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _records(pages, page, dim):
    """Views of a pool: K codes and V codes [pages, heads_kv, records, 16, dim / 2], parameters [.., 16, 4]."""
    r = pages.view(pages.shape[0], pages.shape[1], page // 16, 16 * (dim + 8))
    half = 8 * dim
    codes = lambda x: x.unflatten(-1, (16, dim // 2))  # noqa: E731
    return codes(r[..., :half]), codes(r[..., half:2 * half]), r[..., 2 * half:].view(torch.float16).unflatten(-1, (16, 4))


def _quantise(x, slot):
    """x [tokens, heads_kv, dim] -> (codes uint8 [tokens, heads_kv, dim / 2], scale, offset float16 [tokens, heads_kv]).

    15 equal steps between the row's smallest and largest value.  Even slots count up from the smallest value, odd slots
    down from the largest (their scale is negative)."""
    x = x.float().clamp(-65504.0, 65504.0)
    low, high = x.amin(-1), x.amax(-1)
    odd = (slot % 2 == 1)[:, None]
    # the quotient is rounded once more, to 16 bits: a value next to a border goes by 32 bits
    scale = ((high - low) / 15.0).to(torch.float16)
    scale = torch.where(odd, -scale, scale)
    offset = torch.where(odd, high, low).to(torch.float16)
    step = scale.float()
    inverse = torch.where(step == 0, 0.0, 1.0 / step)
    code = torch.round((x - offset.float()[..., None]) * inverse[..., None]).clamp(0, 15)
    code = torch.nan_to_num(code).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale, offset


def _store4(pages, k, v, slot, page):
    dim = k.shape[-1]
    kc, vc, params = _records(pages, page, dim)
    at = (slot.long() // page, slice(None), slot.long() % page // 16, slot.long() % 16)
    kq, ks, km = _quantise(k, slot)
    vq, vs, vm = _quantise(v, slot)
    kc[at], vc[at], params[at] = kq, vq, torch.stack([ks, km, vs, vm], -1)


def _values(codes, params):
    """codes [.., dim / 2] and (scale, offset) [.., 2] -> values [.., dim] in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return code.float().mul_(params[..., :1].float()).add_(params[..., 1:].float())


def _gather4(s):
    page, dim = s["page"], s["dim"]
    slot, _ = _slots_of(s["table"], s["total_lens"], s["total"], page)
    kc, vc, params = _records(s["pages"], page, dim)
    at = (slot // page, slice(None), slot % page // 16, slot % 16)
    dtype = s["k"].dtype
    return _values(kc[at], params[at][..., :2]).to(dtype), _values(vc[at], params[at][..., 2:]).to(dtype)


def _slots_of(table, lens, total, page):
    lens = lens.long()
    end = torch.cumsum(lens, 0)
    row = torch.arange(total, device="cuda")
    request = torch.searchsorted(end, row, right=True)
    position = row - (end - lens)[request]
    return table.long()[request, position // page] * page + position % page, position


def _norm_rope(x, weight, positions, rotary):
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()
    half = rotary // 2
    freq = torch.pow(_ROPE_BASE, -torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = positions.double()[:, None, None] * freq
    c, n = angle.cos().float(), angle.sin().float()
    a, b = y[..., :half], y[..., half:rotary]
    return torch.cat([a * c - b * n, b * c + a * n, y[..., rotary:]], -1)


def _plan(s):
    page, table, seq, new, total = s["page"], s["table"], s["seq"].long(), s["new"].long(), s["total"]
    width = table.shape[1]
    held = (seq + page - 1) // page
    need = (seq + new + page - 1) // page - held
    refused = (seq < 0) | (new < 0) | (seq + new > width * page)
    need = torch.where(refused, 0, need)
    taken = torch.cumsum(need, 0)
    free = s["free_count"].long()
    granted = ~refused & ((need == 0) | (taken <= free))
    column = torch.arange(width, device="cuda")
    nth = column - held[:, None]
    fresh = (nth >= 0) & (nth < need[:, None]) & granted[:, None]
    popped = s["free"][(free - 1 - (taken - need)[:, None] - nth).clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where(fresh, popped, table))
    count = new.clamp(min=0)
    end = torch.cumsum(count, 0)
    row = torch.arange(total, device="cuda")
    request = torch.searchsorted(end, row, right=True)
    inside = request < seq.numel()
    request = request.clamp(max=seq.numel() - 1)
    position = torch.where(inside, seq[request] + row - (end - count)[request], 0)
    slot = table.long()[request, (position // page).clamp(0, width - 1)] * page + position % page
    slot = torch.where(inside & granted[request], slot, -1)
    left = free - torch.where(granted, need, 0).sum()
    cu = torch.cat([torch.zeros_like(end[:1]), end])
    return [x.to(torch.int32) for x in (cu, slot, position, torch.where(granted, seq + new, seq), left, granted)]


def _decode(s):
    """Scores, probabilities and sums of every request over the whole width of the table, masked by length."""
    q, table, page, dim, heads_kv = s["q"], s["table"], s["page"], s["dim"], s["heads_kv"]
    n, heads = q.shape[:2]
    kc, vc, params = (x[table.long()].transpose(1, 2).flatten(2, 4) for x in _records(s["pages"], page, dim))
    live = (torch.arange(kc.shape[2], device="cuda") < s["lens"][:, None])[:, None, None]
    score = q.float().view(n, heads_kv, -1, dim) @ _values(kc, params[..., :2]).transpose(2, 3) * dim ** -0.5
    if s["softcap"]:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    score = torch.where(live, score, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    v = torch.where(live.transpose(2, 3), _values(vc, params[..., 2:]), 0.0)
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    return out.reshape(n, heads, dim).to(q.dtype)


def run(state):
    s = state
    if s["op"] == "plan":
        if own:
            out = s["plan"](s["seq"], s["new"], s["table"], s["free"], s["free_count"], s["total"])
        else:
            out = _plan(s)
        return dict(zip(("cu_seqlens", "slots", "positions", "seq_lens", "free_count", "granted"), out), table=s["table"])
    if s["op"] == "decode4":
        return {"o": s["attend"](s["q"], s["pages"], s["lens"], s["table"]) if own else _decode(s)}
    if s["op"] == "qk16":
        if own:
            q = s["append"](s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"], s["slots"], s["k_pages"], s["v_pages"])
        else:
            dtype = s["q"].dtype
            q = _norm_rope(s["q"], s["q_weight"], s["positions"], s["rotary"]).to(dtype)
            s["k_pages"][s["slots"].long()] = _norm_rope(s["k"], s["k_weight"], s["positions"], s["rotary"]).to(dtype)
            s["v_pages"][s["slots"].long()] = s["v"]
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    # a 4-bit cache: the append, and the cached rows read back as the values they stand for
    if s["op"] == "qk4":
        if own:
            q = s["append"](s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"], s["slots"], s["pages"])
        else:
            dtype = s["q"].dtype
            q = _norm_rope(s["q"], s["q_weight"], s["positions"], s["rotary"]).to(dtype)
            k = _norm_rope(s["k"], s["k_weight"], s["positions"], s["rotary"]).to(dtype)
            _store4(s["pages"], k, s["v"], s["slots"], s["page"])
    elif own:
        s["append"](s["k"], s["v"], s["slots"], s["pages"])
    else:
        _store4(s["pages"], s["k"], s["v"], s["slots"], s["page"])
    k, v = s["gather"](s["pages"], s["table"], s["cu"], s["total"]) if own else _gather4(s)
    return {"q": q, "k": k, "v": v} if s["op"] == "qk4" else {"k": k, "v": v}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    op, page = case["op"], case["page"]
    if op == "plan":
        cached, new = _lengths(case)
        fresh = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(cached, new))
        # lengths in, pages taken off the stack and entered in the table, lengths, grants and slot map out
        return {"bytes": 4 * (5 * case["requests"] + 1 + 2 * fresh + 2 * sum(new)), "flops": 0}
    heads_kv, dim = case["heads_kv"], case["dim"]
    if op == "decode4":
        lens = _lengths(case)
        pages = sum(-(-n // page) for n in lens)
        return {"bytes": sum(lens) * heads_kv * (dim + 8) + 4 * case["requests"] * case["heads"] * dim + 4 * (pages + len(lens)),
                "flops": 4 * case["heads"] * dim * sum(lens)}
    if op == "cache4":
        cached, new = _lengths(case)
        total = sum(cached) + sum(new)
        row = heads_kv * dim * 4                      # K and V of a token in 16 bits
        four = heads_kv * (dim + 8)
        return {"bytes": sum(new) * (row + four) + total * (row + four), "flops": 8 * heads_kv * dim * total}
    tokens, heads = case["tokens"], case["heads"]
    bytes_in = 2 * tokens * (heads + 2 * heads_kv) * dim + 8 * tokens + 4 * dim
    flops = tokens * (heads + heads_kv) * (4 * dim + 3 * case["rotary"])
    if op == "qk16":
        return {"bytes": bytes_in + 2 * tokens * (heads + 2 * heads_kv) * dim, "flops": flops}
    four = tokens * heads_kv * (dim + 8)
    return {"bytes": bytes_in + 2 * tokens * heads * dim + 2 * four + 4 * tokens * heads_kv * dim, "flops": flops}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_code_row(x, slot):
    """The 4-bit values of rows x [tokens, heads_kv, dim] (16-bit numbers): what the cache holds, in 64 bits."""
    x = x.double().clamp(-65504.0, 65504.0)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    down = (slot.long() & 1).bool().view(-1, 1, 1)
    scale = ((high - low) / 15).to(torch.float16).double()
    start = torch.where(down, high, low).to(torch.float16).double()
    away = (x - start).abs()
    steps = torch.where(scale > 0, away / scale, 0.0).round().clamp(max=15)
    # a value on the wrong side of its start (which is rounded to 16 bits) stays at the start
    steps = torch.where(torch.where(down, x > start, x < start), 0.0, steps)
    return start + torch.where(down, -scale, scale) * steps


def _exact_rotated(x, weight, positions, rotary):
    x = x.double()
    y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt() * weight.double()
    half = rotary // 2
    exponent = torch.arange(half, dtype=torch.float64, device="cuda") / half
    turn = torch.polar(torch.ones(positions.numel(), half, dtype=torch.float64, device="cuda"),
                       positions.double()[:, None] * _ROPE_BASE ** -exponent)
    z = torch.complex(y[..., :half], y[..., half:rotary]) * turn[:, None]
    y[..., :half], y[..., half:rotary] = z.real, z.imag
    return y


def _exact_cached(s, b, length):
    """K and V [length, heads_kv, dim] of request b as the cache holds them, in 64 bits."""
    page, heads_kv, dim = s["page"], s["heads_kv"], s["dim"]
    held = s["pages"][s["table"][b, :-(-length // page)].long()]                       # [pages, heads_kv, bytes]
    held = held.transpose(0, 1).reshape(heads_kv, -1, 16 * (dim + 8))                  # [heads_kv, records, bytes]
    params = held[..., 16 * dim:].contiguous().view(torch.float16).double().view(heads_kv, -1, 4)[:, :length]
    found = []
    for first, at in ((0, 0), (8 * dim, 2)):
        byte = held[..., first:first + 8 * dim].reshape(heads_kv, -1, dim // 2)[:, :length].double()
        high = (byte / 16).floor()
        value = torch.empty(heads_kv, length, dim, dtype=torch.float64, device="cuda")
        value[..., 0::2], value[..., 1::2] = byte - 16 * high, high
        found.append((value * params[..., at:at + 1] + params[..., at + 1:at + 2]).transpose(0, 1))
    return found


def _exact_attention(s):
    n, heads, dim = s["q"].shape
    group = heads // s["heads_kv"]
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lens"].tolist()):
        if length == 0:
            continue
        k, v = _exact_cached(s, b, length)
        for h in range(s["heads_kv"]):
            q = s["q"][b, h * group:(h + 1) * group].double()
            score = (k[:, h] @ q.T) / math.sqrt(dim)
            if s["softcap"]:
                score = (score / s["softcap"]).tanh() * s["softcap"]
            out[b, h * group:(h + 1) * group] = score.softmax(0).T @ v[:, h]
    return out


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None
    s = prepare(case, seed)
    if op == "decode4":
        return {"o": _exact_attention(s)}
    new = _exact_rotated(s["k"], s["k_weight"], s["positions"], s["rotary"]) if op != "cache4" else s["k"]
    if op == "qk16":
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        k_pages[s["slots"].long()], v_pages[s["slots"].long()] = new, s["v"].double()
        return {"q": _exact_rotated(s["q"], s["q_weight"], s["positions"], s["rotary"]), "k_pages": k_pages, "v_pages": v_pages}
    slot = s["slots"]
    k_new, v_new = _exact_code_row(new.to(s["k"].dtype), slot), _exact_code_row(s["v"], slot)
    if op == "qk4":
        return {"q": _exact_rotated(s["q"], s["q_weight"], s["positions"], s["rotary"]), "k": k_new, "v": v_new}
    k, v, row = [], [], 0
    for b, (held, count) in enumerate(zip(*_lengths(case))):   # what is cached already stands as it is, the new rows behind it
        for whole, part, fresh in zip((k, v), _exact_cached(s, b, held), (k_new, v_new)):
            whole += [part, fresh[row:row + count]]
        row += count
    return {"k": torch.cat(k), "v": torch.cat(v)}
