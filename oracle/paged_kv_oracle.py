"""CPU restatement of the operators around a paged KV cache, for the tests: plans with Python integers, norm and rotation
and attention in 64 bits, the 4-bit quantiser step by step in the 32-bit arithmetic it is defined in."""

from __future__ import annotations

import math

import torch


def plan_ref(seq_lens, new_lens, table, free_pages, free_count, total_tokens, page):
    """Plain lists in, plain lists out: (table, cu, slots, positions, seq_after, free_after, granted)."""
    table = [list(row) for row in table]
    width = len(table[0])
    allocates = free_pages is not None
    count = min(max(free_count, 0), len(free_pages)) if allocates else 0
    cu, slots, positions, after, granted = [0], [], [], [], []
    wanted, taken = 0, 0
    for b, (s, n) in enumerate(zip(seq_lens, new_lens)):
        fits = s >= 0 and n >= 0 and s + n <= width * page
        held = -(-s // page)
        need = -(-(s + n) // page) - held if fits and allocates else 0
        wanted += need
        ok = fits and (need == 0 or wanted <= count)
        if ok:
            for j in range(need):
                table[b][held + j] = free_pages[count - 1 - taken]
                taken += 1
        granted.append(int(ok))
        after.append(s + n if ok else s)
        cu.append(cu[-1] + max(n, 0))
        for i in range(max(n, 0)):
            pos = s + i
            positions.append(pos)
            slots.append(table[b][pos // page] * page + pos % page if ok else -1)
    slots = (slots + [-1] * total_tokens)[:total_tokens]
    positions = (positions + [0] * total_tokens)[:total_tokens]
    return table, cu, slots, positions, after, count - taken, granted


def norm_rope_ref(x, weight, positions, rotary_dim, eps, base=10000.0, inv_freq=None):
    """x [T,H,D] -> float64."""
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.double()
    half = rotary_dim // 2
    freq = (torch.tensor([base ** (-j / half) for j in range(half)], dtype=torch.float64) if inv_freq is None
            else inv_freq.double())
    angle = positions.double()[:, None, None] * freq
    a, b = y[..., :half], y[..., half:rotary_dim]
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), y[..., rotary_dim:]], -1)


def quantise_ref(x, odd):
    """Rows x [..., D] (16-bit), odd bool [...] -> (codes uint8 [..., D], scale, offset float16 [...])."""
    x = x.float()
    nan = x.isnan().any(-1)
    x = torch.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0)
    lo, hi = x.amin(-1), x.amax(-1)
    step = ((hi - lo) / torch.tensor(15.0)).half()
    scale = torch.where(odd, -step, step)
    offset = torch.where(odd, hi, lo).half()
    s = scale.float()
    inverse = torch.where(s == 0, torch.zeros_like(s), 1.0 / s)
    code = torch.round((x - offset.float()[..., None]) * inverse[..., None]).clamp(0, 15).to(torch.uint8)
    code[nan] = 0
    scale[nan] = float("nan")
    offset[nan] = float("nan")
    return code, scale, offset


def store_ref(pages, k, v, slots, page):
    """Append k, v [T,Hkv,D] to the pool uint8 [pages, Hkv, page*(D+8)] (CPU, in place); slots outside are skipped."""
    D = k.shape[-1]
    records = pages.view(pages.shape[0], pages.shape[1], page // 16, 16 * (D + 8))
    for t, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pages.shape[0] * page:
            continue
        rec = records[slot // page, :, slot % page // 16]
        i = slot % 16
        for part, x in ((0, k[t]), (1, v[t])):
            code, scale, offset = quantise_ref(x, torch.full((x.shape[0],), slot % 2 == 1))
            rec[:, part * 8 * D + i * (D // 2):part * 8 * D + (i + 1) * (D // 2)] = code[:, 0::2] | (code[:, 1::2] << 4)
            at = 16 * D + i * 8 + part * 4
            rec[:, at:at + 4] = torch.stack([scale, offset], -1).contiguous().view(torch.uint8)


def rows_ref(pages, table_row, length, page, dim):
    """(K, V) float64 [length, Hkv, D] of one request, and its V scales and K parameters [length, Hkv, 4]."""
    records = pages.view(pages.shape[0], pages.shape[1], page // 16, 16 * (dim + 8))
    t = torch.arange(length)
    rec = records[table_row.long()[t // page], :, t % page // 16]              # [length, Hkv, bytes]
    i = t % 16
    params = rec[..., 16 * dim:].contiguous().view(torch.float16).view(length, -1, 16, 4)[t, :, i].double()
    out = []
    for part in (0, 1):
        byte = rec[..., part * 8 * dim:(part + 1) * 8 * dim].reshape(length, -1, 16, dim // 2)[t, :, i]
        code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2).double()
        out.append(code * params[..., 2 * part:2 * part + 1] + params[..., 2 * part + 1:2 * part + 2])
    return out[0], out[1], params


def decode_ref(q, pages, lens, table, page, sm_scale=None, softcap=0.0):
    """float64 (o [B,H,D], log2-domain lse [B,H])."""
    B, H, D = q.shape
    group = H // pages.shape[1]
    scale = D ** -0.5 if sm_scale is None else sm_scale
    o = torch.zeros(B, H, D, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v, _ = rows_ref(pages, table[b], n, page, D)
        for h in range(H):
            s = (k[:, h // group] @ q[b, h].double()) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            o[b, h] = torch.softmax(s, 0) @ v[:, h // group]
            lse[b, h] = torch.logsumexp(s, 0) / math.log(2)
    return o, lse
