"""The operators around the paged 4-bit KV cache in 64 bits on the CPU, from their definitions."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def half_step(dtype):
    return HALF_STEP[dtype]


def quantise(x):
    """x [..., d] -> codes (int64), scale, zero (fp16)."""
    x = x.double()
    nan = x.isnan().any(-1)
    x = x.nan_to_num(0.0, math.inf, -math.inf).clamp(-65504, 65504)
    lo, hi = x.amin(-1), x.amax(-1)
    # the difference and the quotient are taken in fp32, as the definition of the stored scale says
    scale = ((hi.float() - lo.float()) / torch.full_like(hi, 15, dtype=torch.float32)).half().clamp(min=2.0 ** -24)
    zero = lo.float().half()
    s, z = scale.double()[..., None], zero.double()[..., None]
    code = torch.round((x - z) / s).clamp(0, 15).long()          # torch.round: ties to even
    code[nan] = 0
    scale, zero = scale.clone(), zero.clone()
    scale[nan] = math.nan
    zero[nan] = math.nan
    return code, scale, zero


def pack(code, words):
    full = torch.zeros(*code.shape[:-1], words * 8, dtype=torch.int64)
    full[..., :code.shape[-1]] = code
    full = (full.view(*code.shape[:-1], words, 8) << (4 * torch.arange(8))).sum(-1)
    return torch.where(full >= 2 ** 31, full - 2 ** 32, full).to(torch.int32)


def unpack(words, d):
    return ((words.long()[..., None] >> (4 * torch.arange(8))) & 15).flatten(-2)[..., :d]


def append(k, v, slots, codes, scales):
    page = codes.shape[3]
    for t, slot in enumerate(slots.tolist()):
        if slot < 0 or slot >= codes.shape[0] * page:
            continue
        for i, x in enumerate((k, v)):
            c, s, z = quantise(x[t])
            codes[slot // page, i, :, slot % page] = pack(c, codes.shape[-1])
            scales[slot // page, i, :, slot % page] = torch.stack((s, z), -1)


def cached(codes, scales, row, i, d, n):
    """The first n tokens of a request with table row `row`: (values [n, heads, d] in 64 bits, scale, codes, present [n])."""
    page = codes.shape[3]
    heads = codes.shape[2]
    val = torch.zeros(n, heads, d, dtype=torch.float64)
    step = torch.zeros(n, heads, dtype=torch.float64)
    there = torch.zeros(n, dtype=torch.bool)
    t = torch.arange(n)
    pages = row[:-(-n // page)].long()[t // page] if n else t
    ok = (pages >= 0) & (pages < codes.shape[0])
    if ok.any():
        w = codes[pages[ok], i, :, (t % page)[ok]]
        m = scales[pages[ok], i, :, (t % page)[ok]].double()
        val[ok] = m[..., 1:] + m[..., :1] * unpack(w, d).double()
        step[ok] = m[..., 0]
        there[ok] = True
    return val, step, there


def attend(q, k, v, seen, scale):
    """q [m, heads, dk], k [n, kv, dk], v [n, kv, dv] (64 bits), seen [m, n] -> out [m, heads, dv], p [m, heads, n] and the largest
    sum of |q||k| products of each query, which bounds how far 32-bit scores can be off."""
    g = q.shape[1] // k.shape[1]
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    x = torch.einsum("mhd,nhd->mhn", q, kk) * scale
    size = torch.einsum("mhd,nhd->mhn", q.abs(), kk.abs()) * scale
    x = x.masked_fill(~seen[:, None, :], -math.inf)
    top = x.amax(-1, keepdim=True) if x.shape[-1] else torch.zeros(*x.shape[:2], 1, dtype=x.dtype)
    e = torch.where(seen[:, None, :], (x - torch.where(top.isinf(), 0.0, top)).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total.clamp(min=1e-300), 0.0)
    out = torch.einsum("mhn,nhd->mhd", p, torch.where(seen.any(0)[:, None, None], vv, 0.0))
    size = torch.where(seen[:, None, :], size, 0.0).amax(-1) if x.shape[-1] else torch.zeros(x.shape[:2], dtype=x.dtype)
    return out, p, size, vv


def plan(lens, new_lens, table, free, count, page, total):
    """Request by request, page by page."""
    table = table.clone()
    width = table.shape[1]
    stack = free[:count].tolist()
    left = count
    slots, pos, cu, short = [], [], [0], False
    for i, (n, add) in enumerate(zip(lens.tolist(), new_lens.tolist())):
        n, add = max(n, 0), max(add, 0)
        for b in range(-(-n // page), min(-(-(n + add) // page), width)):
            left -= 1
            table[i, b] = stack[left] if left >= 0 else -1
            short |= left < 0
        short |= add > 0 and -(-(n + add) // page) > width
        for t in range(n, n + add):
            at = table[i, t // page].item() if t // page < width else -1
            slots.append(at * page + t % page if at >= 0 else -1)
            pos.append(t)
        cu.append(cu[-1] + add)
    short |= len(slots) > total
    slots = (slots + [-1] * total)[:total]
    pos = (pos + [0] * total)[:total]
    after = [max(n, 0) + max(a, 0) for n, a in zip(lens.tolist(), new_lens.tolist())]
    return table, slots, pos, cu, after, max(left, 0), short
