"""The attention part of a decoder block around a paged KV cache held in 4 bits, as cases that can be timed and compared.

Five operators, in the order a serving loop calls them:

  plan     block tables, slot map and positions of a step's new tokens from the requests' lengths (pages come off a stack)
  append   new K/V rows quantised to 4 bits and stored at their slots; read back with `gather`, so that what is held in 4 bits
           comes out as the values it stands for
  gather   a range of each request's cached rows, dequantised and packed (what a later chunk of a prompt attends to)
  decode   one query token per request over its cached rows
  prompt   causal attention of packed prompts of different lengths, with keys that may reach further back than the queries

Cache: int32 codes [pages, 2, kv_heads, page_size, Dp / 8] (0 is K, 1 is V; channel d of a row in bits 4 (d % 8) of word
d / 8; Dp is the head size rounded up to 64 or 128) and fp16 [pages, 2, kv_heads, page_size, 2] with scale and zero of each
row: value = zero + scale * code.

`run` computes the plain form with elementary torch operations, or, with `own`, makes the library's calls.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"

# Head layouts of the benchmark and the tests: Llama-3.1-8B, Qwen2.5-7B, and the Llama layer after structured compression
# (28 of 32 query heads; 112 of 128 channels).
LLAMA = dict(heads=32, kv_heads=8, dk=128, dv=128)
QWEN = dict(heads=28, kv_heads=4, dk=128, dv=128)
SLICED = dict(heads=32, kv_heads=8, dk=112, dv=112)


def listed():
    return [
        # a decode step of a served batch: one new token for each of 64 requests
        dict(name="plan_decode64", op="plan", batch=64, old=8192, new=1, page=64, mix=1),
        # a large step that mixes prompts and single tokens
        dict(name="plan_mixed1024", op="plan", batch=1024, old=2048, new=512, page=16, mix=2),
        # the cache write of the same decode step
        dict(name="append_decode64", op="append", batch=64, old=8192, new=1, page=64, mix=3, dtype="float16", **LLAMA),
        # the cache write of a batch of long prompts
        dict(name="append_prompts", op="append", batch=8, old=0, new=4096, page=64, mix=4, dtype="bfloat16", **LLAMA),
        # the prefix that a prompt's next chunk attends to, on a layer with sliced heads
        dict(name="gather_prefix_sliced", op="gather", batch=3, old=2001, page=32, mix=5, dtype="float16", **SLICED),
        # the cached rows of a whole batch
        dict(name="gather_batch32", op="gather", batch=32, old=8192, page=64, mix=6, dtype="float16", **LLAMA),
        # interactive decoding: one request
        dict(name="decode_single", op="decode", batch=1, old=1000, page=64, mix=0, dtype="float16", **LLAMA),
        # a served batch of requests of very different lengths, an idle one among them
        dict(name="decode_ragged64", op="decode", batch=64, old=8192, page=64, mix=7, dtype="bfloat16", **QWEN),
        # long contexts
        dict(name="decode_long8", op="decode", batch=8, old=131072, page=128, mix=0, dtype="float16", **LLAMA),
        # a short prompt
        dict(name="prompt_short", op="prompt", batch=1, old=0, new=77, mix=0, dtype="float16", **QWEN),
        # packed prompts of different lengths, some behind a cached prefix
        dict(name="prompt_packed16", op="prompt", batch=16, old=1500, new=2048, mix=8, dtype="bfloat16", **LLAMA),
        # one long prompt: the largest case
        dict(name="prompt_long", op="prompt", batch=1, old=0, new=16384, mix=0, dtype="float16", **LLAMA),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    if rng.random() < 0.5:
        return dict(rng.choice([LLAMA, QWEN, SLICED]))
    kv = rng.choice([1, 2, 4, 5, 8])
    d = rng.choice([64, 128, 128, 8 * rng.randint(5, 16)])
    return dict(heads=kv * rng.choice([1, 2, 3, 4, 6, 7, 8]), kv_heads=kv, dk=d, dv=d)


def draw(rng):
    """One more case of the same ranges: lengths and batches over their logarithm, other head layouts, pages and types."""
    op = rng.choice(["plan", "append", "gather", "decode", "decode", "prompt", "prompt"])
    case = dict(op=op, mix=rng.randint(0, 1) * rng.randint(1, 10 ** 6))
    if op == "plan":
        case.update(batch=_log_int(rng, 1, 1024), old=_log_int(rng, 1, 16384), new=_log_int(rng, 1, 512), page=rng.choice([16, 32, 64, 128]))
        return case
    case.update(dtype=rng.choice(["float16", "bfloat16"]), **_heads(rng))
    if op == "prompt":
        new = _log_int(rng, 1, 4096)
        batch = _log_int(rng, 1, max(1, min(32, 8192 // new)))
        case.update(batch=batch, new=new, old=0 if rng.random() < 0.6 else _log_int(rng, 1, 4096))
        return case
    batch = _log_int(rng, 1, 128)
    case.update(batch=batch, old=_log_int(rng, 1, min(65536, 262144 // batch)), page=rng.choice([16, 32, 64, 128]))
    if op == "append":
        case.update(new=_log_int(rng, 1, max(1, 16384 // batch)))
    return case


# ------------------------------------------------------------------------------------------------ lengths
def _lengths(case):
    """(cached tokens, new tokens) of each request. `mix` 0: all as long as the case says; else ragged, drawn from it."""
    b, old, new = case["batch"], case["old"], case.get("new", 0)
    if not case["mix"]:
        return [old] * b, [new] * b
    r = random.Random(case["mix"])
    olds = [r.randint(0, old) for _ in range(b)]
    news = [r.randint(1, new) if new else 0 for _ in range(b)]
    if case["op"] in ("decode", "gather") and b > 1:
        olds[r.randrange(b)] = 0                       # an idle row of a padded batch
    if case["op"] in ("decode", "gather"):
        olds[-1] = max(1, olds[-1])
    return olds, news


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEVICE)


def _pad(d):
    return 64 if d <= 64 else 128


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, part):
    return torch.Generator(device=DEVICE).manual_seed((int(seed) * 1009 + part) % (2 ** 62))


def _rows(seed, part, tokens, heads, d, dtype, outliers):
    """N(0, 1) rows; `outliers`: every 16th channel four times as large, as the key channels of real models are."""
    x = torch.randn(tokens, heads, d, generator=_gen(seed, part), device=DEVICE)
    if outliers:
        x[..., ::16] *= 4
    return x.to(getattr(torch, dtype))


def _tables(case, seed, totals):
    """Block table for `totals` tokens per request over shuffled pages, the number of pages, and each token's slot."""
    page = case["page"]
    blocks = [-(-n // page) for n in totals]
    width = max(1, max(blocks))
    pages = sum(blocks) + 3
    order = torch.randperm(pages, generator=_gen(seed, 90), device=DEVICE).to(torch.int32)
    col = torch.arange(width, device=DEVICE)[None, :]
    nb = _ints(blocks, torch.int64)[:, None]
    first = _ints(_cu(blocks)[:-1], torch.int64)[:, None]
    table = torch.where(col < nb, order[(first + col).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=DEVICE))
    return table.contiguous(), pages


def _spread(lens, total):
    """For packed tokens of `lens`: their request and their place in it."""
    n = _ints(lens, torch.int64)
    req = torch.repeat_interleave(torch.arange(len(lens), device=DEVICE), n, output_size=total)
    return req, torch.arange(total, device=DEVICE) - _ints(_cu(lens)[:-1], torch.int64)[req]


def _slots(case, table, starts, lens):
    req, at = _spread(lens, sum(lens))
    at = at + _ints(starts, torch.int64)[req]
    return table[req, at // case["page"]].long() * case["page"] + at % case["page"]


def _fill(case, seed, table, pages, lens):
    """A cache that holds `lens` tokens per request."""
    dp, kv, page = _pad(max(case["dk"], case["dv"])), case["kv_heads"], case["page"]
    codes = torch.zeros(pages, 2, kv, page, dp // 8, dtype=torch.int32, device=DEVICE)
    scales = torch.zeros(pages, 2, kv, page, 2, dtype=torch.float16, device=DEVICE)
    slots = _slots(case, table, [0] * len(lens), lens)
    step = max(1, (1 << 25) // (kv * 128))
    for part, at in enumerate(range(0, slots.numel(), step)):
        s = slots[at:at + step]
        k = _rows(seed, 1000 + 2 * part, s.numel(), kv, case["dk"], case["dtype"], True)
        v = _rows(seed, 1001 + 2 * part, s.numel(), kv, case["dv"], case["dtype"], False)
        _store(codes, scales, s, k, v)
    return codes, scales


def prepare(case, seed):
    op = case["op"]
    olds, news = _lengths(case)
    state = dict(op=op, case=case)
    if op == "plan":
        page = case["page"]
        table, used = _tables(case, seed, olds)
        width = max(-(-(o + n) // page) for o, n in zip(olds, news))
        extra = sum(-(-(o + n) // page) for o, n in zip(olds, news)) + 5
        wide = torch.full((len(olds), width), -1, dtype=torch.int32, device=DEVICE)
        wide[:, :table.shape[1]] = table[:, :width]
        free = (used + torch.randperm(extra, generator=_gen(seed, 91), device=DEVICE)).to(torch.int32)
        state.update(lens=_ints(olds), new_lens=_ints(news), table=wide, free=free, count=_ints([extra]), total=sum(news), page=page)
        return state
    dtype = case["dtype"]
    state.update(dk=case["dk"], dv=case["dv"], dtype=getattr(torch, dtype))
    if op == "prompt":
        keys = [o + n for o, n in zip(olds, news)]
        state.update(q=_rows(seed, 1, sum(news), case["heads"], case["dk"], dtype, False), k=_rows(seed, 2, sum(keys), case["kv_heads"], case["dk"], dtype, False),
                     v=_rows(seed, 3, sum(keys), case["kv_heads"], case["dv"], dtype, False), cu_q=_ints(_cu(news)), cu_k=_ints(_cu(keys)), news=news, keys=keys)
        return state
    totals = [o + n for o, n in zip(olds, news)]
    table, pages = _tables(case, seed, totals)
    state.update(table=table, page=case["page"])
    if op == "append":
        tokens = sum(news)
        dp, kv = _pad(max(case["dk"], case["dv"])), case["kv_heads"]
        state.update(codes=torch.zeros(pages, 2, kv, case["page"], dp // 8, dtype=torch.int32, device=DEVICE),
                     scales=torch.zeros(pages, 2, kv, case["page"], 2, dtype=torch.float16, device=DEVICE),
                     k=_rows(seed, 2, tokens, kv, case["dk"], dtype, True), v=_rows(seed, 3, tokens, kv, case["dv"], dtype, False),
                     slots=_slots(case, table, olds, news), starts=_ints(olds), cu=_ints(_cu(news)), total=tokens, lens=news)
        return state
    codes, scales = _fill(case, seed, table, pages, olds)
    state.update(codes=codes, scales=scales, lens=olds)
    if op == "gather":
        state.update(cu=_ints(_cu(olds)), total=sum(olds), starts=None)
    else:
        state.update(q=_rows(seed, 1, len(olds), case["heads"], case["dk"], dtype, False), cached=_ints(olds))
    return state


# ------------------------------------------------------------------------------------------------ plain form
def _quantise(x):
    """Codes (whole numbers 0 to 15), scale and zero of each row. The quotient is taken in 64 bits: codes next to a tie."""
    f = x.float().clamp(-65504.0, 65504.0)
    lo, hi = f.amin(-1), f.amax(-1)
    scale = torch.clamp(((hi - lo) / torch.full_like(hi, 15.0)).to(torch.float16), min=2.0 ** -24)
    zero = lo.to(torch.float16)
    code = torch.round((f.double() - zero[..., None].double()) / scale[..., None].double()).clamp(0, 15)
    return code, scale, zero


def _pack(code, words):
    shape = code.shape[:-1]
    full = torch.zeros(*shape, words * 8, dtype=torch.int64, device=code.device)
    full[..., :code.shape[-1]] = code.to(torch.int64)
    full = (full.view(*shape, words, 8) << (4 * torch.arange(8, device=code.device))).sum(-1)
    return torch.where(full >= 1 << 31, full - (1 << 32), full).to(torch.int32)


def _unpack(words, d):
    c = (words[..., None] >> (4 * torch.arange(8, device=words.device, dtype=torch.int32))) & 15
    return c.flatten(-2)[..., :d].float()


def _store(codes, scales, slots, k, v):
    page = codes.shape[3]
    block, at = slots // page, slots % page
    for i, x in enumerate((k, v)):
        code, scale, zero = _quantise(x)
        codes[block, i, :, at] = _pack(code, codes.shape[-1])
        scales[block, i, :, at] = torch.stack((scale, zero), -1)


def _values(words, meta, d):
    return meta[..., 1:2].float() + meta[..., 0:1].float() * _unpack(words, d)


def _plain_gather(s):
    req, at = _spread(s["lens"], s["total"])
    if s["starts"] is not None:
        at = at + s["starts"].long()[req]
    block, at = s["table"][req, at // s["page"]].long(), at % s["page"]
    return [_values(s["codes"][block, i, :, at], s["scales"][block, i, :, at], d).to(s["dtype"]) for i, d in ((0, s["dk"]), (1, s["dv"]))]


def _softmax(x):
    """Softmax of the last axis, overwriting it; a row of minus infinities becomes zeros."""
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    return x.div_(torch.where(total == 0, torch.ones_like(total), total))


def _plain_decode(s):
    q, kv = s["q"].float(), s["codes"].shape[2]
    block = s["table"].long().clamp(min=0)
    b, width = block.shape
    place = torch.arange(width * s["page"], device=q.device)
    mask = (place[None, :] >= s["cached"][:, None])[:, None, None, :]

    def rows(i, d):
        x = _values(s["codes"][block, i], s["scales"][block, i], d)             # [b, blocks, kv, page, d]
        return x.transpose(1, 2).reshape(b, kv, width * s["page"], d)

    x = (q.view(b, kv, -1, s["dk"]) @ rows(0, s["dk"]).transpose(-1, -2)).mul_(1.0 / math.sqrt(s["dk"]))
    p = _softmax(x.masked_fill_(mask, float("-inf")))
    return (p @ rows(1, s["dv"])).reshape(b, -1, s["dv"]).to(s["dtype"])


def _plain_prompt(s):
    kv, b = s["k"].shape[1], len(s["news"])
    lq, lk = max(s["news"]), max(s["keys"])
    iq, ik = torch.arange(lq, device=DEVICE), torch.arange(lk, device=DEVICE)
    nq, nk = s["cu_q"].diff().long()[:, None], s["cu_k"].diff().long()[:, None]
    q = s["q"][(s["cu_q"][:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)].float()          # [b, lq, heads, dk]
    at = (s["cu_k"][:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    k, v = s["k"][at].float(), s["v"][at].float()
    g = q.shape[2] // kv
    q = q.view(b, lq, kv, g, s["dk"]).permute(0, 2, 3, 1, 4).reshape(b, kv, g * lq, s["dk"])
    x = (q @ k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(s["dk"])).view(b, kv, g, lq, lk)
    hidden = (ik[None, None, :] > (iq[None, :] + nk - nq)[..., None]) | (ik[None, None, :] >= nk[..., None])
    p = _softmax(x.masked_fill_(hidden[:, None, None], float("-inf"))).view(b, kv, g * lq, lk)
    out = (p @ v.transpose(1, 2)).view(b, kv, g, lq, s["dv"]).permute(0, 3, 1, 2, 4).reshape(b, lq, kv * g, s["dv"]).to(s["dtype"])
    req, place = _spread(s["news"], s["q"].shape[0])
    return out[req, place]


def _plain_plan(s):
    page, table, old, new = s["page"], s["table"], s["lens"].long(), s["new_lens"].long()
    had, has = (old + page - 1) // page, (old + new + page - 1) // page
    need = has - had
    first = need.cumsum(0) - need
    col = torch.arange(table.shape[1], device=DEVICE)[None, :]
    fresh = (col >= had[:, None]) & (col < has[:, None])
    rank = first[:, None] + col - had[:, None]
    table.copy_(torch.where(fresh, s["free"][(s["count"].long() - 1 - rank).clamp(0, s["free"].numel() - 1)], table))
    req = torch.repeat_interleave(torch.arange(old.numel(), device=DEVICE), new, output_size=s["total"])
    ends = new.cumsum(0)
    at = torch.arange(s["total"], device=DEVICE) - (ends - new)[req] + old[req]
    slots = table[req, at // page].long() * page + at % page
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=DEVICE), ends)).to(torch.int32)
    return table, slots, at, cu, (old + new).to(torch.int32), (s["count"].long() - need.sum()).to(torch.int32)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        from uniql_b200 import ops
        if s["op"] == "plan":
            return (s["table"], *ops.kv_page_plan(s["lens"], s["new_lens"], s["table"], s["free"], s["count"], s["page"], s["total"]))
        if s["op"] == "append":
            ops.kv4_append(s["k"], s["v"], s["slots"], s["codes"], s["scales"])
        if s["op"] in ("append", "gather"):
            return ops.kv4_gather(s["codes"], s["scales"], s["table"], s["cu"], s["total"], s["dk"], s["dv"], dtype=s["dtype"], starts=s["starts"])
        if s["op"] == "decode":
            return ops.kv4_attention(s["q"], s["codes"], s["scales"], s["table"], s["cached"], head_dim_v=s["dv"])
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
    if s["op"] == "plan":
        return _plain_plan(s)
    if s["op"] == "append":
        _store(s["codes"], s["scales"], s["slots"], s["k"], s["v"])
    if s["op"] in ("append", "gather"):
        return _plain_gather(s)
    return _plain_decode(s) if s["op"] == "decode" else _plain_prompt(s)


def work(case):
    """Each input read once, each output written once; products of visible query-key pairs."""
    olds, news = _lengths(case)
    if case["op"] == "plan":
        page = case["page"]
        taken = sum(-(-(o + n) // page) - -(-o // page) for o, n in zip(olds, news))
        return {"bytes": 16.0 * len(olds) + 8.0 * taken + 16.0 * sum(news), "flops": float(sum(news))}
    h, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    row = (dk + dv) / 2 + 8                                              # cached bytes of a token and kv head
    if case["op"] == "append":
        t = sum(news) * kv
        return {"bytes": t * (2 * 2.0 * (dk + dv) + 2 * row) + 8.0 * sum(news), "flops": 6.0 * t * (dk + dv)}
    if case["op"] == "gather":
        t = sum(olds) * kv
        return {"bytes": t * (2.0 * (dk + dv) + row), "flops": 2.0 * t * (dk + dv)}
    if case["op"] == "decode":
        return {"bytes": sum(olds) * kv * row + 2.0 * len(olds) * h * (dk + dv), "flops": 2.0 * sum(olds) * h * (dk + dv)}
    pairs = sum(n * o + n * (n + 1) / 2 for o, n in zip(olds, news))
    keys = sum(olds) + sum(news)
    return {"bytes": 2.0 * (sum(news) * h + keys * kv) * (dk + dv), "flops": 2.0 * pairs * h * (dk + dv)}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The operators from their definitions, request by request, in 64 bits; whole numbers with Python's."""
    s = prepare(case, seed)
    olds, news = _lengths(case)
    op = case["op"]
    if op == "plan":
        page, free, table = case["page"], s["free"].tolist(), s["table"].tolist()
        slots, places = [], []
        for row, o, n in zip(table, olds, news):
            for t in range(o, o + n):
                if t % page == 0:
                    row[t // page] = free.pop()
                slots.append(row[t // page] * page + t % page)
                places.append(t)
        return (_ints(table), _ints(slots, torch.int64), _ints(places, torch.int64), _ints(_cu(news)), _ints([o + n for o, n in zip(olds, news)]), _ints([len(free)]))

    def nearest(x):
        """What 4 bits hold of a row: the nearest of sixteen steps from its least value."""
        x = x.double().clamp(-65504, 65504)
        base = x.min(-1, keepdim=True).values
        step = ((x.max(-1, keepdim=True).values - base) / 15).half().double().clamp(min=2.0 ** -24)
        base = base.half().double()
        y = (x - base) / step
        down = y.floor()
        up = (y - down > 0.5) | ((y - down == 0.5) & (down % 2 == 1))
        return base + step * (down + up).clamp(0, 15)

    if op == "append":
        return [nearest(s["k"]), nearest(s["v"])]

    def cached(i, d, r, n):
        """The first n rows of request r as they are held: [kv, n, d]."""
        used = s["table"][r, :-(-n // s["page"])].long()
        w = s["codes"][used, i].transpose(0, 1).flatten(1, 2)[:, :n].long()
        m = s["scales"][used, i].transpose(0, 1).flatten(1, 2)[:, :n].double()
        c = torch.stack([(w >> (4 * j)) & 15 for j in range(8)], -1).flatten(-2)[..., :d]
        return m[..., 1:] + m[..., :1] * c.double()

    def attend(q, k, v, first):
        """q [h, m, d] over k, v [kv, n, d]; query i sees the keys below first + i."""
        g = q.shape[0] // k.shape[0]
        seen = torch.arange(k.shape[1], device=DEVICE)[None, :] < (first + torch.arange(q.shape[1], device=DEVICE))[:, None]
        out = []
        for h in range(q.shape[0]):
            e = (q[h] @ k[h // g].T / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf)
            e = torch.where(seen, (e - e.max(-1, keepdim=True).values).exp(), torch.zeros_like(e))
            out.append(e @ v[h // g] / e.sum(-1, keepdim=True).clamp(min=1e-300))
        return torch.stack(out, 1)

    if op == "gather":
        return [torch.cat([cached(i, d, r, n).transpose(0, 1) for r, n in enumerate(olds)]) for i, d in ((0, s["dk"]), (1, s["dv"]))]
    if op == "decode":
        out = torch.zeros(len(olds), case["heads"], s["dv"], dtype=torch.float64, device=DEVICE)
        for r, n in enumerate(olds):
            if n:
                out[r] = attend(s["q"][r].double()[:, None], cached(0, s["dk"], r, n), cached(1, s["dv"], r, n), n)[0]
        return out
    out, cq, ck = [], _cu(news), _cu(s["keys"])
    for r, o in enumerate(olds):
        q, k, v = (s[x][c[r]:c[r + 1]].double().transpose(0, 1) for x, c in (("q", cq), ("k", ck), ("v", ck)))
        out.append(attend(q, k, v, o + 1))
    return torch.cat(out)
