"""GPU: steps around the paged 4-bit KV cache where they can go wrong: consecutive items, large batches, shortages, plans ahead of layers."""
import math

import pytest
import torch

import kv_reference as ref
from test_gpu_kv_attention import _cu, _gen, _prompt_check, _rows

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(params=["binding", "ctypes"])
def route(request, monkeypatch):
    """Both ways into the library: the torch binding and ctypes."""
    from uniql_b200 import ops
    if request.param == "ctypes":
        monkeypatch.setattr(ops, "torch_ext", lambda: None)
    ops.read_and_clear_status("cuda")
    return request.param


@pytest.mark.parametrize("lens,heads,kv", [([3 + i % 60 for i in range(96)], 16, 16), ([1] * 300, 8, 4), ([5, 130, 7, 129, 128, 1] * 20, 24, 8)])
def test_prompt_many_items_with_foreign_rows(lens, heads, kv):
    """A CTA takes many short items one behind the other whose last tile of values reaches into the next request."""
    from uniql_b200 import ops
    g = _gen(len(lens))
    q, k, v = (_rows(g, sum(lens), h, 64, F16) for h in (heads, kv, kv))
    args = q.cuda(), k.cuda(), v.cuda(), _cu(lens).cuda()
    first = ops.prompt_attention(*args)
    for _ in range(20):
        assert torch.equal(ops.prompt_attention(*args), first)
    _prompt_check(first.cpu(), q, k, v, lens, lens, True, 1 / 8)
    assert ops.read_and_clear_status("cuda") == 0


@pytest.mark.parametrize("batch", [4050, 4051, 4095, 4096, 16384])
def test_plan_large_batches(batch):
    """Around the size at which the plan's tables no longer fit the shared memory that a kernel gets by default, and the largest."""
    from uniql_b200 import ops
    g = _gen(batch)
    lens, new = torch.randint(0, 40, (batch,), generator=g), torch.randint(0, 4, (batch,), generator=g)
    table = torch.full((batch, 3), -1, dtype=torch.int32)
    for i, n in enumerate(lens.tolist()):
        table[i, :-(-n // 16)] = i % 7
    free = torch.randperm(batch * 3, generator=g).int()
    total = int(new.sum()) + 2
    want = ref.plan(lens, new, table, free, free.numel(), 16, total)
    d_table = table.cuda()
    got = ops.kv_page_plan(lens.int().cuda(), new.int().cuda(), d_table, free.cuda(), torch.tensor([free.numel()], dtype=torch.int32).cuda(), 16, total)
    assert torch.equal(d_table.cpu(), want[0]) and got[0].tolist() == want[1] and got[1].tolist() == want[2]
    assert got[2].tolist() == want[3] and got[3].tolist() == want[4] and got[4].tolist() == [want[5]]


def test_bounds_behind_the_rows_raise_the_status(route):
    """cu that names more rows than there are: gather fills what there is, prompt attention gives zeros for the requests it cannot
    serve whole and leaves the others as they are; both say so."""
    from uniql_b200 import ops
    g = _gen(40)
    nq, nk = [20, 30, 25], [40, 300, 90]
    q, k, v = _rows(g, 75, 8, 128, F16), _rows(g, 430, 2, 128, F16), _rows(g, 430, 2, 128, F16)
    d = [t.cuda() for t in (q, k, v)]
    clean = ops.prompt_attention(*d, _cu(nq).cuda(), _cu(nk).cuda())
    assert ops.read_and_clear_status("cuda") == 0
    for rows, served in ((429, 2), (341, 2), (340, 2), (339, 1), (40, 1), (39, 0), (0, 0)):
        got = ops.prompt_attention(d[0], d[1][:rows], d[2][:rows], _cu(nq).cuda(), _cu(nk).cuda())
        assert ops.read_and_clear_status("cuda") == 4
        own = sum(nq[:served])
        assert torch.equal(got[:own], clean[:own]) and (got[own:] == 0).all(), rows
    got = ops.prompt_attention(d[0][:60], d[1], d[2], _cu(nq).cuda(), _cu(nk).cuda())          # the last request's queries leave q
    assert ops.read_and_clear_status("cuda") == 4 and torch.equal(got[:50], clean[:50]) and (got[50:] == 0).all()
    got = ops.prompt_attention(*d, _cu(nq).cuda(), torch.tensor([0, 40, 30, 430], dtype=torch.int32).cuda())
    assert ops.read_and_clear_status("cuda") == 4 and torch.equal(got[:20], clean[:20]) and (got[20:50] == 0).all()

    codes, scales = ops.kv4_cache(4, 2, 16, 64)
    ops.kv4_append(k[:64, :, :64].cuda(), v[:64, :, :64].cuda(), torch.arange(64).cuda(), codes, scales)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    whole = ops.kv4_gather(codes, scales, table, _cu([30, 20]).cuda(), 50, 64)
    assert ops.read_and_clear_status("cuda") == 0
    cut = ops.kv4_gather(codes, scales, table, _cu([30, 20]).cuda(), 49, 64)
    assert ops.read_and_clear_status("cuda") == 4
    assert all(torch.equal(a[:49], b) for a, b in zip(whole, cut))


def test_too_few_keys_for_a_chunk():
    """`max_keys` below what the step's requests hold: said in the status word, the requests that fit are served, the rest gives zeros."""
    from uniql_b200 import ops
    from uniql_b200.kv_cache import PagedKV4Cache
    g = _gen(41)
    cache = PagedKV4Cache(1, 30, 2, 64, page_size=16, requests=2, max_tokens=160)
    first, second = [50, 60], [7, 9]
    for new, kw in ((first, dict(fresh=True)), (second, dict(max_keys=126))):
        step = cache.plan(torch.tensor(new, dtype=torch.int32).cuda(), sum(new), **kw)
        q, k, v = (_rows(g, sum(new), h, 64, F16).cuda() for h in (4, 2, 2))
        cache.append(0, k, v, step)
        out = cache.attend(0, q, k, v, step)
    assert ops.read_and_clear_status("cuda") == 0                 # 126 are just enough
    cut = cache.attend(0, q, k, v, step._replace(max_keys=125))
    assert ops.read_and_clear_status("cuda") == 4
    assert torch.equal(cut[:7], out[:7]) and (cut[7:] == 0).all()


@pytest.mark.parametrize("kind", ["decode", "chunk"])
def test_a_step_keeps_its_lengths(kind):
    """The next step may be planned before the layers of this one have run: a step attends to the keys that it was planned with."""
    from uniql_b200.kv_cache import PagedKV4Cache
    g = _gen(42)
    caches = [PagedKV4Cache(1, 30, 2, 64, page_size=16, requests=3, max_tokens=160) for _ in range(2)]
    new = [30, 47, 16]
    rows = [_rows(g, sum(new), h, 64, F16).cuda() for h in (4, 2, 2)]
    more = [1, 1, 1] if kind == "decode" else [5, 20, 1]
    rows2 = [_rows(g, sum(more), h, 64, F16).cuda() for h in (4, 2, 2)]
    outs = []
    for ahead, cache in enumerate(caches):
        step = cache.plan(torch.tensor(new, dtype=torch.int32).cuda(), sum(new), fresh=True)
        cache.append(0, *rows[1:], step)
        cache.codes[0][cache.block_table.max() + 1:] = 0x33333333     # what pages of ended requests hold
        cache.scales[0][cache.block_table.max() + 1:] = 1.0
        step = cache.plan_decode(3) if kind == "decode" else cache.plan(torch.tensor(more, dtype=torch.int32).cuda(), sum(more))
        if ahead:
            cache.plan(torch.tensor([9, 30, 2], dtype=torch.int32).cuda(), 41)
        cache.append(0, *rows2[1:], step)
        outs.append(cache.attend(0, *rows2, step))
    assert torch.equal(*outs)


def _whole(lens, new, table, count, page, width, total):
    """Which requests a step serves: those whose pages, columns and places all fit, in order; an impossible one stands in nobody's way."""
    left, at, stop, served = count, 0, False, []
    for n, add in zip(lens, new):
        need = -(-(n + add) // page) - -(-n // page)
        at += add
        if (add and -(-(n + add) // page) > width) or need > count:
            served.append(False)
            continue
        left -= need
        served.append(not (add and at > total) and not (need and left < 0))
    return served


@pytest.mark.parametrize("new,total,served", [
    ([320, 10, 3], 333, [False, True, True]),                     # more pages than there are: the others are served
    ([64, 70, 8], 142, [True, False, True]),                      # what the first leaves is too little for the second; the third needs none
    ([96, 0, 0], 96, [True, True, True]), ([1, 1, 1], 3, [True, True, True]),
    ([10, 10, 400], 420, [True, True, False]),                    # more columns than the table has
    ([10, 10, 4], 22, [True, True, False]),                       # fewer rows in the step than tokens
    ([0, 700, 0], 700, [True, False, True])])
def test_shortage_leaves_whole_requests_out(route, new, total, served):
    """A request that cannot have all its pages keeps its length and pages, gives zeros, and is served once there are pages again; the
    others of the step are not touched by it."""
    from uniql_b200 import ops
    from uniql_b200.kv_cache import PagedKV4Cache
    g = _gen(sum(new))
    d, heads, kv = 64, 4, 2
    cache = PagedKV4Cache(1, 10, kv, d, page_size=16, requests=3, max_tokens=320)
    old = [0, 48, 5]
    step = cache.plan(torch.tensor(old, dtype=torch.int32).cuda(), 53, fresh=True)
    cache.append(0, *(_rows(g, 53, kv, d, F16).cuda() for _ in range(2)), step)
    before = cache.block_table.clone(), cache.free_pages.clone()
    assert cache.free_count.item() == 6 and ops.read_and_clear_status("cuda") == 0
    assert _whole(old, new, None, 6, 16, 20, total) == served

    step = cache.plan(torch.tensor(new, dtype=torch.int32).cuda(), total)
    held = [o + n * s for o, n, s in zip(old, new, served)]
    taken = sum(-(-h // 16) - -(-o // 16) for h, o in zip(held, old))
    assert ops.read_and_clear_status("cuda") == (0 if all(served) else 8)
    assert cache.lens.tolist() == held and cache.free_count.item() == 6 - taken
    q, k, v = (_rows(g, total, h, d, F16) for h in (heads, kv, kv))
    cache.append(0, k.cuda(), v.cuda(), step)
    out = cache.attend(0, q.cuda(), k.cuda(), v.cuda(), step).cpu()
    assert ops.read_and_clear_status("cuda") == 0                 # what is left out is no key of anybody
    codes, scales, table = cache.codes[0].cpu(), cache.scales[0].cpu(), cache.block_table.cpu()
    at = 0
    for r, (o, n, s) in enumerate(zip(old, new, served)):
        rows = slice(at, min(at + n, total))
        at += n
        slots = step.slots.cpu()[rows]
        if not s:
            assert torch.equal(table[r], before[0].cpu()[r]) and (slots == -1).all() and (out[rows] == 0).all()
            continue
        t = torch.arange(o, o + n)
        assert torch.equal(slots, table[r].long()[t // 16] * 16 + t % 16)
        assert (table[r, :-(-held[r] // 16)] >= 0).all() and (table[r, -(-held[r] // 16):] == -1).all()
        keys, vals = (ref.cached(codes, scales, table[r], i, d, o + n)[0].to(F16) for i in (0, 1))
        _prompt_check(out[rows], q[rows], keys, vals, [n], [o + n], True, 1 / math.sqrt(d))
    # every page is free or in the table, once
    pages = cache.free_pages[:cache.free_count.item()].tolist() + table[table >= 0].tolist()
    assert sorted(pages) == list(range(10))
    # with a request gone its pages serve the one that was left out
    if served == [True, False, True] and total == 142:
        cache.release([0])
        step = cache.plan(torch.tensor([0, 70, 0], dtype=torch.int32).cuda(), 70)
        assert cache.lens.tolist() == [0, 118, 13] and (step.slots >= 0).all() and ops.read_and_clear_status("cuda") == 0


def test_decode_without_a_page_for_one_request(route):
    from uniql_b200 import ops
    from uniql_b200.kv_cache import PagedKV4Cache
    g = _gen(43)
    cache = PagedKV4Cache(1, 4, 2, 64, page_size=16, requests=3, max_tokens=64)
    old = [16, 20, 3]                                             # the first needs a page, and there is none
    step = cache.plan(torch.tensor(old, dtype=torch.int32).cuda(), 39, fresh=True)
    cache.append(0, *(_rows(g, 39, 2, 64, F16).cuda() for _ in range(2)), step)
    q, k, v = (_rows(g, 3, h, 64, F16).cuda() for h in (4, 2, 2))
    step = cache.plan_decode(3)
    cache.append(0, k, v, step)
    out = cache.attend(0, q, k, v, step)
    assert ops.read_and_clear_status("cuda") == 8
    assert cache.lens.tolist() == [16, 21, 4] and step.slots.tolist()[0] == -1 and (out[0] == 0).all()
    args = cache.codes[0], cache.scales[0], cache.block_table
    assert torch.equal(out[1:], ops.kv4_attention(q[1:], *args[:2], cache.block_table[1:], cache.lens[1:])) and (out[1:] != 0).any()
    cache.release([2])
    step = cache.plan_decode(2)
    cache.append(0, k[:2], v[:2], step)
    cache.attend(0, q[:2], k[:2], v[:2], step)
    assert cache.lens.tolist() == [17, 22, 0] and ops.read_and_clear_status("cuda") == 0


@pytest.mark.parametrize("seed", range(4))
def test_whole_requests_step_after_step(route, seed):
    """Many ragged requests over few pages, in place, above and below the size at which a plan becomes two launches."""
    from uniql_b200 import ops
    g = _gen(100 + seed)
    batch, page, width, most = ((7, 16, 9, 40), (300, 16, 12, 90), (1100, 32, 9, 30), (40, 256, 5, 700))[seed]
    pages = batch * 2
    lens, table = [0] * batch, torch.full((batch, width), -1, dtype=torch.int32)
    free, count = torch.randperm(pages, generator=g).int(), pages
    d = [torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda(), free.cuda(), torch.tensor([count], dtype=torch.int32).cuda()]
    some = False
    for step in range(6):
        new = torch.randint(0, most, (batch,), generator=g)
        new[torch.rand(batch, generator=g) < 0.2] = 0
        total = int(new.sum()) - (3 if step == 4 else -5)
        served = _whole(lens, new.tolist(), None, count, page, width, total)
        some |= not all(served)
        got = ops.kv_page_plan(d[0], new.int().cuda(), d[1], d[2], d[3], page, total, in_place=True, whole=True)
        slots, at = [], 0
        for r, (n, add, s) in enumerate(zip(list(lens), new.tolist(), served)):
            if s:
                for b in range(-(-n // page), -(-(n + add) // page)):
                    count -= 1
                    table[r, b] = free[count]
                lens[r] = n + add
            slots += [int(table[r, t // page]) * page + t % page if s else -1 for t in range(n, n + add)]
        slots = (slots + [-1] * total)[:total]
        assert torch.equal(d[1].cpu(), table) and got[0].tolist() == slots and d[0].tolist() == lens and d[3].item() == count
        keys = [n if s else 0 for n, s in zip(lens, served)]
        assert got[2].tolist() == _cu(new.tolist()).clamp(max=total).tolist() and got[5].tolist() == keys and got[6].tolist() == _cu(keys).tolist()
        assert ops.read_and_clear_status("cuda") == (0 if all(served) else 8)
        if step == 2:                                             # half of the requests end: their pages go back
            for r in range(0, batch, 2):
                back = table[r][table[r] >= 0]
                free[count:count + back.numel()] = back
                count += back.numel()
                table[r], lens[r] = -1, 0
            for t, x in zip(d, (torch.tensor(lens, dtype=torch.int32), table, free, torch.tensor([count], dtype=torch.int32))):
                t.copy_(x)
    assert some


# ------------------------------------------------------------------------------------------------ branches of large calls
@pytest.mark.parametrize("short", [False, True])
def test_plan_in_place_as_two_launches(route, short):
    """More than 8192 new tokens of many ragged requests, in place, step after step; in the last one pages run out."""
    from uniql_b200 import ops
    g = _gen(50)
    batch, page, width = 1200, 16, 12
    free = torch.randperm(6 * batch, generator=g).int()
    count = free.numel() if not short else 3 * batch
    lens, table = torch.zeros(batch, dtype=torch.int32), torch.full((batch, width), -1, dtype=torch.int32)
    d = [t.cuda() for t in (lens, table, free, torch.tensor([count], dtype=torch.int32))]
    for step in range(4):
        new = torch.randint(0, 30, (batch,), generator=g).int()
        total = int(new.sum()) + 7
        assert total > 8192
        want = ref.plan(lens, new, table, free, count, page, total)
        got = ops.kv_page_plan(d[0], new.cuda(), d[1], d[2], d[3], page, total, in_place=True)
        table, lens, count = want[0], torch.tensor(want[4], dtype=torch.int32), want[5]
        assert got[0].tolist() == want[1] and got[1].tolist() == want[2] and got[2].tolist() == want[3]
        assert torch.equal(d[1].cpu(), table) and torch.equal(d[0].cpu(), lens) and d[3].item() == count
        assert ops.read_and_clear_status("cuda") == (8 if want[6] else 0)
    assert want[6] == short


@pytest.mark.parametrize("batch", [1023, 1024, 1025, 3000])
def test_gather_of_many_requests(route, batch):
    """Up to 1024 requests the bounds are searched in shared memory, beyond them in global memory; many are empty, all start late."""
    from uniql_b200 import ops
    g = _gen(batch)
    pages, page, d, kv = 64, 16, 64, 2
    codes, scales = ops.kv4_cache(pages, kv, page, d)
    n = pages * page
    ops.kv4_append(_rows(g, n, kv, d, F16).cuda(), _rows(g, n, kv, d, F16).cuda(), torch.arange(n).cuda(), codes, scales)
    table = torch.randint(0, pages, (batch, 3), generator=g).int()
    counts = torch.randint(0, 5, (batch,), generator=g)
    counts[torch.rand(batch, generator=g) < 0.5] = 0
    counts[-1] = 3
    starts = torch.randint(0, 40, (batch,), generator=g).int()
    total = int(counts.sum()) + 9
    got = ops.kv4_gather(codes, scales, table.cuda(), _cu(counts.tolist()).cuda(), total, d, starts=starts.cuda())
    req = torch.repeat_interleave(torch.arange(batch), counts)
    at = torch.cat([torch.arange(s, s + c) for s, c in zip(starts.tolist(), counts.tolist())])
    slots = table[req, at // page].long() * page + at % page
    every = ops.kv4_gather(codes, scales, torch.arange(pages, dtype=torch.int32)[None].cuda(), _cu([n]).cuda(), n, d)
    for x, rows in zip(got, every):
        assert torch.equal(x[:total - 9], rows[slots.cuda()]) and (x[total - 9:] == 0).all()
    assert ops.read_and_clear_status("cuda") == 0


def _striped(lens, heads, kv, d, g):
    """Queries and a cache in which every 64 tokens raise two channels of the values, which no part of a list can be left out without
    changing: all weights are alike within a factor of two."""
    page = 64
    blocks = [-(-n // page) for n in lens]
    pages = sum(blocks)
    order, table, at = torch.randperm(pages, generator=g).int(), torch.zeros(len(lens), max(blocks), dtype=torch.int32), 0
    codes = torch.zeros(pages, 2, kv, page, 8, dtype=torch.int32)
    scales = torch.zeros(pages, 2, kv, page, 2, dtype=F16)
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b]
        at += b
    c, s, z = ref.quantise(torch.randn(pages, kv, page, d, generator=g).half() * 0.1)
    codes[:, 0], scales[:, 0] = ref.pack(c, 8), torch.stack((s, z), -1)
    for i, b in enumerate(blocks):
        for t in range(b):
            x = torch.zeros(kv, page, d)
            x[..., (7 * t + i) % d] = 1.0
            x[..., (11 * t + 3 * i + 5) % d] = 1.0
            c, s, z = ref.quantise(x)
            codes[table[i, t].item(), 1], scales[table[i, t].item(), 1] = ref.pack(c, 8), torch.stack((s, z), -1)
    return torch.randn(len(lens), heads, d, generator=g).half(), codes, scales, table


@pytest.mark.parametrize("lens", [[40000], [24700] * 6, [24700] * 7, [25000] * 8, [24700] * 13, [24800] * 14, [24800] * 15, [30000, 24700, 100, 50000]])
def test_no_part_of_a_long_list_is_lost(lens):
    """Lists that are cut into 30 to 450 parts, more than 32 of which take the second turn of the join: each 64 tokens show in the result.
    Bound per value: the result's rounding, weights rounded to fp16 next to codes centred by 8 steps of 1/15, scores in 32 bits."""
    from uniql_b200 import ops
    g = _gen(len(lens))
    d = 64
    q, codes, scales, table = _striped(lens, 2, 1, d, g)
    got = ops.kv4_attention(*(t.cuda() for t in (q, codes, scales, table)), torch.tensor(lens, dtype=torch.int32).cuda()).cpu()
    for b, n in enumerate(lens):
        k = ref.cached(codes, scales, table[b], 0, d, n)[0]
        v = ref.cached(codes, scales, table[b], 1, d, n)[0]
        out, p, size, _ = ref.attend(q[b:b + 1].double(), k, v, torch.ones(1, n, dtype=torch.bool), 1 / 8)
        # rounded weights: independent errors of at most 2^-11 of each term |c - 8| / 15 <= 8 / 15, so five deviations of their sum stay
        # within 5 * 2^-11 * 8 / 15 * sqrt(sum p^2); their mean is zero because rounding is to nearest
        off = 2 * (d + 16) * 2.0 ** -23 * (size[0] + 1.0)[:, None] + 2.0 ** -18
        tol = out[0].abs() * (2.0 ** -11 + off) + 5 * 2.0 ** -11 * 8 / 15 * p[0].norm(dim=-1)[:, None] + 2.0 ** -18
        assert ((got[b].double() - out[0]).abs() <= tol).all(), b
        # any 64 tokens missing from the plain result would show
        for t in range(0, n - 63, max(64, n // 64 // 40 * 64)):
            rest = torch.ones(n, dtype=torch.bool)
            rest[t:t + 64] = False
            w = p[0][:, rest]
            less = (w @ v[rest, 0]) / w.sum(-1, keepdim=True)
            assert ((less - out[0]).abs() > 2 * tol).any(), (b, t)


@pytest.mark.parametrize("bad", [0, 31, 4000, 5999])
def test_bounds_of_thousands_of_requests_are_looked_over(bad):
    """Most of the grid's CTAs never begin (others take their places): the look at the bounds must not be theirs."""
    from uniql_b200 import ops
    g = _gen(60)
    n = 6000
    q, k, v = (_rows(g, n, h, 64, F16).cuda() for h in (2, 1, 1))
    cu = torch.arange(n + 1, dtype=torch.int32).cuda()
    clean = ops.prompt_attention(q, k, v, cu, cu)
    assert ops.read_and_clear_status("cuda") == 0
    cu_k = cu.clone()
    cu_k[bad] = n + 5 if bad else -1                              # one or two requests whose keys do not all exist
    got = ops.prompt_attention(q, k, v, cu, cu_k)
    assert ops.read_and_clear_status("cuda") == 4
    hit = torch.zeros(n, dtype=torch.bool)
    hit[max(bad - 1, 0):bad + 1] = True
    assert (got[hit] == 0).all() and torch.equal(got[~hit], clean[~hit])


def test_step_plan_without_requests_and_out_of_place(route):
    from uniql_b200 import ops
    from uniql_b200.kv_cache import PagedKV4Cache
    cache = PagedKV4Cache(1, 9, 1, 64, page_size=16, requests=2, max_tokens=64)
    step = cache.plan(torch.zeros(0, dtype=torch.int32).cuda(), 3)
    assert step.slots.tolist() == [-1] * 3 and step.cu_keys.tolist() == [0] and step.lens.numel() == 0
    out = cache.attend(0, *(torch.ones(3, h, 64, dtype=F16).cuda() for h in (2, 1, 1)), step)
    assert (out == 0).all() and cache.free_count.item() == 9
    new = torch.tensor([20, 70], dtype=torch.int32).cuda()        # the second has more tokens than the table columns
    got = ops.kv_page_plan(cache.lens, new, cache.block_table, cache.free_pages, cache.free_count, 16, 90, whole=True)
    assert cache.lens.tolist() == [0, 0] and cache.free_count.item() == 9
    assert [t.tolist() for t in got[2:]] == [[0, 20, 90], [20, 0], [7], [20, 0], [0, 20, 20]]
    assert (got[0][:20] >= 0).all() and (got[0][20:] == -1).all() and ops.read_and_clear_status("cuda") == 8
