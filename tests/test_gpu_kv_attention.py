"""GPU: paged 4-bit KV cache and the attention around it against 64-bit references (tests/kv_reference.py)."""
import math

import pytest
import torch

import kv_reference as ref

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


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(g, tokens, heads, d, dtype, spread=1.0):
    return (torch.randn(tokens, heads, d, generator=g) * spread).to(dtype)


def _table(g, lens, page, pages=None, width=None):
    """Shuffled pages for `lens` tokens per request; returns the table and the number of pages."""
    blocks = [-(-n // page) for n in lens]
    width = max([1] + blocks) if width is None else width
    total = sum(blocks) + 2 if pages is None else pages
    order = torch.randperm(total, generator=g).int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _slots(table, lens, page, starts=None):
    out = []
    for i, n in enumerate(lens):
        s = starts[i] if starts else 0
        out += [table[i, t // page].item() * page + t % page for t in range(s, s + n)]
    return torch.tensor(out, dtype=torch.int64)


def _cu(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32) if lens else torch.zeros(1, dtype=torch.int32)


def _filled(g, lens, page, heads, dk, dv, dtype=F16, spread=1.0):
    """A cache filled by the reference's quantiser: codes, scales, table on the CPU."""
    table, pages = _table(g, lens, page)
    words = 8 if max(dk, dv) <= 64 else 16
    codes = torch.randint(-2 ** 31, 2 ** 31 - 1, (pages, 2, heads, page, words), generator=g).int()     # what nobody wrote is junk
    scales = torch.full((pages, 2, heads, page, 2), math.nan, dtype=F16)
    n = sum(lens)
    slots = _slots(table, lens, page)
    for i, (d, sp) in enumerate(((dk, 1.0), (dv, spread))):
        x = _rows(g, n, heads, d, dtype, sp)
        c, s, z = ref.quantise(x)
        codes[slots // page, i, :, slots % page] = ref.pack(c, words)
        scales[slots // page, i, :, slots % page] = torch.stack((s, z), -1)
    return codes, scales, table


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("lens,new,page", [
    ([0], [1], 16), ([16], [1], 16), ([15], [1], 16), ([15], [2], 16), ([0, 0, 0], [0, 0, 0], 32), ([5], [0], 16),
    ([100, 0, 63, 64, 65], [1, 1, 1, 1, 1], 64), ([0, 31, 32, 33], [4000, 0, 700, 33], 32), ([7] * 1300, [1] * 1300, 128),
    (list(range(700)), [i % 5 for i in range(700)], 16), ([0], [9000], 256), ([-3, 4], [2, -1], 16)])
def test_plan(route, lens, new, page):
    from uniql_b200 import ops
    g = _gen(len(lens))
    width = max(1, max(-(-(max(a, 0) + max(b, 0)) // page) for a, b in zip(lens, new))) + 1
    table, used = _table(g, [max(n, 0) for n in lens], page, width=width)
    free = used + torch.randperm(600 + 40 * len(lens), generator=g).int()
    count = free.numel() - 7
    total = sum(max(n, 0) for n in new) + 3                      # three rows of padding
    want = ref.plan(torch.tensor(lens), torch.tensor(new), table, free, count, page, total)
    d_table = table.cuda()
    got = ops.kv_page_plan(torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(new, dtype=torch.int32).cuda(), d_table,
                           free.cuda(), torch.tensor([count], dtype=torch.int32).cuda(), page, total)
    assert torch.equal(d_table.cpu(), want[0])
    assert got[0].tolist() == want[1] and got[1].tolist() == want[2] and got[2].tolist() == want[3]
    assert got[3].tolist() == want[4] and got[4].tolist() == [want[5]]
    assert ops.read_and_clear_status("cuda") == 0


def test_plan_in_place_step_after_step(route):
    from uniql_b200 import ops
    g = _gen(3)
    page, batch, width = 16, 5, 9
    lens = torch.zeros(batch, dtype=torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32)
    free = torch.randperm(80, generator=g).int()
    count = 80
    d = [t.cuda() for t in (lens, table, free, torch.tensor([count], dtype=torch.int32))]
    for step in range(12):
        new = torch.randint(0, 14, (batch,), generator=g).int()
        total = int(new.sum())
        want = ref.plan(lens, new, table, free, count, page, total)
        got = ops.kv_page_plan(d[0], new.cuda(), d[1], d[2], d[3], page, total, in_place=True)
        table, lens, count = want[0], torch.tensor(want[4], dtype=torch.int32), want[5]
        assert got[0].tolist() == want[1] and torch.equal(d[1].cpu(), table)
        assert torch.equal(d[0].cpu(), lens) and d[3].item() == count
        assert got[3].data_ptr() == d[0].data_ptr() and got[4].data_ptr() == d[3].data_ptr()


@pytest.mark.parametrize("count,width,total", [(3, 8, 90), (0, 8, 90), (30, 2, 90), (30, 8, 40), (30, 0, 90)])
def test_plan_shortage(route, count, width, total):
    """Too few pages, too narrow a table, too few places: what fits is planned, the rest gets -1 and the status bit."""
    from uniql_b200 import ops
    lens, new = torch.tensor([0, 5, 16], dtype=torch.int32), torch.tensor([40, 30, 20], dtype=torch.int32)
    table = torch.full((3, width), -1, dtype=torch.int32)
    for i, n in enumerate((0, 1, 1)):
        table[i, :min(n, width)] = 100 + i
    free = torch.arange(30, dtype=torch.int32)
    want = ref.plan(lens, new, table, free, count, 16, total)
    assert want[6]
    d_table = table.cuda()
    got = ops.kv_page_plan(lens.cuda(), new.cuda(), d_table, free.cuda(), torch.tensor([count], dtype=torch.int32).cuda(), 16, total)
    assert torch.equal(d_table.cpu(), want[0]) and got[0].tolist() == want[1] and got[4].tolist() == [want[5]]
    assert got[2].tolist() == want[3] and got[3].tolist() == want[4]
    assert ops.read_and_clear_status("cuda") == 8


# ------------------------------------------------------------------------------------------------ append, gather
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,heads,dk,dv,page", [(1, 1, 128, 128, 16), (5, 3, 112, 112, 32), (33, 8, 128, 128, 64), (7, 2, 64, 64, 16),
                                                     (9, 5, 40, 64, 128), (50, 2, 128, 56, 256), (2, 1, 8, 8, 16)])
def test_append_is_bit_exact(route, dtype, tokens, heads, dk, dv, page):
    from uniql_b200 import ops
    g = _gen(tokens + dk)
    k, v = _rows(g, tokens, heads, dk, dtype), _rows(g, tokens, heads, dv, dtype)
    k[..., ::7] *= 8
    k[0, 0] = 3.25                                                # a constant row
    v[-1, -1] = torch.arange(dv).to(dtype) % 31                   # quotients on half-way points
    v[0, 0, 0], v[0, 0, -1] = 1e-7, -60000.0
    codes, scales = ops.kv4_cache(6, heads, page, max(dk, dv), device="cpu")
    codes += 0x11111111
    slots = torch.randperm(6 * page, generator=g)[:tokens]
    if tokens > 2:
        slots[1] = -1                                             # padding
    want_c, want_s = codes.clone(), scales.clone()
    ref.append(k, v, slots, want_c, want_s)
    codes, scales = codes.cuda(), scales.cuda()
    ops.kv4_append(k.cuda(), v.cuda(), slots.cuda(), codes, scales)
    assert torch.equal(codes.cpu(), want_c)
    assert torch.equal(scales.cpu().view(torch.int16), want_s.view(torch.int16))
    assert ops.read_and_clear_status("cuda") == 0


def test_append_ties_of_every_step():
    """Rows whose quotients are every k + 1/2, one fp16 step to either side of it, and the ends."""
    from uniql_b200 import ops
    rows = []
    for base, step in ((0.0, 1.0), (-7.5, 1.0), (0.0, 2.0 ** -20), (1000.0, 2.0), (-0.001, 0.0371)):
        hi = base + 15 * step
        x = torch.tensor([base, hi] + [base + (i + 0.5) * step for i in range(15)], dtype=F16)
        near = torch.cat([torch.nextafter(x[2:].float(), torch.tensor(1e9)).half(), torch.nextafter(x[2:], torch.tensor(1e9, dtype=F16)),
                          torch.nextafter(x[2:], torch.tensor(-1e4, dtype=F16))])
        row = torch.cat((x, near.clamp(min(base, hi), max(base, hi))))
        rows.append(torch.nn.functional.pad(row, (0, 64 - row.numel()), value=float(x[0]))[:64])
    k = torch.stack(rows)[:, None]
    codes, scales = ops.kv4_cache(1, 1, 16, 64)
    slots = torch.arange(len(rows))
    ops.kv4_append(k.cuda(), k.flip(-1).cuda(), slots.cuda(), codes, scales)
    want = [t.cpu().clone() for t in ops.kv4_cache(1, 1, 16, 64, device="cpu")]
    ref.append(k, k.flip(-1), slots, *want)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu().view(torch.int16), want[1].view(torch.int16))


def test_append_special_values(route):
    from uniql_b200 import ops
    k = torch.randn(6, 1, 128, generator=_gen(1)).to(BF16)
    k[0, 0, 5] = math.inf
    k[1, 0, 6] = -math.inf
    k[2, 0, 7] = math.nan
    k[3] = 1e30
    k[4, 0, 9] = -1e30
    k[5] = 0.0
    codes, scales = ops.kv4_cache(1, 1, 16, 128)
    ops.kv4_append(k.cuda(), k.cuda(), torch.arange(6).cuda(), codes, scales)
    want = ops.kv4_cache(1, 1, 16, 128, device="cpu")
    ref.append(k, k, torch.arange(6), *want)
    assert torch.equal(codes.cpu(), want[0])
    assert torch.equal(scales.cpu().isnan(), want[1].isnan())
    assert torch.equal(scales.cpu().nan_to_num(), want[1].nan_to_num())
    back, _ = ops.kv4_gather(codes, scales, torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.tensor([0, 6], dtype=torch.int32).cuda(), 6, 128)
    assert back[2].isnan().all() and not back[[0, 1, 3, 4, 5]].isnan().any()
    assert (back[3] == 65504).all() and (back[5] == 0).all()


def test_append_takes_views_and_skips_bad_slots(route):
    from uniql_b200 import ops
    g = _gen(5)
    fused = torch.randn(11, 6 * 128, generator=g).half()          # heads 2 q, 2 k, 2 v side by side
    d = fused.cuda()
    k, v = (d[:, o * 128:(o + 2) * 128].view(11, 2, 128) for o in (2, 4))
    odd = torch.randn(11, 2, 131, generator=g).half().cuda()[..., 3:]          # rows that are not 16-byte aligned
    turned = torch.randn(2, 11, 128, generator=g).half().cuda().transpose(0, 1)
    slots = torch.arange(11) * 3
    slots[4], slots[5], slots[6] = 48, 2 ** 40, -7                # behind the cache, far behind it, negative
    slots[3] = -1
    for a, b in ((k, v), (odd, v), (turned, odd)):
        codes, scales = ops.kv4_cache(3, 2, 16, 128)
        want = ops.kv4_cache(3, 2, 16, 128, device="cpu")
        ref.append(a.cpu(), b.cpu(), slots, *want)
        ops.kv4_append(a, b, slots.cuda(), codes, scales)
        assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu().view(torch.int16), want[1].view(torch.int16))
        assert ops.read_and_clear_status("cuda") == 4


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,heads,dk,dv,page", [([1], 1, 128, 128, 16), ([0, 33, 1], 3, 112, 112, 32), ([200, 0, 0, 65, 129], 8, 128, 128, 64),
                                                   ([17, 16, 15], 2, 64, 64, 16), ([40], 1, 72, 128, 256), ([0, 0], 2, 8, 24, 16)])
def test_gather(route, dtype, lens, heads, dk, dv, page):
    """fp16 values are zero + scale * code rounded once; bf16 passes through fp32: half a step and the fp32 rounding."""
    from uniql_b200 import ops
    g = _gen(sum(lens) + dk)
    codes, scales, table = _filled(g, lens, page, heads, dk, dv)
    total = sum(lens) + 5
    got = ops.kv4_gather(codes.cuda(), scales.cuda(), table.cuda(), _cu(lens).cuda(), total, dk, dv, dtype=dtype)
    for i, (d, x) in enumerate(((dk, got[0]), (dv, got[1]))):
        assert x.shape == (total, heads, d) and x.dtype == dtype
        want = torch.cat([ref.cached(codes, scales, table[r], i, d, n)[0] for r, n in enumerate(lens)])
        x = x.cpu()
        assert (x[sum(lens):] == 0).all()
        if dtype == F16:
            assert torch.equal(x[:sum(lens)], want.to(F16))       # fp64 to fp16 through fp32: 11 + 4 + 11 bits at most matter
        else:
            assert ((x[:sum(lens)].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -23) + 1e-38).all()
    assert ops.read_and_clear_status("cuda") == 0


def test_gather_ranges_and_bad_pages(route):
    from uniql_b200 import ops
    g = _gen(8)
    lens, page = [100, 40, 70], 16
    codes, scales, table = _filled(g, lens, page, 2, 128, 64)
    table[1, 1] = 10 ** 6                                         # outside the cache
    table[2, 0] = -1
    starts, counts = [37, 0, 64], [63, 40, 6]
    args = (codes.cuda(), scales.cuda(), table.cuda(), _cu(counts).cuda(), sum(counts), 128, 64)
    k, v = ops.kv4_gather(*args, starts=torch.tensor(starts, dtype=torch.int32).cuda())
    for i, (d, x) in enumerate(((128, k), (64, v))):
        want = torch.cat([ref.cached(codes, scales, table[r], i, d, n)[0][s:s + c] for r, (n, s, c) in enumerate(zip(lens, starts, counts))])
        assert torch.equal(x.cpu(), want.to(F16))
    assert ops.read_and_clear_status("cuda") == 4
    # a range that leaves the table reads as zeros
    k, _ = ops.kv4_gather(*args, starts=torch.tensor([2 ** 31 - 1, 0, 64], dtype=torch.int32).cuda())
    assert (k[:63] == 0).all() and ops.read_and_clear_status("cuda") == 4


# ------------------------------------------------------------------------------------------------ decode
def _decode_check(got, q, codes, scales, table, lens, dk, dv, scale):
    """Bound per value: the rounded result (half a step), the rounded weights (2^-11 of every term next to centred codes, 2^-25 each
    below fp16's normal range; a weight never sums below 1 over the largest scale), and scores off by fp32 sums of dk + 16 terms."""
    for b, n in enumerate(lens):
        k, _, there = ref.cached(codes, scales, table[b], 0, dk, n)
        v, step, _ = ref.cached(codes, scales, table[b], 1, dv, n)
        out, p, size, _ = ref.attend(q[b:b + 1].double(), k, v, there[None], scale)
        if not there.any():
            assert (got[b] == 0).all()
            continue
        g = q.shape[1] // codes.shape[2]
        # |code - 8| * scale <= 8 scale, per token and head
        spread = torch.einsum("hn,nh->h", p[0], (8 * step).repeat_interleave(g, 1))[:, None]
        tiny = n * 2.0 ** -22 * step.max()
        mass = torch.einsum("hn,nhd->hd", p[0], v.abs().repeat_interleave(g, 1)) + spread
        off = 2 * ((dk + 16) * 2.0 ** -23 * (size[0] + 1.0))[:, None] + 2.0 ** -18
        tol = out[0].abs() * ref.half_step(got.dtype) + 2.0 ** -11 * spread + tiny + off * mass + 1e-7
        assert ((got[b].double() - out[0]).abs() <= tol).all(), (b, n, ((got[b].double() - out[0]).abs() / tol).max())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,heads,kv,dk,dv,page", [
    ([1], 1, 1, 128, 128, 16), ([16], 8, 8, 128, 128, 16), ([15, 17], 4, 1, 64, 64, 16), ([0], 4, 2, 128, 128, 16), ([64, 65, 63], 32, 8, 128, 128, 64),
    ([1000, 0, 1, 333], 28, 4, 128, 128, 32), ([777], 16, 1, 112, 112, 64), ([300, 129], 24, 2, 128, 72, 128), ([50, 2100], 40, 2, 64, 40, 256),
    ([90] * 70, 8, 2, 64, 64, 16), ([5000], 32, 8, 128, 128, 64), ([130, 70], 33, 1, 128, 128, 16), ([0, 0, 4, 0], 6, 3, 8, 8, 16)])
def test_decode(route, dtype, lens, heads, kv, dk, dv, page):
    from uniql_b200 import ops
    g = _gen(sum(lens) + heads)
    codes, scales, table = _filled(g, lens, page, kv, dk, dv, dtype)
    q = _rows(g, len(lens), heads, dk, dtype)
    got = ops.kv4_attention(q.cuda(), codes.cuda(), scales.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), head_dim_v=dv)
    assert got.shape == (len(lens), heads, dv) and got.dtype == dtype
    _decode_check(got.cpu(), q, codes, scales, table, lens, dk, dv, 1 / math.sqrt(dk))
    assert ops.read_and_clear_status("cuda") == 0


@pytest.mark.parametrize("qs,vs,scale", [(30.0, 1.0, None), (1e-6, 1e-3, None), (1.0, 1e3, 2.5), (300.0, 0.01, 0.02)])
def test_decode_magnitudes(qs, vs, scale):
    """Sharp and flat softmax, small and large values: scales of the values from 1e-4 to 1e3."""
    from uniql_b200 import ops
    g = _gen(9)
    lens = [700, 64, 3]
    codes, scales, table = _filled(g, lens, 32, 2, 128, 128, F16, vs)
    q = _rows(g, 3, 8, 128, F16, qs)
    got = ops.kv4_attention(q.cuda(), codes.cuda(), scales.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), softmax_scale=scale)
    _decode_check(got.cpu(), q, codes, scales, table, lens, 128, 128, scale or 1 / math.sqrt(128))


def test_decode_is_deterministic_and_independent_of_the_batch():
    """The same request alone, twice, and beside others of other lengths: split differently, within two roundings of fp16."""
    from uniql_b200 import ops
    g = _gen(10)
    lens = [4000, 129, 900]
    codes, scales, table = (t.cuda() for t in _filled(g, lens, 64, 8, 128, 128))
    q = _rows(g, 3, 32, 128, F16).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    first = ops.kv4_attention(q, codes, scales, table, n)
    for _ in range(3):
        assert torch.equal(first, ops.kv4_attention(q, codes, scales, table, n))
    for i in range(3):
        alone = ops.kv4_attention(q[i:i + 1], codes, scales, table[i:i + 1], n[i:i + 1])
        # both within 2^-11 (result) + 2^-11 * spread (weights) of the same value; outputs here are below 1
        assert (alone - first[i]).abs().max() < 2 * (2 ** -11 + 2 ** -11 * 4)


@pytest.mark.parametrize("lens,kv", [
    ([128] * 32, 1), ([129] * 33, 1), ([0] * 31 + [257], 2), ([0] * 32 + [257], 2), ([256, 255, 1, 0, 1536, 1537], 1), ([1535] * 9, 6),
    ([384 * 12 + 1], 8), ([768 * 24], 4), ([768 * 24 + 1, 5], 4), ([32 * 4 * 12 + 1, 256], 3), ([1] * 131, 4), ([2000, 0, 33] * 43, 1)])
def test_decode_cuts(lens, kv):
    """Where the way that lists are cut changes: parts of every size, the longest lists that get them, batches of 32 and 33."""
    from uniql_b200 import ops
    g = _gen(len(lens) * 7 + kv)
    codes, scales, table = _filled(g, lens, 64, kv, 64, 64)
    q = _rows(g, len(lens), 2 * kv, 64, F16)
    args = q.cuda(), codes.cuda(), scales.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    got = ops.kv4_attention(*args)
    _decode_check(got.cpu(), q, codes, scales, table, lens, 64, 64, 1 / 8)
    assert torch.equal(got, ops.kv4_attention(*args))


def test_decode_bad_pages_and_lengths(route):
    """Pages outside the cache are absent tokens; lengths beyond the table and below zero are cut."""
    from uniql_b200 import ops
    g = _gen(11)
    lens, page = [100, 48, 30, 20], 16
    codes, scales, table = _filled(g, lens, page, 2, 128, 128)
    q = _rows(g, 4, 8, 128, F16)
    table[0, 2], table[0, 6] = -1, 2 ** 30
    table[2, :] = -5                                              # nothing of this request is left
    asked = [10 ** 9, 48, 30, -4]
    got = ops.kv4_attention(q.cuda(), codes.cuda(), scales.cuda(), table.cuda(), torch.tensor(asked, dtype=torch.int32).cuda()).cpu()
    assert ops.read_and_clear_status("cuda") == 4
    cut = [table.shape[1] * page, 48, 30, 0]
    _decode_check(got, q, codes, scales, table, cut, 128, 128, 1 / math.sqrt(128))
    assert (got[2:] == 0).all()


def test_decode_strided_queries_and_tables(route):
    from uniql_b200 import ops
    g = _gen(12)
    lens = [70, 200]
    codes, scales, table = _filled(g, lens, 16, 2, 128, 128)
    wide = torch.full((2, table.shape[1] + 9), 7, dtype=torch.int32)
    wide[:, 4:4 + table.shape[1]] = table
    fused = torch.randn(2, 12 * 128 + 5, generator=g).half()
    q = fused[:, 5:5 + 8 * 128].view(2, 8, 128)
    d_q = fused.cuda()[:, 5:5 + 8 * 128].view(2, 8, 128)
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    got = ops.kv4_attention(d_q, codes.cuda(), scales.cuda(), wide.cuda()[:, 4:4 + table.shape[1]], n)
    _decode_check(got.cpu(), q, codes, scales, table, lens, 128, 128, 1 / math.sqrt(128))
    turned = q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    assert torch.equal(ops.kv4_attention(turned, codes.cuda(), scales.cuda(), table.cuda(), n), got)
    apart = torch.randn(2, 8, 256, generator=g).half().cuda()
    apart[..., ::2] = d_q
    assert torch.equal(ops.kv4_attention(apart[..., ::2], codes.cuda(), scales.cuda(), table.cuda(), n), got)


# ------------------------------------------------------------------------------------------------ prompt
def _prompt_check(got, q, k, v, nq, nk, causal, scale):
    """Bound per value: the rounded result, P rounded to the type (each term; in fp16 2^-25 each below its normal range), and
    scores off by fp32 sums of dk terms."""
    cq, ck = _cu(nq).tolist(), _cu(nk).tolist()
    step = ref.half_step(got.dtype)
    for r in range(len(nq)):
        a, b = slice(cq[r], cq[r + 1]), slice(ck[r], ck[r + 1])
        i, j = torch.arange(nq[r])[:, None], torch.arange(nk[r])[None]
        seen = (j <= i + nk[r] - nq[r]) if causal else torch.ones(nq[r], nk[r], dtype=torch.bool)
        out, p, size, vv = ref.attend(q[a].double(), k[b].double(), v[b].double(), seen, scale)
        mass = torch.einsum("mhn,nhd->mhd", p, vv.abs())
        off = 2 * ((q.shape[2] + 8) * 2.0 ** -23 * (size + 1.0))[..., None] + 2.0 ** -20
        tiny = nk[r] * 2.0 ** -25 * (vv.abs().max() if vv.numel() else 0.0)
        tol = out.abs() * step + mass * (step + off) + tiny + 1e-7
        bad = (got[a].double() - out).abs() / tol
        assert not bad.numel() or bad.max() <= 1, (r, bad.max())
    assert (got[cq[-1]:] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq,nk,heads,kv,dk,dv,causal", [
    ([1], [1], 1, 1, 128, 128, True), ([1], [300], 4, 2, 128, 128, True), ([77], [77], 28, 4, 128, 128, True), ([128], [128], 2, 1, 64, 64, True),
    ([129], [129], 2, 2, 128, 128, True), ([256, 255, 257], [256, 255, 257], 4, 1, 128, 128, True), ([300, 1, 0, 40], [300, 1, 0, 700], 6, 2, 112, 112, True),
    ([5, 130, 64], [133, 130, 1000], 7, 1, 64, 64, True), ([200, 90], [70, 90], 4, 4, 128, 128, True), ([50, 300], [0, 129], 3, 1, 128, 64, True),
    ([100, 33], [257, 20], 4, 2, 128, 128, False), ([700], [700], 2, 1, 72, 40, True), ([17, 18], [17, 18], 5, 5, 8, 16, True),
    ([1] * 40, [1 + 9 * i for i in range(40)], 8, 2, 128, 128, True), ([1100], [1500], 3, 1, 128, 128, True)])
def test_prompt(route, dtype, nq, nk, heads, kv, dk, dv, causal):
    from uniql_b200 import ops
    g = _gen(sum(nq) + sum(nk) + heads)
    q, k, v = _rows(g, sum(nq) + 3, heads, dk, dtype), _rows(g, sum(nk) + 2, kv, dk, dtype), _rows(g, sum(nk) + 2, kv, dv, dtype)
    got = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), _cu(nq).cuda(), _cu(nk).cuda(), causal=causal)
    assert got.shape == (sum(nq) + 3, heads, dv) and got.dtype == dtype
    _prompt_check(got.cpu(), q, k, v, nq, nk, causal, 1 / math.sqrt(dk))
    assert ops.read_and_clear_status("cuda") == 0


@pytest.mark.parametrize("qs,scale", [(40.0, None), (1e-4, None), (1.0, 3.0)])
def test_prompt_magnitudes(qs, scale):
    from uniql_b200 import ops
    g = _gen(20)
    n = [500, 90]
    q, k, v = _rows(g, 590, 4, 128, F16, qs), _rows(g, 590, 2, 128, F16), _rows(g, 590, 2, 128, F16, 100.0)
    k[300:] *= 5                                                  # the bound of a row's scores rises late
    got = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), _cu(n).cuda(), softmax_scale=scale)
    _prompt_check(got.cpu(), q, k, v, n, n, True, scale or 1 / math.sqrt(128))


def test_prompt_requests_do_not_see_each_other():
    """Infinities and NaN in other requests' rows, and in keys that the mask hides, change nothing."""
    from uniql_b200 import ops
    g = _gen(21)
    n = [100, 60, 300, 7]
    q, k, v = _rows(g, 467, 4, 128, F16), _rows(g, 467, 2, 128, F16), _rows(g, 467, 2, 128, F16)
    cu = _cu(n).cuda()
    clean = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu)
    for value in (math.inf, math.nan, -math.inf, 65504.0):
        for r in range(4):
            a = slice(int(cu[r]), int(cu[r + 1]))
            q2, k2, v2 = q.clone(), k.clone(), v.clone()
            q2[a], k2[a], v2[a] = value, value, value
            got = ops.prompt_attention(q2.cuda(), k2.cuda(), v2.cuda(), cu)
            keep = torch.ones(467, dtype=torch.bool)
            keep[a] = False
            assert torch.equal(got[keep], clean[keep])
    k2 = k.clone()
    k2[399] = math.nan                                            # a future key of the third request
    got = ops.prompt_attention(q.cuda(), k2.cuda(), v.cuda(), cu)
    keep = torch.arange(467) != 399
    keep[400:460] = False
    assert torch.equal(got[:399], clean[:399]) and got[399:460].isnan().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq,nk,heads,kv,dk,dv,causal", [
    ([300, 1, 0, 40], [300, 1, 0, 700], 42, 6, 64, 64, True), ([5, 130, 64], [133, 130, 1000], 49, 7, 64, 40, True), ([148], [148], 75, 75, 64, 64, True),
    ([129], [400], 75, 25, 128, 112, False), ([200, 90], [70, 90], 40, 8, 128, 128, True)])
def test_prompt_two_units_an_item(route, dtype, nq, nk, heads, kv, dk, dv, causal):
    """More row blocks and heads than the GPU has SMs."""
    test_prompt(route, dtype, nq, nk, heads, kv, dk, dv, causal)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq,nk,heads,kv,dk,dv,causal", [
    ([1] * 9, [3] * 9, 128, 1, 64, 64, True), ([2, 0, 5], [200, 7, 5], 130, 1, 64, 64, True), ([3, 1], [3, 129], 65, 1, 128, 128, True),
    ([18, 19, 17, 1], [18, 190, 17, 0], 14, 2, 128, 128, True), ([43, 42], [43, 300], 9, 3, 128, 72, True), ([1] * 150, [1] * 150, 10, 2, 64, 64, True),
    ([33] * 20, [40] * 20, 64, 16, 112, 112, False), ([64, 65, 63], [64, 65, 200], 4, 2, 128, 128, True)])
def test_prompt_short_requests(route, dtype, nq, nk, heads, kv, dk, dv, causal):
    """A group's heads share a row block: groups that divide it, that do not, that fill it and that are larger."""
    test_prompt(route, dtype, nq, nk, heads, kv, dk, dv, causal)


@pytest.mark.parametrize("heads", [4, 80])
def test_prompt_padding(heads):
    """Rows behind the last request: NaN there reaches nothing, and their results are zeros."""
    from uniql_b200 import ops
    g = _gen(23)
    n = [100, 61]
    q, k, v = (_rows(g, 200, h, 64, F16) for h in (heads, heads // 2, heads // 2))
    cu = _cu(n).cuda()
    clean = ops.prompt_attention(q[:161].cuda(), k[:161].cuda(), v[:161].cuda(), cu)
    _prompt_check(clean.cpu(), q[:161], k[:161], v[:161], n, n, True, 1 / 8)
    for t in (q, k, v):
        t[161:] = math.nan
    got = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu)
    assert torch.equal(got[:161], clean) and (got[161:] == 0).all()


def test_prompt_views(route):
    from uniql_b200 import ops
    g = _gen(22)
    fused = torch.randn(150, (8 + 2 + 2) * 128, generator=g).half()
    parts = [fused[:, a * 128:b * 128].view(150, b - a, 128) for a, b in ((0, 8), (8, 10), (10, 12))]
    d = fused.cuda()
    views = [d[:, a * 128:b * 128].view(150, b - a, 128) for a, b in ((0, 8), (8, 10), (10, 12))]
    cu = _cu([150]).cuda()
    got = ops.prompt_attention(*views, cu)
    _prompt_check(got.cpu(), *parts, [150], [150], True, 1 / math.sqrt(128))
    odd = torch.zeros(150, 8, 131, dtype=F16, device="cuda")[..., 3:]
    odd.copy_(views[0])
    assert torch.equal(ops.prompt_attention(odd, views[1].transpose(0, 1).contiguous().transpose(0, 1), views[2].contiguous(), cu), got)


def test_empty_calls(route):
    from uniql_b200 import ops
    z = lambda *s, t=F16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    codes, scales = ops.kv4_cache(2, 2, 16, 128)
    i32 = torch.int32
    ops.kv4_append(z(0, 2, 128), z(0, 2, 128), z(0, t=torch.int64), codes, scales)
    k, v = ops.kv4_gather(codes, scales, z(0, 1, t=i32), z(1, t=i32), 0, 128)
    assert k.shape == (0, 2, 128)
    k, v = ops.kv4_gather(codes, scales, z(0, 1, t=i32), z(1, t=i32), 3, 128)
    assert (k == 0).all() and (v == 0).all()
    assert ops.kv4_attention(z(0, 4, 128), codes, scales, z(0, 1, t=i32), z(0, t=i32)).shape == (0, 4, 128)
    assert (ops.kv4_attention(z(2, 4, 128), codes, scales, z(2, 0, t=i32), torch.ones(2, dtype=i32, device="cuda")) == 0).all()
    assert ops.prompt_attention(z(0, 4, 128), z(0, 2, 128), z(0, 2, 128), z(1, t=i32)).shape == (0, 4, 128)
    assert (ops.prompt_attention(z(5, 4, 128) + 1, z(0, 2, 128), z(0, 2, 128), torch.tensor([0, 5], dtype=i32, device="cuda"), z(2, t=i32)) == 0).all()
    assert (ops.prompt_attention(z(5, 4, 128) + 1, z(0, 2, 128), z(0, 2, 128), z(1, t=i32)) == 0).all()
    out = ops.kv_page_plan(z(0, t=i32), z(0, t=i32), z(0, 4, t=i32), z(0, t=i32), z(1, t=i32), 16, 2)
    assert out[0].tolist() == [-1, -1] and out[2].tolist() == [0]
    assert (ops.kv4_attention(z(2, 4, 128), codes[:0], scales[:0], z(2, 3, t=i32), torch.full((2,), 40, dtype=i32, device="cuda")) == 0).all()
    assert ops.read_and_clear_status("cuda") == 4
    assert ops.read_and_clear_status("cuda") == 0
