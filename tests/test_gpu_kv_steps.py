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
