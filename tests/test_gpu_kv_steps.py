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
