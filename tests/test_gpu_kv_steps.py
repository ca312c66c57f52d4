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
