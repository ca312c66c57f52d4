"""CPU: argument checks of the KV cache and attention entry points, which come before any CUDA call, and the reference itself."""
import math

import pytest
import torch

import kv_reference as ref

P = 1 << 20                                                       # stands for a pointer: 16- and 256-byte aligned, never read


def _lib():
    from uniql_b200._lib import lib
    return lib()


def _plan(**kw):
    a = dict(lens=P, new=P, batch=4, table=P, ld=8, width=8, free=P, cap=9, count=P, page=16, total=5, slots=P, pos=P, cu=P, lens_out=P, count_out=P)
    a.update(kw)
    return _lib().uniql_kv_page_plan(a["lens"], a["new"], a["batch"], a["table"], a["ld"], a["width"], a["free"], a["cap"], a["count"],
                                     a["page"], a["total"], a["slots"], a["pos"], a["cu"], a["lens_out"], a["count_out"], None, None)


def _append(**kw):
    a = dict(k=P, kt=256, kh=128, v=P, vt=256, vh=128, dtype=0, tokens=3, heads=2, dk=128, dv=128, slots=P, codes=P, scales=P, pages=4, page=16, dp=128)
    a.update(kw)
    return _lib().uniql_kv4_append(*a.values(), None, None)


def _gather(**kw):
    a = dict(codes=P, scales=P, pages=4, page=16, dp=128, heads=2, table=P, ld=8, width=8, batch=2, starts=None, cu=P, total=3, dk=128, dv=128, dtype=0,
             k=P, v=P)
    a.update(kw)
    return _lib().uniql_kv4_gather(*a.values(), None, None)


def _decode(**kw):
    a = dict(q=P, qb=1024, qh=128, codes=P, scales=P, pages=4, page=16, dp=128, table=P, ld=8, width=8, lens=P, batch=2, heads=8, kv=2, dk=128,
             dv=128, scale=0.1, dtype=0, out=P, scratch=P, bytes=1 << 40)
    a.update(kw)
    return _lib().uniql_kv4_attention(*a.values(), None, None)


def _prompt(**kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, cu_q=P, cu_k=P, batch=2, total_q=9, total_k=9, heads=8, kv=2, dk=128,
             dv=128, scale=0.1, causal=1, dtype=0, out=P)
    a.update(kw)
    return _lib().uniql_prompt_attention(*a.values(), None, None)


EINVAL, ESHAPE, ESCRATCH, EDTYPE = -1, -3, -4, -6


@pytest.mark.parametrize("call,kw,code", [
    (_plan, dict(batch=-1), EINVAL), (_plan, dict(total=-1), EINVAL), (_plan, dict(ld=7), EINVAL), (_plan, dict(page=48), ESHAPE), (_plan, dict(page=8), ESHAPE),
    (_plan, dict(batch=16385), ESHAPE), (_plan, dict(lens=None), EINVAL), (_plan, dict(table=None), EINVAL), (_plan, dict(slots=None), EINVAL),
    (_plan, dict(cu=None), EINVAL), (_plan, dict(free=None), EINVAL), (_plan, dict(count=None), EINVAL), (_plan, dict(total=1 << 30), ESHAPE),
    (_append, dict(tokens=-1), EINVAL), (_append, dict(dtype=2), EDTYPE), (_append, dict(dk=130), ESHAPE), (_append, dict(dk=12), ESHAPE),
    (_append, dict(dv=136), ESHAPE), (_append, dict(dp=64), ESHAPE), (_append, dict(dp=96, dk=64, dv=64), ESHAPE), (_append, dict(page=20), ESHAPE),
    (_append, dict(kt=257), EINVAL), (_append, dict(vh=4), EINVAL), (_append, dict(k=P + 8), EINVAL), (_append, dict(slots=None), EINVAL),
    (_append, dict(codes=P + 4), EINVAL), (_append, dict(heads=0), EINVAL), (_append, dict(tokens=0), 0),
    (_gather, dict(total=-1), EINVAL), (_gather, dict(dtype=2), EDTYPE), (_gather, dict(page=512), ESHAPE), (_gather, dict(dk=0), EINVAL),
    (_gather, dict(dv=20), ESHAPE), (_gather, dict(cu=None), EINVAL), (_gather, dict(k=None), EINVAL), (_gather, dict(v=P + 2), EINVAL),
    (_gather, dict(ld=2), EINVAL), (_gather, dict(total=0), 0),
    (_decode, dict(batch=-1), EINVAL), (_decode, dict(heads=7), ESHAPE), (_decode, dict(dtype=2), EDTYPE), (_decode, dict(scale=math.nan), EINVAL),
    (_decode, dict(scale=0.0), EINVAL), (_decode, dict(scale=math.inf), EINVAL), (_decode, dict(scratch=None), ESCRATCH), (_decode, dict(scratch=P + 16), ESCRATCH),
    (_decode, dict(bytes=16384), ESCRATCH), (_decode, dict(dk=4), ESHAPE), (_decode, dict(q=None), EINVAL), (_decode, dict(lens=None), EINVAL),
    (_decode, dict(codes=None), EINVAL), (_decode, dict(batch=16385), ESHAPE), (_decode, dict(batch=0), 0),
    (_prompt, dict(total_q=-1), EINVAL), (_prompt, dict(heads=7), ESHAPE), (_prompt, dict(dk=136), ESHAPE), (_prompt, dict(dv=12), ESHAPE), (_prompt, dict(dtype=2), EDTYPE),
    (_prompt, dict(scale=-1.0), EINVAL), (_prompt, dict(qt=1023), EINVAL), (_prompt, dict(kh=-128), EINVAL), (_prompt, dict(q=P + 2), EINVAL),
    (_prompt, dict(k=None), EINVAL), (_prompt, dict(cu_k=None), EINVAL), (_prompt, dict(out=None), EINVAL), (_prompt, dict(batch=16385), ESHAPE), (_prompt, dict(total_k=(1 << 26) + 1), ESHAPE),
    (_prompt, dict(total_q=0), 0)])
def test_refusals(built_lib, call, kw, code):
    assert call(**kw) == code


def test_scratch_size(built_lib):
    f = _lib().uniql_kv4_attention_scratch_bytes
    assert f(1, 8, 3, 128) == 0 and f(0, 8, 2, 128) == 0 and f(1, 8, 2, 100) == 0
    assert f(1, 8, 2, 128) > 16384 and f(1, 32, 2, 128) > f(1, 32, 2, 64)


def test_ops_refuse_cpu_tensors():
    from uniql_b200 import ops
    i32 = torch.int32
    codes, scales = ops.kv4_cache(2, 2, 16, 128, device="cpu")
    x, n, t = torch.zeros(1, 2, 128).half(), torch.zeros(1, dtype=i32), torch.zeros(1, 1, dtype=i32)
    for call in (lambda: ops.kv_page_plan(n, n, t, n, n, 16, 1), lambda: ops.kv4_append(x, x, n.long(), codes, scales),
                 lambda: ops.kv4_gather(codes, scales, t, torch.zeros(2, dtype=i32), 1, 128), lambda: ops.kv4_attention(x, codes, scales, t, n),
                 lambda: ops.prompt_attention(x, x, x, torch.zeros(2, dtype=i32))):
        with pytest.raises(RuntimeError):
            call()
    for bad in (dict(page_size=24), dict(head_dim=132), dict(head_dim=0), dict(head_dim=12)):
        with pytest.raises(RuntimeError):
            ops.kv4_cache(**{**dict(num_pages=1, kv_heads=1, page_size=16, head_dim=64, device="cpu"), **bad})


def test_reference_quantiser_is_within_half_a_step():
    """The definition itself: values come back within half a step plus the roundings of scale and zero."""
    x = torch.randn(50, 3, 128, generator=torch.Generator().manual_seed(0)).half()
    code, scale, zero = ref.quantise(x)
    assert code.min() == 0 and code.max() == 15 and torch.equal(ref.unpack(ref.pack(code, 16), 128), code)
    back = zero.double()[..., None] + scale.double()[..., None] * code
    # 15 steps of a scale that is off by at most 2^-11 of itself
    assert ((back - x.double()).abs() <= scale.double()[..., None] * (0.5 + 15 * 2.0 ** -11)).all()


def test_cache_moves_and_releases_rows():
    from uniql_b200.kv_cache import PagedKV4Cache
    cache = PagedKV4Cache(1, 5, 1, 64, page_size=16, requests=3, max_tokens=64, device="cpu")
    cache.block_table[0, :2], cache.lens[0] = torch.tensor([4, 3], dtype=torch.int32), 20
    cache.block_table[2, :1], cache.lens[2] = torch.tensor([2], dtype=torch.int32), 7
    cache.free_count -= 3
    cache.move(2, 2)                                              # onto itself: nothing changes
    assert cache.block_table[2].tolist() == [2, -1, -1, -1] and cache.lens.tolist() == [20, 0, 7]
    cache.move(2, 1)
    assert cache.block_table[1].tolist() == [2, -1, -1, -1] and cache.lens.tolist() == [20, 7, 0] and (cache.block_table[2] == -1).all()
    cache.release([0, 0])                                         # the second time there is nothing to give back
    assert cache.free_count.item() == 4 and cache.free_pages[:4].tolist() == [4, 3, 4, 3] and cache.lens.tolist() == [0, 7, 0]
