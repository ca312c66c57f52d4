"""CPU: argument checks of a step's plan, which come before any CUDA call."""
import pytest
import torch

P = 1 << 20                                                       # stands for a pointer, never read
EINVAL, ESHAPE = -1, -3


@pytest.mark.parametrize("kw,code", [(dict(cu_keys=None), EINVAL), (dict(key_lens=None), EINVAL), (dict(batch=-1), EINVAL), (dict(page=24), ESHAPE),
                                     (dict(batch=16385), ESHAPE), (dict(ld=7), EINVAL), (dict(lens_out=None), EINVAL), (dict(cu=None), EINVAL)])
def test_refusals(built_lib, kw, code):
    from uniql_b200._lib import lib
    a = dict(lens=P, new=P, batch=4, table=P, ld=8, width=8, free=P, cap=9, count=P, page=16, total=5, slots=P, pos=P, cu=P, lens_out=P, count_out=P,
             key_lens=P, cu_keys=P)
    a.update(kw)
    assert lib().uniql_kv_step_plan(*a.values(), None, None) == code


def test_cache_refuses_too_many_requests_and_cpu_lengths():
    from uniql_b200.kv_cache import PagedKV4Cache
    cache = PagedKV4Cache(1, 5, 1, 64, page_size=16, requests=2, max_tokens=64, device="cpu")
    for n in (3, 1):
        with pytest.raises(RuntimeError):
            cache.plan(torch.ones(n, dtype=torch.int32), n)


@pytest.mark.parametrize("n", [3, -1])
def test_decode_steps_of_requests_that_are_not_there(n):
    """Refused before anything moves: the slice of one-token lengths would quietly be shorter than n."""
    from uniql_b200.kv_cache import PagedKV4Cache
    cache = PagedKV4Cache(1, 5, 1, 64, page_size=16, requests=2, max_tokens=64, device="cpu")
    with pytest.raises(RuntimeError, match="room for 2"):
        cache.plan_decode(n)
