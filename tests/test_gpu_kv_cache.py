"""GPU: the cache class and the operators as a decoder block uses them: prompts, chunks, decode steps, graphs, streams."""
import math

import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class _Plain:
    """The cache kept as plain lists of quantised rows per request, in 64 bits."""

    def __init__(self, requests):
        self.k = [torch.zeros(0) for _ in range(requests)]
        self.v = [torch.zeros(0) for _ in range(requests)]

    def add(self, r, k, v):
        for rows, x in ((self.k, k), (self.v, v)):
            c, s, z = ref.quantise(x)
            y = z.double()[..., None] + s.double()[..., None] * c
            rows[r] = y if rows[r].numel() == 0 else torch.cat((rows[r], y))


def _near(got, want, mass):
    """Result and weights rounded to fp16 (2^-11 each, the latter of what the values and their codes' spread weigh), scores in 32
    bits: 2^-10 of `mass`, and the cached rows once more where they were gathered to fp16."""
    assert ((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -10 * mass + 1e-6).all()


@pytest.mark.parametrize("dk,dv,heads,kv,page", [(128, 128, 8, 2, 64), (112, 112, 4, 4, 16), (64, 40, 6, 1, 32)])
def test_prompts_chunks_and_decode(dk, dv, heads, kv, page):
    """Fresh prompts, a second chunk behind them, then decode steps; a request ends and another takes its pages."""
    from uniql_b200 import ops
    from uniql_b200.kv_cache import PagedKV4Cache
    g = _gen(dk)
    cache = PagedKV4Cache(2, 120, kv, dk, dv, page_size=page, requests=4, max_tokens=40 * page)
    plain = [_Plain(4), _Plain(4)]
    ops.read_and_clear_status("cuda")

    def run(new, step, pad, check=True):
        total = sum(new) + pad
        for layer in range(2):
            q, k, v = (torch.randn(total, h, d, generator=g).to(F16) for h, d in ((heads, dk), (kv, dk), (kv, dv)))
            d_q, d_k, d_v = q.cuda(), k.cuda(), v.cuda()
            cache.append(layer, d_k, d_v, step)
            got = cache.attend(layer, d_q, d_k, d_v, step).cpu()
            at = 0
            for r, n in enumerate(new):
                plain[layer].add(r, k[at:at + n], v[at:at + n])
                keys, vals = (k[at:at + n].double(), v[at:at + n].double()) if step.fresh else (plain[layer].k[r], plain[layer].v[r])
                seen = torch.arange(keys.shape[0])[None] <= torch.arange(n)[:, None] + keys.shape[0] - n
                want, p, _, vv = ref.attend(q[at:at + n].double(), keys, vals, seen, 1 / math.sqrt(dk))
                mass = torch.einsum("mhn,nhd->mhd", p, vv.abs()).amax(-1, keepdim=True) + 4.0
                if check:
                    _near(got[at:at + n], want, mass)
                at += n
            if pad and not step.single:
                assert (got[at:] == 0).all()

    new = [70, 1, 150, 33]
    step = cache.plan(torch.tensor(new, dtype=torch.int32).cuda(), sum(new) + 2, fresh=True)
    run(new, step, 2)
    assert cache.lens.tolist() == new
    more = [10, 130, 0, 64]
    step = cache.plan(torch.tensor(more, dtype=torch.int32).cuda(), sum(more) + 1, max_keys=sum(new) + sum(more))
    run(more, step, 1)
    for _ in range(3):
        run([1] * 4, cache.plan_decode(4), 0)
    held = [a + b + 3 for a, b in zip(new, more)]
    assert cache.lens.tolist() == held
    used = sum(-(-n // page) for n in held)
    assert cache.free_count.item() == 120 - used and ops.read_and_clear_status("cuda") == 0
    cache.release([1])
    cache.move(3, 1)
    for p in plain:
        p.k[1], p.v[1] = p.k[3], p.v[3]
    assert cache.free_count.item() == 120 - used + -(-held[1] // page)
    run([1] * 3, cache.plan_decode(3), 0)
    # every page is either free or in the table, once
    pages = cache.free_pages[:cache.free_count.item()].tolist() + cache.block_table[cache.block_table >= 0].tolist()
    assert sorted(pages) == list(range(120))


def test_prompt_and_decode_agree():
    """A decode step's output is the last row of the prompt that holds the same tokens, up to the 4-bit rows: equal to the plain result
    over the same cached rows (checked above), and both paths read the same cache through gather."""
    from uniql_b200 import ops
    g = _gen(1)
    n, heads, kv, d, page = 333, 8, 2, 128, 32
    codes, scales = ops.kv4_cache(20, kv, page, d)
    table = torch.randperm(20, generator=g)[:12].int()[None].contiguous().cuda()
    slots = torch.cat([table[0, t // page:t // page + 1].long() * page + t % page for t in range(n)])
    k, v, q = torch.randn(n, kv, d, generator=g).to(F16).cuda(), torch.randn(n, kv, d, generator=g).to(F16).cuda(), torch.randn(1, heads, d, generator=g).to(F16).cuda()
    ops.kv4_append(k, v, slots, codes, scales)
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    one = ops.kv4_attention(q, codes, scales, table, lens)
    cu = torch.tensor([0, n], dtype=torch.int32).cuda()
    kk, vv = ops.kv4_gather(codes, scales, table, cu, n, d)
    other = ops.prompt_attention(q, kk, vv, torch.tensor([0, 1], dtype=torch.int32).cuda(), cu)
    # two results within 2^-11 of themselves and of their weights' mass (below 1), and rows rounded to fp16 in one of them (2^-11)
    assert (one - other).abs().max() < 5 * 2.0 ** -11


def _layer(g, hidden, out, bias=False):
    from uniql_b200.quantize.quant_linear_layers import W4A16B16O16Linear
    lin = torch.nn.Linear(hidden, out, bias=bias).half()
    lin.weight.data = (torch.randn(out, hidden, generator=g) * 0.02).half()
    if bias:
        lin.bias.data = (torch.randn(out, generator=g) * 0.1).half()
    return W4A16B16O16Linear.from_fp16(lin.cuda()).cuda()


def _rotary(q, k, positions):
    d = q.shape[-1]
    ang = positions.double()[:, None] / 10000.0 ** (torch.arange(0, d, 2, device=q.device).double() / d)
    cos, sin = (torch.cat((f(ang), f(ang)), -1)[:, None].to(q.dtype) for f in (torch.cos, torch.sin))
    turn = lambda x: x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin  # noqa: E731
    return turn(q), turn(k)


def test_decoder_block_prompt_then_captured_decode_steps():
    """attention_block on a W4A16 block with rotary positions: a prompt step eagerly, decode steps as one captured graph that is replayed
    with new inputs, against the same steps run eagerly on a second cache."""
    from uniql_b200 import ops
    from uniql_b200.kv_cache import PagedKV4Cache, attention_block
    g = _gen(2)
    hidden, heads, kv, d, batch = 1024, 8, 2, 128, 3
    mods = [_layer(g, hidden, n * d, bias=True) for n in (heads, kv, kv)] + [_layer(g, heads * d, hidden)]
    caches = [PagedKV4Cache(1, 40, kv, d, page_size=16, requests=batch, max_tokens=160) for _ in range(2)]
    new = [20, 47, 5]
    x = torch.randn(sum(new), hidden, generator=g).half().cuda()
    outs = []
    for c in caches:
        step = c.plan(torch.tensor(new, dtype=torch.int32).cuda(), sum(new), fresh=True)
        outs.append(attention_block(*mods, x, x, c, 0, step, _rotary))
    assert torch.equal(*outs) and outs[0].isfinite().all()
    xs = [torch.randn(batch, hidden, generator=g).half().cuda() for _ in range(9)]
    want = [attention_block(*mods, y, y, caches[0], 0, caches[0].plan_decode(batch), _rotary) for y in xs[:1]]

    # warm up the second cache's path on a throw-away copy, then capture
    spare = PagedKV4Cache(1, 40, kv, d, page_size=16, requests=batch, max_tokens=160)
    static = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_block(*mods, static, static, spare, 0, spare.plan_decode(batch), _rotary)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention_block(*mods, static, static, caches[1], 0, caches[1].plan_decode(batch), _rotary)
    want += [attention_block(*mods, y, y, caches[0], 0, caches[0].plan_decode(batch), _rotary) for y in xs[1:]]
    for y, w in zip(xs, want):
        static.copy_(y)
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(caches[0].lens, caches[1].lens) and torch.equal(caches[0].block_table, caches[1].block_table)
    assert caches[1].lens.tolist() == [n + 9 for n in new]
    # the same codes: every row of both caches reads back alike
    cu = torch.tensor([0, 29, 29 + 56, 29 + 56 + 14], dtype=torch.int32).cuda()
    a, b = (ops.kv4_gather(c.codes[0], c.scales[0], c.block_table, cu, 99, d) for c in caches)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert ops.read_and_clear_status("cuda") == 0


def _decode_inputs(g, lens, page=64, heads=32, kv=8, d=128):
    from uniql_b200 import ops
    blocks = [-(-n // page) for n in lens]
    codes, scales = ops.kv4_cache(sum(blocks), kv, page, d)
    table = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
    order = torch.randperm(sum(blocks), generator=g).int()
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b]
        at += b
    table = table.cuda()
    n = sum(lens)
    req = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).cuda()
    t = torch.cat([torch.arange(m) for m in lens]).cuda()
    slots = table[req, t // page].long() * page + t % page
    ops.kv4_append(torch.randn(n, kv, d, generator=g).half().cuda(), torch.randn(n, kv, d, generator=g).half().cuda(), slots, codes, scales)
    return torch.randn(len(lens), heads, d, generator=g).half().cuda(), codes, scales, table, torch.tensor(lens, dtype=torch.int32).cuda()


@pytest.mark.parametrize("route", ["binding", "ctypes"])
def test_two_graphs_and_eager_calls_at_once(route, monkeypatch):
    """Two captured decode calls and eager ones run on three streams at the same time: each has scratch of its own."""
    from uniql_b200 import ops
    if route == "ctypes":
        monkeypatch.setattr(ops, "torch_ext", lambda: None)
    g = _gen(4)
    sets = [_decode_inputs(g, lens) for lens in ([3000, 900], [2500, 64, 1200], [5000])]
    want = [ops.kv4_attention(*s) for s in sets]
    graphs, outs = [], []
    for s in sets[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([ops.kv4_attention(*s) for _ in range(3)])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    eager = []
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager.append(ops.kv4_attention(*sets[2]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for row, w in zip(outs, want) for o in row) and all(torch.equal(o, want[2]) for o in eager)


def test_calls_follow_each_other_on_one_stream():
    """Plan, append, decode, gather and prompt back to back, each reading what the one in front wrote, many times without a wait
    between (the launches overlap their predecessors' ends), give what they give with a wait behind each."""
    from uniql_b200 import ops
    from uniql_b200.kv_cache import PagedKV4Cache
    g = _gen(5)
    kv, heads, d, rows = 4, 8, 128, 6
    ks = [torch.randn(rows, kv, d, generator=g).half().cuda() for _ in range(2 * 40)]
    qs = [torch.randn(rows, heads, d, generator=g).half().cuda() for _ in range(40)]

    def go(wait):
        cache = PagedKV4Cache(1, 60, kv, d, page_size=16, requests=rows, max_tokens=80)
        outs = []
        for i in range(40):
            step = cache.plan_decode(rows)
            if wait:
                torch.cuda.synchronize()
            cache.append(0, ks[2 * i], ks[2 * i + 1], step)
            if wait:
                torch.cuda.synchronize()
            outs.append(cache.attend(0, qs[i], None, None, step))
            if wait:
                torch.cuda.synchronize()
            outs.append(cache.attend(0, qs[i], None, None, step._replace(single=False, cu=torch.arange(rows + 1, dtype=torch.int32, device="cuda"))))
        return outs

    assert all(torch.equal(a, b) for a, b in zip(go(False), go(True)))
    assert ops.read_and_clear_status("cuda") == 0


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device_than_the_current_one():
    from uniql_b200 import ops
    sets = _decode_inputs(_gen(6), [300, 20])
    want = ops.kv4_attention(*sets)
    moved = [t.to("cuda:1") for t in sets]
    assert torch.equal(ops.kv4_attention(*moved).cpu(), want.cpu())


def test_long_cache_offsets_pass_32_bits():
    """A cache of more than 4 GB: rows at its end are found."""
    from uniql_b200 import ops
    pages, kv, page, d = 140000, 8, 64, 128                       # 140000 * 2 * 8 * 64 * 64 bytes = 9.2 GB of codes
    codes, scales = ops.kv4_cache(pages, kv, page, d)
    g = _gen(7)
    n = 200
    last = torch.tensor([[pages - 1, 3, pages - 2, pages // 2]], dtype=torch.int32).cuda()
    slots = torch.cat([last[0, t // page:t // page + 1].long() * page + t % page for t in range(n)])
    k, v = torch.randn(n, kv, d, generator=g).half().cuda(), torch.randn(n, kv, d, generator=g).half().cuda()
    ops.kv4_append(k, v, slots, codes, scales)
    small = ops.kv4_cache(4, kv, page, d)
    near = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32).cuda()
    ops.kv4_append(k, v, torch.arange(n).cuda(), *small)
    q, lens, cu = torch.randn(1, 32, d, generator=g).half().cuda(), torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    assert torch.equal(ops.kv4_attention(q, codes, scales, last, lens), ops.kv4_attention(q, *small, near, lens))
    for a, b in zip(ops.kv4_gather(codes, scales, last, cu, n, d), ops.kv4_gather(*small, near, cu, n, d)):
        assert torch.equal(a, b)


def test_large_group_split_and_many_parts():
    """One request split over the whole GPU (more than 32 parts a list), and groups beyond 16 query heads."""
    from uniql_b200 import ops
    g = _gen(8)
    for lens, heads, kv in (([40000], 8, 1), ([6000, 100], 40, 1)):
        q, codes, scales, table, n = _decode_inputs(g, lens, heads=heads, kv=kv)
        got = ops.kv4_attention(q, codes, scales, table, n).cpu()
        for b, m in enumerate(lens):
            k = ref.cached(codes.cpu(), scales.cpu(), table[b].cpu(), 0, 128, m)[0]
            v = ref.cached(codes.cpu(), scales.cpu(), table[b].cpu(), 1, 128, m)[0]
            want, p, _, vv = ref.attend(q[b:b + 1].cpu().double(), k, v, torch.ones(1, m, dtype=torch.bool), 1 / math.sqrt(128))
            _near(got[b], want[0], torch.einsum("mhn,nhd->mhd", p, vv.abs())[0].amax(-1, keepdim=True) + 4.0)
