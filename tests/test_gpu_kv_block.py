"""GPU: attention_block against a plain decoder block in 64 bits, and mistakes planted in the plain one, which have to show."""
import math

import numpy as np
import pytest
import torch

import kv_reference as ref
from helpers import linear_tolerance_check
from oracle import uniql_oracle as orc

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, D, PAGE = 512, 8, 2, 64, 16
HALF = 2.0 ** -11


def _layer(g, n_in, n_out, bias):
    from uniql_b200.quantize.quant_linear_layers import W4A16B16O16Linear
    lin = torch.nn.Linear(n_in, n_out, bias=bias).half()
    lin.weight.data = (torch.randn(n_out, n_in, generator=g) * 0.04).half()
    if bias:
        lin.bias.data = (torch.randn(n_out, generator=g) * 0.3).half()
    q = W4A16B16O16Linear.from_fp16(lin.cuda()).cuda()
    w = torch.from_numpy(orc.dequantize(q.weight.cpu().numpy(), q.scale.cpu().numpy())[:n_in, :n_out].astype(np.float64))
    return q, w, lin.bias.data.double().cpu() if bias else torch.zeros(n_out, dtype=torch.float64)


def _rotary(q, k, positions):
    """Turned in 64 bits and rounded once, so that block and reference hold the same bits."""
    d = q.shape[-1]
    ang = positions.double()[:, None] / 10000.0 ** (torch.arange(0, d, 2, device=q.device).double() / d)
    cos, sin = (torch.cat((f(ang), f(ang)), -1)[:, None] for f in (torch.cos, torch.sin))
    turn = lambda x: (x.double() * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1).double() * sin).to(q.dtype)  # noqa: E731
    return turn(q), turn(k)


def _attend(q, k, v, step, seen, interleaved=False):
    """Attention in 64 bits of q [m, heads, d] over k, v [n, kv, d] and how far the kernels may be off, value by value: the result's
    rounding, the rounded weights (of every term; next to codes also of what 8 steps of scale weigh), fp16's denormals, scores as
    sums in 32 bits."""
    if interleaved:
        k, v = (x.repeat(1, HEADS // KV, 1) for x in (k, v))
    out, p, size, vv = ref.attend(q.double(), k.double(), v.double(), seen, 1 / math.sqrt(D))
    mass = torch.einsum("mhn,nhd->mhd", p, vv.abs())
    if step is not None:
        mass = mass + torch.einsum("mhn,nh->mh", p, (8 * step).repeat_interleave(HEADS // KV, 1))[..., None]
    off = 2 * ((D + 16) * 2.0 ** -23 * (size + 1.0))[..., None] + 2.0 ** -18
    return out, out.abs() * HALF + mass * (HALF + off) + k.shape[0] * 2.0 ** -22 * vv.abs().max() + 1e-7


def _far(got, want, attn, tol, w):
    """How far each row is off, in units of its bound: the attention's error through the weights (their largest singular value), the
    linear's own gate of 1e-2, and the sum's rounding."""
    bound = torch.linalg.matrix_norm(w, 2) * tol.flatten(1).norm(dim=1) + 1e-2 * (attn.flatten(1) @ w).norm(dim=1) + HALF * want.norm(dim=1)
    return (got.double() - want).norm(dim=1) / bound


MISTAKES = ["keys not turned", "k and v swapped", "heads interleaved", "no residual", "positions one too far"]


def test_attention_block_against_a_plain_block():
    from uniql_b200 import fused, ops
    from uniql_b200.kv_cache import PagedKV4Cache, attention_block
    g = torch.Generator().manual_seed(0)
    layers = [_layer(g, HIDDEN, n * D, True) for n in (HEADS, KV, KV)] + [_layer(g, HEADS * D, HIDDEN, False)]
    mods, w_o = [x[0] for x in layers], layers[3][1]
    cache = PagedKV4Cache(1, 40, KV, D, page_size=PAGE, requests=3, max_tokens=160)
    codes, scales = (t[0].cpu().clone() for t in (cache.codes, cache.scales))
    ops.read_and_clear_status("cuda")
    held = [0, 0, 0]
    for new, kind in (([20, 47, 5], "fresh"), ([9, 1, 30], "chunk"), ([1, 1, 1], "decode"), ([1, 1, 1], "decode")):
        total = sum(new)
        x, r = (torch.randn(total, HIDDEN, generator=g).half().cuda() for _ in range(2))
        step = cache.plan_decode(3) if kind == "decode" else cache.plan(torch.tensor(new, dtype=torch.int32).cuda(), total, fresh=kind == "fresh")
        got = attention_block(*mods, x, r, cache, 0, step, _rotary).cpu()

        # q, k and v: the linears' own gate, then the same bits go through the plain block
        qkv = fused.qkv_proj(*mods[:3], x)
        for y, (_, w, b) in zip(qkv, layers):
            linear_tolerance_check(y.cpu().numpy(), (x.cpu().double() @ w + b).numpy())
        at = torch.cat([torch.arange(h, h + n) for h, n in zip(held, new)])
        assert step.positions.tolist() == at.tolist()
        q, k, v = (y.view(total, -1, D) for y in qkv)
        turned, later = _rotary(q, k, at.cuda()), _rotary(q, k, at.cuda() + 1)
        (q, kt), v, raw = (t.cpu() for t in turned), v.cpu(), k.cpu()
        ref.append(kt, v, step.slots.cpu(), codes, scales)
        assert torch.equal(cache.codes[0].cpu(), codes) and torch.equal(cache.scales[0].cpu(), scales)

        plain = {m: [] for m in [None] + MISTAKES}
        bounds, first = [], 0
        for i, n in enumerate(new):
            own, h = slice(first, first + n), held[i] + n
            first += n
            seen = torch.arange(h)[None] <= torch.arange(n)[:, None] + h - n
            table = cache.block_table[i].cpu()
            if kind == "fresh":
                rows, step_v = (kt[own], v[own]), None
            else:
                rows, step_v = tuple(ref.cached(codes, scales, table, j, D, h)[0] for j in (0, 1)), ref.cached(codes, scales, table, 1, D, h)[1]
                if kind == "chunk":                               # gathered: rounded to fp16
                    rows = tuple(t.half() for t in rows)
            out, tol = _attend(q[own], *rows, step_v, seen)
            plain[None].append(out)
            bounds.append(tol)
            plain["heads interleaved"].append(_attend(q[own], *rows, None, seen, True)[0])
            plain["k and v swapped"].append(_attend(q[own], rows[1], rows[0], None, seen)[0])
            plain["positions one too far"].append(_attend(later[0][own].cpu(), *rows, None, seen)[0])
            bare = rows[0].clone()
            bare[h - n:] = raw[own].to(bare.dtype)
            plain["keys not turned"].append(_attend(q[own], bare, rows[1], None, seen)[0])
            held[i] = h
        plain = {m: torch.cat(t).flatten(1) for m, t in plain.items() if t}
        plain["no residual"] = plain[None]
        tol = torch.cat(bounds)
        y = r.cpu().double() + plain[None] @ w_o
        assert _far(got, y, plain[None], tol, w_o).max() <= 1
        for m in MISTAKES:
            if kind == "fresh" and m == "positions one too far":
                continue                                          # seen in the first chunk, where queries and cached keys part
            wrong = plain[m] @ w_o + (0 if m == "no residual" else r.cpu().double())
            assert _far(wrong, y, plain[None], tol, w_o).max() > 1.5, m
    assert cache.lens.tolist() == held and ops.read_and_clear_status("cuda") == 0
