"""A paged KV cache held in 4 bits for all layers of a model, and a decoder block's attention over it.

The reference keeps fp16 keys and values in a transformers cache and leaves attention to torch; this is what a served model with
4-bit weights has next to its linears.  Everything that a step decides (pages, slots, positions) is worked out on the GPU by
ops.kv_page_plan, so a decode step has no host synchronisation and can be captured in a CUDA graph and replayed.

    cache = PagedKV4Cache(layers, pages, kv_heads, head_dim, requests=64, max_tokens=8192)
    step = cache.plan(new_lens, total)                 # pages and slots of the step's tokens, the same for every layer
    out = attention_block(q, k, v, o, x, residual, cache, layer, step)          # per layer: q/k/v, append, attention, o + residual
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import fused, ops


class KVStep(NamedTuple):
    """One step's tokens, packed request after request, and the keys they attend to: another step may be planned before the layers of
    this one have run.  `release` and `move` change the block table that all steps read: they come behind the layers."""
    rows: int                    # requests 0 .. rows - 1 take part
    single: bool                 # one new token for each of them: a decode step
    fresh: bool                  # no request had cached tokens before: keys and values of the step are all there is
    slots: torch.Tensor          # int64 [total]: where each token's rows go (-1: padding, or no page was left)
    positions: torch.Tensor      # int64 [total]
    cu: torch.Tensor             # int32 [rows + 1]: first token of each request
    max_keys: int                # bound of the keys of all requests together, for a step that is neither single nor fresh
    lens: torch.Tensor           # int32 [rows]: keys of each request, the step's own included (0: left out of the step)
    cu_keys: torch.Tensor        # int32 [rows + 1]: their exclusive sums


class PagedKV4Cache:
    """Pages of every layer, the block table, the requests' lengths and the stack of free pages, all on the GPU.

    Layer l's cache is (codes[l], scales[l]) as the operators take it; a page number means the same page in every layer."""

    def __init__(self, layers, num_pages, kv_heads, head_dim_k, head_dim_v=None, page_size=64, requests=64, max_tokens=8192, device="cuda"):
        self.head_dim_k, self.head_dim_v = head_dim_k, head_dim_k if head_dim_v is None else head_dim_v
        if self.head_dim_v <= 0 or self.head_dim_v > 128 or self.head_dim_v % 8 or head_dim_k % 8 or not 0 < head_dim_k <= 128:
            raise RuntimeError("head sizes must be multiples of 8 up to 128")
        codes, scales = ops.kv4_cache(layers * num_pages, kv_heads, page_size, max(head_dim_k, self.head_dim_v), device)
        self.codes = codes.view(layers, num_pages, *codes.shape[1:])
        self.scales = scales.view(layers, num_pages, *scales.shape[1:])
        self.page_size, self.num_pages = page_size, num_pages
        device = codes.device
        self.block_table = torch.full((requests, max(1, -(-max_tokens // page_size))), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self._ones = torch.ones_like(self.lens)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)

    def plan(self, new_lens, total, fresh=False, max_keys=None) -> KVStep:
        """Take pages for new_lens[i] (int32, CUDA) tokens of requests 0 .. len(new_lens) - 1, `total` rows of tokens in all (rows
        behind the last token are padding), and move their lengths on.  fresh: the caller knows that all of them were empty.
        max_keys: bound of the requests' keys together after the step, where they are known to be fewer than their tables can
        hold (a prompt step behind a prefix gathers that many rows); requests that do not fit into it give zeros and raise
        status bit 2.

        A request that cannot have all its pages, within `total` rows and the table, is left out (status bit 3): it keeps its
        length and pages, nothing of it is stored, and its rows of a decode step or of a chunk come out as zeros (a fresh step
        works out its rows, but the cache does not hold them).  It may be planned again once `release` has given pages back."""
        n = new_lens.shape[0]
        if n > self.block_table.shape[0]:
            raise RuntimeError(f"the cache has room for {self.block_table.shape[0]} requests")
        slots, positions, cu, _, _, lens, cu_keys = ops.kv_page_plan(self.lens[:n], new_lens, self.block_table[:n], self.free_pages,
                                                                     self.free_count, self.page_size, total, in_place=True, whole=True)
        bound = min(n * self.block_table.shape[1], self.num_pages) * self.page_size
        return KVStep(n, False, fresh, slots, positions, cu, bound if max_keys is None else min(bound, max_keys), lens, cu_keys)

    def plan_decode(self, n) -> KVStep:
        """One new token for each of requests 0 .. n - 1."""
        if not 0 <= n <= self.block_table.shape[0]:
            raise RuntimeError(f"the cache has room for {self.block_table.shape[0]} requests")
        return self.plan(self._ones[:n], n)._replace(single=True)

    def append(self, layer, k, v, step) -> None:
        ops.kv4_append(k, v, step.slots, self.codes[layer], self.scales[layer])

    def attend(self, layer, q, k, v, step, softmax_scale=None):
        """Attention of the step's queries q [total, heads, channels]; k and v are the step's own rows, already appended.  Decode
        steps read the cache in 4 bits, fresh prompts their own keys and values, later chunks of a prompt the cached rows of
        their requests, gathered."""
        codes, scales, table, lens = self.codes[layer], self.scales[layer], self.block_table[:step.rows], step.lens
        if step.single:
            return ops.kv4_attention(q, codes, scales, table, lens, self.head_dim_v, softmax_scale)
        if step.fresh:
            return ops.prompt_attention(q, k, v, step.cu, None, True, softmax_scale)
        kk, vv = ops.kv4_gather(codes, scales, table, step.cu_keys, step.max_keys, self.head_dim_k, self.head_dim_v, q.dtype)
        return ops.prompt_attention(q, kk, vv, step.cu, step.cu_keys, True, softmax_scale)

    def release(self, rows) -> None:
        """Give the pages of finished requests back.  Synchronises with the host: not for the inside of a captured step.  The rows
        of a step are always 0 .. n - 1; what keeps running above a finished row is moved down with `move`."""
        for r in rows:
            used = self.block_table[r][self.block_table[r] >= 0]
            n = int(self.free_count.item())
            self.free_pages[n:n + used.numel()] = used
            self.free_count += used.numel()
            self.block_table[r] = -1
            self.lens[r] = 0

    def move(self, src, dst) -> None:
        """Make the request of row src the one of the (released) row dst: what dst still holds is not given back."""
        if src == dst:
            return
        self.block_table[dst] = self.block_table[src]
        self.lens[dst] = self.lens[src]
        self.block_table[src] = -1
        self.lens[src] = 0


def attention_block(q_proj, k_proj, v_proj, o_proj, x, residual, cache, layer, step, rotary=None, softmax_scale=None):
    """residual + o_proj(attention(x)) of one decoder block (modeling/llama/llama_qblocks.py:104-106 and the attention between): q/k/v in
    one launch, the new rows quantised into the cache, attention, o_proj with the residual.  x and residual [tokens, hidden], tokens
    as packed in `step`; rotary(q, k, positions) -> (q, k) turns [tokens, heads, channels] by position where the model does."""
    q, k, v = fused.qkv_proj(q_proj, k_proj, v_proj, x)
    t = x.shape[0]
    q, k, v = q.view(t, -1, cache.head_dim_k), k.view(t, -1, cache.head_dim_k), v.view(t, -1, cache.head_dim_v)
    if rotary is not None:
        q, k = rotary(q, k, step.positions)
    cache.append(layer, k, v, step)
    out = cache.attend(layer, q, k, v, step, softmax_scale)
    return fused.linear_residual(o_proj, out.view(t, -1), residual)
