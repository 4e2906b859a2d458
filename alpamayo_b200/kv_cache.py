"""The int8 paged key/value cache as a program holds it, and the attention of
a decoder stack over it.

* KV8Cache — one layer's pool of pages: int8 codes with one float32 scale per
  (page, KV head) for keys and for values, and the operators on it.
* ClipCache — the caches of all layers for a batch of clips: which pages each
  clip has, how many tokens it holds, and the attention between a layer's qkv
  and o projections for prompts (whole or in chunks), decode steps,
  speculative verification and, where attention totals are kept, eviction.

The reference keeps bf16 keys and values in a StaticCache and calls
scaled_dot_product_attention on it (src/alpamayo_r1/utils/system/patches.py:
381-548); rotary embedding and the query/key norms happen before, in the
caller's `position` function here.
"""
from __future__ import annotations

import torch

from . import ops

PAGE_SIZES, HEAD_DIMS = (16, 32, 64, 128), (64, 128)
MAX_ROWS = 512   # of ops.attention_kv8: new tokens times query heads per KV head


class KV8Cache:
    """One layer's pages.  A page holds `page_size` tokens of one sequence for
    every KV head; an element stands for code * scale."""

    def __init__(self, pages, kv_heads, head_dim, page_size=64, device="cuda"):
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}")
        shape = (pages, kv_heads, page_size, head_dim)
        self.page_size = page_size
        self.k_codes = torch.zeros(shape, dtype=torch.int8, device=device)
        self.v_codes = torch.zeros(shape, dtype=torch.int8, device=device)
        self.k_scale = torch.zeros(shape[:2], device=device)
        self.v_scale = torch.zeros(shape[:2], device=device)

    @property
    def tensors(self):
        """(k_codes, v_codes, k_scale, v_scale), as the operators take them."""
        return self.k_codes, self.v_codes, self.k_scale, self.v_scale

    def append(self, k, v, cu_seqlens, starts, page_table):
        """Write new tokens behind starts[b] tokens (ops.kv8_append)."""
        ops.kv8_append(k, v, cu_seqlens, starts, *self.tensors, page_table)

    def gather(self, page_table, starts, cu_seqlens, rows, dtype=torch.bfloat16):
        """Token ranges back as (k, v) [rows, kv_heads, head_dim] (ops.kv8_gather)."""
        return ops.kv8_gather(*self.tensors, page_table, starts, cu_seqlens, rows, dtype)

    def attend(self, q, page_table, seq_lens, scale=None, weights=None, weights_out=None):
        """Attention of the newest tokens q [B, T, heads, head_dim] (ops.attention_kv8)."""
        return ops.attention_kv8(q, *self.tensors, page_table, seq_lens, scale, weights, weights_out)

    def evict(self, weights, page_table, seq_lens, out_table, budget, sink=4, recent=0):
        """Keep `budget` tokens per sequence and KV head, in other pages (ops.kv8_evict)."""
        return ops.kv8_evict(weights, *self.tensors, page_table, seq_lens, out_table, budget, sink, recent)


def _send(values, device, dtype=torch.int32):
    """Host integers on the device without waiting for its stream: the copy
    comes from pinned memory, which the allocator keeps until it has run."""
    if torch.device(device).type != "cuda":
        return torch.tensor(values, dtype=dtype, device=device)
    return torch.tensor(values, dtype=dtype, pin_memory=True).to(device, non_blocking=True)


def _offsets(lens, device):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return _send(cu, device)


class ClipCache:
    """Key/value caches of `layers` decoder layers for `clips` sequences of up
    to `capacity` tokens.

    prompt(), step() and verify() return the attention of the next forward
    pass, a callable (layer, qkv) -> attention output for
    ``DecoderStack.forward(x, attention=...)``, with qkv [rows, (heads + 2 *
    kv_heads) * head_dim].  Lengths and pages are counted on the host and sent to
    the device on the current stream, which orders all of a cache's calls; no
    call waits for the device.  With ``totals`` the softmax weight of every
    cached token is accumulated by step() and verify(), which evict() needs.
    `spare` tokens of pages per clip are held free for evict(), which moves the
    clips that it cuts.

    `position` (q [rows, heads, head_dim], k [rows, kv_heads, head_dim]) -> (q,
    k) is called for each layer's new rows before they are cached; it keeps its
    own count of positions, which after evict() are no longer the lengths."""

    def __init__(self, layers, clips, capacity, heads, kv_heads, head_dim=128, page_size=64, totals=False, spare=0,
                 position=None, device="cuda"):
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        self.device, self.position = device, position
        self.width = -(-capacity // page_size)
        pages = clips * (self.width + -(-spare // page_size))
        self.caches = [KV8Cache(pages, kv_heads, head_dim, page_size, device) for _ in range(layers)]
        self.free = list(range(pages))
        self.pages = [[] for _ in range(clips)]
        self.lens = [0] * clips
        cap = self.width * page_size
        self.totals = [torch.zeros(clips, kv_heads, cap, device=device) for _ in range(layers)] if totals else None
        self._state()

    def _state(self):
        rows = [p + [-1] * (self.width - len(p)) for p in self.pages]
        self.table = _send(rows, self.device)
        self.seq_lens = _send(self.lens, self.device)

    def _take(self, n):
        if n > len(self.free):
            raise RuntimeError(f"key/value cache is out of pages ({n} wanted, {len(self.free)} free)")
        return [self.free.pop() for _ in range(n)]

    def _grow(self, new):
        """Room for new[b] more tokens of each clip; returns the lengths before."""
        if len(new) != len(self.lens):
            raise ValueError(f"{len(new)} lengths for {len(self.lens)} clips")
        before = list(self.lens)
        after = [n + m for n, m in zip(before, new)]
        need = [-(-n // self.page_size) - len(p) for n, p in zip(after, self.pages)]
        if any(n < 0 for n in new) or any(n > self.width * self.page_size for n in after):
            raise ValueError("a clip would pass the cache's capacity (or a length is negative)")
        if sum(max(0, n) for n in need) > len(self.free):
            raise RuntimeError("key/value cache is out of pages")
        for p, n in zip(self.pages, need):
            p += self._take(max(0, n))
        self.lens = after
        self._state()
        return before

    def _split(self, qkv):
        x = qkv.view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = x.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        if self.position is not None:
            q, k = self.position(q, k)
        return q, k, v

    def prompt(self, lens):
        """Attention for lens[b] packed new tokens of each clip: causal among
        themselves and, where the clip has cached tokens, over those too.  New
        tokens are seen as they are, cached ones as the cache holds them, so a
        clip's result does not depend on the other clips."""
        before = self._grow(list(lens))
        cu = _offsets(lens, self.device)
        starts = _send(before, self.device)
        table, behind = self.table, any(n and m for n, m in zip(before, lens))
        if behind:
            # only clips with new tokens need their keys; `new`: the rows of the new tokens among all keys
            ends = [n if m else 0 for n, m in zip(self.lens, lens)]
            cu_k, rows, zero = _offsets(ends, self.device), sum(ends), torch.zeros_like(starts)
            new, at = [], 0
            for n, m in zip(ends, lens):
                at += n
                new += range(at - m, at)
            new = _send(new, self.device, torch.int64)

        def attention(layer, qkv):
            q, k, v = self._split(qkv)
            cache = self.caches[layer]
            cache.append(k, v, cu, starts, table)
            if behind:
                kk, vv = cache.gather(table, zero, cu_k, rows, q.dtype)
                kk.index_copy_(0, new, k)
                vv.index_copy_(0, new, v)
                out = ops.attention_prefill(q, kk, vv, cu, cu_k)
            else:
                out = ops.attention_prefill(q, k, v, cu)
            return out.view(-1, self.heads * self.head_dim)

        return attention

    def verify(self, new):
        """Attention for `new` tokens of every clip (rows clip by clip), as a
        draft's verification runs them; accept() says how many of them stay."""
        if new * (self.heads // self.kv_heads) > MAX_ROWS:
            raise ValueError(f"{new} tokens at a time: at most {MAX_ROWS // (self.heads // self.kv_heads)}")
        clips = len(self.lens)
        before = self._grow([new] * clips)
        cu = _offsets([new] * clips, self.device)
        starts = _send(before, self.device)
        table, seq_lens = self.table, self.seq_lens

        def attention(layer, qkv):
            q, k, v = self._split(qkv)
            cache = self.caches[layer]
            cache.append(k, v, cu, starts, table)
            out = cache.attend(q.view(clips, new, self.heads, self.head_dim) if q.is_contiguous()
                               else q.unflatten(0, (clips, new)), table, seq_lens,
                               weights=self.totals[layer] if self.totals else None)
            return out.view(-1, self.heads * self.head_dim)

        return attention

    def step(self):
        """Attention for one new token of every clip."""
        return self.verify(1)

    def accept(self, rejected):
        """Take back the last rejected[b] tokens of each clip; their places are
        written again by the next call.  (Page scales that they raised stay,
        and so do the totals that they added to other tokens.)"""
        if len(rejected) != len(self.lens) or any(r < 0 or r > n for r, n in zip(rejected, self.lens)):
            raise ValueError("rejected: one count per clip, at most its length")
        self.lens = [n - r for n, r in zip(self.lens, rejected)]
        for b, n in enumerate(self.lens):
            keep = -(-n // self.page_size)
            self.free += self.pages[b][keep:]
            del self.pages[b][keep:]
            if self.totals and rejected[b]:
                for t in self.totals:
                    t[b, :, n:] = 0
        self._state()

    def evict(self, budget, sink=4, recent=0):
        """Cut every clip of more tokens to its `budget` most attended ones per
        KV head (and layer), its first `sink` and last `recent` ones among
        them; a shorter clip stays in its pages as it is.  Returns the tokens
        kept, per layer: int32 [clips, kv_heads, budget], -1 behind the last."""
        if self.totals is None:
            raise RuntimeError("eviction needs a ClipCache with totals=True")
        if sink < 0 or recent < 0 or budget <= 0 or sink + recent > budget:
            raise ValueError("budget must be positive and hold sink + recent tokens")
        width = -(-budget // self.page_size)
        if width > self.width:
            raise ValueError("budget is larger than the cache's capacity")
        over = [n > budget for n in self.lens]
        places = torch.arange(budget, dtype=torch.int32, device=self.device)
        whole = torch.where(places < self.seq_lens[:, None], places, -1)[:, None]     # a clip that keeps all
        if not any(over):
            return [whole.repeat(1, self.kv_heads, 1) for _ in self.caches]
        need = [width if o else 0 for o in over]
        taken = self._take(sum(need))
        fresh = [[taken.pop() for _ in range(n)] for n in need]
        try:
            out_table = _send([p + [-1] * (width - len(p)) for p in fresh], self.device)
            cuts = (self.seq_lens > budget)[:, None, None]
            lens = torch.where(cuts[:, 0, 0], self.seq_lens, 0)                       # nothing is moved for the others
            cut = [cache.evict(totals, self.table, lens, out_table, budget, sink, recent)
                   for cache, totals in zip(self.caches, self.totals)]
        except BaseException:
            self.free += [p for pages in fresh for p in pages]
            raise
        kept = []
        for totals, (tokens, new_totals, _) in zip(self.totals, cut):
            kept.append(torch.where(cuts, tokens, whole))
            totals[:, :, :budget] = torch.where(cuts, new_totals, totals[:, :, :budget])
            totals[:, :, budget:] = 0
        for b, o in enumerate(over):
            if o:
                self.free += self.pages[b]
                self.pages[b] = fresh[b]
                self.lens[b] = budget
        self._state()
        return kept
