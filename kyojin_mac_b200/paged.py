"""A paged key/value cache and the attention block of a decoder layer over the package's quantized linears: q | k | v product, rotary positions and cache append, attention
over the cache, o product. It stands beside `foreign_moe.RoutedBlock`, as the other half of a layer; the reference keeps its attention outside the quantized-linear path that
this package replaces, so the names here are the package's own.

    cache = PagedCache(layers=1, pages=4096, kv_heads=8, head_dim=128, requests=64, max_tokens=16384)
    block = AttentionBlock(qkv, o, heads=64, kv_heads=8, head_dim=128, base=500000.0)      # qkv: one linear of (heads + 2 kv_heads) head_dim outputs, or (q, k, v)
    step = cache.step(new_lens, rows=64)                # int32 [requests] on the device: new tokens of each request; the lengths grow
    y = block(x, cache, step, max_q=1)                  # x [rows, hidden], packed by request -> [rows, hidden]
    cache.release(done)                                 # bool [requests]: their pages are free again

Nothing here waits for the device, so a step may be captured (`host_graph.HostGraph`, torch.cuda.graph) and replayed: lengths, table and free list live on the device."""
from __future__ import annotations

import torch

from . import ops


class PagedCache:
    """`pages` pages of `page` tokens for every layer, a block table for `requests` requests of up to `max_tokens` tokens, and the list of free pages. keys[i] and values[i]
    are [pages, kv_heads, page, head_dim]; `table` int32 [requests, columns], `lens` int32 [requests], `free_pages` int32 [pages] with the first `free_count` of them free."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, requests: int, max_tokens: int, page: int = 64, dtype=torch.float16, device="cuda"):
        if page not in (16, 32, 64, 128, 256):
            raise ValueError(f"{page} tokens a page: 16, 32, 64, 128 or 256")
        if min(layers, pages, kv_heads, requests, max_tokens) < 1 or head_dim not in (64, 128) or dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("a cache has layers, pages, heads of 64 or 128, requests and tokens, in float16 or bfloat16")
        self.page, self.requests, self.max_tokens = page, requests, max_tokens
        both = torch.zeros((layers, 2, pages, kv_heads, page, head_dim), dtype=dtype, device=device)
        self.keys, self.values = [both[i, 0] for i in range(layers)], [both[i, 1] for i in range(layers)]
        self.table = torch.full((requests, -(-max_tokens // page)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros((requests,), dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)

    def step(self, new_lens: torch.Tensor, rows: int) -> ops.PagedStep:
        """Slots for the step's tokens; lengths, table and free list move on. Requests that cannot be served are counted in `refused` and keep their lengths: their rows
        have no slot and their attention is zeros."""
        return ops.paged_step(self.table, self.lens, new_lens, self.free_pages, self.free_count, self.page, rows, in_place=True)

    def release(self, which: torch.Tensor) -> torch.Tensor:
        return ops.paged_release(self.table, self.lens, which, self.free_pages, self.free_count, self.page)


class AttentionBlock(torch.nn.Module):
    """qkv: a linear whose outputs are all query heads, then all key heads, then all value heads, or the three linears (members of a same-input group, for instance); o: the
    output linear. Rotary positions from `ops.rope_frequencies(rot, base, scaling)` over the first `rot` values of a head (all unless given); window and sinks as in
    `ops.paged_attention`. x [rows, hidden] packed by request; rows behind the last request come out finite and without meaning."""

    def __init__(self, qkv, o, heads: int, kv_heads: int, head_dim: int, rot: int | None = None, base: float = 10000.0, scaling: dict | None = None, interleaved: bool = False,
                 window: int = 0, sinks: int = 0, scale: float | None = None, device="cuda"):
        super().__init__()
        parts = [qkv] if isinstance(qkv, torch.nn.Module) else list(qkv)
        widths = [heads * head_dim, kv_heads * head_dim, kv_heads * head_dim]
        if len(parts) not in (1, 3) or [m.out_features for m in parts] != ([sum(widths)] if len(parts) == 1 else widths) or o.in_features != widths[0]:
            raise ValueError(f"qkv gives {widths} outputs (one linear or three), o takes {widths[0]}")
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError("query heads are a multiple of the key-value heads")
        if rot is not None and rot > head_dim:
            raise ValueError(f"rot={rot}: at most {head_dim}")
        self.qkv, self.o = torch.nn.ModuleList(parts), o
        self.heads, self.kv_heads, self.head_dim, self.widths = heads, kv_heads, head_dim, widths
        self.interleaved, self.window, self.sinks, self.scale = interleaved, window, sinks, scale
        self.inv_freq, self.mscale = ops.rope_frequencies(head_dim if rot is None else rot, base, scaling, device)

    def forward(self, x: torch.Tensor, cache: PagedCache, step: ops.PagedStep, max_q: int, layer: int = 0) -> torch.Tensor:
        if x.dim() != 2 or x.shape[0] != step.positions.shape[0]:
            raise ValueError(f"x is [{step.positions.shape[0]}, hidden], the step's rows, got {tuple(x.shape)}")
        ys = self.qkv[0](x).split(self.widths, dim=1) if len(self.qkv) == 1 else [m(x) for m in self.qkv]
        q, k, v = (y.unflatten(1, (-1, self.head_dim)) for y in ys)
        kc, vc = cache.keys[layer], cache.values[layer]
        # queries are turned, and attention written, where the product left them: no other buffers, and rows behind the last request stay finite
        ops.rope_append(q, k, v, step.positions, step.slots, self.inv_freq, kc, vc, interleaved=self.interleaved, mscale=self.mscale, out=q)
        ops.paged_attention(q, kc, vc, cache.table, step.kv_lens, step.cu_q, max_q, scale=self.scale, window=self.window, sinks=self.sinks, out=q)
        return self.o(q.flatten(1))
