"""KV4Cache: the tensors of a 4-bit paged K/V cache and the calls on them.

A video that is generated frame after frame, a prompt shared by several guidance branches or a
sequence answered token by token keeps its K and V here between calls at D + D / 16 bytes a token
and kv head (136 for D = 128, against 512 in bf16):

    cache = KV4Cache(num_pages=4096, num_kv_heads=24, head_dim=128, max_sequences=4, layers=60)
    starts = cache.reserve([3600], seq_ids=[0])            # room for a frame in sequence 0
    for i, layer in enumerate(model):
        q, k, v = layer.qkv(x)                             # [1, 24, 3600, 128]
        cache.store(k, v, starts, seq_ids=[0], layer=i)
        x = layer.rest(x, cache.attend(q, seq_ids=[0], layer=i))
    cache.fork([0], [1])                                   # a second branch on the same pages
    cache.check()                                          # the one call that synchronises

No call but `check` waits for the GPU; each runs on torch's current stream of the cache's device (calls
on one cache from several streams are the caller's to order).  Lists become device tensors, by a copy
from pinned memory that nothing waits for (11 us of host time each); a captured graph, which would
replay what that memory holds later, refuses them: pass int32 tensors there.
The calls that change pages happen whole or not at all (kernels/kv4.py)."""

from __future__ import annotations

import torch

from .kernels import kv4


class KV4Cache:
    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, max_sequences: int, *, page_size: int = 64,
                 max_pages: int | None = None, layers: int = 1, device: torch.device | str | None = None):
        """`max_pages` is what one sequence can hold (default: all pages, at most 2^30 tokens)."""
        width = kv4.kv4_page_bytes(page_size, head_dim)
        wide = min(num_pages, 2**30 // page_size) if max_pages is None else max_pages
        for name, n in (("num_pages", num_pages), ("num_kv_heads", num_kv_heads), ("max_sequences", max_sequences),
                        ("max_pages", wide), ("layers", layers)):
            if n < 1:
                raise RuntimeError(f"4-bit cache: {name} must be at least 1, got {n}")
        if wide * page_size > 2**30:
            raise RuntimeError(f"4-bit cache: {wide} pages of {page_size} tokens pass 2^30 tokens a sequence")
        dev = torch.device("cuda" if device is None else device)
        self.page_size, self.head_dim = page_size, head_dim
        self.pages = torch.zeros((layers, num_pages, num_kv_heads, width), dtype=torch.uint8, device=dev)
        self.block_table = torch.full((max_sequences, wide), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(max_sequences, dtype=torch.int32, device=dev)
        self.ref_count = torch.zeros(num_pages, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    def _ints(self, x) -> torch.Tensor | None:
        if x is None or isinstance(x, torch.Tensor):
            return x
        dev = self.pages.device
        if dev.type != "cuda":
            return torch.tensor(list(x), dtype=torch.int32)
        with torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("4-bit cache: a captured graph cannot hold a list; pass an int32 tensor")
            # the pinned memory goes back to torch's host allocator, which keeps it until the copy has ended
            return torch.tensor(list(x), dtype=torch.int32, pin_memory=True).to(dev, non_blocking=True)

    def reserve(self, counts, seq_ids=None) -> torch.Tensor:
        """kv4_reserve: room for counts[i] more tokens of seq_ids[i]; the place of the first of each."""
        return kv4.kv4_reserve(self.block_table, self.lengths, self.ref_count, self.page_size, self._ints(counts),
                               seq_ids=self._ints(seq_ids), status=self.status)

    def store(self, k, v, starts, *, counts=None, seq_ids=None, layer: int = 0) -> None:
        """kv4_store into one layer, at the places `reserve` gave."""
        kv4.kv4_store(self.pages[layer], self.block_table, k, v, self._ints(starts), counts=self._ints(counts),
                      seq_ids=self._ints(seq_ids), page_size=self.page_size)

    def append(self, k, v, *, counts=None, seq_ids=None) -> torch.Tensor:
        """reserve and store K and V [B, Hkv, T, D] of a cache of one layer; returns the starts.  What a store
        would refuse is refused before anything is reserved, and so are counts above T (on the device,
        as reserve refuses)."""
        if self.pages.shape[0] != 1:
            raise RuntimeError("4-bit cache append: a cache of several layers takes reserve, then store per layer")
        rows = k.shape[2] if k.dim() == 4 else 0
        if counts is None:
            counts = torch.full((k.shape[0],), rows, dtype=torch.int32, device=self.pages.device)
        counts, ids = self._ints(counts), self._ints(seq_ids)
        put = kv4.store_call(self.pages[0], self.block_table, k, v, counts=counts, seq_ids=ids,
                             page_size=self.page_size)
        starts = kv4.kv4_reserve(self.block_table, self.lengths, self.ref_count, self.page_size, counts, seq_ids=ids,
                                 status=self.status, most=rows)
        put(starts)
        return starts

    def load(self, starts, counts, rows: int, *, seq_ids=None, layer: int = 0, dtype: torch.dtype = torch.bfloat16):
        """kv4_load from one layer."""
        return kv4.kv4_load(self.pages[layer], self.block_table, self._ints(starts), self._ints(counts), rows,
                            self.head_dim, seq_ids=self._ints(seq_ids), dtype=dtype, page_size=self.page_size)

    def attend(self, q, *, counts=None, seq_ids=None, layer: int = 0, causal: bool = False, scale: float | None = None,
               max_length: int | None = None, return_lse: bool = False):
        """kv4_attention over one layer."""
        return kv4.kv4_attention(q, self.pages[layer], self.block_table, self.lengths, counts=self._ints(counts),
                                 seq_ids=self._ints(seq_ids), causal=causal, scale=scale, max_length=max_length,
                                 return_lse=return_lse, page_size=self.page_size)

    def free(self, seq_ids, *, first_pages=None, page_counts=None) -> None:
        """kv4_free: whole sequences, or a range of each one's pages."""
        kv4.kv4_free(self.block_table, self.lengths, self.ref_count, self.page_size, self._ints(seq_ids),
                     first_pages=self._ints(first_pages), page_counts=self._ints(page_counts), status=self.status)

    def fork(self, src, dst, *, share: bool = True) -> None:
        """kv4_fork: the empty sequences dst become what src are, in every layer."""
        kv4.kv4_fork(self.pages, self.block_table, self.lengths, self.ref_count, self.page_size, self._ints(src),
                     self._ints(dst), share=share, status=self.status)

    def compact(self) -> torch.Tensor:
        """kv4_compact: the held pages are the lowest ones; their number, on the device."""
        return kv4.kv4_compact(self.pages, self.block_table, self.ref_count)

    def check(self) -> None:
        """Raise what the first call that could not happen found since the last check (waits for the GPU)."""
        code = int(self.status.item())
        if code != 0:
            self.status.zero_()
            raise RuntimeError(f"4-bit cache: {kv4.STATUS.get(code, f'status {code}')}")
