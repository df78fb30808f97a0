"""A paged K/V cache held in 4 bits: attention over it, rows stored and loaded, pages reserved,
freed, forked and moved together, on the HIP kernels of csrc/spr_kv4.hip and
csrc/spr_kv4_attention.hip.  `sparsepr_amd.kv4_cache.KV4Cache` keeps the tensors these functions
take.

pages        uint8 [P, Hkv, page_bytes], or [layers, P, Hkv, page_bytes] for the page calls: pages of
             page_size tokens, K and V as 4-bit floats with one power-of-two scale per 32 dims
             (kv4_page_bytes; D + D / 16 bytes a token and kv head, against 4 D in bf16).
block_table  int32 [sequences, wide], a sequence's pages in order, -1 past the last.
lengths      int32 [sequences], tokens.
ref_count    int32 [P], how many sequences hold a page; 0 is free.

All metadata lives on the device and no call synchronises.  The page calls (kv4_reserve, kv4_free,
kv4_fork) check everything on the device first and change all or nothing; what was wrong is left in
`status` (int32 [1], see STATUS), which keeps its first entry until the caller clears it."""

from __future__ import annotations

import math

import torch

from .. import _lib

HEAD_DIMS = (64, 128)
PAGE_SIZES = (32, 64, 128, 256)
MAX_NAMED = 2048

STATUS = {
    1: "a sequence outside the table",
    2: "a sequence named twice",
    3: "a negative count, or a range outside the sequence's pages",
    4: "more tokens than a row of the block table has pages for",
    5: "not enough free pages",
    6: "a fork onto a sequence that holds tokens",
    7: "a length outside the table, or a table entry outside the pool",
}


def kv4_page_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one kv head's part of a page."""
    if page_size not in PAGE_SIZES:
        raise RuntimeError(f"4-bit cache: page size {page_size} not supported {PAGE_SIZES}")
    if head_dim not in HEAD_DIMS:
        raise RuntimeError(f"4-bit cache: head dim {head_dim} not supported {HEAD_DIMS}")
    return page_size * (head_dim + head_dim // 16)


def _page_size(pages: torch.Tensor, head_dim: int, what: str) -> int:
    if head_dim not in HEAD_DIMS:
        raise RuntimeError(f"{what}: head dim {head_dim} not supported {HEAD_DIMS}")
    size = pages.shape[-1] // (head_dim + head_dim // 16)
    if size not in PAGE_SIZES or pages.shape[-1] != kv4_page_bytes(size, head_dim):
        raise RuntimeError(f"{what}: pages of {pages.shape[-1]} bytes a head are not whole pages of head dim {head_dim}")
    return size


def _int32(t: torch.Tensor, shape: tuple, name: str, what: str) -> torch.Tensor:
    """An int32 tensor of this shape, as the kernels read it."""
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} "
                           f"{tuple(t.shape)}")
    return t


def _check_pool(pages: torch.Tensor, what: str) -> None:
    if pages.dtype != torch.uint8 or pages.ndim != 3 or not pages.is_contiguous() or pages.numel() == 0:
        raise RuntimeError(f"{what}: pages must be a contiguous uint8 tensor [P, Hkv, bytes], got {pages.dtype} "
                           f"{tuple(pages.shape)}")


def _check_table(block_table: torch.Tensor, what: str) -> tuple[int, int]:
    if block_table.dtype != torch.int32 or block_table.ndim != 2 or not block_table.is_contiguous():
        raise RuntimeError(f"{what}: block_table must be a contiguous int32 tensor [sequences, wide], got "
                           f"{block_table.dtype} {tuple(block_table.shape)}")
    return block_table.shape[0], block_table.shape[1]


def _batch_ids(seq_ids, batch: int, sequences: int, what: str):
    if seq_ids is None:
        if batch > sequences:
            raise RuntimeError(f"{what}: a batch of {batch} without seq_ids on a table of {sequences} sequences")
        return None
    return _int32(seq_ids, (batch,), "seq_ids", what)


def _rows_in_place(x: torch.Tensor) -> torch.Tensor:
    """x [B, H, T, D] by its strides where rows are packed and 16-byte aligned, else a copy."""
    step = 16 // x.element_size()
    ok = (x.stride(3) == 1 and x.data_ptr() % 16 == 0
          and all(x.shape[i] <= 1 or (x.stride(i) % step == 0 and x.stride(i) >= 0) for i in range(3)))
    return x if ok else x.contiguous()


def _strides(x: torch.Tensor) -> list[int]:
    return [x.stride(i) if x.shape[i] > 1 else 0 for i in range(3)]


def kv4_store(pages: torch.Tensor, block_table: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
              *, counts: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None) -> None:
    """Write K and V rows [B, Hkv, T, D] (bf16, fp16 or fp32, any strides with packed rows) to the
    cache: row t < counts[b] becomes token starts[b] + t of sequence seq_ids[b] (default b).

    The pages have to be there (kv4_reserve): rows without one are not written.  No two rows of a call
    may name one token, and no other sequence may share the page written to (kv4_fork sees to that).
    A group of 32 dims with an infinity or a NaN is stored as NaN."""
    what = "4-bit cache store"
    dev = _lib.require_gpu(pages, block_table, k, v, starts, counts, seq_ids, what=what)
    _check_pool(pages, what)
    if k.ndim != 4 or v.shape != k.shape or v.dtype != k.dtype or k.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: K and V must be [B, Hkv, T, D] of one dtype (bfloat16, float16, float32), got "
                           f"{k.dtype} {tuple(k.shape)} / {v.dtype} {tuple(v.shape)}")
    b, h, t, d = k.shape
    size = _page_size(pages, d, what)
    if pages.shape[1] != h:
        raise RuntimeError(f"{what}: K has {h} heads, the pages {pages.shape[1]}")
    sequences, wide = _check_table(block_table, what)
    ids = _batch_ids(seq_ids, b, sequences, what)
    _int32(starts, (b,), "starts", what)
    if counts is not None:
        _int32(counts, (b,), "counts", what)
    if k.numel() == 0:
        return
    kc, vc = _rows_in_place(k), _rows_in_place(v)
    with torch.cuda.device(dev):
        _lib.call("spr_kv4_store", _lib.ptr(pages), pages.shape[0], h, size, d, _lib.ptr(block_table), sequences, wide,
                  _lib.ptr(ids), _lib.ptr(starts), _lib.ptr(counts), _lib.ptr(kc), _lib.ptr(vc),
                  _lib.DTYPE_CODE[k.dtype], b, t, *_strides(kc), *_strides(vc), _lib.stream(dev))


def kv4_load(pages: torch.Tensor, block_table: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor, rows: int,
             head_dim: int, *, seq_ids: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16):
    """Tokens starts[b] .. starts[b] + counts[b] - 1 of every named sequence as (K, V) [B, Hkv, rows, D]
    in `dtype` (exact in bf16 and fp32); rows past the count are 0, rows with no page NaN."""
    what = "4-bit cache load"
    dev = _lib.require_gpu(pages, block_table, starts, counts, seq_ids, what=what)
    _check_pool(pages, what)
    size = _page_size(pages, head_dim, what)
    if dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: dtype must be bfloat16, float16 or float32, got {dtype}")
    if rows < 0 or starts.ndim != 1:
        raise RuntimeError(f"{what}: rows {rows}, starts {tuple(starts.shape)}")
    b, h = starts.shape[0], pages.shape[1]
    sequences, wide = _check_table(block_table, what)
    ids = _batch_ids(seq_ids, b, sequences, what)
    _int32(starts, (b,), "starts", what)
    _int32(counts, (b,), "counts", what)
    k = torch.empty((b, h, rows, head_dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    with torch.cuda.device(dev):
        _lib.call("spr_kv4_load", _lib.ptr(pages), pages.shape[0], h, size, head_dim, _lib.ptr(block_table), sequences,
                  wide, _lib.ptr(ids), _lib.ptr(starts), _lib.ptr(counts), _lib.ptr(k), _lib.ptr(v),
                  _lib.DTYPE_CODE[dtype], b, rows, _lib.stream(dev))
    return k, v


def kv4_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
                  counts: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None, causal: bool = False,
                  scale: float | None = None, max_length: int | None = None, return_lse: bool = False):
    """softmax(q K^T * scale) V over the cached tokens: q [B, Hq, T, D] bf16 or fp16 (any strides with
    packed rows) -> out [B, Hq, T, D] in q's dtype (and lse fp32 [B, Hq, T], natural log).

    Hq is a multiple of Hkv; query head h reads kv head h // (Hq // Hkv).  Batch entry b attends
    sequence seq_ids[b] (default b) with its first counts[b] rows (default all).  With `causal` the last
    row in use is the sequence's last token and each row sees the tokens up to its own (store them
    first).  Rows that see nothing, and rows past the count, are 0 with lse -inf.  `max_length`, the
    longest length the caller knows of (default: what the table can hold), only sizes the launch."""
    what = "4-bit cache attention"
    dev = _lib.require_gpu(q, pages, block_table, lengths, counts, seq_ids, what=what)
    _check_pool(pages, what)
    if q.ndim != 4 or q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"{what}: q must be [B, Hq, T, D] in bfloat16 or float16, got {q.dtype} {tuple(q.shape)}")
    b, h, t, d = q.shape
    size = _page_size(pages, d, what)
    hk = pages.shape[1]
    if h == 0 or h % hk != 0:
        raise RuntimeError(f"{what}: Q heads ({h}) must be a multiple of KV heads ({hk})")
    sequences, wide = _check_table(block_table, what)
    ids = _batch_ids(seq_ids, b, sequences, what)
    _int32(lengths, (sequences,), "lengths", what)
    if counts is not None:
        _int32(counts, (b,), "counts", what)
    longest = wide * size if max_length is None else min(int(max_length), wide * size)
    sc = float(scale) if scale is not None else 1.0 / math.sqrt(d)
    out = torch.empty((b, h, t, d), dtype=q.dtype, device=dev)
    lse = torch.empty((b, h, t), dtype=torch.float32, device=dev) if return_lse else None
    if out.numel() > 0:
        qc = _rows_in_place(q)
        need = int(_lib.query("spr_kv4_attention_workspace", b, h, hk, t, d, longest))
        ws = _lib.workspace(need, dev) if need > 0 else None
        with torch.cuda.device(dev):
            _lib.call("spr_kv4_attention", _lib.ptr(qc), *_strides(qc), _lib.DTYPE_CODE[q.dtype], b, h, hk, t, d,
                      _lib.ptr(pages), pages.shape[0], size, _lib.ptr(block_table), sequences, wide, _lib.ptr(lengths),
                      _lib.ptr(counts), _lib.ptr(ids), int(causal), sc, longest, _lib.ptr(out), _lib.ptr(lse),
                      _lib.ptr(ws), need, _lib.stream(dev))
    return (out, lse) if return_lse else out


def _check_metadata(block_table, lengths, ref_count, page_size, what):
    sequences, wide = _check_table(block_table, what)
    if lengths is not None:
        _int32(lengths, (sequences,), "lengths", what)
    if ref_count.ndim != 1 or ref_count.shape[0] == 0:
        raise RuntimeError(f"{what}: ref_count must be [P], got {tuple(ref_count.shape)}")
    _int32(ref_count, (ref_count.shape[0],), "ref_count", what)
    if page_size not in PAGE_SIZES:
        raise RuntimeError(f"{what}: page size {page_size} not supported {PAGE_SIZES}")
    return sequences, wide


def _named(ids: torch.Tensor, name: str, what: str) -> int:
    if ids.ndim != 1 or ids.shape[0] > MAX_NAMED:
        raise RuntimeError(f"{what}: {name} must be a vector of at most {MAX_NAMED}, got {tuple(ids.shape)}")
    _int32(ids, (ids.shape[0],), name, what)
    return ids.shape[0]


def _check_status(status, what):
    return None if status is None else _int32(status, (1,), "status", what)


def _layers(pages: torch.Tensor, num_pages: int, what: str) -> tuple[int, int, int]:
    """(bytes of a page, bytes from layer to layer, layers) of [P, H, bytes] or [layers, P, H, bytes]."""
    p = pages if pages.ndim == 4 else pages.unsqueeze(0)
    if pages.dtype != torch.uint8 or p.ndim != 4 or p.numel() == 0 or not p.is_contiguous():
        raise RuntimeError(f"{what}: pages must be a contiguous uint8 tensor [P, Hkv, bytes] or [layers, P, Hkv, "
                           f"bytes], got {pages.dtype} {tuple(pages.shape)}")
    if p.shape[1] != num_pages:
        raise RuntimeError(f"{what}: {p.shape[1]} pages, ref_count of {num_pages}")
    if (p.shape[2] * p.shape[3]) % 16 != 0:
        raise RuntimeError(f"{what}: pages of {p.shape[2]} x {p.shape[3]} bytes are not whole 16-byte pieces")
    page = p.shape[2] * p.shape[3]
    return page, page * num_pages, p.shape[0]


def kv4_reserve(block_table: torch.Tensor, lengths: torch.Tensor, ref_count: torch.Tensor, page_size: int,
                counts: torch.Tensor, *, seq_ids: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """Room for counts[i] more tokens of sequence seq_ids[i] (default i): new pages (the lowest free
    ones) in its row of the table, the length with them.  Returns starts int32 [n], the place of the
    first new token of each, or -1 for all when the call could not happen."""
    what = "4-bit cache reserve"
    dev = _lib.require_gpu(block_table, lengths, ref_count, counts, seq_ids, status, what=what)
    sequences, wide = _check_metadata(block_table, lengths, ref_count, page_size, what)
    n = _named(counts, "counts", what)
    ids = _batch_ids(seq_ids, n, sequences, what)
    _check_status(status, what)
    starts = torch.empty(n, dtype=torch.int32, device=dev)
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev)
    with torch.cuda.device(dev):
        _lib.call("spr_kv4_reserve", _lib.ptr(block_table), _lib.ptr(lengths), _lib.ptr(ref_count), _lib.ptr(counts),
                  _lib.ptr(ids), n, sequences, wide, page_size, ref_count.shape[0], _lib.ptr(starts), _lib.ptr(status),
                  _lib.ptr(ws), ws.numel(), _lib.stream(dev))
    return starts


def kv4_free(block_table: torch.Tensor, lengths: torch.Tensor, ref_count: torch.Tensor, page_size: int,
             seq_ids: torch.Tensor, *, first_pages: torch.Tensor | None = None,
             page_counts: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """The named sequences give their pages back and are empty; or only page_counts[i] pages from the
    first_pages[i]-th on (default 0, and all from there on), as a sliding window does: the pages behind
    close up and the length loses the tokens that lay there.  A page is free when nobody holds it."""
    what = "4-bit cache free"
    dev = _lib.require_gpu(block_table, lengths, ref_count, seq_ids, first_pages, page_counts, status, what=what)
    sequences, wide = _check_metadata(block_table, lengths, ref_count, page_size, what)
    n = _named(seq_ids, "seq_ids", what)
    for t, name in ((first_pages, "first_pages"), (page_counts, "page_counts")):
        if t is not None:
            _int32(t, (n,), name, what)
    _check_status(status, what)
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev)
    with torch.cuda.device(dev):
        _lib.call("spr_kv4_free", _lib.ptr(block_table), _lib.ptr(lengths), _lib.ptr(ref_count), _lib.ptr(seq_ids),
                  _lib.ptr(first_pages), _lib.ptr(page_counts), n, sequences, wide, page_size, ref_count.shape[0],
                  _lib.ptr(status), _lib.ptr(ws), ws.numel(), _lib.stream(dev))


def kv4_fork(pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, ref_count: torch.Tensor,
             page_size: int, src: torch.Tensor, dst: torch.Tensor, *, share: bool = True,
             status: torch.Tensor | None = None) -> None:
    """The empty sequence dst[i] becomes what src[i] is.  share: it holds the same full pages, and a
    copy of the last one where that is not full, so either may grow; else it gets copies of all pages.
    A source may be named more than once, and in every layer of `pages` the same pages are copied."""
    what = "4-bit cache fork"
    dev = _lib.require_gpu(pages, block_table, lengths, ref_count, src, dst, status, what=what)
    sequences, wide = _check_metadata(block_table, lengths, ref_count, page_size, what)
    n = _named(src, "src", what)
    _int32(dst, (n,), "dst", what)
    _check_status(status, what)
    page, layer, layers = _layers(pages, ref_count.shape[0], what)
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev)
    with torch.cuda.device(dev):
        _lib.call("spr_kv4_fork", _lib.ptr(pages), page, layer, layers, _lib.ptr(block_table), _lib.ptr(lengths),
                  _lib.ptr(ref_count), _lib.ptr(src), _lib.ptr(dst), n, sequences, wide, page_size, ref_count.shape[0],
                  int(share), _lib.ptr(status), _lib.ptr(ws), ws.numel(), _lib.stream(dev))


def kv4_compact(pages: torch.Tensor, block_table: torch.Tensor, ref_count: torch.Tensor) -> torch.Tensor:
    """The held pages move down to 0 .. live - 1 (the i-th lowest one from `live` on to the i-th lowest
    free one below it), in every layer, the table and ref_count.  Returns live, int32 []: the pages from
    there on are free, and a pool cut to that many holds all sequences."""
    what = "4-bit cache compact"
    dev = _lib.require_gpu(pages, block_table, ref_count, what=what)
    sequences, wide = _check_metadata(block_table, None, ref_count, PAGE_SIZES[0], what)
    page, layer, layers = _layers(pages, ref_count.shape[0], what)
    live = torch.empty((), dtype=torch.int32, device=dev)
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev)
    with torch.cuda.device(dev):
        _lib.call("spr_kv4_compact", _lib.ptr(pages), page, layer, layers, _lib.ptr(block_table), _lib.ptr(ref_count),
                  sequences, wide, ref_count.shape[0], _lib.ptr(live), _lib.ptr(ws), ws.numel(), _lib.stream(dev))
    return live
