"""A paged K/V cache held in 4 bits: attention over it, rows stored and loaded, pages reserved,
freed, forked and moved together, on the HIP kernels of csrc/spr_kv4.hip and
csrc/spr_kv4_attention.hip.  `sparsepr_amd.kv4_cache.KV4Cache` keeps the tensors these functions
take.

pages        uint8 [P, Hkv, page_bytes], or [layers, P, Hkv, page_bytes] for the page calls: pages of
             page_size tokens, K and V as 4-bit floats with one power-of-two scale per 32 dims
             (kv4_page_bytes; D + D / 16 bytes a token and kv head, against 4 D in bf16).  What slots
             without a token hold does not matter, so a pool need not be cleared.
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
    3: "a negative count or one past the rows given, or a range outside the sequence's pages",
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


def _page_size(pages: torch.Tensor, head_dim: int, page_size: int | None, what: str) -> int:
    """Tokens of a page, from the pages of one layer and the head dim; `page_size`, if the caller gives it."""
    shape = pages.shape
    if pages.dtype is not torch.uint8 or len(shape) != 3 or not pages.is_contiguous() or pages.numel() == 0:
        raise RuntimeError(f"{what}: pages must be a contiguous uint8 tensor [P, Hkv, bytes], got {pages.dtype} "
                           f"{tuple(shape)}")
    if head_dim not in HEAD_DIMS:
        raise RuntimeError(f"{what}: head dim {head_dim} not supported {HEAD_DIMS}")
    size = shape[2] // (head_dim + head_dim // 16)
    if size not in PAGE_SIZES or shape[2] != size * (head_dim + head_dim // 16):
        raise RuntimeError(f"{what}: pages of {shape[2]} bytes a head are not whole pages of head dim {head_dim}")
    if page_size is not None and size != page_size:
        raise RuntimeError(f"{what}: pages of {shape[2]} bytes a head are not {page_size} tokens of head dim {head_dim}")
    return size


def _int32(t: torch.Tensor, n: int, name: str, what: str) -> None:
    """An int32 vector of n, as the kernels read it."""
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be a contiguous int32 tensor of shape {(n,)}, got {t.dtype} "
                           f"{tuple(t.shape)}")


def _check_table(block_table: torch.Tensor, what: str) -> tuple[int, int]:
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or not block_table.is_contiguous():
        raise RuntimeError(f"{what}: block_table must be a contiguous int32 tensor [sequences, wide], got "
                           f"{block_table.dtype} {tuple(block_table.shape)}")
    return block_table.shape


def _check_entries(batch: int, sequences: int, seq_ids, counts, what: str) -> None:
    if seq_ids is not None:
        _int32(seq_ids, batch, "seq_ids", what)
    elif batch > sequences:
        raise RuntimeError(f"{what}: a batch of {batch} without seq_ids on a table of {sequences} sequences")
    if counts is not None:
        _int32(counts, batch, "counts", what)


def _by_rows(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """x [B, H, T, D] and the strides of its first three dims: itself where rows are packed and 16-byte
    aligned, else a copy."""
    (b, h, t, d), (sb, sh, st, sd) = x.shape, x.stride()
    if b == 1:
        sb = 0
    if h == 1:
        sh = 0
    if t == 1:
        st = 0
    if sd == 1 and x.data_ptr() % 16 == 0 and (sb | sh | st) * x.element_size() % 16 == 0:
        return x, sb, sh, st
    # (contiguous() hands packed rows that start off 16 bytes back as they are)
    return x.clone(memory_format=torch.contiguous_format), h * t * d, t * d, d


def store_call(pages: torch.Tensor, block_table: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
               counts: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None, page_size: int | None = None):
    """Everything of kv4_store but the starts checked, as a function of them: whoever reserves first has
    no refusal to expect after it."""
    what = "4-bit cache store"
    dev = _lib.require_gpu(pages, block_table, k, v, counts, seq_ids, what=what)
    if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or k.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: K and V must be [B, Hkv, T, D] of one dtype (bfloat16, float16, float32), got "
                           f"{k.dtype} {tuple(k.shape)} / {v.dtype} {tuple(v.shape)}")
    b, h, t, d = k.shape
    size = _page_size(pages, d, page_size, what)
    if pages.shape[1] != h:
        raise RuntimeError(f"{what}: K has {h} heads, the pages {pages.shape[1]}")
    sequences, wide = _check_table(block_table, what)
    _check_entries(b, sequences, seq_ids, counts, what)
    if h * t * (d // 8) > 2**32 - 256:  # threads of a launch
        raise RuntimeError(f"{what}: {t} rows of {h} heads are too many for one call")
    code, live = _lib.DTYPE_CODE[k.dtype], k.numel() > 0
    k, *k_strides = _by_rows(k)
    v, *v_strides = _by_rows(v)

    def put(starts: torch.Tensor) -> None:
        _lib.require_gpu(pages, starts, what=what)
        _int32(starts, b, "starts", what)
        if live:
            _lib.launch("spr_kv4_store", dev, pages.data_ptr(), pages.shape[0], h, size, d, block_table.data_ptr(),
                        sequences, wide, _lib.ptr(seq_ids), starts.data_ptr(), _lib.ptr(counts), k.data_ptr(),
                        v.data_ptr(), code, b, t, *k_strides, *v_strides)

    return put


def kv4_store(pages: torch.Tensor, block_table: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
              *, counts: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None,
              page_size: int | None = None) -> None:
    """Write K and V rows [B, Hkv, T, D] (bf16, fp16 or fp32, any strides with packed rows) to the
    cache: row t < counts[b] becomes token starts[b] + t of sequence seq_ids[b] (default b).

    The pages have to be there (kv4_reserve): rows without one are not written.  No two rows of a call
    may name one token, and no other sequence may share the page written to (kv4_fork sees to that).
    A group of 32 dims with an infinity or a NaN is stored as NaN.  `page_size` is for the caller's
    check of what it hands over: a page of 2 n tokens of head dim 64 has the bytes of n of 128."""
    store_call(pages, block_table, k, v, counts=counts, seq_ids=seq_ids, page_size=page_size)(starts)


def kv4_load(pages: torch.Tensor, block_table: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor, rows: int,
             head_dim: int, *, seq_ids: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
             page_size: int | None = None):
    """Tokens starts[b] .. starts[b] + counts[b] - 1 of every named sequence as (K, V) [B, Hkv, rows, D]
    in `dtype` (exact in bf16 and fp32); rows past the count are 0, rows with no page NaN.  `page_size` is
    checked, as in kv4_store."""
    what = "4-bit cache load"
    dev = _lib.require_gpu(pages, block_table, starts, counts, seq_ids, what=what)
    size = _page_size(pages, head_dim, page_size, what)
    if dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"{what}: dtype must be bfloat16, float16 or float32, got {dtype}")
    if rows < 0 or starts.dim() != 1:
        raise RuntimeError(f"{what}: rows {rows}, starts {tuple(starts.shape)}")
    b, h = starts.shape[0], pages.shape[1]
    sequences, wide = _check_table(block_table, what)
    _check_entries(b, sequences, seq_ids, counts, what)
    _int32(starts, b, "starts", what)
    k = pages.new_empty((b, h, rows, head_dim), dtype=dtype)
    v = torch.empty_like(k)
    if k.numel() > 0:
        _lib.launch("spr_kv4_load", dev, pages.data_ptr(), pages.shape[0], h, size, head_dim, block_table.data_ptr(),
                    sequences, wide, _lib.ptr(seq_ids), starts.data_ptr(), counts.data_ptr(), k.data_ptr(),
                    v.data_ptr(), _lib.DTYPE_CODE[dtype], b, rows)
    return k, v


def kv4_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
                  counts: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None, causal: bool = False,
                  scale: float | None = None, max_length: int | None = None, return_lse: bool = False,
                  page_size: int | None = None):
    """softmax(q K^T * scale) V over the cached tokens: q [B, Hq, T, D] bf16 or fp16 (any strides with
    packed rows) -> out [B, Hq, T, D] in q's dtype (and lse fp32 [B, Hq, T], natural log).

    Hq is a multiple of Hkv; query head h reads kv head h // (Hq // Hkv).  Batch entry b attends
    sequence seq_ids[b] (default b) with its first counts[b] rows (default all).  With `causal` the last
    row in use is the sequence's last token and each row sees the tokens up to its own (store them
    first).  Rows that see nothing, and rows past the count, are 0 with lse -inf.  `max_length`, the
    longest length the caller knows of (default: what the table can hold), only sizes the launch and its
    workspace, and may be passed: the keys are dealt by the lengths as they are.  `page_size` is checked,
    as in kv4_store.

    Sums, maxima and scores are fp32.  Probabilities keep 16 bits into the product with V in fp16 calls and
    in bf16 calls of up to 8 rows (T * Hq // Hkv); in longer bf16 calls they are rounded to bf16 once.  A
    row whose scores are all -inf is NaN."""
    what = "4-bit cache attention"
    dev = _lib.require_gpu(q, pages, block_table, lengths, counts, seq_ids, what=what)
    if q.dim() != 4 or q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"{what}: q must be [B, Hq, T, D] in bfloat16 or float16, got {q.dtype} {tuple(q.shape)}")
    b, h, t, d = q.shape
    size = _page_size(pages, d, page_size, what)
    hk = pages.shape[1]
    if h == 0 or h % hk != 0:
        raise RuntimeError(f"{what}: Q heads ({h}) must be a multiple of KV heads ({hk})")
    sequences, wide = _check_table(block_table, what)
    _check_entries(b, sequences, seq_ids, counts, what)
    _int32(lengths, sequences, "lengths", what)
    longest = wide * size if max_length is None else min(int(max_length), wide * size)
    sc = float(scale) if scale is not None else 1.0 / math.sqrt(d)
    out = q.new_empty((b, h, t, d))
    lse = q.new_empty((b, h, t), dtype=torch.float32) if return_lse else None
    if out.numel() > 0:
        q, *strides = _by_rows(q)
        need = _lib.query("spr_kv4_attention_workspace", b, h, hk, t, d, longest)
        ws = _lib.workspace(need, dev) if need > 0 else None
        _lib.launch("spr_kv4_attention", dev, q.data_ptr(), *strides, _lib.DTYPE_CODE[q.dtype], b, h, hk, t, d,
                    pages.data_ptr(), pages.shape[0], size, block_table.data_ptr(), sequences, wide, lengths.data_ptr(),
                    _lib.ptr(counts), _lib.ptr(seq_ids), int(causal), sc, longest, out.data_ptr(), _lib.ptr(lse),
                    _lib.ptr(ws), need)
    return (out, lse) if return_lse else out


def _check_metadata(block_table, lengths, ref_count, page_size, status, what):
    sequences, wide = _check_table(block_table, what)
    if lengths is not None:
        _int32(lengths, sequences, "lengths", what)
    if ref_count.dim() != 1 or ref_count.shape[0] == 0:
        raise RuntimeError(f"{what}: ref_count must be [P], got {tuple(ref_count.shape)}")
    _int32(ref_count, ref_count.shape[0], "ref_count", what)
    if page_size not in PAGE_SIZES:
        raise RuntimeError(f"{what}: page size {page_size} not supported {PAGE_SIZES}")
    if status is not None:
        _int32(status, 1, "status", what)
    return sequences, wide


def _named(ids: torch.Tensor, name: str, what: str) -> int:
    if ids.dim() != 1 or ids.shape[0] > MAX_NAMED:
        raise RuntimeError(f"{what}: {name} must be a vector of at most {MAX_NAMED}, got {tuple(ids.shape)}")
    _int32(ids, ids.shape[0], name, what)
    return ids.shape[0]


def _layers(pages: torch.Tensor, num_pages: int, what: str) -> tuple[int, int, int]:
    """(bytes of a page, bytes from layer to layer, layers) of [P, H, bytes] or [layers, P, H, bytes]."""
    shape = pages.shape if pages.dim() == 4 else (1, *pages.shape)
    if pages.dtype is not torch.uint8 or len(shape) != 4 or pages.numel() == 0 or not pages.is_contiguous():
        raise RuntimeError(f"{what}: pages must be a contiguous uint8 tensor [P, Hkv, bytes] or [layers, P, Hkv, "
                           f"bytes], got {pages.dtype} {tuple(pages.shape)}")
    if shape[1] != num_pages:
        raise RuntimeError(f"{what}: {shape[1]} pages, ref_count of {num_pages}")
    page = shape[2] * shape[3]
    if page % 16 != 0:
        raise RuntimeError(f"{what}: pages of {shape[2]} x {shape[3]} bytes are not whole 16-byte pieces")
    return page, page * num_pages, shape[0]


def kv4_reserve(block_table: torch.Tensor, lengths: torch.Tensor, ref_count: torch.Tensor, page_size: int,
                counts: torch.Tensor, *, seq_ids: torch.Tensor | None = None,
                status: torch.Tensor | None = None, most: int | None = None) -> torch.Tensor:
    """Room for counts[i] more tokens of sequence seq_ids[i] (default i): new pages (the lowest free
    ones) in its row of the table, the length with them.  Returns starts int32 [n], the place of the
    first new token of each, or -1 for all when the call could not happen, as where a count passes
    `most`."""
    what = "4-bit cache reserve"
    dev = _lib.require_gpu(block_table, lengths, ref_count, counts, seq_ids, status, what=what)
    sequences, wide = _check_metadata(block_table, lengths, ref_count, page_size, status, what)
    n = _named(counts, "counts", what)
    _check_entries(n, sequences, seq_ids, None, what)
    starts = counts.new_empty(n)
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev)
    _lib.launch("spr_kv4_reserve_ex", dev, block_table.data_ptr(), lengths.data_ptr(), ref_count.data_ptr(),
                counts.data_ptr(), _lib.ptr(seq_ids), n, 2**31 - 1 if most is None else most, sequences, wide,
                page_size, ref_count.shape[0], starts.data_ptr(), _lib.ptr(status), ws.data_ptr(), ws.numel())
    return starts


def kv4_free(block_table: torch.Tensor, lengths: torch.Tensor, ref_count: torch.Tensor, page_size: int,
             seq_ids: torch.Tensor, *, first_pages: torch.Tensor | None = None,
             page_counts: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """The named sequences give their pages back and are empty; or only page_counts[i] pages from the
    first_pages[i]-th on (default 0, and all from there on), as a sliding window does: the pages behind
    close up and the length loses the tokens that lay there.  A page is free when nobody holds it."""
    what = "4-bit cache free"
    dev = _lib.require_gpu(block_table, lengths, ref_count, seq_ids, first_pages, page_counts, status, what=what)
    sequences, wide = _check_metadata(block_table, lengths, ref_count, page_size, status, what)
    n = _named(seq_ids, "seq_ids", what)
    for t, name in ((first_pages, "first_pages"), (page_counts, "page_counts")):
        if t is not None:
            _int32(t, n, name, what)
    # up to 64 sequences are one launch, which hands nothing on
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev) if n > 64 else None
    _lib.launch("spr_kv4_free", dev, block_table.data_ptr(), lengths.data_ptr(), ref_count.data_ptr(),
                seq_ids.data_ptr(), _lib.ptr(first_pages), _lib.ptr(page_counts), n, sequences, wide, page_size,
                ref_count.shape[0], _lib.ptr(status), _lib.ptr(ws), 0 if ws is None else ws.numel())


def kv4_fork(pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, ref_count: torch.Tensor,
             page_size: int, src: torch.Tensor, dst: torch.Tensor, *, share: bool = True,
             status: torch.Tensor | None = None) -> None:
    """The empty sequence dst[i] becomes what src[i] is.  share: it holds the same full pages, and a
    copy of the last one where that is not full, so either may grow; else it gets copies of all pages.
    A source may be named more than once, and in every layer of `pages` the same pages are copied."""
    what = "4-bit cache fork"
    dev = _lib.require_gpu(pages, block_table, lengths, ref_count, src, dst, status, what=what)
    sequences, wide = _check_metadata(block_table, lengths, ref_count, page_size, status, what)
    n = _named(src, "src", what)
    _int32(dst, n, "dst", what)
    page, layer, layers = _layers(pages, ref_count.shape[0], what)
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev)
    _lib.launch("spr_kv4_fork", dev, pages.data_ptr(), page, layer, layers, block_table.data_ptr(), lengths.data_ptr(),
                ref_count.data_ptr(), src.data_ptr(), dst.data_ptr(), n, sequences, wide, page_size,
                ref_count.shape[0], int(share), _lib.ptr(status), ws.data_ptr(), ws.numel())


def kv4_compact(pages: torch.Tensor, block_table: torch.Tensor, ref_count: torch.Tensor) -> torch.Tensor:
    """The held pages move down to 0 .. live - 1 (the i-th lowest one from `live` on to the i-th lowest
    free one below it), in every layer, the table and ref_count.  Returns live, int32 []: the pages from
    there on are free, and a pool cut to that many holds all sequences."""
    what = "4-bit cache compact"
    dev = _lib.require_gpu(pages, block_table, ref_count, what=what)
    sequences, wide = _check_metadata(block_table, None, ref_count, PAGE_SIZES[0], None, what)
    page, layer, layers = _layers(pages, ref_count.shape[0], what)
    live = ref_count.new_empty(())
    ws = _lib.workspace(_lib.query("spr_kv4_pages_workspace", ref_count.shape[0]), dev)
    _lib.launch("spr_kv4_compact", dev, pages.data_ptr(), page, layer, layers, block_table.data_ptr(),
                ref_count.data_ptr(), sequences, wide, ref_count.shape[0], live.data_ptr(), ws.data_ptr(), ws.numel())
    return live
