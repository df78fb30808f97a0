"""Timed cases of the 4-bit K/V cache: attention over its pages, rows written into them and read
back, sequences freed, forked and copied, pages moved together.

A cache is one uint8 tensor `pages` [num_pages, kv_heads, page_bytes].  A page holds `page_size`
tokens of every kv head; one head's part is the K codes [page_size, D / 2], the V codes
[page_size, D / 2], the K scales [page_size, D / 32] and the V scales [page_size, D / 32].  A code
is a 4-bit float (sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even dim in the low
half; a scale byte b stands for 2^(b - 127) and belongs to 32 dims of one token.  `block_table`
[sequences, max_pages] int32 names the pages of a sequence (-1: none), `lengths` its tokens and
`ref_count` the sequences that hold a page.

`own` False computes each operator from elementary torch operations in 32 bits; True calls the
library."""

import math

import numpy as np
import torch

own = False

GROUP = 32  # dims that share a scale
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a short prompt answered token by token: the latency of one call
        dict(name="attend token, short", op="attend", batch=1, heads=12, kv_heads=12, dim=64, rows=1, longest=301,
             page=32, causal=False, dtype="bf16", even=True),
        # one new row of every head against the whole video of 33 frames of 60 x 60 patches
        dict(name="attend token, whole video", op="attend", batch=1, heads=24, kv_heads=24, dim=128, rows=1,
             longest=118800, page=64, causal=False, dtype="bf16", even=True),
        # a serving step: ragged sequences, an empty one among them, four query heads to a kv head
        dict(name="attend token, 48 sequences", op="attend", batch=48, heads=32, kv_heads=8, dim=128, rows=1,
             longest=8191, page=64, causal=True, dtype="bf16", even=False),
        # 128 probe rows of every head against the whole video
        dict(name="attend probes, whole video", op="attend", batch=1, heads=24, kv_heads=24, dim=128, rows=128,
             longest=118800, page=128, causal=False, dtype="bf16", even=True),
        # ragged chunks of prompts behind their own cached prefix, causal, fp16, head dim 64
        dict(name="attend prompts, causal", op="attend", batch=5, heads=16, kv_heads=4, dim=64, rows=777,
             longest=4999, page=64, causal=True, dtype="fp16", even=False),
        # the next frame of a video against all frames before it and itself
        dict(name="attend frame, whole video", op="attend", batch=1, heads=24, kv_heads=24, dim=128, rows=3600,
             longest=118800, page=64, causal=False, dtype="bf16", even=True),
        # the new row of every sequence of a serving step, kept and read back
        dict(name="store tokens", op="store", batch=48, kv_heads=8, dim=128, rows=1, longest=8191, page=64,
             dtype="bf16", even=False, tokens_first=True),
        # a frame's K and V, as the projections leave them ([B, S, H, D]), kept and read back
        dict(name="store frame", op="store", batch=1, kv_heads=24, dim=128, rows=3600, longest=118800, page=64,
             dtype="bf16", even=True, tokens_first=True),
        # a beam step: the old beams go, each of the kept ones continues as four that share its pages
        dict(name="fork beams", op="fork", parents=4, children=16, kv_heads=8, dim=128, layers=2, longest=4001,
             page=64, share=True),
        # two guidance branches with pages of their own, one layer of a half video
        dict(name="copy branches", op="fork", parents=1, children=2, kv_heads=24, dim=128, layers=1, longest=59407,
             page=128, share=False),
        # a few short sequences left in a small pool
        dict(name="compact small pool", op="compact", batch=6, kv_heads=4, dim=64, layers=2, longest=700, page=32,
             held=0.4),
        # long sequences in a pool that is two fifths full
        dict(name="compact large pool", op="compact", batch=24, kv_heads=8, dim=128, layers=2, longest=16384,
             page=64, held=0.4),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "attend", "attend", "store", "store", "fork", "fork", "compact"])
    page, dim = rng.choice([32, 64, 128]), rng.choice([64, 128, 128])
    if op == "attend":
        while True:
            kv_heads = rng.choice([1, 2, 4, 8, 12, 24])
            heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
            batch, rows = _log_int(rng, 1, 64), rng.choice([1, _log_int(rng, 1, 64), _log_int(rng, 1, 3600)])
            longest = _log_int(rng, 40, 118800)
            # at most what one frame against the whole video costs, in the cache and in the products
            if batch * kv_heads * longest <= 4e6 and batch * heads * rows * longest <= 2.5e9:
                break
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, rows=rows, longest=longest, page=page,
                    causal=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16"]), even=rng.random() < 0.3)
    if op == "store":
        while True:
            kv_heads, batch = rng.choice([1, 2, 4, 8, 12, 24]), _log_int(rng, 1, 64)
            rows, longest = rng.choice([1, _log_int(rng, 1, 8000)]), _log_int(rng, 40, 60000)
            if rows <= longest and batch * kv_heads * longest <= 3e6 and batch * kv_heads * rows <= 4e5:
                break
        return dict(op=op, batch=batch, kv_heads=kv_heads, dim=dim, rows=rows, longest=longest, page=page,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), even=rng.random() < 0.3,
                    tokens_first=rng.random() < 0.5)
    if op == "fork":
        while True:
            parents, share = _log_int(rng, 1, 8), rng.random() < 0.5
            children = parents * rng.choice([1, 2, 3, 4])
            kv_heads, layers, longest = rng.choice([1, 4, 8, 24]), rng.choice([1, 2, 3]), _log_int(rng, 30, 60000)
            if (parents + children * (not share)) * kv_heads * layers * longest <= 4.2e6:
                break
        return dict(op=op, parents=parents, children=children, kv_heads=kv_heads, dim=dim, layers=layers,
                    longest=longest, page=page, share=share)
    while True:
        batch, kv_heads, layers = _log_int(rng, 1, 64), rng.choice([1, 4, 8, 24]), rng.choice([1, 2, 3])
        longest, held = _log_int(rng, 40, 20000), rng.uniform(0.15, 0.8)
        if batch * kv_heads * layers * longest / held <= 8e6:
            break
    return dict(op=op, batch=batch, kv_heads=kv_heads, dim=dim, layers=layers, longest=longest, page=page, held=held)


def _lengths_of(case, seed):
    """The tokens of each sequence: all `longest`, or spread over its logarithm with one at the
    top and, among four or more, one empty; the seed says which sequence has which."""
    n, top = case.get("batch", case.get("parents")), case["longest"]
    if case.get("even", False):
        return np.full(n, top, np.int64)
    low = max(1, top // 16)
    got = np.exp(np.random.RandomState(n).uniform(math.log(low), math.log(top + 1), n)).astype(np.int64).clip(1, top)
    got[0] = top
    if n >= 4 and case["op"] != "fork":
        got[1] = 0
    return np.random.RandomState(seed % (2**31)).permutation(got)


def _counts_of(case, lengths, seed):
    """The rows of each sequence in this call: all, or a part of them (none for an empty one)."""
    r = np.random.RandomState((seed + 17) % (2**31))
    full = np.full(len(lengths), case["rows"], np.int64)
    if not case["even"] and case["rows"] > 1:
        full = r.randint(1, case["rows"] + 1, len(lengths))
        full[int(np.argmax(lengths))] = case["rows"]
    return full


# ------------------------------------------------------------------ the format, plain


def _page_size(pages, dim):
    return pages.shape[-1] // (dim + dim // 16)


def _part(pages, dim, what):
    """A view of pages [..., page_bytes]: the codes or scales of K or V, [..., page_size, n]."""
    s = _page_size(pages, dim)
    at = {"k": (0, dim // 2), "v": (s * dim // 2, dim // 2), "ks": (s * dim, dim // GROUP),
          "vs": (s * dim + s * dim // GROUP, dim // GROUP)}[what]
    return pages[..., at[0]:at[0] + s * at[1]].unflatten(-1, (s, at[1]))


def _encode(x):
    """x [..., D] -> codes uint8 [..., D / 2], scales uint8 [..., D / 32]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1, keepdim=True).contiguous().view(torch.int32)
    byte = (((top + 0x200000) >> 23) - 2).clamp(2, 252)
    y = g.abs() * torch.exp2((127 - byte).float())
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)
            + torch.signbit(g).to(torch.uint8) * 8)
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | (code[..., 1] << 4), byte.squeeze(-1).to(torch.uint8)


def _decode(codes, scales):
    """The values, float32 [..., D]."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return (grid[both].unflatten(-1, (-1, GROUP)) * torch.exp2(scales.float() - 127).unsqueeze(-1)).flatten(-2)


def _rows_of(pages, table, dim, n):
    """K and V of the first n tokens of every row of table, float32 [B, H, n, D]."""
    held = pages[table[:, : -(-n // _page_size(pages, dim))].clamp(min=0).long()]  # [B, N, H, bytes]
    put = lambda c, s: _decode(_part(held, dim, c), _part(held, dim, s)).transpose(1, 2).flatten(2, 3)[:, :, :n]  # noqa: E731
    return put("k", "ks"), put("v", "vs")


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool(case, num_pages, gen, layers=None):
    """Pages of K and V rows as the projections give them: channels of unlike size, K above V."""
    dim, page, heads = case["dim"], case["page"], case["kv_heads"]
    pages = torch.zeros((layers or 1, num_pages, heads, page * (dim + dim // 16)), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (heads * page * dim))
    for layer in pages:
        for p in range(0, num_pages, step):
            n = min(step, num_pages - p)
            for c, s, spread in (("k", "ks", 0.6), ("v", "vs", 0.3)):
                width = torch.exp(spread * torch.randn((heads, 1, dim), generator=gen, device="cuda"))
                codes, scales = _encode(torch.randn((n, heads, page, dim), generator=gen, device="cuda") * width)
                _part(layer[p:p + n], dim, c).copy_(codes)
                _part(layer[p:p + n], dim, s).copy_(scales)
    return pages if layers else pages[0]


def _table(lengths, page, num_pages, max_pages, seed):
    """Each sequence's pages, in no order, and how many sequences hold each page."""
    r = np.random.RandomState((seed + 5) % (2**31))
    free, table, at = r.permutation(num_pages), np.full((len(lengths), max_pages), -1, np.int32), 0
    for i, n in enumerate(-(-lengths // page)):
        table[i, :n] = free[at:at + n]
        at += n
    refs = np.zeros(num_pages, np.int32)
    refs[free[:at]] = 1
    return table, refs


def _gpu(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def prepare(case, seed):
    op, page, dim = case["op"], case["page"], case["dim"]
    gen, lengths = _gen(seed), _lengths_of(case, seed)
    wide = -(-case["longest"] // page)
    state = dict(case=case, page_size=page, longest=case["longest"])
    if op in ("attend", "store"):
        num_pages = int((-(-lengths // page)).sum()) + 3
        table, _ = _table(lengths, page, num_pages, wide, seed)
        counts = _counts_of(case, lengths, seed)
        state |= dict(pages=_pool(case, num_pages, gen), table=_gpu(table), counts=_gpu(counts))
        if op == "attend":
            q = torch.randn((case["batch"], case["heads"], case["rows"], dim), generator=gen, device="cuda")
            state |= dict(q=(0.8 * q).to(TYPES[case["dtype"]]), lengths=_gpu(lengths))
        else:
            # the call writes the last rows of every sequence
            counts = np.minimum(counts, lengths)
            shape = (case["batch"], case["kv_heads"], case["rows"], dim)
            if case["tokens_first"]:
                shape = (shape[0], shape[2], shape[1], shape[3])
            k, v = (torch.randn(shape, generator=gen, device="cuda").to(TYPES[case["dtype"]]) for _ in range(2))
            k, v = (x.transpose(1, 2) if case["tokens_first"] else x for x in (k, v))
            state |= dict(k=k, v=v, counts=_gpu(counts), starts=_gpu(lengths - counts))
        return state
    if op == "fork":
        more = case["children"]
        per = -(-lengths // page)
        spare = more if case["share"] else int(per.sum()) * (more // case["parents"])
        num_pages = int(per.sum()) + spare + 2
        table, refs = _table(lengths, page, num_pages, wide, seed)
        table = np.concatenate([table, np.full((more, wide), -1, np.int32)])
        lengths = np.concatenate([lengths, np.zeros(more, np.int64)])
        state |= dict(src=_gpu(np.arange(more) % case["parents"]), dst=_gpu(case["parents"] + np.arange(more)),
                      share=case["share"])
    else:
        num_pages = int((-(-lengths // page)).sum() / case["held"]) + 1
        table, refs = _table(lengths, page, num_pages, wide, seed)
    return state | dict(pages=_pool(case, num_pages, gen, case["layers"]), table=_gpu(table), lengths=_gpu(lengths),
                        refs=_gpu(refs), table0=_gpu(table), lengths0=_gpu(lengths), refs0=_gpu(refs))


# ------------------------------------------------------------------ the operators, plain


def _attend(state):
    case, q, lengths, counts = state["case"], state["q"], state["lengths"].long(), state["counts"].long()
    b, h, t, d = q.shape
    k, v = _rows_of(state["pages"], state["table"], d, state["longest"])
    hk, n = k.shape[1], k.shape[2]
    s = (q.float() * (1.0 / math.sqrt(d))).reshape(b, hk, -1, d) @ k.transpose(2, 3)
    s = s.view(b, h, t, n)
    row, key = torch.arange(t, device=q.device), torch.arange(n, device=q.device)
    end = lengths[:, None].expand(b, t)
    if case["causal"]:
        end = end - counts[:, None] + row + 1
    end = torch.where(row < counts[:, None], end, 0)
    if not case["even"] or case["causal"]:
        s.masked_fill_((key >= end[:, :, None])[:, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3.0e38)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, hk, -1, n) @ v).view(b, h, t, d) / total.clamp(min=1e-37)
    return out.to(q.dtype), (top + total.log()).squeeze(-1)


def _store_and_load(state):
    pages, table, k, v = state["pages"], state["table"], state["k"], state["v"]
    starts, counts = state["starts"].long(), state["counts"].long()
    b, h, t, d = k.shape
    size = _page_size(pages, d)
    row = torch.arange(t, device=k.device)
    live = row < counts[:, None]  # [B, T]
    at = (starts[:, None] + row).clamp(max=table.shape[1] * size - 1)
    page, slot = table.long().gather(1, at // size), at % size
    back = []
    for x, c, s in ((k, "k", "ks"), (v, "v", "vs")):
        codes, scales = _encode(x.transpose(1, 2)[live])  # [M, H, .]
        _part(pages, d, c).transpose(1, 2)[page[live], slot[live]] = codes
        _part(pages, d, s).transpose(1, 2)[page[live], slot[live]] = scales
        got = torch.zeros((b, t, h, d), device=k.device)
        got[live] = _decode(_part(pages, d, c).transpose(1, 2)[page[live], slot[live]],
                            _part(pages, d, s).transpose(1, 2)[page[live], slot[live]])
        back.append(got.transpose(1, 2).contiguous().to(k.dtype))
    return back


def _free_and_fork(state):
    """The children's pages are given back, then every child i becomes a copy of src[i]: its full
    pages are the parent's own (share) or new ones, its last page, where it is not full, a new one.
    New pages are the lowest free ones, in the children's order."""
    pages, table, lengths, refs = state["pages"], state["table"], state["lengths"], state["refs"]
    src, dst, size = state["src"].long(), state["dst"].long(), state["page_size"]
    wide = table.shape[1]
    col = torch.arange(wide, device=table.device)
    gone = table[dst]
    refs.index_add_(0, gone.clamp(min=0).flatten().long(), -(gone >= 0).flatten().int())
    n = lengths[src].long()
    full = n // size if state["share"] else torch.zeros_like(n)
    every = (n + size - 1) // size
    need = every - full
    order = torch.argsort((refs != 0).int(), stable=True)  # free pages first, ascending
    first = need.cumsum(0) - need
    parent = table[src].long()
    new = (col >= full[:, None]) & (col < every[:, None])
    fresh = order[(first[:, None] + col - full[:, None]).clamp(0, len(order) - 1)]
    child = torch.where(new, fresh, torch.where(col < every[:, None], parent, -1))
    pages[:, child[new]] = pages[:, parent[new]]
    refs.index_add_(0, child.clamp(min=0).flatten(), (child >= 0).flatten().int())
    table[dst], lengths[dst] = child.int(), lengths[src]
    return table, lengths, refs, pages


def _compact(state):
    """The i-th lowest held page whose number is not below the count of held pages moves to the
    i-th lowest free page whose number is."""
    pages, table, refs = state["pages"], state["table"], state["refs"]
    held = refs > 0
    count = held.sum()
    number = torch.arange(len(refs), device=refs.device)
    low = number < count
    source, hole = number[held & ~low], number[~held & low]
    place = number.clone()
    place[source] = hole
    pages[:, hole] = pages[:, source]
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()].int(), table))
    refs[hole] = refs[source]
    refs[source] = 0
    return table, state["lengths"], refs, count.int(), pages


def run(state):
    op = state["case"]["op"]
    if op == "attend":
        if own:
            from sparsepr_amd.kernels.kv4 import kv4_attention

            return kv4_attention(state["q"], state["pages"], state["table"], state["lengths"], counts=state["counts"],
                                 causal=state["case"]["causal"], max_length=state["longest"], return_lse=True)
        return _attend(state)
    if op == "store":
        if own:
            from sparsepr_amd.kernels.kv4 import kv4_load, kv4_store

            k = state["k"]
            kv4_store(state["pages"], state["table"], k, state["v"], state["starts"], counts=state["counts"])
            return kv4_load(state["pages"], state["table"], state["starts"], state["counts"], k.shape[2], k.shape[3],
                            dtype=k.dtype)
        return _store_and_load(state)
    if op == "fork":
        if own:
            from sparsepr_amd.kernels.kv4 import kv4_fork, kv4_free

            pages, table, lengths, refs = state["pages"], state["table"], state["lengths"], state["refs"]
            kv4_free(table, lengths, refs, state["page_size"], state["dst"])
            kv4_fork(pages, table, lengths, refs, state["page_size"], state["src"], state["dst"],
                     share=state["share"])
            return table, lengths, refs, pages
        return _free_and_fork(state)
    # the same scattered pages are moved together in every pass
    for name in ("table", "lengths", "refs"):
        state[name].copy_(state[name + "0"])
    if own:
        from sparsepr_amd.kernels.kv4 import kv4_compact

        count = kv4_compact(state["pages"], state["table"], state["refs"])
        return state["table"], state["lengths"], state["refs"], count, state["pages"]
    return _compact(state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    dim, page = case["dim"], case["page"]
    row = dim + dim // 16  # bytes of one token's K and V of one head in the cache
    lengths = _lengths_of(case, 1)
    if case["op"] == "attend":
        counts, bits = _counts_of(case, lengths, 1), 2
        pairs, keys = 0, 0
        for n, t in zip(lengths.tolist(), counts.tolist()):
            if case["causal"]:
                first = max(0, t - n)  # rows that see nothing
                seen = t - first
                pairs += seen * n - seen * (seen - 1) // 2
            else:
                pairs += t * n
            keys += n
        return {"bytes": keys * case["kv_heads"] * row + int(counts.sum()) * case["heads"] * (2 * bits * dim + 4),
                "flops": 4 * dim * case["heads"] * pairs}
    if case["op"] == "store":
        rows = int(np.minimum(_counts_of(case, lengths, 1), lengths).sum()) * case["kv_heads"]
        wide = TYPES[case["dtype"]].itemsize * 2 * dim
        return {"bytes": 2 * rows * (wide + row), "flops": 0}
    page_bytes = case["layers"] * case["kv_heads"] * page * row
    per = -(-lengths // page)
    if case["op"] == "fork":
        each = case["children"] // case["parents"]
        moved = each * int((lengths % page > 0).sum() if case["share"] else per.sum())
        return {"bytes": 2 * moved * page_bytes + 12 * each * int(per.sum()), "flops": 0}
    held = int(per.sum())
    num_pages = int(held / case["held"]) + 1
    moved = held * (1 - held / num_pages)  # on average, for pages in no order
    return {"bytes": 2 * int(moved) * page_bytes + 8 * num_pages + 8 * held, "flops": 0}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    size, dim = state["page_size"], case["dim"]
    pages, table = state["pages"], state["table"].cpu().numpy()
    half = size * dim // 2

    def values(page, where, scales):
        """[..., size, dim] float64 of a head's part of a page: where and scales are byte offsets."""
        raw = page[..., where:where + half].reshape(*page.shape[:-1], size, dim // 2)
        bits = torch.stack([raw % 16, raw // 16], -1).reshape(*raw.shape[:-1], dim).double()
        neg, mag = bits >= 8, bits % 8
        exponent, mantissa = torch.div(mag, 2, rounding_mode="floor"), mag % 2
        value = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * 2.0 ** (exponent - 1))
        scale = page[..., scales:scales + size * dim // 32].reshape(*page.shape[:-1], size, dim // 32).double()
        return torch.where(neg, -value, value) * (2.0 ** (scale - 127)).repeat_interleave(32, -1)

    if case["op"] == "attend":
        q, group = state["q"], case["heads"] // case["kv_heads"]
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
        for b, (n, t) in enumerate(zip(state["lengths"].tolist(), state["counts"].tolist())):
            if n == 0:
                continue
            ids = torch.from_numpy(table[b, : -(-n // size)].astype(np.int64)).cuda()
            for hk in range(case["kv_heads"]):
                mine = pages[ids, hk]
                k = values(mine, 0, 2 * half).reshape(-1, dim)[:n]
                v = values(mine, half, 2 * half + size * dim // 32).reshape(-1, dim)[:n]
                for h in range(hk * group, (hk + 1) * group):
                    s = (q[b, h, :t].double() @ k.T) / math.sqrt(dim)
                    if case["causal"]:
                        last = n - t + torch.arange(t, device="cuda")
                        s[torch.arange(n, device="cuda")[None, :] > last[:, None]] = -math.inf
                    lse[b, h, :t] = torch.logsumexp(s, -1)
                    seen = lse[b, h, :t] > -math.inf
                    out[b, h, :t][seen] = torch.exp(s[seen] - lse[b, h, :t][seen, None]) @ v
        return out, lse
    if case["op"] == "store":
        got = []
        for x in (state["k"], state["v"]):
            g = x.double().reshape(*x.shape[:-1], dim // 32, 32)
            top = g.abs().amax(-1, keepdim=True)
            # the exponent of the largest value rounded to two binary digits, half up
            part, e = torch.frexp(top)
            e = (e - 1 + (part >= 0.875).int()).double()
            scale = 2.0 ** (e - 2).clamp(-125, 125)
            grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
            y = (g.abs() / scale).unsqueeze(-1)
            off = (y - grid).abs()
            # the nearest value, of two equally near ones that with an even code
            pick = (off * 4 + torch.tensor([0, 1, 0, 1, 0, 1, 0, 1], device="cuda") * 1e-9).argmin(-1)
            got.append((torch.copysign(grid[pick] * scale, g)).reshape(x.shape))
        live = torch.arange(case["rows"], device="cuda") < state["counts"][:, None]
        return [torch.where(live[:, None, :, None], x, 0.0) for x in got]
    lengths, refs = state["lengths"].cpu().numpy(), state["refs"].cpu().numpy()
    if case["op"] == "fork":
        free = [p for p in range(len(refs)) if refs[p] == 0]
        moves = []
        for s, d in zip(state["src"].tolist(), state["dst"].tolist()):
            lengths[d] = lengths[s]
            for j in range(-(-int(lengths[s]) // size)):
                page = int(table[s, j])
                if not state["share"] or (j + 1) * size > lengths[s]:
                    moves.append((page, free[0]))
                    page = free.pop(0)
                table[d, j] = page
                refs[page] += 1
        for a, b in moves:
            pages[:, b] = pages[:, a]
        return [torch.from_numpy(x.astype(np.int32)) for x in (table, lengths, refs)] + [pages]
    count = int((refs > 0).sum())
    holes = [p for p in range(count) if refs[p] == 0]
    place = {}
    for p in range(count, len(refs)):
        if refs[p]:
            place[p] = holes[len(place)]
    for a, b in place.items():
        pages[:, b] = pages[:, a]
        refs[b], refs[a] = refs[a], 0
    table = np.array([[place.get(int(p), int(p)) for p in line] for line in table])
    return [torch.from_numpy(x.astype(np.int32)) for x in (table, lengths, refs)] + [torch.tensor(count, dtype=torch.int32), pages]
