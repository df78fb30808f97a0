"""The 4-bit paged K/V cache on the GPU against its definitions in 64 bits."""

import math

import numpy as np
import pytest
import torch

from tests import _kv4_model as model

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gpu(a, dev, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).to(dev)


def _pool(rng, num_pages, heads, size, d, amp=1.0):
    """Pages of rows as the encoder makes them, uint8 numpy, and every byte of them in use."""
    pages = np.zeros((num_pages, heads, size * (d + d // 16)), np.uint8)
    kc, vc, ks, vs = model.parts(pages, size, d)
    for c, s, a in ((kc, ks, amp), (vc, vs, 1.0)):
        codes, scales = model.encode(rng.standard_normal((num_pages, heads, size, d)) * a)
        c[...], s[...] = codes, scales
    return pages


def _table(rng, lengths, size, num_pages, wide):
    order, at = rng.permutation(num_pages), 0
    table = np.full((len(lengths), wide), -1, np.int32)
    for i, n in enumerate(lengths):
        k = -(-n // size)
        table[i, :k] = order[at:at + k]
        at += k
    return table


def _same_nan(got, want):
    return np.array_equal(np.isnan(got), np.isnan(want))


# ------------------------------------------------------------------ rows in and out


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,size", [(64, 32), (128, 64), (128, 256)])
def test_store_bytes_are_the_encoders_and_load_gives_their_values(dev, dtype, d, size):
    from sparsepr_amd.kernels.kv4 import kv4_load, kv4_store

    rng = np.random.default_rng(d + size)
    b, h, t = 3, 2, 77
    x = rng.standard_normal((2, b, h, t, d)) * np.exp(2.5 * rng.standard_normal((2, b, h, t, 1)))
    x[0, 0, 0, 0] = 0.0
    x[0, 0, 0, 1, :32] = -0.0
    # values on the borders between codes, of every sign, at three scales
    edge = np.array([0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 6.96875, 7.0, 7.5])
    for i, s in enumerate((1.0, 2.0**-9, 2.0**6)):
        x[0, 0, 1, i, :34] = np.concatenate([edge, -edge]) * s
        x[1, 0, 1, i, :34] = np.concatenate([-edge, edge]) * s * 0.5
    # largest and smallest magnitudes of the type, and a group that passes the scale's range
    big = float(torch.finfo(DT[dtype]).max)
    x[0, 1, 0, 0, 0], x[0, 1, 0, 1, 3], x[0, 1, 0, 2, :] = big, -big, float(torch.finfo(DT[dtype]).tiny)
    x[1, 1, 0, 0, 5] = float(torch.finfo(DT[dtype]).tiny) * 2.0**-6
    x[1, 1, 1, 0, 7], x[1, 1, 1, 1, 40], x[1, 1, 1, 2, 1] = np.inf, -np.inf, np.nan
    k, v = (torch.from_numpy(y).to(DT[dtype]).to(dev) for y in x)
    lengths = [200, 0, 130]
    starts, counts = np.array([123, 0, 53]), np.array([t, 0, t])
    wide = 300 // size + 1
    num_pages = 2 * wide + 3
    table = _table(rng, [wide * size, 0, wide * size], size, num_pages, wide)
    table[1] = -1
    pages = rng.integers(0, 256, (num_pages, h, size * (d + d // 16)), np.uint8)
    want = pages.copy()
    for s in (0, 2):
        for name, y, (ci, si) in (("k", k, (0, 2)), ("v", v, (1, 3))):
            codes, scales = model.encode(y[s].double().cpu().numpy())
            for i in range(t):
                page, slot = table[s, (starts[s] + i) // size], (starts[s] + i) % size
                model.parts(want[page], size, d)[ci][:, slot] = codes[:, i]
                model.parts(want[page], size, d)[si][:, slot] = scales[:, i]
    gp, gt = _gpu(pages, dev, torch.uint8), _gpu(table, dev)
    kv4_store(gp, gt, k, v, _gpu(starts, dev), counts=_gpu(counts, dev))
    assert np.array_equal(gp.cpu().numpy(), want)  # its own rows, and no other byte
    for out in (torch.bfloat16, torch.float32, torch.float16):
        gk, gv = kv4_load(gp, gt, _gpu(starts, dev), _gpu(counts, dev), t, d, dtype=out)
        for got, y in ((gk, k), (gv, v)):
            ref = model.decode(*model.encode(y.double().cpu().numpy()))
            ref[1] = 0.0
            want_t = torch.from_numpy(ref).to(out)  # exact in bf16 and fp32; fp16 rounds and overflows as torch does
            assert _same_nan(got.double().cpu().numpy(), want_t.double().numpy())
            assert torch.equal(torch.nan_to_num(got.cpu(), nan=0.0, posinf=9e4, neginf=-9e4),
                               torch.nan_to_num(want_t, nan=0.0, posinf=9e4, neginf=-9e4))


def test_store_reads_strided_rows_in_place_and_odd_ones_by_copy(dev):
    from sparsepr_amd.kernels.kv4 import kv4_load, kv4_store

    rng = np.random.default_rng(5)
    b, h, t, d, size = 2, 3, 40, 64, 32
    table = _table(rng, [64, 64], size, 5, 2)
    zero, cnt = torch.zeros(b, dtype=torch.int32, device=dev), torch.full((b,), t, dtype=torch.int32, device=dev)
    base = torch.randn((b, t, h, d), device=dev).to(torch.bfloat16)
    odd = torch.randn((b, h, t, d + 1), device=dev).to(torch.bfloat16)[..., 1:]  # rows off 16 bytes
    flipped = torch.randn((b, h, d, t), device=dev).to(torch.bfloat16).transpose(2, 3)  # rows not packed
    one = torch.randn((b, 1, t, d), device=dev).to(torch.bfloat16).expand(b, h, t, d)  # one head for all
    for k, v in ((base.transpose(1, 2), odd), (flipped, one)):
        pages = torch.zeros((5, h, size * (d + d // 16)), dtype=torch.uint8, device=dev)
        kv4_store(pages, _gpu(table, dev), k, v, zero)
        gk, gv = kv4_load(pages, _gpu(table, dev), zero, cnt, t, d)
        for got, x in ((gk, k), (gv, v)):
            ref = model.decode(*model.encode(x.double().cpu().numpy()))
            assert np.array_equal(got.double().cpu().numpy(), ref)


def test_rows_without_a_page_are_not_written_and_read_as_nan(dev):
    from sparsepr_amd.kernels.kv4 import kv4_load, kv4_store

    rng = np.random.default_rng(6)
    b, h, t, d, size, wide, num = 6, 2, 5, 128, 32, 2, 4
    # 0: fine; 1: start -1 (a reserve that did not happen); 2: past the table; 3: no page; 4: a page
    # number past the pool; 5: a sequence outside the table
    table = np.array([[2, 0], [1, 3], [1, 3], [-1, 3], [num, 3], [1, 1]], np.int32)
    starts, ids = np.array([30, -1, 62, 28, 0, 0]), np.array([0, 1, 2, 3, 4, 6])
    k = torch.randn((b, h, t, d), device=dev).to(torch.bfloat16)
    pages = rng.integers(0, 200, (num, h, size * (d + d // 16)), np.uint8)
    gp, gt = _gpu(pages, dev, torch.uint8), _gpu(table, dev)
    kv4_store(gp, gt, k, k, _gpu(starts, dev), seq_ids=_gpu(ids, dev))
    live = np.zeros((b, t), bool)
    live[0], live[2, :2], live[3, 4:] = True, True, True
    want = pages.copy()
    codes, scales = model.encode(k.double().cpu().numpy())
    for i, j in zip(*np.nonzero(live)):
        page, slot = table[i, (starts[i] + j) // size], (starts[i] + j) % size
        kc, vc, ks, vs = model.parts(want[page], size, d)
        kc[:, slot] = vc[:, slot] = codes[i, :, j]
        ks[:, slot] = vs[:, slot] = scales[i, :, j]
    assert np.array_equal(gp.cpu().numpy(), want)
    gk, gv = kv4_load(gp, gt, _gpu(starts, dev), torch.full((b,), t, dtype=torch.int32, device=dev), t, d,
                      seq_ids=_gpu(ids, dev))
    for got in (gk, gv):
        got = got.float().cpu().numpy()
        assert np.array_equal(np.isnan(got).all((1, 3)), ~live) and np.array_equal(np.isnan(got).any((1, 3)), ~live)


# ------------------------------------------------------------------ attention


def _check_attention(got, lse, q, pages, table, lengths, counts, size, causal, scale, dtype, ids=None):
    """Error bounds, element by element, u = 2^-24:
    - a score is a sum of D exact products in fp32, D u sum|q k| at most, times the scale (2 u more);
      with the subtraction and the argument of exp2 in fp32 and exp2 good to 2^-22, a probability is off
      by e = (D + 6) u L + 2^-21 of itself, L the row's largest sum |q k| scale;
    - bf16 calls round it once more, 2^-8; fp16 calls hold it in two bf16 terms, cut off or rounded: what
      the first leaves is below 2^-7 of it, what the second leaves below 2^-7 of that, 2^-14;
    - sums of n terms in fp32, n u of softmax |v| = A; numerator and denominator: twice e and n u;
    - the output is rounded once, half a step of its type."""
    b, hq, t, d = q.shape
    u = 2.0**-24
    rounds, last = (2.0**-8, 2.0**-8) if dtype == "bf16" else (2.0**-14, 2.0**-11)
    for i in range(b):
        s = i if ids is None else ids[i]
        n = int(lengths[s])
        k, v = model.tokens(pages, table[s], n, size, d)
        out, ref_lse, spread, logit = model.attend(q[i].double().cpu().numpy(), k, v, int(counts[i]), causal, scale)
        e = ((d + 6) * u * logit + 2.0**-21)[..., None]
        tol = spread * (rounds + 2 * e + 2 * n * u) + last * np.abs(out) + 1e-30
        if dtype == "fp16":
            tol = tol + 2.0**-25  # half a step of the smallest fp16
        o = got[i].double().cpu().numpy()
        assert _same_nan(o, out), f"entry {i}"
        bad = np.nan_to_num(np.abs(o - out)) > np.nan_to_num(tol, nan=np.inf)
        assert not bad.any(), f"entry {i}: {np.argwhere(bad)[:4].tolist()} off by {np.abs(o - out)[bad][:4]}, {tol[bad][:4]}"
        got_l = lse[i].double().cpu().numpy()
        assert np.array_equal(np.isneginf(got_l), np.isneginf(ref_lse)) and _same_nan(got_l, ref_lse)
        fin = np.isfinite(ref_lse) & (ref_lse > -1e30)
        # the maximum and log2 of the sum, joined in fp32
        tol_l = e[..., 0] + n * u + 2.0**-21 + 4 * u * np.abs(ref_lse)
        assert (np.abs(got_l[fin] - ref_lse[fin]) <= tol_l[fin]).all(), f"entry {i}: lse"


CASES = [
    # hq, hk, d, rows, page, lengths, counts, causal, dtype
    (1, 1, 128, 1, 32, [1], None, False, "bf16"),
    (3, 1, 64, 1, 32, [0, 1, 31, 32, 33], None, False, "bf16"),
    (4, 4, 128, 1, 64, [64, 63, 65, 128, 700], None, True, "bf16"),
    (8, 2, 128, 1, 128, [129, 2500], None, True, "fp16"),
    (5, 1, 64, 3, 64, [2, 3, 4, 100, 0], None, True, "fp16"),
    (6, 2, 128, 5, 32, [3, 40, 333], [5, 2, 0], True, "bf16"),
    (2, 2, 64, 16, 256, [16, 17, 300], [16, 16, 9], True, "bf16"),
    (2, 1, 128, 16, 64, [100, 65], None, False, "bf16"),
    (12, 4, 64, 11, 32, [44, 45], [11, 7], True, "bf16"),
    (2, 2, 128, 33, 64, [33, 20, 150], None, True, "bf16"),
    (4, 2, 128, 70, 64, [64, 200], [70, 64], True, "fp16"),
    (3, 3, 64, 129, 128, [129, 400, 1], [129, 100, 129], True, "bf16"),
    (2, 1, 128, 150, 32, [500, 31], [150, 1], False, "bf16"),
    (2, 2, 128, 257, 64, [1000], None, True, "bf16"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_attention_matches_the_formula(dev, case):
    from sparsepr_amd.kernels.kv4 import kv4_attention

    hq, hk, d, rows, size, lengths, counts, causal, dtype = case
    rng = np.random.default_rng(hash((hq, d, rows)) % 1000)
    b, wide = len(lengths), max(1, max(-(-n // size) for n in lengths)) + 1
    num = sum(-(-n // size) for n in lengths) + 2
    pages = _pool(rng, num, hk, size, d)
    table = _table(rng, lengths, size, num, wide)
    # what lies past a sequence's end, in its last page and in pages of nobody, is NaN
    used = np.zeros((num, size), bool)
    for i, n in enumerate(lengths):
        for j in range(n):
            used[table[i, j // size], j % size] = True
    for part in model.parts(pages, size, d)[2:]:
        part[np.broadcast_to(~used[:, None], (num, hk, size))] = 255
    q = (torch.randn((b, hq, rows, d), generator=torch.Generator().manual_seed(3)) * 0.9).to(DT[dtype]).to(dev)
    cnt = np.array(counts if counts is not None else [rows] * b)
    scale = 1.0 / math.sqrt(d)
    out, lse = kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu(lengths, dev),
                             counts=None if counts is None else _gpu(cnt, dev), causal=causal, return_lse=True)
    _check_attention(out, lse, q, pages, table, lengths, cnt, size, causal, scale, dtype)


def test_seq_ids_share_scale_and_strides(dev):
    """Two entries on one sequence, a scale of the caller's, q by its strides and q off 16 bytes."""
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(8)
    hq, hk, d, size, rows = 6, 3, 64, 32, 4
    lengths, ids = [70, 5, 33], [2, 0, 2, 1]
    num = sum(-(-n // size) for n in lengths)
    pages, table = _pool(rng, num, hk, size, d), _table(rng, lengths, size, num, 3)
    args = (_gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu(lengths, dev))
    base = torch.randn((4, rows, hq, d), device=dev).to(torch.bfloat16)
    odd = torch.randn((4, hq, rows, d + 3), device=dev).to(torch.bfloat16)[..., 3:]
    for q in (base.transpose(1, 2), odd, base.transpose(1, 2)[:, :, :1]):
        out, lse = kv4_attention(q, *args, seq_ids=_gpu(ids, dev), causal=True, scale=0.3, return_lse=True)
        _check_attention(out, lse, q, pages, table, lengths, [q.shape[2]] * 4, size, True, 0.3, "bf16", ids)


@pytest.mark.parametrize("rows,hq", [(1, 2), (40, 2), (130, 2)])
def test_nan_groups_reach_the_rows_that_see_them_and_no_others(dev, rows, hq):
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(9)
    hk, d, size, n = 2, 128, 64, 200
    for where in (0, n - rows // 2 - 1, n - 1):
        for part, group in ((2, 1), (3, 2), (3, 0)):  # a K scale, V scales
            pages, table = _pool(rng, 4, hk, size, d), _table(rng, [n], size, 4, 4)
            model.parts(pages[table[0, where // size]], size, d)[part][1, where % size, group] = 255
            q = torch.randn((1, hq, rows, d), device=dev).to(torch.bfloat16)
            out, lse = kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu([n], dev), causal=True,
                                     return_lse=True)
            _check_attention(out, lse, q, pages, table, [n], [rows], size, True, d**-0.5, "bf16")


@pytest.mark.parametrize("rows", [1, 50, 200])
def test_broken_tables_give_nan_and_leave_the_others_alone(dev, rows):
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(10)
    hk, d, size, wide = 1, 64, 32, 4
    lengths = [100, 100, 129, -3, 100]  # 1: a page past the pool; 2: longer than the table; 3: negative
    pages, table = _pool(rng, 12, hk, size, d), _table(rng, [100, 100, 128, 0, 0], size, 12, wide)
    table[1, 2] = 99
    table[4] = [0, -1, 1, 2]
    ids = [0, 1, 2, 3, 4, 7, -1]
    q = torch.randn((len(ids), 2, rows, d), device=dev).to(torch.bfloat16)
    out, lse = kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu(lengths, dev),
                             seq_ids=_gpu(ids, dev), return_lse=True)
    _check_attention(out[:1], lse[:1], q[:1], pages, table, lengths, [rows], size, False, d**-0.5, "bf16")
    assert torch.isnan(out[1:]).all() and torch.isnan(lse[1:]).all()


def test_sharp_scores_and_long_sequences(dev):
    """Scores far apart (one key takes all, the maximum moves late) and 40,000 keys in many shares."""
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(11)
    for rows, n, amp in ((1, 40001, 1.0), (20, 3000, 25.0), (70, 3000, 25.0), (130, 9000, 4.0)):
        hk, d, size = 1, 128, 64
        num = -(-n // size)
        pages, table = _pool(rng, num, hk, size, d, amp), _table(rng, [n], size, num, num)
        q = torch.randn((1, 2, rows, d), device=dev).to(torch.bfloat16)
        for longest in (None, 64, n):  # a wrong bound sizes the launch and nothing else
            out, lse = kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu([n], dev),
                                     max_length=longest, return_lse=True)
            _check_attention(out, lse, q, pages, table, [n], [rows], size, False, d**-0.5, "bf16")


@pytest.mark.parametrize("rows,group", [(1, 4), (9, 1), (5, 5), (20, 2), (65, 1), (130, 2)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ragged_batches_in_shares(dev, rows, group, dtype):
    """Sequences of unlike length, in no order, with keys in several shares (long ones), in one and in
    none, for every kernel: each row comes out with its own sequence's."""
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(15)
    hk, d, size = 2, 64, 64
    lengths = [700, 5000, 0, 31, 9000, 2500, 5000]
    ids = [3, 0, 5, 2, 4, 1, 6, 5]
    counts = [rows, rows, max(1, rows // 2), rows, rows, 0, rows, rows]
    num = sum(-(-n // size) for n in lengths)
    pages, table = _pool(rng, num, hk, size, d), _table(rng, lengths, size, num, 141)
    q = torch.randn((len(ids), hk * group, rows, d), device=dev).to(DT[dtype])
    for causal in (False, True):
        out, lse = kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu(lengths, dev),
                                 counts=_gpu(counts, dev), seq_ids=_gpu(ids, dev), causal=causal, return_lse=True)
        # two heads and some rows of each, so that the reference stays quick
        heads = [0, hk * group - 1]
        for i, s in enumerate(ids):
            k, v = model.tokens(pages, table[s], lengths[s], size, d)
            n = lengths[s]
            for h in heads:
                for t in {0, counts[i] // 3, counts[i] - 1, rows - 1} - {-1}:
                    one = q[i:i + 1, h:h + 1, t:t + 1]
                    seen = (min(max(n - counts[i] + t + 1, 0), n) if causal else n) if t < counts[i] else 0
                    kv = k[None, h // group, :seen], v[None, h // group, :seen]
                    ref, ref_lse, spread, logit = model.attend(one[0].double().cpu().numpy(), *kv, 1, False, d**-0.5)
                    u = 2.0**-24  # the bounds of _check_attention
                    rounds, last = (2.0**-8, 2.0**-8) if dtype == "bf16" else (2.0**-14, 2.0**-11)
                    e = (d + 6) * u * logit[0, 0] + 2.0**-21
                    tol = spread * (rounds + 2 * e + 2 * n * u) + last * np.abs(ref) + 2.0**-25
                    assert (np.abs(out[i, h, t].double().cpu().numpy() - ref[0, 0]) <= tol[0, 0]).all(), (i, h, t)
                    if seen == 0:
                        assert torch.isneginf(lse[i, h, t])
                    else:
                        assert abs(float(lse[i, h, t]) - ref_lse[0, 0]) <= e + n * u + 2.0**-21 + 4 * u * abs(ref_lse[0, 0])


def test_pages_past_two_gigabytes(dev):
    from sparsepr_amd.kernels.kv4 import kv4_attention, kv4_compact, kv4_fork, kv4_load, kv4_store

    rng = np.random.default_rng(12)
    h, d, size = 16, 128, 256
    each = h * size * (d + d // 16)
    num = (5 << 29) // each + 1  # 2.5 GiB
    pages = torch.zeros((num, h, each // h), dtype=torch.uint8, device=dev)
    table = np.array([[num - 1, num - 3, num // 2, 1], [-1] * 4], np.int32)
    refs = np.zeros(num, np.int32)
    refs[table[0]] = 1
    gt, gl, gr = _gpu(table, dev), _gpu([900, 0], dev), _gpu(refs, dev)
    k, v = torch.randn((2, 1, h, 900, d), device=dev).to(torch.bfloat16)
    zero, cnt = _gpu([0], dev), _gpu([900], dev)
    kv4_store(pages, gt, k, v, zero)
    want = [torch.from_numpy(model.decode(*model.encode(x.double().cpu().numpy()))) for x in (k, v)]

    def check(seq):
        got = kv4_load(pages, gt, zero, cnt, 900, d, seq_ids=_gpu([seq], dev))
        assert all(torch.equal(a.double().cpu(), b) for a, b in zip(got, want))

    check(0)
    q = torch.randn((1, h, 3, d), device=dev).to(torch.bfloat16)
    before = kv4_attention(q, pages, gt, gl, seq_ids=zero, causal=True)
    kv4_fork(pages, gt, gl, gr, size, _gpu([0], dev), _gpu([1], dev), share=False)
    check(1)
    live = kv4_compact(pages, gt, gr)
    assert int(live) == 8 and int(gt.max()) == 7 and int(gr.sum()) == 8
    check(0), check(1)
    for seq in (0, 1):
        assert torch.equal(before, kv4_attention(q, pages, gt, gl, seq_ids=_gpu([seq], dev), causal=True))


# ------------------------------------------------------------------ pages


def _assert_same(cache, m):
    assert np.array_equal(cache.block_table.cpu().numpy(), m.table)
    assert np.array_equal(cache.lengths.cpu().numpy(), m.lengths)
    assert np.array_equal(cache.ref_count.cpu().numpy(), m.refs)


def _status(cache):
    got = int(cache.status.item())
    cache.status.zero_()
    return got


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("size,num,wide", [(32, 40, 9), (64, 5000, 3)])
def test_a_run_of_page_calls_follows_the_lists(dev, seed, size, num, wide):
    """Random reserves, stores, frees of ranges, forks, copies and compactions, good ones and refused
    ones: tables, lengths, holders and status after each call, the tokens of every sequence, and
    attention over them, now and then."""
    from sparsepr_amd.kv4_cache import KV4Cache

    rng = np.random.default_rng(100 * seed + size)
    seqs, h, d, layers = 7, 2, 64, 2
    cache = KV4Cache(num, h, d, seqs, page_size=size, max_pages=wide, layers=layers, device=dev)
    m = model.Pages(num, seqs, wide, size)
    text = [[np.zeros((2, h, 0, d)) for _ in range(seqs)] for _ in range(layers)]  # K, V values of each sequence
    seen = set()
    for step in range(60):
        op = rng.choice(["append", "append", "append", "free", "range", "fork", "copy", "compact"])
        n = int(rng.integers(1, 4))
        ids = [int(i) for i in rng.integers(-1 if rng.random() < 0.1 else 0, seqs + (rng.random() < 0.1), n)]
        if rng.random() < 0.85:
            ids = list(dict.fromkeys(ids))
        if op == "append":
            counts = [int(c) for c in rng.integers(-1 if rng.random() < 0.1 else 0, size * 2, len(ids))]
            code, starts = m.reserve(ids, counts)
            got = cache.reserve(counts, ids)
            assert got.cpu().tolist() == starts
            t = max(max(counts), 1)
            for layer in range(layers):
                k, v = torch.randn((2, len(ids), h, t, d), device=dev).to(torch.bfloat16)
                cache.store(k, v, got, counts=counts, seq_ids=ids, layer=layer)
                if code == 0:
                    for x, (i, c) in enumerate(zip(ids, counts)):
                        new = np.stack([model.decode(*model.encode(y[x, :, :c].double().cpu().numpy())) for y in (k, v)])
                        text[layer][i] = np.concatenate([text[layer][i], new], 2)
        elif op == "free":
            code = m.free(ids)
            cache.free(ids)
            if code == 0:
                for layer in range(layers):
                    for i in ids:
                        text[layer][i] = text[layer][i][:, :, :0]
        elif op == "range":
            firsts, counts = ([int(c) for c in rng.integers(0, 3, len(ids))] for _ in range(2))
            counts = [c if rng.random() < 0.8 else -1 for c in counts]
            before = m.lengths.copy()
            code = m.free(ids, firsts, counts)
            cache.free(ids, first_pages=firsts, page_counts=counts)
            if code == 0:
                for layer in range(layers):
                    for i, f, c in zip(ids, firsts, counts):
                        end = min((f + c) * size, before[i]) if c >= 0 else before[i]
                        text[layer][i] = np.delete(text[layer][i], np.s_[f * size:end], 2)
        elif op == "compact":
            code, live = 0, m.compact()[0]
            assert int(cache.compact()) == live
        else:
            to = [int(i) for i in rng.integers(0, seqs, len(ids))]
            if rng.random() < 0.8:  # mostly onto empty ones
                empty = [i for i in range(seqs) if m.lengths[i] == 0]
                to = empty[:len(ids)]
                ids = ids[:len(to)]
            if not ids:
                continue
            code, _ = m.fork(ids, to, op == "fork")
            cache.fork(ids, to, share=op == "fork")
            if code == 0:
                for layer in range(layers):
                    for s, t in zip(ids, to):
                        text[layer][t] = text[layer][s]
        assert _status(cache) == code, (step, op, ids)
        seen.add((op, code))
        _assert_same(cache, m)
        if step % 6 == 5:
            longest = max(int(m.lengths.max()), 1)
            for layer in range(layers):
                got = cache.load([0] * seqs, m.lengths, longest, layer=layer)
                for i in range(seqs):
                    for g, want in zip(got, text[layer][i]):
                        assert np.array_equal(g[i, :, :m.lengths[i]].double().cpu().numpy(), want), (step, i)
            q = torch.randn((seqs, 4, 2, d), device=dev).to(torch.bfloat16)
            out, lse = cache.attend(q, layer=1, causal=True, return_lse=True)
            _check_attention(out, lse, q, cache.pages[1].cpu().numpy(), m.table, m.lengths, [2] * seqs, size, True,
                             d**-0.5, "bf16")
    assert len({op for op, code in seen if code == 0}) >= 4  # kinds of call, of six


def test_every_refusal_is_named_and_changes_nothing(dev):
    from sparsepr_amd.kv4_cache import KV4Cache

    cache = KV4Cache(6, 1, 64, 4, page_size=32, max_pages=4, device=dev)
    m = model.Pages(6, 4, 4, 32)
    cache.reserve([70, 40], [0, 1])
    m.reserve([0, 1], [70, 40])
    cache.check()
    for code, call, text in [
        (1, lambda: cache.reserve([1], [4]), "outside the table"),
        (1, lambda: cache.free([-1]), "outside the table"),
        (1, lambda: cache.fork([0], [9]), "outside the table"),
        (2, lambda: cache.reserve([1, 1], [2, 2]), "named twice"),
        (2, lambda: cache.free([0, 1, 0]), "named twice"),
        (2, lambda: cache.fork([0, 1], [2, 2]), "named twice"),
        (2, lambda: cache.fork([0, 2], [3, 2]), "named twice"),
        (3, lambda: cache.reserve([-1], [2]), "negative count"),
        (3, lambda: cache.free([0], first_pages=[2], page_counts=[2]), "range outside"),
        (3, lambda: cache.free([1], first_pages=[3]), "range outside"),
        (4, lambda: cache.reserve([1, 129], [0, 2]), "more tokens than a row"),
        (4, lambda: cache.reserve([2**31 - 1], [0]), "more tokens than a row"),
        (5, lambda: cache.reserve([58, 10], [0, 2]), "not enough free pages"),
        (5, lambda: cache.fork([0], [2], share=False), "not enough free pages"),
        (5, lambda: cache.fork([0, 1], [2, 3]), "not enough free pages"),
        (6, lambda: cache.fork([0], [1]), "holds tokens"),
    ]:
        got = call()
        if got is not None:
            assert (got == -1).all()
        _assert_same(cache, m)
        with pytest.raises(RuntimeError, match=text):
            cache.check()
        cache.check()
    # the first one stays until it is read
    cache.free([7])
    cache.reserve([1, 1], [2, 2])
    with pytest.raises(RuntimeError, match="outside the table"):
        cache.check()
    # tables that cannot be
    cache.block_table[0, 1] = 6
    for call in (lambda: cache.free([0]), lambda: cache.fork([0], [2])):
        call()
        with pytest.raises(RuntimeError, match="entry outside the pool"):
            cache.check()
    cache.lengths[1] = 129
    for call in (lambda: cache.free([1]), lambda: cache.reserve([1], [1]), lambda: cache.fork([1], [2])):
        call()
        with pytest.raises(RuntimeError, match="length outside the table"):
            cache.check()


def test_as_many_sequences_as_a_call_may_name(dev):
    from sparsepr_amd.kernels.kv4 import MAX_NAMED
    from sparsepr_amd.kv4_cache import KV4Cache

    rng = np.random.default_rng(13)
    n = MAX_NAMED
    cache = KV4Cache(9000, 1, 64, n, page_size=32, max_pages=3, device=dev)
    m = model.Pages(9000, n, 3, 32)
    ids = rng.permutation(n).tolist()
    counts = rng.integers(0, 96, n).tolist()
    code, starts = m.reserve(ids, counts)
    assert cache.reserve(counts, ids).tolist() == starts and code == 0
    _assert_same(cache, m)
    m.free(ids[::2])
    cache.free(ids[::2])
    half = n // 2
    assert m.fork(ids[1::2], ids[::2], True)[0] == 0
    cache.fork(ids[1::2], ids[::2])
    _assert_same(cache, m)
    assert int(cache.compact()) == m.compact()[0] and half > 0
    _assert_same(cache, m)
    cache.check()
    with pytest.raises(RuntimeError, match="at most"):
        cache.free([0] * (n + 1))


# ------------------------------------------------------------------ streams, graphs, repeats


def _decode_step(cache, q, k, v):
    cache.append(k, v)
    return cache.attend(q, causal=True, max_length=300)


def _filled(dev, seqs, h, d, tokens, seed):
    from sparsepr_amd.kv4_cache import KV4Cache

    g = torch.Generator(device=dev).manual_seed(seed)
    cache = KV4Cache(60, h, d, seqs, page_size=32, max_pages=12, device=dev)
    k, v = torch.randn((2, seqs, h, max(tokens), d), generator=g, device=dev).to(torch.bfloat16)
    cache.append(k, v, counts=tokens)
    return cache


def test_a_captured_step_replays_as_eager_calls_do(dev):
    seqs, h, d = 3, 2, 128
    g = torch.Generator(device=dev).manual_seed(2)
    steps = [[torch.randn((seqs, n, 1, d), generator=g, device=dev).to(torch.bfloat16) for n in (4, h, h)] for _ in range(70)]
    eager, graphed = (_filled(dev, seqs, h, d, [200, 31, 0], 1) for _ in range(2))
    ins = [x.clone() for x in steps[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _decode_step(_filled(dev, seqs, h, d, [5, 5, 5], 4), *ins)  # warm
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _decode_step(graphed, *ins)
    for x in steps:  # two graphs' worth of steps, eager work and a synchronisation between replays
        want = _decode_step(eager, *x)
        for a, b in zip(ins, x):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(eager.block_table, graphed.block_table) and torch.equal(eager.lengths, graphed.lengths)
    assert torch.equal(eager.pages, graphed.pages)
    eager.check(), graphed.check()


def test_calls_on_two_streams_and_repeats_give_the_same_bits(dev):
    seqs, h, d = 4, 2, 64
    caches = [_filled(dev, seqs, h, d, [300, 7, 128, 33], 5 + i) for i in range(2)]
    q = [torch.randn((seqs, 8, t, d), device=dev).to(torch.float16) for t in (1, 60)]
    want = [[c.attend(x, causal=True) for x in q] for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    for _ in range(5):
        got = []
        for c, s in zip(caches, streams):
            with torch.cuda.stream(s):
                got.append([c.attend(x, causal=True) for x in q])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


# ------------------------------------------------------------------ refusals, odd calls


def test_calls_with_the_wrong_tensors_are_refused(dev):
    from sparsepr_amd.kernels import kv4

    n, h, d, size = 4, 2, 64, 32
    pages = torch.zeros((n, h, kv4.kv4_page_bytes(size, d)), dtype=torch.uint8, device=dev)
    table = torch.zeros((3, 2), dtype=torch.int32, device=dev)
    lengths, refs, one = (torch.zeros(k, dtype=torch.int32, device=dev) for k in (3, n, 1))
    x = torch.zeros((1, h, 5, d), dtype=torch.bfloat16, device=dev)

    def store(p=pages, t=table, k=x, v=x, s=one, **kw):
        kv4.kv4_store(p, t, k, v, s, **kw)

    def load(p=pages, t=table, s=one, c=one, rows=5, dim=d, **kw):
        kv4.kv4_load(p, t, s, c, rows, dim, **kw)

    def attend(q=x, p=pages, t=table, n=lengths, **kw):
        kv4.kv4_attention(q, p, t, n, **kw)

    for call, text in [
        (lambda: store(p=pages.int()), "contiguous uint8"), (lambda: store(p=pages[:, :1]), "contiguous uint8"),
        (lambda: store(p=pages[..., :-16].contiguous()), "not whole pages"), (lambda: store(p=pages[:0]), "contiguous uint8"),
        (lambda: store(k=x[..., :32], v=x[..., :32]), "head dim 32"), (lambda: store(v=x.float()), "of one dtype"),
        (lambda: store(k=x.int(), v=x.int()), "of one dtype"), (lambda: store(v=x[:, :, :4]), "of one dtype"),
        (lambda: store(k=x[:, :1], v=x[:, :1]), "K has 1 heads, the pages 2"),
        (lambda: store(t=table.long()), "block_table must be"), (lambda: store(t=table[0]), "block_table must be"),
        (lambda: store(t=table.t()), "block_table must be"), (lambda: store(s=lengths), "starts must be"),
        (lambda: store(s=one.long()), "starts must be"), (lambda: store(counts=lengths), "counts must be"),
        (lambda: store(seq_ids=lengths), "seq_ids must be"), (lambda: store(s=one.cpu()), "require GPU tensors"),
        (lambda: store(k=x.expand(5, h, 5, d), v=x.expand(5, h, 5, d), s=torch.zeros(5, dtype=torch.int32, device=dev)),
         "a batch of 5 without seq_ids"),
        (lambda: load(dim=128), "not whole pages"), (lambda: load(rows=-1), "rows -1"),
        (lambda: load(dtype=torch.float64), "dtype must be"), (lambda: load(c=lengths), "counts must be"),
        (lambda: attend(q=x.float()), "bfloat16 or float16"), (lambda: attend(q=x[0]), "bfloat16 or float16"),
        (lambda: attend(q=x[:, :1]), "multiple of KV heads"), (lambda: attend(n=one), "lengths must be"),
        (lambda: attend(counts=lengths), "counts must be"), (lambda: attend(scale=0.0), "scale must be positive"),
        (lambda: attend(scale=float("nan")), "scale must be positive"), (lambda: attend(max_length=-1), "max_length -1"),
        (lambda: kv4.kv4_reserve(table, lengths, refs, 48, lengths), "page size 48"),
        (lambda: kv4.kv4_reserve(table, one, refs, size, lengths), "lengths must be"),
        (lambda: kv4.kv4_reserve(table, lengths, refs, size, refs), "a batch of 4 without seq_ids"),
        (lambda: kv4.kv4_reserve(table, lengths, refs, size, lengths, status=lengths), "status must be"),
        (lambda: kv4.kv4_free(table, lengths, refs, size, one, first_pages=lengths), "first_pages must be"),
        (lambda: kv4.kv4_free(table, lengths, refs, size, one.float()), "seq_ids must be"),
        (lambda: kv4.kv4_fork(pages, table, lengths, refs, size, one, lengths), "dst must be"),
        (lambda: kv4.kv4_fork(pages, table, lengths, one, size, one, one), "4 pages, ref_count of 1"),
        (lambda: kv4.kv4_compact(pages.float(), table, refs), "contiguous uint8"),
        (lambda: kv4.kv4_compact(pages[None, None], table, refs), "contiguous uint8"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()
    assert int(pages.sum()) == 0


def test_empty_calls_and_no_sequences(dev):
    from sparsepr_amd.kv4_cache import KV4Cache

    cache = KV4Cache(4, 2, 64, 3, page_size=32, device=dev)
    x = torch.zeros((0, 2, 5, 64), dtype=torch.bfloat16, device=dev)
    assert cache.attend(x).shape == x.shape
    out, lse = cache.attend(torch.ones((3, 4, 0, 64), dtype=torch.float16, device=dev), return_lse=True)
    assert out.shape == (3, 4, 0, 64) and lse.shape == (3, 4, 0)
    out, lse = cache.attend(torch.ones((3, 4, 2, 64), dtype=torch.float16, device=dev), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()  # sequences without tokens
    out, lse = cache.attend(torch.ones((3, 4, 40, 64), dtype=torch.float16, device=dev), causal=True, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    assert cache.reserve(none, none).shape == (0,)
    cache.free(none), cache.fork(none, none), cache.store(x, x, none)
    k, v = cache.load([0, 0, 0], [0, 0, 0], 0)
    assert k.shape == (3, 2, 0, 64)
    k, v = cache.load([0, 0, 0], [0, 1, 0], 2)
    assert (k[[0, 2]] == 0).all() and torch.isnan(k[1, :, 0]).all() and (v[1, :, 1] == 0).all()
    assert int(cache.compact()) == 0
    cache.check()
    # the lengths themselves as counts: sequences twice as long
    cache.reserve([20, 0, 30])
    starts = cache.reserve(cache.lengths)
    assert starts.tolist() == [20, 0, 30] and cache.lengths.tolist() == [40, 0, 60]


def test_a_window_that_slides_over_a_video(dev):
    """Frame after frame: reserve, store, attend, and past four frames the oldest whole pages but the
    first go; attention is over what is left, in order."""
    from sparsepr_amd.kv4_cache import KV4Cache

    rng = np.random.default_rng(14)
    h, d, size, frame, layers = 3, 128, 32, 50, 2
    cache = KV4Cache(9, h, d, 2, page_size=size, max_pages=9, layers=layers, device=dev)
    kept = [np.zeros((2, h, 0, d)) for _ in range(layers)]
    for i in range(12):
        starts = cache.reserve([frame], [1])
        for layer in range(layers):
            k, v = torch.randn((2, 1, frame, h, d), device=dev).to(torch.bfloat16).transpose(2, 3)
            cache.store(k, v, starts, seq_ids=[1], layer=layer)
            new = np.stack([model.decode(*model.encode(y[0].double().cpu().numpy())) for y in (k, v)])
            kept[layer] = np.concatenate([kept[layer], new], 2)
            q = torch.randn((1, h, frame, d), device=dev).to(torch.bfloat16)
            out, lse = cache.attend(q, seq_ids=[1], layer=layer, return_lse=True)
            n = kept[layer].shape[2]
            assert int(cache.lengths[1]) == n
            # 2^-8 for each rounding (probabilities, output), and as much again for what is in fp32
            ref, ref_lse, spread, _ = model.attend(q[0].double().cpu().numpy(), *kept[layer], frame, False, d**-0.5)
            assert (np.abs(out[0].double().cpu().numpy() - ref) <= 2.0**-7 * (spread + np.abs(ref)) + 1e-6).all()
            got = cache.load([0], [n], n, seq_ids=[1], layer=layer)
            assert all(np.array_equal(g[0].double().cpu().numpy(), w) for g, w in zip(got, kept[layer]))
        over = (n - 3 * frame) // size
        if over > 0:
            cache.free([1], first_pages=[1], page_counts=[over])
            kept = [np.delete(x, np.s_[size:size * (1 + over)], 2) for x in kept]
    cache.check()


def test_captured_attention_with_shares_of_the_keys(dev):
    """Calls whose keys are dealt in shares (workspaces, merges), of each kernel: two graphs over one
    cache, replayed in turns with eager calls between, as the sequences grow."""
    from sparsepr_amd.kv4_cache import KV4Cache

    g = torch.Generator(device=dev).manual_seed(7)
    h, d = 2, 64
    cache = KV4Cache(220, h, d, 2, page_size=64, max_pages=110, device=dev)
    k, v = torch.randn((2, 2, h, 6000, d), generator=g, device=dev).to(torch.bfloat16)
    cache.append(k, v, counts=[6000, 1500])
    qs = [torch.randn((2, 4, t, d), generator=g, device=dev).to(torch.bfloat16) for t in (1, 14, 30, 60, 200)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for q in qs:
            cache.attend(q, causal=True, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for part in (qs[:3], qs[3:]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [cache.attend(q, causal=True, return_lse=True) for q in part]
        graphs.append((graph, part, outs))
    for step in range(4):
        cache.append(k[:, :, :200], v[:, :, :200])
        for graph, part, outs in graphs:
            for q in part:
                q.copy_(torch.randn(q.shape, generator=g, device=dev))
            want = [cache.attend(q, causal=True, return_lse=True) for q in part]
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), step
    cache.check()


ROWS = [(1, 2), (9, 1), (10, 2), (20, 2), (70, 1), (140, 2)]  # both kernels, 8, 16, 32 rows, 64, 128 and 256


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,group", ROWS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_slots_that_hold_no_token_change_nothing(dev, d, rows, group, dtype):
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(21)
    hk, size, lengths = 2, 64, [1, 33, 200, 0, 95]
    num = sum(-(-n // size) for n in lengths) + 2
    pages, table = _pool(rng, num, hk, size, d), _table(rng, lengths, size, num, 5)
    unused = np.ones((num, size), bool)
    for i, n in enumerate(lengths):
        for j in range(n):
            unused[table[i, j // size], j % size] = False
    unused = np.broadcast_to(unused[:, None], (num, hk, size))
    q = torch.randn((len(lengths), hk * group, rows, d), device=dev).to(DT[dtype])
    outs = []
    for scale in (100, 252, 253, 254, 255, None):  # None: any bytes at all
        for part in model.parts(pages, size, d)[:2]:
            part[unused] = rng.integers(0, 256, part[unused].shape, np.uint8)
        for part in model.parts(pages, size, d)[2:]:
            part[unused] = rng.integers(0, 256, part[unused].shape, np.uint8) if scale is None else scale
        for causal in (False, True):
            outs.append(kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu(lengths, dev),
                                      causal=causal, return_lse=True))
    for i, got in enumerate(outs):
        assert all(torch.equal(a, b) for a, b in zip(got, outs[i % 2])), i // 2
    assert torch.isfinite(outs[0][0]).all()


@pytest.mark.parametrize("byte", [253, 254])
@pytest.mark.parametrize("rows", [1, 40, 130])
def test_scale_bytes_past_the_encoders_are_nan(dev, rows, byte):
    from sparsepr_amd.kernels.kv4 import kv4_attention, kv4_load

    rng = np.random.default_rng(22)
    hk, d, size, n = 2, 128, 64, 200
    for where in (0, n - rows // 2 - 1, n - 1):
        for part, group in ((2, 1), (3, 2)):
            pages, table = _pool(rng, 4, hk, size, d), _table(rng, [n], size, 4, 4)
            said = model.parts(pages[table[0, where // size]], size, d)[part][1, where % size]
            said[group] = byte
            gp, gt = _gpu(pages, dev, torch.uint8), _gpu(table, dev)
            said[group] = 255
            q = torch.randn((1, 2, rows, d), device=dev).to(torch.bfloat16)
            out, lse = kv4_attention(q, gp, gt, _gpu([n], dev), causal=True, return_lse=True)
            _check_attention(out, lse, q, pages, table, [n], [rows], size, True, d**-0.5, "bf16")
            loaded = kv4_load(gp, gt, _gpu([0], dev), _gpu([n], dev), n, d)
            for got, want in zip(loaded, model.tokens(pages, table[0], n, size, d)):
                assert np.array_equal(got[0].double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("rows,group", ROWS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 6000])
def test_rows_whose_scores_are_all_minus_infinity_are_nan(dev, rows, group, dtype, n):
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(23)
    d, size = 64, 64
    num = -(-n // size)
    pages, table = _pool(rng, num, 1, size, d), _table(rng, [n], size, num, num)
    codes = model.parts(pages, size, d)[0]
    codes[..., 0] = codes[..., 0] & 0xF0 | 2  # K's first dim is positive
    q = torch.randn((1, group, rows, d), device=dev).to(DT[dtype])
    q[0, 0, 0, 0] = -math.inf
    out, lse = kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu([n], dev), return_lse=True)
    bad = torch.zeros((1, group, rows), dtype=torch.bool, device=dev)
    bad[0, 0, 0] = True
    assert torch.equal(torch.isnan(lse), bad) and torch.equal(torch.isnan(out).all(-1), bad)
    assert torch.equal(torch.isnan(out).any(-1), bad)


def test_tensors_of_another_head_dim_are_refused(dev):
    from sparsepr_amd.kernels import kv4
    from sparsepr_amd.kv4_cache import KV4Cache

    for d, size, other in ((64, 64, 128), (64, 256, 128), (128, 32, 64), (128, 128, 64), (64, 32, 128)):
        cache = KV4Cache(8, 2, d, 2, page_size=size, device=dev)
        starts = cache.reserve([5], [0])
        x = torch.ones((1, 2, 5, other), dtype=torch.bfloat16, device=dev)
        for call in (lambda: cache.store(x, x, starts, seq_ids=[0]), lambda: cache.attend(x, seq_ids=[0])):
            with pytest.raises(RuntimeError, match=f"head dim {other}|pages of"):
                call()
        assert int(cache.pages.sum()) == 0 and cache.lengths.tolist() == [5, 0]
    # the same of the functions, where the caller says what the pages hold
    x = torch.ones((1, 2, 5, 128), dtype=torch.bfloat16, device=dev)
    pages = torch.zeros((2, 2, kv4.kv4_page_bytes(64, 64)), dtype=torch.uint8, device=dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    five = torch.full((1,), 5, dtype=torch.int32, device=dev)
    for call in (lambda **kw: kv4.kv4_store(pages, table, x, x, five, **kw),
                 lambda **kw: kv4.kv4_attention(x, pages, table, five, **kw),
                 lambda **kw: kv4.kv4_load(pages, table, five, five, 5, 128, **kw)):
        with pytest.raises(RuntimeError, match="are not 64 tokens of head dim 128"):
            call(page_size=64)
        call(page_size=32)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_packed_rows_off_sixteen_bytes_are_taken(dev, dtype):
    from sparsepr_amd.kv4_cache import KV4Cache

    b, h, t, d = 2, 2, 9, 64
    k, v, q = (torch.randn(b * h * t * d + 1, device=dev).to(DT[dtype]) for _ in range(3))
    odd = [x[1:].view(b, h, t, d) for x in (k, v, q)]
    assert all(x.is_contiguous() and x.data_ptr() % 16 != 0 for x in odd)
    got = []
    for x in (odd, [y.clone() for y in odd]):
        cache = KV4Cache(4, h, d, b, page_size=32, device=dev)
        cache.append(x[0], x[1])
        got.append([cache.pages, *cache.load([0, 0], [t, t], t)])
        if dtype != "fp32":
            got[-1] += [cache.attend(x[2]), cache.attend(x[2][:, :1, :1].expand(b, h, t, d))]
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_a_refused_append_changes_nothing(dev):
    from sparsepr_amd.kv4_cache import KV4Cache

    cache = KV4Cache(8, 2, 64, 3, page_size=32, device=dev)
    x = torch.ones((1, 2, 5, 64), dtype=torch.bfloat16, device=dev)
    cache.append(x, x, seq_ids=[1])
    before = [t.clone() for t in (cache.pages, cache.block_table, cache.lengths, cache.ref_count)]
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    for call in (
        lambda: cache.append(x, x.float(), seq_ids=[1]), lambda: cache.append(x, x[:, :, :4], seq_ids=[1]),
        lambda: cache.append(x[:, :1], x[:, :1], seq_ids=[1]), lambda: cache.append(x.int(), x.int(), seq_ids=[1]),
        lambda: cache.append(x[..., :32], x[..., :32], seq_ids=[1]), lambda: cache.append(x[0], x[0], seq_ids=[1]),
        lambda: cache.append(x.repeat(1, 1, 1, 2), x.repeat(1, 1, 1, 2), seq_ids=[1]),
        lambda: cache.append(x, x, counts=[3, 3], seq_ids=[0, 1]), lambda: cache.append(x, x.cpu(), seq_ids=[1]),
    ):
        with pytest.raises(RuntimeError):
            call()
        for a, b in zip(before, (cache.pages, cache.block_table, cache.lengths, cache.ref_count)):
            assert torch.equal(a, b)
    cache.check()
    # counts are looked at on the device
    for counts in ([6], ints(6), [-1]):
        assert cache.append(x, x, counts=counts, seq_ids=[1]).tolist() == [-1]
        with pytest.raises(RuntimeError, match="past the rows given"):
            cache.check()
        for a, b in zip(before, (cache.pages, cache.block_table, cache.lengths, cache.ref_count)):
            assert torch.equal(a, b)
    assert cache.append(x, x, counts=ints(5), seq_ids=[1]).tolist() == [5] and cache.lengths.tolist() == [0, 10, 0]
    cache.check()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_the_workspace_query_is_what_a_call_needs_for_the_same_arguments(dev, dtype):
    from sparsepr_amd import _lib

    size, d = 64, 128
    for wide in (1, 3, 17, 40, 90):
        for rows, heads in ((1, 2), (20, 4), (64, 3), (128, 24), (200, 7)):
            q = torch.ones((1, heads, rows, d), dtype=DT[dtype], device=dev)
            out = torch.empty_like(q)
            pages = torch.zeros((1, heads, size * (d + d // 16)), dtype=torch.uint8, device=dev)
            table = torch.zeros((1, wide), dtype=torch.int32, device=dev)
            n = torch.full((1,), wide * size, dtype=torch.int32, device=dev)
            for bound in (0, 500, 2000, 9000, 1 << 20, (1 << 63) - 1):
                need = _lib.query("spr_kv4_attention_workspace", 1, heads, heads, rows, d, bound)
                ws = _lib.workspace(need, dev)
                out.fill_(7)
                _lib.launch("spr_kv4_attention", dev, q.data_ptr(), *q.stride()[:3], _lib.DTYPE_CODE[q.dtype], 1, heads,
                            heads, rows, d, pages.data_ptr(), 1, size, table.data_ptr(), 1, wide, n.data_ptr(), None,
                            None, 0, 0.1, bound, out.data_ptr(), None, ws.data_ptr(), need)
                assert (out == 0).all()


@pytest.mark.filterwarnings("ignore:Synchronization debug mode")
def test_calls_with_lists_do_not_wait_for_the_gpu(dev):
    from sparsepr_amd.kv4_cache import KV4Cache

    h, d = 2, 64
    cache = KV4Cache(200, h, d, 3, page_size=32, max_pages=40, layers=2, device=dev)
    one = KV4Cache(20, h, d, 3, page_size=32, device=dev)
    k, v = torch.randn((2, 1, h, 8, d), device=dev).to(torch.bfloat16)

    def run():
        starts = cache.reserve([8], [0])
        for layer in range(2):
            cache.store(k, v, starts, counts=[8], seq_ids=[0], layer=layer)
            cache.attend(k, seq_ids=[0], counts=[8], layer=layer, causal=True)
        cache.fork([0], [1])
        cache.load([0, 0], [8, 4], 8, seq_ids=[1, 0])
        cache.free([0], first_pages=[0], page_counts=[1])
        cache.free([1])
        one.append(k, v, seq_ids=[0])
        one.append(k, v, counts=[3], seq_ids=[0])
        cache.compact()

    run()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        run()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    cache.check(), one.check()
    assert one.lengths.tolist() == [22, 0, 0]


def test_lists_hold_what_they_held_when_the_call_was_made(dev):
    """Hundreds of calls behind a GPU that is busy, with lists that are changed right after."""
    from sparsepr_amd.kv4_cache import KV4Cache

    rng = np.random.default_rng(26)
    cache, m = KV4Cache(3000, 1, 64, 40, page_size=32, max_pages=200, device=dev), model.Pages(3000, 40, 200, 32)
    busy = torch.randn((8192, 8192), device=dev).to(torch.bfloat16)
    for _ in range(30):
        busy @ busy
    starts = []
    for _ in range(300):
        ids = rng.permutation(40)[:3].tolist()
        counts = rng.integers(0, 20, 3).tolist()
        starts.append((cache.reserve(counts, ids), m.reserve(ids, counts)[1]))
        ids[:], counts[:] = [39, 39, 39], [-1, -1, -1]
    for got, want in starts:
        assert got.tolist() == want
    _assert_same(cache, m)
    cache.check()


def test_a_captured_graph_refuses_lists(dev):
    cache = _filled(dev, 3, 2, 64, [5, 6, 7], 8)
    ids, q = _gpu([2, 0], dev), torch.randn((2, 2, 1, 64), device=dev).to(torch.bfloat16)
    want = cache.attend(q, seq_ids=ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="pass an int32 tensor"):
            cache.attend(q, seq_ids=[2, 0])
        with pytest.raises(RuntimeError, match="pass an int32 tensor"):
            cache.reserve([1], [0])
        out = cache.attend(q, seq_ids=ids)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert cache.lengths.tolist() == [5, 6, 7]


@pytest.mark.parametrize("rows,heads,lengths", [
    (1, 24, [3600]), (1, 24, [20000]), (12, 24, [3600]), (30, 8, [20000]), (128, 24, [3600]), (128, 24, [20000]),
    (1, 8, [3600, 0, 9000]), (64, 4, [3600, 9000, 33])])
def test_a_loose_bound_deals_the_keys_as_the_exact_one(dev, rows, heads, lengths):
    """The bits depend on how the keys are dealt out: they do not move with `max_length`."""
    from sparsepr_amd.kv4_cache import KV4Cache

    d, b = 128, len(lengths)
    cache = KV4Cache(sum(-(-n // 64) for n in lengths), heads, d, b, max_pages=4096, device=dev)
    k, v = torch.randn((2, b, heads, max(lengths), d), device=dev).to(torch.bfloat16)
    cache.append(k, v, counts=lengths)
    q = torch.randn((b, heads, rows, d), device=dev).to(torch.bfloat16)
    want = cache.attend(q, max_length=max(lengths), return_lse=True)
    for bound in (max(lengths) + 1000, 60000, None):
        got = cache.attend(q, max_length=bound, return_lse=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), bound


@pytest.mark.parametrize("count", [1, 63, 64, 65, 100, -1])
def test_ranges_of_long_rows_close_up(dev, count):
    from sparsepr_amd.kv4_cache import KV4Cache

    tokens = [300 * 32, 130 * 32 - 5, 257 * 32 + 1]
    for firsts in ([0, 199, 1], [63, 1, 30], [128, 64, 0]):
        cache = KV4Cache(700, 1, 64, 3, page_size=32, max_pages=300, device=dev)
        m = model.Pages(700, 3, 300, 32)
        cache.reserve(tokens), m.reserve([0, 1, 2], tokens)
        cache.free([2, 0, 1], first_pages=firsts, page_counts=[count] * 3)
        assert m.free([2, 0, 1], firsts, [count] * 3) == 0
        _assert_same(cache, m)
        cache.check()


def test_ranges_of_more_sequences_than_one_launch_frees(dev):
    from sparsepr_amd.kv4_cache import KV4Cache

    rng = np.random.default_rng(24)
    n = 70
    tokens = rng.integers(1, 130 * 32, n).tolist()
    num = sum(-(-t // 32) for t in tokens) + n
    cache, m = KV4Cache(num, 1, 64, 2 * n, page_size=32, max_pages=130, device=dev), model.Pages(num, 2 * n, 130, 32)
    cache.reserve(tokens, list(range(n))), m.reserve(list(range(n)), tokens)
    cache.fork(list(range(n)), list(range(n, 2 * n))), m.fork(list(range(n)), list(range(n, 2 * n)), True)
    ids = rng.permutation(2 * n)[:100].tolist()
    held = [-(-tokens[i % n] // 32) for i in ids]
    firsts = [int(rng.integers(0, k + 1)) for k in held]
    counts = [int(rng.integers(-1, k - f + 1)) for f, k in zip(firsts, held)]
    cache.free(ids, first_pages=firsts, page_counts=counts)
    assert m.free(ids, firsts, counts) == 0
    _assert_same(cache, m)
    before = m.table.copy()
    cache.free(ids, first_pages=[0] * 99 + [131], page_counts=[0] * 99 + [1])  # refused whole
    assert _status(cache) == 3 and np.array_equal(before, m.table)
    _assert_same(cache, m)


@pytest.mark.parametrize("rows", [1, 40])
def test_more_sequences_than_a_wave_ranks(dev, rows):
    from sparsepr_amd.kernels.kv4 import kv4_attention

    rng = np.random.default_rng(25)
    hk, d, size, n = 1, 64, 64, 70
    lengths = rng.integers(0, 900, n).tolist()
    lengths[5] = 2900  # several shares, and the last one in the batch
    num = sum(-(-t // size) for t in lengths)
    pages, table = _pool(rng, num, hk, size, d), _table(rng, lengths, size, num, 46)
    ids = [i for i in rng.permutation(n).tolist() if i != 5] + [5]
    q = torch.randn((n, 1, rows, d), device=dev).to(torch.bfloat16)
    out, lse = kv4_attention(q, _gpu(pages, dev, torch.uint8), _gpu(table, dev), _gpu(lengths, dev),
                             seq_ids=_gpu(ids, dev), causal=True, return_lse=True)
    _check_attention(out, lse, q, pages, table, lengths, [rows] * n, size, True, d**-0.5, "bf16", ids)


def test_a_captured_call_deals_a_growing_sequence_as_eager_calls_do(dev):
    """One sequence, no bound: the shares follow its length from replay to replay."""
    from sparsepr_amd.kv4_cache import KV4Cache

    g = torch.Generator(device=dev).manual_seed(9)
    h, d = 3, 128
    cache = KV4Cache(400, h, d, 2, page_size=64, max_pages=300, device=dev)
    ids = _gpu([1], dev)
    k, v = torch.randn((2, 1, h, 1500, d), generator=g, device=dev).to(torch.bfloat16)
    qs = [torch.randn((1, 6, t, d), generator=g, device=dev).to(dt)
          for t, dt in ((1, DT["bf16"]), (12, DT["fp16"]), (20, DT["bf16"]), (60, DT["fp16"]), (300, DT["bf16"]))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for q in qs:
            cache.attend(q, seq_ids=ids, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [cache.attend(q, seq_ids=ids, return_lse=True) for q in qs]
    for count in (0, 1, 600, 1500, 1500, 1500, 1500, 1500, 1500):
        cache.append(k[:, :, :count], v[:, :, :count], seq_ids=ids)
        want = [cache.attend(q, seq_ids=ids, return_lse=True) for q in qs]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), int(cache.lengths[1])
    cache.check()
