"""8-bit matrices and their product on the GPU against the definitions in 64 bits.

Quantisation is exact: its bytes are the model's.  A product of codes that are small whole numbers has sums
below 2^24, which fp32 holds exactly in any order: the output is the exact one, rounded once.  For other
codes, K additions of which each is off by at most 2^-23 (a rounding to fp32 or a cut) of the sum of
magnitudes, then half a step of the output's type.  Outputs in 16 bits come from the 8-bit matrix
instruction, which cuts the other seven of eight neighbouring products 2^-13 below the largest: 7 * 2^-13 of
each eight's largest product more.  (Whole numbers up to 16 with scales alike in a block lose nothing there.)"""

# Outputs in 16 bits come from the 8-bit instruction only where fast sums are asked for (test_gpu_fp8_sums.py); the bound
# above holds for both ways of summing.
import numpy as np
import pytest
import torch

from tests import _fp8_model as model

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {t: torch.finfo(t).eps / 2 for t in DT.values()}


def _f64(t):
    return t.double().cpu().numpy()


def _bytes(t):
    return t.view(torch.uint8).cpu().numpy()


def _put(codes, scales, dev):
    return (torch.from_numpy(codes).to(dev).view(torch.float8_e4m3fn), torch.from_numpy(scales).to(dev))


# ------------------------------------------------------------------ rows to codes and back


def _rows(rng, r, c, dtype):
    x = rng.standard_normal((r, c)) * np.exp(2.5 * rng.standard_normal((r, 1))) * np.exp(rng.standard_normal(c))
    t = torch.from_numpy(x).to(dtype)
    if r > 4:
        t[0] = 0.0
        t[1, : min(c, 5)] = -0.0
        t[2, c // 2] = float(torch.finfo(dtype).max) * 0.9
        t[3] = t[3] * float(torch.finfo(dtype).tiny)
        # ties between two codes, at the scale that a top of 1.75 * 2^n gives
        edge = torch.tensor([448.0, 17.0, 19.0, 2.0**-10, 3 * 2.0**-10, -17.0, 232.0, 248.0])[:c]
        t[4, : len(edge)] = edge.to(dtype)
    return t


def _same_values(codes, want_codes, scales, want_scales):
    """Bytes alike where the group is a number; any bytes under a NaN scale."""
    assert np.array_equal(scales, want_scales)
    got, want = model.values(codes, scales), model.values(want_codes, want_scales)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    assert np.array_equal(codes[~nan], want_codes[~nan])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("square,transpose", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("shape", [(1, 1), (1, 300), (5, 16), (130, 40), (129, 257), (300, 1000)])
def test_codes_are_the_models_and_read_back_exactly(dev, dtype, square, transpose, shape):
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_quantize

    rng = np.random.default_rng(shape[1])
    x = _rows(rng, *shape, DT[dtype])
    codes, scales = fp8_quantize(x.to(dev), square=square, transpose=transpose)
    want = model.quantise(_f64(x.t() if transpose else x), square)
    assert codes.dtype == torch.float8_e4m3fn and tuple(codes.shape) == want[0].shape
    _same_values(_bytes(codes), want[0], scales.cpu().numpy(), want[1])
    v = model.values(*want)
    for out in DT.values():
        got = fp8_dequantize(codes, scales, dtype=out)
        assert torch.equal(got.cpu(), torch.from_numpy(v).to(out))  # fp32 and bf16 hold them; fp16 rounds as torch does


@pytest.mark.parametrize("square,transpose", [(False, False), (True, False), (False, True), (True, True)])
def test_a_group_with_an_infinity_or_a_nan_is_nan_and_no_other(dev, square, transpose):
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_quantize

    x = torch.randn(200, 300, generator=torch.Generator().manual_seed(1))
    x[3, 5], x[140, 290], x[60, 130] = float("inf"), float("nan"), float("-inf")
    codes, scales = fp8_quantize(x.to(dev), square=square, transpose=transpose)
    want = model.quantise(_f64(x.t() if transpose else x), square)
    _same_values(_bytes(codes), want[0], scales.cpu().numpy(), want[1])
    assert np.array_equal(np.isnan(_f64(fp8_dequantize(codes, scales))), np.isnan(model.values(*want)))


def test_quantisation_reads_strided_rows_and_copies_others(dev):
    from sparsepr_amd.kernels.fp8 import fp8_quantize

    base = torch.randn(70, 3, 250, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    for x in (base[:, 1], base[:, 2, 3:], base[:, 0].t(), base[:, 0, ::2], base[:1, 0].expand(9, 250)):
        for transpose in (False, True):
            codes, scales = fp8_quantize(x, transpose=transpose)
            want = model.quantise(_f64(x.t() if transpose else x))
            assert np.array_equal(_bytes(codes), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


# ------------------------------------------------------------------ the product

SIZES = [(1, 1, 16), (1, 16, 128), (1, 500, 1040), (3, 70, 144), (16, 48, 4112), (17, 33, 272), (33, 129, 640), (64, 64, 256),
         (65, 130, 400), (128, 128, 128), (200, 300, 1168), (257, 129, 96), (333, 1000, 528), (1, 500, 4112), (17, 33, 5136),
         (60, 32, 20016)]  # the last three: the kernel of few rows, with 16, 32 and 64 of them


def _whole(rng, m, k, square):
    codes = model.encode(rng.integers(-4, 5, (m, k)).astype(float))
    scales = rng.integers(126, 129, (-(-m // 128) if square else m, -(-k // 128))).astype(np.uint8)
    return codes, scales


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("squares", [(False, True), (False, False), (True, False)])
def test_products_of_whole_numbers_are_exact(dev, m, n, k, squares):
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    # |a b| <= 16 at scales up to 4, in steps of 1/4: sums of 20,016 of them stay below 2^24 steps
    rng = np.random.default_rng(m * 1000 + n)
    a, b = _whole(rng, m, k, squares[0]), _whole(rng, n, k, squares[1])
    want = model.values(*a) @ model.values(*b).T
    bias = torch.from_numpy(rng.integers(-8, 9, n).astype(np.float32)).to(dev)
    for out in DT.values():
        got = fp8_matmul(*_put(*a, dev), *_put(*b, dev), out_dtype=out)
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(out))
        for dt in DT.values():
            got = fp8_matmul(*_put(*a, dev), *_put(*b, dev), bias=bias.to(dt), out_dtype=out)
            assert torch.equal(got.cpu(), torch.from_numpy(want + _f64(bias)).to(out))


@pytest.mark.parametrize("m,n,k", [(4000, 3500, 256), (3328, 4097, 8320), (49152 + 7, 260, 144), (4000, 3585, 16),
                                   (1030, 5000, 4240), (500, 5000, 4240), (300, 700, 4240), (90, 5000, 8208), (30, 16, 20016)])
def test_products_on_tiles_of_every_size_are_exact(dev, m, n, k):
    """Past the edges of tiles of 256 x 256, 128 x 128, 64 x 128 and 64 x 64, and with more blocks than their windows of
    scales hold; a summed dim shorter than a block on each."""
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    g = torch.Generator(device=dev).manual_seed(3)
    a, b = (torch.randint(-2, 3, (r, k), generator=g, device=dev).to(torch.float8_e4m3fn) for r in (m, n))
    sa = torch.randint(126, 129, (m, -(-k // 128)), generator=g, device=dev).to(torch.uint8)
    sb = torch.randint(126, 129, (-(-n // 128), -(-k // 128)), generator=g, device=dev).to(torch.uint8)
    spread = lambda s, r: torch.exp2(s.float() - 127)[torch.arange(r, device=dev) // (1 if len(s) == r else 128)]  # noqa: E731
    af = a.float() * spread(sa, m).repeat_interleave(128, 1)[:, :k]
    bf = b.float() * spread(sb, n).repeat_interleave(128, 1)[:, :k]
    want = af @ bf.t()  # exact: |a b| <= 16 in steps of 1/4, 20,016 of them at most
    for out in DT.values():
        assert torch.equal(fp8_matmul(a, sa, b, sb, out_dtype=out), want.to(out))


@pytest.mark.parametrize("out", DT)
@pytest.mark.parametrize("m,n,k", [(1, 200, 4096), (60, 24, 20000), (40, 77, 592), (150, 190, 2064), (513, 260, 400)])
def test_products_of_rows_as_they_come(dev, out, m, n, k):
    from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize

    rng = np.random.default_rng(k)
    x = torch.from_numpy(rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k))).to(torch.bfloat16).to(dev)
    w = torch.from_numpy(rng.standard_normal((n, k)) * 0.03).to(torch.bfloat16).to(dev)
    bias = torch.from_numpy(rng.standard_normal(n)).to(DT[out]).to(dev)
    a, b = fp8_quantize(x), fp8_quantize(w, square=True)
    av, bv = model.values(_bytes(a[0]), a[1].cpu().numpy()), model.values(_bytes(b[0]), b[1].cpu().numpy())
    want, size = av @ bv.T + _f64(bias), np.abs(av) @ np.abs(bv).T + np.abs(_f64(bias))
    got = fp8_matmul(*a, *b, bias=bias, out_dtype=DT[out])
    bound = k * 2.0**-23 * size + HALF[DT[out]] * np.abs(want) + 2.0**-25
    if out != "fp32":
        for i in range(0, k, 8):
            bound += 7 * 2.0**-13 * (np.abs(av[:, None, i:i + 8]) * np.abs(bv[None, :, i:i + 8])).max(-1)
    assert got.dtype == DT[out] and (np.abs(_f64(got) - want) <= bound).all()
    assert torch.equal(got, fp8_matmul(*a, *b, bias=bias, out_dtype=DT[out]))  # the same bits again


def test_scales_at_the_ends_of_their_range(dev):
    """2^-127 to 2^127, products whose scales cancel, and the two kinds of NaN."""
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_matmul

    for m in (4, 100):
        n, k = 36, 256
        codes = np.full((m, k), model.encode(np.array([1.0]))[0])
        bcodes = np.full((n, k), model.encode(np.array([1.0]))[0])
        sa = np.full((m, 2), 127, np.uint8)
        sb = np.full((n, 2), 127, np.uint8)
        sa[0], sb[1] = 254, 0  # their product 2^0
        sa[1], sb[0] = 1, 253
        sa[2, 1] = 255  # NaN row
        sb[2, 0] = 255  # NaN column
        codes[3, 200], bcodes[3, 7] = 0x7F, 0xFF  # NaN codes
        want = model.values(codes, sa) @ model.values(bcodes, sb).T
        for out in (torch.float32, torch.bfloat16):
            got = _f64(fp8_matmul(*_put(codes, sa, dev), *_put(bcodes, sb, dev), out_dtype=out))
            assert np.array_equal(np.isnan(got), np.isnan(want))
            ok = ~np.isnan(want) & (np.abs(want) >= 2.0**-100)  # (subnormal results are flushed or not)
            assert np.array_equal(got[ok], _f64(torch.from_numpy(want).to(out))[ok])
            low = ~np.isnan(want) & (np.abs(want) < 2.0**-100)
            assert (np.abs(got[low]) <= 2.0**-99).all()
        assert np.array_equal(_f64(fp8_dequantize(*_put(codes, sa, dev), dtype=torch.float32))[:2], model.values(codes, sa)[:2])


def test_codes_and_scales_with_strides(dev):
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    rng = np.random.default_rng(9)
    m, n, k = 90, 150, 304
    (ac, asc), (bc, bsc) = _whole(rng, m, k, False), _whole(rng, n, k, True)
    want = model.values(ac, asc) @ model.values(bc, bsc).T
    a, sa = _put(ac, asc, dev)
    b, sb = _put(bc, bsc, dev)
    wide = torch.full((m, 3, k), 0x7F, dtype=torch.uint8, device=dev)  # NaN codes all around
    wide[:, 1] = a.view(torch.uint8)
    off = torch.full((m, k + 5), 0x7F, dtype=torch.uint8, device=dev)
    off[:, 5:] = a.view(torch.uint8)
    more = torch.full((m, 7), 255, dtype=torch.uint8, device=dev)
    more[:, 2:5] = sa
    for codes in (wide.view(torch.float8_e4m3fn)[:, 1], off.view(torch.float8_e4m3fn)[:, 5:],
                  a.view(torch.uint8).t().contiguous().view(torch.float8_e4m3fn).t()):
        for scales in (sa, more[:, 2:5], sa.t().contiguous().t()):
            got = fp8_matmul(codes, scales, b, sb, out_dtype=torch.float32)
            assert np.array_equal(_f64(got), want)


def test_gradients_of_a_linear_layer_are_products_of_the_same_weight(dev):
    from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize

    rng = np.random.default_rng(10)
    m, n, k = 203, 150, 330
    x, dy = (torch.from_numpy(rng.standard_normal((m, c))).to(torch.bfloat16).to(dev) for c in (k, n))
    w = torch.from_numpy(rng.standard_normal((n, k)) * 0.05).to(torch.bfloat16).to(dev)
    wv = model.values(*model.quantise(_f64(w), True))[:, :k]
    forth, back = fp8_quantize(w, square=True), fp8_quantize(w, square=True, transpose=True)
    assert np.array_equal(model.values(_bytes(back[0]), back[1].cpu().numpy())[:, :n], wv.T)
    dv = model.values(*model.quantise(_f64(dy)))[:, :n]
    dx = _f64(fp8_matmul(*fp8_quantize(dy), *back, out_dtype=torch.float32))
    assert (np.abs(dx - dv @ wv) <= n * 2.0**-23 * (np.abs(dv) @ np.abs(wv))).all()
    dt, xt = (model.values(*model.quantise(_f64(t).T))[:, :m] for t in (dy, x))
    dw = _f64(fp8_matmul(*fp8_quantize(dy, transpose=True), *fp8_quantize(x, transpose=True), out_dtype=torch.float32))
    assert dw.shape == (n, k) and (np.abs(dw - dt @ xt.T) <= m * 2.0**-23 * (np.abs(dt) @ np.abs(xt).T)).all()
    # against a difference of the layer itself, whose weight stays: y is linear in x's codes
    xq = fp8_quantize(x)
    y = _f64(fp8_matmul(*xq, *forth, out_dtype=torch.float32))
    xv = model.values(_bytes(xq[0]), xq[1].cpu().numpy())[:, :k]
    assert (np.abs(y - xv @ wv.T) <= k * 2.0**-23 * (np.abs(xv) @ np.abs(wv).T)).all()


def test_empty_sides(dev):
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_matmul, fp8_quantize

    none, some = torch.zeros(0, 64, device=dev), torch.zeros(5, 64, device=dev)
    a, b = fp8_quantize(none), fp8_quantize(some)
    assert a[0].shape == (0, 64) and a[1].shape == (0, 1) and fp8_quantize(none, transpose=True)[0].shape == (64, 0)
    assert fp8_matmul(*a, *b).shape == (0, 5) and fp8_matmul(*b, *a).shape == (5, 0)
    assert fp8_dequantize(*a).shape == (0, 64)
    assert torch.equal(fp8_matmul(*b, *b), torch.zeros(5, 5, device=dev, dtype=torch.bfloat16))
    # the weight's gradient of no rows, and a sum over nothing with a bias
    t = fp8_quantize(none, transpose=True)
    assert torch.equal(fp8_matmul(*t, *t, out_dtype=torch.float32), torch.zeros(64, 64, device=dev))
    assert torch.equal(fp8_matmul(*t, *t, bias=torch.arange(64, device=dev).float())[3], torch.arange(64, device=dev).bfloat16())


def test_refusals(dev):
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_matmul, fp8_quantize

    x = torch.zeros(8, 64, device=dev)
    a, s = fp8_quantize(x)
    with pytest.raises(RuntimeError, match=r"x must be \[rows, width\]"):
        fp8_quantize(x[0])
    with pytest.raises(RuntimeError, match="in bfloat16, float16 or float32"):
        fp8_quantize(x.double())
    with pytest.raises(RuntimeError, match="autograd"):
        fp8_quantize(x.clone().requires_grad_())
    with torch.no_grad():
        fp8_quantize(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="multiple of 16"):
        fp8_matmul(a[:, :40], s, a, s)
    with pytest.raises(RuntimeError, match="scales of b"):
        fp8_matmul(a, s, a, s[:3])
    with pytest.raises(RuntimeError, match="scales of a"):
        fp8_matmul(a, s.int(), a, s)
    with pytest.raises(RuntimeError, match=r"a is \[8, 64\], b \[8, 32\]"):
        fp8_matmul(a, s, a[:, :32], s)
    with pytest.raises(RuntimeError, match="bias must be"):
        fp8_matmul(a, s, a, s, bias=x[0])
    with pytest.raises(RuntimeError, match="out_dtype"):
        fp8_matmul(a, s, a, s, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        fp8_matmul(a.view(torch.uint8), s, a, s)
    with pytest.raises(RuntimeError, match="dtype must be"):
        fp8_dequantize(a, s, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="require GPU tensors"):
        fp8_matmul(a, s.cpu(), a, s)


def test_another_stream_and_replays(dev):
    """A captured quantisation and product over buffers whose contents change, and a call on a side stream."""
    from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize

    g = torch.Generator(device=dev).manual_seed(4)
    w = fp8_quantize(torch.randn(300, 520, generator=g, device=dev), square=True)
    for m in (5, 150):
        x = torch.zeros(m, 520, device=dev, dtype=torch.bfloat16)
        inputs = [torch.randn(m, 520, generator=g, device=dev).to(torch.bfloat16) for _ in range(4)]
        eager = [fp8_matmul(*fp8_quantize(i), *w) for i in inputs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = fp8_matmul(*fp8_quantize(inputs[0]), *w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(beside, eager[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8_matmul(*fp8_quantize(x), *w)
        for i, want in zip(inputs, eager):
            x.copy_(i)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_sizes_past_what_an_entry_point_counts(dev):
    """Views of one value: a column count that 32 bits would cut down to a small one is refused before anything is
    allocated."""
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_matmul, fp8_quantize

    n = 2**32 + 16
    x = torch.zeros(1, 1, device=dev)
    for shape in ((1, n), (n, 1)):
        for how in (dict(), dict(square=True), dict(transpose=True)):
            with pytest.raises(RuntimeError, match="rows or columns"):
                fp8_quantize(x.expand(shape), **how)
    codes = torch.zeros(1, 1, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    scale = torch.zeros(1, 1, dtype=torch.uint8, device=dev)
    wide, scales = codes.expand(1, n), scale.expand(1, -(-n // 128))
    with pytest.raises(RuntimeError, match="rows or columns"):
        fp8_dequantize(wide, scales)
    with pytest.raises(RuntimeError, match="rows or columns"):
        fp8_matmul(wide, scales, wide, scales)
    k = 2**22 + 16
    wide, scales = codes.expand(1, k), scale.expand(1, -(-k // 128))
    with pytest.raises(RuntimeError, match=f"sums of {k} terms"):
        fp8_matmul(wide, scales, wide, scales)


def test_more_rows_than_a_launch_of_tiles_has(dev):
    from sparsepr_amd.kernels.fp8 import fp8_quantize

    rows = 65535 * 128 + 100
    x = (torch.arange(rows, device=dev)[:, None] % 1021 - 500 + torch.arange(8, device=dev)).to(torch.bfloat16)
    codes, scales = (t.view(torch.uint8) for t in fp8_quantize(x))
    for part in (slice(0, 1000), slice(rows - 1000, rows)):
        c, s = (t.view(torch.uint8) for t in fp8_quantize(x[part].clone()))
        assert torch.equal(codes[part], c) and torch.equal(scales[part], s)
    with pytest.raises(RuntimeError, match="rows of 8"):
        fp8_quantize(x, square=True)


def test_one_row_on_more_columns_than_a_launch_of_few_rows_has(dev):
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    n = 2**27 + 5
    one = torch.full((1, 16), 0x38, dtype=torch.uint8, device=dev)  # 1.0
    scale = torch.full((1, 1), 127, dtype=torch.uint8, device=dev)
    b = torch.zeros(n, 16, dtype=torch.uint8, device=dev)
    b[-3:] = 0x38
    y = fp8_matmul(one.view(torch.float8_e4m3fn), scale, b.view(torch.float8_e4m3fn), scale.expand(n, 1))
    assert (y[0, -3:] == 16).all() and not y[0, :-3].any()


@pytest.mark.parametrize("m,n,k", [(64, 64, 640), (70, 100, 4496), (130, 700, 1296), (300, 1500, 8208), (77, 4096, 3984)])
def test_products_of_few_tiles_whose_waves_share_the_sum_are_exact(dev, m, n, k):
    """Odd and even counts of blocks between two groups of waves, more of them than a window of scales holds."""
    test_products_on_tiles_of_every_size_are_exact(dev, m, n, k)


def test_a_sum_in_parts_that_one_call_does_not_take(dev):
    """Columns of codes whose rows are further apart than an entry point takes: a sum of 2^22 + 272 terms as two."""
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    m, n, k, half = 40, 3, 2**22 + 272, 2**21
    g = torch.Generator(device=dev).manual_seed(5)
    a, b = (torch.randint(-1, 2, (r, k), generator=g, device=dev).to(torch.float8_e4m3fn) for r in (m, n))
    sa, sb = (torch.full((r, -(-k // 128)), 127, dtype=torch.uint8, device=dev) for r in (m, n))
    parts = [fp8_matmul(a[:, p], sa[:, s], b[:, p], sb[:, s], out_dtype=torch.float32)
             for p, s in ((slice(0, half), slice(0, half // 128)), (slice(half, k), slice(half // 128, None)))]
    assert torch.equal(parts[0] + parts[1], a.float() @ b.float().t())  # whole numbers below 2^24
    for last in (0, 16, 128):  # one row of them, narrow columns at the end
        p = slice(k - 128 - last, k - last)
        for rows in (slice(0, 1), slice(5, 8)):
            got = fp8_matmul(a[rows, p], sa[rows, :1], b[:, p], sb[:, :1], out_dtype=torch.float32)
            assert torch.equal(got, a[rows, p].float() @ b[:, p].float().t())


@pytest.mark.parametrize("fast", [False, True])
def test_more_rows_than_the_fastest_kernels_launch_takes(dev, fast):
    """2^22 tiles of 128 x 128, the kernel that such a shape would get by its time: 2^21 of 256 x 256 do it."""
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    m, n = 2**29, 65
    if torch.cuda.mem_get_info()[0] < 100 * 2**30:
        pytest.skip("needs 80 GB")
    a = torch.zeros(m, 16, dtype=torch.uint8, device=dev)
    a[-300:] = a[m // 2] = 0x38  # 1.0
    b = torch.full((n, 16), 0x38, dtype=torch.uint8, device=dev)
    scale = torch.full((1, 1), 127, dtype=torch.uint8, device=dev)
    y = fp8_matmul(a.view(torch.float8_e4m3fn), scale.expand(m, 1), b.view(torch.float8_e4m3fn), scale.expand(n, 1), fast_sums=fast)
    assert (y[-300:] == 16).all() and (y[m // 2] == 16).all()
    for i in (0, m // 4, m // 2 - 5000, m // 2 + 1, m - 5300):
        assert not y[i:i + 5000].any()
    del a, y
    torch.cuda.empty_cache()


def test_more_rows_than_one_launch_quantises(dev):
    """Rows with scales of their own: past 2^24 of them, packed and with a stride, and past 2^28 groups."""
    from sparsepr_amd.kernels.fp8 import fp8_quantize

    for rows, width, stride in ((2**24 + 1000, 16, 24), (2**24 - 1, 8, 8), (2**24, 8, 8), (2**28 + 5, 4, 0)):
        x = torch.arange(max(1, (rows if stride else 1) * stride // 8), device=dev)[:, None] % 1021 - 500 + torch.arange(8, device=dev)
        x = x.to(torch.bfloat16).flatten().as_strided((rows, width), (stride, 1))
        codes, scales = fp8_quantize(x)
        assert codes.shape == (rows, 16) and scales.shape == (rows, 1)
        for part in (slice(0, 100), slice(2**24 - 60, min(rows, 2**24 + 60)), slice(rows - 100, rows)):
            c, s = fp8_quantize(x[part].clone())
            assert torch.equal(codes[part].view(torch.uint8), c.view(torch.uint8)) and torch.equal(scales[part], s)
        if stride == 0:
            assert (codes.view(torch.uint8) == codes[0].view(torch.uint8)).all() and (scales == scales[0]).all()
    torch.cuda.empty_cache()
