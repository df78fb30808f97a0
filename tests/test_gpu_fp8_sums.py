"""The 8-bit product on every kernel that its rule picks: how it adds, what it reads and where it writes.

With sums in fp32 (the default) rows are built so that the 8-bit matrix instruction would lose every digit of the
result: of eight neighbouring products one is 2^12, which the next eight take off again, and seven are 2^-2, 2^-14 of
it.  All partial sums are multiples of 2^-2 below 2^12 K / 16, so fp32 holds them in any order up to K = 2^14 and the
output is the exact one, rounded once.

With fast sums an output is off by the seven other products' cut, 7 * 2^-13 of each eight's largest product, by K
additions in fp32 of 2^-23 of the sum of magnitudes each, and by half a step of its type."""

import numpy as np
import pytest
import torch

from tests import _fp8_model as model

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {t: torch.finfo(t).eps / 2 for t in DT.values()}
# Tiles of 256 x 256, 128 x 128, 64 x 128 (two sizes, the first with sums in fp32 128 x 128), 64 x 64 (two, the second
# with sums in fp32 two groups of waves), two groups (two), few rows (16, 32 and, with sums in fp32, 64); each
# with a last block and last tiles that are not whole.
SIZES = [(4000, 3500, 272), (2100, 2300, 784), (500, 5000, 4240), (700, 1800, 528), (513, 260, 400), (90, 5000, 8208),
         (300, 1500, 8208), (70, 100, 4496), (1, 500, 4112), (17, 33, 5136), (60, 32, 12048)]


def _f64(t):
    return t.double().cpu().numpy()


def _put(codes, dev):
    return torch.from_numpy(codes).to(dev).view(torch.float8_e4m3fn)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_what_cancels_leaves_the_small_products(dev, m, n, k):
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    rng = np.random.default_rng(m + k)
    a, b = (_put(c, dev) for c in model.cancelling(rng, m, n, k))
    sa = torch.from_numpy(np.repeat(rng.integers(126, 129, (m, 1)), -(-k // 128), 1).astype(np.uint8)).to(dev)
    sb = torch.full((-(-n // 128), -(-k // 128)), 127, dtype=torch.uint8, device=dev)
    want = (a.float() * torch.exp2(sa[:, :1].float() - 127)) @ b.float().t()  # exact in any order
    assert (want != 0).any()
    for out in DT.values():
        assert torch.equal(fp8_matmul(a, sa, b, sb, out_dtype=out), want.to(out))


@pytest.mark.parametrize("out", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_fast_sums_lose_what_the_instruction_cuts_and_no_more(dev, out, m, n, k):
    """At 24 rows and 40 columns, the last ones among them."""
    from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize

    g = torch.Generator(device=dev).manual_seed(k)
    x = torch.randn(m, k, generator=g, device=dev) * torch.exp(torch.randn(k, generator=g, device=dev))
    a, b = fp8_quantize(x), fp8_quantize(torch.randn(n, k, generator=g, device=dev) * 0.03, square=True)
    bias = torch.randn(n, generator=g, device=dev)
    got = fp8_matmul(*a, *b, bias=bias, out_dtype=DT[out], fast_sums=True)
    assert torch.equal(got, fp8_matmul(*a, *b, bias=bias, out_dtype=DT[out], fast_sums=True))  # the same bits again
    rows, cols = (np.unique(np.r_[np.linspace(0, s - 1, c).astype(int), s - 1]) for s, c in ((m, 24), (n, 40)))
    av = model.values(a[0].view(torch.uint8).cpu().numpy(), a[1].cpu().numpy())[rows]
    bv = model.values(b[0].view(torch.uint8).cpu().numpy(), b[1].cpu().numpy())[cols]
    bias = _f64(bias)[cols]
    want, bound = av @ bv.T + bias, k * 2.0**-23 * (np.abs(av) @ np.abs(bv).T + np.abs(bias)) + 2.0**-25
    bound += HALF[DT[out]] * np.abs(want)
    for i in range(0, k, 8):
        bound += 7 * 2.0**-13 * (np.abs(av[:, None, i:i + 8]) * np.abs(bv[None, :, i:i + 8])).max(-1)
    assert (np.abs(_f64(got)[rows][:, cols] - want) <= bound).all()


def test_fast_sums_are_for_outputs_in_16_bits(dev):
    from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize
    from sparsepr_amd.qkv_projection import QKVProjection

    a = fp8_quantize(torch.ones(8, 64, device=dev))
    with pytest.raises(RuntimeError, match="fast sums are for outputs in 16 bits"):
        fp8_matmul(*a, *a, out_dtype=torch.float32, fast_sums=True)
    g = torch.Generator(device=dev).manual_seed(1)
    w, x = (torch.randn(192, 64, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    fast, full = (QKVProjection(w, heads=1, axis_dims=(0,), fast_sums=f) for f in (True, False))
    codes = fp8_quantize(w, square=True)
    for front in (fast, full):
        from sparsepr_amd.kernels.rms_norm import rms_norm_fp8

        v = fp8_matmul(*rms_norm_fp8(x), *codes, fast_sums=front is fast)[:, 128:]
        assert torch.equal(front(x[None], torch.zeros(192, 1, device=dev))[2][0, 0], v)


@pytest.mark.parametrize("byte", [0, 1, 2, 3, 246, 247, 254, 255])
def test_values_are_multiplied_as_bf16_holds_them(dev, byte):
    """All codes at the ends of the scales' range, by ones: what fp8_dequantize gives, exact for bytes 3 to 246."""
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_matmul

    for n in (16, 200):
        codes = torch.zeros(256, 128, dtype=torch.uint8, device=dev)
        codes[:, 3] = torch.arange(256, device=dev)
        codes = codes.view(torch.float8_e4m3fn)
        scales = torch.full((256, 1), byte, dtype=torch.uint8, device=dev)
        one = torch.zeros(n, 128, device=dev)
        one[:, 3] = 1
        one_scale = torch.full((n, 1), 127, dtype=torch.uint8, device=dev)
        for r in (slice(0, 256), slice(100, 140)):
            got = fp8_matmul(codes[r], scales[r], one.to(torch.float8_e4m3fn), one_scale, out_dtype=torch.float32)
            want = fp8_dequantize(codes[r], scales[r], dtype=torch.bfloat16)[:, 3:4].float().expand(-1, n)
            assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(got.isnan(), want.isnan())
            full = fp8_dequantize(codes[r], scales[r], dtype=torch.float32)[:, 3:4].expand(-1, n)
            assert not 3 <= byte <= 246 or torch.equal(got.nan_to_num(7.0), full.nan_to_num(7.0))


WAYS = [(out, fast) for out in DT.values() for fast in (False, True) if not (fast and out is torch.float32)]


def _spread(scales, rows, k):
    """The scales of every value, in 64 bits."""
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    s = s if len(scales) == rows else s.repeat_interleave(128, 0)[:rows]
    return s.repeat_interleave(128, 1)[:, :k]


@pytest.mark.parametrize("squares", [(False, True), (True, False)])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_rows_and_scales_inside_others(dev, m, n, k, squares):
    """Codes and scales as slices of larger tensors that hold NaN in front of, behind and between them: whole numbers up
    to 4 at scales up to 4, whose sums are exact in any order."""
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    g = torch.Generator(device=dev).manual_seed(n)
    sides = []
    for rows, square, gap in ((m, squares[0], 48), (n, squares[1], 16)):
        whole = torch.full((rows + 3, k + gap + 16), 0x7F, dtype=torch.uint8, device=dev)
        codes = torch.randint(-2, 3, (rows, k), generator=g, device=dev).to(torch.float8_e4m3fn)
        whole[2:-1, 16:16 + k] = codes.view(torch.uint8)
        blocks, groups = -(-k // 128), -(-rows // 128) if square else rows
        around = torch.full((groups + 3, blocks + 5), 255, dtype=torch.uint8, device=dev)
        around[1:-2, 3:-2] = torch.randint(126, 129, (groups, blocks), generator=g, device=dev)
        sides.append((whole.view(torch.float8_e4m3fn)[2:-1, 16:16 + k], around[1:-2, 3:-2]))
    (a, sa), (b, sb) = sides
    want = (a.float() * _spread(sa, m, k).float()) @ (b.float() * _spread(sb, n, k).float()).t()
    for out, fast in WAYS:
        assert torch.equal(fp8_matmul(a, sa, b, sb, out_dtype=out, fast_sums=fast), want.to(out))


@pytest.mark.parametrize("m,n,k", SIZES)
def test_nan_and_the_ends_of_the_scales(dev, m, n, k):
    """A NaN code or scale reaches its row or column and nothing else; scales of 2^127 and 2^-127 meet.  (Results below
    2^-100 are flushed or not.)"""
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    g = torch.Generator(device=dev).manual_seed(k)
    blocks = -(-k // 128)
    (a, sa), (b, sb) = ((torch.randint(0, 3, (r, k), generator=g, device=dev).to(torch.float8_e4m3fn).view(torch.uint8),
                         torch.full((r, blocks), 127, dtype=torch.uint8, device=dev)) for r in (m, n))
    one = 0x38
    a[0] = b[:2] = one
    sa[0], sb[1] = 254, 0  # 2^127 and 2^-127
    if m > 1:
        a[1], sa[1], sb[0] = one, 1, 253  # 2^-126 and 2^126
    if m > 4:
        a[m - 1, k - 1], sa[m - 2, blocks - 1], a[m // 2, 0] = 0x7F, 255, 0xFF
    b[n - 1, k - 1], sb[n - 2, blocks - 1], b[n // 2, 17] = 0xFF, 255, 0x7F
    a, b = a.view(torch.float8_e4m3fn), b.view(torch.float8_e4m3fn)
    want = (a.double() * _spread(sa, m, k)) @ (b.double() * _spread(sb, n, k)).t().contiguous()
    assert want[0, 1] == k and want.isnan().any(0).sum() == (n if m > 4 else 3)
    low = want.abs() < 2.0**-100
    for out, fast in WAYS:
        got = fp8_matmul(a, sa, b, sb, out_dtype=out, fast_sums=fast)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(torch.where(low, 0, got).nan_to_num(7.0, 9.0), torch.where(low, 0, want).to(out).nan_to_num(7.0, 9.0))
        assert (got[low].double().abs() <= 2.0**-99).all()


@pytest.mark.parametrize("m,n", [(32900, 4112), (32771, 4099)])
def test_outputs_that_the_caches_do_not_hold(dev, m, n):
    """Above 256 MB in 16 bits, every value of them, rows that start on 16 bytes or anywhere."""
    from sparsepr_amd.kernels.fp8 import fp8_matmul

    g, k = torch.Generator(device=dev).manual_seed(m), 272
    a, b = (torch.randint(-2, 3, (r, k), generator=g, device=dev).to(torch.float8_e4m3fn) for r in (m, n))
    sa, sb = (torch.randint(126, 129, (r, 3), generator=g, device=dev).to(torch.uint8) for r in (m, -(-n // 128)))
    want = (a.float() * _spread(sa, m, k).float()) @ (b.float() * _spread(sb, n, k).float()).t()
    assert m * n * 2 > 256 << 20
    for out, fast in WAYS:
        assert torch.equal(fp8_matmul(a, sa, b, sb, out_dtype=out, fast_sums=fast), want.to(out))
