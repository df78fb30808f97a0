"""The norm of the hidden rows, its 8-bit output and its gradient on the GPU against the formulas in 64 bits.

Errors in fp32: a sum of C squares, 32 terms a lane in a chain and at most 16 joins, is off by at most 48 half
steps (2^-24) of itself, its root by half of that; with the division, the root and the two products a value is off by
at most 32 * 2^-24.  Then half a step of the output's type."""

# A lane's chain is one or two squares now and the roundings of the products are carried along, so that the bound above is
# wide; test_an_output_is_rounded_once holds what those roundings leave.
import numpy as np
import pytest
import torch

from tests import _fp8_model as model

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {t: torch.finfo(t).eps / 2 for t in DT.values()}
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-126}
F32 = 2.0**-24
WIDTHS = [1, 7, 16, 64, 100, 128, 129, 500, 512, 1111, 2048, 2050, 5120, 8192, 9000, 16384]


def _f64(t):
    return t.double().cpu().numpy()


def _x(seed, shape, dtype, dev, spread=1.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[-1])) * np.exp(rng.standard_normal((*shape[:-1], 1)))
    return torch.from_numpy(x).to(dtype).to(dev)


def _near(got, want, dtype, rel=32 * F32):
    got = _f64(got)
    bound = np.abs(want) * (HALF[dtype] + rel) * (1 + 1e-6) + TINY[dtype]
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,stream,wd", [("bf16", "bf16", "bf16"), ("bf16", "fp32", "fp32"), ("fp16", "fp16", "fp32"),
                                            ("fp16", "fp32", "fp16"), ("fp32", "fp32", "fp32"), ("bf16", None, None)])
def test_norm_and_sum(dev, width, dtype, stream, wd):
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_fp8

    x = _x(width, (37, width), DT[dtype], dev)
    w = None if wd is None else (1 + 0.3 * torch.randn(width, generator=torch.Generator().manual_seed(1))).to(DT[wd]).to(dev)
    res = None if stream is None else _x(width + 1, (37, width), DT[stream], dev)
    s = x
    if res is None:
        y, codes, scales = rms_norm(x, w), *rms_norm_fp8(x, w)
    else:
        y, s = rms_norm(x, w, residual=res)
        codes, scales, again = rms_norm_fp8(x, w, residual=res)
        assert s.dtype == res.dtype and torch.equal(s, again)
        _near(s, _f64(x) + _f64(res), s.dtype, rel=F32)
    want = model.norm(_f64(s), 1.0 if w is None else _f64(w), 1e-6)
    assert y.dtype == x.dtype and y.shape == x.shape
    _near(y, want, y.dtype)
    # 8 bits: the scale that the unrounded row gives, up to the fp32 errors at a border, and half a step
    blocks = -(-width // 128)
    assert codes.shape == (37, -(-width // 16) * 16) and scales.shape == (37, blocks)
    sc = scales.cpu().numpy()
    top = np.abs(model.blocks_of(want, False)).max((1, 3))
    e = np.ldexp(1.0, sc.astype(int) - 127)
    assert (top <= 448 * e * (1 + 32 * F32)).all() and ((top >= 224 * e * (1 - 32 * F32)) | (sc == 1)).all()
    got = model.values(codes.view(torch.uint8).cpu().numpy(), sc)
    assert (got[:, width:] == 0).all()
    unit = e.repeat(128, 1)[:, :width]
    assert (np.abs(got[:, :width] - want) <= np.maximum(np.abs(want) * 2.0**-4, unit * 2.0**-10) * (1 + 1e-5)).all()


def test_the_8_bit_output_is_the_quantised_norm(dev):
    """In fp32, where the norm's output is unrounded: the same bytes."""
    from sparsepr_amd.kernels.fp8 import fp8_quantize
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_fp8

    for width in (100, 640, 1111, 5120):
        x = _x(width, (50, width), torch.float32, dev)
        codes, scales = rms_norm_fp8(x)
        want = fp8_quantize(rms_norm(x))
        assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])


def test_rows_with_strides_and_leading_dims(dev):
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_backward, rms_norm_fp8

    b, t, h, d = 2, 9, 5, 64
    qkv = _x(3, (b, t, 3 * h * d), torch.bfloat16, dev)
    q = qkv[..., h * d: 2 * h * d].unflatten(-1, (h, d))  # [B, T, H, D], rows of one token side by side
    res = _x(4, (b, h, t, d), torch.bfloat16, dev).transpose(1, 2)
    for x, r in ((q, None), (q, res), (res, q), (q.transpose(1, 2), res.transpose(1, 2)), (q[..., 1:], res[..., :-1]),
                 (qkv[:, ::2, 3:200], None), (q[0, 0, 0], None), (q[:, :, :1].expand(b, t, h, d), q), (q[..., ::2], None)):
        xc, rc = x.contiguous(), None if r is None else r.contiguous()
        got, want = rms_norm(x, residual=r), rms_norm(xc, residual=rc)
        for g, w in zip(got if r is not None else [got], want if r is not None else [want]):
            assert g.shape == x.shape and torch.equal(g, w)
        got, want = rms_norm_fp8(x, residual=r), rms_norm_fp8(xc, residual=rc)
        assert all(torch.equal(g.view(torch.uint8), w.view(torch.uint8)) for g, w in zip(got, want))
        w = torch.ones(x.shape[-1], device=dev)
        dy = x if r is None else r
        got, want = rms_norm_backward(dy, x, w, dsum=x), rms_norm_backward(dy.contiguous(), xc, w, dsum=xc)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_zero_rows_infinities_and_epsilon(dev):
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_fp8

    for width in (40, 300, 3000):
        x = torch.randn(6, width, generator=torch.Generator().manual_seed(5))
        x[0], x[1] = 0.0, 1e-12
        x[2, 1], x[3, 2] = float("inf"), float("nan")
        x = x.to(dev)
        y = _f64(rms_norm(x, epsilon=1e-6))
        assert (y[0] == 0).all() and (np.abs(y[1] - 1e-9) < 1e-14).all()
        assert np.isnan(y[2, 1]) and (np.delete(y[2], 1) == 0).all() and np.isnan(y[3]).all()  # inf / inf; x / inf
        assert np.isfinite(y[4:]).all()
        assert np.isnan(_f64(rms_norm(x, epsilon=0.0))[0]).all()  # 0 / 0
        codes, scales = rms_norm_fp8(x)
        v = model.values(codes.view(torch.uint8).cpu().numpy(), scales.cpu().numpy())
        assert np.isnan(v[2, : min(128, v.shape[1])]).all() and np.isnan(v[3]).all() and np.isfinite(v[[0, 1, 4, 5]]).all()


@pytest.mark.parametrize("width", [1, 16, 100, 128, 500, 640, 2048, 2051, 5120, 8192, 12000])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("dtype,stream,wd,given", [("bf16", "bf16", "bf16", True), ("bf16", "fp32", "fp32", True),
                                                  ("fp16", "fp16", "fp32", False), ("fp16", "fp32", "fp16", True),
                                                  ("fp32", "fp32", "fp32", True), ("bf16", "bf16", None, False)])
def test_gradient(dev, width, rows, dtype, stream, wd, given):
    _gradient(dev, width, rows, dtype, stream, wd, given)


@pytest.mark.parametrize("width,rows", [(128, 40003), (640, 9001), (2560, 3001), (9000, 700)])
def test_gradient_of_many_rows(dev, width, rows):
    _gradient(dev, width, rows, "bf16", "fp32", "bf16", True)


def _gradient(dev, width, rows, dtype, stream, wd, given):
    from sparsepr_amd.kernels.rms_norm import rms_norm_backward

    dy = _x(width, (rows, width), DT[dtype], dev, 0.3)
    s = _x(width + 1, (rows, width), DT[stream], dev)
    dsum = _x(width + 2, (rows, width), DT[stream], dev, 0.3) if given else None
    w = None if wd is None else (1 + 0.3 * torch.randn(width, generator=torch.Generator().manual_seed(1))).to(DT[wd]).to(dev)
    dx, dw = rms_norm_backward(dy, s, w, dsum=dsum, epsilon=1e-5)
    y64, s64, w64 = _f64(dy), _f64(s), np.ones(width) if w is None else _f64(w)
    d64 = 0.0 if dsum is None else _f64(dsum)
    want_x, want_w = model.norm_backward(y64, s64, w64, d64, 1e-5)
    # what cancels in dx: each term is off by 96 half steps at most (two sums, their products)
    r = 1.0 / np.sqrt((s64 * s64).mean(-1, keepdims=True) + 1e-5)
    g = np.abs(y64 * w64)
    size = r * (g + np.abs(s64) * r * r * (g * np.abs(s64)).mean(-1, keepdims=True)) + np.abs(d64)
    assert dx.dtype == s.dtype
    assert (np.abs(_f64(dx) - want_x) <= 96 * F32 * size + HALF[dx.dtype] * np.abs(want_x) + TINY[dx.dtype]).all()
    if w is None:
        assert dw is None
    else:
        terms = np.abs(y64 * s64 * r).sum(0)
        assert dw.dtype == torch.float32 and (np.abs(_f64(dw) - want_w) <= (rows + 64) * F32 * terms + 1e-30).all()
        again = rms_norm_backward(dy, s, w, dsum=dsum, epsilon=1e-5)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_gradient_against_differences_of_the_norm_itself(dev):
    """Central differences of the fp32 norm along random directions: (y(s + h d) - y(s - h d)) . dy / 2 h is the
    gradient along d up to h^2 terms and 2^-21 |y| |dy| / h of rounding."""
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_backward

    g = torch.Generator(device=dev).manual_seed(6)
    for width in (96, 700):
        s, dy, d = (torch.randn(8, width, generator=g, device=dev) for _ in range(3))
        w = 1 + 0.3 * torch.randn(width, generator=g, device=dev)
        dx, dw = rms_norm_backward(dy, s, w)
        h = 2.0**-7
        diff = ((rms_norm(s + h * d, w).double() - rms_norm(s - h * d, w).double()) * dy.double()).sum(-1) / (2 * h)
        along = (dx.double() * d.double()).sum(-1)
        scale = dy.double().norm(dim=-1) * d.double().norm(dim=-1)
        assert ((diff - along).abs() <= scale * (h * h + 2.0**-21 / h)).all()
        dwd = torch.randn(width, generator=g, device=dev)
        diff = ((rms_norm(s, w + h * dwd).double() - rms_norm(s, w - h * dwd).double()) * dy.double()).sum() / (2 * h)
        assert abs(diff - (dw.double() * dwd.double()).sum()) <= 2.0**-21 / h * (dy.double().abs() * 5).sum()


def test_empty_and_refused(dev):
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_backward, rms_norm_fp8

    x = torch.zeros(4, 32, device=dev)
    none = x[:0]
    assert rms_norm(none).shape == (0, 32) and rms_norm_fp8(none)[1].shape == (0, 1)
    dx, dw = rms_norm_backward(none, none, x[0])
    assert dx.shape == (0, 32) and torch.equal(dw, torch.zeros(32, device=dev))
    for bad, text in [(lambda: rms_norm(x.double()), "in bfloat16, float16 or float32"), (lambda: rms_norm(x[:, :0]), "width 0"),
                      (lambda: rms_norm(torch.zeros(1, 16385, device=dev)), "width 16385"),
                      (lambda: rms_norm(x, x[0, :5]), "weight must be"), (lambda: rms_norm(x, x[0].half()), "weight must be"),
                      (lambda: rms_norm(x, residual=x[:2]), "residual must be"),
                      (lambda: rms_norm(x, residual=x.half()), "residual must be"),
                      (lambda: rms_norm(x, epsilon=float("nan")), "epsilon"), (lambda: rms_norm(x, epsilon=-1.0), "epsilon"),
                      (lambda: rms_norm(x, x[0].clone().requires_grad_()), "autograd"),
                      (lambda: rms_norm_backward(x, x[:2]), "s must be"),
                      (lambda: rms_norm_backward(x.half(), x, dsum=x.half()), "dsum must be"),
                      (lambda: rms_norm_backward(x, x.half()), "s must be"),
                      (lambda: rms_norm(x, residual=x.cpu()), "require GPU tensors")]:
        with pytest.raises(RuntimeError, match=text):
            bad()


def test_replays_and_another_stream(dev):
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_backward

    g = torch.Generator(device=dev).manual_seed(7)
    x, r = torch.zeros(200, 640, device=dev), torch.zeros(200, 640, device=dev)
    w = torch.randn(640, generator=g, device=dev)
    pairs = [(torch.randn(200, 640, generator=g, device=dev), torch.randn(200, 640, generator=g, device=dev)) for _ in range(4)]

    def step(x, r):
        y, s = rms_norm(x, w, residual=r)
        return y, s, *rms_norm_backward(y, s, w, dsum=s)

    eager = [step(*p) for p in pairs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = step(*pairs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(beside, eager[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, r)
    for p, want in zip(pairs, eager):
        x.copy_(p[0]), r.copy_(p[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_more_rows_than_an_entry_point_counts(dev):
    """Views of one row: 2^32 + 8 rows, which 32 bits would cut down to 8, are refused before anything is allocated."""
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_backward, rms_norm_fp8

    x = torch.zeros(1, 16, device=dev).expand(2**32 + 8, 16)
    for call in (rms_norm, rms_norm_fp8, lambda t: rms_norm_backward(t, t)):
        with pytest.raises(RuntimeError, match="too many rows"):
            call(x)


@pytest.mark.parametrize("scale", [2.0**-66, 2.0**-60, 2.0**56])
@pytest.mark.parametrize("width", [64, 300, 2000])
def test_gradient_of_very_small_and_large_rows(dev, width, scale):
    """With no epsilon, where 1 / mean(s^2) is outside of fp32's range: at 2^-66 a square is about 2^-132, a subnormal
    that is off by 2^-150, so the sum by 2^-18 of itself, the root by half and its cube by three halves of that."""
    from sparsepr_amd.kernels.rms_norm import rms_norm_backward

    dy = _x(width, (20, width), torch.float32, dev, 0.3)
    g = torch.Generator(device=dev).manual_seed(3)
    s = (1 + torch.rand(20, width, generator=g, device=dev)) * scale * torch.where(torch.rand(20, width, generator=g, device=dev) < 0.5, 1, -1)
    w = torch.linspace(0.5, 1.5, width, device=dev)
    dx, dw = rms_norm_backward(dy, s, w, epsilon=0.0)
    y64, s64, w64 = _f64(dy), _f64(s), _f64(w)
    want_x, want_w = model.norm_backward(y64, s64, w64, 0.0, 0.0)
    r = 1.0 / np.sqrt((s64 * s64).mean(-1, keepdims=True))
    g = np.abs(y64 * w64)
    size = r * (g + np.abs(s64) * r * r * (g * np.abs(s64)).mean(-1, keepdims=True))
    low = 2.0**-17 if scale < 2.0**-63 else 0.0
    assert (np.abs(_f64(dx) - want_x) <= (97 * F32 + low) * size).all()
    assert (np.abs(_f64(dw) - want_w) <= (84 * F32 + low) * np.abs(y64 * s64 * r).sum(0)).all()


@pytest.mark.parametrize("width", [1, 16, 100, 128, 300, 512, 640, 2050, 5120, 16384])
def test_an_output_is_rounded_once(dev, width):
    """Whole numbers up to 8, whose squares add up exactly: the root is then 64 bits, and what is left is the rounding
    of s r w to fp32, at most half a step of the output (2^-44 of it more, from the root's and the products' low parts)."""
    from sparsepr_amd.kernels.rms_norm import rms_norm

    rng = np.random.default_rng(width)
    s = torch.from_numpy(rng.integers(1, 9, (60, width)) * rng.choice([-1.0, 1.0], (60, width)))
    w = torch.from_numpy(rng.uniform(0.5, 2.0, width).astype(np.float32))
    want = model.norm(_f64(s), _f64(w), 2.0**-20)
    half = np.spacing(np.abs(want).astype(np.float32)).astype(np.float64) / 2
    got = _f64(rms_norm(s.float().to(dev), w.to(dev), epsilon=2.0**-20))
    assert (np.abs(got - want) <= half + 2.0**-44 * np.abs(want)).all()
    # a residual of the same numbers: the sum is exact too
    y, total = rms_norm(torch.zeros(60, width, dtype=torch.float16, device=dev), w.to(dev), residual=s.half().to(dev), epsilon=2.0**-20)
    assert torch.equal(total.cpu(), s.half())
    assert (np.abs(_f64(y) - want) <= (HALF[torch.float16] + F32) * np.abs(want) * (1 + 2.0**-10)).all()
