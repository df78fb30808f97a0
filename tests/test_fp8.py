"""What stands in front of the attention, without a GPU: the 8-bit format's definition, the formulas of the
gradients against differences, and the refusals that the host gives."""

import numpy as np
import pytest
import torch

from tests import _fp8_model as model


def test_encoder_picks_the_nearest_code_and_the_smallest_scale():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((60, 300)) * np.exp(3 * rng.standard_normal((60, 1)))
    x[3] = 0.0
    for square in (False, True):
        codes, scales = model.quantise(x, square)
        assert codes.shape == (60, 304) and scales.shape == (1 if square else 60, 3)
        y = model.values(codes, scales)
        s = np.ldexp(1.0, (scales.repeat(60, 0) if square else scales).astype(int) - 127).repeat(128, 1)[:, :300]
        # half a step: 2^-4 of the value, of the smallest normal code's below it
        assert (np.abs(y[:, :300] - x) <= np.maximum(np.abs(x) * 2.0**-4, s * 2.0**-10)).all()
        assert (y[:, 300:] == 0).all()
        top = np.abs(model.blocks_of(x, square)).max((1, 3))
        e = np.ldexp(1.0, scales.astype(int) - 127)
        assert (top <= 448 * e).all() and ((top > 224 * e) | (scales == 1)).all()
        again = model.quantise(y, square)
        assert np.array_equal(model.values(*again), y)
    assert np.array_equal(model.encode(np.array([0.0, -0.0, 448.0, -448.0, 2.0**-9, 2.0**-10, 3 * 2.0**-10, 17.0, 19.0])),
                          np.array([0, 128, 126, 254, 1, 0, 2, 88, 90], np.uint8))
    assert model.scale_byte(np.array([0.0, 448.0, 448.1, 1e-45, np.inf, np.nan])).tolist() == [1, 127, 128, 1, 255, 255]


def test_torchs_codes_are_the_models():
    y = model.grid()
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.isnan(t), np.isnan(y)) and np.array_equal(t[~np.isnan(t)], y[~np.isnan(y)])


def test_gradient_formulas_against_differences():
    rng = np.random.default_rng(2)
    s, dy, w = rng.standard_normal((3, 10)), rng.standard_normal((3, 10)), rng.standard_normal(10)
    dsum, eps, h = rng.standard_normal((3, 10)), 0.03, 1e-6
    dx, dw = model.norm_backward(dy, s, w, dsum, eps)
    loss = lambda s, w: (model.norm(s, w, eps) * dy).sum() + (s * dsum).sum()  # noqa: E731
    for i in np.ndindex(s.shape):
        d = np.zeros(s.shape)
        d[i] = h
        assert abs((loss(s + d, w) - loss(s - d, w)) / (2 * h) - dx[i]) < 1e-7
    for i in range(10):
        d = np.zeros(10)
        d[i] = h
        assert abs((loss(s, w + d) - loss(s, w - d)) / (2 * h) - dw[i]) < 1e-7
    x, p = rng.standard_normal((1, 2, 3, 12)), rng.uniform(-9, 9, (1, 3, 2))
    f, axis = rng.uniform(0, 2, 4), np.array([0, 1, 1, 0])
    for pairs in ("interleaved", "halves"):
        g = rng.standard_normal(x.shape)
        back, _ = model.rotate(g, p, f, axis, pairs, inverse=True)
        for i in np.ndindex(x.shape):
            d = np.zeros(x.shape)
            d[i] = h
            diff = (model.rotate(x + d, p, f, axis, pairs)[0] - model.rotate(x - d, p, f, axis, pairs)[0]) * g
            assert abs(diff.sum() / (2 * h) - back[i]) < 1e-7


def test_rows_that_cancel_tell_full_sums_from_cut_ones():
    """What the GPU tests of the sums are built on: cut at 2^-13, nothing is left of products that are 2^-14 of the
    largest; fp32's 24 digits keep them all, and normal rows tell the cut from fp32 only by little."""
    rng = np.random.default_rng(4)
    a, b = (model.grid()[c] for c in model.cancelling(rng, 5, 7, 256))
    want = a @ b.T
    assert (want != 0).sum() > 25 and np.abs(want).max() <= 2.0**-2 * 224
    assert (cut := model.cut_product(a, b, 13)).shape == want.shape and not cut.any()
    assert np.array_equal(model.cut_product(a, b, 14), want)
    a, b = (model.values(*model.quantise(rng.standard_normal((r, 512)))) for r in (6, 9))
    off = np.abs(model.cut_product(a, b, 13) - a @ b.T)
    assert off.max() > 0 and (off <= 7 * 2.0**-13 * (np.abs(a[:, None]) * np.abs(b)).reshape(6, 9, -1, 8).max(-1).sum(-1)).all()


def test_products_entry_point_refuses_fast_sums_of_fp32_outputs():
    lib = _lib()
    st = lib.spr_fp8_matmul_ex(16, 64, 16, 1, 0, 16, 64, 16, 1, 0, 4, 4, 64, None, 0, 2, 1, 16, None)
    assert "fast sums are for outputs in 16 bits" in _refused(lib, st)


def _refused(lib, st):
    assert st in (1, 3)
    return lib.spr_last_error().decode()


def _lib():
    from sparsepr_amd import _lib

    return _lib.load()


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype 3"), (dict(width=0), "width 0"), (dict(width=16385), "width 16385"), (dict(n0=-1), "rows"),
    (dict(n0=1 << 20, n1=1 << 12), "too many rows"), (dict(eps=-1.0), "epsilon"), (dict(eps=float("nan")), "epsilon"),
    (dict(eps=float("inf")), "epsilon"), (dict(wd=1), "weights of dtype 1"), (dict(rd=1), "residual of dtype 1"),
    (dict(x=None), "null pointer"), (dict(sum=None), "null pointer"), (dict(out=4), "8-byte aligned"),
    (dict(s0=-8), "negative stride")])
def test_norm_refuses_bad_arguments_before_any_launch(kw, text):
    lib = _lib()
    a = dict(x=16, s0=64, n0=2, n1=3, width=64, dtype=0, rd=0, wd=0, eps=1e-6, out=16, scales=16, sum=16)
    a.update(kw)
    st = lib.spr_rms_norm(a["x"], a["s0"], 64, 16, 64, 64, a["n0"], a["n1"], a["width"], a["dtype"], a["rd"], 16, a["wd"],
                          a["eps"], a["out"], a["scales"], a["sum"], None)
    assert text in _refused(lib, st)


def test_empty_norms_are_no_work():
    assert _lib().spr_rms_norm(None, 0, 0, None, 0, 0, 0, 5, 64, 0, 0, None, 0, 1e-6, None, None, None, None) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=-1), "dtype -1"), (dict(sd=1), "sum of dtype 1"), (dict(width=20000), "width 20000"),
    (dict(eps=-1e-9), "epsilon"), (dict(wd=1), "weights of dtype 1"), (dict(dy=None), "null pointer"),
    (dict(ws=0), "workspace 0 < "), (dict(s0=-1), "negative stride"), (dict(at=8), "not 16-byte aligned")])
def test_norm_gradient_refuses_bad_arguments_before_any_launch(kw, text):
    lib = _lib()
    a = dict(dy=16, s0=64, width=64, dtype=0, sd=2, wd=0, eps=1e-6, ws=1 << 20, at=16)
    a.update(kw)
    st = lib.spr_rms_norm_backward(a["dy"], a["s0"], 64, 16, 64, 64, None, 0, 0, 2, 3, a["width"], a["dtype"], a["sd"], 16,
                                   a["wd"], a["eps"], 16, 16, a["at"], a["ws"], None)
    assert text in _refused(lib, st)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype 3"), (dict(rows=1 << 24), "rows of"), (dict(rows=-1), "rows of"),
    (dict(rows=8000000, width=1 << 14), "too many groups"), (dict(x=None), "null pointer"), (dict(codes=24), "16-byte aligned"),
    (dict(ld=-1), "negative stride")])
def test_quantisation_refuses_bad_arguments_before_any_launch(kw, text):
    lib = _lib()
    a = dict(x=16, ld=64, rows=4, width=64, dtype=0, codes=32)
    a.update(kw)
    assert text in _refused(lib, lib.spr_fp8_quantize(a["x"], a["ld"], a["rows"], a["width"], a["dtype"], 0, 0, a["codes"],
                                                      16, None))


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=5), "dtype 5"), (dict(width=40), "rows of 40"), (dict(rows=1 << 31), "rows of"), (dict(out=None), "null"),
    (dict(ld=72), "strides 72"), (dict(codes=40), "16-byte aligned"), (dict(rows=1 << 30, width=128), "too many values")])
def test_values_refuse_bad_arguments_before_any_launch(kw, text):
    lib = _lib()
    a = dict(codes=16, ld=64, rows=4, width=64, dtype=0, out=16)
    a.update(kw)
    assert text in _refused(lib, lib.spr_fp8_dequantize(a["codes"], a["ld"], 16, 1, 0, a["rows"], a["width"], a["dtype"],
                                                        a["out"], None))


@pytest.mark.parametrize("kw,text", [
    (dict(od=3), "output dtype 3"), (dict(bd=4), "bias dtype 4"), (dict(K=40), "sizes"), (dict(K=1 << 23), "sizes"),
    (dict(M=-1), "sizes"), (dict(M=1 << 31), "sizes"), (dict(K=0), "nothing to sum"), (dict(a=None), "null pointer"),
    (dict(a_ld=48), "row strides 48"), (dict(b_ld=72), "row strides 64, 72"), (dict(a=24), "16-byte aligned"),
    (dict(s_ld=-1), "negative scale stride"), (dict(M=1 << 30, N=1 << 16), "too many outputs"),
    (dict(M=1, N=1 << 29, K=16, a_ld=16, b_ld=16), "too many outputs"), (dict(M=1 << 22, N=1 << 22), "too many outputs")])
def test_product_refuses_bad_arguments_before_any_launch(kw, text):
    lib = _lib()
    a = dict(a=16, a_ld=64, b_ld=64, s_ld=1, M=4, N=4, K=64, bd=0, od=0)
    a.update(kw)
    st = lib.spr_fp8_matmul(a["a"], a["a_ld"], 16, a["s_ld"], 0, 16, a["b_ld"], 16, 1, 0, a["M"], a["N"], a["K"], 16,
                            a["bd"], a["od"], 16, None)
    assert text in _refused(lib, st)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype 3"), (dict(code=4), "position code 4"), (dict(dim=60), "head dim 60"), (dict(dim=1032), "head dim"),
    (dict(rotated=72), "72 rotated dims"), (dict(rotated=12), "12 rotated dims"), (dict(axes=0), "0 axes"),
    (dict(axes=17), "17 axes"), (dict(batch=-1), "bad size"), (dict(q=None), "null pointer"), (dict(pos=None), "null pointer"),
    (dict(batch=1 << 30, tokens=1 << 30), "too many rows"), (dict(batch=1 << 10, tokens=1 << 20), "too many rows")])
def test_rotation_refuses_bad_arguments_before_any_launch(kw, text):
    lib = _lib()
    a = dict(q=16, dtype=0, batch=2, tokens=3, dim=64, rotated=64, pos=16, code=0, axes=3)
    a.update(kw)
    st = lib.spr_axial_rope(a["q"], 64, 64, 64, 2, 16, 64, 64, 64, 1, a["dtype"], a["batch"], a["tokens"], a["dim"],
                            a["rotated"], a["pos"], a["code"], 0, a["axes"], 16, 16, 0, 0, 16, 16, None)
    assert text in _refused(lib, st)


def test_functions_refuse_host_tensors_and_host_tables_are_right():
    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope, grid_positions
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_matmul, fp8_quantize
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_backward, rms_norm_fp8

    x = torch.zeros(4, 64)
    codes, scales = x.to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8)
    q, f, i = torch.zeros(1, 2, 4, 64), torch.zeros(32, dtype=torch.float64), torch.zeros(32, dtype=torch.int32)
    for call in (lambda: rms_norm(x), lambda: rms_norm_fp8(x), lambda: rms_norm_backward(x, x), lambda: fp8_quantize(x),
                 lambda: fp8_dequantize(codes, scales), lambda: fp8_matmul(codes, scales, codes, scales),
                 lambda: axial_rope(q, q, torch.zeros(4, 1), f, i)):
        with pytest.raises(RuntimeError, match="require GPU tensors"):
            call()
    f, a = axial_frequencies((4, 0, 6), theta=100.0, device="cpu")
    assert a.tolist() == [0, 0, 2, 2, 2]
    assert np.allclose(f.numpy(), [1.0, 0.1, 1.0, 100.0 ** (-2 / 6), 100.0 ** (-4 / 6)], rtol=1e-15)
    p = grid_positions(2, 3, 4, first=(5, 0, 1), device="cpu")
    assert p.shape == (24, 3) and p.dtype == torch.int32
    assert p[0].tolist() == [5, 0, 1] and p[1].tolist() == [5, 0, 2] and p[4].tolist() == [5, 1, 1] and p[23].tolist() == [6, 2, 4]
    for bad in (dict(axis_dims=(3, 4)), dict(axis_dims=(4,), theta=0.0), dict(axis_dims=(-2,))):
        with pytest.raises(RuntimeError, match="axial RoPE"):
            axial_frequencies(bad.pop("axis_dims"), device="cpu", **bad)


def test_lost_gradients_are_found():
    from torch.autograd import forward_ad

    from sparsepr_amd.kernels.fp8 import no_gradient

    x = torch.ones(2, 3)
    leaf = x.clone().requires_grad_()
    no_gradient("call", x, None, torch.zeros(2, dtype=torch.uint8))
    for lost in (leaf, leaf[1:], leaf.to(torch.float8_e4m3fn)):
        with pytest.raises(RuntimeError, match="call: autograd does not record"):
            no_gradient("call", x, lost)
    with torch.no_grad():
        no_gradient("call", leaf)
    with forward_ad.dual_level():
        no_gradient("call", x, torch.zeros(2, dtype=torch.uint8))
        dual = forward_ad.make_dual(x, x)
        for lost in (dual, dual[1:], dual.to(torch.float8_e4m3fn)):
            with pytest.raises(RuntimeError, match="call: autograd's forward mode"):
                no_gradient("call", lost)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                no_gradient("call", x, lost)
        no_gradient("call", forward_ad.unpack_dual(dual).primal)
